"""The plain operator set with an 8-bit cache, page copies and token scores: for the engine's host side without a GPU."""
from __future__ import annotations

import numpy as np
import torch

from plain_kv8 import PlainCache8
from torch_ops import TorchOps


class TorchOps8(TorchOps):
    def rope_kv8_write(self, qkv, positions, inv_freq, rot, slots, codes, words, nq, nkv, d, page_size):
        own = qkv.clone()
        self.rope_kv_write(own, positions, inv_freq, rot, None, None, nq, nkv, d, page_size)
        qkv[:, :nq * d] = own[:, :nq * d]
        kv = own[:, nq * d:].reshape(-1, 2, nkv, d)
        for t, s in enumerate(slots.tolist()):
            if s < 0:
                continue
            page, off, b = s // page_size, s % page_size, s % page_size // 16
            cell = PlainCache8(nkv, d, page_size)
            first = page * page_size + b * 16
            for o in range(off % 16):           # what the block's tokens before this one stand for
                cell.blocks.setdefault(first // 16, {})[o] = self._value(codes, words, page, b * 16 + o)[0]
            cell.write(kv[t:t + 1], [s])
            e = cell.exponent(first // 16)
            if off % 16:
                e = np.maximum(e, (words[page, :, b].T & 255).numpy())
            step = np.ldexp(1.0, e - 133)[..., None]
            for o, x in cell.blocks[first // 16].items():
                u = np.where(e[..., None] > 0, np.floor(np.nan_to_num(x, posinf=0, neginf=0) / step) + 128, 128)
                codes[page, :, :, b * 16 + o] = torch.from_numpy(u).to(torch.uint8)
            words[page, :, b] = torch.from_numpy(e.T.astype(np.int32))

    @staticmethod
    def _value(codes, words, page, off):
        e = (words[page, :, off // 16].T & 255).numpy()[..., None]
        v = np.where(e > 0, (codes[page, :, :, off].numpy().astype(np.float64) - 127.5) * np.ldexp(1.0, e - 133), 0.0)
        return v, e

    def _expanded(self, codes, words):
        e = (words & 255).permute(0, 3, 1, 2).repeat_interleave(16, -1)[..., None].double()
        return torch.where(e > 0, (codes.double() - 127.5) * torch.exp2(e - 133), torch.zeros((), dtype=torch.float64)).float()

    def paged_attention8(self, q, codes, words, block_table, tok_req, positions, nq, nkv, d, page_size, scale, window=0, hints=None):
        return self.paged_attention(q, self._expanded(codes, words), block_table, tok_req, positions, nq, nkv, d, page_size, scale, window=window)

    def read_kv8(self, codes, words, block_table, contexts, dtype):
        v, ps = self._expanded(codes, words), codes.shape[3]
        out = [v[block_table[r, p // ps].long(), :, :, p % ps] for r, n in enumerate(contexts) for p in range(n)]
        return torch.stack(out).to(dtype)

    def copy_pages(self, tensors, src, dst):
        assert len(src) == len(dst) and len(set(dst)) == len(dst) and not set(src) & set(dst)
        for t in tensors:
            t[list(dst)] = t[list(src)]

    def token_scores(self, logits, tokens, top=0):
        full = torch.log_softmax(logits.double(), -1)
        lp = full.gather(1, tokens.long()[:, None])[:, 0]
        order = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :top]
        return lp.float(), -(full.exp() * full).sum(-1).float(), full.gather(1, order).float(), order.int()
