"""Keys and values in 8 bits, restated token by token in 64 bits from their definition, and attention over them."""
from __future__ import annotations

import math

import numpy as np
import torch

BLOCK = 16


class PlainCache8:
    """One layer's 8-bit cache as the values that were written: a block of 16 positions remembers, per head and for k and v, the
    value of each of its tokens, and works out from all of them what is held."""

    def __init__(self, heads, d, page_size):
        self.heads, self.d, self.page_size = heads, d, page_size
        self.blocks = {}                       # block -> {offset: float64 [2, heads, d]}

    def write(self, kv: torch.Tensor, slots):
        """kv [T, 2, heads, d] in the order in which it is written; slots host integers."""
        for x, s in zip(kv.double().cpu().numpy(), slots):
            if s < 0:
                continue
            if s % BLOCK == 0:
                self.blocks[s // BLOCK] = {}
            self.blocks.setdefault(s // BLOCK, {})[s % BLOCK] = x

    def exponent(self, block):
        """[2, heads] biased exponents of a block."""
        x = np.stack(list(self.blocks[block].values()))
        big = np.where(np.isfinite(x), np.abs(x), 0.0).max(axis=(0, 3))
        return np.where(big > 0, np.maximum(16, np.frexp(big)[1] - 1 + 127), 0)

    def held(self, slot):
        """(values float64 [2, heads, d] as read back, a value that is not finite taken as 0; marks [2, heads])."""
        x = self.blocks[slot // BLOCK][slot % BLOCK]
        e = self.exponent(slot // BLOCK)[..., None]
        step = np.ldexp(1.0, e - 133)
        fin = np.where(np.isfinite(x), x, 0.0)
        v = np.where(e > 0, (np.floor(fin / step) + 0.5) * step, 0.0)
        return v, ~np.isfinite(x).all(-1)

    def read(self, table, n):
        """Values [n, 2, heads, d] and marks [n, 2, heads] of the first n positions of a request with these pages."""
        ps = self.page_size
        out = [self.held(table[i // ps] * ps + i % ps) for i in range(n)]
        v, bad = np.stack([o[0] for o in out]), np.stack([o[1] for o in out])
        return torch.from_numpy(v), torch.from_numpy(bad)


def attend(q, values, bad, positions, scale, window=0):
    """q float64 [T, H, d] of one request, values [n, 2, G, d], positions [T]: (out [T, H, d], the sum of p |v|, the largest bound on
    |q| |k| scale of a row's scores [T, H])."""
    T, H, d = q.shape
    G = values.shape[2]
    out, size, score = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(T, H, dtype=torch.float64)
    key = torch.arange(values.shape[0])
    for t, p in enumerate(positions):
        seen = (key <= p) & (key > p - window) if window else key <= p
        if p < 0 or not bool(seen.any()):
            continue
        for h in range(H):
            g = h // (H // G)
            k, v = values[seen, 0, g], values[seen, 1, g]
            s = (k @ q[t, h]) * scale
            score[t, h] = q[t, h].abs().max() * k.abs().sum(-1).max() * scale
            w = torch.softmax(s, 0)
            out[t, h], size[t, h] = w @ v, w @ v.abs()
            if bool(bad[seen, :, g].any()):
                out[t, h] = math.nan
    return out, size, score


def tolerance(dtype, out, size, score, d, keys, weights=torch.float16, largest=0.0):
    """How far a kernel may be off: the output's rounding, half a step of the type; weights rounded to ``weights`` (bfloat16 rows: half floats for
    single tokens, bfloat16 for portions on the fifth-generation tensor cores), half a step of each, 2^-11 or 2^-8
    (and 2^-25 of the largest where half floats leave the normal numbers, keys of them at most); 2 eps for a relative error eps of
    e^s, where a score's d products and sums in float32, two more for its scale and the exponential's few ulps, err by
    (d + 8) 2^-24 of |q| |k| scale; and the float32 sums over the keys.

    ``largest``: the largest |v| of the request, where values lie so far apart that the smallest weights matter.  Weights are half floats (float32:
    two, the second of what the first leaves) in units of 2^-7, and half floats are 2^-24 apart below 2^-14, so a weight is off by up to
    2^-25 of those units, 2^-32 of the largest weight, which is at least 1 of the row's sum's terms; in blocks whose weights carry their
    step, by as much in units of the largest step, whose block has a value of at least 64 of its steps where codes count up to 128: 2^-31 |v| a key."""
    half = torch.finfo(dtype).eps / 2
    eps = (d + 8) * 2.0 ** -24 * (1 + score[..., None])
    rounding = torch.finfo(weights).eps / 2 + keys * 2.0 ** -25 if dtype == torch.bfloat16 else 2.0 ** -22
    return half * out.abs() + size * (2 * eps + 2 * rounding + (keys + 64) * 2.0 ** -24) + keys * 2.0 ** -31 * largest + 1e-30
