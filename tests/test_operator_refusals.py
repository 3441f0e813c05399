"""What the operators of the 8-bit cache, page copies and token scores refuse.  No kernel runs: the wrappers check their arguments on
any device, and the library's entries check theirs before they launch."""
import ctypes

import pytest
import torch

from pytriton_llama_b200.ops.cuda import CudaOps, KernelError, load_library


class _NoLibrary:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


@pytest.fixture()
def ops():
    o = CudaOps.__new__(CudaOps)
    o.device, o.lib, o._raw_stream, o._device_index, o.launches = torch.device("cpu"), _NoLibrary(), lambda i: 0, 0, 0
    return o


I32, BF = torch.int32, torch.bfloat16


def cache(pages=4, G=2, ps=16, d=64):
    return dict(codes=torch.zeros((pages, 2, G, ps, d), dtype=torch.uint8), words=torch.zeros((pages, G, max(1, ps // 16), 2), dtype=I32))


def write_args(**over):
    a = dict(qkv=torch.zeros((3, (4 + 2 * 2) * 64), dtype=BF), positions=torch.zeros(3, dtype=I32), inv_freq=torch.zeros(32), rot=64,
             slots=torch.zeros(3, dtype=I32), nq=4, nkv=2, d=64, page_size=16, **cache())
    a.update(over)
    return a


@pytest.mark.parametrize("over,message", [
    (dict(qkv=torch.zeros((3, 500), dtype=BF)), "rows of 512"),
    (dict(qkv=torch.zeros((6, 512), dtype=BF)[::2]), "contiguous"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions has element type"),
    (dict(slots=torch.zeros(3, dtype=torch.int64)), "slots has element type"),
    (dict(slots=torch.zeros(2, dtype=I32)), "fewer positions or slots"),
    (dict(positions=torch.zeros(2, dtype=I32)), "fewer positions or slots"),
    (dict(inv_freq=torch.zeros(31)), "inv_freq shorter"),
    (dict(inv_freq=torch.zeros(32, dtype=torch.float64)), "inv_freq has element type"),
    (dict(page_size=8), "no whole blocks"),
    (dict(d=60), "no multiple of 16"),
    (dict(codes=torch.zeros((4, 2, 2, 16, 64), dtype=torch.int8)), "codes has element type"),
    (dict(codes=torch.zeros((4, 2, 2, 16, 32), dtype=torch.uint8)), "do not fit"),
    (dict(words=torch.zeros((4, 2, 1, 2), dtype=torch.int64)), "words has element type"),
    (dict(words=torch.zeros((4, 2, 2, 1), dtype=I32)), "expected"),
    (dict(words=torch.zeros((3, 2, 1, 2), dtype=I32)), "expected"),
    (dict(qkv=torch.zeros((3, 512), dtype=torch.float16)), "unsupported element type"),
])
def test_write(ops, over, message):
    with pytest.raises(KernelError, match=message):
        ops.rope_kv8_write(**write_args(**over))


def test_tensors_of_another_device(ops):
    ops.device = torch.device("cuda:0")
    with pytest.raises(KernelError, match="lives on"):
        ops.rope_kv8_write(**write_args())
    with pytest.raises(KernelError, match="lives on"):
        ops.copy_pages([torch.zeros(3, 3)], [0], [1])
    with pytest.raises(KernelError, match="lives on"):
        ops.token_scores(torch.zeros(2, 5), torch.zeros(2, dtype=I32), 1)


@pytest.mark.parametrize("over,message", [
    (dict(q=torch.zeros((3, 100), dtype=BF)), "for 4 heads"),
    (dict(nq=3), "for 3 heads"),
    (dict(nq=0), "for 0 heads"),
    (dict(block_table=torch.zeros((1, 2), dtype=torch.int64)), "block_table has element type"),
    (dict(block_table=torch.zeros(4, dtype=I32)), "the block table is"),
    (dict(tok_req=torch.zeros(2, dtype=I32)), "fewer requests or positions"),
    (dict(positions=torch.zeros(2, dtype=I32)), "fewer requests or positions"),
    (dict(page_size=24), "no whole blocks"),
    (dict(d=512), "up to 256"),
    (dict(window=-1), "window"),
    (dict(window=1 << 31), "window"),
    (dict(scale=-0.125), "scores times"),
    (dict(scale=float("nan")), "scores times"),
])
def test_attention(ops, over, message):
    a = dict(q=torch.zeros((3, 256), dtype=BF), block_table=torch.zeros((1, 2), dtype=I32), tok_req=torch.zeros(3, dtype=I32),
             positions=torch.zeros(3, dtype=I32), nq=4, nkv=2, d=64, page_size=16, scale=0.125, **cache())
    a.update(over)
    with pytest.raises(KernelError, match=message):
        ops.paged_attention8(**a)


@pytest.mark.parametrize("over,message", [
    (dict(contexts=[3, 4]), "2 requests"),
    (dict(contexts=[-1]), "of -1 tokens"),
    (dict(contexts=[33]), "of 33 tokens"),
    (dict(codes=torch.zeros((4, 64), dtype=torch.uint8)), "expected .pages"),
    (dict(block_table=torch.zeros((1, 2), dtype=torch.int64)), "block_table has element type"),
])
def test_reading(ops, over, message):
    a = dict(block_table=torch.zeros((1, 2), dtype=I32), contexts=[3], dtype=BF, **cache())
    a.update(over)
    with pytest.raises(KernelError, match=message):
        ops.read_kv8(**a)


@pytest.mark.parametrize("src,dst,message", [
    ([0], [1, 2], "1 rows to read, 2"),
    ([0, 1], [2, 2], "written twice"),
    ([0, 1], [1, 2], "read is written"),
    ([0], [0], "read is written"),
    ([0], [4], "rows 0..4"),
    ([-1], [1], "rows -1..1"),
    ([1 << 40], [1], "rows 1.."),
])
def test_copies(ops, src, dst, message):
    with pytest.raises(KernelError, match=message):
        ops.copy_pages([torch.zeros(5, 3), torch.zeros(4, 8)], src, dst)


def test_copies_of_tensors_that_overlap(ops):
    base = torch.zeros(8, 4)
    with pytest.raises(KernelError, match="share memory"):
        ops.copy_pages([base[:5], base[3:]], [0], [1])
    with pytest.raises(KernelError, match="share memory"):
        ops.copy_pages([base, base], [0], [1])
    with pytest.raises(KernelError, match="contiguous"):
        ops.copy_pages([base.t()], [0], [1])


@pytest.mark.parametrize("over,message", [
    (dict(logits=torch.zeros((3, 50), dtype=BF)), "logits has element type"),
    (dict(logits=torch.zeros((50, 3)).t()), "contiguous"),
    (dict(logits=torch.zeros(50)), "expected .rows, vocabulary"),
    (dict(logits=torch.zeros((3, 0))), "expected .rows, vocabulary"),
    (dict(tokens=torch.zeros(3, dtype=torch.int64)), "tokens has element type"),
    (dict(tokens=torch.zeros(2, dtype=I32)), "2 tokens for 3 rows"),
    (dict(top=33), "at most 32"),
    (dict(top=-1), "at most 32"),
])
def test_scores(ops, over, message):
    a = dict(logits=torch.zeros((3, 50)), tokens=torch.zeros(3, dtype=I32), top=2)
    a.update(over)
    with pytest.raises(KernelError, match=message):
        ops.token_scores(**a)


def test_the_library_refuses_before_it_launches():
    lib = load_library()
    err = lambda: lib.ptl_last_error().decode()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 63) // 64 * 64
    w = lambda **o: lib.ptl_rope_kv8_write_bf16(CudaOps._KV8_WRITE_ARGS.pack(at, at, 0, at, o.get("codes", at), at, 0, 64, 1, 1, 1, o.get("d", 64),
                                                                             o.get("rot", 0), o.get("ps", 16)))
    assert w(d=40) == -1 and "head size 40" in err()
    assert w(ps=20) == -1 and "pages of 20" in err()
    assert w(rot=65) == -1 and "rotary width" in err()
    assert w(codes=at + 8) == -1 and "aligned" in err()
    a = lambda **o: lib.ptl_attention8_simt_f32(at, None, None, at, at, o.get("words", at), at, at, at, 1, 64, 64, 1, o.get("nq", 1), o.get("nkv", 1),
                                                o.get("d", 64), o.get("ps", 16), 1.0, 0, o.get("splits", 1), 4, None)
    assert a(d=272) == -1 and "head size 272" in err()
    assert a(nq=3, nkv=2) == -1 and "no multiple" in err()
    assert a(ps=8) == -1 and "whole blocks" in err()
    assert a(words=at + 4) == -1 and "aligned" in err()
    assert a(splits=2) == -1 and "scratch" in err()
    n = (ctypes.c_int * 1)(17)
    read = CudaOps._KV8_READ_ARGS.pack(at, at, at, at, ctypes.addressof(n), 0, 1, 1, 1, 64, 16, 4)
    assert lib.ptl_read_kv8_f32(read) == -1 and "17 tokens" in err()
    scores = lambda logits, vocab, top: lib.ptl_token_scores(CudaOps._TOKEN_SCORES_ARGS.pack(at, at, at, at, logits, at, 0, 1, vocab, top, 0))
    assert scores(at, 40, 33) == -1 and "at most 32" in err()
    assert scores(at, 4, 5) == -1 and "at most 32" in err()
    assert scores(at + 2, 4, 1) == -1 and "aligned" in err()
    launches = ctypes.c_int(7)
    ptrs, rows = (ctypes.c_void_p * 1)(at), (ctypes.c_longlong * 1)(0)
    assert lib.ptl_copy_pages(ptrs, rows, 1, ctypes.addressof(n), ctypes.addressof(n), 1, ctypes.byref(launches), None) == -1 and "no rows" in err()


def test_every_entry_that_the_operators_call_has_its_signature():
    """Without one, addresses would be cut to 32 bits."""
    import re
    from pathlib import Path

    import pytriton_llama_b200.ops.cuda as module
    lib = load_library()
    text = Path(module.__file__).read_text()
    names = set(re.findall(r"lib\.(ptl_\w+)\((?!\))", text)) | {n + t for n in re.findall(r'"(ptl_\w+)" \+ ', text) for t in ("_f32", "_bf16")}
    assert len(names) > 50
    without = [n for n in sorted(names) if hasattr(lib, n) and getattr(lib, n).argtypes is None]
    assert without == []
