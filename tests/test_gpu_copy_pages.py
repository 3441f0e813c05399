"""Rows copied inside many tensors at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pytriton_llama_b200.ops.cuda import CudaOps
    return CudaOps(torch.device("cuda:0"))


def filled(shape, dtype, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * torch.empty((), dtype=dtype).element_size()), dtype=torch.uint8, device="cuda",
                         generator=g).view(dtype)


CASES = [
    ([((40, 2, 2, 16, 64), torch.bfloat16)], 1),
    ([((40, 2, 2, 16, 64), torch.bfloat16)] * 3 + [((40, 7), torch.float32)], 19),
    ([((50, 4097), torch.float32), ((60, 3), torch.int32)], 25),                     # four bytes at a time
    ([((50, 5), torch.uint8), ((50, 70001), torch.uint8)], 20),                      # one byte at a time
    ([((9000, 16), torch.uint8)], 4400),                                             # more pairs than one launch takes
    ([((20, 64), torch.float32)] * 300, 9),                                          # more tensors
    ([((3, 20000, 16), torch.bfloat16)], 1),                                         # one large row
    ([((10, 0, 4), torch.float32), ((10, 4), torch.float32)], 2),                    # a tensor without elements
]


@pytest.mark.parametrize("shapes,pairs", CASES)
def test_rows_are_copied(ops, shapes, pairs):
    tensors = [filled(s, t, i) for i, (s, t) in enumerate(shapes)]
    rows = min(t.shape[0] for t in tensors)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(pairs)).tolist()
    dst, rest = order[:pairs], order[pairs:]
    src = [rest[i % len(rest)] for i in range(pairs)]                                # a row may be read for several
    want = [t.clone() for t in tensors]
    for w in want:
        w[torch.tensor(dst, device="cuda")] = w[torch.tensor(src, device="cuda")]
    ops.copy_pages(tensors, src, dst)
    for t, w in zip(tensors, want):
        assert torch.equal(t.view(torch.uint8) if t.numel() else t, w.view(torch.uint8) if w.numel() else w)


def test_a_view_that_is_not_aligned(ops):
    base = filled((4 * 33 + 8,), torch.uint8, 1)
    for off in (1, 4, 8):
        t = base[off:off + 4 * 33].view(4, 33)
        before = base.clone()
        ops.copy_pages([t], [1], [3])
        want = before.clone()
        want[off + 99:off + 132] = before[off + 33:off + 66]
        assert torch.equal(base, want)


def test_nothing_to_copy(ops):
    t = filled((4, 8), torch.float32, 1)
    before = t.clone()
    launches = ops.launches
    ops.copy_pages([t], [], [])
    ops.copy_pages([], [1], [2])
    assert torch.equal(t.view(torch.uint8), before.view(torch.uint8)) and ops.launches == launches


def test_captured_copies_hold_their_own_rows(ops):
    t = filled((8, 1024), torch.bfloat16, 2)
    first = t.clone()
    graphs = []
    for src, dst in (([0, 1], [6, 7]), ([2], [5])):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.copy_pages([t], src, dst)
        graphs.append(g)
    for g in graphs:
        g.replay()
    want = first.clone()
    want[6], want[7], want[5] = first[0], first[1], first[2]
    assert torch.equal(t.view(torch.uint8), want.view(torch.uint8))
