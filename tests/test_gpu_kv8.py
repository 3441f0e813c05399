"""Keys and values in 8 bits: writing, reading back, attention, on the device against 64-bit restatements."""
import math

import numpy as np
import pytest
import torch

from plain_kv8 import BLOCK, PlainCache8, attend, tolerance

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from pytriton_llama_b200.ops.cuda import CudaOps
    return CudaOps(torch.device("cuda:0"))


class Pool:
    """A device cache and its plain restatement, with the pages of a few requests."""

    def __init__(self, ops, G, d, ps, lengths, seed, spare=2):
        self.ops, self.G, self.d, self.ps = ops, G, d, ps
        g = np.random.default_rng(seed)
        blocks = [max(1, -(-n // ps)) for n in lengths]
        self.pages = sum(blocks) + spare
        ids = g.permutation(self.pages)
        self.tables, at = [], 0
        for b in blocks:
            self.tables.append(ids[at:at + b].tolist())
            at += b
        self.unused = ids[at:].tolist()
        self.table = torch.full((len(lengths), max(blocks) + 1), -1, dtype=torch.int32)
        for r, t in enumerate(self.tables):
            self.table[r, :len(t)] = torch.tensor(t)
        self.table = self.table.cuda()
        # whatever pages held before
        gen = torch.Generator("cuda").manual_seed(seed)
        self.codes = torch.randint(0, 256, (self.pages, 2, G, ps, d), dtype=torch.uint8, device="cuda", generator=gen)
        self.words = torch.randint(-2 ** 31, 2 ** 31 - 1, (self.pages, G, ps // BLOCK, 2), dtype=torch.int32, device="cuda", generator=gen)
        self.plain = PlainCache8(G, d, ps)
        self.held = [0] * len(lengths)

    def slots(self, r, positions):
        return [self.tables[r][p // self.ps] * self.ps + p % self.ps for p in positions]

    def append(self, counts, kv, nq=0, q=None, inv_freq=None, rot=0, dtype=torch.bfloat16):
        """The next counts[r] tokens of every request, kv [T, 2, G, d]; returns the qkv buffer."""
        T = sum(counts)
        slots, pos = [], []
        for r, n in enumerate(counts):
            p = range(self.held[r], self.held[r] + n)
            slots += self.slots(r, p)
            pos += list(p)
            self.held[r] += n
        qkv = torch.cat([q if q is not None else torch.zeros(T, 0), kv.reshape(T, -1)], 1).to(dtype).cuda()
        self.ops.rope_kv8_write(qkv, torch.tensor(pos, dtype=torch.int32, device="cuda"), inv_freq, rot,
                                torch.tensor(slots, dtype=torch.int32, device="cuda"), self.codes, self.words, nq, self.G, self.d, self.ps)
        self.plain.write(kv.to(dtype), slots)
        return qkv, slots, pos

    def check(self, lengths=None):
        n = lengths or self.held
        got = self.ops.read_kv8(self.codes, self.words, self.table, n, torch.float32).cpu().double()
        want = [self.plain.read(t, k) for t, k in zip(self.tables, n) if k]
        v, bad = torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want])
        v[bad] = math.nan
        assert torch.equal(torch.isnan(got), torch.isnan(v))
        assert torch.equal(got.nan_to_num(), v.nan_to_num())
        as_bf16 = self.ops.read_kv8(self.codes, self.words, self.table, n, torch.bfloat16).cpu().double()
        assert torch.equal(as_bf16.nan_to_num(), v.nan_to_num())


def values(T, G, d, seed, spread=4):
    """Values of very different sizes from token to token, so that blocks' exponents grow."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn((T, 2, G, d), generator=g) * torch.exp2(torch.randint(-spread, spread + 1, (T, 2, G, 1), generator=g).float())


# ----------------------------------------------------------------------------- writing and reading
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G,d,ps", [(2, 64, 16), (1, 128, 32), (3, 48, 16), (5, 16, 48), (1, 256, 64)])
def test_written_values_are_read_back(ops, dtype, G, d, ps):
    counts = [[1, 17, 40, 2], [1, 1, 1, 1], [3, 16, 0, 30], [1, 0, 1, 64], [15, 33, 5, 1]]
    total = [sum(c[i] for c in counts) for i in range(4)]
    pool = Pool(ops, G, d, ps, total, seed=G * d)
    for i, c in enumerate(counts):
        pool.append(c, values(sum(c), G, d, seed=i), dtype=DTYPES[dtype])
        pool.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_held_does_not_depend_on_the_portions(ops, dtype):
    n, x = 83, values(83, 2, 64, seed=3, spread=20)
    whole, single, cut = (Pool(ops, 2, 64, 32, [n], seed=s) for s in (1, 2, 3))
    whole.append([n], x, dtype=DTYPES[dtype])
    for t in range(n):
        single.append([1], x[t:t + 1], dtype=DTYPES[dtype])
    at = 0
    for k in (5, 11, 1, 30, 3, 33):
        cut.append([k], x[at:at + k], dtype=DTYPES[dtype])
        at += k
    got = [ops.read_kv8(p.codes, p.words, p.table, [n], torch.float32) for p in (whole, single, cut)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    whole.check()


def test_error_is_half_a_step(ops):
    x = values(64, 2, 64, seed=5, spread=0)
    pool = Pool(ops, 2, 64, 16, [64], seed=5)
    pool.append([64], x, dtype=torch.float32)
    got = ops.read_kv8(pool.codes, pool.words, pool.table, [64], torch.float32).cpu()
    big = x.view(4, 16, 2, 2, 64).abs().amax((1, 4), keepdim=True).expand(4, 16, 2, 2, 64).reshape(64, 2, 2, 64)
    assert ((got - x).abs() <= torch.exp2(torch.floor(torch.log2(big)) - 7)).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_zeros_tiny_huge_and_marked_values(ops, dtype):
    x = values(70, 1, 64, seed=7, spread=1)
    top = float(torch.finfo(DTYPES[dtype]).max)
    x[0:3] = 0                                  # a block that begins with zeros
    x[16:32] = 0                                # a block of zeros
    x[32, 0, 0, 5], x[33, 1, 0, 9] = math.nan, math.inf
    x[47, 0, 0, 63] = -math.inf
    x[48:64] = torch.randn(16, 2, 1, 64) * 1e-38
    x[50, 0, 0, 1] = -1e-40
    x[64, 0, 0, 3], x[65, 1, 0, 4] = top, -top
    x[66, 0, 0, 3] = -1e-37                     # beside the largest number there is
    for step in (70, 1, 9):
        pool = Pool(ops, 1, 64, 16, [70], seed=step)
        for at in range(0, 70, step):
            pool.append([min(step, 70 - at)], x[at:at + step], dtype=DTYPES[dtype])
        pool.check()
    # a marked token that is written again with finite numbers loses its mark
    pool = Pool(ops, 1, 64, 16, [20], seed=1)
    pool.append([20], x[30:50])
    s = pool.slots(0, [2, 3])
    y = values(2, 1, 64, seed=9, spread=0)
    ops.rope_kv8_write(y.reshape(2, -1).bfloat16().cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"), None, 0,
                       torch.tensor(s, dtype=torch.int32, device="cuda"), pool.codes, pool.words, 0, 1, 64, 16)
    pool.plain.write(y.bfloat16(), s)
    pool.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 128), (48, 24), (80, 20), (64, 16), (64, 0)])
def test_rotation_is_that_of_the_other_cache(ops, dtype, d, rot):
    G, nq, T, t = 2, 3, 37, DTYPES[dtype]
    g = torch.Generator().manual_seed(d + rot)
    qkv = torch.randn((T, (nq + 2 * G) * d), generator=g).to(t).cuda()
    inv_freq = (10000.0 ** (-torch.arange(0, max(rot, 2), 2).float() / max(rot, 2))).cuda() if rot else None
    pos = torch.cat([torch.arange(5, 21), torch.arange(100000, 100021)]).int().cuda()
    slots = torch.cat([torch.arange(5, 21), torch.arange(64, 85)]).int().cuda()
    full = torch.zeros((8, 2, G, 16, d), dtype=t, device="cuda")
    turned = qkv.clone()
    ops.rope_kv_write(turned, pos, inv_freq, rot, slots, full, nq, G, d, 16)
    codes, words = torch.zeros((8, 2, G, 16, d), dtype=torch.uint8, device="cuda"), torch.zeros((8, G, 1, 2), dtype=torch.int32, device="cuda")
    mine = qkv.clone()
    ops.rope_kv8_write(mine, pos, inv_freq, rot, slots, codes, words, nq, G, d, 16)
    assert torch.equal(mine[:, :nq * d], turned[:, :nq * d])
    assert torch.equal(mine[:, nq * d:], qkv[:, nq * d:])
    plain = PlainCache8(G, d, 16)
    k = full.transpose(2, 3).reshape(8, 2, 16, G, d).transpose(1, 2).reshape(128, 2, G, d)[slots.long()].cpu()
    plain.write(k, slots.tolist())
    got = ops.read_kv8(codes, words, torch.arange(8, dtype=torch.int32, device="cuda")[None], [128], torch.float32)[slots.long()].cpu().double()
    want = torch.stack([torch.from_numpy(plain.held(s)[0]) for s in slots.tolist()])
    assert torch.equal(got, want)


def test_rows_without_a_slot_write_nothing(ops):
    pool = Pool(ops, 2, 64, 16, [40], seed=11)
    before = pool.codes.clone(), pool.words.clone()
    kv = values(6, 2, 64, seed=1).reshape(6, -1).bfloat16().cuda()
    pos = torch.zeros(6, dtype=torch.int32, device="cuda")
    behind = pool.pages * 16
    ops.rope_kv8_write(kv, pos, None, 0, torch.tensor([-1, -5, behind, behind + 7, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda"),
                       pool.codes, pool.words, 0, 2, 64, 16)
    assert torch.equal(before[0], pool.codes) and torch.equal(before[1], pool.words)
    # among rows that have one
    s = pool.slots(0, [0, 1, 2])
    x = values(6, 2, 64, seed=2)
    ops.rope_kv8_write(x.reshape(6, -1).bfloat16().cuda(), pos, None, 0, torch.tensor([-1, s[0], s[1], s[2], -1, behind], dtype=torch.int32, device="cuda"),
                       pool.codes, pool.words, 0, 2, 64, 16)
    pool.plain.write(x[1:4].bfloat16(), s)
    pool.check([3])
    touched = s[0] // 16
    rest = [p for p in range(pool.pages) if p != touched]
    assert torch.equal(before[0][rest], pool.codes[rest]) and torch.equal(before[1][rest], pool.words[rest])
    ops.rope_kv8_write(torch.zeros((0, 256), dtype=torch.bfloat16, device="cuda"), pos, None, 0, pos, pool.codes, pool.words, 0, 2, 64, 16)
    assert ops.read_kv8(pool.codes, pool.words, pool.table, [0], torch.bfloat16).shape == (0, 2, 2, 64)


def test_many_requests_are_read(ops):
    """More than one launch's worth of requests, some without tokens, a page that is missing."""
    n = 2000
    lengths = [(7 * i) % 4 for i in range(n)]
    codes = torch.randint(0, 256, (600, 2, 1, 16, 16), dtype=torch.uint8, device="cuda")
    words = torch.randint(120, 140, (600, 1, 1, 2), dtype=torch.int32, device="cuda")
    table = torch.arange(n, dtype=torch.int32, device="cuda").remainder(601)[:, None].contiguous()       # page 600 does not exist
    got = ops.read_kv8(codes, words, table, lengths, torch.float32)
    v = (codes.double() - 127.5) * torch.exp2((words[..., 0, :].double() - 133)).transpose(1, 2)[:, :, :, None, None]
    v = torch.cat([v, torch.zeros_like(v[:1])])
    want = torch.cat([v[r % 601].permute(2, 0, 1, 3)[:k] for r, k in enumerate(lengths)])
    assert torch.equal(got.double(), want)


# ----------------------------------------------------------------------------- attention
SHAPES = [(4, 2, 64, 16), (8, 1, 128, 32), (6, 2, 128, 16), (16, 1, 64, 48), (5, 5, 48, 16), (20, 1, 64, 16), (4, 1, 256, 64), (3, 3, 80, 16), (2, 2, 16, 16),
          (32, 1, 128, 16)]
STEPS = {  # (new tokens, tokens cached before) of the requests
    "singles": [(1, 0), (1, 1), (1, 14), (1, 15), (1, 16), (1, 62), (1, 63), (1, 64), (1, 129), (1, 300)],
    "long": [(1, 1500), (1, 700)],
    "prompts": [(2, 0), (17, 0), (130, 0), (15, 1), (33, 31), (257, 70)],
    "mixed": [(1, 40), (5, 0), (1, 0), (129, 3), (1, 200), (64, 64), (2, 500)],
}


def run_attention(ops, nq, G, d, ps, step, dtype, window=0, spoil=None, extra=0, seed=0, gain=1.0, far=False):
    t = DTYPES[dtype]
    lens = [n + c for n, c in step]
    pool = Pool(ops, G, d, ps, lens, seed=seed + d)
    kv = [values(n, G, d, seed=seed + i, spread=1) for i, n in enumerate(lens)]
    if spoil:
        spoil(kv)
    if any(c for _, c in step):
        pool.append([c for _, c in step], torch.cat([x[:c] for x, (_, c) in zip(kv, step)]), dtype=t)
    T = sum(n for n, _ in step)
    g = torch.Generator().manual_seed(seed + 77)
    q = (torch.randn((T, nq * d), generator=g) * gain).to(t)
    qkv, slots, pos = pool.append([n for n, _ in step], torch.cat([x[c:] for x, (_, c) in zip(kv, step)]), nq=nq, q=q, dtype=t)
    req = torch.cat([torch.full((n,), r) for r, (n, _) in enumerate(step)]).int()
    if extra:       # rows behind the last request, as a padded step has them
        qkv = torch.cat([qkv, torch.full((extra, qkv.shape[1]), math.nan, dtype=t, device="cuda")])
        req = torch.cat([req, torch.full((extra,), -1).int()])
        pos = pos + [0] * extra
    hints = ops.hints_for([n for n, _ in step], lens)
    scale = d ** -0.5
    got = ops.paged_attention8(qkv, pool.codes, pool.words, pool.table, req.cuda(), torch.tensor(pos, dtype=torch.int32, device="cuda"), nq, G, d, ps,
                               scale, window=window, hints=hints)
    assert got.shape == (T + extra, nq * d) and got.dtype == t
    at = 0
    for r, (n, c) in enumerate(step):
        v, bad = pool.plain.read(pool.tables[r], n + c)
        out, size, score = attend(q[at:at + n].double().view(n, nq, d), v, bad, list(range(c, c + n)), scale, window)
        mine = got[at:at + n].double().cpu().view(n, nq, d)
        assert torch.equal(torch.isnan(mine), torch.isnan(out)), (r, n, c)
        fine = ~torch.isnan(out)
        off = (mine - out).abs()[fine] / tolerance(t, out, size, score, d, n + c, torch.float16 if n == 1 else torch.bfloat16,
                                                   v[:, 1].abs().max() if far else 0.0)[fine]
        assert off.numel() == 0 or off.max() <= 1, (r, n, c, float(off.max()))
        at += n
    return got, pool, qkv, req, pos, hints


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("nq,G,d,ps", SHAPES)
def test_attention(ops, nq, G, d, ps, step, dtype):
    run_attention(ops, nq, G, d, ps, STEPS[step], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 7, 16, 65, 10000])
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (6, 2, 128, 32), (5, 5, 48, 16)])
def test_attention_within_a_window(ops, nq, G, d, ps, window, dtype):
    run_attention(ops, nq, G, d, ps, STEPS["mixed"], dtype, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (6, 2, 128, 32), (5, 5, 48, 16)])
def test_pages_before_the_window_may_be_gone(ops, nq, G, d, ps, dtype):
    step, window = [(1, 200), (40, 100), (1, 33)], 50
    got, pool, qkv, req, pos, hints = run_attention(ops, nq, G, d, ps, step, dtype, window=window)
    table = pool.table.clone()
    for r, (n, c) in enumerate(step):
        table[r, :max(0, c - window + 1) // ps] = -1
    again = ops.paged_attention8(qkv, pool.codes, pool.words, table, req.cuda(), torch.tensor(pos, dtype=torch.int32, device="cuda"), nq, G, d, ps,
                                 d ** -0.5, window=window, hints=hints)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (8, 2, 128, 32), (5, 5, 48, 16)])
def test_numbers_that_are_not_finite_reach_only_rows_that_see_them(ops, nq, G, d, ps, dtype):
    def spoil(kv):
        kv[0][0, 0, 0, 0] = math.nan            # a single token sees it, in one kv head
        kv[1][20, 1, G - 1, 3] = math.inf       # in the middle of a prompt, the block's other tokens before and after it
        kv[3][5, 0, 0, 2] = -math.inf           # cached before a portion
        kv[4][90, 1, 0, 1] = math.nan           # the last but one position of a portion's request
    run_attention(ops, nq, G, d, ps, [(1, 9), (40, 0), (1, 30), (20, 16), (70, 22), (1, 0)], dtype, spoil=spoil)
    # a marked token that fell out of the window
    run_attention(ops, nq, G, d, ps, [(1, 40), (30, 40)], dtype, window=8, spoil=lambda kv: [x.__setitem__((10, 0, 0, 0), math.nan) for x in kv])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (8, 2, 128, 32), (5, 5, 48, 16)])
def test_rows_without_a_request(ops, nq, G, d, ps, dtype):
    """Rows behind the last request, and their NaN, leave the others alone; where the step lists its rows, they may hold anything."""
    run_attention(ops, nq, G, d, ps, STEPS["mixed"], dtype, extra=3)
    run_attention(ops, nq, G, d, ps, STEPS["singles"], dtype, extra=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (8, 2, 128, 32), (5, 5, 48, 16)])
def test_scores_far_apart(ops, nq, G, d, ps, dtype):
    """One key takes all of a row's weight, and rows of zeros give every key the same."""
    run_attention(ops, nq, G, d, ps, STEPS["mixed"], dtype, gain=30.0)
    run_attention(ops, nq, G, d, ps, STEPS["mixed"], dtype, gain=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_missing_pages_are_not_seen(ops, dtype):
    """A page id of -1 or behind the pool in the middle of a request: its positions are left out."""
    nq, G, d, ps, t = 4, 2, 64, 16, DTYPES[dtype]
    for n, c in ((1, 99), (20, 80)):
        pool = Pool(ops, G, d, ps, [100], seed=3)
        kv = values(100, G, d, seed=4, spread=1)
        pool.append([100], kv, dtype=t)
        q = torch.randn((n, nq * d), generator=torch.Generator().manual_seed(1)).to(t)
        table = pool.table.clone()
        table[0, 1], table[0, 3] = -1, pool.pages
        hints = ops.hints_for([n], [100])
        got = ops.paged_attention8(q.cuda(), pool.codes, pool.words, table, torch.zeros(n, dtype=torch.int32, device="cuda"),
                                   torch.arange(c, c + n, dtype=torch.int32, device="cuda"), nq, G, d, ps, d ** -0.5, hints=hints)
        v, bad = pool.plain.read(pool.tables[0], 100)
        keep = [i for i in range(100) if i // 16 not in (1, 3)]
        for t_ in range(n):
            have = [i for i in keep if i <= c + t_]
            out, size, score = attend(q[t_:t_ + 1].double().view(1, nq, d), v[have], bad[have], [len(have) - 1], d ** -0.5)
            off = (got[t_].double().cpu().view(1, nq, d) - out).abs() / tolerance(t, out, size, score, d, 100, torch.float16 if n == 1 else torch.bfloat16)
            assert off.max() <= 1
    # no page at all
    table = torch.full_like(pool.table, -1)
    got = ops.paged_attention8(q.cuda(), pool.codes, pool.words, table, torch.zeros(n, dtype=torch.int32, device="cuda"),
                               torch.arange(c, c + n, dtype=torch.int32, device="cuda"), nq, G, d, ps, d ** -0.5, hints=hints)
    assert torch.equal(got, torch.zeros_like(got))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_from_a_graph_and_on_another_stream(ops, dtype):
    nq, G, d, ps, t = 8, 2, 64, 16, DTYPES[dtype]
    step = [(1, 99), (1, 399), (1, 30)]
    first, pool, qkv, req, pos, hints = run_attention(ops, nq, G, d, ps, step, dtype, seed=1)
    req, pos, q = req.cuda(), torch.tensor(pos, dtype=torch.int32, device="cuda"), qkv[:, :nq * d].contiguous()
    call = lambda: ops.paged_attention8(q, pool.codes, pool.words, pool.table, req, pos, nq, G, d, ps, d ** -0.5, hints=hints)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    graphs = []
    for _ in range(2):      # two captured calls, replayed together on two streams
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out, torch.cuda.Stream()))
    for _ in range(20):
        for graph, out, stream in graphs:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        for graph, out, stream in graphs:
            torch.cuda.current_stream().wait_stream(stream)
        assert torch.equal(graphs[0][1], first) and torch.equal(graphs[1][1], first)
    # the same graph at other positions
    pos.copy_(torch.tensor([50, 200, 29]))
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], call())


@pytest.mark.parametrize("dtype", DTYPES)
def test_bits_of_a_row_do_not_depend_on_the_call_before(ops, dtype):
    a = run_attention(ops, 8, 2, 64, 16, STEPS["mixed"], dtype, seed=5)[0]
    run_attention(ops, 8, 2, 64, 16, STEPS["long"], dtype, seed=6)
    b = run_attention(ops, 8, 2, 64, 16, STEPS["mixed"], dtype, seed=5)[0]
    assert torch.equal(a, b)
