"""Attention over an 8-bit cache by each of the forms that its kernels have, whichever the sizes would choose; and far corners of the cache."""
import math

import pytest
import torch

from conftest import PAGE_SIZE, TINY, random_tokens
from gpu_common import stored_dtype
from plain_kv8 import attend, tolerance
from test_gpu_kv8 import DTYPES, STEPS, Pool, run_attention, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pytriton_llama_b200.ops.cuda import CudaOps
    return CudaOps(torch.device("cuda:0"))


class Forced:
    """The operators with hints that name a form."""

    def __init__(self, ops, **form):
        self.ops, self.form = ops, form

    def __getattr__(self, name):
        return getattr(self.ops, name)

    def hints_for(self, *lengths):
        hints = self.ops.hints_for(*lengths)
        for name, value in self.form.items():
            setattr(hints, name, value)
        return hints


def spoil(kv):
    kv[0][0, 0, 0, 0] = math.nan
    kv[4][min(60, len(kv[4]) - 1), 1, -1, 3] = math.inf
    kv[9][17, 0, 0, 1] = -math.inf


FORMS = [(parts, warps) for parts in (0, 1, 2, 4, 8) for warps in (4, 8) if parts or warps == 4]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (8, 1, 128, 32), (3, 1, 64, 48)])
def test_single_tokens_in_every_form(ops, nq, G, d, ps, form, dtype):
    forced = Forced(ops, single_form=form)
    run_attention(forced, nq, G, d, ps, STEPS["singles"], dtype)
    run_attention(forced, nq, G, d, ps, STEPS["long"], dtype)
    run_attention(forced, nq, G, d, ps, STEPS["singles"], dtype, spoil=spoil, extra=2)
    run_attention(forced, nq, G, d, ps, STEPS["long"], dtype, window=129)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("parts", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("nq,G,d", [(18, 2, 64), (16, 1, 128)])
def test_single_tokens_of_wide_groups_in_every_form(ops, nq, G, d, parts, dtype):
    forced = Forced(ops, single_form=(parts, 4))
    run_attention(forced, nq, G, d, 16, STEPS["singles"], dtype, spoil=spoil)
    run_attention(forced, nq, G, d, 16, STEPS["long"], dtype)


LONG_PORTIONS = {"one": [(20, 1500)], "pair": [(131, 900), (3, 1200)], "mixed": [(1, 700), (40, 600), (1, 3), (130, 0), (300, 5)]}


def scale_blocks(kv):
    """Values of neighbouring blocks apart by up to 2^24."""
    g = torch.Generator().manual_seed(1)
    for x in kv:
        e = torch.randint(-12, 13, (-(-len(x) // 16), 1, x.shape[2], 1), generator=g).float().repeat_interleave(16, 0)[:len(x)]
        x[:, 1:] *= torch.exp2(e)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("step", LONG_PORTIONS)
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (3, 1, 128, 32), (12, 1, 64, 48), (16, 1, 128, 16), (9, 1, 64, 256)])
def test_portions_in_every_form(ops, nq, G, d, ps, step, split, dtype):
    forced = Forced(ops, split_portions=split)
    run_attention(forced, nq, G, d, ps, LONG_PORTIONS[step], dtype)
    run_attention(forced, nq, G, d, ps, LONG_PORTIONS[step], dtype, window=333)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (3, 1, 128, 32)])
def test_values_far_apart(ops, nq, G, d, ps, split, dtype):
    forced = Forced(ops, split_portions=split)
    run_attention(forced, nq, G, d, ps, LONG_PORTIONS["mixed"], dtype, spoil=scale_blocks, far=True)
    run_attention(forced, nq, G, d, ps, LONG_PORTIONS["mixed"], dtype, spoil=scale_blocks, gain=8.0, window=100, far=True)
    run_attention(forced, nq, G, d, ps, STEPS["singles"], dtype, spoil=scale_blocks, far=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [False, True])
def test_marks_in_split_portions(ops, split, dtype):
    def some(kv):
        kv[0][700, 0, 0, 0] = math.nan
        kv[1][1201, 1, 0, 5] = math.inf
    run_attention(Forced(ops, split_portions=split), 4, 2, 64, 16, LONG_PORTIONS["pair"], dtype, spoil=some)
    run_attention(Forced(ops, split_portions=split), 4, 2, 64, 16, LONG_PORTIONS["pair"], dtype, spoil=some, window=300)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("d,ps", [(64, 16), (128, 32)])
def test_missing_pages_in_split_portions(ops, d, ps, split, dtype):
    """Whole parts of the keys among them."""
    nq, G, t, n, total = 4, 2, DTYPES[dtype], 24, 1400
    pool = Pool(ops, G, d, ps, [total], seed=3)
    pool.append([total], values(total, G, d, seed=4, spread=1), dtype=t)
    q = torch.randn((n, nq * d), generator=torch.Generator().manual_seed(1)).to(t)
    table = pool.table.clone()
    gone = {1, 3, *range(600 // ps, 1100 // ps)}
    for b in gone:
        table[0, b] = -1 if b % 2 else pool.pages + b
    hints = Forced(ops, split_portions=split).hints_for([n], [total])
    pos = torch.arange(total - n, total, dtype=torch.int32, device="cuda")
    got = ops.paged_attention8(q.cuda(), pool.codes, pool.words, table, torch.zeros(n, dtype=torch.int32, device="cuda"), pos, nq, G, d, ps, d ** -0.5,
                               hints=hints).double().cpu()
    v, bad = pool.plain.read(pool.tables[0], total)
    for i in range(n):
        have = [k for k in range(total - n + i + 1) if k // ps not in gone]
        out, size, score = attend(q[i:i + 1].double().view(1, nq, d), v[have], bad[have], [len(have) - 1], d ** -0.5)
        assert ((got[i].view(1, nq, d) - out).abs() <= tolerance(t, out, size, score, d, total, torch.bfloat16)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,G,d", [(4, 2, 64), (5, 5, 48)])
def test_positions_behind_the_table_are_not_seen(ops, nq, G, d, dtype):
    t = DTYPES[dtype]
    for n in (1, 20):
        pool = Pool(ops, G, d, 16, [96], seed=3)
        pool.append([96], values(96, G, d, seed=4, spread=1), dtype=t)
        q = torch.randn((n, nq * d), generator=torch.Generator().manual_seed(1)).to(t).cuda()
        where = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(96 - n, 96, dtype=torch.int32, device="cuda")
        narrow, wide = pool.table[:, :4].contiguous(), pool.table.clone()
        wide[:, 4:] = -1
        call = lambda table, hints: ops.paged_attention8(q, pool.codes, pool.words, table, *where, nq, G, d, 16, d ** -0.5, hints=hints)
        assert torch.equal(call(narrow, ops.hints_for([n], [96])), call(wide, ops.hints_for([n], [96])))
        assert torch.equal(call(narrow, None), call(wide, None))


def test_pages_far_into_a_large_pool(ops):
    """Offsets of codes that pass 32 bits: written, read, attended, copied."""
    nq, G, d, ps = 16, 8, 128, 64
    spare = 2 ** 32 // (2 * G * ps * d) + 200
    pool = Pool(ops, G, d, ps, [200], seed=1, spare=spare)
    assert pool.codes.numel() > 2 ** 32
    last = list(range(pool.pages - 4, pool.pages))
    pool.tables = [last]
    pool.table[0, :4] = torch.tensor(last)
    kv = values(200, G, d, seed=5, spread=1)
    pool.append([200], kv)
    pool.check()
    v, bad = pool.plain.read(last, 200)
    for n, split in ((1, None), (30, True), (30, False)):
        q = torch.randn((n, nq * d), generator=torch.Generator().manual_seed(n)).bfloat16()
        hints = Forced(ops, split_portions=split).hints_for([n], [200])
        got = ops.paged_attention8(q.cuda(), pool.codes, pool.words, pool.table, torch.zeros(n, dtype=torch.int32, device="cuda"),
                                   torch.arange(200 - n, 200, dtype=torch.int32, device="cuda"), nq, G, d, ps, d ** -0.5, hints=hints)
        out, size, score = attend(q.double().view(n, nq, d), v, bad, list(range(200 - n, 200)), d ** -0.5)
        assert ((got.double().cpu().view(n, nq, d) - out).abs() <= tolerance(torch.bfloat16, out, size, score, d, 200, torch.float16 if n == 1 else torch.bfloat16)).all()
    ops.copy_pages([pool.codes, pool.words], last, [0, 1, 2, 3])
    first = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    assert torch.equal(ops.read_kv8(pool.codes, pool.words, first, [200], torch.bfloat16), ops.read_kv8(pool.codes, pool.words, pool.table, [200], torch.bfloat16))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", ["D", "H"])
def test_captured_mixed_steps(model_folders, name, dtype):
    """Steps of single tokens beside portions: captured and replayed they give the same again."""
    from pytriton_llama_b200 import EngineConfig, SamplingParams
    from pytriton_llama_b200.engine.llm import LLM
    folder = model_folders(name, stored_dtype(dtype))
    vocab = TINY[name]["vocab_size"]
    prompts = [random_tokens(n, vocab, n) for n in (33, 5, 200, 17, 64, 150, 90)]
    got = []
    for compiled in (True, True):
        llm = LLM(folder, EngineConfig(dtype=dtype, page_size=max(16, PAGE_SIZE[name]), max_gpu_num_blocks=120, max_seq_len=256, max_num_seqs=4, seed=5, cache_bits=8,
                                       max_batched_tokens=48, compiled_model=compiled, capture_mixed_steps=compiled))
        reqs = [llm.add_request(p, SamplingParams(temperature=0.0, max_gen_len=12, top_logprobs=3)) for p in prompts]
        for _ in llm.run():
            pass
        llm.engine.check_device_status()
        llm.engine.cache.check_invariants()
        assert all(len(r.output) == 12 and all(map(math.isfinite, r.logprobs)) for r in reqs)
        got.append([(r.output, r.logprobs, r.entropies, r.top_logprobs) for r in reqs])
    assert got[0] == got[1]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [False, True])
def test_a_captured_mixed_step(ops, split, dtype):
    nq, G, d, ps = 8, 2, 64, 16
    forced = Forced(ops, split_portions=split)
    first, pool, qkv, req, pos, hints = run_attention(forced, nq, G, d, ps, LONG_PORTIONS["mixed"], dtype)
    req, pos = req.cuda(), torch.tensor(pos, dtype=torch.int32, device="cuda")
    call = lambda: ops.paged_attention8(qkv, pool.codes, pool.words, pool.table, req, pos, nq, G, d, ps, d ** -0.5, hints=hints)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    side = torch.cuda.Stream()
    for _ in range(5):
        out.fill_(math.nan)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        between = call()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, first) and torch.equal(between, first)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("d,ps", [(64, 16), (64, 64), (128, 32)])
@pytest.mark.parametrize("held", [0, 90, 640])
def test_portions_whose_table_ends_before_their_positions(ops, held, d, ps, split, dtype):
    """Positions behind the table's width have no page: they are not seen, whichever kernel runs, by parts of the keys too, and a row
    that sees no other is zeros."""
    nq, G, t, total = 4, 2, DTYPES[dtype], 1400
    pool = Pool(ops, G, d, ps, [total], seed=3)
    pool.append([total], values(total, G, d, seed=4, spread=1), dtype=t)
    v, bad = pool.plain.read(pool.tables[0], total)
    width = max(1, held // ps)
    keys = width * ps if held else 0
    narrow, wide = pool.table[:, :width].contiguous(), pool.table.clone()
    wide[:, width:] = -1
    if not held:
        narrow, wide = torch.full_like(narrow, -1), torch.full_like(wide, -1)
    for n, window in ((24, 0), (150, 0), (300, 0), (24, 33), (300, 900)):
        q = torch.randn((n, nq * d), generator=torch.Generator().manual_seed(n)).to(t)
        pos = torch.arange(total - n, total, dtype=torch.int32, device="cuda")
        got = []
        for table in (narrow, wide):
            hints = Forced(ops, split_portions=split).hints_for([n], [total])
            got.append(ops.paged_attention8(q.cuda(), pool.codes, pool.words, table, torch.zeros(n, dtype=torch.int32, device="cuda"), pos, nq, G, d, ps,
                                            d ** -0.5, window=window, hints=hints))
        assert torch.equal(*got)
        mine = got[0].double().cpu().view(n, nq, d)
        for i in range(0, n, 23):
            first = max(0, total - n + i - window + 1) if window else 0
            seen = slice(first, keys)
            if first >= keys:
                assert not mine[i].any()
                continue
            out, size, score = attend(q[i:i + 1].double().view(1, nq, d), v[seen], bad[seen], [keys - first - 1], d ** -0.5)
            assert ((mine[i] - out[0]).abs() <= tolerance(t, out, size, score, d, total, torch.bfloat16)[0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", [{}, {"single_form": (0, 4)}, {"single_form": (4, 8)}, {"split_portions": True}, {"split_portions": False}],
                         ids=["chosen", "units", "cluster", "mma", "tensor memory"])
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 16), (3, 1, 128, 32), (5, 5, 48, 16)])
def test_a_scale_of_zero_is_the_mean_of_the_values_in_sight(ops, nq, G, d, ps, form, dtype):
    """Masked keys among them: 0 times their -inf is no number.  With a missing page and a window too."""
    t, step = DTYPES[dtype], [(1, 700), (40, 600), (1, 3), (130, 0), (300, 5)]
    lens = [n + c for n, c in step]
    pool = Pool(ops, G, d, ps, lens, seed=d)
    kv = [values(n, G, d, seed=i, spread=1) for i, n in enumerate(lens)]
    pool.append(lens, torch.cat(kv), dtype=t)
    table = pool.table.clone()
    gone = {r: 0 if n < 3 * ps else 2 for r, n in enumerate(lens)}
    for r, b in gone.items():
        if b:
            table[r, b] = -1
    T = sum(n for n, _ in step)
    q = torch.randn((T, nq * d), generator=torch.Generator().manual_seed(1)).to(t)
    req = torch.cat([torch.full((n,), r) for r, (n, _) in enumerate(step)]).int()
    pos = torch.cat([torch.arange(c, c + n) for n, c in step]).int()
    for window in (0, 77):
        hints = Forced(ops, **form).hints_for([n for n, _ in step], lens)
        got = ops.paged_attention8(q.cuda(), pool.codes, pool.words, table, req.cuda(), pos.cuda(), nq, G, d, ps, 0.0, window=window, hints=hints)
        at = 0
        for r, (n, c) in enumerate(step):
            v, bad = pool.plain.read(pool.tables[r], n + c)
            for i in range(0, n, 13):
                p = c + i
                keys = [k for k in range(max(0, p - window + 1) if window else 0, p + 1) if not gone[r] or k // ps != gone[r]]
                mine = got[at + i].double().cpu().view(nq, d)
                out, size, score = attend(torch.zeros((1, nq, d), dtype=torch.float64), v[keys], bad[keys], [len(keys) - 1], 0.0)
                assert ((mine - out[0]).abs() <= tolerance(t, out, size, score, d, n + c, torch.float16 if n == 1 else torch.bfloat16)[0]).all(), (r, i, window)
            at += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [False, True])
def test_integers_worked_out_on_the_device_right_before_the_call(ops, split, dtype):
    """Slots, positions, table and tiles are results of the kernel before: the same as with integers that were there long ago."""
    nq, G, d, ps, t, total = 4, 2, 64, 16, DTYPES[dtype], 700
    forced = Forced(ops, split_portions=split)
    pool = Pool(ops, G, d, ps, [total], seed=3)
    kv = values(total, G, d, seed=4, spread=1)
    q = torch.randn((total, nq * d), generator=torch.Generator().manual_seed(1))
    f = (1.0 / 10000 ** (torch.arange(0, d, 2) / d)).cuda()
    qkv, slots, pos = pool.append([total], kv, nq=nq, q=q, inv_freq=f, rot=d, dtype=t)
    hints = forced.hints_for([total], [total])
    where = torch.zeros(total, dtype=torch.int32, device="cuda"), torch.tensor(pos, dtype=torch.int32, device="cuda")
    args = (nq, G, d, ps, d ** -0.5)
    first = ops.paged_attention8(qkv, pool.codes, pool.words, pool.table, *where, *args, hints=hints)
    held = ops.read_kv8(pool.codes, pool.words, pool.table, [total], t)
    codes, words = torch.zeros_like(pool.codes), torch.zeros_like(pool.words)
    ints = {k: torch.zeros_like(v) for k, v in dict(pos=where[1], slots=where[1], table=pool.table, f=f.int()).items()}
    f_new = torch.zeros_like(f)
    tiles = hints.work["prefill_tiles"].tensor
    right = tiles.clone()
    slots = torch.tensor(slots, dtype=torch.int32, device="cuda")
    for _ in range(10):
        again = torch.cat([q, kv.reshape(total, -1)], 1).to(t).cuda()
        for x in (codes, words, f_new, tiles, *ints.values()):
            x.zero_()
        torch.add(where[1], 0, out=ints["pos"])
        torch.mul(f, 1, out=f_new)
        torch.add(slots, 0, out=ints["slots"])
        ops.rope_kv8_write(again, ints["pos"], f_new, d, ints["slots"], codes, words, *args[:4])
        torch.add(pool.table, 0, out=ints["table"])
        assert torch.equal(ops.read_kv8(codes, words, ints["table"], [total], t), held)
        ints["table"].zero_()
        torch.add(right, 0, out=tiles)
        torch.add(pool.table, 0, out=ints["table"])
        out = ops.paged_attention8(again, codes, words, ints["table"], where[0], ints["pos"], *args, hints=hints)
        assert torch.equal(out, first) and torch.equal(again, qkv)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", [{}, {"single_form": (0, 4)}, {"single_form": (4, 8)}, {"split_portions": True}, {"split_portions": False}],
                         ids=["chosen", "units", "cluster", "mma", "tensor memory"])
@pytest.mark.parametrize("nq,G,d,ps", [(4, 2, 64, 32), (8, 1, 128, 64), (3, 3, 64, 128), (5, 5, 48, 48)])
def test_what_memory_held_before_reaches_no_row(ops, nq, G, d, ps, form, dtype):
    """Words and codes of blocks that no token was written to, in pages that the last tokens lie in: exponents that no value has, marks, and codes at both
    ends.  What comes out is the same as over zeros."""
    t, step = DTYPES[dtype], [(1, 700), (13, 825), (40, 600), (1, 3), (256, 4), (3, 0)]
    lens = [n + c for n, c in step]
    T = sum(n for n, _ in step)
    kv = torch.cat([values(n, G, d, seed=i, spread=1) for i, n in enumerate(lens)])
    q = torch.randn((T, nq * d), generator=torch.Generator().manual_seed(1)).to(t).cuda()
    req = torch.cat([torch.full((n,), r) for r, (n, _) in enumerate(step)]).int().cuda()
    pos = torch.cat([torch.arange(c, c + n) for n, c in step]).int().cuda()
    got = []
    for word, code in ((0, 0), (-1, 255), (-1, 0), (255, 255), (254, 0), (1, 255), (4, 0), (6, 255), (7, 0), (15, 255), (16, 0)):
        pool = Pool(ops, G, d, ps, lens, seed=5)
        pool.words.fill_(word)
        pool.codes.fill_(code)
        pool.append(lens, kv, dtype=t)
        hints = Forced(ops, **form).hints_for([n for n, _ in step], lens)
        got.append(ops.paged_attention8(q, pool.codes, pool.words, pool.table, req, pos, nq, G, d, ps, d ** -0.5, hints=hints))
    assert torch.isfinite(got[0]).all()
    for other in got[1:]:
        assert torch.equal(other, got[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", [{}, {"single_form": (0, 4)}, {"single_form": (4, 8)}, {"split_portions": True}, {"split_portions": False}],
                         ids=["chosen", "units", "cluster", "mma", "tensor memory"])
@pytest.mark.parametrize("step", [[(1, 300)], [(40, 300)], [(1, 300), (40, 600), (1, 3), (300, 4)]], ids=["singles", "portion", "mixed"])
def test_rows_behind_the_last_request_are_zeros(ops, step, form, dtype):
    """Whatever the memory of the output held before."""
    torch.full((5000, 256), math.nan, dtype=DTYPES[dtype], device="cuda")
    got = run_attention(Forced(ops, **form), 4, 2, 64, 16, step, dtype, extra=5)[0]
    assert not got[sum(n for n, _ in step):].any()
