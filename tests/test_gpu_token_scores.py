"""Log-probabilities of given tokens, entropy and the best alternatives, against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pytriton_llama_b200.ops.cuda import CudaOps
    return CudaOps(torch.device("cuda:0"))


def check(ops, logits, tokens, top):
    lp, ent, best, ids = [t.cpu() for t in ops.token_scores(logits, tokens, top)]
    x, tok = logits.cpu(), tokens.cpu().long()
    rows, vocab = x.shape
    k = min(top, vocab)
    assert lp.shape == (rows,) and ent.shape == (rows,) and best.shape == (rows, k) and ids.shape == (rows, k) and ids.dtype == torch.int32
    # ids: NaN behind -inf, equal ones by their index
    order = torch.where(torch.isnan(x), torch.tensor(-math.inf), x)
    rank = torch.sort(order.double() - torch.isnan(x).double() * 1e-300, dim=-1, descending=True, stable=True)[1]
    fine = [j for j in range(rows) if not torch.isnan(x[j]).any()]
    assert torch.equal(ids[fine].long(), rank[fine, :k])
    for j in range(rows):
        if j not in fine:      # numbers first
            n = int((~torch.isnan(x[j])).sum())
            have = [i for i in rank[j].tolist() if not math.isnan(x[j, i])] + [i for i in range(vocab) if math.isnan(x[j, i])]
            assert ids[j].tolist() == have[:k], (j, n)
    full = torch.log_softmax(x.double(), -1)
    p = full.exp()
    H = -torch.where(p > 0, p * full, torch.zeros((), dtype=torch.float64)).sum(-1)
    odd = torch.isnan(x).any(-1) | (x == math.inf).any(-1) | (x.amax(-1) == -math.inf)
    H[odd] = math.nan
    inside = (tok >= 0) & (tok < vocab)
    want = full.gather(1, tok.clamp(0, vocab - 1)[:, None])[:, 0].masked_fill(~inside, -math.inf)
    want[odd] = math.nan
    alt = full.gather(1, rank[:, :k])
    alt[odd] = math.nan
    # log S: float32 sums along chains of at most 400 and a few exponentials' ulps; x - m and the difference round once each, half a step
    # of a result of size |x - m|; U's terms e^z z are at most 1/e, their number counts through S, its chains as S's
    eps = 2.0 ** -24
    size = torch.where(torch.isfinite(x), x, torch.zeros(())).abs().amax(-1).double()
    lse_err = 450 * eps + 4 * eps * (size * 2 + math.log(vocab))

    def close(got, ref, tol):
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
        ok = torch.isfinite(ref)
        err = ((got.double() - ref).abs() / tol)[ok]
        assert err.numel() == 0 or err.max() <= 1, float(err.max())
    close(lp, want, lse_err + 2 * eps * want.abs().nan_to_num(posinf=0))
    close(best, alt, (lse_err[:, None] + 2 * eps * alt.abs().nan_to_num(posinf=0)))
    close(ent, H, lse_err + 450 * eps * (H.abs().nan_to_num() + math.log(vocab)))


def logits_of(rows, vocab, seed, gain=3.0):
    return torch.randn((rows, vocab), generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * gain


def tokens_of(rows, vocab, seed=0):
    return torch.randint(0, vocab, (rows,), generator=torch.Generator("cuda").manual_seed(seed), device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 33), (1, 4095), (2, 8191), (2, 8193), (4, 32001), (3, 128256), (1, 65537), (7, 50257),
                                        (301, 10007), (2400, 515)])
def test_scores(ops, rows, vocab, top):
    check(ops, logits_of(rows, vocab, vocab), tokens_of(rows, vocab), top)


@pytest.mark.parametrize("rows,vocab", [(2, 8200), (1, 128256), (3, 40001)])
def test_orders_that_fill_the_list(ops, rows, vocab):
    up = torch.arange(vocab, device="cuda", dtype=torch.float32)[None].expand(rows, vocab) / vocab * 20
    for x in (up, up.flip(1), torch.zeros_like(up), (up * 3).floor(), torch.where(up.long() % 7 == 0, up, torch.zeros_like(up))):
        check(ops, x.contiguous(), tokens_of(rows, vocab), 32)
        check(ops, x.contiguous(), tokens_of(rows, vocab), 3)
    # the largest all in neighbouring places, at the end, and ties across the slices' borders
    x = logits_of(rows, vocab, 1)
    x[:, -40:] = 50.0 + torch.arange(40, device="cuda") % 3
    check(ops, x, tokens_of(rows, vocab), 32)


def test_masked_rows(ops):
    vocab = 20011
    x = logits_of(8, vocab, 2)
    x[0] = -math.inf                            # nothing left
    x[1] = -math.inf
    x[1, 17000] = 2.0                           # one token left
    x[2, ::2] = -math.inf
    x[3, 5] = math.nan
    x[4, 19999] = math.inf
    x[5] = torch.finfo(torch.float32).min       # the lowest numbers everywhere
    x[6, :-1] = torch.finfo(torch.float32).min
    x[7] = math.nan
    x[7, 3], x[7, 4] = 1.0, -math.inf
    t = tokens_of(8, vocab)
    t[1], t[2], t[6] = 17000, 2, vocab - 1
    check(ops, x, t, 12)
    t[0], t[1], t[2], t[5] = -1, vocab, 3, 2 ** 31 - 1       # outside the vocabulary
    check(ops, x, t, 0)
    x[:, :] = -0.0
    x[:, 7::9] = 0.0                            # equal to -0
    check(ops, x, t.clamp(0, vocab - 1), 32)


def test_agrees_with_the_token_logprobs(ops):
    x, t = logits_of(64, 128256, 5), tokens_of(64, 128256)
    assert (ops.token_scores(x, t)[0] - ops.token_logprobs(x, t)).abs().max() < 1e-5


def test_rows_of_a_view_and_no_rows(ops):
    base = logits_of(1, 4 * 5003 + 3, 1).flatten()
    for off in (1, 2, 3):
        check(ops, base[off:off + 4 * 5003].view(4, 5003), tokens_of(4, 5003), 7)
    out = ops.token_scores(torch.empty((0, 50), device="cuda"), tokens_of(0, 50), 4)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 4), (0, 4)]


def test_two_graphs_at_once_and_the_same_bits(ops):
    calls = []
    for seed, rows in ((1, 3), (2, 40)):
        x, t = logits_of(rows, 60001, seed), tokens_of(rows, 60001)
        want = ops.token_scores(x, t, 20)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.token_scores(x, t, 20)
        calls.append((g, out, want, torch.cuda.Stream()))
    for _ in range(10):
        for g, out, want, s in calls:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for g, out, want, s in calls:
            torch.cuda.current_stream().wait_stream(s)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
