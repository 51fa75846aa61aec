"""The draw of tokens on the GPU against the 64-bit restatement: tokens equal, log probabilities to f32 rounding."""

import numpy as np
import pytest
import torch

from oracle import prefix as OP
from sgl_amd_mono_b200.sampling import SampleOp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, op=None, out=None):
    """Draws and compares every row.  A draw may differ only where u lies within 2^-36 of a border of the running sum:
    masses are exact sums of weights rounded to 2^-45 of the largest (and of f64 exponentials)."""
    rows, vocab = logits.shape
    d = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    if out is None:
        op = op or SampleOp(vocab, DEV, max_rows=rows)
        out = op(d(logits), d(u), d(temperature), d(top_k), d(top_p), d(min_p))
    token, logprob = (x.cpu() for x in out)
    x = logits.float().numpy()
    for r in range(rows):
        args = [float("nan") if a is None else a[r].item() for a in (temperature, top_k, top_p, min_p)]
        want, lp, gap = OP.sample_row(x[r], float(u[r]), 1.0 if temperature is None else args[0], 0 if top_k is None else args[1],
                                      1.0 if top_p is None else args[2], 0.0 if min_p is None else args[3])
        assert gap > 2.0**-36, "the test's own numbers lie on a border"
        assert int(token[r]) == want, f"row {r}: token {int(token[r])}, expected {want}"
        if want >= 0:
            # every weight is rounded by at most 2^-45 of the largest, so their sum Z, which is at least the largest, by at
            # most vocab 2^-45 of itself, and log Z by as much
            assert abs(float(logprob[r]) - lp) <= abs(lp) * 2.0**-24 + 2.0**-40 + vocab * 2.0**-45, f"row {r}"
        else:
            assert float(logprob[r]) == -np.inf
    return token


def _logits(rows, vocab, seed=0, rounded=False, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    return x.bfloat16().float() if rounded else x


def _u(rows, seed=7):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 33), (4, 1000), (3, 4097), (2, 50001), (20, 129280), (1, 300001)])
@pytest.mark.parametrize("rounded", [False, True])
def test_no_filter(rows, vocab, rounded):
    _check(_logits(rows, vocab, rounded=rounded), _u(rows))


@pytest.mark.parametrize("vocab", [7, 1000, 129280])
@pytest.mark.parametrize("rounded", [False, True])
def test_each_filter_and_all_together(vocab, rounded):
    rows = 24
    x, u = _logits(rows, vocab, 1, rounded), _u(rows, 3)
    g = torch.Generator().manual_seed(5)
    temperature = 0.25 + torch.rand(rows, generator=g) * 2
    top_k = torch.randint(1, max(2, min(vocab, 400)), (rows,), generator=g).to(torch.int32)
    top_p = torch.rand(rows, generator=g) * 0.98 + 0.01
    min_p = torch.rand(rows, generator=g) * 0.2
    _check(x, u, temperature)
    _check(x, u, top_k=top_k)
    _check(x, u, top_p=top_p)
    _check(x, u, min_p=min_p)
    _check(x, u, temperature, top_k, top_p, min_p)


def test_values_that_switch_filters_off_and_greedy_rows():
    x = _logits(8, 5000, 2)
    u = _u(8)
    inf, nan = float("inf"), float("nan")
    temperature = torch.tensor([0.0, -1.0, nan, 1.0, 1.0, 1.0, 1.0, inf])
    top_k = torch.tensor([5, 0, 7, 0, -1, 9999, 5000, 2**31 - 1], dtype=torch.int32)
    top_p = torch.tensor([0.5, 1.0, 0.3, 1.0, 2.0, nan, 1.0, inf])
    min_p = torch.tensor([0.0, 0.1, 0.0, -1.0, nan, 0.0, -inf, 0.0])
    token = _check(x, u, temperature, top_k, top_p, min_p)
    assert token[:3].tolist() == x[:3].argmax(1).tolist()


def test_borders_of_u_and_small_filters():
    x = torch.tensor([0.0, 1.0, 2.0, 1.0]).repeat(8, 1)
    op = SampleOp(4, DEV, max_rows=8)
    u = torch.tensor([0.0, -1.0, float("nan"), 1.0, 5.0, 2.0**-149, float(np.nextafter(np.float32(1), np.float32(0))), 0.25])
    token, _ = op(x.to(DEV), u.to(DEV))
    assert token.tolist()[:7] == [0, 0, 0, 3, 3, 0, 3]
    one = torch.ones(8)
    # filters that keep only the best token, whatever u is
    for kw in (dict(top_k=torch.ones(8, dtype=torch.int32)), dict(top_p=one * 0), dict(top_p=one * 1e-9), dict(top_p=-one), dict(min_p=one), dict(min_p=one * 3)):
        token, _ = op(x.to(DEV), u.to(DEV), **{k: v.to(DEV) for k, v in kw.items()})
        assert token.tolist() == [2] * 8, kw


def test_equal_logits_keep_the_lowest_indices():
    rows, vocab = 16, 3000
    x = torch.full((rows, vocab), 1.5)
    x[8:, ::3] = 2.5
    u = _u(rows, 11)
    _check(x, u)
    _check(x, u, top_k=torch.full((rows,), 1200, dtype=torch.int32))
    token = _check(x, u, top_k=torch.full((rows,), 7, dtype=torch.int32))
    assert int(token[:8].max()) < 7 and int(token[8:].max()) <= 18 and not (token[8:] % 3).any()
    _check(x, u, top_p=torch.full((rows,), 0.37))


def test_borders_at_zero_and_among_the_smallest_numbers():
    """Ties at 0 and -0 (equal), the filter's border there, and subnormal logits on both sides of it."""
    rows, vocab = 12, 900
    x = torch.full((rows, vocab), -1.0)
    x[:, ::3] = 0.0
    x[:, 1::3] = -0.0
    x[:, 5] = 2.0
    x[:, 2] = -(2.0**-149)
    x[:, 8] = 2.0**-149
    u = _u(rows, 13)
    for k in (1, 2, 3, 300, 601, 602, 603):
        _check(x, u, top_k=torch.full((rows,), k, dtype=torch.int32))
    _check(x, u, top_p=torch.full((rows,), 0.5))
    _check(x, u, min_p=torch.full((rows,), 0.1353))
    _check(x, u, min_p=torch.full((rows,), 0.1354))


def test_infinities_nan_and_empty_rows():
    rows, vocab = 8, 1300
    x = _logits(rows, vocab, 4)
    inf, nan = float("inf"), float("nan")
    x[0] = -inf
    x[1] = nan
    x[2, 100:] = -inf
    x[3, ::2] = nan
    x[4, [5, 900]] = inf
    x[5] = -inf
    x[5, 77] = -3e38
    x[6] = 3e38
    x[7, 3] = -0.0
    x[7, 4:] = 0.0
    u = _u(rows, 2)
    k = torch.full((rows,), 50, dtype=torch.int32)
    token = _check(x, u)
    assert token[:2].tolist() == [-1, -1] and int(token[5]) == 77 and int(token[4]) in (5, 900)
    _check(x, u, top_k=k, top_p=torch.full((rows,), 0.9))
    _check(x, u, temperature=torch.full((rows,), 1e-6), min_p=torch.full((rows,), 0.5))
    assert _check(x, u, temperature=torch.zeros(rows)).tolist()[4] == 5


@pytest.mark.parametrize("spread", [0.01, 30.0])
def test_flat_and_sharp_rows(spread):
    rows = 12
    x, u = _logits(rows, 129280, 6, spread=spread), _u(rows, 8)
    _check(x, u, top_p=torch.linspace(0.05, 0.99, rows))
    _check(x, u, top_k=torch.arange(1, 120001, 10000)[:rows].to(torch.int32))


def test_bf16_logits_strided_rows_and_odd_addresses():
    x, u = _logits(5, 4099, 9), _u(5)
    kw = dict(top_k=torch.full((5,), 77, dtype=torch.int32), top_p=torch.full((5,), 0.8))
    _check(x.bfloat16(), u, **kw)
    for dt in (torch.float32, torch.bfloat16):
        wide = torch.full((5, 4099 + 10), 99.0, dtype=dt, device=DEV)
        for first in (0, 1, 3):
            wide[:] = 99.0
            wide[:, first : first + 4099] = x.to(DEV)
            op = SampleOp(4099, DEV, max_rows=9)
            out = op(wide[:, first : first + 4099], u.to(DEV), **{k: v.to(DEV) for k, v in kw.items()})
            _check(x.to(dt), u, **kw, out=out)


def test_many_rows_repeat_to_the_bit_and_follow_a_graph():
    rows, vocab = 300, 2000
    x, u = _logits(rows, vocab, 10), _u(rows, 1)
    op = SampleOp(vocab, DEV, max_rows=rows)
    p = torch.full((rows,), 0.9)
    xd, ud, pd = x.to(DEV), u.to(DEV), p.to(DEV)
    token, logprob = (t.clone() for t in op(xd, ud, top_p=pd))
    _check(x, u, top_p=p, out=(token, logprob))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = op(xd, ud, top_p=pd)
    torch.cuda.current_stream().wait_stream(side)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], token) and torch.equal(out[1], logprob)
    u2 = _u(rows, 99)
    ud.copy_(u2)
    g.replay()
    torch.cuda.synchronize()
    _check(x, u2, top_p=p, out=out)


def test_refusals():
    op = SampleOp(100, DEV, max_rows=4)
    x, u = torch.zeros(4, 100, device=DEV), torch.zeros(4, device=DEV)
    op(x, u)
    for bad in (x.half(), x[:, :99], x.repeat(2, 1), x[0], x.cpu(), x.t().contiguous().t()):
        with pytest.raises(ValueError, match="logits"):
            op(bad, u)
    for name, bad in (("u", u.double()), ("u", u[:3]), ("top_k", u), ("top_p", u.int()), ("temperature", u.cpu()), ("min_p", u.repeat(2))):
        with pytest.raises(ValueError, match=name):
            op(**{"logits": x, "u": u, name: bad})


@pytest.mark.parametrize("together", [True, False])
@pytest.mark.parametrize("n", [1, 63, 64, 65, 127, 255, 256, 257, 700])
def test_borders_among_many_close_logits(n, together):
    """``n`` logits within a thousandth of each other (some equal) hold nearly all the mass, in one run or all over the
    row: the border lies among them, whether they are few enough to be ranked at once or not."""
    vocab, rows = 20000, 8
    g = torch.Generator().manual_seed(n)
    x = torch.randn(rows, vocab, generator=g) - 12
    for r in range(rows):
        at = torch.arange(n) + 4100 if together else torch.randperm(vocab, generator=g)[:n]
        x[r, at] = 3 + torch.randint(0, 8, (n,), generator=g) * 1e-4
    k = torch.tensor([1, max(1, n // 2), n, n + 1, 0, max(1, n - 1), 1, n // 3 + 1], dtype=torch.int32)
    p = torch.tensor([1.0, 1.0, 0.999, 1.0, 0.37, 0.5, 0.0, 0.9])
    mp = torch.tensor([0.0, 0.0, 0.0, 0.5, 0.0, 0.9997, 1.0, 0.0])
    _check(x, _u(rows, seed=n + 1), torch.tensor([0.7, 1.0, 1.3, 1.0, 2.0, 1.0, 1.0, 0.5]), k, p, mp)


def test_rank_zero_alone_is_the_first_of_the_largest():
    x = _logits(4, 5000, seed=3)
    x[:, [77, 4000]] = 9.0
    one = torch.ones(4, dtype=torch.int32)
    token = _check(x, torch.tensor([0.0, 0.5, 0.999, 0.3]), torch.tensor([1.0, 0.3, 5.0, 0.0]), one, torch.tensor([1.0, 0.0, 0.5, 1.0]), torch.tensor([0.0, 1.0, 0.2, 0.0]))
    assert (token == 77).all()


@pytest.mark.parametrize("rows,vocab", [(60, 7), (60, 1000), (60, 4099), (60, 20480), (60, 20481), (90, 8193), (90, 40960), (150, 9000), (40, 81920), (40, 81921)])
@pytest.mark.parametrize("rounded", [False, True])
def test_many_rows_of_small_vocabularies(rows, vocab, rounded):
    x, u = _logits(rows, vocab, vocab, rounded), _u(rows, vocab)
    g = torch.Generator().manual_seed(5)
    k = torch.randint(0, min(vocab, 300) + 1, (rows,), generator=g).to(torch.int32)
    p = torch.where(torch.arange(rows) % 3 == 0, torch.ones(rows), torch.rand(rows, generator=g) * 0.98 + 0.01)
    mp = torch.where(torch.arange(rows) % 4 == 0, torch.rand(rows, generator=g) * 0.2, torch.zeros(rows))
    t = torch.where(torch.arange(rows) % 7 == 6, torch.zeros(rows), torch.rand(rows, generator=g) + 0.4)
    x[1], x[2, : vocab // 2] = -float("inf"), float("nan")
    _check(x, u)
    _check(x.bfloat16() if rounded else x, u, t, k, p, mp)


@pytest.mark.parametrize("rows,vocab", [(4, 129280), (90, 40000), (150, 40000), (40, 20000), (24, 9000)])
def test_rows_of_rank_zero_alone_repeat_their_log_probability(rows, vocab):
    """Greedy rows and rows with top_k = 1 need no search of a border: what their CTAs exchange must not meet."""
    x, u = _logits(rows, vocab, vocab + rows), _u(rows, 3)
    temperature = torch.where(torch.arange(rows) % 2 == 0, torch.zeros(rows), torch.full((rows,), 1.7))
    k = torch.where(torch.arange(rows) % 2 == 0, torch.zeros(rows), torch.ones(rows)).to(torch.int32)
    op = SampleOp(vocab, DEV, max_rows=rows)
    args = [t.to(DEV) for t in (x, u, temperature, k)]
    token, logprob = (t.clone() for t in op(*args))
    _check(x, u, temperature, k, out=(token, logprob))
    for _ in range(30):
        again = op(*args)
        assert torch.equal(again[0], token) and torch.equal(again[1], logprob)


@pytest.mark.parametrize("rows,vocab", [(1, 8193), (18, 4097), (2, 40001)])
def test_short_loads_of_whole_clusters(rows, vocab):
    """Clusters of eight whose CTAs have next to nothing to load, one launch right after another."""
    op = SampleOp(vocab, DEV, max_rows=rows)
    x, u = _logits(rows, vocab, vocab), _u(rows, 5)
    p = torch.full((rows,), 0.8)
    args = [t.to(DEV) for t in (x, u)]
    outs = [tuple(t.clone() for t in op(*args, top_p=p.to(DEV))) for _ in range(20)]
    _check(x, u, top_p=p, out=outs[0])
    assert all(torch.equal(t, outs[0][0]) and torch.equal(lp, outs[0][1]) for t, lp in outs)


@pytest.mark.parametrize("vocab", [4, 3000, 50001])
def test_min_p_above_one_keeps_the_first_of_the_largest_alone(vocab):
    x = torch.zeros(6, vocab)
    x[:, 1:vocab:2] = 2.0
    mp = torch.tensor([1.0, float(np.nextafter(np.float32(1), np.float32(2))), 1.5, float("inf"), 3.0, 1.5])
    u = torch.tensor([0.9, 0.9, 0.9, 0.9, 0.0, 0.999])
    token = _check(x, u, min_p=mp)
    assert int(token[0]) > 1 and token[1:].tolist() == [1] * 5
    _check(x, u, torch.full((6,), 0.3), torch.full((6,), 3, dtype=torch.int32), torch.full((6,), 0.9), mp)


@pytest.mark.parametrize("rows", [1, 40])
def test_the_largest_vocabulary(rows):
    vocab = 393216
    x, u = _logits(rows, vocab, 21), _u(rows, 22)
    x[0] = 1.25  # all alike
    p = torch.where(torch.arange(rows) % 2 == 0, torch.full((rows,), 0.9), torch.ones(rows))
    k = torch.where(torch.arange(rows) % 3 == 2, torch.full((rows,), 200000), torch.zeros(rows)).to(torch.int32)
    _check(x, u)
    _check(x, u, top_k=k, top_p=p)
