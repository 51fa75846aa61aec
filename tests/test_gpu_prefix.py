"""Cache append and shared-prefix attention on the GPU through the public ops, against the 64-bit restatement."""

import pytest
import torch

from oracle import prefix as OP
from sgl_amd_mono_b200 import _lib as L
from sgl_amd_mono_b200 import ops
from sgl_amd_mono_b200.prefix import PrefixTables, QkvAppendOp, SharedPrefixAttnOp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
K_SCALE, V_SCALE = 0.0625, 0.046875


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------- append
def _append_inputs(tokens, hq, hk, rot, table=torch.bfloat16, seed=0, pages=None):
    g = _gen(seed)
    pages = pages or -(-tokens // 64) + 2
    x = torch.randn(tokens, (hq + 2 * hk) * 128, generator=g)
    ang = torch.arange(512, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    d = dict(x=x.bfloat16(), g_q=(torch.randn(128, generator=g) * 0.2).bfloat16(), g_k=(torch.randn(128, generator=g) * 0.2).bfloat16(),
             cos=ang.cos().to(table), sin=ang.sin().to(table), positions=torch.randint(0, 512, (tokens,), generator=g),
             slots=torch.randperm(pages * 64, generator=g)[:tokens])
    caches = [(torch.randn(pages, 64, hk, 128, generator=g) * 16).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2)]
    return d, caches


def _check_append(q, kc, vc, x, d, caches, hq, hk, interleaved, norm=True, eps=1e-6):
    gq, gk = (d["g_q"], d["g_k"]) if norm else (None, None)
    rq, rk, rv = OP.append_rows(x, hq, hk, gq, gk, eps, d["cos"], d["sin"], d["positions"], interleaved)
    # f32 arithmetic: a norm is a 128-term sum, a root and two products (relative 2^-20 of the value at most), a
    # rotation adds two products of the pair's size
    slack = 2.0**-19
    top = rq.abs().amax(-1, keepdim=True)
    assert torch.isfinite(q.float()).all()
    assert ((q.cpu().double() - rq).abs() <= rq.abs() * 2.0**-8 + top * slack).all()
    for got, before, ref, scale in ((kc, caches[0], rk, K_SCALE), (vc, caches[1], rv, V_SCALE)):
        want = OP.cache_values(before).reshape(-1, hk, 128)
        tol = torch.zeros_like(want)
        live = (d["slots"] >= 0) & (d["slots"] < want.shape[0])
        v = (ref / scale).clamp(-448, 448)
        at = d["slots"][live]
        want[at] = v[live]
        # E4M3: half a step is 2^-4 of the value, or 2^-10 below the smallest normal number
        tol[at] = (v.abs() * 2.0**-4).clamp(min=2.0**-10)[live] + v.abs().amax(-1, keepdim=True)[live] * slack
        have = OP.cache_values(got.cpu()).reshape(-1, hk, 128)
        assert ((have - want).abs() <= tol).all()
        # the other slots keep their bytes
        rest = torch.ones(want.shape[0], dtype=torch.bool)
        rest[at] = False
        assert torch.equal(got.cpu().reshape(-1, hk, 128)[rest], before.reshape(-1, hk, 128)[rest])


@pytest.mark.parametrize("tokens,hq,hk,rot,interleaved,table", [
    (1, 1, 1, 64, False, torch.bfloat16), (1, 12, 2, 64, False, torch.float32), (5, 3, 3, 16, True, torch.bfloat16),
    (16, 12, 2, 128, False, torch.bfloat16), (33, 7, 1, 48, False, torch.float32), (33, 5, 5, 96, True, torch.float32),
    (700, 48, 8, 64, True, torch.bfloat16), (1203, 20, 4, 112, False, torch.bfloat16)])
def test_append_rows(tokens, hq, hk, rot, interleaved, table):
    d, caches = _append_inputs(tokens, hq, hk, rot, table)
    op = QkvAppendOp(hq, hk, DEV, max_tokens=tokens, rot_dim=rot, interleaved=interleaved, k_scale=K_SCALE, v_scale=V_SCALE)
    kc, vc = (c.to(DEV) for c in caches)
    q = op(d["x"].to(DEV), *(d[k].to(DEV) for k in ("g_q", "g_k", "cos", "sin", "positions", "slots")), kc, vc)
    _check_append(q, kc, vc, d["x"], d, caches, hq, hk, interleaved)


def test_append_strided_rows_pads_far_positions_and_no_norm():
    tokens, hq, hk = 70, 12, 2
    d, caches = _append_inputs(tokens, hq, hk, 64)
    wide = torch.full((tokens, 2048 + 24), float("nan"), dtype=torch.bfloat16)
    wide[:, 8 : 8 + 2048] = d["x"]
    d["slots"][[0, 3]] = -1
    d["slots"][5] = caches[0].shape[0] * 64  # behind the cache: inserts nothing
    d["positions"][[1, 2]] = torch.tensor([-7, 10**12])
    op = QkvAppendOp(hq, hk, DEV, max_tokens=128, k_scale=K_SCALE, v_scale=V_SCALE)
    kc, vc = (c.to(DEV) for c in caches)
    q = op(wide.to(DEV)[:, 8 : 8 + 2048], None, None, *(d[k].to(DEV) for k in ("cos", "sin", "positions", "slots")), kc, vc)
    _check_append(q, kc, vc, d["x"], d, caches, hq, hk, False, norm=False)
    # without slots nothing is inserted
    k2 = kc.clone()
    op(d["x"].to(DEV), None, None, *(d[k].to(DEV) for k in ("cos", "sin", "positions")), None, kc, vc)
    assert torch.equal(k2, kc)


@pytest.mark.parametrize("tokens,nsum", [(1, 1), (16, 3), (9, 7)])
def test_append_from_partial_sums(tokens, nsum):
    hq, hk = 12, 2
    d, caches = _append_inputs(tokens, hq, hk, 64)
    parts = torch.randn(nsum, 16, 2048, generator=_gen(3))
    op = QkvAppendOp(hq, hk, DEV, max_tokens=16, k_scale=K_SCALE, v_scale=V_SCALE)
    kc, vc = (c.to(DEV) for c in caches)
    q = op(parts.to(DEV), *(d[k].to(DEV) for k in ("g_q", "g_k", "cos", "sin", "positions", "slots")), kc, vc, tokens=tokens)
    # the f32 sum of the parts is the operator's input: added in order, as the kernel does
    x = torch.zeros(16, 2048)
    for p in parts:
        x = x + p
    _check_append(q, kc, vc, x[:tokens], d, caches, hq, hk, False)


def test_append_extreme_values():
    hq, hk = 2, 1
    d, caches = _append_inputs(4, hq, hk, 64)
    x = d["x"].float().view(4, 4, 128)
    x[0] = 0  # a zero head stays zero under eps
    x[1] *= 1e4  # saturates V
    x[2, 3, 5] = float("inf")
    x[3, 3, 7] = float("nan")
    op = QkvAppendOp(hq, hk, DEV, max_tokens=4, k_scale=K_SCALE, v_scale=V_SCALE)
    kc, vc = (c.to(DEV) for c in caches)
    q = op(x.bfloat16().view(4, -1).to(DEV), *(d[k].to(DEV) for k in ("g_q", "g_k", "cos", "sin", "positions", "slots")), kc, vc)
    v = OP.cache_values(vc.cpu()).reshape(-1, 128)[d["slots"]]
    assert (q[0] == 0).all() and (v[0] == 0).all()
    assert v[1].abs().max() == 448
    assert v[2, 5] == 448 and torch.isfinite(v[2]).all()
    assert torch.isnan(v[3, 7]) and torch.isnan(v[3]).sum() == 1
    assert torch.isfinite(q).all()


def test_append_far_cache_offsets():
    """Slots behind 2^31 bytes of a cache (and the attention that reads them) use 64-bit offsets."""
    pages, hk, hq = 33000, 8, 8  # 2.16 GB a cache
    kc, vc = (torch.zeros(pages, 64, hk, 128, dtype=torch.uint8, device=DEV) for _ in range(2))
    d, _ = _append_inputs(64, hq, hk, 64, pages=4)
    d["slots"] = (pages - 1) * 64 + torch.arange(64)
    op = QkvAppendOp(hq, hk, DEV, max_tokens=64, k_scale=K_SCALE, v_scale=V_SCALE)
    q = op(d["x"].to(DEV), *(d[k].to(DEV) for k in ("g_q", "g_k", "cos", "sin", "positions", "slots")), kc, vc)
    last = [c[-1:].cpu() for c in (kc, vc)]
    d2 = dict(d, slots=torch.arange(64))
    _check_append(q, last[0], last[1], d["x"], d2, [torch.zeros(1, 64, hk, 128, dtype=torch.uint8)] * 2, hq, hk, False)
    assert int(kc[:-1].count_nonzero()) == 0
    attn = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=1, max_seqs=1, k_scale=K_SCALE, v_scale=V_SCALE)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    t = PrefixTables(i32(0, 1), i32(pages - 1).view(1, 1), i32(64))
    out = attn(q[63:64], kc, vc, _dev(t))
    _check_attend(out, q[63:64].cpu(), last, PrefixTables(t.q_start, i32(0).view(1, 1), t.lens), attn)


# ---------------------------------------------------------------- attention
def _dev(t: PrefixTables) -> PrefixTables:
    return PrefixTables(*(None if x is None else x.to(DEV) for x in (t.q_start, t.page_table, t.lens, t.group_start, t.prefix_table, t.prefix_lens)))


def _tables(ntok, own, starts, prefix, seed=0, spare=1, columns=0):
    """Tables over pages in random order; returns (tables, pages)."""
    need = [-(-n // 64) for n in list(prefix) + list(own)]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=_gen(seed)).to(torch.int32)
    rows, at = [], 0
    for n in need:
        rows.append(order[at : at + n])
        at += n

    def table(part, extra):
        w = max([len(r) for r in part] + [1]) + extra
        t = torch.full((len(part), w), -1, dtype=torch.int32)
        for i, r in enumerate(part):
            t[i, : len(r)] = r
        return t

    i32 = lambda v: torch.tensor(list(v), dtype=torch.int32)  # noqa: E731
    q_start = i32([0] + torch.tensor(ntok).cumsum(0).tolist())
    p = len(prefix)
    if not p:
        return PrefixTables(q_start, table(rows, columns), i32(own)), pages
    return PrefixTables(q_start, table(rows[p:], columns), i32(own), i32(starts), table(rows[:p], columns), i32(prefix)), pages


def _caches(pages, hk, seed=1):
    g = _gen(seed)
    return [(torch.randn(pages, 64, hk, 128, generator=g) * 16).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2)]


def _check_attend(out, q, caches, t, op, rows=None):
    ref, mag, big, seen = OP.attend(q, *caches, t.q_start, t.page_table, t.lens, t.group_start, t.prefix_table, t.prefix_lens,
                                    op.k_scale, op.v_scale, op.sm_scale)
    # weights: f16 rounding 2^-11; a score is 128 products added in f32 steps that may truncate (2^-23 of the running
    # sum each) and enters numerator and denominator; the value sums add one step per 16 keys; the store rounds to bf16
    tol = ref.abs() * 2.0**-8 + mag * (2.0**-11 + 2 * (128 * 2.0**-23 * big[..., None] + 2.0**-20) + (seen[:, None, None] / 16 + 16) * 2.0**-23)
    live = ~torch.isnan(ref) if rows is None else rows
    err = (out.cpu().double() - ref).abs()
    assert (err[live] <= tol[live]).all(), f"off by {(err - tol)[live].max():.3g} beyond the bound, {int((err > tol)[live].sum())} values"
    return ref


def _attend(hq, hk, ntok, own, starts, prefix, seed=0, columns=0, qmul=2.0, **kw):
    t, pages = _tables(ntok, own, starts, prefix, seed, columns=columns)
    caches = _caches(pages, hk)
    tokens = sum(ntok)
    q = (torch.randn(tokens, hq, 128, generator=_gen(seed + 5)) * qmul).bfloat16()
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=tokens, max_seqs=len(own), max_groups=max(1, len(prefix)), k_scale=K_SCALE, v_scale=V_SCALE, **kw)
    dc = [c.to(DEV) for c in caches]
    out = op(q.to(DEV), *dc, _dev(t))
    torch.cuda.synchronize()
    rc, words = ops.guard_read(op.guard)
    assert rc == 0, f"guard words {words}"
    _check_attend(out, q, caches, t, op)
    return op, q, caches, dc, t, out


@pytest.mark.parametrize("hq,hk,ntok,own,starts,prefix", [
    (1, 1, [1], [1], [0, 1], [1]),                                   # one key each
    (12, 2, [1], [64], [], []),                                      # no prefix, a whole page
    (12, 2, [1] * 4, [1, 63, 64, 65], [0, 4], [129]),                # page borders
    (8, 8, [1] * 3, [7, 200, 31], [0, 3], [64]),                     # one q head per kv head
    (16, 1, [1] * 5, [3, 70, 128, 1, 33], [0, 5], [700]),            # sixteen q heads on one
    (20, 4, [1] * 9, list(range(1, 200, 23))[:9], [0, 2, 3, 9], [300, 1, 65]),  # three groups
    (12, 2, [1] * 6, [5, 6, 7, 8, 9, 10], [1, 4], [100]),            # some sequences have no group
    (12, 2, [3, 1, 5, 2], [40, 1, 5, 130], [0, 4], [500]),           # several query tokens, causal
    (6, 1, [1] * 40, [1 + 7 * i for i in range(40)], [0, 40], [190]),   # more rows than one tile of the prefix
    (6, 3, [70, 1, 200], [70, 65, 333], [0, 2, 3], [77, 130]),       # prompt chunks
    (24, 2, [1] * 33, [9] * 33, [0, 33], [1111]),
    # kv heads that do not fill a group of heads, and more than one group
    (6, 3, [1, 2], [130, 70], [0, 2], [200]),
    (5, 5, [1, 1], [65, 3], [0, 2], [129]),
    (14, 7, [2, 1], [40, 300], [0, 1, 2], [10, 64]),
    (12, 12, [1] * 3, [63, 64, 1000], [0, 3], [65]),
    (16, 16, [1] * 2, [17, 200], [], []),
    (32, 2, [1] * 7, [500, 1, 16, 17, 31, 48, 49], [0, 7], [2000])])
def test_attend(hq, hk, ntok, own, starts, prefix):
    _attend(hq, hk, ntok, own, starts, prefix, columns=2)


def test_attend_empty_sides():
    """No prefix keys, no own keys, neither: the last gives zeros."""
    hq, hk = 6, 2
    t, pages = _tables([1, 1, 2, 1], [5, 1, 1, 1], [0, 2, 4], [64, 1], spare=2)
    t.lens[:] = torch.tensor([5, 0, 1, 0])   # sequence 2: its first token comes before its only key
    t.prefix_lens[:] = torch.tensor([64, 0])
    caches = _caches(pages, hk)
    q = torch.randn(5, hq, 128, generator=_gen(9)).bfloat16()
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=5, max_seqs=4, max_groups=2, k_scale=K_SCALE, v_scale=V_SCALE)
    out = op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t))
    ref = _check_attend(out, q, caches, t, op)
    assert (ref[2] == 0).all() and (out[2] == 0).all() and (out[4] == 0).all() and (ref[3] != 0).all()


def test_attend_rows_of_no_sequence_keep_their_values():
    hq, hk = 12, 2
    t, pages = _tables([1, 2], [30, 70], [0, 2], [100])
    t.q_start += 1  # token 0 and the tokens behind the last sequence belong to nobody
    caches = _caches(pages, hk)
    q = torch.randn(7, hq, 128, generator=_gen(2)).bfloat16()
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=7, max_seqs=2, k_scale=K_SCALE, v_scale=V_SCALE)
    mine = torch.full((7, hq, 128), 3.25, dtype=torch.bfloat16, device=DEV)
    out = op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t), out=mine)
    assert out.data_ptr() == mine.data_ptr()
    _check_attend(out, q, caches, t, op)
    assert (out[0] == 3.25).all() and (out[4:] == 3.25).all()


def test_attend_ignores_what_lies_in_masked_places():
    """Keys and values behind a length, pages outside the cache and unused columns: NaN bytes there change nothing."""
    hq, hk = 12, 2
    op, q, caches, dc, t, out = _attend(hq, hk, [1, 2, 1], [10, 70, 129], [0, 3], [200])
    want = out.clone()
    n = [c.clone() for c in caches]
    for tab, lens in ((t.page_table, t.lens), (t.prefix_table, t.prefix_lens)):
        for row, ln in zip(tab, lens):
            full, part = divmod(int(ln), 64)
            if part:
                for c in n:
                    c[int(row[full]), part:] = 0x7F
    used = set(int(p) for tab in (t.page_table, t.prefix_table) for p in tab.flatten() if p >= 0)
    for c in n:
        c[[p for p in range(c.shape[0]) if p not in used]] = 0xFF
    assert torch.equal(op(q.to(DEV), *(c.to(DEV) for c in n), _dev(t)), want)
    # a page number outside the cache is a page without keys
    t2 = PrefixTables(t.q_start, t.page_table.clone(), t.lens, t.group_start, t.prefix_table.clone(), t.prefix_lens)
    t2.prefix_table[0, 1] = caches[0].shape[0]
    t2.page_table[2, 0] = -5
    got = op(q.to(DEV), *dc, _dev(t2))
    _check_attend(got, q, caches, t2, op)
    # lengths beyond the columns are cut
    t3 = PrefixTables(t.q_start, t.page_table[:, :1].contiguous(), t.lens, t.group_start, t.prefix_table, t.prefix_lens)
    got = op(q.to(DEV), *dc, _dev(t3))
    _check_attend(got, q, caches, t3, op)


def test_attend_sharp_scores_and_nan_rows():
    """Scores far apart (one key takes all the weight, a sink in another block), and a NaN query: its own rows only."""
    hq, hk = 12, 2
    t, pages = _tables([1, 1], [100, 30], [0, 2], [640])
    caches = _caches(pages, hk)
    q = (torch.randn(2, hq, 128, generator=_gen(2)) * 30).bfloat16()
    q[0, 3] = float("nan")
    q[1, 5] *= 1e-30
    q[1, 6] = 0
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=2, max_seqs=2, k_scale=K_SCALE, v_scale=V_SCALE)
    out = op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t))
    assert torch.isnan(out[0, 3]).all() and int(torch.isnan(out).any(-1).sum()) == 1
    _check_attend(out, q, caches, t, op)


def test_attend_strided_queries_and_repeats_to_the_bit():
    hq, hk = 12, 2
    op, q, caches, dc, t, out = _attend(hq, hk, [1] * 5, [70] * 5, [0, 5], [900])
    want = out.clone()
    wide = torch.full((5, hq * 128 + 512), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, : hq * 128] = q.to(DEV).view(5, -1)
    again = op(wide[:, : hq * 128].unflatten(1, (hq, 128)), *dc, _dev(t))
    assert torch.equal(again, want)


def test_attend_in_a_graph_follows_the_tables():
    hq, hk = 12, 2
    op, q, caches, dc, t, _ = _attend(hq, hk, [1] * 3, [70, 10, 64], [0, 3], [300], columns=2)
    dt, qd = _dev(t), q.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = op(qd, *dc, dt)
    torch.cuda.current_stream().wait_stream(side)
    for lens, plen in (([70, 10, 64], 300), ([3, 1, 2], 17), ([70, 9, 33], 0)):
        t.lens[:], t.prefix_lens[:] = torch.tensor(lens), plen
        dt.lens.copy_(t.lens)
        dt.prefix_lens.copy_(t.prefix_lens)
        g.replay()
        torch.cuda.synchronize()
        _check_attend(out, q, caches, t, op)


def test_attend_refuses_starts_that_fall():
    hq, hk = 12, 2
    op, q, caches, dc, t, _ = _attend(hq, hk, [1] * 3, [70, 10, 64], [0, 3], [300])
    bad = _dev(t)
    bad.q_start.copy_(torch.tensor([0, 3, 0, 3]))
    op(q.to(DEV), *dc, bad)
    torch.cuda.synchronize()
    rc, words = ops.guard_read(op.guard)
    assert rc != 0 and words[2] == 105  # argument word: the tables' site + 1
    op.guard.zero_()
    bad = _dev(t)
    bad.group_start.copy_(torch.tensor([0, 9]))
    op(q.to(DEV), *dc, bad)
    rc, words = ops.guard_read(op.guard)
    assert rc != 0 and words[2] == 105
    op.guard.zero_()
    _check_attend(op(q.to(DEV), *dc, _dev(t)), q, caches, t, op)


def test_attend_on_a_side_stream_with_its_own_op():
    hq, hk = 12, 2
    a = _attend(hq, hk, [1] * 8, [70] * 8, [0, 8], [2000])
    b = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=8, max_seqs=8, k_scale=K_SCALE, v_scale=V_SCALE)
    op, q, caches, dc, t, out = a
    want, qd, dt = out.clone(), q.to(DEV), _dev(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            o2 = b(qd, *dc, dt)
        o1 = op(qd, *dc, dt)
    torch.cuda.synchronize()
    assert torch.equal(o1, want) and torch.equal(o2, want)


def test_append_then_attend_then_append():
    """A prompt's rows go to the cache once; three samples of it then take two steps each on the same pages."""
    hq, hk, eps = 12, 2, 1e-6
    prompt, seqs = 150, 3
    pages = 3 + seqs
    g = _gen(4)
    width = (hq + 2 * hk) * 128
    ang = torch.arange(512, dtype=torch.float64)[:, None] / 1e6 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    cos, sin = ang.cos().bfloat16(), ang.sin().bfloat16()
    gq, gk = ((torch.randn(128, generator=g) * 0.1).bfloat16() for _ in range(2))
    kc, vc = (torch.zeros(pages, 64, hk, 128, dtype=torch.uint8, device=DEV) for _ in range(2))
    app = QkvAppendOp(hq, hk, DEV, max_tokens=prompt, k_scale=K_SCALE, v_scale=V_SCALE)
    att = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=prompt, max_seqs=seqs, k_scale=K_SCALE, v_scale=V_SCALE)
    w = [x.to(DEV) for x in (gq, gk, cos, sin)]
    order = torch.tensor([4, 0, 2])
    at = torch.arange(prompt)
    x = torch.randn(prompt, width, generator=g).bfloat16()
    q = app(x.to(DEV), *w, at.to(DEV), (order[at // 64] * 64 + at % 64).to(DEV), kc, vc)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    # the prompt attends itself: one sequence, causal, no prefix
    t = PrefixTables(i32([0, prompt]), order.to(torch.int32).view(1, 3), i32([prompt]))
    out = att(q, kc, vc, _dev(t))
    _check_attend(out, q.cpu(), [kc.cpu(), vc.cpu()], t, att)
    own = torch.tensor([1, 3, 5])
    for step in range(2):
        x = torch.randn(seqs, width, generator=g).bfloat16()
        q = app(x.to(DEV), *w, torch.full((seqs,), prompt + step, device=DEV), (own * 64 + step).to(DEV), kc, vc)
        t = PrefixTables(i32([0, 1, 2, 3]), own.to(torch.int32).view(3, 1), i32([step + 1] * 3), i32([0, 3]), order.to(torch.int32).view(1, 3), i32([prompt]))
        out = att(q, kc, vc, _dev(t))
        _check_attend(out, q.cpu(), [kc.cpu(), vc.cpu()], t, att)


def test_ops_refuse_other_shapes_types_and_devices():
    app = QkvAppendOp(12, 2, DEV, max_tokens=8)
    att = SharedPrefixAttnOp(12, 2, DEV, max_tokens=8, max_seqs=2)
    d, caches = _append_inputs(8, 12, 2, 64)
    kc, vc = (c.to(DEV) for c in caches)
    good = dict(qkv=d["x"].to(DEV), g_q=None, g_k=None, cos=d["cos"].to(DEV), sin=d["sin"].to(DEV), positions=d["positions"].to(DEV),
                slots=d["slots"].to(DEV), k_cache=kc, v_cache=vc)
    app(**good)
    for name, bad in [("qkv", good["qkv"].half()), ("qkv", good["qkv"].cpu()), ("qkv", good["qkv"][:, :-128]), ("qkv", good["qkv"].repeat(2, 1)),
                      ("qkv", good["qkv"].float()), ("g_q", torch.zeros(64, device=DEV).bfloat16()), ("cos", good["cos"][:, :16]),
                      ("sin", good["sin"].float()), ("positions", good["positions"].int()), ("slots", good["slots"][:4]),
                      ("k_cache", kc[:, :32]), ("v_cache", vc[:1].contiguous()), ("k_cache", kc.cpu())]:
        with pytest.raises(ValueError, match=name):
            app(**{**good, name: bad})
    t, pages = _tables([1, 1], [9, 9], [0, 2], [70])
    kc, vc = (c.to(DEV) for c in _caches(pages, 2))
    q, dt = torch.zeros(2, 12, 128, device=DEV).bfloat16(), _dev(t)
    att(q, kc, vc, dt)
    for bad_q in (q.float(), q[:, :6], q.repeat(5, 1, 1), q.transpose(0, 1), q.cpu()):
        with pytest.raises(ValueError, match="q"):
            att(bad_q, kc, vc, dt)
    for field, bad in [("q_start", dt.q_start[:2]), ("page_table", dt.page_table.long()), ("lens", dt.lens.repeat(2)), ("group_start", dt.group_start[:1]),
                       ("prefix_table", dt.prefix_table[0]), ("prefix_lens", None), ("prefix_lens", dt.prefix_lens.repeat(2))]:
        with pytest.raises(ValueError, match=field):
            att(q, kc, vc, PrefixTables(**{**dt.__dict__, field: bad}))
    for guard in (torch.zeros(L.GUARD_WORDS, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(L.GUARD_WORDS, dtype=torch.int32)):
        with pytest.raises(ValueError, match="guard"):
            SharedPrefixAttnOp(12, 2, DEV, max_tokens=8, max_seqs=2, guard=guard)
    with pytest.raises(ValueError, match="out"):
        att(q, kc, vc, dt, out=torch.zeros(2, 12, 128, device=DEV))
    assert L.load().mono_prefix_attn_scratch_bytes(8, 12, 2, 2, 1) == att.scratch.numel()


# ---------------------------------------------------------------- entries of many rows, and both kinds in one launch
@pytest.mark.parametrize("hq,hk,ntok,own,starts,prefix", [
    (12, 2, [3] * 20, [5 + 13 * i for i in range(20)], [0, 20], [333]),        # 18 rows a sequence, 360 a prefix
    (4, 2, [5] * 7, [5, 64, 65, 6, 300, 129, 9], [0, 2, 7], [640, 63]),        # 10 rows a sequence: half a tile and more
    (4, 2, [4] * 9, [4, 5, 63, 64, 65, 66, 130, 200, 7], [0, 9], [100]),       # 8 rows a sequence: less than that
    (8, 8, [1] * 17, [1 + 9 * i for i in range(17)], [0, 17], [700]),          # 17 rows of a prefix in tiles of 8
    (8, 8, [1] * 16, [1 + 9 * i for i in range(16)], [0, 16], [700]),          # 16 of them
    (16, 1, [3], [3], [0, 1], [1]),                                            # 48 rows, four keys
    (16, 1, [2], [2], [0, 1], [64]),                                           # 32 rows in the whole step
    (33, 3, [12, 1, 24], [12, 1, 90], [0, 2, 3], [65, 1000]),                  # 132 and 264 rows: a tile's halves and borders
    (5, 1, [52], [1600], [], []),                                              # no prefix
    (6, 1, [43, 1], [43, 2000], [0, 2], [5])])
def test_attend_many_rows(hq, hk, ntok, own, starts, prefix):
    _attend(hq, hk, ntok, own, starts, prefix, columns=1)


def test_attend_many_rows_scores_far_apart_and_nan_rows():
    """Maxima that rise by hundreds between blocks, and a NaN and an infinite query: their own rows only."""
    hq, hk = 12, 2
    t, pages = _tables([1] * 30 + [40], [9] * 30 + [400], [0, 30], [1500])
    caches = _caches(pages, hk)
    q = (torch.randn(70, hq, 128, generator=_gen(2)) * 30).bfloat16()
    q[3, 7], q[50, 2, 5], q[12, 1, 100] = float("nan"), float("nan"), float("inf")
    q[1, 5] *= 1e-30
    q[1, 6] = 0
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=70, max_seqs=31, k_scale=K_SCALE, v_scale=V_SCALE)
    out = op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t))
    bad = torch.isnan(out).any(-1).cpu()
    assert bad[3, 7] and bad[50, 2] and int(bad.sum()) <= 3
    keep = ~bad[..., None].expand_as(out).clone()
    keep[12, 1] = False  # infinite scores have no restated value
    _check_attend(out, q, caches, t, op, rows=keep)


@pytest.mark.parametrize("hq,hk,ntok,own,starts,prefix", [
    (12, 2, [5, 2, 1], [70, 130, 20], [0, 3], [200]),   # tiles of few rows (and 30 rows of one sequence)
    (3, 1, [2, 3, 2], [20, 80, 64], [], []),
    (8, 8, [6, 7], [9, 200], [0, 2], [64]),
    (12, 2, [70, 3], [150, 66], [0, 2], [129]),         # prompt chunks
    (16, 1, [20], [20], [], [])])
def test_attend_nan_keys_and_values_of_later_tokens(hq, hk, ntok, own, starts, prefix):
    """A NaN in a key (or in one dim of a value) of a token reaches the tokens that see it, and no earlier one."""
    t, pages = _tables(ntok, own, starts, prefix)
    caches = _caches(pages, hk)
    for b, (n, ln) in enumerate(zip(ntok, own)):
        for back, dim, which, head in ((0, 3, 1, 0), (max(n - 2, 0), 77, 1, hk - 1), (n // 2, 5, 0, 0)):
            if n == 1 and which == 0:
                continue
            key = ln - 1 - back
            caches[which][int(t.page_table[b, key // 64]), key % 64, head, dim] = 0xFF if back else 0x7F
    tokens = sum(ntok)
    q = torch.randn(tokens, hq, 128, generator=_gen(11)).bfloat16()
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=tokens, max_seqs=len(own), max_groups=max(1, len(prefix)), k_scale=K_SCALE, v_scale=V_SCALE)
    out = op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t))
    ref = _check_attend(out, q, caches, t, op)
    assert torch.equal(torch.isnan(out).cpu(), torch.isnan(ref))
    assert torch.isnan(ref).any() and torch.isfinite(ref[0]).all() == (ntok[0] > 2)


def test_attend_many_rows_ignore_masked_places_and_bad_pages():
    hq, hk = 12, 2
    op, q, caches, dc, t, out = _attend(hq, hk, [20, 1, 30], [33, 70, 129], [0, 3], [200])
    want = out.clone()
    n = [c.clone() for c in caches]
    for tab, lens in ((t.page_table, t.lens), (t.prefix_table, t.prefix_lens)):
        for row, ln in zip(tab, lens):
            full, part = divmod(int(ln), 64)
            if part:
                for c in n:
                    c[int(row[full]), part:] = 0x7F
    assert torch.equal(op(q.to(DEV), *(c.to(DEV) for c in n), _dev(t)), want)
    t2 = PrefixTables(t.q_start, t.page_table.clone(), t.lens, t.group_start, t.prefix_table.clone(), t.prefix_lens)
    t2.prefix_table[0, 1] = caches[0].shape[0]
    t2.page_table[2, 0] = -5
    _check_attend(op(q.to(DEV), *dc, _dev(t2)), q, caches, t2, op)


def test_attend_steps_of_other_sizes_share_an_op():
    """Steps with and without entries of many rows, one after another on one op's buffers, each as on fresh ones."""
    hq, hk = 12, 2
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=200, max_seqs=40, max_groups=3, k_scale=K_SCALE, v_scale=V_SCALE)
    for seed, (ntok, own, starts, prefix) in enumerate([
            ([1] * 40, [9 + i for i in range(40)], [0, 20, 39, 40], [500, 77, 3]), ([1], [700], [], []), ([3] * 10, [40] * 10, [0, 10], [300]),
            ([150, 2], [150, 2], [0, 1, 2], [64, 900]), ([1] * 2, [5, 6], [0, 2], [2000])]):
        t, pages = _tables(ntok, own, starts, prefix, seed)
        caches = _caches(pages, hk)
        q = torch.randn(sum(ntok), hq, 128, generator=_gen(seed)).bfloat16()
        _check_attend(op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t)), q, caches, t, op)
        assert ops.guard_read(op.guard)[0] == 0


def test_a_decode_step_in_one_graph():
    """Append, attention, LM head and draw captured as one step; the replays follow the tables and the random numbers."""
    from sgl_amd_mono_b200.sampling import SampleOp
    from sgl_amd_mono_b200.tail import LmHeadOp

    hq, hk, seqs, vocab, prompt = 12, 2, 6, 1000, 100
    hidden, width = hq * 128, (hq + 2 * hk) * 128
    g = _gen(21)
    ang = torch.arange(256, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    cos, sin = ang.cos().bfloat16().to(DEV), ang.sin().bfloat16().to(DEV)
    pages = 2 + seqs
    kc, vc = (c.to(DEV) for c in _caches(pages, hk))
    app = QkvAppendOp(hq, hk, DEV, max_tokens=seqs, k_scale=K_SCALE, v_scale=V_SCALE)
    att = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=seqs, max_seqs=seqs, k_scale=K_SCALE, v_scale=V_SCALE)
    w = (torch.randn(vocab, hidden, generator=g) * hidden**-0.5).bfloat16().to(DEV)
    head = LmHeadOp(hidden, w, torch.zeros(hidden, dtype=torch.bfloat16, device=DEV), 1e-6, DEV)
    draw = SampleOp(vocab, DEV, max_rows=seqs)
    x = torch.zeros(seqs, width, dtype=torch.bfloat16, device=DEV)
    positions, slots = (torch.zeros(seqs, dtype=torch.int64, device=DEV) for _ in range(2))
    u, temp = torch.zeros(seqs, device=DEV), torch.full((seqs,), 0.8, device=DEV)
    top_p = torch.full((seqs,), 0.9, device=DEV)
    own = torch.arange(2, pages)
    t = PrefixTables(torch.arange(seqs + 1, dtype=torch.int32), own.to(torch.int32).view(seqs, 1), torch.ones(seqs, dtype=torch.int32),
                     torch.tensor([0, seqs], dtype=torch.int32), torch.tensor([[1, 0]], dtype=torch.int32), torch.tensor([prompt], dtype=torch.int32))
    dt = _dev(t)

    def step():
        out = att(app(x, None, None, cos, sin, positions, slots, kc, vc), kc, vc, dt)
        logits = head(out.view(seqs, hidden))
        return out, logits, *draw(logits, u, temp, None, top_p)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        x.copy_(torch.randn(seqs, width, generator=g))
        u.copy_(torch.rand(seqs, generator=g))
        positions.fill_(prompt + k)
        slots.copy_(own * 64 + k)
        t.lens.fill_(k + 1)
        dt.lens.copy_(t.lens)
        graph.replay()
        torch.cuda.synchronize()
        out, logits, tokens, logprobs = (r.cpu() for r in res)
        _check_attend(out, app.q.cpu(), [kc.cpu(), vc.cpu()], t, att)
        for r in range(seqs):
            token, lp, gap = OP.sample_row(logits[r].numpy(), float(u[r]), 0.8, 0, float(top_p[r]), 0.0)
            # the draw decides to 2^-44 of the largest weight; sums in the restatement round at 2^-52 of theirs
            assert gap < 1e-9 or (int(tokens[r]) == token and abs(float(logprobs[r]) - lp) <= abs(lp) * 2.0**-23 + 1e-9)


@pytest.mark.parametrize("qmul", [1.0, 3.0])
def test_attend_long_prefix_of_many_rows(qmul):
    """Single keys that hold much of a row's weight, anywhere in a long prefix: none may be lost when a maximum rises."""
    op, q, caches, dc, t, out = _attend(12, 2, [1] * 64, [33] * 64, [0, 64], [7000], seed=3, qmul=qmul)
    qd, dt, want = q.to(DEV), _dev(t), out.clone()
    for _ in range(20):
        assert torch.equal(op(qd, *dc, dt), want)


def test_attend_as_many_entries_as_a_launch_takes():
    n = 2047
    _attend(1, 1, [1] * n, [1 + i % 5 for i in range(n)], [0, n], [70])
    _attend(2, 1, [0] * 1023 + [1] * 1024, [0] * 1023 + [1 + i % 70 for i in range(1024)], [], [])


def test_attend_one_launch_after_another_without_overlap():
    """The same bits whether a launch's kernels may start before the one before has ended or not."""
    cases = [_attend(12, 2, [3] * 20, [40] * 20, [0, 20], [900]), _attend(12, 2, [1] * 3, [70] * 3, [0, 3], [300])]
    want = [out.clone() for *_, out in cases]
    try:
        L.load().mono_set_pdl(0)
        for (op, q, caches, dc, t, _), w in zip(cases, want):
            assert torch.equal(op(q.to(DEV), *dc, _dev(t)), w)
    finally:
        L.load().mono_set_pdl(1)


@pytest.mark.parametrize("spread", [9, 13, 20])
@pytest.mark.parametrize("hq,hk,ntok,own,starts,prefix", [
    (12, 2, [1] * 60, [30] * 60, [0, 60], [500]),     # one prefix of 360 rows
    (6, 1, [100, 40], [100, 300], [], []),            # tiles of both sizes on their own keys
    (12, 2, [1] * 4, [70] * 4, [0, 2, 4], [90, 64])])  # few rows
def test_attend_queries_with_one_large_dim(hq, hk, ntok, own, starts, prefix, spread):
    """A query dim up to 2^spread times the others, at a dim where the keys are zero, changes no score."""
    t, pages = _tables(ntok, own, starts, prefix)
    caches = _caches(pages, hk)
    caches[0][..., 17] = 0
    tokens = sum(ntok)
    g = _gen(31)
    sign = lambda *s: torch.randint(0, 2, s, generator=g) * 2.0 - 1.0  # noqa: E731
    q = (sign(tokens, hq, 128) * (0.5 + 1.5 * torch.rand(tokens, hq, 128, generator=g))).bfloat16()  # 0.5 .. 2
    q[..., 17] = (sign(tokens, hq) * 2.0 ** torch.randint(spread - 4, spread, (tokens, hq), generator=g)).bfloat16()
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=tokens, max_seqs=len(own), max_groups=max(1, len(prefix)), k_scale=K_SCALE, v_scale=V_SCALE)
    out = op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t))
    if spread <= 13:
        _check_attend(out, q, caches, t, op)
        return
    # beyond 2^13 a query value is held to 2^-21 of the row's largest: scores are off by that times the sum of a key's values,
    # which enters numerator and denominator
    ref, mag, big, seen = OP.attend(q, *caches, t.q_start, t.page_table, t.lens, t.group_start, t.prefix_table, t.prefix_lens, op.k_scale, op.v_scale, op.sm_scale)
    most = float(OP.cache_values(caches[0]).abs().sum(-1).max()) * op.k_scale * op.sm_scale
    score = 2.0**-21 * q.double().abs().amax(-1) * most + 128 * 2.0**-23 * big
    tol = ref.abs() * 2.0**-8 + mag * (2.0**-11 + torch.expm1(2 * score)[..., None] + 2.0**-19 + (seen[:, None, None] / 16 + 16) * 2.0**-23)
    assert ((out.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("hq,hk,ntok,own,starts,prefix", [
    (6, 1, [2100], [2100], [], []),                                      # a prompt on its own keys
    (12, 2, [4096, 1, 2001], [4096, 800, 3000], [], []),                 # prompts, one of them in a second chunk
    (12, 2, [700, 442, 300], [1500, 442, 901], [0, 3], [4100])])         # prompt chunks behind a shared prefix
def test_attend_long_prompts(hq, hk, ntok, own, starts, prefix):
    t, pages = _tables(ntok, own, starts, prefix)
    caches = _caches(pages, hk)
    tokens = sum(ntok)
    q = (torch.randn(tokens, hq, 128, generator=_gen(17)) * 2).bfloat16()
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=tokens, max_seqs=len(own), max_groups=max(1, len(prefix)), k_scale=K_SCALE, v_scale=V_SCALE)
    out = op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t)).cpu()
    assert ops.guard_read(op.guard)[0] == 0
    # some tokens, as sequences of one token each: token j of n sees its sequence's keys up to its own
    pick = torch.unique(torch.cat([torch.arange(0, tokens, 97), torch.arange(40, 46), torch.tensor([tokens - 1]), torch.randperm(tokens, generator=_gen(1))[:40]]))
    seq = torch.searchsorted(t.q_start[1:].long(), pick, right=True)
    lens = t.lens[seq] - t.q_start[1:][seq] + pick.to(torch.int32) + 1
    one = PrefixTables(torch.arange(len(pick) + 1, dtype=torch.int32), t.page_table[seq], lens.to(torch.int32),
                       None if t.group_start is None else torch.tensor([0, len(pick)], dtype=torch.int32), t.prefix_table, t.prefix_lens)
    _check_attend(out[pick], q[pick], caches, one, op)


@pytest.mark.parametrize("k_scale,sm_scale", [(2.0**-40, None), (2.0**-100, 2.0**-100), (2.0**-100, 2.0**60), (2.0**100, 2.0**-100), (2.0**40, 2.0**-43)])
def test_attend_small_scores_and_far_scales(k_scale, sm_scale):
    """Scores next to 0 under the smallest scales weigh all visible keys alike, and masked keys not at all."""
    hq, hk = 12, 2
    t, pages = _tables([3, 1, 20], [40, 70, 30], [0, 3], [100])
    caches = _caches(pages, hk)
    q = torch.randn(24, hq, 128, generator=_gen(3)).bfloat16()
    q[1, 4] = 0
    q[2, 5] *= 2.0**-120
    q[9, 7] = 0
    q[13, 2] *= 2.0**-120
    for n in (24, 4):  # entries of many rows, and of few
        part = t if n == 24 else PrefixTables(t.q_start[:3], t.page_table[:2], t.lens[:2], torch.tensor([0, 2], dtype=torch.int32), t.prefix_table, t.prefix_lens)
        op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=24, max_seqs=3, k_scale=k_scale, v_scale=V_SCALE, sm_scale=sm_scale)
        out = op(q[:n].to(DEV), *(c.to(DEV) for c in caches), _dev(part))
        _check_attend(out, q[:n], caches, part, op)


@pytest.mark.parametrize("tokens,nsum,rows", [(1, 1, 1), (16, 3, 16), (9, 2, 9), (1, 4, 1)])
def test_append_from_partial_sums_of_wider_rows(tokens, nsum, rows):
    """The block-sparse layer's projection leaves its index heads behind q | k | v: the rows are taken where they lie."""
    from sgl_amd_mono_b200.gqa import CFG_GQA

    hq, hk, width = CFG_GQA.q_local, CFG_GQA.kv_local, CFG_GQA.qkv_rows
    d, caches = _append_inputs(tokens, hq, hk, 64)
    parts = torch.randn(nsum, rows, width, generator=_gen(3))
    op = QkvAppendOp(hq, hk, DEV, max_tokens=16, k_scale=K_SCALE, v_scale=V_SCALE)
    w = [d[k].to(DEV) for k in ("g_q", "g_k", "cos", "sin", "positions", "slots")]
    kc, vc = (c.to(DEV) for c in caches)
    part = parts.to(DEV)[..., : (hq + 2 * hk) * 128]
    q = op(part, *w, kc, vc, tokens=tokens).clone()
    x = torch.zeros(rows, (hq + 2 * hk) * 128)
    for p in parts:
        x = x + p[:, : x.shape[1]]
    _check_append(q, kc, vc, x[:tokens], d, caches, hq, hk, False)
    # the same bits as of rows that lie close
    k2, v2 = (c.to(DEV) for c in caches)
    assert torch.equal(op(part.contiguous(), *w, k2, v2, tokens=tokens), q) and torch.equal(k2, kc) and torch.equal(v2, vc)
    for bad in (parts.to(DEV), parts.to(DEV)[..., 1 : 1 + x.shape[1]], part[0]):
        with pytest.raises(ValueError, match="qkv"):
            op(bad, *w, kc, vc, tokens=tokens)
    if rows > 1:
        odd = torch.zeros(nsum, rows, x.shape[1] + 4, device=DEV)[..., : x.shape[1]]
        turned = part.transpose(1, 2).contiguous().transpose(1, 2)  # (of a single row that is the row itself)
        for bad in (odd, turned):
            with pytest.raises(ValueError, match="qkv"):
                op(bad, *w, kc, vc, tokens=tokens)


@pytest.mark.parametrize("hq,hk,ntok,own,starts,prefix", [
    (72, 9, [2, 0] * 20, [9, 0] * 20, list(range(0, 41, 2)), [5] * 20),   # two full tiles of 8 rows of every sequence and group
    (8, 8, [16] + [0] * 15 + [1] * 3, [40] + [0] * 15 + [300] * 3, [0, 16, 19], [70, 90]),
    (32, 2, [1] * 2, [700, 800], [0, 1, 2], [900, 300]),                  # fewer rows than the other kernel is started for
    (7, 7, [4] * 8, [10 + i for i in range(8)], [0, 4, 8], [65, 200]),
    (16, 1, [16, 1, 15, 1], [16, 40, 500, 1], [], [])])
def test_attend_scratch_holds_what_a_step_leaves(hq, hk, ntok, own, starts, prefix):
    """Steps of as many parts of tiles as their sizes allow, on a scratch of just the size asked for."""
    t, pages = _tables(ntok, own, starts, prefix)
    caches = _caches(pages, hk)
    tokens = sum(ntok)
    q = torch.randn(tokens, hq, 128, generator=_gen(8)).bfloat16()
    op = SharedPrefixAttnOp(hq, hk, DEV, max_tokens=tokens, max_seqs=len(own), max_groups=len(prefix), k_scale=K_SCALE, v_scale=V_SCALE)
    size = op.scratch.numel()
    room = torch.full((size + 8192,), 0xA5, dtype=torch.uint8, device=DEV)
    op._fixed.scratch = room.data_ptr()
    assert room.data_ptr() % 256 == 0
    out = op(q.to(DEV), *(c.to(DEV) for c in caches), _dev(t))
    assert ops.guard_read(op.guard)[0] == 0
    _check_attend(out, q, caches, t, op)
    assert (room[size:] == 0xA5).all()
