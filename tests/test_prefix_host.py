"""Host side of the append, attention and sampling operators: what is refused before any launch, the scratch sizes, and
the restatement they are compared with against a second form of each definition."""

import ctypes as C
import math
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import prefix as OP
from sgl_amd_mono_b200 import _lib as L
from sgl_amd_mono_b200 import prefix
from sgl_amd_mono_b200.build import build_library
from sgl_amd_mono_b200.prefix import QkvAppendOp, SharedPrefixAttnOp
from sgl_amd_mono_b200.sampling import SampleOp


@pytest.fixture(scope="module")
def lib():
    build_library()
    return L.load()


def _append_args(**kw):
    a = L.QkvAppendArgs()
    base = dict(tokens=4, q_heads=12, kv_heads=2, rot_dim=64, src_bf16=4096, src_ld=2048, eps=1e-6, cos=4096, sin=4096, table_rows=8,
                positions=4096, slots=4096, k_scale=1.0, v_scale=1.0, k_cache=4096, v_cache=4096, n_pages=3, q_out=4096)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    dict(tokens=0), dict(q_heads=0), dict(kv_heads=0), dict(rot_dim=8), dict(rot_dim=72), dict(rot_dim=144), dict(src_bf16=None),
    dict(src_f32=4096), dict(src_ld=2040), dict(src_ld=2052), dict(src_bf16=4098), dict(cos=None), dict(table_rows=0), dict(positions=None),
    dict(q_out=None), dict(k_cache=None), dict(v_cache=4100), dict(n_pages=0), dict(k_scale=0.0), dict(v_scale=-1.0), dict(k_scale=1e-39), dict(eps=float("nan")),
    dict(src_bf16=None, src_f32=4096, nsum=0), dict(src_bf16=None, src_f32=4096, nsum=2, tokens=17), dict(src_bf16=None, src_f32=4096, nsum=2, sum_stride=6)])
def test_append_refuses(lib, bad):
    assert lib.mono_qkv_append_launch(C.byref(_append_args(**bad)), None) == -1
    assert lib.mono_last_error()


def _attn_args(**kw):
    a = L.PrefixAttnArgs()
    base = dict(tokens=4, q_heads=12, kv_heads=2, seqs=4, groups=1, q=4096, q_ld=1536, k_cache=4096, v_cache=4096, n_pages=9, q_start=4096,
                page_table=4096, pt_ld=2, lens=4096, group_start=4096, prefix_table=4096, prefix_ld=5, prefix_lens=4096, k_scale=1.0,
                v_scale=1.0, sm_scale=1.0, scratch=4096, scratch_bytes=1 << 30, out=4096)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    dict(tokens=0), dict(q_heads=13), dict(q_heads=34), dict(kv_heads=0), dict(seqs=0), dict(groups=-1), dict(seqs=2048), dict(q=None),
    dict(q_ld=1528), dict(q_ld=1540), dict(q=4104), dict(out=4104), dict(scratch=4112), dict(scratch=None), dict(scratch_bytes=1000), dict(lens=None),
    dict(pt_ld=0), dict(prefix_ld=0), dict(group_start=None), dict(k_scale=0.0), dict(v_scale=float("inf")), dict(sm_scale=1e-40), dict(n_pages=0), dict(n_pages=1 << 26),
    dict(tokens=1 << 20, pt_ld=1 << 20)])
def test_attention_refuses(lib, bad):
    assert lib.mono_prefix_attn_launch(C.byref(_attn_args(**bad)), None) == -1
    assert lib.mono_last_error()


@pytest.mark.parametrize("bad", [dict(rows=0), dict(rows=70000), dict(vocab=0), dict(vocab=L.SAMPLE_MAX_VOCAB + 1), dict(logits=None), dict(u=None),
                                 dict(tokens=None), dict(ld=99), dict(logits=4098), dict(tokens=4100), dict(logits=4097, logits_bf16=1)])
def test_sampling_refuses(lib, bad):
    a = L.SampleArgs()
    for k, v in {**dict(rows=2, vocab=100, logits=4096, ld=100, u=4096, tokens=4096), **bad}.items():
        setattr(a, k, v)
    assert lib.mono_sample_launch(C.byref(a), None) == -1
    assert lib.mono_last_error()


def test_ops_refuse_before_they_touch_a_device():
    for kw, name in [(dict(q_heads=13), "q_heads"), (dict(q_heads=34), "q_heads"), (dict(max_tokens=0), "max_tokens"), (dict(rot_dim=40), "rot_dim"),
                     (dict(k_scale=0.0), "k_scale"), (dict(v_scale=float("inf")), "v_scale"), (dict(eps=-1.0), "eps"), (dict(device="cpu"), "device")]:
        with pytest.raises(ValueError, match=name):
            QkvAppendOp(**{**dict(q_heads=12, kv_heads=2, device="cuda:0", max_tokens=4), **kw})
    for kw, name in [(dict(q_heads=0), "q_heads"), (dict(max_seqs=0), "max_seqs"), (dict(max_seqs=2048), "max_seqs"), (dict(k_scale=-1.0), "k_scale"),
                     (dict(device="cpu"), "device")]:
        with pytest.raises(ValueError, match=name):
            SharedPrefixAttnOp(**{**dict(q_heads=12, kv_heads=2, device="cuda:0", max_tokens=4, max_seqs=4), **kw})
    for kw, name in [(dict(vocab=0), "vocab"), (dict(vocab=L.SAMPLE_MAX_VOCAB + 1), "vocab"), (dict(max_rows=0), "max_rows"), (dict(device="cpu"), "device")]:
        with pytest.raises(ValueError, match=name):
            SampleOp(**{**dict(vocab=100, device="cuda:0", max_rows=4), **kw})


def test_attention_scratch_grows_with_every_size(lib):
    f = lib.mono_prefix_attn_scratch_bytes
    base = f(64, 12, 2, 16, 1)
    assert 0 < base < 64 << 20
    assert f(65 * 16, 12, 2, 16, 1) > base and f(64, 12, 2, 17, 1) > base and f(64, 12, 2, 16, 2) > base
    assert f(0, 12, 2, 16, 1) == 0 and f(64, 13, 2, 16, 1) == 0


def test_restated_attention_is_softmax_over_the_visible_keys():
    g = torch.Generator().manual_seed(0)
    kc, vc = ((torch.randn(5, 64, 1, 128, generator=g) * 16).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2))
    q = torch.randn(3, 2, 128, generator=g).bfloat16()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    out, _, _, seen = OP.attend(q, kc, vc, i32([0, 1, 3]), i32([[2, -1], [4, 1]]), i32([10, 66]), i32([0, 2]), i32([[3, 0]]), i32([100]), 0.5, 0.25, 0.1)
    assert seen.tolist() == [110, 165, 166]
    k, v = OP.cache_values(kc)[:, :, 0] * 0.5, OP.cache_values(vc)[:, :, 0] * 0.25
    keys = torch.cat([k[3], k[0][:36], k[4], k[1][:2]])
    vals = torch.cat([v[3], v[0][:36], v[4], v[1][:2]])
    s = q[2].double() @ keys.T * 0.1
    want = (s - s.amax(1, keepdim=True)).exp()
    want = want / want.sum(1, keepdim=True) @ vals
    assert torch.allclose(out[2], want, rtol=1e-12, atol=1e-14)


def test_restated_draw_follows_its_definition():
    x = np.array([1.0, 3.0, 2.0, 3.0, -np.inf, np.nan], dtype=np.float32)
    w = np.array([np.exp(-2.0), 1.0, np.exp(-1.0), 1.0, 0.0, 0.0])
    c = np.cumsum(w) / w.sum()
    for u in (0.0, 0.03, 0.2, 0.5, 0.9):
        assert OP.sample_row(x, u)[0] == int(np.argmax(c > u))
    assert OP.sample_row(x, 0.999, top_k=1)[0] == 1 and OP.sample_row(x, 0.999, top_k=2)[0] == 3
    assert OP.sample_row(x, 0.0, top_p=0.5)[0] == 1 and OP.sample_row(x, 0.999, top_p=0.3)[0] == 1
    assert OP.sample_row(x, 0.0, min_p=0.2)[0] == 1 and OP.sample_row(x, 0.4, min_p=0.2)[0] == 1 and OP.sample_row(x, 0.999, min_p=0.5)[0] == 3
    assert OP.sample_row(x, 0.7, temperature=0.0)[0] == 1
    assert OP.sample_row(np.full(3, -np.inf), 0.5)[0] == -1


def test_draw_waits_for_its_cluster_before_it_writes_to_peers():
    """Another CTA's shared memory may be touched only once that CTA is known to run, so the kernel's first use of it lies
    behind a wait for the whole cluster."""
    src = (Path(L.__file__).parent / "csrc" / "sample.cu").read_text()
    body = src[src.index("sample_kernel(") : src.index("static cudaError_t launch_with")]
    first = min(body.index(use) for use in ("map_shared_rank(", "st_peer(", "hist_merge<"))
    waits = [body.find(w) for w in ("cluster.barrier_wait()", "cluster.sync()")]
    assert any(0 <= at < first for at in waits)


def test_restated_draw_keeps_the_first_alone_where_no_weight_passes():
    x = np.array([0.0, 2.0, 1.0, 2.0], dtype=np.float32)
    assert OP.sample_row(x, 0.9, min_p=1.0)[0] == 3
    for min_p in (float(np.nextafter(np.float32(1), np.float32(2))), 1.5, math.inf):
        assert OP.sample_row(x, 0.9, min_p=min_p)[0] == 1


def test_attention_refuses_scales_whose_product_leaves_no_room_for_scores(lib):
    assert lib.mono_prefix_attn_launch(C.byref(_attn_args(k_scale=2.0**60, sm_scale=2.0**41)), None) == -1
    assert b"2^100" in lib.mono_last_error()
    with pytest.raises(ValueError, match="sm_scale"):
        SharedPrefixAttnOp(12, 2, "cuda:0", max_tokens=4, max_seqs=4, k_scale=2.0**60, sm_scale=2.0**41)


def test_ops_are_not_built_for_what_every_launch_refuses(lib):
    """Each size at its largest passes the launch's check of it (and fails at the next), and so does the op."""
    assert lib.mono_qkv_append_launch(C.byref(_append_args(q_heads=257)), None) == -1 and b"256 q heads" in lib.mono_last_error()
    with pytest.raises(ValueError, match="q_heads"):
        QkvAppendOp(272, 17, "cuda:0", max_tokens=4)
    with pytest.raises(ValueError, match="device"):  # (what comes after the sizes)
        QkvAppendOp(256, 16, "cpu", max_tokens=1 << 24)
    with pytest.raises(ValueError, match="max_tokens"):
        QkvAppendOp(12, 2, "cuda:0", max_tokens=(1 << 24) + 1)
    with pytest.raises(ValueError, match="max_tokens"):
        SharedPrefixAttnOp(12, 2, "cuda:0", max_tokens=(1 << 20) + 1, max_seqs=4)
    with pytest.raises(ValueError, match="device"):
        SharedPrefixAttnOp(12, 2, "cpu", max_tokens=1 << 20, max_seqs=4)


def test_an_op_keeps_few_views_of_its_buffers():
    base = torch.arange(4000).view(1000, 4)
    views = {0: base}
    for n in list(range(1, 1001)) + [7, 7, 1000]:
        v = prefix._front(views, n)
        assert v.shape == (n, 4) and v.data_ptr() == base.data_ptr() and len(views) <= 100
    assert prefix._front(views, 7) is prefix._front(views, 7) and views[0] is base


def test_attention_scratch_of_long_prompts(lib):
    """What 16384 tokens of 48 heads need: their rows in f32 once for a sequence and once for a group, and their queries."""
    f = lib.mono_prefix_attn_scratch_bytes
    rows = 16384 * 48
    assert f(16384, 48, 8, 1, 0) < 1.25 * rows * (128 * 4 + 256)
    assert f(16384, 48, 8, 4, 1) < 1.25 * rows * (2 * 128 * 4 + 256)
    # a step of fewer tokens, sequences or groups fits what was reserved for more
    sizes = [(t, s, g) for t in (1, 2, 5, 6, 33, 200, 3001) for s in (1, 3, 40) for g in (0, 1, 7)]
    for hq, hk in ((12, 2), (48, 8), (72, 9), (5, 5)):
        for a in sizes:
            for b in sizes:
                if all(x <= y for x, y in zip(a, b)):
                    assert f(a[0], hq, hk, a[1], a[2]) <= f(b[0], hq, hk, b[1], b[2])
