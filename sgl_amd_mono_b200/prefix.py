"""Many continuations of shared prompts on the paged E4M3 K / V caches: append and attention.

``QkvAppendOp`` takes the rows of the fused q | k | v projection (a prompt's or a step's, any number of tokens) to
normed, rotated queries and writes keys and values to the caches; ``SharedPrefixAttnOp`` attends a prefix that a group
of sequences shares, read once for the group, and every sequence's own pages.  The caches are those of ``gqa.GqaCore``
(``[pages, 64, kv_heads, 128]`` E4M3 bytes with one fixed scale each); dense attention here stands beside the
block-sparse attention there.

An op allocates its buffers when it is built; a call only enqueues kernels on its device's current stream and may be
captured into a CUDA graph (the tables are device data that a replay reads afresh).  Calls of ONE op object share its
buffers and must be ordered (one stream, or streams that wait for one another); the returned tensor is overwritten by
the next call.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib as L
from . import ops

HEAD_DIM = 128
PAGE = 64
MAX_GROUP = 16  # q heads per kv head
MAX_ENTRIES = 2048  # sequences + prefix groups of one launch


def _device(device) -> torch.device:
    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError(f"device: {d}, needs a CUDA device (there is no CPU path)")
    return d if d.index is not None else torch.device("cuda", torch.cuda.current_device())


def _heads(q_heads: int, kv_heads: int) -> None:
    if q_heads < 1 or not 1 <= kv_heads <= 256 or q_heads % kv_heads or q_heads // kv_heads > MAX_GROUP:
        raise ValueError(f"q_heads {q_heads} / kv_heads {kv_heads}: needs a whole number of q heads per kv head, 1..{MAX_GROUP}")


def _scale(x: float, name: str) -> float:
    x = float(x)
    if not 0.0 < x < float("inf"):
        raise ValueError(f"{name}: {x}, needs a positive finite number")
    return x


def _on(t: torch.Tensor, name: str, dev: torch.device, dtype=None, shape=None) -> torch.Tensor:
    ops.require(t, name, dtype, shape)
    if t.device != dev:
        raise ValueError(f"{name}: on {t.device}, the op was built for {dev}")
    return t


def _aligned(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.data_ptr() % 16:
        raise ValueError(f"{name}: must start on a 16-byte address")
    return t


def _caches(k_cache, v_cache, kv_heads: int, dev) -> None:
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _aligned(_on(t, name, dev, torch.uint8), name)
        if t.dim() != 4 or tuple(t.shape[1:]) != (PAGE, kv_heads, HEAD_DIM) or t.shape[0] < 1:
            raise ValueError(f"{name}: shape {tuple(t.shape)}, needs [pages, {PAGE}, {kv_heads}, {HEAD_DIM}]")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"v_cache: {v_cache.shape[0]} pages, k_cache has {k_cache.shape[0]}")


class QkvAppendOp:
    """``q = rope(norm(q))`` per head, and K / V of the same rows into the paged caches.

    Per q and k head: RMSNorm over the 128 dims with weight ``1 + g``, then the rotation of the first ``rot_dim`` dims
    in pairs ``(i, i + rot_dim / 2)`` or, ``interleaved``, ``(2i, 2i + 1)``.  f32 arithmetic, rounded once at the store:
    q to bf16, k and v to E4M3 of ``value / scale``."""

    def __init__(self, q_heads: int, kv_heads: int, device, max_tokens: int, rot_dim: int = 64, interleaved: bool = False,
                 eps: float = 1e-6, k_scale: float = 1.0, v_scale: float = 1.0):
        _heads(q_heads, kv_heads)
        if max_tokens < 1:
            raise ValueError(f"max_tokens: {max_tokens}, needs at least 1")
        if rot_dim % 16 or not 16 <= rot_dim <= HEAD_DIM:
            raise ValueError(f"rot_dim: {rot_dim}, needs a multiple of 16 in 16..{HEAD_DIM}")
        if not float(eps) >= 0.0:
            raise ValueError(f"eps: {eps}, needs at least 0")
        self.k_scale, self.v_scale = _scale(k_scale, "k_scale"), _scale(v_scale, "v_scale")
        self.dev = _device(device)
        L.load()
        self.q_heads, self.kv_heads, self.max_tokens = q_heads, kv_heads, max_tokens
        self.rot_dim, self.interleaved, self.eps = rot_dim, bool(interleaved), float(eps)
        self.q = torch.zeros(max_tokens, q_heads, HEAD_DIM, dtype=torch.bfloat16, device=self.dev)

    def __call__(self, qkv: torch.Tensor, g_q, g_k, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, slots,
                 k_cache: torch.Tensor, v_cache: torch.Tensor, tokens: int | None = None) -> torch.Tensor:
        """``qkv``: bf16 ``[tokens, (q_heads + 2 kv_heads) * 128]`` (rows may lie further apart), or f32 partial sums
        ``[nsum, rows, ..]`` of at most 16 ``tokens`` as the projection's GEMV leaves them (``tokens`` is then required).
        ``g_q`` / ``g_k``: bf16 ``[128]``, None for no norm.  ``cos`` / ``sin``: bf16 or f32 ``[positions, rot_dim / 2]``.
        ``positions``, ``slots``: int64 ``[tokens]``; a position outside the table is taken to its nearest row, a slot
        (page * 64 + offset) outside the cache inserts nothing, and the slots inside it must differ.
        Returns q ``[tokens, q_heads, 128]`` (the op's own buffer)."""
        width = (self.q_heads + 2 * self.kv_heads) * HEAD_DIM
        a = L.QkvAppendArgs()
        if not isinstance(qkv, torch.Tensor) or not qkv.is_cuda or qkv.device != self.dev:
            raise ValueError(f"qkv: must be a tensor on {self.dev} (there is no CPU path)")
        if qkv.dtype == torch.bfloat16:
            if qkv.dim() != 2 or qkv.shape[1] != width or qkv.stride(1) != 1 or (qkv.shape[0] > 1 and qkv.stride(0) < width):
                raise ValueError(f"qkv: shape {tuple(qkv.shape)} strides {qkv.stride()}, needs [tokens, {width}] with contiguous rows")
            if tokens is not None and tokens != qkv.shape[0]:
                raise ValueError(f"qkv: {qkv.shape[0]} rows, tokens says {tokens}")
            n = qkv.shape[0]
            a.src_bf16, a.src_ld = qkv.data_ptr(), qkv.stride(0) if n > 1 else width
        elif qkv.dtype == torch.float32:
            if qkv.dim() != 3 or not qkv.is_contiguous() or qkv.shape[2] != width:
                raise ValueError(f"qkv: shape {tuple(qkv.shape)}, needs contiguous f32 partial sums [nsum, rows, {width}]")
            if tokens is None or not 1 <= tokens <= min(L.MAX_ROWS, qkv.shape[1]):
                raise ValueError(f"tokens: {tokens}, partial sums of {qkv.shape[1]} rows serve 1..{min(L.MAX_ROWS, qkv.shape[1])}")
            n = tokens
            a.src_f32, a.nsum, a.src_ld, a.sum_stride = qkv.data_ptr(), qkv.shape[0], width, qkv.shape[1] * width
        else:
            raise ValueError(f"qkv: dtype {qkv.dtype}, needs bfloat16 rows or float32 partial sums")
        if not 1 <= n <= self.max_tokens:
            raise ValueError(f"qkv: {n} tokens, the op was built for 1..{self.max_tokens}")
        if a.src_ld % 8:
            raise ValueError(f"qkv: rows {a.src_ld} values apart, needs a multiple of 8")
        _aligned(qkv, "qkv")
        for g, name in ((g_q, "g_q"), (g_k, "g_k")):
            if g is not None:
                _aligned(_on(g, name, self.dev, torch.bfloat16, (HEAD_DIM,)), name)
        if not isinstance(cos, torch.Tensor) or cos.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("cos: needs a bfloat16 or float32 tensor")
        for t, name in ((cos, "cos"), (sin, "sin")):
            _aligned(_on(t, name, self.dev, cos.dtype), name)
            if t.dim() != 2 or t.shape[0] < 1 or t.shape[1] != self.rot_dim // 2 or t.shape != cos.shape:
                raise ValueError(f"{name}: shape {tuple(t.shape)}, needs [positions, {self.rot_dim // 2}]")
        _on(positions, "positions", self.dev, torch.int64, (n,))
        if slots is not None:
            _on(slots, "slots", self.dev, torch.int64, (n,))
        _caches(k_cache, v_cache, self.kv_heads, self.dev)
        a.tokens, a.q_heads, a.kv_heads = n, self.q_heads, self.kv_heads
        a.rot_dim, a.interleaved = self.rot_dim, int(self.interleaved)
        a.g_q, a.g_k, a.eps = ops._p(g_q), ops._p(g_k), self.eps
        a.cos, a.sin, a.table_f32, a.table_rows = cos.data_ptr(), sin.data_ptr(), int(cos.dtype == torch.float32), cos.shape[0]
        a.positions, a.slots = positions.data_ptr(), ops._p(slots)
        a.k_scale, a.v_scale = self.k_scale, self.v_scale
        a.k_cache, a.v_cache, a.n_pages = k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0]
        a.q_out = self.q.data_ptr()
        with torch.cuda.device(self.dev):
            L.check(L.load().mono_qkv_append_launch(C.byref(a), ops._stream()), "mono_qkv_append_launch")
        return self.q[:n]


@dataclass
class PrefixTables:
    """One step's tables, all int32 on the device.

    Sequence b has the query tokens ``q_start[b] .. q_start[b + 1] - 1`` and ``lens[b]`` keys of its own, its query
    tokens' among them, in pages ``page_table[b]``.  Sequences ``group_start[g] .. group_start[g + 1] - 1`` share the
    ``prefix_lens[g]`` keys in pages ``prefix_table[g]``; without groups (None) there is no prefix."""

    q_start: torch.Tensor      # [seqs + 1]
    page_table: torch.Tensor   # [seqs, columns]
    lens: torch.Tensor         # [seqs]
    group_start: torch.Tensor | None = None   # [groups + 1]
    prefix_table: torch.Tensor | None = None  # [groups, columns]
    prefix_lens: torch.Tensor | None = None   # [groups]


class SharedPrefixAttnOp:
    """Dense attention of every query token over its group's shared prefix and its sequence's own keys.

    Token j of a sequence's n sees the whole prefix and the sequence's keys ``0 .. lens - n + j``.  The output is
    ``softmax((q . k) k_scale sm_scale) v v_scale``; a token that sees no key gives zeros, and rows of ``out`` behind
    the last sequence's tokens keep what they held.  ``guard`` holds the error words (``ops.guard_read``): starts that
    fall or leave their range set the argument word."""

    def __init__(self, q_heads: int, kv_heads: int, device, max_tokens: int, max_seqs: int, max_groups: int = 1,
                 k_scale: float = 1.0, v_scale: float = 1.0, sm_scale: float | None = None, guard: torch.Tensor | None = None,
                 deadline_s: float = 5.0):
        _heads(q_heads, kv_heads)
        if max_tokens < 1 or max_seqs < 1 or max_groups < 0 or max_seqs + max_groups > MAX_ENTRIES:
            raise ValueError(f"max_tokens {max_tokens}, max_seqs {max_seqs}, max_groups {max_groups}: needs at least one token and "
                             f"sequence, and at most {MAX_ENTRIES} sequences and groups")
        self.k_scale, self.v_scale = _scale(k_scale, "k_scale"), _scale(v_scale, "v_scale")
        self.dev = _device(device)
        self.q_heads, self.kv_heads = q_heads, kv_heads
        self.max_tokens, self.max_seqs, self.max_groups = max_tokens, max_seqs, max_groups
        self.sm_scale = _scale(sm_scale, "sm_scale") if sm_scale is not None else HEAD_DIM ** -0.5
        self.deadline_s = deadline_s
        with torch.cuda.device(self.dev):
            nbytes = L.load().mono_prefix_attn_scratch_bytes(max_tokens, q_heads, kv_heads, max_seqs, max_groups)
        self.scratch = torch.zeros(nbytes, dtype=torch.uint8, device=self.dev)
        self.out = torch.zeros(max_tokens, q_heads, HEAD_DIM, dtype=torch.bfloat16, device=self.dev)
        self.guard = guard if guard is not None else torch.zeros(L.GUARD_WORDS, dtype=torch.int32, device=self.dev)

    def _table(self, t, name: str, rows: int) -> torch.Tensor:
        _on(t, name, self.dev, torch.int32)
        if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
            raise ValueError(f"{name}: shape {tuple(t.shape)}, needs [{rows}, at least 1]")
        return t

    def __call__(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, t: PrefixTables,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """``q``: bf16 ``[tokens, q_heads, 128]`` (token rows may lie further apart).  Returns ``out`` (default: the
        op's own buffer), bf16 ``[tokens, q_heads, 128]``."""
        if not isinstance(q, torch.Tensor) or q.device != self.dev:
            raise ValueError(f"q: must be a tensor on {self.dev} (there is no CPU path)")
        if q.dtype != torch.bfloat16:
            raise ValueError(f"q: dtype {q.dtype}, needs torch.bfloat16")
        if q.dim() != 3 or tuple(q.shape[1:]) != (self.q_heads, HEAD_DIM):
            raise ValueError(f"q: shape {tuple(q.shape)}, needs [tokens, {self.q_heads}, {HEAD_DIM}]")
        n = q.shape[0]
        if not 1 <= n <= self.max_tokens:
            raise ValueError(f"q: {n} tokens, the op was built for 1..{self.max_tokens}")
        width = self.q_heads * HEAD_DIM
        ld = q.stride(0) if n > 1 else width
        if q.stride(2) != 1 or (self.q_heads > 1 and q.stride(1) != HEAD_DIM) or ld < width or ld % 8:
            raise ValueError(f"q: strides {q.stride()}, needs contiguous heads and token rows a multiple of 8 values apart")
        _aligned(q, "q")
        _caches(k_cache, v_cache, self.kv_heads, self.dev)
        _on(t.lens, "lens", self.dev, torch.int32)
        seqs = t.lens.numel()
        if t.lens.dim() != 1 or not 1 <= seqs <= self.max_seqs:
            raise ValueError(f"lens: shape {tuple(t.lens.shape)}, the op was built for 1..{self.max_seqs} sequences")
        _on(t.q_start, "q_start", self.dev, torch.int32, (seqs + 1,))
        self._table(t.page_table, "page_table", seqs)
        groups = 0
        if t.prefix_lens is not None:
            _on(t.prefix_lens, "prefix_lens", self.dev, torch.int32)
            groups = t.prefix_lens.numel()
            if t.prefix_lens.dim() != 1 or not 1 <= groups <= self.max_groups:
                raise ValueError(f"prefix_lens: shape {tuple(t.prefix_lens.shape)}, the op was built for up to {self.max_groups} groups")
            _on(t.group_start, "group_start", self.dev, torch.int32, (groups + 1,))
            self._table(t.prefix_table, "prefix_table", groups)
        elif t.group_start is not None or t.prefix_table is not None:
            raise ValueError("prefix_lens: missing beside group_start / prefix_table")
        if out is None:
            out = self.out[:n]
        else:
            _aligned(_on(out, "out", self.dev, torch.bfloat16, (n, self.q_heads, HEAD_DIM)), "out")
        a = L.PrefixAttnArgs()
        a.tokens, a.q_heads, a.kv_heads, a.seqs, a.groups = n, self.q_heads, self.kv_heads, seqs, groups
        a.q, a.q_ld = q.data_ptr(), ld
        a.k_cache, a.v_cache, a.n_pages = k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0]
        a.q_start, a.page_table, a.pt_ld, a.lens = t.q_start.data_ptr(), t.page_table.data_ptr(), t.page_table.shape[1], t.lens.data_ptr()
        if groups:
            a.group_start, a.prefix_lens = t.group_start.data_ptr(), t.prefix_lens.data_ptr()
            a.prefix_table, a.prefix_ld = t.prefix_table.data_ptr(), t.prefix_table.shape[1]
        a.k_scale, a.v_scale, a.sm_scale = self.k_scale, self.v_scale, self.sm_scale
        a.scratch, a.scratch_bytes = self.scratch.data_ptr(), self.scratch.numel()
        a.out, a.guard, a.wait_ns = out.data_ptr(), self.guard.data_ptr(), int(self.deadline_s * 1e9)
        with torch.cuda.device(self.dev):
            L.check(L.load().mono_prefix_attn_launch(C.byref(a), ops._stream()), "mono_prefix_attn_launch")
        return out
