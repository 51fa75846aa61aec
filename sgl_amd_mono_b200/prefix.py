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
_VIEWS = 64  # views that an op keeps of one of its buffers


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
    if not 2.0**-100 <= x <= 2.0**100:
        raise ValueError(f"{name}: {x}, needs a positive number, 2**-100 .. 2**100")
    return x


def _on(t: torch.Tensor, name: str, dev: torch.device, dtype=None, shape=None) -> int:
    """The address of a tensor that is what it has to be (a step makes some thirty of these checks: the common case is
    four comparisons)."""
    if not (isinstance(t, torch.Tensor) and t.device == dev and (dtype is None or t.dtype is dtype) and (shape is None or t.shape == shape)
            and t.is_contiguous()):
        ops.require(t, name, dtype, shape)
        raise ValueError(f"{name}: on {t.device}, the op was built for {dev}")
    return t.data_ptr()


def _aligned(address: int, name: str) -> int:
    if address % 16:
        raise ValueError(f"{name}: must start on a 16-byte address")
    return address


def _caches(a, k_cache, v_cache, kv_heads: int, dev) -> None:
    a.k_cache = _aligned(_on(k_cache, "k_cache", dev, torch.uint8), "k_cache")
    shape = k_cache.shape
    if len(shape) != 4 or shape[0] < 1 or shape[1:] != (PAGE, kv_heads, HEAD_DIM):
        raise ValueError(f"k_cache: shape {tuple(shape)}, needs [pages, {PAGE}, {kv_heads}, {HEAD_DIM}]")
    a.v_cache = _aligned(_on(v_cache, "v_cache", dev, torch.uint8, shape), "v_cache")
    a.n_pages = shape[0]


def _front(views: dict, n: int) -> torch.Tensor:
    """The first ``n`` rows of an op's buffer (``views[0]``), the views of some row counts kept: a slice costs what a launch
    costs, and prompts come in any length."""
    v = views.get(n)
    if v is None:
        if len(views) > _VIEWS:
            base = views[0]
            views.clear()
            views[0] = base
        v = views[n] = views[0][:n]
    return v


def _launch(fn, a, index: int, what: str) -> None:
    """Enqueues on the current stream of device ``index``, whichever device is current."""
    stream = torch._C._cuda_getCurrentRawStream(index)  # (the Stream object around it costs a microsecond)
    if torch.cuda.current_device() == index:
        rc = fn(C.byref(a), stream)
    else:
        with torch.cuda.device(index):
            rc = fn(C.byref(a), stream)
    if rc:
        L.check(rc, what)


class QkvAppendOp:
    """``q = rope(norm(q))`` per head, and K / V of the same rows into the paged caches.

    Per q and k head: RMSNorm over the 128 dims with weight ``1 + g``, then the rotation of the first ``rot_dim`` dims
    in pairs ``(i, i + rot_dim / 2)`` or, ``interleaved``, ``(2i, 2i + 1)``.  f32 arithmetic, rounded once at the store:
    q to bf16, k and v to E4M3 of ``value / scale``."""

    def __init__(self, q_heads: int, kv_heads: int, device, max_tokens: int, rot_dim: int = 64, interleaved: bool = False,
                 eps: float = 1e-6, k_scale: float = 1.0, v_scale: float = 1.0):
        _heads(q_heads, kv_heads)
        if q_heads > 256:
            raise ValueError(f"q_heads: {q_heads}, needs at most 256")
        if not 1 <= max_tokens <= 1 << 24:
            raise ValueError(f"max_tokens: {max_tokens}, needs 1..2**24")
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
        self._views = {0: self.q}
        self.width = (q_heads + 2 * kv_heads) * HEAD_DIM
        self._fn = L.load().mono_qkv_append_launch
        self._fixed = f = L.QkvAppendArgs()  # what no call changes
        f.q_heads, f.kv_heads, f.rot_dim, f.interleaved, f.eps = q_heads, kv_heads, rot_dim, int(self.interleaved), self.eps
        f.k_scale, f.v_scale, f.q_out = self.k_scale, self.v_scale, self.q.data_ptr()

    def __call__(self, qkv: torch.Tensor, g_q, g_k, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, slots,
                 k_cache: torch.Tensor, v_cache: torch.Tensor, tokens: int | None = None) -> torch.Tensor:
        """``qkv``: bf16 ``[tokens, (q_heads + 2 kv_heads) * 128]`` (rows may lie further apart), or f32 partial sums
        ``[nsum, rows, ..]`` of at most 16 ``tokens`` as the projection's GEMV leaves them (``tokens`` is then required).  Of
        wider rows, such as those of ``gqa.GqaConfig.qkv_rows`` with index heads at their end, the q | k | v part is given,
        ``qkv[..., : (q_heads + 2 * kv_heads) * 128]``.
        ``g_q`` / ``g_k``: bf16 ``[128]``, None for no norm.  ``cos`` / ``sin``: bf16 or f32 ``[positions, rot_dim / 2]``.
        ``positions``, ``slots``: int64 ``[tokens]``; a position outside the table is taken to its nearest row, a slot
        (page * 64 + offset) outside the cache inserts nothing, and the slots inside it must differ.
        Returns q ``[tokens, q_heads, 128]`` (the op's own buffer)."""
        width, dev = self.width, self.dev
        a = L.QkvAppendArgs.from_buffer_copy(self._fixed)
        if not isinstance(qkv, torch.Tensor) or qkv.device != dev:
            raise ValueError(f"qkv: must be a tensor on {dev} (there is no CPU path)")
        shape = qkv.shape
        if qkv.dtype is torch.bfloat16:
            if len(shape) != 2 or shape[1] != width or qkv.stride(1) != 1 or (shape[0] > 1 and qkv.stride(0) < width):
                raise ValueError(f"qkv: shape {tuple(shape)} strides {qkv.stride()}, needs [tokens, {width}] with contiguous rows")
            n = shape[0]
            if tokens is not None and tokens != n:
                raise ValueError(f"qkv: {n} rows, tokens says {tokens}")
            ld = qkv.stride(0) if n > 1 else width
            if ld % 8:
                raise ValueError(f"qkv: rows {ld} values apart, needs a multiple of 8")
            a.src_bf16, a.src_ld = _aligned(qkv.data_ptr(), "qkv"), ld
        elif qkv.dtype is torch.float32:
            if len(shape) != 3 or shape[0] < 1 or shape[2] != width or qkv.stride(2) != 1 or (shape[1] > 1 and qkv.stride(1) < width):
                raise ValueError(f"qkv: shape {tuple(shape)} strides {qkv.stride()}, needs f32 partial sums [nsum, rows, {width}] with contiguous rows")
            if tokens is None or not 1 <= tokens <= min(L.MAX_ROWS, shape[1]):
                raise ValueError(f"tokens: {tokens}, partial sums of {shape[1]} rows serve 1..{min(L.MAX_ROWS, shape[1])}")
            n = tokens
            ld, apart = qkv.stride(1) if shape[1] > 1 else width, qkv.stride(0) if shape[0] > 1 else 0
            if ld % 8 or apart % 4:
                raise ValueError(f"qkv: rows {ld} and partial sums {apart} values apart, needs multiples of 8 and 4")
            a.src_f32, a.nsum, a.src_ld, a.sum_stride = _aligned(qkv.data_ptr(), "qkv"), shape[0], ld, apart
        else:
            raise ValueError(f"qkv: dtype {qkv.dtype}, needs bfloat16 rows or float32 partial sums")
        if not 1 <= n <= self.max_tokens:
            raise ValueError(f"qkv: {n} tokens, the op was built for 1..{self.max_tokens}")
        if g_q is not None:
            a.g_q = _aligned(_on(g_q, "g_q", dev, torch.bfloat16, (HEAD_DIM,)), "g_q")
        if g_k is not None:
            a.g_k = _aligned(_on(g_k, "g_k", dev, torch.bfloat16, (HEAD_DIM,)), "g_k")
        if not isinstance(cos, torch.Tensor) or cos.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("cos: needs a bfloat16 or float32 tensor")
        table = cos.shape
        a.cos = _aligned(_on(cos, "cos", dev), "cos")
        if len(table) != 2 or table[0] < 1 or table[1] != self.rot_dim // 2:
            raise ValueError(f"cos: shape {tuple(table)}, needs [positions, {self.rot_dim // 2}]")
        a.sin = _aligned(_on(sin, "sin", dev, cos.dtype, table), "sin")
        a.table_f32, a.table_rows = cos.dtype is torch.float32, table[0]
        a.positions = _on(positions, "positions", dev, torch.int64, (n,))
        if slots is not None:
            a.slots = _on(slots, "slots", dev, torch.int64, (n,))
        _caches(a, k_cache, v_cache, self.kv_heads, dev)
        a.tokens = n
        _launch(self._fn, a, dev.index, "mono_qkv_append_launch")
        return _front(self._views, n)


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
    the last sequence's tokens keep what they held.  Scores are f32; where many rows share their keys, a query's values are
    held exactly within 2^13 of the row's largest, and to 2^-21 of the largest below that.  Weights are rounded to f16 for
    their product with the values: to 2^-11 of themselves, those below 2^-21 of a row's largest to 2^-32 of the largest.
    ``guard`` holds the error words (``ops.guard_read``): starts that
    fall or leave their range set the argument word."""

    def __init__(self, q_heads: int, kv_heads: int, device, max_tokens: int, max_seqs: int, max_groups: int = 1,
                 k_scale: float = 1.0, v_scale: float = 1.0, sm_scale: float | None = None, guard: torch.Tensor | None = None,
                 deadline_s: float = 5.0):
        _heads(q_heads, kv_heads)
        if not 1 <= max_tokens <= 1 << 20 or max_seqs < 1 or max_groups < 0 or max_seqs + max_groups > MAX_ENTRIES:
            raise ValueError(f"max_tokens {max_tokens}, max_seqs {max_seqs}, max_groups {max_groups}: needs 1..2**20 tokens, at least "
                             f"one sequence, and at most {MAX_ENTRIES} sequences and groups")
        self.k_scale, self.v_scale = _scale(k_scale, "k_scale"), _scale(v_scale, "v_scale")
        self.sm_scale = _scale(sm_scale, "sm_scale") if sm_scale is not None else HEAD_DIM ** -0.5
        if self.k_scale * self.sm_scale > 2.0**100:
            raise ValueError(f"sm_scale: {self.sm_scale}, needs at most 2**100 / k_scale")
        self.dev = _device(device)
        self.q_heads, self.kv_heads = q_heads, kv_heads
        self.max_tokens, self.max_seqs, self.max_groups = max_tokens, max_seqs, max_groups
        with torch.cuda.device(self.dev):
            nbytes = L.load().mono_prefix_attn_scratch_bytes(max_tokens, q_heads, kv_heads, max_seqs, max_groups)
        self.scratch = torch.zeros(nbytes, dtype=torch.uint8, device=self.dev)
        self.out = torch.zeros(max_tokens, q_heads, HEAD_DIM, dtype=torch.bfloat16, device=self.dev)
        self._views = {0: self.out}
        self.guard = guard if guard is not None else torch.zeros(L.GUARD_WORDS, dtype=torch.int32, device=self.dev)
        _on(self.guard, "guard", self.dev, torch.int32)
        if self.guard.numel() < L.GUARD_WORDS:
            raise ValueError(f"guard: {self.guard.numel()} words, needs {L.GUARD_WORDS}")
        self._fn = L.load().mono_prefix_attn_launch
        self._fixed = f = L.PrefixAttnArgs()  # what no call changes
        f.q_heads, f.kv_heads, f.k_scale, f.v_scale, f.sm_scale = q_heads, kv_heads, self.k_scale, self.v_scale, self.sm_scale
        f.scratch, f.scratch_bytes, f.out = self.scratch.data_ptr(), nbytes, self.out.data_ptr()
        f.guard, f.wait_ns = self.guard.data_ptr(), int(deadline_s * 1e9)

    def _table(self, t, name: str, rows: int) -> tuple[int, int]:
        address = _on(t, name, self.dev, torch.int32)
        if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
            raise ValueError(f"{name}: shape {tuple(t.shape)}, needs [{rows}, at least 1]")
        return address, t.shape[1]

    def __call__(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, t: PrefixTables,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """``q``: bf16 ``[tokens, q_heads, 128]`` (token rows may lie further apart).  Returns ``out`` (default: the
        op's own buffer), bf16 ``[tokens, q_heads, 128]``."""
        dev = self.dev
        if not isinstance(q, torch.Tensor) or q.device != dev:
            raise ValueError(f"q: must be a tensor on {dev} (there is no CPU path)")
        if q.dtype is not torch.bfloat16:
            raise ValueError(f"q: dtype {q.dtype}, needs torch.bfloat16")
        shape, strides = q.shape, q.stride()
        if len(shape) != 3 or shape[1] != self.q_heads or shape[2] != HEAD_DIM:
            raise ValueError(f"q: shape {tuple(shape)}, needs [tokens, {self.q_heads}, {HEAD_DIM}]")
        n = shape[0]
        if not 1 <= n <= self.max_tokens:
            raise ValueError(f"q: {n} tokens, the op was built for 1..{self.max_tokens}")
        width = self.q_heads * HEAD_DIM
        ld = strides[0] if n > 1 else width
        if strides[2] != 1 or (self.q_heads > 1 and strides[1] != HEAD_DIM) or ld < width or ld % 8:
            raise ValueError(f"q: strides {strides}, needs contiguous heads and token rows a multiple of 8 values apart")
        a = L.PrefixAttnArgs.from_buffer_copy(self._fixed)
        a.tokens, a.q, a.q_ld = n, _aligned(q.data_ptr(), "q"), ld
        _caches(a, k_cache, v_cache, self.kv_heads, dev)
        a.lens = _on(t.lens, "lens", dev, torch.int32)
        seqs = t.lens.shape[0] if t.lens.dim() == 1 else 0
        if not 1 <= seqs <= self.max_seqs:
            raise ValueError(f"lens: shape {tuple(t.lens.shape)}, the op was built for 1..{self.max_seqs} sequences")
        a.seqs = seqs
        a.q_start = _on(t.q_start, "q_start", dev, torch.int32, (seqs + 1,))
        a.page_table, a.pt_ld = self._table(t.page_table, "page_table", seqs)
        if t.prefix_lens is not None:
            a.prefix_lens = _on(t.prefix_lens, "prefix_lens", dev, torch.int32)
            groups = t.prefix_lens.shape[0] if t.prefix_lens.dim() == 1 else 0
            if not 1 <= groups <= self.max_groups:
                raise ValueError(f"prefix_lens: shape {tuple(t.prefix_lens.shape)}, the op was built for up to {self.max_groups} groups")
            a.groups = groups
            a.group_start = _on(t.group_start, "group_start", dev, torch.int32, (groups + 1,))
            a.prefix_table, a.prefix_ld = self._table(t.prefix_table, "prefix_table", groups)
        elif t.group_start is not None or t.prefix_table is not None:
            raise ValueError("prefix_lens: missing beside group_start / prefix_table")
        if out is None:
            out = _front(self._views, n)
        else:
            a.out = _aligned(_on(out, "out", dev, torch.bfloat16, (n, self.q_heads, HEAD_DIM)), "out")
        _launch(self._fn, a, dev.index, "mono_prefix_attn_launch")
        return out
