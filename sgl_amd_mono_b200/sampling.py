"""Next tokens from the LM head's logits and given random numbers (``tail.LmHeadOp`` makes the logits).

Row r: ``w_i = exp((logit_i - max) / temperature)``.  The tokens in order of (logit descending, index ascending); kept is
the front part with rank < ``top_k``, mass before the token < ``top_p`` of the whole mass, and ``w_i >= min_p``, at
least the first token.  The drawn token is the first, by index, whose running kept mass passes ``u`` times the kept
mass, so the same numbers draw the same tokens on every run.

An op allocates its outputs when it is built; a call enqueues one kernel on its device's current stream and may be
captured into a CUDA graph.  The returned tensors are overwritten by the next call.
"""

from __future__ import annotations


import torch

from . import _lib as L
from .prefix import _device, _front, _launch, _on


class SampleOp:
    def __init__(self, vocab: int, device, max_rows: int):
        if not 1 <= vocab <= L.SAMPLE_MAX_VOCAB:
            raise ValueError(f"vocab: {vocab}, needs 1..{L.SAMPLE_MAX_VOCAB}")
        if not 1 <= max_rows <= 65535:
            raise ValueError(f"max_rows: {max_rows}, needs 1..65535")
        self.dev = _device(device)
        L.load()
        self.vocab, self.max_rows = vocab, max_rows
        self.tokens = torch.zeros(max_rows, dtype=torch.int64, device=self.dev)
        self.logprobs = torch.zeros(max_rows, dtype=torch.float32, device=self.dev)
        self._tokens, self._logprobs = {0: self.tokens}, {0: self.logprobs}  # and their views by rows
        self._fn, self._out = L.load().mono_sample_launch, (self.tokens.data_ptr(), self.logprobs.data_ptr())

    def __call__(self, logits: torch.Tensor, u: torch.Tensor, temperature=None, top_k=None, top_p=None, min_p=None):
        """``logits``: f32 or bf16 ``[rows, vocab]`` (rows may lie further apart); ``u``: f32 ``[rows]`` in [0, 1);
        ``temperature``, ``top_p``, ``min_p``: f32 ``[rows]``, ``top_k``: int32 ``[rows]``, each None for "not used".
        Temperature 0 or below takes the best token.  Returns (tokens int64 ``[rows]``, logprobs f32 ``[rows]``): the
        drawn token's log probability at the row's temperature before any filter (at temperature 1 for greedy rows).  A
        row whose logits are all -inf or NaN gives token -1."""
        dev = self.dev
        if not isinstance(logits, torch.Tensor) or logits.device != dev:
            raise ValueError(f"logits: must be a tensor on {dev} (there is no CPU path)")
        if logits.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"logits: dtype {logits.dtype}, needs float32 or bfloat16")
        shape = logits.shape
        if len(shape) != 2 or shape[1] != self.vocab or not 1 <= shape[0] <= self.max_rows:
            raise ValueError(f"logits: shape {tuple(shape)}, needs [1..{self.max_rows}, {self.vocab}]")
        rows = shape[0]
        ld = logits.stride(0) if rows > 1 else self.vocab
        if (self.vocab > 1 and logits.stride(1) != 1) or ld < self.vocab:
            raise ValueError(f"logits: strides {logits.stride()}, needs contiguous rows")
        a = L.SampleArgs()
        a.rows, a.vocab, a.logits, a.ld, a.logits_bf16 = rows, self.vocab, logits.data_ptr(), ld, logits.dtype is torch.bfloat16
        n = (rows,)
        a.u = _on(u, "u", dev, torch.float32, n)
        if temperature is not None:
            a.temperature = _on(temperature, "temperature", dev, torch.float32, n)
        if top_k is not None:
            a.top_k = _on(top_k, "top_k", dev, torch.int32, n)
        if top_p is not None:
            a.top_p = _on(top_p, "top_p", dev, torch.float32, n)
        if min_p is not None:
            a.min_p = _on(min_p, "min_p", dev, torch.float32, n)
        a.tokens, a.logprobs = self._out
        _launch(self._fn, a, dev.index, "mono_sample_launch")
        return _front(self._tokens, rows), _front(self._logprobs, rows)
