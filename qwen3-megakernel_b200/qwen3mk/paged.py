"""Many sequences in one pool of cache pages: the operators of a server that keeps more conversations than it decodes at once.

  pool = PagePool.empty(layers=28, pages=4096, page_size=64)       K and V pages of every layer
  batch = PagedBatch(pool, page_table, q_start, kv_len)            which pages belong to whom, who brings how many new tokens
  q = rope_append(batch, q, k, v, table, layer, q_gain=..., k_gain=...)    head norm and rotary embedding; k and v rows into the pages
  o = attention(batch, q, layer)                                   the new tokens attend their sequences' pages

Position p of sequence b is slot p % page_size of page page_table[b, p // page_size].  An entry outside the pool (-1, say) is a page that is
not there: nothing is written to it and its positions are not attended; so are positions behind the table's row.  The new tokens' rows lie one sequence after the other, sequence b's from
q_start[b] to q_start[b + 1]; they are its last positions of kv_len[b], which counts them.  One new token is a decode step, many are a prompt or
a chunk of one, none is a sequence that sits this call out.

As everywhere in this package nothing here synchronises, the descriptors are read on the device when the call runs (so a captured call may be replayed
with others), every tensor is borrowed, and there is no path without the CUDA library.  The reference keeps one contiguous cache of 128 positions
(qwen3mk/kernel.py:27-50); `Megakernel.extend` is the whole model over such a pool.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import _cabi
from ._stream import raw_stream as _raw_stream

HEAD_DIM = 128
ROPE_THETA = 1e6
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NO_SWITCH = contextlib.nullcontext()
_current_device = torch.cuda.current_device


def _on(device: torch.device):
    """The library launches on the current device: the tensors' own for the length of a call."""
    return _NO_SWITCH if _current_device() == device.index else torch.cuda.device(device)


class PagePool:
    """K and V pages of every layer: two CUDA tensors [layers, pages, page_size, kv_heads, 128] of bf16 or fp16, with the same strides; the last dimension is
    contiguous, the others may be permuted (pass a view)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 5 or k.shape[-1] != HEAD_DIM or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            raise ValueError(f"PagePool: expected K and V pages [layers, pages, page_size, kv_heads, {HEAD_DIM}] alike in shape, strides, type and device, "
                             f"got {tuple(k.shape)} {k.dtype} on {k.device} and {tuple(v.shape)} {v.dtype} on {v.device}")
        if k.dtype not in (torch.bfloat16, torch.float16) or not k.is_cuda or k.stride(-1) != 1:
            raise ValueError(f"PagePool: expected CUDA bf16 or fp16 pages with a contiguous last dimension, got {k.dtype} on {k.device}, strides {k.stride()}")
        self.k, self.v = k, v
        self.layers, self.pages, self.page_size, self.kv_heads = (int(x) for x in k.shape[:4])
        self.device, self.dtype = k.device, k.dtype
        self._status = torch.zeros(4, dtype=torch.int32, device=k.device)      # what `attention` reports of a wait that gave up

    def status(self, stream=None) -> list[int]:
        """Synchronise a stream (the current one, a Stream or its address) and read the status words of `attention` over this pool; raises RuntimeError, and clears them, if a wait inside a kernel gave
        up: rows of that call are NaN.  (`Megakernel.extend` reports to `Megakernel.status`.)"""
        if stream is None:
            stream = torch.cuda.current_stream(self.device)
        elif isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=self.device)
        stream.synchronize()
        words = self._status.tolist()
        if words[0]:
            self._status.zero_()
            raise RuntimeError(f"paged attention: device status: code {words[0]} at site {words[1]}, CTA {words[2]}, value {words[3]}")
        return words

    @classmethod
    def empty(cls, *, layers: int = 28, pages: int, page_size: int = 64, kv_heads: int = 8, dtype=torch.bfloat16, device="cuda") -> "PagePool":
        shape = (layers, pages, page_size, kv_heads, HEAD_DIM)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


class PagedBatch:
    """The sequences of a call, described on the device: page_table int32 [B, most pages of a sequence], q_start int32 [B + 1], kv_len int32 [B].

    tokens: rows of q (default: q_start[-1]); rows behind the last sequence's are left as they were.  max_new: most new tokens of a sequence, which
    chooses the kernels and bounds nothing (default: read from q_start).  Both defaults read q_start on the host, once, here.  The tensors are kept
    and may be changed in place between calls.  wait_limit_us: patience of the waits inside `attention`'s kernel (0: 200 ms), as an engine has it; tests set it low."""

    def __init__(self, pool: PagePool, page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, *, tokens: int | None = None, max_new: int | None = None,
                 wait_limit_us: int = 0):
        batch = kv_len.numel()
        for name, t, ok in (("page_table", page_table, page_table.dim() == 2 and page_table.shape[0] == batch and (page_table.shape[1] == 1 or page_table.stride(1) == 1)),
                            ("q_start", q_start, q_start.shape == (batch + 1,) and q_start.is_contiguous()),
                            ("kv_len", kv_len, kv_len.dim() == 1 and batch > 0 and kv_len.is_contiguous())):
            if t.dtype != torch.int32 or t.device != pool.device or not ok:
                raise ValueError(f"PagedBatch: {name}: expected int32 page_table [B, pages], q_start [B + 1], kv_len [B] on {pool.device}, "
                                 f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        if tokens is None or max_new is None:
            starts = q_start.tolist()
            tokens = starts[-1] if tokens is None else tokens
            max_new = max(b - a for a, b in zip(starts, starts[1:])) if max_new is None else max_new
        self.pool, self.page_table, self.q_start, self.kv_len = pool, page_table, q_start, kv_len
        self.device, self.dtypes = pool.device, (pool.dtype,)
        self.batch, self.tokens, self.max_new = batch, int(tokens), int(max_new)
        self.wait_limit_us, self._status = int(wait_limit_us), pool._status.data_ptr()
        self.lib = _cabi.load()
        self._views: dict = {}
        self._space: dict = {}

    def view(self, layer: int) -> _cabi.Paged:
        """The C ABI's descriptor of one layer."""
        c = self._views.get(layer)
        if c is None:
            p = self.pool
            if not 0 <= layer < p.layers:
                raise ValueError(f"layer {layer} outside 0..{p.layers - 1}")
            at = layer * p.k.stride(0) * p.k.element_size()
            t = self.page_table
            c = self._views[layer] = _cabi.Paged(p.k.data_ptr() + at, p.v.data_ptr() + at, t.data_ptr(), self.q_start.data_ptr(), self.kv_len.data_ptr(),
                                                 p.k.stride(1), p.k.stride(2), p.k.stride(3), t.stride(0) if self.batch > 1 else t.shape[1], t.shape[1], p.pages,
                                                 p.page_size, self.batch, self.tokens, self.max_new, p.kv_heads, _TYPES[p.dtype])
        return c

    def workspace_bytes(self, q_heads: int) -> int:
        n = self._space.get(q_heads)
        if n is None:
            with _on(self.pool.device):
                n = self.lib.q3_paged_attn_workspace(self.view(0), q_heads)
            if n < 0:
                _cabi.check(self.lib, None, int(n), "q3_paged_attn_workspace")
            self._space[q_heads] = n
        return n


def _strides(what: str, t: torch.Tensor, batch: PagedBatch, dtypes, heads: int | None = None):
    """The strides of rows [tokens, heads, 128], or ValueError."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 3 or shape[0] != batch.tokens or shape[2] != HEAD_DIM or t.dtype not in dtypes or t.device != batch.device or strides[2] != 1 or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what}: expected [{batch.tokens}, {'heads' if heads is None else heads}, {HEAD_DIM}] of {' or '.join(map(str, dtypes))} on {batch.device} with a contiguous "
                         f"last dimension, got {t.dtype} {tuple(shape)} on {t.device}")
    return strides


def attention(batch: PagedBatch, q: torch.Tensor, layer: int = 0, *, scale: float = HEAD_DIM ** -0.5, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the new tokens over their sequences' pages (whose rows of the new tokens have been written, see rope_append).

    q: [tokens, heads, 128] in the pages' type, heads 1, 2, 4 or 8 times the pool's.  Returns out (q's shape and type; rows that share no memory with one another or with q's).  A token that sees no position gets zeros;
    rows that a token does not see (later tokens', slots behind the last position) do not touch its result, whatever they hold.  Equal bits on every run.  A wait inside the
    kernel that gives up leaves NaN in the rows it could not finish and is reported by `batch.pool.status()`."""
    sq = _strides("attention: q", q, batch, batch.dtypes)
    heads = q.shape[1]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    so = _strides("attention: out", out, batch, batch.dtypes, heads)
    view = batch.view(layer)
    with _on(batch.device):
        space = torch.empty(batch.workspace_bytes(heads), dtype=torch.uint8, device=batch.device)
        a = _cabi.PagedAttnArgs(q.data_ptr(), out.data_ptr(), sq[0], sq[1], so[0], so[1], heads, scale, space.data_ptr(), space.numel(), batch._status)
        rc = batch.lib.q3_paged_attn_limited(view, a, batch.wait_limit_us, _raw_stream(batch.device.index))
    if rc:
        _cabi.check(batch.lib, None, rc, "q3_paged_attn")
    return out


def rope_append(batch: PagedBatch, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rope: torch.Tensor | None, layer: int = 0, *, q_gain: torch.Tensor | None = None,
                k_gain: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False, positions: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """The new tokens' rows: RMS norm of every q and k head (where a gain, bf16 [128], is given), rotary embedding, k and v into the pages.  Returns q's rows in the
    pages' type (`out` when given: q itself where the types agree, or rows that share no memory with q, k and v), as `attention` reads them.

    q [tokens, heads, 128], k and v [tokens, kv_heads, 128]: fp32, bf16 or fp16, all three alike; slices of one projection's rows serve.  rope: fp32
    [positions, rotary_dim], contiguous, a row the cosines and then the sines (`rope_table`); its width says how many dims of a head are rotated (a multiple of 8
    up to 128), None rotates nothing.  interleaved: pairs are neighbours instead of half the rotated dims apart.  positions (int32 [tokens]): rotate by these instead of
    the tokens' places in their sequences.  fp32 inside, one rounding at the end."""
    dev, kv_heads = batch.device, batch.pool.kv_heads
    sq = _strides("rope_append: q", q, batch, _TYPES)
    kind = (q.dtype,)
    sk, sv = _strides("rope_append: k", k, batch, kind, kv_heads), _strides("rope_append: v", v, batch, kind, kv_heads)
    if rope is not None and (rope.dim() != 2 or rope.dtype != torch.float32 or not rope.is_contiguous() or rope.device != dev):
        raise ValueError(f"rope_append: rope: expected a contiguous float32 [positions, rotary_dim] on {dev}, got {rope.dtype} {tuple(rope.shape)} on {rope.device}")
    for name, g in (("q_gain", q_gain), ("k_gain", k_gain)):
        if g is not None and (g.shape != (HEAD_DIM,) or g.dtype != torch.bfloat16 or g.device != dev or not g.is_contiguous()):
            raise ValueError(f"rope_append: {name}: expected a contiguous bfloat16 [{HEAD_DIM}] on {dev}, got {g.dtype} {tuple(g.shape)} on {g.device}")
    if positions is not None and (positions.shape != (batch.tokens,) or positions.dtype != torch.int32 or positions.device != dev or not positions.is_contiguous()):
        raise ValueError(f"rope_append: positions: expected a contiguous int32 [{batch.tokens}] on {dev}")
    heads = q.shape[1]
    if out is None:
        out = torch.empty(q.shape, dtype=batch.pool.dtype, device=dev)
    so = _strides("rope_append: out", out, batch, batch.dtypes, heads)
    n, width = (0, 0) if rope is None else rope.shape
    a = _cabi.PagedRopeArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), sq[0], sq[1], sk[0], sk[1], sv[0], sv[1], so[0], so[1],
                            None if q_gain is None else q_gain.data_ptr(), None if k_gain is None else k_gain.data_ptr(), None if rope is None else rope.data_ptr(),
                            None if positions is None else positions.data_ptr(), heads, _TYPES[q.dtype], n, width, interleaved, eps)
    view = batch.view(layer)
    with _on(dev):
        rc = batch.lib.q3_paged_rope(view, a, _raw_stream(dev.index))
    if rc:
        _cabi.check(batch.lib, None, rc, "q3_paged_rope")
    return out


def rope_table(n_positions: int, device="cuda", *, rotary_dim: int = HEAD_DIM, theta: float = ROPE_THETA, scaling: dict | None = None) -> torch.Tensor:
    """Table of rotary angles, fp32 [n_positions, rotary_dim]: row p is cos(p f) and then sin(p f) of the rotary_dim / 2 frequencies f = theta^(-2i/rotary_dim), from
    angles in 64 bits.  `Megakernel.set_rope` takes one of 128 columns, `rope_append` any.

    scaling stretches the table beyond the `original` positions that a model was trained on, by `factor`:
      {"type": "linear", "factor"}                              angles divided by the factor
      {"type": "ntk", "factor"}                                 a larger theta: the slowest frequency divided by the factor, the fastest kept
      {"type": "yarn", "factor", "original", "beta_fast" = 32, "beta_slow" = 1, "attention" = 0.1 ln(factor) + 1}
                                                                frequencies of more than beta_fast turns over the original length kept, of fewer than beta_slow divided
                                                                by the factor, a ramp between; cosines and sines times `attention`, so scores grow by its square
      {"type": "llama3", "factor", "original", "low" = 1, "high" = 4}     the same idea: kept above `high` turns, divided below `low`, a ramp in the turns between"""
    if rotary_dim < 2 or rotary_dim > HEAD_DIM or rotary_dim % 2 or n_positions < 1:
        raise ValueError(f"rope_table: rotary_dim {rotary_dim} (even, 2..{HEAD_DIM}) or n_positions {n_positions} out of range")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    freq, gain = theta ** (-2 * i / rotary_dim), 1.0
    if scaling is not None:
        known = {"linear": (), "ntk": (), "yarn": ("original", "beta_fast", "beta_slow", "attention"), "llama3": ("original", "low", "high")}
        kind = scaling.get("type")
        if kind not in known or set(scaling) - {"type", "factor", *known[kind]} or not scaling.get("factor", 0) >= 1 or ("original" in known[kind] and not scaling.get("original", 0) > 0):
            raise ValueError(f"rope_table: scaling {scaling}: expected type linear, ntk, yarn or llama3, factor >= 1 and what the type takes")
        factor = float(scaling["factor"])
        if kind == "linear":
            freq = freq / factor
        elif kind == "ntk":
            freq = (theta * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2 * i / rotary_dim) if rotary_dim > 2 else freq / factor
        elif kind == "yarn":
            # the frequency that makes `turns` turns over the original length has this (fractional) index
            at = lambda turns: rotary_dim * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            low = max(math.floor(at(scaling.get("beta_fast", 32))), 0)
            high = min(math.ceil(at(scaling.get("beta_slow", 1))), rotary_dim - 1)
            divided = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
            freq = freq / factor * divided + freq * (1 - divided)
            gain = float(scaling.get("attention", 0.1 * math.log(factor) + 1))
        else:
            turns = scaling["original"] * freq / (2 * math.pi)
            lo, hi = float(scaling.get("low", 1)), float(scaling.get("high", 4))
            kept = ((turns - lo) / (hi - lo)).clamp(0, 1)
            freq = freq / factor * (1 - kept) + freq * kept
    ang = torch.arange(n_positions, dtype=torch.float64)[:, None] * freq
    return (torch.cat([ang.cos(), ang.sin()], dim=1) * gain).float().contiguous().to(device)
