"""Sampling on the GPU over the fp32 logits of a decode step: `sample` with one temperature and top-k, `sample_rows` with a temperature, top-k, top-p and
min-p of its own for every row.

The reference decodes greedily and returns the fp32 logits "for the caller" (qwen3mk/kernel.py:44-50); this module is
the step after that: `sample` picks one token per row through the C ABI (`q3_sample`), with the uniform numbers drawn
from a seeded generator so that a run can be repeated, and can write straight into the token buffer the next launch
reads.  `sample_reference` states the same rule in plain PyTorch on whatever device the logits are on; it is the
documentation of the rule, not a fallback (`sample` fails without the CUDA library).
"""
from __future__ import annotations

import contextlib

import torch

from . import _cabi
from ._stream import raw_stream as _raw_stream


def sample(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0, *, generator: torch.Generator | None = None,
           u: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of `logits` (CUDA fp32 [vocab] or [batch, vocab]).  top_k = 0 keeps the whole vocabulary;
    temperature <= 0 or top_k = 1 is the arg-max.  `u` (CUDA fp32 [batch], values in [0, 1)) overrides the generator.
    Enqueues on the current stream and returns the int64 tensor of tokens (`out` when given) without synchronising."""
    if not logits.is_cuda or logits.dtype != torch.float32 or not logits.is_contiguous():
        raise ValueError("sample: logits must be a contiguous CUDA float32 tensor")
    rows = logits.reshape(-1, logits.shape[-1])
    batch, vocab = rows.shape
    if u is None:
        u = torch.rand(batch, device=logits.device, dtype=torch.float32, generator=generator)
    if u.dtype != torch.float32 or u.numel() != batch or not u.is_cuda:
        raise ValueError(f"sample: u must be a CUDA float32 tensor of {batch} numbers")
    if out is None:
        out = torch.empty(logits.shape[:-1], dtype=torch.int64, device=logits.device)
    elif out.dtype != torch.int64 or out.numel() != batch or not out.is_cuda:
        raise ValueError(f"sample: out must be a CUDA int64 tensor of {batch} elements")
    lib = _cabi.load()
    rc = lib.q3_sample(rows.data_ptr(), batch, vocab, float(temperature), int(top_k), u.data_ptr(), out.data_ptr(),
                       torch.cuda.current_stream(logits.device).cuda_stream)
    _cabi.check(lib, None, rc, "q3_sample")
    return out


def sample_reference(logits: torch.Tensor, temperature: float, top_k: int, u: torch.Tensor) -> torch.Tensor:
    """The sampling rule in PyTorch (fp64): keep logits >= the k-th largest, weigh by exp((l - max) / T), return the first
    index whose cumulative weight exceeds u * total."""
    rows = logits.reshape(-1, logits.shape[-1]).double()
    if temperature <= 0 or top_k == 1:
        return rows.argmax(dim=-1).reshape(logits.shape[:-1])
    keep = rows > float("-inf")         # a masked word weighs nothing, at an infinite temperature too
    if 0 < top_k < rows.shape[-1]:
        kth = rows.topk(top_k, dim=-1).values[:, -1:]
        keep &= rows >= kth
    w = torch.where(keep, torch.exp((rows - rows.max(dim=-1, keepdim=True).values) / temperature), torch.zeros_like(rows))
    cdf = w.cumsum(dim=-1)
    target = u.reshape(-1, 1).double().to(rows.device) * cdf[:, -1:]
    return (cdf > target).double().argmax(dim=-1).reshape(logits.shape[:-1])


_NO_SWITCH = contextlib.nullcontext()
_FILTERS = (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32))


def sample_rows(logits: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, *, u: torch.Tensor | None = None, generator: torch.Generator | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of `logits` (CUDA fp32 [batch, vocab], contiguous words, any row stride), each filter a number or a CUDA tensor [batch] (float32; top_k int32).

    A row keeps its top_k largest logits (0: all; ties are all kept), of these the most likely words until their weights exp((l - max) / temperature) reach top_p of their sum
    (equal words: the lowest index first), of these the words of at least min_p times the most likely one's weight; the token is the first index whose cumulative weight
    exceeds u times the total.  temperature <= 0, top_k = 1, top_p = 0 or min_p > 1: the arg-max.  `u` (CUDA fp32 [batch], in [0, 1)) overrides the generator.
    Enqueues on the current stream of the logits' device and returns the int64 tokens [batch] (`out` when given) without synchronising; equal inputs draw equal words."""
    if not logits.is_cuda or logits.dtype != torch.float32 or logits.dim() != 2 or logits.shape[0] < 1 or (logits.shape[1] != 1 and logits.stride(1) != 1):
        raise ValueError("sample_rows: logits must be a CUDA float32 tensor [batch, vocab] with contiguous words")
    (batch, vocab), dev = logits.shape, logits.device
    ptrs, values, size = [], [], (batch,)
    for (name, dtype), x in zip(_FILTERS, (temperature, top_k, top_p, min_p)):
        if isinstance(x, torch.Tensor):
            if x.dtype != dtype or x.shape != size or x.device != dev or not x.is_contiguous():
                raise ValueError(f"sample_rows: {name} must be a number or a contiguous {dtype} tensor [{batch}] on {dev}")
            ptrs.append(x.data_ptr()), values.append(0)
        else:
            ptrs.append(None), values.append(x)
    if u is None:
        u = torch.rand(batch, device=dev, dtype=torch.float32, generator=generator)
    elif u.dtype != torch.float32 or u.shape != (batch,) or u.device != dev or not u.is_contiguous():
        raise ValueError(f"sample_rows: u must be a contiguous float32 tensor [{batch}] on {dev}")
    if out is None:
        out = torch.empty(batch, dtype=torch.int64, device=dev)
    elif out.dtype != torch.int64 or out.shape != (batch,) or out.device != dev or not out.is_contiguous():
        raise ValueError(f"sample_rows: out must be a contiguous int64 tensor [{batch}] on {dev}")
    lib = _cabi.load()
    a = _cabi.SampleRowsArgs(logits.data_ptr(), logits.stride(0) if batch > 1 else vocab, *ptrs, u.data_ptr(), out.data_ptr(), batch, vocab, float(values[0]), min(int(values[1]), 0x7fffffff),
                             float(values[2]), float(values[3]))
    with _NO_SWITCH if torch.cuda.current_device() == dev.index else torch.cuda.device(dev):
        rc = lib.q3_sample_rows(a, _raw_stream(dev.index))
    if rc:
        _cabi.check(lib, None, rc, "q3_sample_rows")
    return out
