"""Products in 8-bit integers with a factor per token and per channel, and what stands between them in a decoder: rows turned into 8 bits, and
the norms around a block with its gate and residual scale, whose result is a product's left side.

:func:`gemm_int8` is the counterpart of :func:`onnx_genai_b200.ops.gemm` for weights that :func:`quantize_weight` (or
:func:`quantize_gate_up`) has made.  Weights take a byte a value; activations are quantised a token at a time when a product reads them, so
no calibration is needed.  CUDA tensors run the kernels of ``libogb_cuda.so`` on the current stream of the tensors' device; CPU tensors run
the statements of :mod:`onnx_genai_b200.ops.reference`.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from . import _native, _raw_stream, _timed, current_index, launch_counts, reference, status_word

P, I, L, F = _native.P, _native.I, _native.L, _native.F
_native.register("ogb_quantize_rows", [P] * 3 + [I] * 2 + [L] * 2 + [I, P])
_native.register("ogb_gemm_int8_workspace", [I] * 5, L)
_native.register("ogb_gemm_int8", [P, I, L, P, P, L, P, L, P, P, P, L, P, L] + [I] * 5 + [P, L, P, P])
_native.register("ogb_block_norm", [P] * 9 + [L] * 6 + [I] * 8 + [F] * 3 + [P])

ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_K = 131072          # sums of 128 * 127 * K stay below 2^31
MAX_HIDDEN = 16384      # a row of block_norm stays in registers
_EPI = ("none", "residual", "swiglu")


class Int8Rows(NamedTuple):
    """Rows in 8 bits: ``q`` [rows, k] int8 whose rows begin at multiples of 16 bytes, ``scale`` [rows] fp32; a row stands for ``q * scale``."""
    q: torch.Tensor
    scale: torch.Tensor

    def float(self) -> torch.Tensor:
        return self.q.float() * self.scale[:, None]


def _refuse(what):
    raise ValueError(what)


def _padded(rows, k, device):
    """[rows, k] int8 whose rows begin at multiples of 16 bytes."""
    if k % 16 == 0:
        return torch.empty(rows, k, dtype=torch.int8, device=device)
    return torch.empty(rows, (k + 15) // 16 * 16, dtype=torch.int8, device=device)[:, :k]


@_timed("quantize_rows")
def quantize_rows(x) -> Int8Rows:
    """``scale = max |x| / 127`` and ``q = round(127 x / max |x|)`` (halves to even) of every row of ``x`` [rows, k] (fp32, bf16, fp16; any
    strides).  A row of zeros has scale 0; one that holds an infinity or a NaN has scale NaN and zeros."""
    if x.dim() != 2 or x.dtype not in ELEM:
        _refuse(f"x must be a matrix of fp32, bf16 or fp16, not {tuple(x.shape)} {x.dtype}")
    rows, k = x.shape
    if k == 0:
        _refuse("rows without values have no scale")
    if k > 1 and x.stride(1) != 1:
        x = x.contiguous()
    dev = x.device
    q = _padded(rows, k, dev)
    if not x.is_cuda:
        codes, scale = reference.quantize_rows(x)
        q.copy_(codes)
        return Int8Rows(q, scale)
    index = dev.index
    if index != current_index():
        with torch.cuda.device(index):
            return quantize_rows(x)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    rc = _native.load().ogb_quantize_rows(x.data_ptr(), q.data_ptr(), scale.data_ptr(), rows, k, x.stride(0), q.stride(0), ELEM[x.dtype], _raw_stream(index))
    _native.check(rc, "ogb_quantize_rows")
    launch_counts["quantize_rows"] += 1
    return Int8Rows(q, scale)


def quantize_weight(w) -> Int8Rows:
    """A weight [n, k] in 8 bits with a factor per output channel, laid out for :func:`gemm_int8`.  Weights have to be finite."""
    if not bool(torch.isfinite(w).all()):
        _refuse("a weight that is not finite cannot be held in 8 bits")
    return quantize_rows(w)


def quantize_gate_up(gate, up) -> Int8Rows:
    """Gate and up projections [inter, k] as one weight for ``epilogue="swiglu"``: blocks of 128 gate rows and their 128 up rows, ``inter``
    padded with zero rows to a multiple of 128 (the padded columns of the result are zero: pad the next weight's k with anything)."""
    if gate.shape != up.shape or gate.dim() != 2:
        _refuse("gate and up projections have one shape")
    pad = (-gate.shape[0]) % 128
    if pad:
        zero = gate.new_zeros(pad, gate.shape[1])
        gate, up = torch.cat([gate, zero]), torch.cat([up, zero])
    return quantize_weight(reference.pack_gate_up(gate, up, 128))


@_timed("gemm_int8")
def gemm_int8(a, w, w_scale, bias=None, residual=None, epilogue="none", out=None, out_dtype=None):
    """``out[M, N] = a @ (w * w_scale[:, None])^T (+ bias) (+ residual)``, or SwiGLU over a :func:`quantize_gate_up` weight (``epilogue="swiglu"``,
    out [M, N / 2]).

    ``a`` [M, K]: float rows, which the call turns into 8 bits (:func:`quantize_rows`), or :class:`Int8Rows`.  ``w`` [N, K] int8, rows at
    multiples of 16 bytes; ``w_scale`` and ``bias`` [N] fp32.  ``residual`` has the type of the result; ``out`` may be the same tensor.  The result's
    type is ``out_dtype``, that of ``out`` or of ``residual``, or that of float rows, else bf16.  Sums over K are exact; one rounding follows the
    factors, the bias and the residual."""
    rows = isinstance(a, Int8Rows)
    x = a.q if rows else a
    gated = epilogue == "swiglu"
    if epilogue not in _EPI:
        _refuse(f"epilogue {epilogue!r}: one of {', '.join(_EPI)}")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        _refuse(f"a {tuple(x.shape)} and w {tuple(w.shape)} do not multiply")
    m, k = x.shape
    n, dev = w.shape[0], x.device
    if (x.dtype != torch.int8) if rows else (x.dtype not in ELEM):
        _refuse(f"rows of {x.dtype}")
    if not 0 < k <= MAX_K:
        _refuse(f"k = {k}: between 1 and {MAX_K}")
    if w.dtype != torch.int8 or w.device != dev:
        _refuse("w must be int8 on the device of a")
    if w_scale is None or not _channels(w_scale, n, dev) or not (bias is None or _channels(bias, n, dev)):
        _refuse(f"w_scale and bias: {n} contiguous fp32 values each on the device of a")
    if gated and (n % 256 or residual is not None):
        _refuse("swiglu takes a weight of quantize_gate_up and no residual")
    if epilogue == "residual" and residual is None:
        _refuse("the residual is missing")
    n_out = n // 2 if gated else n
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else residual.dtype if residual is not None else torch.bfloat16 if rows else x.dtype
    if out_dtype not in ELEM:
        _refuse(f"results of {out_dtype}")
    for t in (out, residual):
        if t is not None and (t.shape != (m, n_out) or t.dtype != out_dtype or t.device != dev or (n_out > 1 and t.stride(1) != 1)):
            _refuse(f"out and residual: [{m}, {n_out}] {out_dtype} with neighbouring columns on the device of a")
    if not x.is_cuda:
        y = reference.gemm_int8(a, w, w_scale, bias, residual, gated, out_dtype)
        return y if out is None else out.copy_(y)
    ldw, c1 = w.stride()
    ldx, x1 = x.stride()
    if n == 1:                     # one row has no next: any stride will do
        ldw = (k + 15) // 16 * 16
    if m == 1:
        ldx = (k + 15) // 16 * 16
    if out is not None and m > 1 and out.stride(0) < n_out:
        _refuse("rows of out overlap")
    if (c1 != 1 and k > 1) or ldw % 16 or w.data_ptr() % 16 or ldw < k:
        _refuse("rows of w must begin at multiples of 16 bytes: lay it out by quantize_weight")
    if rows:
        if (x1 != 1 and k > 1) or ldx % 16 or x.data_ptr() % 16 or ldx < k:
            _refuse("8-bit rows must begin at multiples of 16 bytes")
        if not _channels(a.scale, m, dev):
            _refuse("a.scale: a contiguous fp32 value a row on the device of a.q")
    elif x1 != 1 and k > 1:
        x = x.contiguous()
        ldx = k
    index = dev.index
    if index != current_index():
        with torch.cuda.device(index):
            return gemm_int8(a, w, w_scale, bias, residual, epilogue, out, out_dtype)
    if out is None:
        out = torch.empty(m, n_out, dtype=out_dtype, device=dev)
    if m == 0 or n == 0:
        return out
    # the caller's own memory for as long as the call: the allocator hands it on in the stream's order, and a captured graph keeps its own
    size = _workspace(m, n, k, gated, not rows)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    rc = _native.load().ogb_gemm_int8(0 if rows else x.data_ptr(), 0 if rows else ELEM[x.dtype], ldx, x.data_ptr() if rows else 0,
                                      a.scale.data_ptr() if rows else 0, ldx, w.data_ptr(), ldw, w_scale.data_ptr(),
                                      0 if bias is None else bias.data_ptr(), 0 if residual is None else residual.data_ptr(),
                                      0 if residual is None else residual.stride(0), out.data_ptr(), out.stride(0), ELEM[out_dtype], m, n, k, gated,
                                      ws.data_ptr() if size else 0, size, status_word(dev).data_ptr(), _raw_stream(index))
    _native.check(rc, "ogb_gemm_int8")
    launch_counts["gemm_int8"] += 1
    return out


def _channels(t, n, dev):
    return t.dtype == torch.float32 and t.dim() == 1 and t.shape[0] == n and t.is_contiguous() and t.device == dev


@functools.lru_cache(maxsize=4096)
def _workspace(m, n, k, gated, quantize):
    """Bytes, from the sizes alone."""
    return _native.load().ogb_gemm_int8_workspace(m, n, k, gated, quantize)


@_timed("block_norm")
def block_norm(x, y=None, post=None, gate=None, pre=None, eps=1e-6, x_scale=1.0, y_scale=1.0, gate_sigmoid=False, x_out=None, out=None, out_dtype=None,
               int8=False):
    """The step between two blocks of a decoder: ``x' = x_scale * x + y_scale * g * post(y)``, then ``h = pre(x')``, which is returned.

    ``x`` [rows, hidden]: the residual stream (fp32, bf16, fp16), replaced by x' unless ``x_out`` (same type) takes it.  ``y``: what the block
    wrote (None: nothing is added; the stream stays as it is unless ``x_out`` or ``x_scale`` says otherwise).  ``post`` and ``pre``: weights [hidden] of RMS norms in one
    type (None: no norm).  ``gate``: [hidden] or [rows, hidden], taken as it is or through a sigmoid.  ``h`` comes in ``out_dtype`` (that of ``out``, else of ``x``), or as
    :class:`Int8Rows` with ``int8=True``.  All of it is computed in 32 bits and rounded where it is stored; h is taken from x' before that is
    rounded.  ``hidden`` is at most 16384 on CUDA; the tensors' columns are neighbours."""
    if x.dim() != 2 or x.dtype not in ELEM:
        _refuse(f"x must be a matrix of fp32, bf16 or fp16, not {tuple(x.shape)} {x.dtype}")
    shape, dev = x.shape, x.device
    rows, n = shape
    if n == 0:
        _refuse("rows without values")
    if x.stride(1) != 1 and n > 1:
        _refuse("x: neighbouring columns")
    wide = gate is not None and gate.dim() == 2
    for t in (y, x_out, out, gate if wide else None):
        if t is not None and (t.shape != shape or t.dtype not in ELEM or t.device != dev or (t.stride(1) != 1 and n > 1)):
            _refuse("y, x_out, out and a gate for each token: matrices of x's shape and device with neighbouring columns")
    for t in (post, pre, None if wide else gate):
        if t is not None and (t.dim() != 1 or t.shape[0] != n or t.dtype not in ELEM or t.device != dev or not t.is_contiguous()):
            _refuse(f"post, pre and a gate for each channel: {n} contiguous values on x's device")
    if y is None and (post is not None or gate is not None):
        _refuse("a post norm or a gate needs y")
    if post is not None and pre is not None and post.dtype != pre.dtype:
        _refuse("post and pre weights have one type")
    if x_out is not None and x_out.dtype != x.dtype:
        _refuse("x_out has the type of x")
    for t in (x_out if x_out is not None else x, out):
        if t is not None and rows > 1 and t.stride(0) < n:
            _refuse("rows of x_out (or x, where it takes the new stream) and out do not overlap")
    if int8:
        if out is not None or out_dtype is not None:
            _refuse("8-bit rows are made by the call")
    else:
        out_dtype = out_dtype or (out.dtype if out is not None else x.dtype)
        if out_dtype not in ELEM or (out is not None and out.dtype != out_dtype):
            _refuse(f"results of {out_dtype}")
    if x_out is None and (y is not None or x_scale != 1.0):
        x_out = x
    if not x.is_cuda:
        new, h = reference.block_norm(x, y, post, gate, pre, eps, x_scale, y_scale, gate_sigmoid)
        if int8:
            codes, scale = reference.quantize_rows(h)
            q = _padded(rows, n, dev)
            q.copy_(codes)
            h = Int8Rows(q, scale)
        else:
            h = h.to(out_dtype) if out is None else out.copy_(h)
        if x_out is not None:
            x_out.copy_(new)
        return h
    if n > MAX_HIDDEN:
        _refuse(f"hidden {n}: at most {MAX_HIDDEN}")
    index = dev.index
    if index != current_index():
        with torch.cuda.device(index):
            return block_norm(x, y, post, gate, pre, eps, x_scale, y_scale, gate_sigmoid, x_out, out, None if int8 else out_dtype, int8)
    q = scale = None
    if int8:
        q, scale = _padded(rows, n, dev), torch.empty(rows, dtype=torch.float32, device=dev)
    elif out is None:
        out = torch.empty(rows, n, dtype=out_dtype, device=dev)
    weight = post if post is not None else pre
    rc = _native.load().ogb_block_norm(
        x.data_ptr(), 0 if y is None else y.data_ptr(), 0 if gate is None else gate.data_ptr(), 0 if post is None else post.data_ptr(),
        0 if pre is None else pre.data_ptr(), 0 if x_out is None else x_out.data_ptr(), 0 if out is None else out.data_ptr(),
        q.data_ptr() if int8 else 0, scale.data_ptr() if int8 else 0, x.stride(0), 0 if y is None else y.stride(0), gate.stride(0) if wide else 0,
        0 if x_out is None else x_out.stride(0), 0 if out is None else out.stride(0), q.stride(0) if int8 else 0, rows, n, ELEM[x.dtype],
        0 if y is None else ELEM[y.dtype], 0 if gate is None else ELEM[gate.dtype], 0 if weight is None else ELEM[weight.dtype],
        0 if out is None else ELEM[out_dtype], gate_sigmoid, eps, x_scale, y_scale, _raw_stream(index))
    _native.check(rc, "ogb_block_norm")
    launch_counts["block_norm"] += 1
    return Int8Rows(q, scale) if int8 else out
