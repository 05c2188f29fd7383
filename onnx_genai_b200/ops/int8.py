"""Products in 8-bit integers with a factor per token and per channel, and what stands between them in a decoder: rows turned into 8 bits, and
the norms around a block with its gate and residual scale, whose result is a product's left side.

:func:`gemm_int8` is the counterpart of :func:`onnx_genai_b200.ops.gemm` for weights that :func:`quantize_weight` (or
:func:`quantize_gate_up`) has made.  Weights take a byte a value; activations are quantised a token at a time when a product reads them, so
no calibration is needed.  CUDA tensors run the kernels of ``libogb_cuda.so`` on the current stream of the tensors' device; CPU tensors run
the statements of :mod:`onnx_genai_b200.ops.reference`.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native, _timed, launch_counts, reference, status_word

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


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _float_rows(t, name):
    _need(t.dim() == 2 and t.dtype in ELEM, f"{name} must be a matrix of fp32, bf16 or fp16, not {tuple(t.shape)} {t.dtype}")
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _padded(rows, k, device, alloc=torch.empty):
    return alloc(rows, (k + 15) // 16 * 16, dtype=torch.int8, device=device)[:, :k]


class _on:
    """Launches go to the tensors' device, whichever is current."""
    __slots__ = ("guard",)

    def __init__(self, device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


@_timed("quantize_rows")
def quantize_rows(x) -> Int8Rows:
    """``scale = max |x| / 127`` and ``q = round(127 x / max |x|)`` (halves to even) of every row of ``x`` [rows, k] (fp32, bf16, fp16; any
    row stride).  A row of zeros has scale 0; one that holds an infinity or a NaN has scale NaN and zeros."""
    x = _float_rows(x, "x")
    rows, k = x.shape
    _need(k > 0, "rows without values have no scale")
    q = _padded(rows, k, x.device)
    if not x.is_cuda:
        codes, scale = reference.quantize_rows(x)
        q.copy_(codes)
        return Int8Rows(q, scale)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    with _on(x.device) as stream:
        rc = _native.load().ogb_quantize_rows(x.data_ptr(), q.data_ptr(), scale.data_ptr(), rows, k, x.stride(0), q.stride(0), ELEM[x.dtype], stream)
    _native.check(rc, "ogb_quantize_rows")
    launch_counts["quantize_rows"] += 1
    return Int8Rows(q, scale)


def quantize_weight(w) -> Int8Rows:
    """A weight [n, k] in 8 bits with a factor per output channel, laid out for :func:`gemm_int8`.  Weights have to be finite."""
    _need(bool(torch.isfinite(w).all()), "a weight that is not finite cannot be held in 8 bits")
    return quantize_rows(w)


def quantize_gate_up(gate, up) -> Int8Rows:
    """Gate and up projections [inter, k] as one weight for ``epilogue="swiglu"``: blocks of 128 gate rows and their 128 up rows, ``inter``
    padded with zero rows to a multiple of 128 (the padded columns of the result are zero: pad the next weight's k with anything)."""
    _need(gate.shape == up.shape and gate.dim() == 2, "gate and up projections have one shape")
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
    _need(epilogue in _EPI, f"epilogue {epilogue!r}: one of {', '.join(_EPI)}")
    rows = isinstance(a, Int8Rows)
    x = a.q if rows else a
    gated = epilogue == "swiglu"
    _need(x.dim() == 2 and w.dim() == 2 and x.shape[1] == w.shape[1], f"a {tuple(x.shape)} and w {tuple(w.shape)} do not multiply")
    _need((x.dtype == torch.int8) if rows else x.dtype in ELEM, f"rows of {x.dtype}")
    m, k = x.shape
    n = w.shape[0]
    _need(0 < k <= MAX_K, f"k = {k}: between 1 and {MAX_K}")
    _need(w.dtype == torch.int8 and w.device == x.device, "w must be int8 on the device of a")
    for t, name in ((w_scale, "w_scale"), (bias, "bias")):
        _need(t is None or (t.dtype == torch.float32 and t.shape == (n,) and t.is_contiguous() and t.device == x.device),
              f"{name}: {n} contiguous fp32 values on the device of a")
    _need(w_scale is not None, "w_scale is needed")
    _need(not gated or (n % 256 == 0 and residual is None), "swiglu takes a weight of quantize_gate_up and no residual")
    _need(epilogue != "residual" or residual is not None, "the residual is missing")
    n_out = n // 2 if gated else n
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else residual.dtype if residual is not None else torch.bfloat16 if rows else x.dtype
    _need(out_dtype in ELEM, f"results of {out_dtype}")
    for t, name in ((out, "out"), (residual, "residual")):
        _need(t is None or (t.shape == (m, n_out) and t.dtype == out_dtype and t.device == x.device and (n_out <= 1 or t.stride(1) == 1)),
              f"{name}: [{m}, {n_out}] {out_dtype} with neighbouring columns on the device of a")
    if not x.is_cuda:
        y = reference.gemm_int8(a, w, w_scale, bias, residual, gated, out_dtype)
        return y if out is None else out.copy_(y)
    _need(w.stride(1) == 1 and w.stride(0) % 16 == 0 and w.data_ptr() % 16 == 0, "rows of w must begin at multiples of 16 bytes: lay it out by quantize_weight")
    if rows:
        _need(x.stride(1) == 1 and x.stride(0) % 16 == 0 and x.data_ptr() % 16 == 0, "8-bit rows must begin at multiples of 16 bytes")
        _need(a.scale.dtype == torch.float32 and a.scale.shape == (m,) and a.scale.is_contiguous() and a.scale.device == x.device, "a.scale: a contiguous fp32 value a row")
    elif k > 1 and x.stride(1) != 1:
        x = x.contiguous()
    if out is None:
        out = torch.empty(m, n_out, dtype=out_dtype, device=x.device)
    if m == 0 or n == 0:
        return out
    lib = _native.load()
    with _on(x.device) as stream:
        # the caller's own memory for as long as the call: the allocator hands it on in the stream's order, and a captured graph keeps its own
        size = lib.ogb_gemm_int8_workspace(m, n, k, gated, not rows)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        rc = lib.ogb_gemm_int8(0 if rows else x.data_ptr(), 0 if rows else ELEM[x.dtype], x.stride(0), x.data_ptr() if rows else 0,
                               a.scale.data_ptr() if rows else 0, x.stride(0) if rows else 0, w.data_ptr(), w.stride(0), w_scale.data_ptr(),
                               bias.data_ptr() if bias is not None else 0, residual.data_ptr() if residual is not None else 0,
                               residual.stride(0) if residual is not None else 0, out.data_ptr(), out.stride(0), ELEM[out_dtype], m, n, k, gated,
                               ws.data_ptr() if size else 0, size, status_word(x.device).data_ptr(), stream)
    _native.check(rc, "ogb_gemm_int8")
    launch_counts["gemm_int8"] += 1
    return out


@_timed("block_norm")
def block_norm(x, y=None, post=None, gate=None, pre=None, eps=1e-6, x_scale=1.0, y_scale=1.0, gate_sigmoid=False, x_out=None, out=None, out_dtype=None,
               int8=False):
    """The step between two blocks of a decoder: ``x' = x_scale * x + y_scale * g * post(y)``, then ``h = pre(x')``, which is returned.

    ``x`` [rows, hidden]: the residual stream (fp32, bf16, fp16), replaced by x' unless ``x_out`` (same type) takes it.  ``y``: what the block
    wrote (None: nothing is added; the stream stays as it is unless ``x_out`` or ``x_scale`` says otherwise).  ``post`` and ``pre``: weights [hidden] of RMS norms in one
    type (None: no norm).  ``gate``: [hidden] or [rows, hidden], taken as it is or through a sigmoid.  ``h`` comes in ``out_dtype`` (that of ``out``, else of ``x``), or as
    :class:`Int8Rows` with ``int8=True``.  All of it is computed in 32 bits and rounded where it is stored; h is taken from x' before that is
    rounded.  ``hidden`` is at most 16384 on CUDA; the tensors' columns are neighbours."""
    _need(x.dim() == 2 and x.dtype in ELEM, f"x must be a matrix of fp32, bf16 or fp16, not {tuple(x.shape)} {x.dtype}")
    rows, n = x.shape
    _need(n > 0, "rows without values")
    dev = x.device
    for t, name in ((y, "y"), (x_out, "x_out"), (out, "out"), (gate if gate is not None and gate.dim() == 2 else None, "gate")):
        _need(t is None or (t.shape == x.shape and t.dtype in ELEM and t.device == dev and (n == 1 or t.stride(1) == 1)),
              f"{name}: a matrix of x's shape and device with neighbouring columns")
    _need(n == 1 or x.stride(1) == 1, "x: neighbouring columns")
    vectors = [(post, "post"), (pre, "pre"), (gate if gate is not None and gate.dim() != 2 else None, "gate")]
    for t, name in vectors:
        _need(t is None or (t.shape == (n,) and t.dtype in ELEM and t.device == dev and t.is_contiguous()), f"{name}: {n} contiguous values on x's device")
    _need(y is not None or (post is None and gate is None), "a post norm or a gate needs y")
    _need(post is None or pre is None or post.dtype == pre.dtype, "post and pre weights have one type")
    _need(x_out is None or x_out.dtype == x.dtype, "x_out has the type of x")
    _need(not int8 or (out is None and out_dtype is None), "8-bit rows are made by the call")
    if x_out is None and (y is not None or x_scale != 1.0):
        x_out = x
    if not int8:
        out_dtype = out_dtype or (out.dtype if out is not None else x.dtype)
        _need(out_dtype in ELEM and (out is None or out.dtype == out_dtype), f"results of {out_dtype}")
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
    _need(n <= MAX_HIDDEN, f"hidden {n}: at most {MAX_HIDDEN}")
    if int8:
        q, scale = _padded(rows, n, dev), torch.empty(rows, dtype=torch.float32, device=dev)
    elif out is None:
        out = torch.empty(rows, n, dtype=out_dtype, device=dev)
    ptr = lambda t: 0 if t is None else t.data_ptr()                      # noqa: E731
    ld = lambda t: 0 if t is None or t.dim() != 2 else t.stride(0)        # noqa: E731
    kind = lambda t: 0 if t is None else ELEM[t.dtype]                    # noqa: E731
    with _on(dev) as stream:
        rc = _native.load().ogb_block_norm(
            x.data_ptr(), ptr(y), ptr(gate), ptr(post), ptr(pre), ptr(x_out), ptr(out), q.data_ptr() if int8 else 0, scale.data_ptr() if int8 else 0,
            x.stride(0), ld(y), ld(gate), ld(x_out), ld(out), q.stride(0) if int8 else 0, rows, n, ELEM[x.dtype], kind(y), kind(gate),
            kind(post if post is not None else pre), kind(out), int(gate_sigmoid), eps, x_scale, y_scale, stream)
    _native.check(rc, "ogb_block_norm")
    launch_counts["block_norm"] += 1
    return Int8Rows(q, scale) if int8 else out
