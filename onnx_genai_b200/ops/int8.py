"""Products in 8-bit integers with a factor per token and per channel, and what stands between them in a decoder: rows turned into 8 bits, and
the norms around a block with its gate and residual scale, whose result is a product's left side.

:func:`gemm_int8` is the counterpart of :func:`onnx_genai_b200.ops.gemm` for weights that :func:`quantize_weight` (or
:func:`quantize_gate_up`) has made.  Weights take a byte a value; activations are quantised a token at a time when a product reads them, so
no calibration is needed.  CUDA tensors run the kernels of ``libogb_cuda.so`` on the current stream of the tensors' device; CPU tensors run
the statements of :mod:`onnx_genai_b200.ops.reference`.
"""
from __future__ import annotations

import functools
import struct
from typing import NamedTuple

import torch

from . import _native, _raw_stream, _timed, current_index, launch_counts, reference, status_ptr

ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_K = 131072          # sums of 127 * 128 * K stay below 2^31: codes of rows are -127 to 127, weights may be -128
MAX_ROWS = 1 << 30       # of rows and of channels
MAX_HIDDEN = 16384      # a row of block_norm stays in registers
_EPI = ("none", "residual", "swiglu")
# arguments of the two calls with many, as 64-bit words (ctypes takes 2 us to convert them one by one)
_pack_gemm = struct.Struct("23q").pack
_pack_norm = struct.Struct("23q3dq").pack


class Int8Rows(NamedTuple):
    """Rows in 8 bits: ``q`` [rows, k] int8, -127 to 127, whose rows begin at multiples of 16 bytes, ``scale`` [rows] fp32; a row stands for
    ``q * scale``."""
    q: torch.Tensor
    scale: torch.Tensor

    def float(self) -> torch.Tensor:
        return self.q.float() * self.scale[:, None]


def _refuse(what):
    raise ValueError(what)


def _padded(rows, k, device):
    """[rows, k] int8 whose rows begin at multiples of 16 bytes."""
    pitch = (k + 15) // 16 * 16
    if pitch == k:
        # (by its strides: torch.empty takes twice as long for two dimensions as for one)
        return torch.empty_strided((rows, k), (k, 1), dtype=torch.int8, device=device)
    return torch.empty(rows, pitch, dtype=torch.int8, device=device)[:, :k]


@_timed("quantize_rows")
def quantize_rows(x) -> Int8Rows:
    """``scale = max |x| / 127`` and ``q = round(127 x / max |x|)`` (halves to even) of every row of ``x`` [rows, k] (fp32, bf16, fp16; any
    strides).  A row of zeros has scale 0; one that holds an infinity or a NaN has scale NaN and zeros."""
    if x.dim() != 2 or x.dtype not in ELEM:
        _refuse(f"x must be a matrix of fp32, bf16 or fp16, not {tuple(x.shape)} {x.dtype}")
    rows, k = x.shape
    if not 0 < k < MAX_ROWS or rows > MAX_ROWS:
        _refuse(f"{rows} rows of {k} values: at most {MAX_ROWS}, and at least one value")
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

    ``a`` [M, K]: float rows, which the call turns into 8 bits (:func:`quantize_rows`), or :class:`Int8Rows` (codes of -127 to 127: at the largest
    K a sum of -128 times -128 would pass 32 bits).  ``w`` [N, K] int8, rows at multiples of 16 bytes; ``w_scale`` and ``bias`` [N] fp32.
    ``residual`` has the type of the result; ``out`` may be the same tensor, and shares no memory with anything else that is read.  The
    result's type is ``out_dtype``, that of ``out`` or of ``residual``, or that of float rows, else bf16.  Sums over K are exact; one rounding
    follows the factors, the bias and the residual."""
    rows = isinstance(a, Int8Rows)
    x = a.q if rows else a
    gated = epilogue == "swiglu"
    if epilogue not in _EPI:
        _refuse(f"epilogue {epilogue!r}: one of {', '.join(_EPI)}")
    shape, wshape = x.shape, w.shape
    if len(shape) != 2 or len(wshape) != 2 or shape[1] != wshape[1]:
        _refuse(f"a {tuple(shape)} and w {tuple(wshape)} do not multiply")
    m, k = shape
    n, dev, dtype = wshape[0], x.device, x.dtype
    kind = ELEM.get(dtype, 0) if rows else ELEM.get(dtype)
    if (dtype is not torch.int8) if rows else (kind is None):
        _refuse(f"rows of {dtype}")
    if not 0 < k <= MAX_K:
        _refuse(f"k = {k}: between 1 and {MAX_K}")
    if m > MAX_ROWS or n > MAX_ROWS:
        _refuse(f"{m} rows and {n} channels: at most {MAX_ROWS}")
    if w.dtype is not torch.int8 or w.device != dev:
        _refuse("w must be int8 on the device of a")
    if w_scale is None or not _channels(w_scale, n, dev) or not (bias is None or _channels(bias, n, dev)):
        _refuse(f"w_scale and bias: {n} contiguous fp32 values each on the device of a")
    n_out = n
    if gated:
        if n % 256 or residual is not None:
            _refuse("swiglu takes a weight of quantize_gate_up and no residual")
        n_out = n // 2
    elif residual is None:
        if epilogue == "residual":
            _refuse("the residual is missing")
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else residual.dtype if residual is not None else torch.bfloat16 if rows else dtype
    out_kind = ELEM.get(out_dtype)
    if out_kind is None:
        _refuse(f"results of {out_dtype}")
    if residual is not None:
        _result(residual, m, n_out, out_dtype, dev)
    if out is not None:
        _result(out, m, n_out, out_dtype, dev)
        place = _place(out)
        if _meet(*place, *_place(x)) or _meet(*place, *_place(w)):
            _refuse("out shares memory with a or w")
        for v in (w_scale, bias, a.scale if rows else None):
            if v is not None and _over(place, v):
                _refuse("out shares memory with factors or the bias")
        if residual is not None and _meet(*place, *_place(residual)) and (out.data_ptr() != residual.data_ptr() or out.stride() != residual.stride()):
            _refuse("out is the residual itself or shares no memory with it")
    if not x.is_cuda:
        y = reference.gemm_int8(a, w, w_scale, bias, residual, gated, out_dtype)
        return y if out is None else out.copy_(y)
    ldw, c1 = w.stride()
    ldx, x1 = x.stride()
    if n == 1:                     # one row has no next: any stride will do
        ldw = (k + 15) // 16 * 16
    if m == 1:
        ldx = (k + 15) // 16 * 16
    x_ptr, w_ptr = x.data_ptr(), w.data_ptr()
    if (c1 != 1 and k > 1) or ldw % 16 or w_ptr % 16 or ldw < k:
        _refuse("rows of w must begin at multiples of 16 bytes: lay it out by quantize_weight")
    if rows:
        if (x1 != 1 and k > 1) or ldx % 16 or x_ptr % 16 or ldx < k:
            _refuse("8-bit rows must begin at multiples of 16 bytes")
        if not _channels(a.scale, m, dev):
            _refuse("a.scale: a contiguous fp32 value a row on the device of a.q")
    elif x1 != 1 and k > 1:
        x = x.contiguous()
        x_ptr, ldx = x.data_ptr(), k
    index = dev.index
    if index != current_index():
        with torch.cuda.device(index):
            return gemm_int8(a, w, w_scale, bias, residual, epilogue, out, out_dtype)
    if out is None:
        out = torch.empty_strided((m, n_out), (n_out, 1), dtype=out_dtype, device=dev)
        ldc = n_out
    else:
        ldc = out.stride(0)
        if m > 1 and ldc < n_out:
            _refuse("rows of out overlap")
    if m == 0 or n == 0:
        return out
    # the caller's own memory for as long as the call: the allocator hands it on in the stream's order, and a captured graph keeps its own
    size = _workspace(m, n, k, gated, not rows)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    rc = _native.load().ogb_gemm_int8_args(_pack_gemm(
        0 if rows else x_ptr, kind, ldx, x_ptr if rows else 0, a.scale.data_ptr() if rows else 0, ldx, w_ptr, ldw, w_scale.data_ptr(),
        0 if bias is None else bias.data_ptr(), 0 if residual is None else residual.data_ptr(), 0 if residual is None else residual.stride(0),
        out.data_ptr(), ldc, out_kind, m, n, k, gated, 0 if ws is None else ws.data_ptr(), size, status_ptr(index), _raw_stream(index)))
    if rc:
        _native.check(rc, "ogb_gemm_int8")
    launch_counts["gemm_int8"] += 1
    return out


def _meet(a, rows_a, pitch_a, width_a, b, rows_b, pitch_b, width_b) -> bool:
    """Whether two matrices share memory (addresses, and pitches and widths in bytes); columns side by side in rows of one pitch do not."""
    if a > b:
        a, rows_a, pitch_a, width_a, b, rows_b, pitch_b, width_b = b, rows_b, pitch_b, width_b, a, rows_a, pitch_a, width_a
    if rows_a == 0 or rows_b == 0 or b >= a + (rows_a - 1) * pitch_a + width_a:
        return False
    if pitch_a == pitch_b > 0:
        beside = (b - a) % pitch_a
        return beside < width_a or beside + width_b > pitch_a
    return True


def _over(place, v):
    """Whether a matrix (:func:`_place`) shares memory with a contiguous vector, which may lie beside its rows."""
    return _meet(*place, v.data_ptr(), 1, place[2], v.numel() * v.element_size())


def _place(t):
    """A matrix for :func:`_meet`."""
    size, (rows, cols), (ld, step) = t.element_size(), t.shape, t.stride()
    return t.data_ptr(), rows if cols else 0, ld * size, ((cols - 1) * step + 1) * size


def _result(t, m, n, dtype, dev):
    if t.shape != (m, n) or t.dtype is not dtype or t.device != dev or (n > 1 and t.stride(1) != 1):
        _refuse(f"out and residual: [{m}, {n}] {dtype} with neighbouring columns on the device of a")


def _channels(t, n, dev):
    return t.dtype is torch.float32 and t.shape == (n,) and t.device == dev and t.is_contiguous()


@functools.lru_cache(maxsize=4096)
def _workspace(m, n, k, gated, quantize):
    """Bytes, from the sizes alone."""
    return _native.load().ogb_gemm_int8_workspace(m, n, k, gated, quantize)


@_timed("block_norm")
def block_norm(x, y=None, post=None, gate=None, pre=None, eps=1e-6, x_scale=1.0, y_scale=1.0, gate_sigmoid=False, x_out=None, out=None, out_dtype=None,
               int8=False):
    """The step between two blocks of a decoder: ``x' = x_scale * x + y_scale * g * post(y)``, then ``h = pre(x')``, which is returned.

    ``x`` [rows, hidden]: the residual stream (fp32, bf16, fp16), replaced by x' unless ``x_out`` (same type) takes it.  ``y``: what the block
    wrote (None: nothing is added; the stream stays as it is unless ``x_out`` or ``x_scale`` says otherwise).  ``post`` and ``pre``: weights
    [hidden] of RMS norms in one type (None: no norm).  ``gate``: [hidden] or [rows, hidden], taken as it is or through a sigmoid.  ``h`` comes
    in ``out_dtype`` (that of ``out``, else of ``x``), or as :class:`Int8Rows` with ``int8=True``.  ``x_out`` and ``out`` may each be a matrix
    that is read; otherwise they share memory with nothing.  All of it is computed in 32 bits and rounded where it is stored; h is taken from x'
    before that is rounded.  ``hidden`` is at most 16384 on CUDA; the tensors' columns are neighbours."""
    shape, dev, dtype = x.shape, x.device, x.dtype
    kind = ELEM.get(dtype)
    if kind is None or len(shape) != 2:
        _refuse(f"x must be a matrix of fp32, bf16 or fp16, not {tuple(shape)} {dtype}")
    rows, n = shape
    if n == 0 or rows > MAX_ROWS:
        _refuse(f"{rows} rows of {n} values: at most {MAX_ROWS}, and at least one value")
    ldx = _matrix(x, shape, dev)
    ldy = ldg = ldo = 0
    y_kind = gate_kind = w_kind = 0
    y_ptr = gate_ptr = post_ptr = pre_ptr = new_ptr = 0
    if y is not None:
        ldy, y_kind, y_ptr = _matrix(y, shape, dev), ELEM[y.dtype], y.data_ptr()
    elif post is not None or gate is not None:
        _refuse("a post norm or a gate needs y")
    if gate is not None:
        if gate.dim() == 2:
            ldg = _matrix(gate, shape, dev)
        else:
            _vector(gate, n, dev)
        gate_kind, gate_ptr = ELEM[gate.dtype], gate.data_ptr()
    if post is not None:
        _vector(post, n, dev)
        w_kind, post_ptr = ELEM[post.dtype], post.data_ptr()
    if pre is not None:
        _vector(pre, n, dev)
        if post is not None and post.dtype is not pre.dtype:
            _refuse("post and pre weights have one type")
        w_kind, pre_ptr = ELEM[pre.dtype], pre.data_ptr()
    ldn = ldx
    if x_out is not None:
        if x_out.dtype is not dtype:
            _refuse("x_out has the type of x")
        ldn = _matrix(x_out, shape, dev)
    elif y is not None or x_scale != 1.0:
        x_out = x
    if x_out is not None:
        if ldn < n and rows > 1:
            _refuse("rows of x_out (or x, where it takes the new stream) overlap")
        new_ptr = x_out.data_ptr()
    if int8:
        if out is not None or out_dtype is not None:
            _refuse("8-bit rows are made by the call")
    else:
        out_dtype = out_dtype or (out.dtype if out is not None else dtype)
        if out_dtype not in ELEM or (out is not None and out.dtype is not out_dtype):
            _refuse(f"results of {out_dtype}")
        if out is not None:
            ldo = _matrix(out, shape, dev)
            if ldo < n and rows > 1:
                _refuse("rows of out overlap")
    # a matrix that is written may stand in the place of one that is read, row for row; any other meeting would change what is still to be read
    x_ptr = x.data_ptr()
    wide = 2 if kind else 4
    reads = [(x_ptr, ldx, kind, wide)]
    if y_ptr:
        reads.append((y_ptr, ldy, y_kind, 2 if y_kind else 4))
    if ldg:
        reads.append((gate_ptr, ldg, gate_kind, 2 if gate_kind else 4))
    if new_ptr:
        _separate(new_ptr, ldn, kind, wide, reads, rows, n)
    if out is not None:
        out_kind, out_ptr = ELEM[out_dtype], out.data_ptr()
        out_wide = 2 if out_kind else 4
        _separate(out_ptr, ldo, out_kind, out_wide, reads, rows, n)
        if new_ptr and _meet(new_ptr, rows, ldn * wide, n * wide, out_ptr, rows, ldo * out_wide, n * out_wide):
            _refuse("the new stream and out share memory")
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
    if int8:
        q, scale = _padded(rows, n, dev), torch.empty(rows, dtype=torch.float32, device=dev)
        q_ptr, ldq, scale_ptr, out_ptr, out_kind = q.data_ptr(), (n + 15) // 16 * 16, scale.data_ptr(), 0, 0
    else:
        if out is None:
            out, ldo = torch.empty_strided((rows, n), (n, 1), dtype=out_dtype, device=dev), n
            out_kind, out_ptr = ELEM[out_dtype], out.data_ptr()
        q_ptr = ldq = scale_ptr = 0
    rc = _native.load().ogb_block_norm_args(_pack_norm(x_ptr, y_ptr, gate_ptr, post_ptr, pre_ptr, new_ptr, out_ptr, q_ptr, scale_ptr, ldx, ldy, ldg, ldn, ldo,
                                                       ldq, rows, n, kind, y_kind, gate_kind, w_kind, out_kind, gate_sigmoid, eps, x_scale, y_scale,
                                                       _raw_stream(index)))
    if rc:
        _native.check(rc, "ogb_block_norm")
    launch_counts["block_norm"] += 1
    return Int8Rows(q, scale) if int8 else out


def _separate(ptr, ld, kind, wide, reads, rows, n):
    end = ptr + ((rows - 1) * ld + n) * wide
    for other, ldr, other_kind, other_wide in reads:
        if other < end and ptr < other + ((rows - 1) * ldr + n) * other_wide:
            same = ptr == other and kind == other_kind and (ld == ldr or rows == 1)
            if not same and _meet(ptr, rows, ld * wide, n * wide, other, rows, ldr * other_wide, n * other_wide):
                _refuse("x_out (or x) and out: matrices that share memory with none, or the very ones that are read")


def _matrix(t, shape, dev):
    """Stride of the rows of a matrix that goes with x."""
    if t.shape == shape and t.dtype in ELEM and t.device == dev:
        ld, step = t.stride()
        if step == 1 or shape[1] == 1:
            return ld
    _refuse("x, y, x_out, out and a gate for each token: matrices of one shape, fp32, bf16 or fp16, on one device, with neighbouring columns")


def _vector(t, n, dev):
    if t.shape != (n,) or t.dtype not in ELEM or t.device != dev or not t.is_contiguous():
        _refuse(f"post, pre and a gate for each channel: {n} contiguous values on x's device")
