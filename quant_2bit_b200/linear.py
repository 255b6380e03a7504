"""Linear layers over the quantizers' weights: products grouped by expert, and
8-bit floating point with a scale for each block of 128.

The reference's QuantizedLinear multiplies its quantized weight with torch
(src/qat/quantized_linear.py:309-315).  Here one launch serves all experts of a layer
(``quant.bcjr_quantize_layer`` quantizes them in one launch too), and layers
that are not being trained -- the teacher, the frozen layers around the one in
training -- can hold their weights in e4m3 and still pass gradients on.

* ``grouped_linear(x, weight, offsets)``: rows sorted by expert, bf16 or fp16,
  differentiable in ``x`` and ``weight``.
* ``fp8_quantize_rows`` / ``fp8_quantize_weight``: e4m3 with one fp32 scale for
  each 1 x 128 row segment / 128 x 128 block: with amax = max(max |x|, 2^-100)
  over the block, scale = amax * (1/448) and q = e4m3(x * (448 * (1/amax))), in fp32.
* ``fp8_matmul``: the product of two such operands, summed in fp32.
* ``fp8_linear(x, q, scale)``: quantizes the rows of ``x`` and multiplies;
  differentiable in ``x`` (straight through the rounding; the upstream gradient
  is quantized by rows in the same way).

Every op runs the sm_100a kernels of libbcjr_b200.so on the caller's current
stream, reads ``offsets`` on the device only, and never synchronises.  There is
no CPU path: CPU tensors raise RuntimeError, wrong shapes AssertionError, wrong
types ValueError.  Feature counts are multiples of 16 (the quantizers' tile).
There is no second and no forward-mode derivative: asking for one raises
RuntimeError (NotImplementedError for a dual tensor).
All of it can be captured into CUDA graphs, backward passes included; as for
any torch op, no eager graph of the same leaves may be alive during the capture
(torch then makes the capturing stream wait for the leaf's own and raises).
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_BLOCK = 128
_TILE = 16
_MAX_GROUPS = 1024
_MAX_STEP = 1 << 32        # elements between rows
_RAW_ROWS = 32             # up to here the 8-bit layer needs no workspace
_F8 = torch.float8_e4m3fn
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_HALVES = (torch.bfloat16, torch.float16)


# Calls with few rows take less time on the GPU than in here, so the checks of
# the usual case are few and their messages are made only when one fails.


def _need_cuda(names, *tensors):
    """All tensors on one GPU (None is skipped); returns its index."""
    device = -1
    for i, t in enumerate(tensors):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError(f"quant_2bit_b200: `{names.split()[i]}` must be a CUDA tensor (the B200 "
                               "kernels have no CPU fallback)")
        d = t.get_device()
        if device < 0:
            device = d
        elif d != device:
            raise AssertionError(f"`{names.split()[i]}` is on cuda:{d}, not on cuda:{device}")
    return device


def _need_dtype(t, name, allowed):
    if t.dtype not in allowed:
        raise ValueError(f"`{name}` must be {' or '.join(str(d) for d in allowed)}, got {t.dtype}")


def _need_features(n, name):
    assert n >= _TILE and n % _TILE == 0, f"{name} must be a multiple of {_TILE}, got {n}"


def _call(fn, device, *args):
    """One C call on `device`'s current stream (appended to the arguments)."""
    stream = torch._C._cuda_getCurrentRawStream(device)
    if torch._C._cuda_getDevice() == device:
        st = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            st = fn(*args, stream)
    if st:
        _lib.check(st, fn.__name__)


def _differentiate(backward, ctx, dy):
    """A backward without a second derivative (asking for one raises); the
    bookkeeping for that is left out when no graph of the backward is made."""
    if torch.is_grad_enabled():
        backward = once_differentiable(backward)
    return backward(ctx, dy)


def _forward_mode():
    """Inside torch.autograd.forward_ad.dual_level: an operand with a tangent does
    not require a gradient, and the autograd Function has to refuse it."""
    return forward_ad._current_level >= 0


def _need_constant(names, *tensors):
    """No derivative is asked for that the operator would lose."""
    for i, t in enumerate(tensors):
        assert not (t.requires_grad and torch.is_grad_enabled()), f"`{names.split()[i]}` has no gradient here"
        assert not _forward_mode() or forward_ad.unpack_dual(t).tangent is None, \
            f"`{names.split()[i]}` has no forward-mode derivative here"


def _blocks(n):
    return -(-n // _BLOCK)


def _rows(t):
    """(tensor, elements between rows) of a 2-D matrix as the kernels read it: the
    matrix itself when its rows are contiguous, start on 16 bytes and lie no
    further apart than the C entry points accept, else a contiguous copy."""
    n = t.size(1)
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t, n
        step = t.stride(0)
        if t.stride(1) == 1 and n <= step <= _MAX_STEP and step * t.element_size() % 16 == 0:
            return t, step
    return _dense(t), n


def _dense(t):
    """Contiguous and 16-byte aligned."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _need_offsets(offsets, groups):
    """Checked and contiguous."""
    if offsets is None:
        return None
    _need_dtype(offsets, "offsets", (torch.int32, torch.int64))
    assert offsets.dim() == 1 and offsets.shape[0] == groups + 1, \
        f"offsets must have one more element than there are experts ({groups}), got {tuple(offsets.shape)}"
    return offsets if offsets.is_contiguous() else offsets.contiguous()


def _bounds(offsets):
    """(pointer, bytes of an element)"""
    return (0, 0) if offsets is None else (offsets.data_ptr(), offsets.element_size())


# --------------------------------------------------------------------------
# bf16 / fp16, grouped by expert


def _grouped_forward(x, weight, offsets):
    E, N, K = weight.shape
    T = x.size(0)
    y = x.new_empty(T, N)
    if T == 0:
        return y
    x, ld = _rows(x)
    weight = _dense(weight)
    off_ptr, off_size = _bounds(offsets)
    _call(_lib.load().bcjr_grouped_mm, x.get_device(), x.data_ptr(), ld, weight.data_ptr(), off_ptr,
          off_size, T, E, N, K, _DTYPES[x.dtype], y.data_ptr(), None)
    return y


def _grouped_backward(ctx, dy):
    x, weight, offsets = ctx.saved_tensors
    need_x, need_w, _ = ctx.needs_input_grad
    E, N, K = ctx.sizes
    T = dy.shape[0]
    dy, ld_dy = _rows(dy if dy.dtype == ctx.dtype else dy.to(ctx.dtype))
    dx = dw = x_ptr = weight_ptr = dx_ptr = dw_ptr = None
    ld_x = 0
    if need_x:
        weight = _dense(weight)
        dx = dy.new_empty(T, K)
        weight_ptr, dx_ptr = weight.data_ptr(), dx.data_ptr()
    if need_w:
        x, ld_x = _rows(x)
        dw = dy.new_empty(E, N, K)
        x_ptr, dw_ptr = x.data_ptr(), dw.data_ptr()
    off_ptr, off_size = _bounds(offsets)
    _call(_lib.load().bcjr_grouped_backward, dy.get_device(), dy.data_ptr(), ld_dy, x_ptr, ld_x, weight_ptr,
          off_ptr, off_size, T, E, N, K, _DTYPES[ctx.dtype], dx_ptr, dw_ptr, None)
    return dx, dw, None


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        # each gradient reads the other operand only: what no gradient reads is
        # not kept alive, and may change before the backward pass
        need_x, need_w, _ = ctx.needs_input_grad
        ctx.save_for_backward(x if need_w else None, weight if need_x else None, offsets)
        ctx.sizes, ctx.dtype = weight.shape, x.dtype
        return _grouped_forward(x, weight, offsets)

    @staticmethod
    def backward(ctx, dy):
        return _differentiate(_grouped_backward, ctx, dy)


def grouped_linear(x, weight, offsets):
    """y[t] = weight[e] @ x[t] for every row t of group e, offsets[e] <= t <
    offsets[e + 1].

    x        (T, K) bf16 or fp16, rows sorted by expert; any row stride
    weight   (E, N, K), x's dtype (``quant.bcjr_quantize_layer`` returns fp32:
             stack and cast, as QuantizedLinear casts to its input's type)
    offsets  (E + 1,) int32 or int64 on x's device, not decreasing, within
             [0, T]; it is not read on the host, and the kernels clamp it

    Returns (T, N).  Groups may be empty; rows before offsets[0] and from
    offsets[E] on belong to no group: their output and gradient are zero.
    Sums are fp32, rounded once; results do not change from run to run."""
    _need_cuda("x weight offsets", x, weight, offsets)
    _need_dtype(x, "x", _HALVES)
    if weight.dtype != x.dtype:
        _need_dtype(weight, "weight", (x.dtype,))
    assert x.dim() == 2 and weight.dim() == 3 and x.size(1) == weight.size(2), \
        f"x must be (T, K) and weight (E, N, K), got {tuple(x.shape)} and {tuple(weight.shape)}"
    E, N, K = weight.shape
    assert 1 <= E <= _MAX_GROUPS, f"1 to {_MAX_GROUPS} experts, got {E}"
    _need_features(N, "out features")
    _need_features(K, "in features")
    offsets = _need_offsets(offsets, E)
    if (x.requires_grad or weight.requires_grad) and torch.is_grad_enabled() or _forward_mode():
        return _GroupedLinear.apply(x, weight, offsets)
    return _grouped_forward(x, weight, offsets)


# --------------------------------------------------------------------------
# e4m3 with block scales


def fp8_quantize_rows(x):
    """(q, scale) of (..., K) bf16, fp16 or fp32: q e4m3 of x's shape, scale fp32
    (..., ceil(K / 128)); q times its segment's scale stands for x.  Not
    differentiable (``fp8_linear`` is)."""
    _need_cuda("x", x)
    code = _DTYPES.get(x.dtype)
    if code is None:
        _need_dtype(x, "x", tuple(_DTYPES))
    assert x.dim() >= 1, "x must have at least one axis"
    K = x.size(-1)
    _need_features(K, "the last axis")
    blocks = _blocks(K)
    rows = x if x.dim() == 2 else x.detach().reshape(-1, K)
    T = rows.size(0)
    q = x.new_empty(T, K, dtype=_F8)
    scale = x.new_empty(T, blocks, dtype=torch.float32)
    if T:
        rows, ld = _rows(rows)
        _call(_lib.load().bcjr_fp8_quantize_rows, x.get_device(), rows.data_ptr(), ld, T, K, code,
              q.data_ptr(), scale.data_ptr(), blocks, 1)
    if x.dim() == 2:
        return q, scale
    return q.view(x.shape), scale.view(*x.shape[:-1], blocks)


def fp8_quantize_weight(weight):
    """(q, scale) of a weight (N, K), or of E weights (E, N, K), bf16, fp16 or
    fp32: q e4m3 of its shape, scale fp32 ([E,] ceil(N / 128), ceil(K / 128)),
    one for each 128 x 128 block.  Not differentiable."""
    _need_cuda("weight", weight)
    code = _DTYPES.get(weight.dtype)
    if code is None:
        _need_dtype(weight, "weight", tuple(_DTYPES))
    assert weight.dim() in (2, 3), f"weight must be (N, K) or (E, N, K), got {tuple(weight.shape)}"
    *lead, N, K = weight.shape
    assert N >= 1, "weight must have rows"
    _need_features(K, "in features")
    w = _dense(weight)
    q = weight.new_empty(*lead, N, K, dtype=_F8)
    scale = weight.new_empty(*lead, _blocks(N), _blocks(K), dtype=torch.float32)
    _call(_lib.load().bcjr_fp8_quantize_blocks, weight.get_device(), w.data_ptr(),
          lead[0] if lead else 1, N, K, code, q.data_ptr(), scale.data_ptr())
    return q, scale


def _need_fp8_weight(q, scale, offsets):
    """(E, N, K, offsets) of a weight in blocks, checked."""
    if q.dtype != _F8:
        _need_dtype(q, "q", (_F8,))
    if scale.dtype != torch.float32:
        _need_dtype(scale, "scale", (torch.float32,))
    assert q.dim() == (2 if offsets is None else 3), \
        f"q must be (N, K), or (E, N, K) with offsets, got {tuple(q.shape)}"
    *lead, N, K = q.shape
    E = lead[0] if lead else 1
    assert 1 <= E <= _MAX_GROUPS, f"1 to {_MAX_GROUPS} experts, got {E}"
    _need_features(N, "out features")
    _need_features(K, "in features")
    assert scale.shape == (*lead, _blocks(N), _blocks(K)), \
        f"scale must be {(*lead, _blocks(N), _blocks(K))}, got {tuple(scale.shape)}"
    assert not scale.requires_grad, "the scales of an e4m3 weight have no gradient"
    return E, N, K, _need_offsets(offsets, E)


def fp8_matmul(xq, x_scale, q, scale, offsets=None, out_dtype=torch.bfloat16):
    """Rows times a weight, both in e4m3: sum over blocks j of 128 of
    x_scale[t, j] * scale[n // 128, j] * (xq[t, block j] . q[n, block j]).

    xq, x_scale  (T, K) and (T, ceil(K / 128)), as ``fp8_quantize_rows`` returns
    q, scale     (N, K) and its block scales, as ``fp8_quantize_weight`` returns;
                 with ``offsets`` (see ``grouped_linear``) (E, N, K) and theirs
    Returns (T, N) in ``out_dtype`` (bf16 or fp16).  Any fp32 scales are
    accepted; the product of two scales is formed in fp32, so it should not
    underflow.  Not differentiable (``fp8_linear`` is): rows and scales that
    require a gradient are refused, and the weight is constant."""
    _need_cuda("xq x_scale q scale offsets", xq, x_scale, q, scale, offsets)
    _need_dtype(xq, "xq", (_F8,))
    _need_dtype(x_scale, "x_scale", (torch.float32,))
    if out_dtype not in _HALVES:
        raise ValueError(f"out_dtype must be torch.bfloat16 or torch.float16, got {out_dtype}")
    E, N, K, offsets = _need_fp8_weight(q, scale, offsets)
    assert xq.dim() == 2 and xq.shape[1] == K, f"xq must be (T, {K}), got {tuple(xq.shape)}"
    assert x_scale.shape == (xq.shape[0], _blocks(K)), \
        f"x_scale must be {(xq.shape[0], _blocks(K))}, got {tuple(x_scale.shape)}"
    _need_constant("xq x_scale scale", xq, x_scale, scale)
    T = xq.shape[0]
    if T == 0:
        return torch.empty((0, N), dtype=out_dtype, device=xq.device)
    xq, ld = _rows(xq)
    q, scale = _dense(q), _dense(scale)
    out = xq.new_empty(T, N, dtype=out_dtype)
    off_ptr, off_size = _bounds(offsets)
    _call(_lib.load().bcjr_fp8_mm, xq.get_device(), xq.data_ptr(), ld, x_scale.data_ptr(),
          x_scale.stride(0), x_scale.stride(1), q.data_ptr(), scale.data_ptr(), off_ptr, off_size,
          T, E, N, K, False, out.data_ptr(), _DTYPES[out_dtype], None)
    return out


def _quantized_product(x, q, scale, offsets, transpose):
    """x's rows, quantized, times the e4m3 weight (or its transpose)."""
    T, C = x.shape
    *lead, N, K = q.shape
    E = lead[0] if lead else 1
    out = x.new_empty(T, K if transpose else N)
    if T == 0:
        return out
    size, ws = 0, None
    if T > _RAW_ROWS:
        size = T * (C + 4 * _blocks(C)) + 16      # bcjr_fp8_linear_workspace_bytes
        ws = x.new_empty(size, dtype=torch.uint8)
    x, ld = _rows(x)
    q, scale = _dense(q), _dense(scale)
    off_ptr, off_size = _bounds(offsets)
    _call(_lib.load().bcjr_fp8_linear, x.get_device(), x.data_ptr(), ld, _DTYPES[x.dtype], q.data_ptr(),
          scale.data_ptr(), off_ptr, off_size, T, E, N, K, transpose, out.data_ptr(),
          None if ws is None else ws.data_ptr(), size, None)
    return out


def _fp8_backward(ctx, dy):
    q, scale, offsets = ctx.saved_tensors
    dx = _quantized_product(dy, q, scale, offsets, True) if ctx.needs_input_grad[0] else None
    return dx, None, None, None


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, q, scale, offsets):
        ctx.save_for_backward(q, scale, offsets)
        return _quantized_product(x, q, scale, offsets, False)

    @staticmethod
    def backward(ctx, dy):
        return _differentiate(_fp8_backward, ctx, dy)


def fp8_linear(x, q, scale, offsets=None):
    """x times an e4m3 weight: x's rows are quantized in segments of 128
    (``fp8_quantize_rows``) and multiplied (``fp8_matmul``).

    x         (..., K) bf16 or fp16; with ``offsets`` (T, K), rows sorted by expert
    q, scale  (N, K) and its block scales, as ``fp8_quantize_weight`` returns;
              with ``offsets`` (E, N, K) and theirs
    Returns (..., N) in x's dtype.  Differentiable in x: the gradient of the
    product with the stored weight, with the upstream gradient quantized in
    row segments of 128; the rounding of x counts as the identity.  The weight
    is constant."""
    _need_cuda("x q scale offsets", x, q, scale, offsets)
    _need_dtype(x, "x", _HALVES)
    E, N, K, offsets = _need_fp8_weight(q, scale, offsets)
    dims = x.dim()
    assert dims >= 1 and x.size(-1) == K, f"x must be (..., {K}), got {tuple(x.shape)}"
    assert offsets is None or dims == 2, f"x must be (T, K) with offsets, got {tuple(x.shape)}"
    rows = x if dims == 2 else x.reshape(-1, K)
    if x.requires_grad and torch.is_grad_enabled() or _forward_mode():
        y = _Fp8Linear.apply(rows, q, scale, offsets)
    else:
        y = _quantized_product(rows, q, scale, offsets, False)
    return y if dims == 2 else y.view(*x.shape[:-1], N)


__all__ = ["grouped_linear", "fp8_quantize_rows", "fp8_quantize_weight", "fp8_matmul", "fp8_linear"]
