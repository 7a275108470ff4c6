"""The training step of a Mamba-1 block on the GPU (CUDA tensors, sm_100a).

* ``selective_scan_backward`` -- gradients of ``selective_scan``
* ``causal_conv1d_silu_backward`` -- gradients of ``causal_conv1d_silu``
* ``add_rms_norm`` / ``add_rms_norm_fp8`` / ``add_rms_norm_backward`` -- RMS
  norm with the residual's addition, its e4m3 form and its gradients
* ``grad_norm`` / ``clip_grads_`` -- global gradient norm over many tensors,
  and clipping in place

``selective_scan``, ``causal_conv1d_silu`` and ``add_rms_norm`` also
differentiate through autograd when an input requires grad.  The reference
trains through torch's own autograd (its ops register no gradient); these
kernels recompute what they need from the forward's inputs.

Activations are float32 or bfloat16; sums, states, statistics and the
gradients of per-channel parameters are fp32.  Every sum over channels, batch
or tensors is added in a fixed order, so a call's results are reproducible to
the bit.
"""

import contextlib
from array import array
from operator import attrgetter
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _ffi
from .layout import m1_layout
from .op import _CALLS, _causal_conv1d_silu, _prep, _ptr, _selective_scan

_DTYPES = {torch.float32: _ffi.DTYPE_F32, torch.bfloat16: _ffi.DTYPE_BF16}
_NO_GUARD = contextlib.nullcontext()


def _guard(dev):
    """Make ``dev`` current for the duration of a call, if it is not."""
    return _NO_GUARD if dev.index == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _stream(dev):
    """Handle of the device's current stream."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _need_cuda(what, *tensors):
    at = tensors[0].get_device()
    if at < 0 or not tensors[0].is_cuda:
        raise ValueError(f"{what} runs on CUDA tensors")
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError(f"{what}: tensors on {tensors[0].device} and {t.device}")
    return tensors[0].device


def _as(t, dtype):
    """``t`` contiguous and of ``dtype``, itself where it is."""
    if t is None or (t.dtype is dtype and t.is_contiguous()):
        return t
    return t.to(dtype).contiguous()


def _like(g, t):
    """Gradient ``g`` in the shape and type of its input ``t``."""
    if t is None or (g.dtype == t.dtype and g.shape == t.shape):
        return g if t is not None else None
    return g.reshape(t.shape).to(t.dtype)


def _new(t, dtype):
    """A contiguous tensor of t's shape."""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def _workspace(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8)


# ---------------------------------------------------------------------------
# selective scan
class SelectiveScanGrads(NamedTuple):
    """Gradients of ``selective_scan``'s inputs; None where the input was."""

    du: torch.Tensor
    ddelta: torch.Tensor
    dA: torch.Tensor
    dB: torch.Tensor
    dC: torch.Tensor
    dD: Optional[torch.Tensor]
    dz: Optional[torch.Tensor]
    ddelta_bias: Optional[torch.Tensor]
    dinitial_state: Optional[torch.Tensor]


def _scan_shape(u, delta, A, B, C, D, z, delta_bias, h0):
    """(batch, dim, len, state, groups); ``m1_layout`` where the plain
    comparisons do not settle it, for its errors."""
    shape, bc = u.shape, B.shape
    if len(shape) == 3 and A.dim() == 2 and bc == C.shape and len(bc) in (3, 4):
        batch, dim, length = shape
        state, groups, row = A.shape[1], bc[1] if len(bc) == 4 else 1, (dim,)
        if (A.shape[0] == dim and delta.shape == shape
                and bc == ((batch, groups, state, length) if len(bc) == 4 else (batch, state, length))
                and groups > 0 and dim % groups == 0 and (z is None or z.shape == shape)
                and (D is None or D.shape == row) and (delta_bias is None or delta_bias.shape == row)
                and (h0 is None or h0.shape == (batch, dim, state))):
            return batch, dim, length, state, groups
    lay = m1_layout(shape, delta.shape, A.shape, bc, C.shape,
                    *[None if t is None else t.shape for t in (D, z, delta_bias, h0)])
    return lay.batch, lay.dim, lay.length, lay.state, lay.groups


def selective_scan_backward(dout, u, delta, A, B, C, D=None, z=None, delta_bias=None,
                            delta_softplus=False, initial_state=None, dlast_state=None,
                            reverse=False):
    """Gradients of ``selective_scan`` with the same arguments.

    ``dout`` (batch, dim, len) is the gradient of its output, ``dlast_state``
    (batch, dim, state) that of its last state (None: zero).  Returns a
    ``SelectiveScanGrads``; each gradient has its input's shape and type.

    Nothing of the forward is needed but its inputs: the states are
    recomputed.  Activations (u, delta, z, B, C) that are all bfloat16 are read
    and their gradients written in 16 bits, with dout in bfloat16 or float32;
    otherwise they are converted to float32.  CUDA tensors only; any strides
    (non-contiguous tensors are copied)."""
    dev = _need_cuda("selective_scan_backward", u, dout, delta, A, B, C, D, z, delta_bias,
                     initial_state, dlast_state)
    shape = u.shape
    batch, dim, length, state, groups = _scan_shape(u, delta, A, B, C, D, z, delta_bias,
                                                    initial_state)
    if dout.shape != shape:
        raise ValueError(f"dout must be {tuple(shape)}, got {tuple(dout.shape)}")
    if dlast_state is not None and dlast_state.shape != (batch, dim, state):
        raise ValueError(f"dlast_state must be {(batch, dim, state)}, got "
                         f"{tuple(dlast_state.shape)}")
    given = (u, delta, A, B, C, D, z, delta_bias, initial_state)
    f32, bf16 = torch.float32, torch.bfloat16
    act = f32
    if u.dtype is bf16 and delta.dtype is bf16 and B.dtype is bf16 and C.dtype is bf16 and \
            (z is None or z.dtype is bf16):
        act = bf16
    do = _as(dout, bf16 if act is bf16 and dout.dtype is bf16 else f32)
    dlast = _as(dlast_state, f32)
    ins = [_as(t, want) for t, want in zip(given, (act, act, f32, act, act, f32, act, f32, f32))]
    grads = [None if t is None else torch.empty_like(t) for t in ins]
    dims = _ffi.ArmScanDims(batch, dim, length, state, groups)
    with _guard(dev):
        nbytes = _ffi.scan_backward_workspace_bytes(dims)
        ws = _workspace(nbytes, do)
        ptrs = [0 if t is None else t.data_ptr() for t in (do, *ins, dlast)]
        _ffi.scan_backward_raw(
            dims, _DTYPES[act], _DTYPES[do.dtype], ptrs[:9], delta_softplus, reverse, ptrs[9],
            ptrs[10], ws.data_ptr(), nbytes, [0 if g is None else g.data_ptr() for g in grads],
            _stream(dev))
    _CALLS["n"] += 1
    # an input that was taken as it is has its gradient's shape and type already
    return SelectiveScanGrads(*[g if i is t else _like(g, t)
                                for g, i, t in zip(grads, ins, given)])


class _Scan(torch.autograd.Function):
    """``selective_scan`` on contiguous tensors with gradients.  The forward runs
    in fp32; what is kept are its inputs as they are (bfloat16 activations)."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, h0, delta_softplus, reverse):
        given = (u, delta, A, B, C, D, z, delta_bias, h0)
        ctx.save_for_backward(*given)
        ctx.flags = (delta_softplus, reverse)
        ctx.set_materialize_grads(False)
        return _selective_scan(*[None if t is None else _prep(t, u.device) for t in given],
                               delta_softplus, reverse)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast):
        given = ctx.saved_tensors
        if dout is None:  # only the last state is used
            dout = torch.zeros_like(given[0])
        return (*selective_scan_backward(dout, *given[:8], ctx.flags[0], given[8], dlast,
                                         ctx.flags[1]), None, None)


# ---------------------------------------------------------------------------
# causal conv1d + SiLU
class _ConvSilu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(x, weight, bias)
        return _causal_conv1d_silu(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return causal_conv1d_silu_backward(dout, *ctx.saved_tensors)


def causal_conv1d_silu_backward(dout, x, weight, bias=None):
    """Gradients (dx, dweight, dbias) of ``causal_conv1d_silu``; dbias is None
    without a bias.  dout and x both bfloat16 are read (and dx written) in 16
    bits, otherwise in float32; CUDA tensors only.  Through autograd dout is
    float32, as the forward's output is: a bfloat16 x is then converted, and dx
    back."""
    if x.dim() != 3:
        raise ValueError("causal_conv1d_silu_backward takes a (batch, dim, len) CUDA tensor")
    dev = _need_cuda("causal_conv1d_silu_backward", x, dout, weight, bias)
    batch, dim, length = x.shape
    if dout.shape != x.shape:
        raise ValueError(f"dout must be {tuple(x.shape)}, got {tuple(dout.shape)}")
    if weight.shape[0] != dim or weight.numel() % dim:
        raise ValueError(f"weight must be ({dim}, kernel), got {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (dim,):
        raise ValueError(f"bias must be ({dim},), got {tuple(bias.shape)}")
    t = torch.bfloat16 if x.dtype == dout.dtype == torch.bfloat16 else torch.float32
    xs, do = _as(x, t), _as(dout, t)
    ws, bs = _as(weight, torch.float32), _as(bias, torch.float32)
    kernel = weight.numel() // dim
    dx, dw = torch.empty_like(xs), torch.empty_like(ws)
    db = None if bs is None else torch.empty_like(bs)
    with _guard(dev):
        nbytes = _ffi.conv_silu_backward_workspace_bytes(batch, dim, length, kernel)
        scratch = _workspace(nbytes, xs)
        _ffi.conv_silu_backward_raw(batch, dim, length, kernel, _DTYPES[t], do.data_ptr(),
                                    xs.data_ptr(), ws.data_ptr(), _ptr(bs), scratch.data_ptr(),
                                    nbytes, dx.data_ptr(), dw.data_ptr(), _ptr(db), _stream(dev))
    return _like(dx, x), _like(dw, weight), _like(db, bias)


# ---------------------------------------------------------------------------
# RMS norm with the residual's addition
def _rows(t, dim):
    """``t`` as rows of ``dim`` with unit element stride, and the row stride."""
    if t.is_contiguous():
        return t, dim
    t = t.reshape(-1, dim)
    if (t.stride(1) != 1 and dim > 1) or (t.shape[0] > 1 and t.stride(0) < dim):
        return t.contiguous(), dim
    return t, (t.stride(0) if t.shape[0] > 1 else dim)


def _norm_weight(weight, dim):
    if weight.shape != (dim,):
        raise ValueError(f"weight must be ({dim},), got {tuple(weight.shape)}")
    return weight if weight.dtype in _DTYPES and weight.is_contiguous() else \
        _as(weight.detach(), torch.bfloat16 if weight.dtype == torch.bfloat16 else torch.float32)


def _norm_args(what, x, weight, residual, residual_dtype):
    dev = _need_cuda(what, x, weight, residual)
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} takes float32 or bfloat16 activations, got {x.dtype}")
    if x.dim() < 1 or x.numel() == 0:
        raise ValueError(f"{what}: x has no elements")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual_dtype not in (None, residual.dtype):
            raise ValueError(f"the residual is {residual.dtype}, not {residual_dtype}")
        residual_dtype = residual.dtype
    if residual_dtype is None:
        residual_dtype = x.dtype
    if residual_dtype not in (torch.float32, x.dtype):
        raise ValueError(f"the residual stream is float32 or x's type, got {residual_dtype}")
    dim = x.shape[-1]
    rows = x.numel() // dim
    xr, x_stride = _rows(x, dim)
    rr, r_stride = _rows(residual, dim) if residual is not None else (None, dim)
    w = _norm_weight(weight, dim)
    res_out = _new(x, residual_dtype)
    head = (rows, dim, _DTYPES[x.dtype], _DTYPES[residual_dtype], _DTYPES[w.dtype],
            xr.data_ptr(), x_stride, _ptr(rr), r_stride, w.data_ptr())
    # the caller keeps xr, rr and w alive until the launch
    return dev, head, res_out, (xr, rr, w)


def _needs_grad(x, weight, residual):
    return torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                        (residual is not None and residual.requires_grad))


def _add_rms_norm(x, weight, residual, eps, residual_dtype, want_rstd):
    dev, head, res_out, held = _norm_args("add_rms_norm", x, weight, residual, residual_dtype)
    y = _new(x, x.dtype)
    rstd = x.new_empty(x.shape[:-1], dtype=torch.float32) if want_rstd else None
    with _guard(dev):
        _ffi.add_rms_norm_raw(*head, eps, y.data_ptr(), res_out.data_ptr(), _ptr(rstd), _stream(dev))
    del held
    return y, res_out, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, residual_dtype):
        y, res_out, rstd = _add_rms_norm(x, weight, residual, eps, residual_dtype, True)
        ctx.save_for_backward(res_out, weight, rstd)
        ctx.has_residual, ctx.y_dtype = residual is not None, y.dtype
        ctx.mark_non_differentiable(rstd)
        ctx.set_materialize_grads(False)
        return y, res_out, rstd

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dres_out, _):
        res_out, weight, rstd = ctx.saved_tensors
        if dy is None:  # only the residual stream is used
            dy = torch.zeros_like(res_out, dtype=ctx.y_dtype)
        dx, dres, dw = add_rms_norm_backward(dy, res_out, weight, rstd, dresidual_out=dres_out)
        return dx, dw, dres if ctx.has_residual else None, None, None


def add_rms_norm(x, weight, residual=None, eps=1e-5, residual_dtype=None, return_rstd=False):
    """RMS norm of ``residual + x`` in one pass: returns (y, residual_out) [,
    rstd], with residual_out = residual + x (x itself without a residual) and
    y = residual_out / sqrt(mean(residual_out^2) + eps) * weight over the last
    axis.

    x, residual: (..., dim) CUDA tensors, dim <= 16384, rows of any stride; y
    has x's type (float32 or bfloat16), residual_out the residual's: float32 or
    x's type (``residual_dtype`` chooses it when there is no residual).  weight
    (dim,).  The norm is taken from the fp32 sum before residual_out is
    rounded.  rstd (...) is what ``add_rms_norm_backward`` takes.  Differentiable."""
    if _needs_grad(x, weight, residual):
        y, res_out, rstd = _AddRmsNorm.apply(x, weight, residual, float(eps), residual_dtype)
    else:
        y, res_out, rstd = _add_rms_norm(x, weight, residual, float(eps), residual_dtype,
                                         return_rstd)
    return (y, res_out, rstd) if return_rstd else (y, res_out)


def _add_rms_norm_fp8(x, weight, residual, eps, residual_dtype):
    dev, head, res_out, held = _norm_args("add_rms_norm_fp8", x, weight, residual, residual_dtype)
    y8 = _new(x, torch.float8_e4m3fn)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    with _guard(dev):
        _ffi.add_rms_norm_fp8_raw(*head, eps, y8.data_ptr(), scale.data_ptr(), res_out.data_ptr(),
                                  _stream(dev))
    del held
    return y8, scale, res_out


class _AddRmsNormFp8(torch.autograd.Function):
    """No gradient exists: a backward that reaches any output raises."""

    @staticmethod
    def forward(ctx, *args):
        return _add_rms_norm_fp8(*args)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: use add_rms_norm where one is needed")


def add_rms_norm_fp8(x, weight, residual=None, eps=1e-5, residual_dtype=None):
    """``add_rms_norm`` with the output in 8 bits: returns (y8, scale,
    residual_out), y8 float8_e4m3fn (..., dim) and scale float32 (...) with
    y = y8 * scale, scale = max|y| / 448 per row, at least 2^-126 (1 for a row of
    zeros).  y8 is rounded from y times 1 / scale in fp32: within 1e-7 of the
    middle between two 8-bit values either may be written.  The row-scaled
    operand of an 8-bit projection; inference only: a backward through any
    output raises."""
    run = _AddRmsNormFp8.apply if _needs_grad(x, weight, residual) else _add_rms_norm_fp8
    return run(x, weight, residual, float(eps), residual_dtype)


def add_rms_norm_backward(dy, residual_out, weight, rstd, dresidual_out=None):
    """Gradients (dx, dresidual, dweight) of ``add_rms_norm`` from its
    residual_out and rstd.  ``dresidual_out``: the gradient that reaches
    residual_out past the norm (None: zero).  dx has dy's type, dresidual
    residual_out's; they hold the same values and are one tensor when the
    types agree."""
    dev = _need_cuda("add_rms_norm_backward", dy, residual_out, weight, rstd, dresidual_out)
    if dy.dtype not in _DTYPES or residual_out.dtype not in (torch.float32, dy.dtype):
        raise ValueError("add_rms_norm_backward takes float32 or bfloat16 dy and a residual_out of "
                         f"float32 or dy's type, got {dy.dtype} and {residual_out.dtype}")
    if residual_out.shape != dy.shape or dy.numel() == 0:
        raise ValueError(f"dy {tuple(dy.shape)} and residual_out {tuple(residual_out.shape)} must be "
                         "of one shape, with elements")
    dim = dy.shape[-1]
    rows = dy.numel() // dim
    if rstd.numel() != rows:
        raise ValueError(f"rstd must hold {rows} values, got {tuple(rstd.shape)}")
    w = _norm_weight(weight, dim)
    dyc, res, rs = dy.contiguous(), residual_out.contiguous(), _as(rstd, torch.float32)
    dro = None
    if dresidual_out is not None:
        if dresidual_out.shape != dy.shape:
            raise ValueError(f"dresidual_out must be {tuple(dy.shape)}, got "
                             f"{tuple(dresidual_out.shape)}")
        dro = _as(dresidual_out, res.dtype)
    dx = torch.empty_like(dyc)
    same = dyc.dtype == res.dtype
    dres = dx if same else torch.empty_like(res)
    dw = dyc.new_empty(dim, dtype=torch.float32)
    with _guard(dev):
        nbytes = _ffi.add_rms_norm_backward_workspace_bytes(rows, dim)
        scratch = _workspace(nbytes, dyc)
        _ffi.add_rms_norm_backward_raw(
            rows, dim, _DTYPES[dyc.dtype], _DTYPES[res.dtype], _DTYPES[w.dtype], dyc.data_ptr(),
            res.data_ptr(), w.data_ptr(), rs.data_ptr(), _ptr(dro), scratch.data_ptr(), nbytes,
            dx.data_ptr(), 0 if same else dres.data_ptr(), dw.data_ptr(), _stream(dev))
    return dx, dres, _like(dw, weight)


# ---------------------------------------------------------------------------
# global gradient norm and clipping
def _dense(t):
    """Whether t's elements fill one block of memory without gaps or overlap."""
    need = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride != need:
            return False
        need *= size
    return True


def _clip(what, grads, max_norm, eps, scale):
    grads = [g for g in ([grads] if isinstance(grads, torch.Tensor) else grads) if g is not None]
    if not grads:
        raise ValueError(f"{what}: no gradients")
    # one C-level pass per attribute: a model has hundreds of gradients
    devices, dtypes = set(map(torch.Tensor.get_device, grads)), list(map(attrgetter("dtype"), grads))
    dev = grads[0].device
    if len(devices) > 1 or dev.type != "cuda":
        raise ValueError(f"{what} runs on CUDA tensors of one device, got "
                         f"{sorted({str(g.device) for g in grads})}")
    kinds = set(dtypes)
    other = kinds - _DTYPES.keys()
    if other:
        raise ValueError(f"{what} takes float32 and bfloat16 gradients, got {other.pop()}")
    if not all(map(torch.Tensor.is_contiguous, grads)):
        for g in grads:
            if not (g.is_contiguous() or _dense(g)):
                raise ValueError(f"{what}: a gradient of shape {tuple(g.shape)} and strides "
                                 f"{g.stride()} does not fill its memory")
    # most lists hold one type: looking each up took 2 us of 32 tensors' call
    codes = (array("i", (_DTYPES[dtypes[0]],)) * len(grads) if len(kinds) == 1
             else array("i", map(_DTYPES.__getitem__, dtypes)))
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with _guard(dev):
        nbytes = _ffi.clip_grads_workspace_bytes()
        ws = _workspace(nbytes, norm)
        _ffi.clip_grads_raw(array("Q", map(torch.Tensor.data_ptr, grads)),
                            array("Q", map(torch.Tensor.numel, grads)), codes, max_norm, eps, scale,
                            ws.data_ptr(), nbytes, norm.data_ptr(), _stream(dev))
    if scale:  # autograd notices tensors that it kept, as with torch's in-place operations
        torch.autograd.graph.increment_version(grads)
    return norm


def grad_norm(grads):
    """The 2-norm of all gradients together, a 0-d float32 CUDA tensor (no
    host synchronization).  ``grads``: CUDA tensors of one device, float32 or
    bfloat16, mixed at will; None entries are skipped."""
    return _clip("grad_norm", grads, 0.0, 0.0, False)


def clip_grads_(grads, max_norm, eps=1e-6):
    """Scale every gradient in place by min(1, max_norm / (norm + eps)), norm
    being ``grad_norm(grads)`` before the call, which is returned.  The rule of
    ``torch.nn.utils.clip_grad_norm_`` on the gradients themselves: a factor of
    1 leaves every bit as it was, a NaN norm makes every gradient NaN.  Autograd
    counts it as an in-place change."""
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return _clip("clip_grads_", grads, max_norm, eps, True)
