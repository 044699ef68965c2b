"""Root-mean-square norms on either side of a recurrent layer.

``launch_add_norm``    r = x + residual; y = r / sqrt(mean(r^2) + eps) * weight, before a layer's projections
``launch_gated_norm``  y = x / sqrt(mean(x^2) + eps) * weight * silu(z) over each head of a recurrence's output
                       (``launch_gdn(..., out_norm=...)`` applies it to its own output)

Both write the inputs' type, or e4m3 codes with fp32 scales for an 8-bit
product: scale = max(amax |y|, 1e-12) / 448 per row or per 128 channels
(``launch_add_norm``) or per head (``launch_gated_norm``), code = e4m3(y /
scale), saturating.  The backward passes and the differentiable ``add_norm``
and ``gated_norm`` are for training.  Inputs are bf16, fp16 or fp32, all of
one type, the weight fp32 or that type; statistics and sums are fp32 and every
output is rounded once.  Everything runs on the current torch stream,
asynchronously; errors in arguments raise ``ValueError`` before a launch.  An
output of the inputs' type may be a contiguous input itself; no output may
otherwise share memory with an input or another output.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _capi
from .recurrence import DTYPES, _call, _dense, _fault, _like, _need, _ptr, _rows

_pack_add, _pack_gated, _pack_grad = (
    _capi.packer(t) for t in (_capi.GdnAddNormArgs, _capi.GdnGatedNormArgs, _capi.GdnNormGradArgs))
QUANT = {None: _capi.QUANT_NONE, "row": _capi.QUANT_ROW, "group": _capi.QUANT_GROUP}
GROUP = 128
MAX_WIDTH = 32768
HEAD_DIMS = (64, 128, 256)


def _weight(weight, width: int, dtype, device) -> int:
    if not isinstance(weight, torch.Tensor) or weight.dtype not in (torch.float32, dtype):
        raise ValueError(f"weight must be float32 or {dtype}, got {getattr(weight, 'dtype', type(weight))}")
    _dense(weight, "weight", weight.dtype, (width,), device)
    return DTYPES[weight.dtype]


def _row_inputs(x, weight, eps) -> tuple[int, int, int]:
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a [rows, width] tensor")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")
    if x.dtype not in DTYPES:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    rows, width = x.shape
    if not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"rows must have 1 to {MAX_WIDTH} elements, got {width}")
    if not eps >= 0:
        raise ValueError("eps must be >= 0")
    return rows, width, _weight(weight, width, x.dtype, x.device)


def launch_add_norm(x, residual, weight, eps=1e-6, output=None, new_residual=None, scale=None, quant=None):
    """Returns ``(output, new_residual)``, or with ``quant`` ``(output, new_residual, scale)``.

    ``x`` and ``residual`` are ``[rows, width]`` with a free row stride;
    ``residual=None`` norms ``x`` alone and returns ``x`` as ``new_residual``.
    ``new_residual`` is the sum in the inputs' type (the norm is of the
    unrounded sum) and may be ``residual`` or ``x`` (in place).  ``quant``:
    ``"row"`` (scale ``[rows, 1]``) or ``"group"`` (one scale per 128
    channels, scale ``[rows, width / 128]``); ``output`` is then
    ``float8_e4m3fn``.
    """
    rows, width, wdt = _row_inputs(x, weight, eps)
    dev = x.device
    if quant not in QUANT:
        raise ValueError(f"quant must be None, 'row' or 'group', got {quant!r}")
    if quant == "group" and width % GROUP:
        raise ValueError(f"group scales need a width that is a multiple of {GROUP}, got {width}")
    x_stride = _rows(x, "x", x.dtype, rows, width, dev)
    res_stride = 0
    if residual is not None:
        res_stride = _rows(residual, "residual", x.dtype, rows, width, dev)
        if new_residual is None:
            new_residual = _like(x)
        else:
            _dense(new_residual, "new_residual", x.dtype, (rows, width), dev)
    else:
        _need(new_residual is None, "new_residual needs a residual")
    odt = torch.float8_e4m3fn if quant else x.dtype
    if output is None:
        output = _like(x, odt)
    else:
        _dense(output, "output", odt, (rows, width), dev)
        _need(rows == 0 or new_residual is None or output.data_ptr() != new_residual.data_ptr(),
              "output must not be new_residual")
    if quant:
        scale_shape = (rows, 1 if quant == "row" else width // GROUP)
        if scale is None:
            scale = x.new_empty(scale_shape, dtype=torch.float32)
        else:
            _dense(scale, "scale", torch.float32, scale_shape, dev)
    else:
        _need(scale is None, "scale needs quant")
    args = _pack_add(_ptr(x), _ptr(residual), x_stride, res_stride, _ptr(weight), wdt, DTYPES[x.dtype],
                                QUANT[quant], eps, rows, width, _ptr(output), _ptr(new_residual), _ptr(scale))
    _call(_capi.load().gdn_add_norm_launch, "gdn_add_norm_launch", dev, args)
    summed = x if residual is None else new_residual
    return (output, summed, scale) if quant else (output, summed)


def launch_add_norm_backward(d_output, new_residual, weight, eps=1e-6, d_new_residual=None, dx=None):
    """Gradients of ``launch_add_norm``: ``(dx, d_weight)``.

    ``new_residual`` is the sum that the forward call returned (``x`` where it
    had no residual).  ``dx`` is the gradient of ``x`` and of ``residual``
    alike, the ``d_new_residual`` that came down the residual stream (``None``:
    zero) included; ``d_weight`` is fp32.  Sums are taken in a fixed order.
    """
    rows, width, wdt = _row_inputs(new_residual, weight, eps)
    dev, dt = new_residual.device, new_residual.dtype
    r_stride = _rows(new_residual, "new_residual", dt, rows, width, dev)
    dy_stride = _rows(d_output, "d_output", dt, rows, width, dev)
    dr_stride = 0 if d_new_residual is None else _rows(d_new_residual, "d_new_residual", dt, rows, width, dev)
    if dx is None:
        dx = _like(new_residual)
    else:
        _dense(dx, "dx", dt, (rows, width), dev)
    d_weight = _like(weight, torch.float32)
    lib = _capi.load()
    need = int(lib.gdn_add_norm_backward_workspace_size(rows, width))
    workspace = weight.new_empty(need, dtype=torch.uint8)
    args = _pack_add(_ptr(new_residual), 0, r_stride, 0, _ptr(weight), wdt, DTYPES[dt], 0, eps, rows, width, 0, 0, 0)
    g = _pack_grad(_ptr(d_output), dy_stride, _ptr(d_new_residual), dr_stride, _ptr(dx), 0, _ptr(d_weight))
    _call(lib.gdn_add_norm_backward_launch, "gdn_add_norm_backward_launch", dev, args, g,
          _ptr(workspace), need)
    return dx, d_weight


def _heads(t, name: str, dtype, shape, device) -> int:
    """Checks a [tokens, heads, dim] tensor whose tokens are contiguous; returns the token stride."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.shape != shape:
        _fault(t, name, dtype, shape, device)
    tokens, heads, dim = shape
    step, head, inner = t.stride()
    if inner != 1 or (head != dim and heads > 1):
        raise ValueError(f"{name} must have contiguous heads, got strides {t.stride()}")
    if tokens <= 1:
        return heads * dim
    if step < heads * dim:
        raise ValueError(f"{name} must not have overlapping tokens, got strides {t.stride()}")
    return step


def _gated_inputs(x, z, weight, eps):
    """x and z as [tokens, heads, dim] with their token strides, and the weight's type."""
    if not isinstance(x, torch.Tensor) or x.dim() < 3:
        raise ValueError("x must be a [tokens, heads, dim] tensor")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")
    if x.dtype not in DTYPES:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if not isinstance(z, torch.Tensor) or z.shape != x.shape:
        raise ValueError(f"z must have the shape of x, {tuple(x.shape)}")
    heads, dim = x.shape[-2:]
    if dim not in HEAD_DIMS:
        raise ValueError(f"the head dim must be one of {HEAD_DIMS}, got {dim}")
    if not 1 <= heads <= 4096:
        raise ValueError(f"x must have 1 to 4096 heads, got {heads}")
    if not eps >= 0:
        raise ValueError("eps must be >= 0")
    if x.dim() > 3:  # [batch, tokens, heads, dim]
        _need(x.is_contiguous() and z.is_contiguous(), "x and z must be contiguous with more than three dimensions")
        x, z = x.view(-1, heads, dim), z.view(-1, heads, dim)
    shape, dev = x.shape, x.device
    if shape[0] * heads > 0x7FFF0000:
        raise ValueError("too many heads in one call")
    return x, z, _heads(x, "x", x.dtype, shape, dev), _heads(z, "z", x.dtype, shape, dev), _weight(weight, dim, x.dtype, dev)


def _prepare_gated_norm(x, z, weight, eps, output, scale, quant, check: bool = False):
    """Checks the arguments and makes the C ones; returns ``(launch, output, scale)``.
    With ``check`` the library's checks, which are the launch's own, come now too."""
    shape = x.shape if isinstance(x, torch.Tensor) else None
    x, z, xs, zs, wdt = _gated_inputs(x, z, weight, eps)
    tokens, heads, dim = x.shape
    dev = x.device
    odt = torch.float8_e4m3fn if quant else x.dtype
    if output is None:
        output = _like(x, odt)
        if output.shape != shape:
            output = output.view(shape)
    else:
        _dense(output, "output", odt, shape, dev)
        _need(tokens == 0 or output.data_ptr() != z.data_ptr(), "output must not be z")
    if quant:
        if scale is None:
            scale = x.new_empty(shape[:-1], dtype=torch.float32)
        else:
            _dense(scale, "scale", torch.float32, shape[:-1], dev)
    else:
        _need(scale is None, "scale needs quant")
    args = _pack_gated(_ptr(x), _ptr(z), xs, zs, _ptr(weight), wdt, DTYPES[x.dtype],
                                  _capi.QUANT_GROUP if quant else _capi.QUANT_NONE, eps, tokens, heads, dim,
                                  _ptr(output), _ptr(scale))
    if check:
        _capi.check(_capi.load().gdn_gated_norm_check(args), "gdn_gated_norm_check")

    def launch():
        _call(_capi.load().gdn_gated_norm_launch, "gdn_gated_norm_launch", dev, args)

    return launch, output, scale


def launch_gated_norm(x, z, weight, eps=1e-6, output=None, scale=None, quant: bool = False):
    """The gated per-head norm; returns ``output``, or with ``quant`` ``(output, scale)``.

    ``x`` and ``z`` are ``[tokens, heads, dim]`` (dim 64, 128 or 256) with a
    free token stride, or contiguous with more leading dimensions; ``weight``
    is ``[dim]``.  ``output`` has ``x``'s shape, contiguous, and may be a
    contiguous ``x`` itself.  With ``quant`` it is ``float8_e4m3fn`` with one
    fp32 scale per head, ``scale`` ``[..., heads]``.
    """
    launch, output, scale = _prepare_gated_norm(x, z, weight, eps, output, scale, quant)
    launch()
    return (output, scale) if quant else output


def launch_gated_norm_backward(d_output, x, z, weight, eps=1e-6, dx=None, dz=None):
    """Gradients of ``launch_gated_norm``: ``(dx, dz, d_weight)``; ``d_weight`` is fp32."""
    shape = x.shape if isinstance(x, torch.Tensor) else None
    x, z, xs, zs, wdt = _gated_inputs(x, z, weight, eps)
    tokens, heads, dim = x.shape
    dev = x.device
    _need(isinstance(d_output, torch.Tensor) and d_output.shape == shape, f"d_output must have shape {tuple(shape)}")
    if d_output.dim() > 3:
        _need(d_output.is_contiguous(), "d_output must be contiguous with more than three dimensions")
        d_output = d_output.view(-1, heads, dim)
    dys = _heads(d_output, "d_output", x.dtype, x.shape, dev)
    if dx is None:
        dx = _like(x).view(shape)
    else:
        _dense(dx, "dx", x.dtype, shape, dev)
    if dz is None:
        dz = _like(x).view(shape)
    else:
        _dense(dz, "dz", x.dtype, shape, dev)
        _need(tokens == 0 or dz.data_ptr() != dx.data_ptr(), "dz must not be dx")
    d_weight = _like(weight, torch.float32)
    lib = _capi.load()
    need = int(lib.gdn_gated_norm_backward_workspace_size(tokens, heads, dim))
    workspace = weight.new_empty(need, dtype=torch.uint8)
    args = _pack_gated(_ptr(x), _ptr(z), xs, zs, _ptr(weight), wdt, DTYPES[x.dtype], 0, eps, tokens, heads, dim, 0, 0)
    g = _pack_grad(_ptr(d_output), dys, 0, 0, _ptr(dx), _ptr(dz), _ptr(d_weight))
    _call(lib.gdn_gated_norm_backward_launch, "gdn_gated_norm_backward_launch", dev, args,
          g, _ptr(workspace), need)
    return dx, dz, d_weight


@dataclass
class OutputNorm:
    """The gated norm that ``launch_gdn(..., out_norm=)`` applies to its output:
    ``z`` in the output's shape, ``weight`` ``[128]``.  With ``codes``
    (``float8_e4m3fn``, the output's shape) and ``scale`` (fp32, the shape
    without its last dimension) the e4m3 form is written there and ``output``
    keeps the recurrence's own values; without them ``output`` is normed in
    place."""

    z: torch.Tensor
    weight: torch.Tensor
    eps: float = 1e-6
    codes: torch.Tensor | None = None
    scale: torch.Tensor | None = None

    def prepare(self, output):
        """Checks the norm against the ``output`` it will be applied to, all of
        it, so that nothing is refused once the recurrence has run, and returns
        the call that launches it."""
        _need((self.codes is None) == (self.scale is None), "codes and scale go together")
        z = self.z
        _need(isinstance(z, torch.Tensor) and z.numel() == output.numel(), f"z must have the output's shape {tuple(output.shape)}")
        if z.shape != output.shape:  # [B, 1, heads, 128] for an output [B, heads, 128], or the other way round
            _need(z.is_contiguous(), "z must be contiguous unless it has the output's shape")
            z = z.view(output.shape)
        _need(z.numel() == 0 or output.data_ptr() != z.data_ptr(), "output must not be z")
        # in place, or at least none of the recurrence's output where the norm reads
        launch = _prepare_gated_norm(output, z, self.weight, self.eps, output, None, False, check=True)[0]
        if self.codes is None:
            return launch
        return _prepare_gated_norm(output, z, self.weight, self.eps, self.codes, self.scale, True, check=True)[0]


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        output, summed = launch_add_norm(x, residual, weight, eps)
        ctx.save_for_backward(summed, weight)
        ctx.eps, ctx.has_residual = eps, residual is not None
        return (output, summed) if ctx.has_residual else output

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_output, d_summed=None):
        summed, weight = ctx.saved_tensors
        if d_summed is not None:
            d_summed = d_summed.contiguous()
        dx, dw = launch_add_norm_backward(d_output.contiguous(), summed, weight, ctx.eps, d_summed)
        return dx, dx if ctx.has_residual else None, dw.to(weight.dtype), None


def add_norm(x, residual, weight, eps=1e-6):
    """Differentiable ``launch_add_norm``: ``(output, new_residual)``, with
    gradients for ``x``, ``residual`` and ``weight``."""
    if residual is None:
        return _AddNorm.apply(x, None, weight, eps), x
    return _AddNorm.apply(x, residual, weight, eps)


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, weight, eps):
        ctx.save_for_backward(x, z, weight)
        ctx.eps = eps
        return launch_gated_norm(x, z, weight, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_output):
        x, z, weight = ctx.saved_tensors
        dx, dz, dw = launch_gated_norm_backward(d_output.contiguous(), x, z, weight, ctx.eps)
        return dx, dz, dw.to(weight.dtype), None


def gated_norm(x, z, weight, eps=1e-6):
    """Differentiable ``launch_gated_norm``, with gradients for ``x``, ``z`` and ``weight``."""
    return _GatedNorm.apply(x, z, weight, eps)
