"""The per-channel gated linear recurrence: packed scan, backward pass, decode step.

    h_t = g_t h_{t-1} + sigmoid(b_t) x_t,   y_t = h_t
    g_t = exp(-exp(A_log) softplus(a_t + dt_bias))

per channel, with the gates of the delta-rule entry points (``decode`` and
``prefill``) and, like them, destination-passing: ``launch_scan`` over packed
sequences (``cu_seqlens`` as ``prefill.launch_gdn``), ``launch_step`` for one
or a few tokens per sequence (as ``decode.launch_gdn``), and
``launch_scan_backward`` for training.  ``gated_scan`` is the differentiable
form.

``x``, ``a`` and ``b`` are ``[T, C]`` bf16, fp16 or fp32, all of one type,
channels contiguous; the token stride is free, so column blocks of one
projection's output need no copy.  ``A_log`` and ``dt_bias`` are fp32 ``[C]``,
states fp32 ``[N, C]``.  The state, the gates and every sum are fp32; outputs
are rounded once.  Everything runs on the current torch stream of the tensors'
device, asynchronously.  Errors in arguments raise ``ValueError`` before
anything launches; bad ``cu_seqlens`` values are reported through
``prefill.device_status``.
"""
from __future__ import annotations

import torch

from . import _capi

_pack_scan, _pack_scan_grad = _capi.packer(_capi.GdnScanArgs), _capi.packer(_capi.GdnScanGradArgs)
# What the kernels' indices hold: elements between tokens, channels, tokens and sequences.
MAX_STRIDE, MAX_CHANNELS, MAX_ROWS = 1 << 29, 1 << 20, 0x7FFF0000
DTYPES = {torch.bfloat16: _capi.DTYPE_BF16, torch.float16: _capi.DTYPE_F16, torch.float32: _capi.DTYPE_F32}


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _fault(t, name: str, dtype, shape, device) -> None:
    """Says what keeps ``t`` from being a tensor of that type, device and shape."""
    _need(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    _need(t.device == device, f"{name} must be on {device}, got {t.device}")
    _need(t.shape == shape, f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


# The checks below run on every call, a decode step's among them: messages are
# made only when there is something to say.
def _rows(t, name: str, dtype, rows: int, width: int, device) -> int:
    """Checks a ``[rows, width]`` tensor with contiguous rows; returns its row stride."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.shape != (rows, width):
        _fault(t, name, dtype, (rows, width), device)
    stride, inner = t.stride()
    if inner != 1 and width > 1:
        raise ValueError(f"{name} must have contiguous rows, got strides {t.stride()}")
    if rows <= 1:
        return width
    if stride < width:
        raise ValueError(f"{name} must not have overlapping rows, got strides {t.stride()}")
    return stride


def _token_rows(t, name: str, dtype, rows: int, width: int, device) -> int:
    """``_rows`` of a tensor that a scan or a step reads or writes."""
    stride = _rows(t, name, dtype, rows, width, device)
    if stride > MAX_STRIDE:
        raise ValueError(f"{name} must have at most {MAX_STRIDE} elements between tokens, got {stride}")
    return stride


def _dense(t, name: str, dtype, shape, device) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.shape != shape:
        _fault(t, name, dtype, shape, device)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _like(x, dtype=None) -> torch.Tensor:
    """A contiguous tensor of ``x``'s shape (``empty_like`` is half the cost of ``empty``)."""
    return torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)


def _call(fn, what: str, device, *args) -> None:
    """``fn(*args, current stream of device)`` with that device current."""
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _capi.check(rc, what)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _inputs(x, A_log, a, dt_bias, b, require_cuda: bool):
    """Checks what every entry point takes; returns (rows, channels, x, a and b strides)."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a [T, C] tensor")
    dtype, dev, shape = x.dtype, x.device, x.shape
    T, C = shape
    if require_cuda and not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")
    if dtype not in DTYPES:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {dtype}")
    if not 1 <= C <= MAX_CHANNELS:
        raise ValueError(f"x must have 1 to {MAX_CHANNELS} channels, got {C}")
    if T > MAX_ROWS:
        raise ValueError(f"x must have at most {MAX_ROWS} tokens, got {T}")
    layout = x.stride()
    stride = (layout[0] if T > 1 and layout[1] == 1 and C <= layout[0] <= MAX_STRIDE
              else _token_rows(x, "x", dtype, T, C, dev))
    strides = [stride]
    for t, name in ((a, "a"), (b, "b")):  # mostly in the layout of x
        if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == dev and t.shape == shape
                and t.stride() == layout):
            strides.append(stride)
        else:
            strides.append(_token_rows(t, name, dtype, T, C, dev))
    for t, name in ((A_log, "A_log"), (dt_bias, "dt_bias")):
        _dense(t, name, torch.float32, (C,), dev)
    return T, C, strides


def _seqlens(cu_seqlens, T: int, device, check: bool) -> int:
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a 1-D tensor of N+1 offsets")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("cu_seqlens must be int32 or int64")
    if cu_seqlens.device != device:
        raise ValueError(f"cu_seqlens must be on {device}")
    if not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be contiguous")
    if check:
        cu = cu_seqlens.to("cpu", torch.int64)
        _need(int(cu[0]) >= 0, "cu_seqlens[0] must be >= 0")
        _need(bool((cu[1:] >= cu[:-1]).all()), "cu_seqlens must be non-decreasing")
        _need(int(cu[-1]) <= T, f"cu_seqlens[-1]={int(cu[-1])} exceeds total tokens {T}")
    if cu_seqlens.numel() - 1 > MAX_ROWS:
        raise ValueError(f"cu_seqlens must have at most {MAX_ROWS} sequences")
    return cu_seqlens.numel() - 1


def validate(x, A_log, a, dt_bias, b, cu_seqlens, state, output, new_state, checkpoints=None,
             check_seqlens: bool = False, require_cuda: bool = True) -> tuple[int, int, int]:
    """Checks every argument of ``launch_scan``; returns ``(T, N, C)``.

    With ``check_seqlens`` the cu_seqlens values are copied to the host and
    checked (a device sync).  ``require_cuda=False`` checks only
    shapes/dtypes/layout (host-side tests).
    """
    T, C, _ = _inputs(x, A_log, a, dt_bias, b, require_cuda)
    dev = x.device
    N = _seqlens(cu_seqlens, T, dev, check_seqlens)
    _token_rows(output, "output", x.dtype, T, C, dev)
    _dense(new_state, "new_state", torch.float32, (N, C), dev)
    if state is not None:
        _dense(state, "state", torch.float32, (N, C), dev)
        _need(N == 0 or state.data_ptr() != new_state.data_ptr(), "state must not alias new_state")
    if checkpoints is not None:
        _dense(checkpoints, "checkpoints", torch.float32, (_checkpoint_rows(T), C), dev)
    _need(T == 0 or output.data_ptr() not in (x.data_ptr(), a.data_ptr(), b.data_ptr()),
          "output must not overlap an input")
    return T, N, C


def _checkpoint_rows(T: int) -> int:
    return int(_capi.load().gdn_scan_checkpoint_rows(T))


def empty_checkpoints(x) -> torch.Tensor:
    """The buffer that ``launch_scan`` fills for ``launch_scan_backward`` (one
    fp32 row of channels per 60 packed tokens)."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a [T, C] tensor")
    return x.new_empty((_checkpoint_rows(x.shape[0]), x.shape[1]), dtype=torch.float32)


def _args(x, A_log, a, dt_bias, b, cu_seqlens, state, strides, seqs, output, new_state, checkpoints):
    rows, C = x.shape
    return _pack_scan(
        x.data_ptr(), a.data_ptr(), b.data_ptr(), *strides, A_log.data_ptr(), dt_bias.data_ptr(), _ptr(state),
        cu_seqlens.data_ptr(), _capi.GDN_SEQLENS_INT64 if cu_seqlens.dtype == torch.int64 else _capi.GDN_SEQLENS_INT32,
        DTYPES[x.dtype], rows, seqs, C, _ptr(output), 0 if output is None else output.stride(0) if rows > 1 else C,
        _ptr(new_state), _ptr(checkpoints))


def launch_scan(x, A_log, a, dt_bias, b, cu_seqlens, state=None, output=None, new_state=None, checkpoints=None,
                check_seqlens: bool = False):
    """The recurrence over packed sequences; returns ``(output, new_state)``.

    ``state`` is ``[N, C]`` fp32 (``None``: zero) and must not be
    ``new_state``; an empty sequence's ``new_state`` row is its ``state`` row.
    Output rows of tokens that belong to no sequence are zeros.
    ``checkpoints`` (``empty_checkpoints(x)``) is filled for the backward pass.
    ``output`` may be row-strided (a column block of a wider buffer).  No
    output may share memory with an input or another output.
    """
    T, C, strides = _inputs(x, A_log, a, dt_bias, b, True)
    if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.device != x.device:
        cu_seqlens = cu_seqlens.to(x.device)
    N = _seqlens(cu_seqlens, T, x.device, check_seqlens)
    if output is None:
        output = _like(x)
    else:
        _token_rows(output, "output", x.dtype, T, C, x.device)
        _need(T == 0 or output.data_ptr() not in (x.data_ptr(), a.data_ptr(), b.data_ptr()),
              "output must not overlap an input")
    if state is not None:
        _dense(state, "state", torch.float32, (N, C), x.device)
    if new_state is None:
        new_state = x.new_empty((N, C), dtype=torch.float32) if state is None else _like(state)
    else:
        _dense(new_state, "new_state", torch.float32, (N, C), x.device)
        _need(N == 0 or state is None or state.data_ptr() != new_state.data_ptr(), "state must not alias new_state")
    if checkpoints is not None:
        _dense(checkpoints, "checkpoints", torch.float32, (_checkpoint_rows(T), C), x.device)
    args = _args(x, A_log, a, dt_bias, b, cu_seqlens, state, strides, N, output, new_state, checkpoints)
    _call(_capi.load().gdn_scan_launch, "gdn_scan_launch", x.device, args)
    return output, new_state


def launch_scan_backward(d_output, x, A_log, a, dt_bias, b, cu_seqlens, state, checkpoints, d_new_state=None, dx=None,
                         da=None, db=None):
    """Gradients of ``launch_scan``: ``(dx, da, db, dA_log, d_dt_bias, d_state)``.

    The arguments are those of the forward call and the ``checkpoints`` that it
    filled; ``d_output`` is ``[T, C]`` of ``x``'s type, ``d_new_state`` fp32
    ``[N, C]`` (``None``: zero).  ``dx``, ``da``, ``db`` may be given
    (row-strided, e.g. column blocks of the projection's gradient) and share no
    memory with each other or an input; ``dA_log``
    and ``d_dt_bias`` are fp32 ``[C]``, ``d_state`` fp32 ``[N, C]`` (``None``
    when ``state`` is).  Sums are taken in a fixed order: the same call gives
    the same bits.
    """
    T, C, strides = _inputs(x, A_log, a, dt_bias, b, True)
    dev = x.device
    if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.device != dev:
        cu_seqlens = cu_seqlens.to(dev)
    N = _seqlens(cu_seqlens, T, dev, False)
    dy_stride = _token_rows(d_output, "d_output", x.dtype, T, C, dev)
    _dense(checkpoints, "checkpoints", torch.float32, (_checkpoint_rows(T), C), dev)
    if state is not None:
        _dense(state, "state", torch.float32, (N, C), dev)
    if d_new_state is not None:
        _dense(d_new_state, "d_new_state", torch.float32, (N, C), dev)
    grads, grad_strides = [], []
    for t, name in ((dx, "dx"), (da, "da"), (db, "db")):
        if t is None:
            t = _like(x)
            grad_strides.append(C)
        else:
            grad_strides.append(_token_rows(t, name, x.dtype, T, C, dev))
            _need(T == 0 or t.data_ptr() not in (x.data_ptr(), a.data_ptr(), b.data_ptr(), d_output.data_ptr()),
                  f"{name} must not overlap an input")
            _need(T == 0 or all(t.data_ptr() != u.data_ptr() for u in grads), f"{name} must not overlap another gradient")
        grads.append(t)
    dA_log, d_dt_bias = _like(A_log), _like(dt_bias)
    d_state = None if state is None else _like(state)
    args = _args(x, A_log, a, dt_bias, b, cu_seqlens, state, strides, N, None, None, checkpoints)
    g = _pack_scan_grad(_ptr(d_output), dy_stride, _ptr(d_new_state), *(_ptr(t) for t in grads), *grad_strides,
                              _ptr(dA_log), _ptr(d_dt_bias), _ptr(d_state))
    _call(_capi.load().gdn_scan_backward_launch, "gdn_scan_backward_launch", dev, args, g)
    return (*grads, dA_log, d_dt_bias, d_state)


def launch_step(x, A_log, a, dt_bias, b, state, output=None, new_state=None):
    """One decode step; returns ``(output, new_state)``.

    ``x``, ``a``, ``b`` are ``[B, C]``, or ``[B, T, C]`` for T tokens per
    sequence applied in order; ``state`` is ``[B, C]`` fp32 and may be
    ``new_state`` (in-place update), and a contiguous ``x``, ``a`` or ``b``
    may be ``output``.
    """
    if not isinstance(x, torch.Tensor) or x.dim() not in (2, 3):
        raise ValueError("x must be a [B, C] or [B, T, C] tensor")
    shape, tokens = x.shape, 1
    B = shape[0]
    if x.dim() == 3:
        tokens = shape[1]
        _need(tokens >= 1, "x must have at least one token per sequence")
        flat = []
        for t, name in ((x, "x"), (a, "a"), (b, "b")):
            _need(isinstance(t, torch.Tensor) and t.shape == shape, f"{name} must have shape {tuple(shape)}")
            _need(B <= 1 or tokens <= 1 or t.stride(0) == tokens * t.stride(1),
                  f"{name} must have evenly spaced tokens, got strides {t.stride()}")
            flat.append(t.flatten(0, 1))
        x, a, b = flat
    rows, C, strides = _inputs(x, A_log, a, dt_bias, b, True)
    dev = x.device
    _dense(state, "state", torch.float32, (B, C), dev)
    if output is None:
        output = _like(x) if tokens == 1 and len(shape) == 2 else x.new_empty(shape)
    else:
        _dense(output, "output", x.dtype, shape, dev)
    if new_state is None:
        new_state = _like(state)
    elif new_state is not state:
        _dense(new_state, "new_state", torch.float32, (B, C), dev)
    args = _pack_scan(x.data_ptr(), a.data_ptr(), b.data_ptr(), *strides, A_log.data_ptr(), dt_bias.data_ptr(),
                      state.data_ptr(), 0, 0, DTYPES[x.dtype], rows, B, C, output.data_ptr(), C, new_state.data_ptr(), 0)
    _call(_capi.load().gdn_scan_step_launch, "gdn_scan_step_launch", dev, args, tokens)
    return output, new_state


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, A_log, a, dt_bias, b, cu_seqlens, state):
        checkpoints = empty_checkpoints(x)
        output, new_state = launch_scan(x, A_log, a, dt_bias, b, cu_seqlens, state, checkpoints=checkpoints)
        ctx.save_for_backward(x, A_log, a, dt_bias, b, cu_seqlens, state, checkpoints)
        return output, new_state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_output, d_new_state):
        x, A_log, a, dt_bias, b, cu_seqlens, state, checkpoints = ctx.saved_tensors
        dx, da, db, dA_log, d_dt_bias, d_state = launch_scan_backward(
            d_output.contiguous(), x, A_log, a, dt_bias, b, cu_seqlens, state, checkpoints, d_new_state.contiguous())
        return dx, dA_log, da, d_dt_bias, db, None, d_state


def gated_scan(x, A_log, a, dt_bias, b, cu_seqlens, state=None):
    """Differentiable ``launch_scan``: ``(output, new_state)`` with gradients
    for ``x``, ``A_log``, ``a``, ``dt_bias``, ``b`` and ``state``."""
    if isinstance(cu_seqlens, torch.Tensor) and isinstance(x, torch.Tensor) and cu_seqlens.device != x.device:
        cu_seqlens = cu_seqlens.to(x.device)
    return _GatedScan.apply(x, A_log, a, dt_bias, b, cu_seqlens, state)
