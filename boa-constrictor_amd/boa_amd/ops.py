"""Operators of the model's training pass and of its streaming by single tokens, on GPU tensors.

  layer_norm          rows of d values, weight and bias (nn.LayerNorm of model.py:45,51)
  causal_conv         the mixer's depthwise convolution over 4 positions with SiLU (model.py:72)
  selective_scan      the mixer's state space recurrence with its gate (model.py:72-81)
  cross_entropy       next-byte loss in nats (train.py:59-63)
  causal_conv_step, selective_scan_step   one token per sequence, states advanced in place

All of them run hand-written kernels of libboa_hip.so (include/boa_hip.h) on the current stream of their tensors' device,
synchronize nothing and can be captured into a graph.  The first four are differentiable (once, backward): gradients reach
every floating input but the states; inputs with a tangent of forward-mode differentiation are refused, and so is every call
that torch.jit.trace or make_fx records.  Activations are float32, bfloat16 or float16, all of a call of the same type; parameters,
scan states and the gradients of parameters are float32; arithmetic is in float32 and each result is rounded once.  The same
inputs give the same bits.

Shapes: activations [batch, length, channels] with any batch and row strides (a last dimension that is not contiguous is
copied); conv states [batch, 3, channels] in the activations' type, oldest position first; scan states
[batch, 16, channels] float32; ``lens``: int32 [batch], the sequences' lengths in a padded batch.  Positions behind a
sequence's end are not read (they may hold anything) and come out, and have gradients, as zeros; a state handed on is the one
behind the sequence's last position, so a sequence of length 0 hands on the state that it was given.

States carry no gradient: a batch that continues from a state trains on its own positions (truncated back-propagation).

Captured backward passes: torch ties a parameter's gradient accumulation to the stream that first used it, so do the warm-up
passes on the capture's side stream and let go of any eager graph of the same parameters before capturing.
"""
from __future__ import annotations

import functools
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from boa_amd import _native as _nat

__all__ = ["layer_norm", "causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "cross_entropy",
           "D_STATE", "D_CONV"]

D_STATE, D_CONV = 16, 4
_DTYPES = {torch.float32: _nat.BOA_DT_F32, torch.bfloat16: _nat.BOA_DT_BF16, torch.float16: _nat.BOA_DT_F16}
_INT_BYTES = {torch.uint8: 1, torch.int32: 4, torch.int64: 8}


# ---- argument checks -------------------------------------------------------------------------------
# A single-token step takes 10 us on the host, a third of it these checks: what is right is seen at once (_is), what is wrong is
# looked at again for the message.
_Tensor, _F32 = torch.Tensor, torch.float32


def _is(t, dtype, shape, device):
    return isinstance(t, _Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == device


def _act(who, name, t, shape=None, like=None):
    """An activation: its type code; a tensor of `like`'s type and device, and of `shape`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{who}: {name} must be a tensor")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{who}: {name} must be float32, bfloat16 or float16 (got {t.dtype})")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{who}: {name} must have the type and device of the other activations "
                         f"({like.dtype}, {like.device}; got {t.dtype}, {t.device})")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{who}: {name} must be {list(shape)} (got {list(t.shape)})")
    return code


def _param(who, name, t, shape, like):
    """A float32 parameter or state of this shape on the activations' device, contiguous; None stays None."""
    if t is None:
        return None
    if _is(t, _F32, shape, like.get_device()):
        return t if t.is_contiguous() else t.contiguous()
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
        raise TypeError(f"{who}: {name} must be a float32 tensor")
    raise ValueError(f"{who}: {name} must be {list(shape)} on {like.device} (got {list(t.shape)} on {t.device})")


def _state(who, t, shape, like, dtype, in_place):
    if t is None:
        return None
    if not _is(t, dtype, shape, like.get_device()):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype:
            raise TypeError(f"{who}: state must be a {dtype} tensor")
        raise ValueError(f"{who}: state must be {list(shape)} on {like.device} (got {list(t.shape)} on {t.device})")
    if t.requires_grad:
        raise ValueError(f"{who}: states carry no gradient; detach() it")
    if not t.is_contiguous():
        if in_place:
            raise ValueError(f"{who}: a state that is advanced in place must be contiguous")
        t = t.contiguous()
    return t


def _lens(who, t, batch, length, like):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{who}: lens must be an int32 tensor")
    if t.device != like.device or t.shape != (batch,):
        raise ValueError(f"{who}: lens must be [{batch}] on {like.device} (got {list(t.shape)} on {t.device})")
    if t.dtype == torch.int64:
        t = t.clamp(0, length).to(torch.int32)  # what the kernels do with int32
    return t.contiguous()


def _rows(t):
    """The tensor with a contiguous last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _written(*ts):
    """Tensors of one channel with lazy negations written out (imaginary parts of conjugates; wider ones have gaps and are copied)."""
    return tuple(t.resolve_neg() if isinstance(t, _Tensor) else t for t in ts)


def _flat(t, d):
    """[..., d] as rows: a tensor that holds them, their stride, their number."""
    if t.is_contiguous():
        return t, d, t.numel() // d
    t = _rows(t if t.ndim == 2 else t.reshape(-1, d))
    return t, t.stride(0), t.shape[0]


def _gpu(who, t):
    if not t.is_cuda:
        raise ValueError(f"{who}: the tensors must be on the GPU (got {t.device})")


def _grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


_raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice  # cheaper than a torch.cuda.Stream


def _call(t, f, *args):
    """An entry point (its last argument is the stream) on the current stream of a tensor's device, made current for it."""
    i = t.get_device()
    if i == _device():
        rc = f(*args, _raw_stream(i))
        if rc:
            _nat.check(rc)
    else:
        with torch.cuda.device(i):
            _nat.check(f(*args, _raw_stream(i)))


_tracing, _modes, _mode, _PROXY = (torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._get_dispatch_mode,
                                   torch._C._TorchDispatchModeKey.PROXY)


def _plain(who, *ts):
    """Refuses what a kernel behind a pointer would drop without a word: tangents, and the recording of the call by a tracer."""
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in ts:
            if isinstance(t, _Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{who}: forward-mode differentiation is not supported")
    if _tracing() or (_modes() and _mode(_PROXY) is not None):
        raise RuntimeError(f"{who}: cannot be traced (torch.jit.trace, make_fx)")


def _once(who, dy):
    """The upstream gradient in memory: autograd hands zeros and negations on without writing them.  The gradients are made by
    kernels, which autograd cannot differentiate again."""
    if torch.is_grad_enabled():
        raise RuntimeError("the operators of boa_amd.ops are differentiable once (create_graph is not supported)")
    _plain(who, dy)
    if dy._is_zerotensor():
        return torch.zeros(dy.shape, dtype=dy.dtype, device=dy.device)
    return dy.resolve_neg()


@functools.lru_cache(maxsize=256)
def _bytes(name, *sizes):
    return getattr(_nat.lib(), name)(*sizes)


def _ptr(t):
    """The address of an input that may be absent.  A tensor that stands for others (a subclass that wraps them, a fake one) has
    none, which would be taken for absence."""
    if t is None:
        return 0
    p = t.data_ptr()
    if not p and t.numel():
        raise ValueError(f"boa_amd.ops: a {type(t).__name__} of shape {list(t.shape)} without memory of its own")
    return p


def _work(nbytes, like):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


# ---- layer norm ------------------------------------------------------------------------------------
def _norm_fwd(x, w, b, eps, keep):
    d = x.shape[-1]
    rows, stride, n = _flat(x, d)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = torch.empty((n, 2), dtype=torch.float32, device=x.device) if keep else None
    _call(x, _nat.lib().boa_layer_norm_fwd, _DTYPES[x.dtype], rows.data_ptr(), stride, _ptr(w), _ptr(b), n, d, eps, y.data_ptr(), d,
          _ptr(stats))
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps):
        y, stats = _norm_fwd(x, w, b, eps, True)
        ctx.save_for_backward(x, w, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        dy = _once("layer_norm", dy)
        x, w, stats = ctx.saved_tensors
        d = x.shape[-1]
        rows, stride, n = _flat(x, d)
        dyr, dy_stride, _ = _flat(dy, d)
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        _, need_w, need_b, _ = ctx.needs_input_grad
        dwb = work = None
        size = 0
        if need_w or need_b:
            dwb = stats.new_empty((2, d))
            size = _bytes("boa_layer_norm_bwd_work_bytes", n, d)
            work = _work(size, x)
        _call(x, _nat.lib().boa_layer_norm_bwd, _DTYPES[x.dtype], dyr.data_ptr(), dy_stride, rows.data_ptr(), stride, _ptr(w),
              stats.data_ptr(), n, d, dx.data_ptr(), d, _ptr(dwb), _ptr(work), size)
        return dx, dwb[0] if need_w else None, dwb[1] if need_b else None, None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (1 to 4096 values), biased variance.

    x: [..., d]; weight, bias: float32 [d] or None.  Returns a contiguous tensor of x's shape and type."""
    _plain("layer_norm", x, weight, bias)
    _act("layer_norm", "x", x)
    if x.ndim < 1 or not 1 <= x.shape[-1] <= _nat.BOA_LAYER_NORM_MAX_D:
        raise ValueError(f"layer_norm: x must be [..., d] with 1 <= d <= {_nat.BOA_LAYER_NORM_MAX_D} (got {list(x.shape)})")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must not be negative (got {eps})")
    if x.shape[-1] == 1:
        weight, bias = _written(weight, bias)
    w = _param("layer_norm", "weight", weight, x.shape[-1:], x)
    b = _param("layer_norm", "bias", bias, x.shape[-1:], x)
    _gpu("layer_norm", x)
    if _grad(x, w, b):
        return _LayerNorm.apply(x, w, b, float(eps))
    return _norm_fwd(x, w, b, float(eps), False)[0]


# ---- cross entropy ---------------------------------------------------------------------------------
class _CrossEntropy(torch.autograd.Function):
    # In one allocation: the forward pass's workspace, the number of rows that count, and what the backward pass needs of each row.
    @staticmethod
    def forward(ctx, x, target, ignore, reduction, keep):
        v = x.shape[-1]
        rows, stride, n = _flat(x, v)
        lib = _nat.lib()
        size = 0 if reduction == "none" else _bytes("boa_cross_entropy_work_bytes")
        buf = torch.empty(size + 16 + (8 * n if keep else 0), dtype=torch.uint8, device=x.device)
        work = buf.data_ptr()
        count, stats = work + size, work + size + 16
        loss = torch.empty(x.shape[:-1] if reduction == "none" else (), dtype=torch.float32, device=x.device)
        each, all_rows = (loss.data_ptr(), 0) if reduction == "none" else (0, loss.data_ptr())
        _call(x, lib.boa_cross_entropy_fwd, _DTYPES[x.dtype], rows.data_ptr(), stride, target.data_ptr(), target.element_size(),
              ignore, n, v, reduction == "mean", stats if keep else 0, each, all_rows, count if all_rows else 0,
              work if all_rows else 0, size)
        if keep:
            ctx.save_for_backward(x, target, buf)
            ctx.ignore, ctx.reduction, ctx.size = ignore, reduction, size
        return loss

    @staticmethod
    def backward(ctx, up):
        up = _once("cross_entropy", up)
        x, target, buf = ctx.saved_tensors
        v = x.shape[-1]
        rows, stride, n = _flat(x, v)
        up = up.contiguous()  # float32, as the loss is
        dx = x.new_empty(x.shape)
        count = buf.data_ptr() + ctx.size
        _call(x, _nat.lib().boa_cross_entropy_bwd, _DTYPES[x.dtype], rows.data_ptr(), stride, target.data_ptr(),
              target.element_size(), ctx.ignore, n, v, count + 16, up.data_ptr(), ctx.reduction == "none",
              count if ctx.reduction == "mean" else 0, dx.data_ptr(), v)
        return dx, None, None, None, None


def cross_entropy(logits, targets, *, ignore_index: int = -100, reduction: str = "mean"):
    """``log(sum(exp(logits))) - logits[target]`` of every row, in nats: their mean over the rows that count, their sum, or
    (reduction "none") one value per row.

    logits: [..., V] (1 to 4096 symbols); targets: uint8, int32 or int64 of the leading shape.  Rows whose target is
    ignore_index count for nothing and have no gradient (a mean over no rows is NaN); any other target outside [0, V) gives
    NaN.  Returns float32."""
    _plain("cross_entropy", logits)
    _act("cross_entropy", "logits", logits)
    if logits.ndim < 1 or not 1 <= logits.shape[-1] <= _nat.BOA_CROSS_ENTROPY_MAX_V:
        raise ValueError(f"cross_entropy: logits must be [..., V] with 1 <= V <= {_nat.BOA_CROSS_ENTROPY_MAX_V} "
                         f"(got {list(logits.shape)})")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"cross_entropy: reduction must be mean, sum or none (got {reduction!r})")
    if not isinstance(targets, torch.Tensor) or targets.dtype not in _INT_BYTES:
        raise TypeError("cross_entropy: targets must be a uint8, int32 or int64 tensor")
    if targets.device != logits.device or targets.shape != logits.shape[:-1]:
        raise ValueError(f"cross_entropy: targets must be {list(logits.shape[:-1])} on {logits.device} "
                         f"(got {list(targets.shape)} on {targets.device})")
    _gpu("cross_entropy", logits)
    return _CrossEntropy.apply(logits, targets.contiguous(), int(ignore_index), reduction, _grad(logits))


# ---- causal convolution ----------------------------------------------------------------------------
def _conv_fwd(x, w, b, silu, state, lens, want_state):
    n, length, c = x.shape
    y = x.new_empty((n, length, c))
    out = x.new_empty((n, D_CONV - 1, c)) if want_state else None
    _call(x, _nat.lib().boa_causal_conv_fwd, _DTYPES[x.dtype], x.data_ptr(), x.stride(0), x.stride(1), w.data_ptr(), _ptr(b), silu,
          n, length, c, _ptr(lens), _ptr(state), _ptr(out), y.data_ptr(), length * c, c)
    return y, out


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, silu, state, lens, want_state):
        y, out = _conv_fwd(x, w, b, silu, state, lens, want_state)
        ctx.save_for_backward(x, w, b, state, lens)
        ctx.silu = silu
        if out is not None:
            ctx.mark_non_differentiable(out)
        return y, out

    @staticmethod
    def backward(ctx, dy, _):
        dy = _once("causal_conv", dy)
        x, w, b, state, lens = ctx.saved_tensors
        n, length, c = x.shape
        dy = _rows(dy)
        dx = x.new_empty((n, length, c))
        need_w, need_b = ctx.needs_input_grad[1:3]
        dwb = work = None
        size = 0
        if need_w or need_b:
            dwb = w.new_empty((D_CONV + 1) * c)
            size = _bytes("boa_causal_conv_bwd_work_bytes", n, length, c)
            work = _work(size, x)
        _call(x, _nat.lib().boa_causal_conv_bwd, _DTYPES[x.dtype], dy.data_ptr(), dy.stride(0), dy.stride(1), x.data_ptr(), x.stride(0),
              x.stride(1), w.data_ptr(), _ptr(b), ctx.silu, n, length, c, _ptr(lens), _ptr(state), dx.data_ptr(), length * c, c,
              _ptr(dwb), _ptr(work), size)
        dw = dwb.as_strided(w.shape, w.stride()) if need_w else None
        db = dwb[D_CONV * c:] if need_b else None
        return dx, dw, db, None, None, None, None


def _conv_args(who, x, ndim, weight, bias):
    _act(who, "x", x)
    if x.ndim != ndim or not 1 <= x.shape[-1] <= _nat.BOA_OPS_MAX_CHANNELS:
        raise ValueError(f"{who}: x must be {'[batch, length, channels]' if ndim == 3 else '[batch, channels]'} "
                         f"(got {list(x.shape)})")
    c = x.shape[-1]
    if c == 1:
        x, bias = _written(x, bias)
    flat = isinstance(weight, torch.Tensor) and weight.ndim == 2
    w = _param(who, "weight", weight, (c, D_CONV) if flat else (c, 1, D_CONV), x)
    if w is None:
        raise TypeError(f"{who}: weight must be a float32 tensor")
    return x, w, _param(who, "bias", bias, (c,), x)


def causal_conv(x, weight, bias=None, *, silu: bool = True, state=None, lens=None, return_state: bool = False):
    """Depthwise convolution of each channel over the last 4 positions, then SiLU unless ``silu`` is false.

    x: [batch, length, channels]; weight: float32 [channels, 1, 4] (nn.Conv1d's) or [channels, 4], oldest tap first; bias:
    float32 [channels]; state: the three positions before the first one (zeros without).  Returns y, with ``return_state``
    also the state behind each sequence's last position, as a new tensor."""
    _plain("causal_conv", x, weight, bias, state)
    x, w, b = _conv_args("causal_conv", x, 3, weight, bias)
    n, length, c = x.shape
    state = _state("causal_conv", state, (n, D_CONV - 1, c), x, x.dtype, False)
    lens = _lens("causal_conv", lens, n, length, x)
    _gpu("causal_conv", x)
    x = _rows(x)
    if _grad(x, w, b):
        y, out = _CausalConv.apply(x, w, b, bool(silu), state, lens, bool(return_state))
    else:
        y, out = _conv_fwd(x, w, b, bool(silu), state, lens, return_state)
    return (y, out) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, silu: bool = True):
    """``causal_conv`` of one position per sequence: x [batch, channels]; state [batch, 3, channels] is advanced in place.
    Returns y [batch, channels]; no gradient."""
    who = "causal_conv_step"
    _plain(who, x, state, weight, bias)
    x, w, b = _conv_args(who, x, 2, weight, bias)
    n, c = x.shape
    if state is None:
        raise TypeError(f"{who}: state must be a tensor")
    state = _state(who, state, (n, D_CONV - 1, c), x, x.dtype, True)
    if _grad(x, w, b):
        raise ValueError(f"{who}: no gradient; call it under torch.no_grad()")
    _gpu(who, x)
    x = _rows(x)
    y = x.new_empty((n, c))
    _call(x, _nat.lib().boa_causal_conv_step, _DTYPES[x.dtype], x.data_ptr(), x.stride(0), state.data_ptr(), w.data_ptr(), _ptr(b),
          bool(silu), n, c, y.data_ptr(), c)
    increment_version(state)  # autograd sees the change, as it does one by an operator of torch
    return y


# ---- selective scan --------------------------------------------------------------------------------
# boa_scan (include/boa_hip.h): dtype, channels, batch, length; u, delta, z, b, c (pointer, two strides); a, d, delta_bias,
# lens, state_in, state_out, marks; y, dy, du, ddelta, dz, db, dc; dpar
_SCAN = struct.Struct("@iiqq15q7q21qq")
_NO_ROWS = (0, 0, 0)
_NO_BACKWARD = (0,) * 19


def _r3(t):
    return _NO_ROWS if t is None else (_ptr(t), t.stride(0), t.stride(1))


def _pack(u, delta, A, B, C, D, z, bias, lens, state_in, state_out, marks, y, back=(None,) * 6, dpar=None):
    n, length, c = u.shape
    return _SCAN.pack(_DTYPES[u.dtype], c, n, length, *_r3(u), *_r3(delta), *_r3(z), *_r3(B), *_r3(C), A.data_ptr(), _ptr(D),
                      _ptr(bias), _ptr(lens), _ptr(state_in), _ptr(state_out), _ptr(marks), *_r3(y), *_r3(back[0]), *_r3(back[1]),
                      *_r3(back[2]), *_r3(back[3]), *_r3(back[4]), *_r3(back[5]), _ptr(dpar))


def _scan_rows(t):
    """Rows as the kernels read them: contiguous, not too far apart."""
    t = _rows(t)
    if t.stride(-2) <= _nat.BOA_SCAN_MAX_ROW_STRIDE:
        return t
    return t.clone(memory_format=torch.contiguous_format)  # contiguous() keeps the stride of a dimension of one


def _scalar_rows(t):
    """The same for B and C, whose rows begin at multiples of 4 bytes."""
    t = _scan_rows(t)
    if t.dtype is not _F32 and (t.data_ptr() % 4 or any(s % 2 for s in t.stride()[:-1])):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _scan_fwd(u, delta, A, B, C, D, z, bias, state, lens, want_state, keep):
    n, length, c = u.shape
    y = u.new_empty((n, length, c))
    out = A.new_empty((n, D_STATE, c)) if want_state else None
    marks = None
    if keep:
        marks = A.new_empty((n, -(-length // _nat.BOA_SCAN_MARK), D_STATE, c))
    args = _pack(u, delta, A, B, C, D, z, bias, lens, state, out, marks, y)
    lib = _nat.lib()
    size = lib.boa_selective_scan_work_bytes(args, 0)
    work = _work(size, u)
    _call(u, lib.boa_selective_scan_fwd, args, _ptr(work), size)
    return y, out, marks


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, state, lens, want_state):
        y, out, marks = _scan_fwd(u, delta, A, B, C, D, z, bias, state, lens, want_state, True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, lens, marks)
        if out is not None:
            ctx.mark_non_differentiable(out)
        return y, out

    @staticmethod
    def backward(ctx, dy, _):
        dy = _once("selective_scan", dy)
        u, delta, A, B, C, D, z, bias, lens, marks = ctx.saved_tensors
        n, length, c = u.shape
        dy = _scan_rows(dy)
        du, ddelta, dz = (u.new_empty((n, length, c)) if t is not None else None for t in (u, delta, z))
        dB, dC = (u.new_empty((n, length, D_STATE)) for _ in range(2))
        dpar = A.new_empty((D_STATE + 2) * c)
        args = _pack(u, delta, A, B, C, D, z, bias, lens, None, None, marks, None, (dy, du, ddelta, dz, dB, dC), dpar)
        lib = _nat.lib()
        size = lib.boa_selective_scan_work_bytes(args, 1)
        work = _work(size, u)
        _call(u, lib.boa_selective_scan_bwd, args, _ptr(work), size)
        dA = dpar.as_strided((c, D_STATE), (D_STATE, 1))
        dD = dpar[D_STATE * c:(D_STATE + 1) * c] if D is not None else None
        dbias = dpar[(D_STATE + 1) * c:] if bias is not None else None
        return du, ddelta, dA, dB, dC, dD, dz, dbias, None, None, None


def _scan_args(who, ndim, u, delta, A, B, C, D, z, bias):
    _act(who, "u", u)
    if u.ndim != ndim or not 1 <= u.shape[-1] <= _nat.BOA_OPS_MAX_CHANNELS:
        raise ValueError(f"{who}: u must be {'[batch, length, channels]' if ndim == 3 else '[batch, channels]'} "
                         f"(got {list(u.shape)})")
    dtype, shape, dev = u.dtype, u.shape, u.get_device()
    c = shape[-1]
    if c == 1:
        u, delta, z, D, bias = _written(u, delta, z, D, bias)
    states = shape[:-1] + (D_STATE,)
    if not _is(delta, dtype, shape, dev):
        _act(who, "delta", delta, shape, u)
    if z is not None and not _is(z, dtype, shape, dev):
        _act(who, "z", z, shape, u)
    if not _is(B, dtype, states, dev):
        _act(who, "B", B, states, u)
    if not _is(C, dtype, states, dev):
        _act(who, "C", C, states, u)
    A = _param(who, "A", A, (c, D_STATE), u)
    if A is None:
        raise TypeError(f"{who}: A must be a float32 tensor")
    D, bias = _param(who, "D", D, (c,), u), _param(who, "delta_bias", bias, (c,), u)
    rows = _scan_rows if ndim == 3 else _rows
    return rows(u), rows(delta), A, _scalar_rows(B), _scalar_rows(C), D, z if z is None else rows(z), bias


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, *, state=None, lens=None, return_state: bool = False):
    """``h = exp(dt A) h + dt B u``, ``y = (C . h + D u) silu(z)`` along the positions, ``dt = softplus(delta + delta_bias)``.

    u, delta, z: [batch, length, channels]; B, C: [batch, length, 16], shared by the channels; A: float32 [channels, 16]
    (negative); D, delta_bias: float32 [channels].  Without z there is no gate, without D no skip.  state: [batch, 16, channels]
    before the first position (zeros without).  Returns y, with ``return_state`` also the state behind each sequence's last
    position, as a new tensor."""
    who = "selective_scan"
    _plain(who, u, delta, A, B, C, D, z, delta_bias, state)
    args = _scan_args(who, 3, u, delta, A, B, C, D, z, delta_bias)
    n, length, c = u.shape
    state = _state(who, state, (n, D_STATE, c), u, torch.float32, False)
    lens = _lens(who, lens, n, length, u)
    _gpu(who, u)
    if _grad(*args):
        y, out = _SelectiveScan.apply(*args, state, lens, bool(return_state))
    else:
        y, out, _ = _scan_fwd(*args, state, lens, return_state, False)
    return (y, out) if return_state else y


def selective_scan_step(u, delta, A, B, C, D=None, z=None, delta_bias=None, *, state):
    """``selective_scan`` of one position per sequence: u, delta, z [batch, channels], B, C [batch, 16]; state
    [batch, 16, channels] is advanced in place.  Returns y [batch, channels]; no gradient."""
    who = "selective_scan_step"
    _plain(who, u, delta, A, B, C, D, z, delta_bias, state)
    args = _scan_args(who, 2, u, delta, A, B, C, D, z, delta_bias)
    n, c = u.shape
    if state is None:
        raise TypeError(f"{who}: state must be a tensor")
    state = _state(who, state, (n, D_STATE, c), u, torch.float32, True)
    if _grad(*args):
        raise ValueError(f"{who}: no gradient; call it under torch.no_grad()")
    _gpu(who, u)
    y = u.new_empty((n, c))
    u, delta, A, B, C, D, z, bias = args
    if A.data_ptr() % 16:
        A = A.clone()

    zp, zs = (0, 0) if z is None else (_ptr(z), z.stride(0))
    packed = _SCAN.pack(_DTYPES[u.dtype], c, n, 1, u.data_ptr(), u.stride(0), 0, delta.data_ptr(), delta.stride(0), 0, zp, zs, 0,
                        B.data_ptr(), B.stride(0), 0, C.data_ptr(), C.stride(0), 0, A.data_ptr(), _ptr(D), _ptr(bias), 0, 0,
                        state.data_ptr(), 0, y.data_ptr(), c, 0, *_NO_BACKWARD)
    _call(u, _nat.lib().boa_selective_scan_step, packed)
    increment_version(state)
    return y
