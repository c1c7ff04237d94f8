"""Operators of a model's training pass and of its streaming by single tokens, on GPU tensors.

  layer_norm          rows of d values, weight and bias (nn.LayerNorm of model.py:45,51)
  causal_conv         the mixer's depthwise convolution over 4 positions with SiLU (model.py:72)
  selective_scan      the mixer's state space recurrence with its gate (model.py:72-81)
  cross_entropy       next-byte loss in nats (train.py:59-63)
  linear_attention    a recurrence like the scan's whose state is a key x value matrix per head
  causal_conv_step, selective_scan_step, linear_attention_step   one token per sequence, states advanced in place
  grad_norm, clip_grad_norm_   the norm of all gradients together, and their scaling by it (before optimizer.step() of train.py:63)
  sample              next symbols drawn from logits by given random numbers, with temperature, top_k, top_p and min_p

All of them run hand-written kernels of libboa_hip.so (include/boa_hip.h) on the current stream of their tensors' device,
synchronize nothing and can be captured into a graph.  The first five are differentiable (once, backward): gradients reach
every floating input but the states; inputs with a tangent of forward-mode differentiation are refused, and so is every call
that torch.jit.trace or make_fx records.  Activations are float32, bfloat16 or float16, all of a call of the same type; parameters,
scan states and the gradients of parameters are float32; arithmetic is in float32 and each result is rounded once.  The same
inputs give the same bits.

Shapes: activations [batch, length, channels] with any batch and row strides (a last dimension that is not contiguous is
copied), of linear attention [batch, length, heads, key or value] with any strides but the last; conv states
[batch, 3, channels] in the activations' type, oldest position first; scan states [batch, 16, channels] and attention's
[batch, heads, key, value] float32; ``lens``: int32 [batch], the sequences' lengths in a padded batch.  Positions behind a
sequence's end are not read (they may hold anything) and come out, and have gradients, as zeros; a state handed on is the one
behind the sequence's last position, so a sequence of length 0 hands on the state that it was given.

States carry no gradient: a batch that continues from a state trains on its own positions (truncated back-propagation).

Captured backward passes: torch ties a parameter's gradient accumulation to the stream that first used it, so do the warm-up
passes on the capture's side stream and let go of any eager graph of the same parameters before capturing.
"""
from __future__ import annotations

import functools
import math
import operator
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from boa_amd import _native as _nat

__all__ = ["layer_norm", "causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "cross_entropy",
           "linear_attention", "linear_attention_step", "grad_norm", "clip_grad_norm_", "sample", "D_STATE", "D_CONV"]

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


# ---- linear attention ------------------------------------------------------------------------------
# boa_attention (include/boa_hip.h): dtype, heads, groups, key, value, decay_per_head, scale, unused; batch, length; q, k, v, y
# (pointer, three strides); decay and its strides; lens, state_in, state_out, marks; dy, dq, dk, dv; ddecay
_ATTENTION = struct.Struct("@6ifi2q16q4q4q16qq")
_NO_HEADS = (0, 0, 0, 0)


def _r4(t):
    return _NO_HEADS if t is None else (t.data_ptr(), *t.stride()[:-1])


def _pack_attention(q, k, v, g, scale, lens, state_in, state_out, marks, y, back=(None,) * 4, dg=None):
    n, length, groups, key = q.shape
    gs = (0, 0, 1) if g.ndim == 1 else g.stride()
    return _ATTENTION.pack(_DTYPES[q.dtype], v.shape[2], groups, key, v.shape[3], g.ndim == 1, scale, 0, n, length, *_r4(q), *_r4(k),
                           *_r4(v), *_r4(y), g.data_ptr(), *gs, _ptr(lens), _ptr(state_in), _ptr(state_out), _ptr(marks),
                           *_r4(back[0]), *_r4(back[1]), *_r4(back[2]), *_r4(back[3]), _ptr(dg))


def _attention_work(lib, args, backward):
    size = lib.boa_linear_attention_work_bytes(args, backward)
    if size < 0:
        _nat.check(_nat.BOA_ERR_ARG)
    return size


def _attention_fwd(q, k, v, g, scale, state, lens, want_state, keep):
    n, length, heads, value = v.shape
    y = v.new_empty((n, length, heads, value))
    out = g.new_empty((n, heads, q.shape[3], value)) if want_state else None
    # the states before every 64th position, of keys and values padded to multiples of 64
    marks = g.new_empty((n * heads, -(-value // 64), -(-length // 64), -(-q.shape[3] // 64) * 4096)) if keep else None
    args = _pack_attention(q, k, v, g, scale, lens, state, out, marks, y)
    lib = _nat.lib()
    size = _attention_work(lib, args, 0)
    work = _work(size, q)
    _call(q, lib.boa_linear_attention_fwd, args, _ptr(work), size)
    return y, out, marks


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, scale, state, lens, want_state):
        y, out, marks = _attention_fwd(q, k, v, g, scale, state, lens, want_state, True)
        ctx.save_for_backward(q, k, v, g, lens, marks)
        ctx.scale = scale
        if out is not None:
            ctx.mark_non_differentiable(out)
        return y, out

    @staticmethod
    def backward(ctx, dy, _):
        dy = _once("linear_attention", dy)
        q, k, v, g, lens, marks = ctx.saved_tensors
        dy = _rows(dy)
        dq, dk, dv, dg = (t.new_empty(t.shape) for t in (q, k, v, g))
        args = _pack_attention(q, k, v, g, ctx.scale, lens, None, None, marks, None, (dy, dq, dk, dv), dg)
        lib = _nat.lib()
        size = _attention_work(lib, args, 1)
        work = _work(size, q)
        _call(q, lib.boa_linear_attention_bwd, args, _ptr(work), size)
        return dq, dk, dv, dg, None, None, None, None


def _attention_args(who, ndim, q, k, v, g, scale):
    _act(who, "q", q)
    lead = "batch, length" if ndim == 4 else "batch"
    if q.ndim != ndim or not 1 <= q.shape[-1] <= _nat.BOA_ATTENTION_MAX_KEY or not q.shape[-2]:
        raise ValueError(f"{who}: q must be [{lead}, groups, key] with 1 <= key <= {_nat.BOA_ATTENTION_MAX_KEY} (got {list(q.shape)})")
    dev = q.get_device()
    if not _is(k, q.dtype, q.shape, dev):
        _act(who, "k", k, q.shape, q)
    _act(who, "v", v, None, q)
    if v.ndim != ndim or v.shape[:-2] != q.shape[:-2] or not 1 <= v.shape[-1] <= _nat.BOA_ATTENTION_MAX_VALUE:
        raise ValueError(f"{who}: v must be [{lead}, heads, value] with 1 <= value <= {_nat.BOA_ATTENTION_MAX_VALUE}, {lead} as q's "
                         f"(got {list(v.shape)} and {list(q.shape)})")
    heads = v.shape[-2]
    if not 1 <= heads <= _nat.BOA_ATTENTION_MAX_HEADS or heads % q.shape[-2]:
        raise ValueError(f"{who}: the heads of v must be a multiple of q's and k's, at most {_nat.BOA_ATTENTION_MAX_HEADS} "
                         f"(got {heads} and {q.shape[-2]})")
    if not isinstance(g, _Tensor) or g.dtype is not _F32:
        raise TypeError(f"{who}: log_decay must be a float32 tensor")
    if g.get_device() != dev or (g.shape != (heads,) and g.shape != v.shape[:-1]):
        raise ValueError(f"{who}: log_decay must be [{heads}] or {list(v.shape[:-1])} on {q.device} (got {list(g.shape)} on {g.device})")
    if g.ndim == 1 and g.stride(0) != 1:
        g = g.contiguous()
    if q.shape[-1] == 1:
        q, k = _written(q, k)
    if v.shape[-1] == 1:
        v, = _written(v)
    g, = _written(g)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    return _rows(q), _rows(k), _rows(v), g, scale


def linear_attention(q, k, v, log_decay, *, scale=None, state=None, lens=None, return_state: bool = False):
    """``S = exp(log_decay) S + k v^T``, ``y = scale S^T q`` along the positions: a state of key x value values per head, which
    ``selective_scan`` would have as 16 per channel with a decay each.

    q, k: [batch, length, groups, key] (1 to 128), each group shared by heads / groups consecutive heads; v: [batch, length, heads,
    value] (1 to 512); log_decay: float32 [heads], or [batch, length, heads] for one of each position's own, 0 or negative (-inf
    forgets everything before); scale: 1 / sqrt(key) unless given.  state: float32 [batch, heads, key, value] before the first
    position (zeros without).  Returns y [batch, length, heads, value], with ``return_state`` also the state behind each
    sequence's last position, as a new tensor.  Products q . k of near positions are made before scale and decay: beyond float32's
    range they are infinite (nothing behind a decay of zero)."""
    who = "linear_attention"
    _plain(who, q, k, v, log_decay, state)
    q, k, v, g, scale = _attention_args(who, 4, q, k, v, log_decay, scale)
    n, length, heads, value = v.shape
    state = _state(who, state, (n, heads, q.shape[-1], value), q, torch.float32, False)
    lens = _lens(who, lens, n, length, q)
    _gpu(who, q)
    if _grad(q, k, v, g):
        y, out = _LinearAttention.apply(q, k, v, g, scale, state, lens, bool(return_state))
    else:
        y, out, _ = _attention_fwd(q, k, v, g, scale, state, lens, return_state, False)
    return (y, out) if return_state else y


def linear_attention_step(q, k, v, log_decay, *, state, scale=None):
    """``linear_attention`` of one position per sequence: q, k [batch, groups, key], v [batch, heads, value], log_decay [heads] or
    [batch, heads]; state [batch, heads, key, value] is advanced in place.  Returns y [batch, heads, value]; no gradient."""
    who = "linear_attention_step"
    _plain(who, q, k, v, log_decay, state)
    q, k, v, g, scale = _attention_args(who, 3, q, k, v, log_decay, scale)
    n, heads, value = v.shape
    key = q.shape[-1]
    if state is None:
        raise TypeError(f"{who}: state must be a tensor")
    state = _state(who, state, (n, heads, key, value), q, torch.float32, True)
    if _grad(q, k, v, g):
        raise ValueError(f"{who}: no gradient; call it under torch.no_grad()")
    _gpu(who, q)
    y = v.new_empty((n, heads, value))
    per_head = g.ndim == 1
    packed = _ATTENTION.pack(_DTYPES[q.dtype], heads, q.shape[1], key, value, per_head, scale, 0, n, 1, q.data_ptr(), q.stride(0), 0,
                             q.stride(1), k.data_ptr(), k.stride(0), 0, k.stride(1), v.data_ptr(), v.stride(0), 0, v.stride(1),
                             y.data_ptr(), heads * value, 0, value, g.data_ptr(), 0 if per_head else g.stride(0), 0,
                             1 if per_head else g.stride(1), 0, 0, state.data_ptr(), 0, *(_NO_HEADS * 4), 0)
    _call(q, _nat.lib().boa_linear_attention_step, packed)
    increment_version(state)
    return y


# ---- gradient norm ---------------------------------------------------------------------------------
# A model has hundreds of gradients, and each look at one costs Python 70 ns: few looks, without calls of functions of our own.
_grad_of, _type_of = operator.attrgetter("grad"), operator.attrgetter("dtype")
_contiguous, _address, _size = _Tensor.is_contiguous, _Tensor.data_ptr, _Tensor.numel


def _grads(who, parameters, in_place):
    """The gradients of parameters, those that have one and memory for it; their number, addresses, sizes and types as the bytes of C
    arrays; copies of those that are not contiguous, with the originals; their device."""
    if isinstance(parameters, _Tensor):
        parameters = (parameters,)
    grads = [g for g in map(_grad_of, parameters) if g is not None]
    copies = []
    if not grads:
        return grads, None, copies, None
    _plain(who, *grads)
    try:
        types = set(map(_type_of, grads))
        codes = [_DTYPES[types.pop()]] * len(grads) if len(types) == 1 else [_DTYPES[g.dtype] for g in grads]
        at = list(map(_address, grads))
    except (KeyError, RuntimeError):  # sparse ones have no address
        raise TypeError(f"{who}: gradients must be dense float32, bfloat16 or float16 "
                        f"(got {', '.join(sorted({f'{g.layout}, {g.dtype}' for g in grads}))})") from None
    dev = grads[0].device
    if len(set(map(_Tensor.get_device, grads))) > 1:
        raise ValueError(f"{who}: the gradients must be on one device (got {', '.join(sorted({str(g.device) for g in grads}))})")
    _gpu(who, grads[0])
    if not all(map(_contiguous, grads)):
        for i, g in enumerate(grads):
            if not g.is_contiguous():
                if in_place and any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
                    raise ValueError(f"{who}: a gradient whose values share memory (strides {g.stride()}) cannot be scaled in place")
                if in_place and at.count(at[i]) > 1 and at[i]:
                    raise ValueError(f"{who}: two gradients share memory and cannot be scaled in place")
                grads[i] = g.contiguous()
                at[i] = grads[i].data_ptr()
                copies.append((g, grads[i]))
    if not all(at):  # empty ones, and zeros that autograd has not written; what stands for others without memory is refused
        for g in grads:
            if not g._is_zerotensor():
                _ptr(g)
        grads, at, codes = zip(*[x for x in zip(grads, at, codes) if x[1]]) if any(at) else ((), (), ())
    n = len(grads)
    return grads, (n, struct.pack(f"{n}q", *at), struct.pack(f"{n}q", *map(_size, grads)), struct.pack(f"{n}i", *codes)), copies, dev


def _norm_type(who, norm_type):
    if norm_type not in (2, math.inf):
        raise ValueError(f"{who}: norm_type must be 2 or inf (got {norm_type})")
    return norm_type != 2


def grad_norm(parameters, *, norm_type: float = 2.0):
    """The norm of the gradients of all parameters together, as if they were one vector: 2-norm, or (inf) the largest magnitude.

    parameters: a tensor or an iterable of them; those without a gradient count for nothing.  Gradients may be float32, bfloat16
    and float16 in one call, on one device.  Returns float32 on it, without waiting for it."""
    who = "grad_norm"
    largest = _norm_type(who, norm_type)
    grads, arrays, _, dev = _grads(who, parameters, False)
    if dev is None:
        return torch.zeros(())
    lib = _nat.lib()
    size = _bytes("boa_grad_norm_work_bytes", len(grads))
    norm, work = torch.empty((), dtype=torch.float32, device=dev), torch.empty(size, dtype=torch.uint8, device=dev)
    _call(norm, lib.boa_grad_norm, *arrays, largest, norm.data_ptr(), work.data_ptr(), size)
    return norm


def clip_grad_norm_(parameters, max_norm: float, *, norm_type: float = 2.0):
    """Scales the gradients of all parameters in place by ``min(1, max_norm / (norm + 1e-6))``, ``norm`` theirs together, between
    ``loss.backward()`` and the optimizer's step.  Returns the norm that they had (``grad_norm``).

    The call waits for nothing, so a norm that is no number makes the gradients so too (an infinite one makes them zeros, and NaN
    where they were infinite)."""
    who = "clip_grad_norm_"
    largest = _norm_type(who, norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{who}: max_norm must not be negative (got {max_norm})")
    grads, arrays, copies, dev = _grads(who, parameters, True)
    if dev is None:
        return torch.zeros(())
    lib = _nat.lib()
    size = _bytes("boa_grad_norm_work_bytes", len(grads))
    norm, work = torch.empty((), dtype=torch.float32, device=dev), torch.empty(size, dtype=torch.uint8, device=dev)
    _call(norm, lib.boa_clip_grads, *arrays, largest, max_norm, norm.data_ptr(), work.data_ptr(), size)
    if copies:
        with torch.no_grad():
            for g, scaled in copies:
                g.copy_(scaled)
    if grads:
        increment_version(grads)
    return norm


# ---- drawing symbols -------------------------------------------------------------------------------
def _limit(who, name, v, shape, like, dtype, lo, hi):
    """A limit of all rows as a number, or one of each row as a contiguous tensor: (number, tensor)."""
    if not isinstance(v, _Tensor):
        if not lo <= v <= hi:
            raise ValueError(f"{who}: {name} must be {lo} to {hi} (got {v})")
        return operator.index(v) if dtype is torch.int32 else float(v), None
    if v.dtype is not dtype:
        raise TypeError(f"{who}: {name} must be a number or a {dtype} tensor (got {v.dtype})")
    if v.shape != shape or v.get_device() != like.get_device():
        raise ValueError(f"{who}: {name} must be a number or {list(shape)} on {like.device} (got {list(v.shape)} on {v.device})")
    return 0, v.resolve_neg().contiguous()


def sample(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Symbols drawn from logits [..., V] (1 to 4096 symbols) by given random numbers u, float32 of the leading shape in [0, 1).

    The weights are exp((x - max) / temperature).  Of all symbols the top_k likeliest are kept (0: all), of those the fewest
    likeliest whose weights sum to top_p of theirs, of those the ones with at least min_p of the likeliest one's weight; equal
    logits count in the symbols' order.  Returns, int64 of the leading shape, the first symbol up to and with which the kept
    weights sum to more than u of them all: the same numbers draw the same symbols.  Temperature 0 takes the likeliest symbol.
    Each limit is a number, or a tensor of the leading shape (float32; top_k int32, where 0 or less keeps all).  A row that is no
    distribution (a NaN in it or its numbers, nothing above -inf) gives -1.  No gradient."""
    who = "sample"
    _plain(who, logits, u, temperature, top_p, min_p)
    _act(who, "logits", logits)
    if logits.ndim < 1 or not 1 <= logits.shape[-1] <= _nat.BOA_SAMPLE_MAX_V:
        raise ValueError(f"{who}: logits must be [..., V] with 1 <= V <= {_nat.BOA_SAMPLE_MAX_V} (got {list(logits.shape)})")
    shape = logits.shape[:-1]
    if not isinstance(u, _Tensor) or u.dtype is not _F32:
        raise TypeError(f"{who}: u must be a float32 tensor")
    if u.shape != shape or u.get_device() != logits.get_device():
        raise ValueError(f"{who}: u must be {list(shape)} on {logits.device} (got {list(u.shape)} on {u.device})")
    t, ts = _limit(who, "temperature", temperature, shape, logits, _F32, 0.0, math.inf)
    k, ks = _limit(who, "top_k", top_k, shape, logits, torch.int32, 0, 0x7FFFFFFF)
    p, ps = _limit(who, "top_p", top_p, shape, logits, _F32, 0.0, 1.0)
    m, ms = _limit(who, "min_p", min_p, shape, logits, _F32, 0.0, 1.0)
    _gpu(who, logits)
    v = logits.shape[-1]
    if v == 1:
        logits, = _written(logits)
    rows, stride, n = _flat(logits, v)
    u = u.resolve_neg().contiguous()
    out = torch.empty(shape, dtype=torch.int64, device=logits.device)
    _call(logits, _nat.lib().boa_sample, _DTYPES[logits.dtype], rows.data_ptr(), stride, n, v, _ptr(u), t, _ptr(ts), k, _ptr(ks), p,
          _ptr(ps), m, _ptr(ms), out.data_ptr())
    return out
