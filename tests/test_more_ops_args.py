"""Calls of linear attention, gradient clipping and sampling that are refused, in Python and at the C ABI, without a GPU."""
import array
import ctypes
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from boa_amd import _native, ops
from test_ops_storage import Wrapper

BF = torch.bfloat16


def _attention(n=2, length=5, heads=4, groups=2, key=6, value=3, dtype=torch.float32):
    z = lambda *s: torch.zeros(s, dtype=dtype)  # noqa: E731
    return dict(q=z(n, length, groups, key), k=z(n, length, groups, key), v=z(n, length, heads, value), log_decay=torch.zeros(n, length, heads))


def _step(args, state=True):
    out = {k: t[:, 0] for k, t in args.items()}
    return {**out, "state": torch.zeros(2, 4, 6, 3)} if state else out


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 5, 2, 6, dtype=torch.float64)), TypeError),
    (dict(q=torch.zeros(2, 5, 12)), ValueError),
    (dict(q=torch.zeros(2, 5, 0, 6), k=torch.zeros(2, 5, 0, 6)), ValueError),
    (dict(q=torch.zeros(2, 5, 2, 0), k=torch.zeros(2, 5, 2, 0)), ValueError),
    (dict(q=torch.zeros(2, 5, 2, 129), k=torch.zeros(2, 5, 2, 129)), ValueError),
    (dict(q=torch.zeros(2, 5, 3, 6), k=torch.zeros(2, 5, 3, 6)), ValueError),  # 4 heads cannot share 3
    (dict(k=torch.zeros(2, 5, 4, 6)), ValueError),
    (dict(k=torch.zeros(2, 5, 2, 6, dtype=BF)), ValueError),
    (dict(k=None), TypeError),
    (dict(v=torch.zeros(2, 4, 4, 3)), ValueError),
    (dict(v=torch.zeros(2, 5, 4, 513)), ValueError),
    (dict(v=torch.zeros(2, 5, 0, 3)), ValueError),
    (dict(v=torch.zeros(2, 5, 4, 0)), ValueError),
    (dict(log_decay=torch.zeros(2)), ValueError),
    (dict(log_decay=torch.zeros(2, 5, 4, dtype=BF)), TypeError),
    (dict(log_decay=-0.5), TypeError),
    (dict(state=torch.zeros(2, 4, 3, 6)), ValueError),
    (dict(state=torch.zeros(2, 4, 6, 3, dtype=BF)), TypeError),
    (dict(state=torch.zeros(2, 4, 6, 3, requires_grad=True)), ValueError),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(lens=torch.zeros(2)), TypeError),
    (dict(), ValueError),  # on the CPU
])
def test_attention_refusals(change, error):
    with pytest.raises(error):
        ops.linear_attention(**{**_attention(), **change})


@pytest.mark.parametrize("change,error", [
    (dict(state=None), TypeError),
    (dict(state=torch.zeros(2, 4, 3, 6).transpose(2, 3)), ValueError),
    (dict(state=torch.zeros(3, 4, 6, 3)), ValueError),
    (dict(q=torch.zeros(2, 1, 2, 6)), ValueError),
    (dict(log_decay=torch.zeros(2, 1, 4)), ValueError),
    (dict(v=torch.zeros(2, 4, 3, requires_grad=True)), ValueError),
    (dict(), ValueError),
])
def test_attention_step_refusals(change, error):
    with pytest.raises(error):
        ops.linear_attention_step(**{**_step(_attention()), **change})


@pytest.mark.parametrize("kw,error", [
    (dict(logits=torch.zeros(2, 256, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(2, 4097)), ValueError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(u=torch.zeros(3)), ValueError),
    (dict(u=torch.zeros(2, dtype=torch.float64)), TypeError),
    (dict(u=0.5), TypeError),
    (dict(temperature=-0.1), ValueError),
    (dict(temperature=math.nan), ValueError),
    (dict(temperature=torch.ones(2, dtype=torch.float64)), TypeError),
    (dict(top_k=-1), ValueError),
    (dict(top_k=torch.ones(2, dtype=torch.int64)), TypeError),
    (dict(top_k=torch.ones(1, dtype=torch.int32)), ValueError),
    (dict(top_p=1.5), ValueError),
    (dict(top_p=-0.1), ValueError),
    (dict(min_p=1.5), ValueError),
    (dict(min_p=math.nan), ValueError),
    (dict(), ValueError),
])
def test_sample_refusals(kw, error):
    with pytest.raises(error):
        ops.sample(**{**dict(logits=torch.zeros(2, 256), u=torch.zeros(2)), **kw})


def _with_grad(g):
    p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype))
    p.grad = g
    return p


@pytest.mark.parametrize("params,kw,error", [
    ([_with_grad(torch.zeros(3, dtype=torch.float64))], {}, TypeError),
    ([_with_grad(torch.zeros(3, dtype=torch.complex64))], {}, TypeError),
    ([_with_grad(torch.zeros(3))], dict(norm_type=1.0), ValueError),
    ([_with_grad(torch.zeros(3))], {}, ValueError),  # on the CPU
])
def test_grad_norm_refusals(params, kw, error):
    with pytest.raises(error):
        ops.grad_norm(params, **kw)
    with pytest.raises(error):
        ops.clip_grad_norm_(params, 1.0, **kw)


def test_clipping_refuses_a_limit_that_is_none():
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            ops.clip_grad_norm_([], bad)
    sparse = torch.nn.Parameter(torch.zeros(3, 2))
    sparse.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 2), (3, 2))
    with pytest.raises(TypeError, match="dense"):
        ops.grad_norm([sparse])


CALLS = {
    "linear_attention": (ops.linear_attention, lambda: dict(_attention(), state=torch.zeros(2, 4, 6, 3))),
    "linear_attention_step": (ops.linear_attention_step, lambda: _step(_attention())),
    "sample": (ops.sample, lambda: dict(logits=torch.zeros(2, 256), u=torch.zeros(2))),
}


@pytest.mark.parametrize("call", CALLS)
def test_tangents_and_tracers_are_refused(call):
    f, make = CALLS[call]
    for name in make():
        args = make()
        with forward_ad.dual_level():
            args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(**args)
    args = make()
    g = lambda *ts: f(**dict(zip(args, ts)))  # noqa: E731
    for trace in (lambda: torch.jit.trace(g, tuple(args.values())), lambda: make_fx(g)(*args.values())):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            trace()


def test_tensors_without_memory_are_not_taken_for_absent_ones(monkeypatch):
    calls = []
    import types

    lib = types.SimpleNamespace(boa_linear_attention_work_bytes=lambda *a: 0, boa_linear_attention_fwd="f", boa_sample="s",
                                boa_grad_norm="n", boa_grad_norm_work_bytes=lambda n: 8)
    monkeypatch.setattr(ops, "_gpu", lambda *a: None)
    monkeypatch.setattr(ops._nat, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_call", lambda *a: calls.append(a))
    args = dict(_attention(), state=torch.zeros(2, 4, 6, 3), lens=torch.zeros(2, dtype=torch.int32))
    ops.linear_attention(**args)
    for name in ("state", "lens"):
        with pytest.raises(ValueError, match="without memory"):
            ops.linear_attention(**{**args, name: Wrapper(args[name])})
    args = dict(logits=torch.zeros(2, 256), u=torch.zeros(2), temperature=torch.ones(2), top_k=torch.ones(2, dtype=torch.int32), top_p=torch.ones(2),
                min_p=torch.ones(2))
    ops.sample(**args)
    for name in list(args)[1:]:
        with pytest.raises((ValueError, NotImplementedError)):
            ops.sample(**{**args, name: Wrapper(args[name])})
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    ops.grad_norm([p])
    assert len(calls) == 3


# ---- the C ABI: every refusal comes before any launch ------------------------------------------------
def _packed(dtype=0, heads=4, groups=2, key=6, value=3, n=2, length=5, p=16, decay=16, state_out=0, ddecay=16, marks=16):
    rows = (p, 1, 1, 1)
    return ops._ATTENTION.pack(dtype, heads, groups, key, value, 0, 1.0, 0, n, length, *(rows * 4), decay, 1, 1, 1, 0, 0, state_out, marks, *(rows * 4), ddecay)


def test_the_struct_has_the_headers_size():
    assert ops._ATTENTION.size == 6 * 4 + 8 + 16 + 4 * 32 + 8 + 24 + 32 + 4 * 32 + 8


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(heads=0), dict(groups=0), dict(groups=3), dict(heads=8192, groups=2), dict(key=0), dict(key=129),
                                dict(value=0), dict(value=513), dict(n=-1), dict(length=-1), dict(n=1 << 40), dict(length=1 << 50)])
def test_c_attention_sizes(kw):
    lib = _native.load_cdll()
    s = _packed(**kw)
    assert lib.boa_linear_attention_work_bytes(s, 0) == -1 and lib.boa_linear_attention_work_bytes(s, 1) == -1
    big = ctypes.c_void_p(16)
    assert lib.boa_linear_attention_fwd(s, big, 1 << 62, None) == _native.BOA_ERR_ARG
    assert lib.boa_linear_attention_bwd(s, big, 1 << 62, None) == _native.BOA_ERR_ARG
    assert lib.boa_linear_attention_step(s, None) == _native.BOA_ERR_ARG


def test_c_attention_pointers_and_workspaces():
    lib = _native.load_cdll()
    big, odd = ctypes.c_void_p(16), ctypes.c_void_p(24)
    s = _packed(n=1, length=200)
    need, back = lib.boa_linear_attention_work_bytes(s, 0), lib.boa_linear_attention_work_bytes(s, 1)
    assert 0 < need < back
    assert lib.boa_linear_attention_bwd(_packed(marks=0), big, 1 << 62, None) == _native.BOA_ERR_ARG
    assert lib.boa_linear_attention_marks_bytes(_packed(n=1, length=200)) == 4 * 4 * 4 * 64 * 64
    assert lib.boa_linear_attention_marks_bytes(_packed(dtype=3)) == -1
    for bad in (_packed(p=0), _packed(decay=0), _packed(marks=8)):
        assert lib.boa_linear_attention_fwd(bad, big, 1 << 62, None) == _native.BOA_ERR_ARG
        assert lib.boa_linear_attention_bwd(bad, big, 1 << 62, None) == _native.BOA_ERR_ARG
    assert lib.boa_linear_attention_bwd(_packed(ddecay=0), big, 1 << 62, None) == _native.BOA_ERR_ARG
    for work, size in ((None, need), (big, need - 1), (odd, need)):
        assert lib.boa_linear_attention_fwd(s, work, size, None) == _native.BOA_ERR_ARG
    for work, size in ((None, back), (big, back - 1), (odd, back)):
        assert lib.boa_linear_attention_bwd(s, work, size, None) == _native.BOA_ERR_ARG
    assert lib.boa_linear_attention_step(_packed(length=2, state_out=16), None) == _native.BOA_ERR_ARG
    assert lib.boa_linear_attention_step(_packed(length=1), None) == _native.BOA_ERR_ARG
    assert lib.boa_linear_attention_fwd(None, big, 0, None) == _native.BOA_ERR_ARG
    assert lib.boa_linear_attention_step(_packed(n=0, length=1), None) == _native.BOA_OK


def test_c_gradients():
    lib = _native.load_cdll()
    work, norm = ctypes.c_void_p(16), ctypes.c_void_p(16)
    size = lib.boa_grad_norm_work_bytes(2)

    def both(p, n, d, count=2, work=work, size=size, norm=norm):
        a = (array.array("q", p).tobytes(), array.array("q", n).tobytes(), array.array("i", d).tobytes())
        return {lib.boa_grad_norm(count, *a, 0, norm, work, size, None), lib.boa_clip_grads(count, *a, 0, 1.0, norm, work, size, None)}

    refused = {_native.BOA_ERR_ARG}
    assert both([64, 256], [4, 4], [0, 3]) == refused
    assert both([64, 256], [4, -1], [0, 0]) == refused
    assert both([64, 256], [4, (1 << 40) + 1], [0, 0]) == refused
    assert both([64, 0], [4, 4], [0, 0]) == refused
    assert both([64, 258], [4, 4], [0, 0]) == refused
    assert both([64, 257], [4, 4], [0, 1]) == refused
    assert both([64, 256], [4, 4], [0, 0], count=-1) == refused
    assert both([64, 256], [4, 4], [0, 0], work=None) == refused
    assert both([64, 256], [4, 4], [0, 0], size=size - 1) == refused
    assert both([64, 256], [4, 4], [0, 0], work=ctypes.c_void_p(20)) == refused
    assert both([64, 256], [4, 4], [0, 0], norm=None) == refused
    a = (array.array("q", [64, 76]).tobytes(), array.array("q", [4, 4]).tobytes(), array.array("i", [0, 0]).tobytes())
    assert lib.boa_clip_grads(2, *a, 0, 1.0, norm, work, size, None) == _native.BOA_ERR_ARG  # four bytes of both
    for bad in (-1.0, math.nan):
        assert lib.boa_clip_grads(1, *a, 0, bad, norm, work, size, None) == _native.BOA_ERR_ARG
    assert lib.boa_grad_norm(1, None, None, None, 0, norm, work, size, None) == _native.BOA_ERR_ARG


def test_c_sample():
    lib = _native.load_cdll()
    p = ctypes.c_void_p(16)

    def call(dtype=0, x=p, rows=2, v=256, u=p, t=1.0, k=0, top_p=1.0, min_p=0.0, out=p):
        return lib.boa_sample(dtype, x, v, rows, v, u, t, None, k, None, top_p, None, min_p, None, out, None)

    for kw in (dict(dtype=3), dict(rows=-1), dict(v=0), dict(v=4097), dict(x=None), dict(u=None), dict(out=None), dict(t=-1.0), dict(t=math.nan),
               dict(top_p=-0.1), dict(top_p=math.nan), dict(min_p=-0.1), dict(min_p=math.nan)):
        assert call(**kw) == _native.BOA_ERR_ARG, kw
    assert call(rows=0) == _native.BOA_OK


def test_limits_agree_with_the_header():
    import os
    import re

    from conftest import REPO

    text = open(os.path.join(REPO, "include", "boa_hip.h")).read()
    for name in ("BOA_ATTENTION_MAX_KEY", "BOA_ATTENTION_MAX_VALUE", "BOA_ATTENTION_MAX_HEADS", "BOA_SAMPLE_MAX_V"):
        assert int(re.search(rf"#define {name} (\d+)", text).group(1)) == getattr(_native, name)


def test_generate_refuses():
    import model

    m = model.BoaConstrictor(256, 1)
    x = torch.zeros(2, 3, dtype=torch.uint8)
    for args, kw in (((x[0], 4), {}), ((x[:, :0], 4), {}), ((x, -1), {}), ((x, 4), dict(u=torch.zeros(2, 4)))):
        with pytest.raises(ValueError):
            m.generate(*args, **kw)
    with pytest.raises(ValueError, match="on the GPU"):
        m.generate(x, 4)


def test_limits_are_numbers_of_their_kind():
    like, shape = torch.zeros(2, 256), (2,)
    for v in (5.0, np.float32(5), "5"):
        with pytest.raises(TypeError):
            ops._limit("sample", "top_k", v, shape, like, torch.int32, 0, 9)
    for v in (np.int64(5), np.uint8(5), 5):
        got, none = ops._limit("sample", "top_k", v, shape, like, torch.int32, 0, 9)
        assert type(got) is int and got == 5 and none is None
    for v in (np.float32(0.5), np.float64(0.5), 0.5):
        got, none = ops._limit("sample", "top_p", v, shape, like, torch.float32, 0.0, 1.0)
        assert type(got) is float and got == 0.5 and none is None
    for name in ("temperature", "top_p", "min_p"):
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            ops.sample(like, torch.zeros(2), **{name: forward_ad.make_dual(torch.ones(2), torch.ones(2))})


def test_c_tensors_longer_than_any_memory():
    lib = _native.load_cdll()
    work, norm = ctypes.c_void_p(16), ctypes.c_void_p(16)
    for dtype, n in ((0, (1 << 37) + 1), (1, (1 << 38) + 1), (2, (1 << 38) + 1)):
        a = (array.array("q", [64]).tobytes(), array.array("q", [n]).tobytes(), array.array("i", [dtype]).tobytes())
        size = lib.boa_grad_norm_work_bytes(1)
        assert lib.boa_grad_norm(1, *a, 0, norm, work, size, None) == _native.BOA_ERR_ARG
        assert lib.boa_clip_grads(1, *a, 0, 1.0, norm, work, size, None) == _native.BOA_ERR_ARG


def test_more_sequences_than_a_launch_takes_are_named(monkeypatch):
    monkeypatch.setattr(_native, "_lib", _native.load_cdll())
    with pytest.raises(ValueError, match="too many for a launch"):
        ops._attention_work(_native._lib, _packed(n=1 << 40), 0)
