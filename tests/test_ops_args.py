"""Calls that the training operators refuse, in Python and at the C ABI, without a GPU."""
import os
import re
import subprocess

import pytest
import torch

from boa_amd import _native, ops
from conftest import REPO

BF = torch.bfloat16


def _scan_args(n=2, length=5, c=6, dtype=torch.float32):
    act = lambda *s: torch.zeros(s, dtype=dtype)  # noqa: E731
    return dict(u=act(n, length, c), delta=act(n, length, c), A=torch.zeros(c, 16), B=act(n, length, 16), C=act(n, length, 16),
                D=torch.zeros(c), z=act(n, length, c), delta_bias=torch.zeros(c))


def _step(args):
    return {k: v[:, 0] if k in ("u", "delta", "B", "C", "z") else v for k, v in args.items()}


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 5, 6)
    w = torch.zeros(6, 1, 4)
    for call in (lambda: ops.layer_norm(x), lambda: ops.cross_entropy(x, torch.zeros(2, 5, dtype=torch.int64)),
                 lambda: ops.causal_conv(x, w), lambda: ops.causal_conv_step(x[:, 0], torch.zeros(2, 3, 6), w),
                 lambda: ops.selective_scan(**_scan_args()),
                 lambda: ops.selective_scan_step(**_step(_scan_args()), state=torch.zeros(2, 16, 6))):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


@pytest.mark.parametrize("change,error", [
    (dict(u=torch.zeros(2, 5, 6, dtype=torch.float64)), TypeError),
    (dict(u=torch.zeros(2, 6)), ValueError),
    (dict(u=torch.zeros(2, 5, 0), delta=torch.zeros(2, 5, 0)), ValueError),
    (dict(delta=torch.zeros(2, 5, 7)), ValueError),
    (dict(delta=torch.zeros(2, 5, 6, dtype=BF)), ValueError),
    (dict(B=torch.zeros(2, 5, 8)), ValueError),
    (dict(C=torch.zeros(2, 4, 16)), ValueError),
    (dict(C=None), TypeError),
    (dict(A=torch.zeros(6, 8)), ValueError),
    (dict(A=torch.zeros(6, 16, dtype=BF)), TypeError),
    (dict(A=None), TypeError),
    (dict(D=torch.zeros(5)), ValueError),
    (dict(z=torch.zeros(1, 5, 6)), ValueError),
    (dict(delta_bias=torch.zeros(6, dtype=torch.float16)), TypeError),
    (dict(state=torch.zeros(2, 6, 16)), ValueError),
    (dict(state=torch.zeros(2, 16, 6, dtype=BF)), TypeError),
    (dict(state=torch.zeros(2, 16, 6, requires_grad=True)), ValueError),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(lens=torch.zeros(2)), TypeError),
    (dict(lens=[5, 5]), TypeError),
])
def test_scan_refusals(change, error):
    with pytest.raises(error):
        ops.selective_scan(**{**_scan_args(), **change})


@pytest.mark.parametrize("change,error", [
    (dict(state=None), TypeError),
    (dict(state=torch.zeros(2, 6, 16).transpose(1, 2)), ValueError),  # not contiguous: it could not be advanced in place
    (dict(state=torch.zeros(3, 16, 6)), ValueError),
    (dict(u=torch.zeros(2, 5, 6)), ValueError),
    (dict(u=torch.zeros(2, 6, requires_grad=True), state=torch.zeros(2, 16, 6)), ValueError),
])
def test_scan_step_refusals(change, error):
    with pytest.raises(error):
        ops.selective_scan_step(**{**_step(_scan_args()), "state": torch.zeros(2, 16, 6), **change})


@pytest.mark.parametrize("kw,error", [
    (dict(weight=torch.zeros(6, 1, 3)), ValueError),
    (dict(weight=torch.zeros(6, 4, dtype=BF)), TypeError),
    (dict(weight=None), TypeError),
    (dict(bias=torch.zeros(7)), ValueError),
    (dict(x=torch.zeros(2, 6)), ValueError),
    (dict(x=torch.zeros(2, 5, 6, dtype=torch.int32)), TypeError),
    (dict(state=torch.zeros(2, 4, 6)), ValueError),
    (dict(state=torch.zeros(2, 3, 6, dtype=BF)), TypeError),
    (dict(state=torch.zeros(2, 3, 6, requires_grad=True)), ValueError),
    (dict(lens=torch.zeros(2, 1, dtype=torch.int32)), ValueError),
])
def test_conv_refusals(kw, error):
    with pytest.raises(error):
        ops.causal_conv(**{**dict(x=torch.zeros(2, 5, 6), weight=torch.zeros(6, 1, 4)), **kw})


def test_conv_step_refusals():
    x, w, st = torch.zeros(2, 6), torch.zeros(6, 4), torch.zeros(2, 3, 6)
    for args, error in (((x, None, w), TypeError), ((x, st[:, :2], w), ValueError), ((x[None], st, w), ValueError),
                        ((x, torch.zeros(2, 6, 3).transpose(1, 2), w), ValueError), ((x, st, w.clone().requires_grad_()), ValueError)):
        with pytest.raises(error):
            ops.causal_conv_step(*args)


@pytest.mark.parametrize("kw,error", [
    (dict(x=torch.zeros(3, 4097)), ValueError), (dict(x=torch.zeros(3, 0)), ValueError), (dict(x=torch.zeros(())), ValueError),
    (dict(weight=torch.zeros(7)), ValueError), (dict(weight=torch.zeros(8, dtype=BF)), TypeError),
    (dict(bias=torch.zeros(8, 1)), ValueError), (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError),
    (dict(x=[1.0]), TypeError),
])
def test_norm_refusals(kw, error):
    with pytest.raises(error):
        ops.layer_norm(**{**dict(x=torch.zeros(3, 8)), **kw})


@pytest.mark.parametrize("kw,error", [
    (dict(logits=torch.zeros(3, 4097)), ValueError), (dict(logits=torch.zeros(3, 0)), ValueError),
    (dict(logits=torch.zeros(3, 8, dtype=torch.int32)), TypeError), (dict(targets=torch.zeros(3)), TypeError),
    (dict(targets=torch.zeros(3, dtype=torch.int16)), TypeError), (dict(targets=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(targets=[0, 1, 2]), TypeError), (dict(reduction="max"), ValueError),
])
def test_loss_refusals(kw, error):
    with pytest.raises(error):
        ops.cross_entropy(**{**dict(logits=torch.zeros(3, 8), targets=torch.zeros(3, dtype=torch.int64)), **kw})


def test_scan_struct_is_the_headers(tmp_path):
    """ops packs boa_scan by hand: its size and the places of its members as the C compiler lays them out."""
    order = ["u", "delta", "z", "b", "c", "a", "d", "delta_bias", "lens", "state_in", "state_out", "marks", "y", "dy", "du",
             "ddelta", "dz", "db", "dc", "dpar"]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "boa_hip.h"\nint main(void) { printf("%zu", sizeof(boa_scan));\n'
                   + "".join(f'printf(" %zu", offsetof(boa_scan, {m}));\n' for m in ["dtype", "channels", "batch", "length"] + order)
                   + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), "-o", str(tmp_path / "s"), str(src)], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()))
    at, want = 24, [0, 4, 8, 16]
    for m in order:
        want.append(at)
        at += 8 if m in ("a", "d", "delta_bias", "lens", "state_in", "state_out", "marks", "dpar") else 24
    assert got == [at] + want and ops._SCAN.size == at


def test_constants_are_the_headers():
    src = open(os.path.join(REPO, "include", "boa_hip.h")).read()
    for name in ("BOA_DT_F32", "BOA_DT_BF16", "BOA_DT_F16", "BOA_LAYER_NORM_MAX_D", "BOA_CROSS_ENTROPY_MAX_V",
                 "BOA_OPS_MAX_CHANNELS", "BOA_SCAN_MARK", "BOA_SCAN_MAX_ROW_STRIDE"):
        assert int(re.search(rf"#define {name} (\d+)", src).group(1)) == getattr(_native, name)


def _pack(dtype=0, c=64, n=2, length=8, p=4096, b_stride=128, back=True, dpar=4096):
    rows = (p, length * c, c)
    bc = (p, b_stride * length, b_stride)
    return ops._SCAN.pack(dtype, c, n, length, *rows, *rows, *rows, *bc, *bc, p, p, p, 0, 0, 0, p if back else 0, *rows,
                          *(rows * 4), *bc, *bc, dpar)


def test_c_abi_refuses_before_it_launches():
    """Arguments that no kernel may see end as BOA_ERR_ARG (the pointers here are never followed)."""
    L, bad = _native.load_cdll(), _native.BOA_ERR_ARG
    P = 4096
    fwd, bwd, step = L.boa_selective_scan_fwd, L.boa_selective_scan_bwd, L.boa_selective_scan_step
    assert fwd(None, None, 0, None) == bad
    for kw in (dict(dtype=3), dict(dtype=-1), dict(c=0), dict(c=65537), dict(n=-1), dict(length=-1), dict(p=0),
               dict(dtype=1, b_stride=33), dict(b_stride=1 << 26), dict(b_stride=-128), dict(dtype=2, p=4098), dict(n=1 << 40)):
        assert fwd(_pack(**kw), None, 0, None) == bad, kw
        assert step(_pack(**kw), None) == bad, kw
    assert step(_pack(), None) == bad  # more than one position
    need = L.boa_selective_scan_work_bytes(_pack(), 1)
    assert need > 0
    assert bwd(_pack(), P, need - 1, None) == bad and b"workspace" in L.boa_last_error()
    assert bwd(_pack(), None, need, None) == bad
    assert bwd(_pack(back=False), P, need, None) == bad  # no marks
    assert bwd(_pack(dpar=0), P, need, None) == bad
    for kw in (dict(dtype=3), dict(rows=-1), dict(d=0), dict(d=4097), dict(x=0)):
        a = {**dict(dtype=0, x=P, rows=4, d=8), **kw}
        assert L.boa_layer_norm_fwd(a["dtype"], a["x"], 8, P, P, a["rows"], a["d"], 1e-5, P, 8, P, None) == bad, kw
        assert L.boa_layer_norm_bwd(a["dtype"], P, 8, a["x"], 8, P, P, a["rows"], a["d"], P, 8, P, P, 1 << 30, None) == bad, kw
        assert L.boa_cross_entropy_fwd(a["dtype"], a["x"], 8, P, 8, -100, a["rows"], a["d"], 1, P, None, P, P, P, 1 << 20, None) == bad
        assert L.boa_cross_entropy_bwd(a["dtype"], a["x"], 8, P, 8, -100, a["rows"], a["d"], P, P, 0, P, P, 8, None) == bad
    assert L.boa_layer_norm_bwd(0, P, 8, P, 8, P, P, 4, 8, P, 8, P, P, 8, None) == bad  # workspace
    assert L.boa_cross_entropy_fwd(0, P, 8, P, 2, -100, 4, 8, 1, P, None, P, P, P, 1 << 20, None) == bad  # targets of 2 bytes
    assert L.boa_cross_entropy_fwd(0, P, 8, P, 8, -100, 4, 8, 1, P, None, P, P, P, 8, None) == bad  # workspace
    assert L.boa_cross_entropy_fwd(0, P, 8, P, 8, -100, 4, 8, 1, P, None, P, None, P, 1 << 20, None) == bad  # loss, no count
    conv = L.boa_causal_conv_fwd
    for kw in (dict(dtype=3), dict(n=-1), dict(length=-1), dict(c=0), dict(c=65537), dict(x=0)):
        a = {**dict(dtype=0, x=P, n=2, length=8, c=8), **kw}
        assert conv(a["dtype"], a["x"], 64, 8, P, P, 1, a["n"], a["length"], a["c"], None, None, None, P, 64, 8, None) == bad, kw
        assert L.boa_causal_conv_bwd(a["dtype"], P, 64, 8, a["x"], 64, 8, P, P, 1, a["n"], a["length"], a["c"], None, None, P, 64, 8,
                                     P, P, 1 << 30, None) == bad, kw
        if "length" not in kw:
            assert L.boa_causal_conv_step(a["dtype"], a["x"], 8, P, P, P, 1, a["n"], a["c"], P, 8, None) == bad, kw
    assert L.boa_causal_conv_bwd(0, P, 64, 8, P, 64, 8, P, P, 1, 2, 8, 8, None, None, P, 64, 8, P, P, 4, None) == bad  # workspace


def test_workspace_sizes():
    L = _native.load_cdll()
    assert L.boa_layer_norm_bwd_work_bytes(0, 8) == 0 and L.boa_layer_norm_bwd_work_bytes(1, 8) == 64
    assert L.boa_causal_conv_bwd_work_bytes(0, 5, 8) == 0 and L.boa_causal_conv_bwd_work_bytes(2, 0, 8) == 0
    assert L.boa_selective_scan_work_bytes(None, 1) == 0


def test_states_are_not_handed_on_in_place():
    """The forward passes of whole sequences read the state while its successor is written."""
    L, bad, P = _native.load_cdll(), _native.BOA_ERR_ARG, 4096
    packed = bytearray(_pack())
    for at in (24 + 5 * 24 + 4 * 8, 24 + 5 * 24 + 5 * 8):  # state_in, state_out
        packed[at:at + 8] = (P).to_bytes(8, "little")
    assert L.boa_selective_scan_fwd(bytes(packed), P, 1 << 30, None) == bad and b"another buffer" in L.boa_last_error()
    assert L.boa_causal_conv_fwd(0, P, 64, 8, P, P, 1, 2, 8, 8, None, P, P, P, 64, 8, None) == bad


def test_a_cache_for_every_block():
    from model import BoaConstrictor

    m = BoaConstrictor(d_model=256, num_layers=2, vocab_size=256, device="cpu")
    with pytest.raises(ValueError, match="2 blocks"):
        m.train_step(torch.zeros(3, dtype=torch.uint8), m.init_caches(3)[:1])
    with pytest.raises(ValueError, match="2 blocks"):
        m.train_forward(torch.zeros(3, 4, dtype=torch.uint8), caches=m.init_caches(3) * 2)


@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_far_rows_of_one_position(dtype):
    """A dimension of one keeps any stride through contiguous(); the kernels are given rows that are near all the same."""
    far = torch.zeros(2, 1, 16, dtype=dtype).as_strided((2, 1, 16), (16, 1 << 27, 1))
    for near in (ops._scan_rows(far), ops._scalar_rows(far)):
        assert near.stride() == (16, 16, 1) and near.shape == far.shape


def test_a_scan_of_no_positions_needs_its_parameters():
    """It hands on the state by the kernel that reads them."""
    L, bad, P = _native.load_cdll(), _native.BOA_ERR_ARG, 4096
    packed = bytearray(_pack(length=0))
    at_a, at_state_out = 24 + 5 * 24, 24 + 5 * 24 + 5 * 8
    packed[at_a:at_a + 8] = bytes(8)
    assert L.boa_selective_scan_fwd(bytes(packed), None, 0, None) == _native.BOA_OK  # no state wanted: nothing to do
    packed[at_state_out:at_state_out + 8] = P.to_bytes(8, "little")
    assert L.boa_selective_scan_fwd(bytes(packed), None, 0, None) == bad and b"null pointer" in L.boa_last_error()


def _put(packed, member, value, at=0):
    """`value` as the at-th 8 bytes of a member of boa_scan."""
    order = ["u", "delta", "z", "b", "c", "a", "d", "delta_bias", "lens", "state_in", "state_out", "marks", "y", "dy", "du",
             "ddelta", "dz", "db", "dc", "dpar"]
    pointers = ("a", "d", "delta_bias", "lens", "state_in", "state_out", "marks", "dpar")
    i = 24 + sum(8 if m in pointers else 24 for m in order[:order.index(member)]) + 8 * at
    packed[i:i + 8] = value.to_bytes(8, "little", signed=True)


@pytest.mark.parametrize("far", [-5, 1 << 40])
def test_members_that_a_call_does_not_use_are_ignored(far):
    """Row strides of a step, y of a backward pass, dz without z: each call goes on to the next refusal (and launches nothing)."""
    L, bad, P = _native.load_cdll(), _native.BOA_ERR_ARG, 4096
    packed = bytearray(_pack(dtype=1, length=1))
    for m in ("u", "delta", "z", "b", "c", "y"):
        _put(packed, m, far, 2)
    assert L.boa_selective_scan_step(bytes(packed), None) == bad and b"null pointer" in L.boa_last_error()  # no state
    packed = bytearray(_pack())
    _put(packed, "y", far, 2)
    assert L.boa_selective_scan_bwd(bytes(packed), P, 0, None) == bad and b"workspace" in L.boa_last_error()
    _put(packed, "dz", far, 2)
    assert L.boa_selective_scan_bwd(bytes(packed), P, 0, None) == bad and b"rows have to be" in L.boa_last_error()
    _put(packed, "z", 0)
    assert L.boa_selective_scan_bwd(bytes(packed), P, 0, None) == bad and b"workspace" in L.boa_last_error()
    packed = bytearray(_pack())
    _put(packed, "y", far, 2)  # the forward pass writes y
    assert L.boa_selective_scan_fwd(bytes(packed), P, 0, None) == bad and b"rows have to be" in L.boa_last_error()
