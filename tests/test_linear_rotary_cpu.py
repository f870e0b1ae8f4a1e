"""Linear attention and rotary positions without a GPU: the mirrors of the C structs, what is refused and how, the workspace sizes, and
the plan's numbers."""
import ctypes as C
import math
import os
import subprocess
import tempfile

import pytest
import torch
import torch.autograd.forward_ad as fwd

from acctransformer_b200 import _lib, build as _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MIRRORS = {"acct_linear_args": "LinearArgs", "acct_linear_bwd_io": "LinearBwdIO", "acct_linear_step_args": "LinearStepArgs", "acct_rotary_args": "RotaryArgs"}


@pytest.fixture(scope="module", autouse=True)
def _built():
    _build.build()


def test_struct_mirrors():
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "acct_b200.h"', "int main(void) {"]
    for st, mirror in MIRRORS.items():
        lines.append(f'printf("{st} %zu\\n", sizeof({st}));')
        lines += [f'printf("{st}.{name} %zu\\n", offsetof({st}, {name}));' for name, _ in getattr(_lib, mirror)._fields_]
    lines.append("return 0; }")
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        with open(src, "w") as f:
            f.write("\n".join(lines))
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        said = dict(x.rsplit(" ", 1) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines())
    for st, mirror in MIRRORS.items():
        cls = getattr(_lib, mirror)
        assert int(said[st]) == C.sizeof(cls), st
        for name, _ in cls._fields_:
            assert int(said[f"{st}.{name}"]) == getattr(cls, name).offset, (st, name)


def _args(**more):
    a = _lib.LinearArgs()
    a.dtype, a.B, a.N, a.S, a.D = _lib.ACCT_BF16, 2, 4, 256, 64
    a.q = a.k = a.v = a.y = a.log_decay = 4096
    a.scale = 1.0
    for name, value in more.items():
        if isinstance(value, tuple):
            for i, x in enumerate(value):
                getattr(a, name)[i] = x
        else:
            setattr(a, name, value)
    return a


REFUSED = [
    (dict(dtype=_lib.ACCT_F32), 3), (dict(B=0), 2), (dict(N=-1), 2), (dict(S=0), 2), (dict(N_kv=3), 2), (dict(D=60), 4), (dict(D=136), 4), (dict(D=0), 4),
    (dict(log_decay=None), 1), (dict(q=None), 1), (dict(k=4104), 5), (dict(q_stride=(0, 0, 68)), 5), (dict(v_stride=(0, 0, 32)), 2),
    (dict(cu_seqlens=4096, seq_lens=4096), 2), (dict(scale=math.inf), 2), (dict(scale=math.nan), 2), (dict(B=1 << 20, N=64), 2)]


@pytest.mark.parametrize("change,code", REFUSED, ids=[str(c) for c, _ in REFUSED])
def test_abi_refuses(change, code):
    lib = _lib.load()
    assert lib.acct_linear_fwd(C.byref(_args(**change)), None) == code, lib.acct_last_error()
    io = _lib.LinearBwdIO()
    io.d_y = io.dq = io.dk = io.dv = 4096
    assert lib.acct_linear_bwd(C.byref(_args(**change)), C.byref(io), None) == code, lib.acct_last_error()


def test_abi_refuses_more():
    lib = _lib.load()
    assert lib.acct_linear_fwd(None, None) == 1
    assert lib.acct_linear_fwd(C.byref(_args(y=None)), None) == 1
    assert lib.acct_linear_fwd(C.byref(_args(state_out=4100)), None) == 5
    io = _lib.LinearBwdIO()
    assert lib.acct_linear_bwd(C.byref(_args()), C.byref(io), None) == 1
    io.d_y = io.dq = io.dk = io.dv = 4096
    assert lib.acct_linear_bwd(C.byref(_args(cu_seqlens=4096)), C.byref(io), None) == 2
    assert lib.acct_linear_bwd(C.byref(_args(state_out=4096)), C.byref(io), None) == 2
    shared = _args(N_kv=2)
    need = lib.acct_linear_bwd_workspace_bytes(C.byref(shared))
    assert need >= 2 * 2 * 4 * 256 * 64 * 4
    assert lib.acct_linear_bwd(C.byref(shared), C.byref(io), None) == 6
    io.workspace, io.workspace_bytes = 4096 + 16, need
    assert lib.acct_linear_bwd(C.byref(shared), C.byref(io), None) == 5
    long = _args(B=1, N=1, S=8192)      # segments: their states
    need = lib.acct_linear_fwd_workspace_bytes(C.byref(long))
    assert need > 0 and need % (64 * 64 * 4) == 0
    assert lib.acct_linear_fwd(C.byref(long), None) == 6


def test_abi_step_and_rotary_refuse():
    lib = _lib.load()
    s = _lib.LinearStepArgs()
    s.dtype, s.B, s.N, s.D, s.scale = _lib.ACCT_F16, 2, 4, 64, 1.0
    assert lib.acct_linear_step(None, None) == 1
    assert lib.acct_linear_step(C.byref(s), None) == 1
    s.q = s.k = s.v = s.y = s.state = s.log_decay = 4096
    for name, value, code in (("dtype", 7, 3), ("B", 0, 2), ("N_kv", 3, 2), ("D", 12, 4), ("D", 256, 4), ("state", 4104, 5)):
        old = getattr(s, name)
        setattr(s, name, value)
        assert lib.acct_linear_step(C.byref(s), None) == code, name
        setattr(s, name, old)
    r = _lib.RotaryArgs()
    r.dtype, r.B, r.S, r.D, r.N, r.N_kv, r.rotated = _lib.ACCT_F16, 1, 8, 64, 2, 2, 64
    assert lib.acct_rotary(None, None) == 1
    assert lib.acct_rotary(C.byref(r), None) == 1
    r.q = r.k = r.q_out = r.k_out = r.positions = r.turns = r.axis = 4096
    for name, value, code in (("dtype", 2, 3), ("S", -1, 2), ("D", 264, 4), ("D", 20, 4), ("rotated", 0, 2), ("rotated", 33, 2), ("rotated", 66, 2), ("k", 4098, 5),
                              ("S", 2 ** 31 - 1, 2)):
        old = getattr(r, name)
        setattr(r, name, value)
        assert lib.acct_rotary(C.byref(r), None) == code, (name, value)
        setattr(r, name, old)


def _half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


def _calls():
    from acctransformer_b200 import linear_attention_packed, linear_attention_step
    g, cu, state = torch.zeros(4), torch.tensor([0, 4], dtype=torch.int32), torch.zeros(1, 4, 64, 64)
    out = {}
    for i, name in enumerate("qkv"):
        def packed(x, i=i):
            rows = [_half(4, 4, 64), _half(4, 2, 64), _half(4, 2, 64)]
            rows[i] = x(rows[i])
            linear_attention_packed(*rows, g, cu)

        def step(x, i=i):
            rows = [_half(1, 4, 1, 64), _half(1, 2, 1, 64), _half(1, 2, 1, 64)]
            rows[i] = x(rows[i])
            linear_attention_step(*rows, g, state)
        out[f"packed {name}"], out[f"step {name}"] = packed, step
    out["packed state"] = lambda x: linear_attention_packed(_half(4, 4, 64), _half(4, 2, 64), _half(4, 2, 64), g, cu, state=x(state.clone()))
    out["step state"] = lambda x: linear_attention_step(_half(1, 4, 1, 64), _half(1, 2, 1, 64), _half(1, 2, 1, 64), g, x(state.clone()))
    return out


@pytest.mark.parametrize("call", ["packed q", "packed k", "packed v", "packed state", "step q", "step k", "step v", "step state"])
def test_serving_refuses_gradients(call):
    call = _calls()[call]
    with pytest.raises(ValueError, match="has no gradient"):
        call(lambda t: t.requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        call(lambda t: t.requires_grad_())
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        call(lambda t: fwd.make_dual(t, torch.ones_like(t)))


def test_python_refuses():
    from acctransformer_b200 import LinearAttention, Rotary, linear_attention
    with pytest.raises(ValueError, match="CUDA"):
        linear_attention(_half(1, 4, 8, 64), _half(1, 4, 8, 64), _half(1, 4, 8, 64), torch.zeros(4))
    with pytest.raises(ValueError, match="CUDA"):
        linear_attention(3, None, None, None)
    for bad in (dict(head_dim=60), dict(head_dim=264), dict(head_dim=64, sections=(40,)), dict(head_dim=64, sections=(-1, 3)), dict(head_dim=64, sections=()),
                dict(head_dim=64, base=0.0), dict(head_dim=64, frequencies=[1.0]), dict(head_dim=64, sections=(1,), frequencies=[math.inf])):
        with pytest.raises(ValueError):
            Rotary(**bad, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        Rotary(64, device="cpu")
    for bad in (dict(log_decay=[0.1, 0.0]), dict(log_decay=[-1.0]), dict(log_decay=[-1.0, math.nan])):
        with pytest.raises(ValueError):
            LinearAttention(2, 64, **bad)
    with pytest.raises(ValueError, match="positions"):
        LinearAttention(2, 64)(_half(1, 2, 4, 64), _half(1, 2, 4, 64), _half(1, 2, 4, 64), positions=torch.zeros(1, 4))


def test_default_decays():
    from acctransformer_b200.linear import default_log_decay
    assert torch.allclose(default_log_decay(8), -(2.0 ** -torch.arange(1.0, 9.0)))
