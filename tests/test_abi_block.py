"""The C entries of the unquantised operators refuse bad arguments on the host
(every call here returns before any HIP call), and their argument blocks have
the header's layout."""
import ctypes
import os
import subprocess

import pytest
import torch

import smoe
from smoe import _C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE, MIS = 0x100000, 0x100001  # never dereferenced


def test_tokens_reject():
    lib = _C.lib()
    p = lambda x=FAKE, ld=64, inv=FAKE, w=None, T=4, K=2, H=64, dt=0, xp=FAKE: lib.smoe_permute_tokens(
        x, ld, inv, w, T, K, H, dt, xp, None)
    assert p(x=None) == -1 and p(inv=None) == -1 and p(xp=None) == -1
    assert p(T=0) == -2 and p(H=0) == -2 and p(ld=-1) == -2 and p(T=1 << 30, K=4) == -2
    assert p(K=0) == -7 and p(K=33) == -7 and p(dt=3) == -8 and p(dt=-1) == -8
    assert p(x=MIS) == -6 and p(xp=MIS) == -6 and p(inv=FAKE + 2) == -6 and p(w=FAKE + 2) == -6
    assert p(x=FAKE + 2, dt=2) == -6
    assert p(T=1 << 30, K=1, H=1) == -2  # more workgroups than a grid holds
    need = lib.smoe_route_sort_workspace_size(4, 2, 8)
    q = lambda idx=FAKE, T=4, K=2, E=8, rm=FAKE, xp=FAKE, ws=FAKE, nb=need, ld=64: lib.smoe_sort_permute_tokens(
        FAKE, ld, idx, None, T, K, E, 64, 0, rm, FAKE, FAKE, FAKE, xp, ws, nb, None)
    assert q(idx=None) == -1 and q(rm=None) == -1 and q(xp=None) == -1 and q(ws=None) == -5 and q(nb=need - 1) == -5
    assert q(E=0) == -4 and q(E=1025) == -4 and q(E=1) == -7 and q(T=0) == -2 and q(ld=-1) == -2 and q(ws=FAKE + 8) == -6
    assert q(T=2000, idx=None, nb=1 << 30) == -1 and q(T=2000, nb=4) == -5
    b = lambda g=FAKE, x=FAKE, dx=FAKE, dw=FAKE, T=4: lib.smoe_permute_tokens_bwd(
        g, 64, x, 64, FAKE, FAKE, T, 2, 64, 0, dx, dw, None)
    assert b(g=None) == -1 and b(x=None) == -1 and b(dx=None) == -1 and b(T=-1) == -2 and b(dw=FAKE + 2) == -6
    assert lib.smoe_unpermute_tokens(None, 64, FAKE, None, 4, 2, 64, 0, FAKE, None) == -1
    u = lambda g=FAKE, y=FAKE, dy=FAKE, dw=FAKE, ld=64: lib.smoe_unpermute_tokens_bwd(
        g, ld, y, 64, FAKE, FAKE, 4, 2, 64, 0, dy, dw, None)
    assert u(g=None) == -1 and u(y=None) == -1 and u(dy=None) == -1 and u(ld=-3) == -2 and u(dw=FAKE + 1) == -6


def test_norms_reject():
    lib = _C.lib()
    n = lambda x=FAKE, ld=64, w=FAKE, pf=0, eps=1e-6, T=4, H=64, dt=0, h=FAKE, r=FAKE: lib.smoe_block_norm_in(
        x, ld, w, pf, eps, T, H, dt, h, r, None)
    assert n(x=None) == -1 and n(h=None) == -1 and n(r=None) == -1
    assert n(T=0) == -2 and n(H=0) == -2 and n(H=65537) == -2 and n(eps=0.0) == -2 and n(eps=float("nan")) == -2
    assert n(ld=-1) == -2 and n(dt=3) == -8 and n(pf=4) == -8 and n(w=FAKE + 2, pf=1) == -6 and n(r=FAKE + 2) == -6
    o = lambda mode=1, gate=FAKE, pf=0, ldg=1, x=FAKE: lib.smoe_block_norm_out(
        FAKE, 64, x, 64, FAKE, gate, ldg, mode, pf, 1.0, 1e-6, 4, 64, 0, FAKE, FAKE, None)
    assert o(mode=4) == -8 and o(mode=-1) == -8 and o(gate=None) == -1 and o(gate=FAKE + 2, pf=2) == -6
    assert o(ldg=-1) == -2 and o(x=None) == -1
    need = lib.smoe_block_norm_bwd_workspace_size(4, 64)
    assert need >= 64 * 4 and lib.smoe_block_norm_bwd_workspace_size(0, 64) == 0
    b = lambda ws=FAKE, nb=need, dw=FAKE, sk=None, r=FAKE: lib.smoe_block_norm_in_bwd(
        FAKE, 64, FAKE, 64, r, FAKE, 0, sk, 64, 1.0, 4, 64, 0, FAKE, dw, ws, nb, None)
    assert b(ws=None) == -5 and b(nb=need - 1) == -5 and b(ws=FAKE + 4) == -6 and b(sk=MIS) == -6 and b(r=None) == -1
    g = lambda gate=FAKE, dg=FAKE, mode=1, ws=FAKE: lib.smoe_block_norm_out_bwd(
        FAKE, 64, FAKE, 64, FAKE, FAKE, gate, 1, mode, 0, 4, 64, 0, FAKE, None, dg, ws, need, None)
    assert g(gate=None) == -1 and g(dg=None) == -1 and g(ws=None) == -5 and g(mode=9) == -8


def fwd(**kw):
    a = dict(R=4, N=32, K=64, E=1, act=0, dtype=0, bias_f32=0, x=FAKE, ldx=64, w=FAKE, bias=None, residual=None,
             ldr=0, offsets=None, out=FAKE, z=None, ws=None, ws_bytes=0)
    a.update(kw)
    return _C.lib().smoe_linear_act(ctypes.byref(_C.LinearFwd(**a)), None)


def bwd(**kw):
    a = dict(R=4, N=32, K=64, E=1, act=2, dtype=0, bias_f32=0, dw_mode=2, dout=FAKE, lddout=32, x=FAKE, ldx=64,
             w=FAKE, z=FAKE, offsets=None, dx=FAKE, dw=FAKE, dbias=None, ws=FAKE, ws_bytes=1 << 20)
    a.update(kw)
    return _C.lib().smoe_linear_act_bwd(ctypes.byref(_C.LinearBwd(**a)), None)


def test_linear_rejects():
    assert _C.lib().smoe_linear_act(None, None) == -1 and _C.lib().smoe_linear_act_bwd(None, None) == -1
    for f in (fwd, bwd):
        assert f(R=0) == -2 and f(N=0) == -2 and f(K=-1) == -2 and f(N=(1 << 20) + 2) == -2 and f(R=1 << 30) == -2
        assert f(E=0) == -4 and f(E=1025, offsets=FAKE) == -4 and f(E=2) == -1 and f(offsets=FAKE + 2) == -6
        assert f(act=6) == -8 and f(act=-1) == -8 and f(dtype=2) == -8 and f(act=5, N=33) == -2
        assert f(x=MIS) == -6 and f(w=MIS) == -6 and f(ldx=-1) == -2
    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(out=None) == -1 and fwd(ldr=-1) == -2
    assert fwd(bias=FAKE + 2, bias_f32=1) == -6 and fwd(residual=MIS) == -6 and fwd(z=MIS) == -6
    assert bwd(dout=None) == -1 and bwd(z=None) == -1 and bwd(x=None) == -1 and bwd(w=None) == -1
    assert bwd(dw_mode=4) == -8 and bwd(dw_mode=-1) == -8 and bwd(dw=FAKE + 2, dw_mode=0) == -6
    assert bwd(ws=None) == -5 and bwd(ws_bytes=8) == -5 and bwd(ws=FAKE + 4) == -6 and bwd(lddout=-1) == -2


def test_argument_blocks_match_the_header(tmp_path):
    """Sizes and offsets of the ctypes structures and of the C structs."""
    src = tmp_path / "s.c"
    lines = []
    for c, name in ((_C.LinearFwd, "smoe_linear_fwd"), (_C.LinearBwd, "smoe_linear_bwd")):
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in c._fields_]
    src.write_text(f'#include <stdio.h>\n#include "{ROOT}/include/smoe.h"\nint main(void) {{ {" ".join(lines)} }}\n')
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for c in (_C.LinearFwd, _C.LinearBwd):
        want += [ctypes.sizeof(c)] + [getattr(c, f[0]).offset for f in c._fields_]
    assert got == want


@pytest.mark.parametrize("call", [
    lambda x, i: smoe.permute_tokens_rows(x, i, 1), lambda x, i: smoe.unpermute_tokens(x, i, 1),
    lambda x, i: smoe.block_norm_in(x), lambda x, i: smoe.block_norm_out(x, x), lambda x, i: smoe.linear_act(x, x),
    lambda x, i: smoe.linear_act_bwd(x, x, x)])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(ValueError, match="GPU tensor"):
        call(torch.zeros(4, 4, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32))
