"""The operators of an unquantised expert block against their formulas in 64
bits on the CPU.

Tolerances are bounds, not measurements.  A result is the exact value with one
rounding to its type (half a step: u = eps/2 relative) on top of what the fp32
arithmetic before it can lose: a sum of n products in any order is off by at
most n 2^-24 times the sum of the magnitudes.  fp16's smallest step, 2^-24,
bounds what a value near zero can lose beyond that.
"""
import math

import pytest
import torch

import smoe

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}
E32 = 2.0 ** -24


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def check(got, ref, slack, what=""):
    """got within half a step of its type plus `slack` (absolute) of ref."""
    got, g = got.cpu().double(), got.dtype
    tol = U[g] * (ref.abs() + slack) + slack + 2.0 ** -24 * (g == F16)
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        i = int(bad.flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: "
                             f"{got.flatten()[i]} for {ref.flatten()[i]} (tolerance {tol.flatten()[i]})")


def routing(T, E, K, seed, drop=0.0):
    g = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]) if T else torch.zeros(0, K)
    idx = idx.to(torch.int32)
    if drop:
        idx[torch.rand(idx.shape, generator=g) < drop] = E + 3
    return idx, torch.rand((T, K), generator=g) + 0.1


def sort_ref(idx, E):
    ids = idx.reshape(-1).tolist()
    rows = sorted((p for p in range(len(ids)) if 0 <= ids[p] < E), key=lambda p: (ids[p], p))
    inv = [-1] * len(ids)
    for r, p in enumerate(rows):
        inv[p] = r
    off = [0]
    for e in range(E):
        off.append(off[-1] + ids.count(e))
    return torch.tensor(inv, dtype=torch.int64), off


# ------------------------------------------------------------------ tokens
TOKENS = [(1, 64, 1, 4), (1, 2048, 8, 128), (7, 33, 3, 8), (130, 2880, 4, 32), (257, 1001, 2, 8), (64, 16, 32, 64),
          (3, 7168, 8, 256), (5000, 40, 2, 8), (9, 1, 5, 16)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("T,H,K,E", TOKENS)
def test_permute(dev, T, H, K, E, weights, dtype):
    idx, w = routing(T, E, K, 1, drop=0.2 if T > 3 else 0.0)
    x = rand((T, H), dtype, 2)
    wd = w.to(dev) if weights else None
    inv, off = sort_ref(idx, E)
    xp, row_map, inv_map, counts, offsets = smoe.permute_tokens(x.to(dev), idx.to(dev), E, topk_w=wd)
    assert inv_map.cpu().long().equal(inv) and offsets.cpu().tolist() == off
    assert counts.cpu().tolist() == [b - a for a, b in zip(off, off[1:])]
    have = inv >= 0
    ref = (x.double()[:, None, :] * (w.double()[:, :, None] if weights else 1.0)).expand(T, K, H).reshape(T * K, H)
    check(xp[inv[have].to(dev)], ref[have], ref[have].abs() * E32, "xp")
    assert row_map.cpu()[:off[-1]].long().equal(torch.argsort(torch.where(have, inv, T * K))[:off[-1]])
    # into a given buffer: rows without a pair keep what they held
    buf = torch.full((T * K, H), 7.0, dtype=dtype, device=dev)
    out = smoe.permute_tokens_rows(x.to(dev), inv_map, K, topk_w=wd, out=buf)
    assert out is buf and bool((buf[off[-1]:] == 7.0).all()) and buf[:off[-1]].equal(xp[:off[-1]])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("T,H,K,E", TOKENS)
def test_unpermute_and_gradients(dev, T, H, K, E, weights, dtype):
    idx, w = routing(T, E, K, 3, drop=0.2 if T > 3 else 0.0)
    inv, _ = sort_ref(idx, E)
    inv_map = inv.to(torch.int32).to(dev)
    y, g, gp, x = (rand(s, dtype, i) for i, s in enumerate([(T * K, H), (T, H), (T * K, H), (T, H)]))
    wd = w.to(dev) if weights else None
    have = (inv >= 0).view(T, K)
    wz = torch.where(have, w.double() if weights else torch.ones(T, K, dtype=torch.float64), torch.zeros(()).double())
    at = inv.clamp(min=0).view(T, K)

    out = smoe.unpermute_tokens(y.to(dev), inv_map, K, topk_w=wd)
    pairs = y.double()[at] * wz[:, :, None]
    check(out, pairs.sum(1), (K + 1) * E32 * pairs.abs().sum(1), "out")

    got = smoe.permute_tokens_bwd(gp.to(dev), inv_map, K, x=x.to(dev), topk_w=wd)
    dx, dw = got if weights else (got, None)
    pairs = gp.double()[at] * wz[:, :, None]
    check(dx, pairs.sum(1), (K + 1) * E32 * pairs.abs().sum(1), "dx")
    if weights:
        prod = gp.double()[at] * x.double()[:, None, :] * have[:, :, None]
        check(dw, prod.sum(2), (H + 1) * E32 * prod.abs().sum(2), "dw of permute")

    got = smoe.unpermute_tokens_bwd(g.to(dev), inv_map, K, y=y.to(dev), topk_w=wd)
    dy, dw = got if weights else (got, None)
    ref = (g.double()[:, None, :] * wz[:, :, None]).reshape(T * K, H)
    flat = have.reshape(-1)
    check(dy[inv[flat].to(dev)], ref[flat], ref[flat].abs() * E32, "dy")
    if weights:
        prod = y.double()[at] * g.double()[:, None, :] * have[:, :, None]
        check(dw, prod.sum(2), (H + 1) * E32 * prod.abs().sum(2), "dw of unpermute")


@pytest.mark.parametrize("T,E,K", [(1, 8, 8), (256, 1024, 8), (1024, 3, 2), (1025, 3, 2), (64, 1000, 32), (2048, 5, 1)])
def test_permute_sort_against_route_sort(dev, T, E, K):
    """Maps, counts, offsets and the status of a small batch in one launch
    and of a larger one are the sort's, repeated and out-of-range ids among
    them."""
    g = torch.Generator().manual_seed(T)
    idx = torch.randint(-2, E + 2, (T, K), generator=g, dtype=torch.int32).to(dev)
    x = rand((T, 24), F16, 1).to(dev)
    got = smoe.permute_tokens(x, idx, E)
    status = int(smoe.last_route_status(dev))
    want = smoe.route_sort(idx, E)
    n = int(want[3][-1])
    assert status == int(smoe.last_route_status(dev)) == T * K - n
    assert got[1][:n].equal(want[0][:n]) and all(a.equal(b) for a, b in zip(got[2:], want[1:]))
    assert got[0][:n].equal(x[(want[0][:n] // K).long()])


def test_tokens_rows_apart_and_odd_starts(dev):
    """Inputs whose rows lie apart or start at an odd element, and one row
    repeated (stride 0), give what contiguous copies give."""
    T, H, K, E = 70, 333, 4, 16
    idx, w = routing(T, E, K, 5)
    inv = sort_ref(idx, E)[0].to(torch.int32).to(dev)
    w = w.to(dev)
    for dtype in (BF16, F16, F32):
        x = rand((T, 2 * H + 5), dtype, 6).to(dev)[:, 3:3 + H]
        y = rand((T * K, H + 7), dtype, 7).to(dev)[:, 1:1 + H]
        one = rand((1, H), dtype, 8).to(dev).expand(T, H)
        eq = lambda a, b: all(p.equal(q) for p, q in zip(a, b)) if isinstance(a, tuple) else a.equal(b)
        for v in (x, one):
            c = v.contiguous()
            assert eq(smoe.permute_tokens_rows(v, inv, K, w), smoe.permute_tokens_rows(c, inv, K, w))
            assert eq(smoe.permute_tokens_bwd(y, inv, K, v, w), smoe.permute_tokens_bwd(y.contiguous(), inv, K, c, w))
            assert eq(smoe.unpermute_tokens_bwd(v, inv, K, y, w), smoe.unpermute_tokens_bwd(c, inv, K, y.contiguous(), w))
        assert eq(smoe.unpermute_tokens(y, inv, K, w), smoe.unpermute_tokens(y.contiguous(), inv, K, w))


def test_tokens_special_values(dev):
    """NaN and infinities stay in the rows they are in; a pair without a row
    brings nothing, whatever its weight."""
    T, H, K, E = 6, 48, 2, 4
    idx, w = routing(T, E, K, 9)
    idx[2, 1] = E
    w[2, 1] = math.nan
    inv = sort_ref(idx, E)[0]
    x = rand((T, H), BF16, 10)
    x[1, 5], x[3, 7] = math.inf, math.nan
    xp = smoe.permute_tokens_rows(x.to(dev), inv.to(torch.int32).to(dev), K, w.to(dev)).cpu()
    rows = inv.view(T, K)
    for t in range(T):
        for k in range(K):
            if rows[t, k] >= 0:
                assert torch.isfinite(xp[rows[t, k]]).all() == (t not in (1, 3))
    y = rand((T * K, H), BF16, 11)
    y[rows[4, 0]] = math.nan
    out = smoe.unpermute_tokens(y.to(dev), inv.to(torch.int32).to(dev), K, w.to(dev)).cpu()
    assert torch.isnan(out[4]).all() and torch.isfinite(out[[0, 1, 2, 3, 5]]).all()


# ------------------------------------------------------------------- norms
NORMS = [(1, 7168), (1, 1), (3, 17), (70, 2880), (129, 1001), (2050, 64), (5, 16384), (2, 65536), (33, 4095)]
EPS = 1e-5


def norm_inputs(T, H, dtype, gate, pdt, seed=0):
    x, y, g, sk = (rand((T, H), dtype, seed + i, 1.0 + i) for i in range(4))
    w = (1.0 + rand((H,), F32, seed + 5, 0.2)).to(pdt)
    shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[gate]
    gt = None if shape is None else rand(shape, pdt, seed + 6, 0.7)
    return x, y, g, sk, w, gt


def d64(t):
    return None if t is None else t.double()


def dv(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


@pytest.mark.parametrize("dtype,pdt", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("T,H", NORMS)
def test_norm_in(dev, T, H, dtype, pdt):
    x, _, g, sk, w, _ = norm_inputs(T, H, dtype, "none", pdt)
    xd, gd, sd, wd = dv(dev, x, g, sk, w)
    h, rstd = smoe.block_norm_in(xd, wd, eps=EPS)
    r = 1 / torch.sqrt(x.double().square().mean(1) + EPS)
    # mean: H roundings of positive terms; rstd: half of that and four more
    rel = (H / 2 + 8) * E32
    check(rstd, r, r * rel, "rstd")
    ref = x.double() * r[:, None] * w.double()
    check(h, ref, ref.abs() * rel, "h")

    dx, dw = smoe.block_norm_in_bwd(gd, xd, rstd, wd, dskip=sd, skip_scale=0.5)
    r = rstd.cpu().double()
    n, c = x.double() * r[:, None], g.double() * w.double()
    mean, mag = (c * n).mean(1, keepdim=True), (c * n).abs().mean(1, keepdim=True)
    ref = r[:, None] * (c - n * mean) + 0.5 * sk.double()
    slack = E32 * (6 * (r[:, None] * (c.abs() + n.abs() * mag) + sk.abs()) + r[:, None] * n.abs() * mag * H)
    check(dx, ref, slack, "dx")
    check(dw, (g.double() * n).sum(0), E32 * (T + 4) * (g.double() * n).abs().sum(0), "dweight")
    plain, none = smoe.block_norm_in_bwd(gd, xd, rstd)
    assert none is None and plain.shape == dx.shape


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("dtype,pdt", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("T,H", NORMS)
def test_norm_out(dev, T, H, dtype, pdt, gate):
    x, y, g, _, w, gt = norm_inputs(T, H, dtype, gate, pdt, seed=20)
    xd, yd, gd, wd, gtd = dv(dev, x, y, g, w, gt)
    s = 0.3
    out, rstd = smoe.block_norm_out(yd, xd, wd, gate=gtd, residual_scale=s, eps=EPS)
    s = float(torch.tensor(s, dtype=F32))
    r = 1 / torch.sqrt(y.double().square().mean(1) + EPS)
    rel = (H / 2 + 12) * E32
    check(rstd, r, r * rel, "rstd")
    gg = torch.ones(1, 1).double() if gt is None else gt.double()
    branch = gg * (y.double() * r[:, None] * w.double())
    ref = s * x.double() + branch
    check(out, ref, branch.abs() * rel + 2 * E32 * ref.abs() + 2 * E32 * x.double().abs(), "out")

    dy, dw, dg = smoe.block_norm_out_bwd(gd, yd, rstd, wd, gate=gtd)
    r = rstd.cpu().double()
    n, up = y.double() * r[:, None], g.double() * gg
    c = up * w.double()
    mean, mag = (c * n).mean(1, keepdim=True), (c * n).abs().mean(1, keepdim=True)
    ref = r[:, None] * (c - n * mean)
    slack = E32 * (8 * r[:, None] * (c.abs() + n.abs() * mag) + r[:, None] * n.abs() * mag * H)
    check(dy, ref, slack, "dy")
    check(dw, (up * n).sum(0), E32 * (T + 6) * (up * n).abs().sum(0), "dweight")
    if gt is None:
        assert dg is None
        return
    full = g.double() * n * w.double()
    if gate == "channel":
        check(dg, full.sum(0), E32 * (T + 6) * full.abs().sum(0), "dgate")
    elif gate == "token" and H > 1:
        check(dg, full.sum(1, keepdim=True), E32 * (H + 6) * full.abs().sum(1, keepdim=True), "dgate")
    else:
        check(dg, full, E32 * 4 * full.abs(), "dgate")
    assert dg.shape == gtd.shape and dg.dtype == gtd.dtype


def test_norm_without_weight_and_rows_apart(dev):
    T, H = 37, 515
    for dtype in (BF16, F16, F32):
        wide = rand((T, 2 * H + 3), dtype, 40).to(dev)
        x, y = wide[:, 1:1 + H], wide[:, H + 3:]
        g = rand((T, H + 1), dtype, 41).to(dev)[:, 1:]
        gt = rand((T, 5), dtype, 42).to(dev)[:, 2:3]
        ones = torch.ones(H, dtype=dtype, device=dev)
        for a, b in (((x, y, g, gt), tuple(v.contiguous() for v in (x, y, g, gt))),):
            for weight in (None, ones):
                o1, r1 = smoe.block_norm_out(a[1], a[0], weight, gate=a[3])
                o2, r2 = smoe.block_norm_out(b[1], b[0], ones, gate=b[3])
                assert o1.equal(o2) and r1.equal(r2)
                d1 = smoe.block_norm_out_bwd(a[2], a[1], r1, weight, gate=a[3])
                d2 = smoe.block_norm_out_bwd(b[2], b[1], r2, ones, gate=b[3])
                assert d1[0].equal(d2[0]) and d1[2].equal(d2[2])
                h1, q1 = smoe.block_norm_in(a[0], weight)
                h2, q2 = smoe.block_norm_in(b[0], ones)
                assert h1.equal(h2) and q1.equal(q2)
                assert smoe.block_norm_in_bwd(a[2], a[0], q1, weight, dskip=a[1])[0].equal(
                    smoe.block_norm_in_bwd(b[2], b[0], q2, ones, dskip=b[1])[0])


def test_norm_zero_rows_and_special_values(dev):
    """A row of zeros gives zeros (eps keeps rstd finite); NaN stays in its row."""
    x = rand((4, 300), BF16, 50)
    x[1] = 0
    x[2, 7] = math.nan
    h, rstd = smoe.block_norm_in(x.to(dev), None, eps=1e-6)
    h = h.cpu()
    assert (h[1] == 0).all() and abs(float(rstd[1]) - 1000.0) < 1e-2
    assert torch.isnan(h[2]).all() and torch.isfinite(h[[0, 1, 3]]).all()


# ------------------------------------------------------------------ linear
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu"]


def act64(z, act):
    if act == "swiglu":
        g, u = z.chunk(2, 1)
        return g * torch.sigmoid(g) * u
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z),
            "gelu_tanh": lambda: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))}[act]()


def bounds_of(offsets, R):
    return [0, R] if offsets is None else offsets


def run_linear(dev, R, K, N, act, dtype, offsets=None, bias=None, residual=False, seed=0):
    """Forward and backward against the formulas; -> the outputs."""
    b, E = bounds_of(offsets, R), 1 if offsets is None else len(offsets) - 1
    lead = () if offsets is None else (E,)
    M = N // 2 if act == "swiglu" else N
    x, w = rand((R, K), dtype, seed), rand(lead + (N, K), dtype, seed + 1, 1 / math.sqrt(K))
    bi = None if bias is None else rand(lead + (N,), bias, seed + 2, 0.5)
    res = rand((R, M), dtype, seed + 3) if residual else None
    dout = rand((R, M), dtype, seed + 4)
    xd, wd, bd, rd, gd = dv(dev, x, w, bi, res, dout)
    od = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=dev)
    out, z = smoe.linear_act(xd, wd, bias=bd, act=act, residual=rd, offsets=od, save_z=True)
    dx, dw, db = smoe.linear_act_bwd(gd, xd, wd, z=z, act=act, bias=bd, offsets=od)
    u, zc = U[dtype], z.cpu().double()
    for e in range(E):
        lo, hi = b[e], b[e + 1]
        we = w[e].double() if lead else w.double()
        ed = dw[e] if lead else dw
        if hi <= lo:
            assert not ed.any() and (db is None or not db[e].any())
            continue
        xe = x[lo:hi].double()
        zr, mag = xe @ we.t(), xe.abs() @ we.t().abs()
        if bi is not None:
            be = bi[e].double() if lead else bi.double()
            zr, mag = zr + be, mag + be.abs()
        tol = (K + 2) * E32 * mag
        check(z[lo:hi], zr, tol, f"z of expert {e}")
        ref = act64(zr, act)
        # every activation here has a slope below 1.13; the products of
        # SwiGLU also scale one factor's error by the other; 2^-20 relative
        # covers the exp2, reciprocal and erf of the fp32 activation
        if act == "swiglu":
            g, up = zr.chunk(2, 1)
            tg, tu = tol.chunk(2, 1)
            slack = 1.13 * tg * (up.abs() + tu) + g.abs() * tu + 2.0 ** -20 * ref.abs()
        else:
            slack = 1.13 * tol + 2.0 ** -20 * (ref.abs() + (zr.abs() * 2.0 ** -3 if act == "gelu" else 0))
        if res is not None:
            ref = ref + res[lo:hi].double()
            slack = slack + E32 * ref.abs()
        check(out[lo:hi], ref, slack, f"out of expert {e}")
        # gradients from the z that the forward stored
        ze = zc[lo:hi].clone().requires_grad_(True)
        act64(ze, act).backward(dout[lo:hi].double())
        dz = ze.grad
        if act == "swiglu":  # |d/dg| <= 1.13 |u|, |d/du| <= |g|: the fp32 slope's error
            dzm = dz.abs() + 2.0 ** -6 * torch.cat([zc[lo:hi, M:].abs(), zc[lo:hi, :M].abs()], 1) * \
                dout[lo:hi].double().abs().repeat(1, 2)
        else:
            dzm = dz.abs() + 2.0 ** -6 * dout[lo:hi].double().abs()
        el = (u * dz.abs() + 2.0 ** -18 * dzm + 2.0 ** -25) if act != "none" else torch.zeros_like(dz)
        n = hi - lo
        check(dx[lo:hi], dz @ we, el @ we.abs() + (N + 2) * E32 * (dz.abs() @ we.abs()), f"dx of expert {e}")
        check(ed, dz.t() @ xe, el.t() @ xe.abs() + (n + 2) * E32 * (dz.abs().t() @ xe.abs()), f"dw of expert {e}")
        if db is not None:
            fl = 2.0 ** -18 * dzm if act != "none" else torch.zeros_like(dz)
            check(db[e] if lead else db, dz.sum(0), fl.sum(0) + (n + 4) * E32 * dz.abs().sum(0), f"db of expert {e}")
    return out, z, dx, dw, db


DENSE = [(1, 64, 64), (1, 1, 2), (16, 512, 256), (5, 40, 24), (63, 65, 66), (130, 264, 200), (17, 1000, 514),
         (300, 33, 130), (257, 512, 384), (600, 1096, 776), (2, 4160, 136), (29, 1544, 1050),
         (50, 704, 96), (200, 2048, 264), (70, 1000, 3000), (2050, 136, 72), (34, 4104, 520)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("R,K,N", DENSE)
def test_linear_dense(dev, R, K, N, act, dtype):
    run_linear(dev, R, K, N, act, dtype, bias=dtype if N % 4 else F32, residual=R % 2 == 0, seed=R)


GROUPED = [(40, 64, 64, [0, 0, 13, 13, 40]), (300, 136, 96, [0, 1, 66, 200, 300]), (7, 129, 34, [0, 7]),
           (513, 256, 256, [0, 128, 256, 257, 257, 257, 513]), (64, 48, 32, [0] * 20 + [64]),
           (200, 72, 640, list(range(0, 201, 2))),
           (70, 1030, 96, [0, 3, 3, 20, 55, 70]), (1500, 328, 520, [0, 700, 1000, 1001, 1500]), (900, 64, 272, [0] + [90 * (e // 7) for e in range(1, 71)])]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("R,K,N,offsets", GROUPED)
def test_linear_grouped(dev, R, K, N, offsets, act, dtype):
    run_linear(dev, R, K, N, act, dtype, offsets=offsets, bias=dtype, residual=act == "none", seed=N)


BIG = [(3136, 200, 4112, None, "gelu"), (6000, 2056, 136, None, "silu"), (2600, 1800, 1032, [0, 700, 700, 1900, 2600], "none"),
       (3000, 72, 8200, [0, 1400, 3000], "swiglu"), (5000, 1032, 2056, None, "swiglu"),
       (4000, 520, 4104, [0, 130, 1000, 1000, 4000], "relu")]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("R,K,N,offsets,act", BIG)
def test_linear_big_tiles(dev, R, K, N, offsets, act, dtype):
    """Sizes whose product, dx or dW take the 256-row tiles, several of them a
    workgroup, the last ones partly empty."""
    run_linear(dev, R, K, N, act, dtype, offsets=offsets, bias=dtype, residual=act != "none", seed=R)


@pytest.mark.parametrize("R,K,N", [(4100, 72, 136), (4099, 73, 135), (300, 4104, 264)])
def test_linear_cut_sums_into_buffers(dev, R, K, N):
    """A dense product of few tiles (its sum cut into shares): dW written and
    added in every mode, aligned and not, and the same bits every time."""
    x, w, g = rand((R, K), BF16, 1).to(dev), rand((N, K), BF16, 2).to(dev), rand((R, N), BF16, 3).to(dev)
    f = torch.empty((N, K), device=dev)
    smoe.linear_act_bwd(g, x, w, need_dx=False, dw_out=f)
    a, b = g.cpu().double(), x.cpu().double()
    check(f, a.t() @ b, (R + 20) * E32 * (a.abs().t() @ b.abs()), "fp32 dw")
    for base in (rand((N, K), F32, 4).to(dev), rand((N, K), BF16, 5).to(dev)):
        acc = base.clone()
        smoe.linear_act_bwd(g, x, w, need_dx=False, dw_out=acc, accumulate=True)
        assert acc.equal((base.float() + f).to(base.dtype))
    first = smoe.linear_act_bwd(g, x, w)
    for _ in range(3):
        assert all(p.equal(q) for p, q in zip(first[:2], smoe.linear_act_bwd(g, x, w)[:2]))
    res = rand((R, N), BF16, 6).to(dev)
    out = smoe.linear_act(x, w, residual=res)
    into = res.clone()
    assert smoe.linear_act(x, w, residual=into, out=into).equal(out)


def test_linear_malformed_offsets_stay_inside(dev):
    """Bounds out of order, negative or past the end give values that mean
    nothing, but touch nothing outside: guard rows around the outputs keep
    what they hold, and the call after is right."""
    R, K, N, E = 300, 64, 48, 6
    x, w = rand((R, K), BF16, 1).to(dev), rand((E, N, K), BF16, 2).to(dev)
    g = rand((R, N), BF16, 3).to(dev)
    for off in ([0, 50, 20, 290, 100, 300, 300], [-5, 10, 1 << 30, 40, -7, 90, 400], [300, 250, 200, 150, 100, 50, 0]):
        od = torch.tensor(off, dtype=torch.int32, device=dev)
        guarded = torch.full((R + 64, N), 3.0, dtype=BF16, device=dev)
        smoe.linear_act(x, w, offsets=od, out=guarded[32:32 + R])
        smoe.linear_act_bwd(g, x, w, offsets=od, bias=w[:, :, 0].contiguous())
        torch.cuda.synchronize()
        assert bool((guarded[:32] == 3.0).all()) and bool((guarded[32 + R:] == 3.0).all())
    run_linear(dev, R, K, N, "none", BF16, offsets=[0, 50, 50, 120, 250, 299, 300], bias=BF16)


def test_linear_plain_forms(dev):
    """Without bias, residual, z: the same values as with a zero bias."""
    R, K, N = 77, 200, 120
    x, w = rand((R, K), BF16, 1).to(dev), rand((N, K), BF16, 2).to(dev)
    zero = torch.zeros(N, dtype=BF16, device=dev)
    for act in ACTS:
        assert smoe.linear_act(x, w, act=act).equal(smoe.linear_act(x, w, bias=zero, act=act, save_z=True)[0])


@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_linear_rows_outside_and_between(dev, act):
    """Rows before the first and behind the last expert's keep what the
    buffers held, and NaN and infinities there reach nothing."""
    R, K, N, off = 150, 96, 64, [20, 50, 50, 121]
    M = N // 2 if act == "swiglu" else N
    x, w = rand((R, K), BF16, 3), rand((3, N, K), BF16, 4, 0.1)
    dout, z0 = rand((R, M), BF16, 5), rand((R, N), BF16, 6)
    inside = torch.zeros(R, dtype=torch.bool)
    inside[20:121] = True
    xn, dn, zn = x.clone(), dout.clone(), z0.clone()
    for t in (xn, dn, zn):
        t[~inside] = math.nan
        t[3] = math.inf
    od = torch.tensor(off, dtype=torch.int32, device=dev)
    buf = torch.full((R, M), 5.0, dtype=BF16, device=dev)
    out = smoe.linear_act(xn.to(dev), w.to(dev), act=act, offsets=od, out=buf).cpu()
    ref = smoe.linear_act(x.to(dev), w.to(dev), act=act, offsets=od).cpu()
    assert (out[~inside] == 5.0).all() and out[inside].equal(ref[inside])
    z = None if act == "none" else zn.to(dev)
    zc = None if act == "none" else z0.to(dev)
    bias = torch.zeros(3, N, dtype=F32, device=dev)
    got = smoe.linear_act_bwd(dn.to(dev), xn.to(dev), w.to(dev), z=z, act=act, bias=bias, offsets=od)
    ref = smoe.linear_act_bwd(dout.to(dev), x.to(dev), w.to(dev), z=zc, act=act, bias=bias, offsets=od)
    assert got[0].cpu()[inside].equal(ref[0].cpu()[inside])
    assert got[1].equal(ref[1]) and got[2].equal(ref[2]) and bool(torch.isfinite(got[1].float()).all())
    assert not got[1][1].any() and not got[2][1].any()


def test_linear_rows_apart(dev):
    R, K, N = 90, 130, 72
    for dtype in (BF16, F16):
        x = rand((R, 2 * K + 3), dtype, 7).to(dev)[:, 3:3 + K]
        w = rand((N, K), dtype, 8).to(dev)
        res = rand((R, N + 1), dtype, 9).to(dev)[:, 1:]
        g = rand((1, N), dtype, 10).to(dev).expand(R, N)
        out, z = smoe.linear_act(x, w, act="silu", residual=res, save_z=True)
        ref, zr = smoe.linear_act(x.contiguous(), w, act="silu", residual=res.contiguous(), save_z=True)
        assert out.equal(ref) and z.equal(zr)
        for act in ("none", "silu"):
            a = smoe.linear_act_bwd(g, x, w, z=z, act=act)
            b = smoe.linear_act_bwd(g.contiguous(), x.contiguous(), w, z=z, act=act)
            assert a[0].equal(b[0]) and a[1].equal(b[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_weight_gradient_buffers(dev, dtype):
    """dw into fp32 and 16-bit buffers, written and added to."""
    R, K, N, off = 120, 80, 48, [0, 50, 50, 120]
    x, w, g = rand((R, K), dtype, 1).to(dev), rand((3, N, K), dtype, 2).to(dev), rand((R, N), dtype, 3).to(dev)
    od = torch.tensor(off, dtype=torch.int32, device=dev)
    kw = dict(offsets=od, need_dx=False)
    f = torch.empty((3, N, K), device=dev)
    dx, dw, db = smoe.linear_act_bwd(g, x, w, dw_out=f, **kw)
    assert dx is None and db is None and dw is f
    for e in range(3):
        a, b = g[off[e]:off[e + 1]].cpu().double(), x[off[e]:off[e + 1]].cpu().double()
        check(f[e], a.t() @ b, 71 * E32 * (a.abs().t() @ b.abs()), "fp32 dw")
    assert smoe.linear_act_bwd(g, x, w, **kw)[1].equal(f.to(dtype))
    base = rand((3, N, K), F32, 4).to(dev)
    acc = base.clone()
    smoe.linear_act_bwd(g, x, w, dw_out=acc, accumulate=True, **kw)
    assert acc.equal(base + f)
    half = base.to(dtype)
    acc = half.clone()
    smoe.linear_act_bwd(g, x, w, dw_out=acc, accumulate=True, **kw)
    assert acc.equal((half.float() + f).to(dtype))


def test_linear_gradient_by_differences(dev):
    """The gradients of the fused call against central differences of the
    formula itself in 64 bits, and the call's loss against that formula's."""
    R, K, N = 24, 40, 32
    for act in ACTS:
        x, w, b = rand((R, K), BF16, 1), rand((N, K), BF16, 2, 0.2), rand((N,), BF16, 3)
        M = N // 2 if act == "swiglu" else N
        g = rand((R, M), BF16, 4)
        f = lambda x, w, b: float((act64(x @ w.t() + b, act) * g.double()).sum())
        xd, wd, bd, gd = dv(dev, x, w, b, g)
        out, z = smoe.linear_act(xd, wd, bias=bd, act=act, save_z=True)
        grads = smoe.linear_act_bwd(gd, xd, wd, z=z, act=act, bias=bd)
        args = [x.double(), w.double(), b.double()]
        for i, grad in enumerate(grads):
            d = rand(args[i].shape, F32, 30 + i).double()
            h = 1e-6
            up = f(*[a + h * d if j == i else a for j, a in enumerate(args)])
            dn = f(*[a - h * d if j == i else a for j, a in enumerate(args)])
            num, got = (up - dn) / (2 * h), float((grad.cpu().double() * d).sum())
            # z, dz and the gradient are each rounded to bf16 (u = 2^-8): each
            # value is off by at most 3u of the magnitudes summed into it
            # (slopes' slope below 1.2); relu's step at 0 is not crossed by
            # such a z except where z itself is below u of its terms
            scale = float(sum((gr.cpu().double().abs() * d.abs()).sum() for gr in [grad]))
            assert abs(num - got) <= 6 * 2.0 ** -8 * (scale + abs(num)), (act, i, num, got)


# ----------------------------------------------------------- all together
def test_empty_batches(dev):
    i32 = dict(dtype=torch.int32, device=dev)
    x = torch.empty((0, 64), dtype=BF16, device=dev)
    inv = torch.empty(0, **i32)
    assert smoe.permute_tokens(x, torch.empty((0, 2), **i32), 4)[0].shape == (0, 64)
    assert smoe.permute_tokens_rows(x, inv, 2).shape == (0, 64)
    assert smoe.unpermute_tokens(x, inv, 2).shape == (0, 64)
    w = torch.empty((0, 2), device=dev)
    assert smoe.permute_tokens_bwd(x, inv, 2, x, w)[1].shape == (0, 2)
    assert smoe.unpermute_tokens_bwd(x, inv, 2, x, w)[0].shape == (0, 64)
    wt = torch.ones(64, dtype=BF16, device=dev)
    h, r = smoe.block_norm_in(x, wt)
    assert h.shape == (0, 64) and not smoe.block_norm_in_bwd(h, x, r, wt)[1].any()
    o, r = smoe.block_norm_out(x, x, wt, gate=wt)
    assert not smoe.block_norm_out_bwd(o, x, r, wt, gate=wt)[2].any()
    W, off = torch.ones((2, 32, 64), dtype=BF16, device=dev), torch.zeros(3, **i32)
    out, z = smoe.linear_act(x, W, act="silu", offsets=off, save_z=True)
    dx, dw, db = smoe.linear_act_bwd(out, x, W, z=z, act="silu", offsets=off, bias=W[:, :, 0].contiguous())
    assert out.shape == (0, 32) and dx.shape == (0, 64) and not dw.any() and not db.any()


def expert_block(x, idx, tw, p, E, K):
    """Norm, sorted experts and back, a dense expert beside them, norm, gate
    and residual: the operators as a block uses them."""
    h, r1 = smoe.block_norm_in(x, p["n1"])
    xp, row_map, inv, counts, off = smoe.permute_tokens(h, idx, E)
    a, z1 = smoe.linear_act(xp, p["w1"], bias=p["b1"], act="swiglu", offsets=off, save_z=True)
    y = smoe.linear_act(a, p["w2"], offsets=off)
    routed = smoe.unpermute_tokens(y, inv, K, tw)
    s, z2 = smoe.linear_act(h, p["s1"], act="gelu_tanh", save_z=True)
    both = smoe.linear_act(s, p["s2"], residual=routed)
    out, r2 = smoe.block_norm_out(both, x, p["n2"], gate=p["g"], residual_scale=0.7)
    return out, (h, r1, xp, inv, off, a, z1, y, s, z2, both, r2)


def expert_block_bwd(dout, x, tw, p, K, st):
    h, r1, xp, inv, off, a, z1, y, s, z2, both, r2 = st
    dboth, dn2, dg = smoe.block_norm_out_bwd(dout, both, r2, p["n2"], gate=p["g"])
    ds, ds2, _ = smoe.linear_act_bwd(dboth, s, p["s2"])
    dh1, ds1, _ = smoe.linear_act_bwd(ds, h, p["s1"], z=z2, act="gelu_tanh")
    dy, dtw = smoe.unpermute_tokens_bwd(dboth, inv, K, y, tw)
    da, dw2, _ = smoe.linear_act_bwd(dy, a, p["w2"], offsets=off)
    dxp, dw1, db1 = smoe.linear_act_bwd(da, xp, p["w1"], z=z1, act="swiglu", bias=p["b1"], offsets=off)
    dh = smoe.permute_tokens_bwd(dxp, inv, K) + dh1
    dx, dn1 = smoe.block_norm_in_bwd(dh, x, r1, p["n1"], dskip=dout, skip_scale=0.7)
    return dx, dn1, dn2, dg, dw1, dw2, db1, ds1, ds2, dtw


def block_inputs(T, H, I, E, K, seed, dtype=BF16):
    idx, tw = routing(T, E, K, seed)
    p = dict(n1=1 + rand((H,), F32, seed + 1, 0.2), n2=1 + rand((H,), F32, seed + 2, 0.2), g=rand((H,), F32, seed + 3),
             w1=rand((E, 2 * I, H), F32, seed + 4, 1 / math.sqrt(H)), b1=rand((E, 2 * I), F32, seed + 5, 0.3),
             w2=rand((E, H, I), F32, seed + 6, 1 / math.sqrt(I)), s1=rand((I, H), F32, seed + 7, 1 / math.sqrt(H)),
             s2=rand((H, I), F32, seed + 8, 1 / math.sqrt(I)))
    return rand((T, H), dtype, seed + 9), idx, tw, {k: v.to(dtype) for k, v in p.items()}, rand((T, H), dtype, seed + 10)


def block64(x, idx, tw, p, E, K):
    norm = lambda v, w: v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * w
    h = norm(x, p["n1"])
    routed = 0
    for k in range(K):
        e = idx[:, k].long()
        z = torch.stack([p["w1"][e[t]] @ h[t] + p["b1"][e[t]] for t in range(x.shape[0])])
        a = act64(z, "swiglu")
        routed = routed + tw[:, k:k + 1] * torch.stack([p["w2"][e[t]] @ a[t] for t in range(x.shape[0])])
    both = act64(h @ p["s1"].t(), "gelu_tanh") @ p["s2"].t() + routed
    return 0.7 * x + p["g"] * norm(both, p["n2"])


@pytest.mark.parametrize("T", [1, 37, 200])
def test_expert_block_against_autograd(dev, T):
    """All of them together, forward and backward, against autograd over the
    formulas in 64 bits.  Every tensor between two operators is rounded to
    bf16 (u = 2^-8 at most, half that on average), about 8 of them on the
    longest way, and rounding errors of unlike sign add as squares: the error
    of each result, root mean square over its root mean square, stays below
    sqrt(8) u < 3 u; 4 u is asked for."""
    H, I, E, K = 72, 56, 6, 2
    x, idx, tw, p, dout = block_inputs(T, H, I, E, K, 60)
    leaves = {k: v.double().requires_grad_(True) for k, v in p.items()}
    x64, tw64 = x.double().requires_grad_(True), tw.double().requires_grad_(True)
    ref = block64(x64, idx, tw64, leaves, E, K)
    ref.backward(dout.double())
    pd = {k: v.to(dev) for k, v in p.items()}
    out, st = expert_block(x.to(dev), idx.to(dev), tw.to(dev), pd, E, K)
    got = expert_block_bwd(dout.to(dev), x.to(dev), tw.to(dev), pd, K, st)
    want = (x64, leaves["n1"], leaves["n2"], leaves["g"], leaves["w1"], leaves["w2"], leaves["b1"], leaves["s1"],
            leaves["s2"], tw64)
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())
    assert rel(out, ref.detach()) <= 4 * 2.0 ** -8
    for i, (a, b) in enumerate(zip(got, want)):
        assert rel(a, b.grad) <= 4 * 2.0 ** -8, i


def test_expert_block_in_a_graph(dev):
    """Forward and backward captured once and replayed on new inputs, with
    eager work in between, gives the eager bits every time; results do not
    change from run to run."""
    T, H, I, E, K = 50, 64, 48, 8, 2
    x, idx, tw, p, dout = block_inputs(T, H, I, E, K, 80)
    xs, ids, tws, gs = dv(dev, x, idx, tw, dout)
    pd = {k: v.to(dev) for k, v in p.items()}

    def step():
        out, st = expert_block(xs, ids, tws, pd, E, K)
        return (out,) + expert_block_bwd(gs, xs, tws, pd, K, st)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x2, idx2, tw2, _, g2 = block_inputs(T, H, I, E, K, 200 + 30 * i)
        for dst, src in ((xs, x2), (ids, idx2), (tws, tw2), (gs, g2)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        for a, b in zip(kept, step()):
            assert a.equal(b)


def test_other_stream(dev):
    """Calls follow the current stream."""
    T, H, I, E, K = 40, 64, 32, 4, 2
    x, idx, tw, p, dout = block_inputs(T, H, I, E, K, 90)
    xs, ids, tws, gs = dv(dev, x, idx, tw, dout)
    pd = {k: v.to(dev) for k, v in p.items()}
    ref, _ = expert_block(xs, ids, tws, pd, E, K)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, _ = expert_block(xs, ids, tws, pd, E, K)
    s.synchronize()
    assert got.equal(ref)


def test_refusals(dev):
    bad = (ValueError, TypeError)
    x = torch.zeros((4, 64), dtype=BF16, device=dev)
    inv = torch.arange(8, dtype=torch.int32, device=dev)
    w = torch.ones((4, 2), device=dev)
    n = torch.ones(64, dtype=BF16, device=dev)
    W = torch.zeros((32, 64), dtype=BF16, device=dev)
    r = torch.ones(4, device=dev)
    off = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    calls = [
        lambda: smoe.permute_tokens_rows(x.double(), inv, 2), lambda: smoe.permute_tokens_rows(x.t(), inv, 2),
        lambda: smoe.permute_tokens_rows(x, inv[:7], 2), lambda: smoe.permute_tokens_rows(x, inv, 0),
        lambda: smoe.permute_tokens_rows(x, inv, 33), lambda: smoe.permute_tokens_rows(x, inv.long(), 2),
        lambda: smoe.permute_tokens_rows(x, inv, 2, topk_w=w[:3]),
        lambda: smoe.permute_tokens_rows(x, inv, 2, topk_w=w.half()),
        lambda: smoe.permute_tokens_rows(x, inv, 2, out=x),
        lambda: smoe.permute_tokens(x, inv.view(4, 2)[:3].contiguous(), 4),
        lambda: smoe.unpermute_tokens(x, inv, 3), lambda: smoe.unpermute_tokens(x, inv, 2),
        lambda: smoe.permute_tokens_bwd(x, inv[:4], 2, None, w[:2]),
        lambda: smoe.unpermute_tokens_bwd(x, inv, 2, x, w),
        lambda: smoe.block_norm_in(x, n[:63]), lambda: smoe.block_norm_in(x, n.half()),
        lambda: smoe.block_norm_in(x, n, eps=0.0), lambda: smoe.block_norm_in(x.cpu(), n),
        lambda: smoe.block_norm_in(torch.zeros((1, 65537), dtype=BF16, device=dev)),
        lambda: smoe.block_norm_out(x, x[:3], n), lambda: smoe.block_norm_out(x, x.half(), n),
        lambda: smoe.block_norm_out(x, x, n, gate=n[:5]), lambda: smoe.block_norm_out(x, x, n, gate=x[:, :2]),
        lambda: smoe.block_norm_in_bwd(x, x, r[:3], n), lambda: smoe.block_norm_out_bwd(x[:, :32], x, r, n),
        lambda: smoe.linear_act(x, W, act="tanh"), lambda: smoe.linear_act(x.float(), W.float()),
        lambda: smoe.linear_act(x[:, :32], W), lambda: smoe.linear_act(x, W[:31], act="swiglu"),
        lambda: smoe.linear_act(x, W, offsets=off), lambda: smoe.linear_act(x, W[None], offsets=off[:1]),
        lambda: smoe.linear_act(x, W[None]), lambda: smoe.linear_act(x, W, bias=n),
        lambda: smoe.linear_act(x, W, residual=x), lambda: smoe.linear_act(x, W, out=x),
        lambda: smoe.linear_act(x, W.half()),
        lambda: smoe.linear_act_bwd(x[:, :32], x, W, act="silu"),
        lambda: smoe.linear_act_bwd(x, x, W), lambda: smoe.linear_act_bwd(x[:, :32], x, W, accumulate=True),
        lambda: smoe.linear_act_bwd(x[:, :32], x, W, dw_out=W.half()),
        lambda: smoe.linear_act_bwd(x[:, :32], x, W, z=x, act="silu"),
    ]
    for i, c in enumerate(calls):
        with pytest.raises(bad):
            c()
            pytest.fail(f"call {i} was accepted")
