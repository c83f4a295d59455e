"""Group norm with an activation, and dropout, against their definitions in 64 bits.

Tolerances are rounding bounds, element by element, with u = 2^-24 (half a step of fp32) and a chain of at most K = 256
additions between an element and any mean or sum it enters:
  statistics   |d mean| <= K u mean|x|,  |d rstd| / rstd <= (K + 8) u + (d mean * rstd)^2
  z            |d z| <= |gamma| (rstd |d mean| + |h| ((K + 8) u + 4 u)) + 4 u (|gamma h| + |beta|)
  y            slopes are at most 1.13; the activations' own error is at most E u (1 + |z|): exp and the reciprocal are
               good to 2 steps each and erf to 4, and the bf16 kernels' exponent is rounded once more, (1.5 |z| or, in the
               Gaussian, 0.75 z^2) u of the result, hence E = 16 (bf16: + 2 z^2)
  storing      one rounding: half a step of the stored type, eps / 2
and in the backward pass, from given statistics, the same terms carried through dx = rstd (t - m1 - h m2)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import norm_oracle as N

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
ACTS = ["none", "relu", "silu", "gelu"]
U, K = 2.0 ** -24, 256


@pytest.fixture(scope="module")
def ua():
    import unet_amd
    unet_amd.lib()
    return unet_amd


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(seed, *shape, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale + shift


def place(t, dtype, before=0, after=0, fill=float("nan")):
    """A (B,H,W,C) tensor in a GPU buffer of the library's layout with `before` channels in front of it and `after`
    behind; those and the padding channels hold `fill`."""
    B, H, W, C = t.shape
    buf = torch.full((B, H, W, before + N.pad_ch(C) + after), fill, dtype=dtype)
    buf[..., before:before + C] = t.to(dtype)
    return buf.cuda()


def check_padding(y, C, off=0):
    pad = y[..., off + C:off + N.pad_ch(C)]
    assert pad.numel() == 0 or (pad == 0).all()


def within(got, want, bound, what):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), ((got - want).abs() / bound).nan_to_num(posinf=1e30).max().item(),
                           got[bad][:4], want[bad][:4])


def stats_bounds(x, mean, rstd, groups):
    cg = x.shape[3] // groups
    dm = K * U * N._group_mean(x.abs(), groups) + U * mean.abs()
    dr = rstd * ((K + 8) * U + (dm * rstd) ** 2)
    return dm, dr, cg


def act_error(z, dtype):
    return (16 + (2 * z * z if dtype == torch.bfloat16 else 0)) * U * (1 + z.abs())


def fwd_bound(x, y, z, mean, rstd, gamma, beta, groups, dtype, factor=1.0):
    dm, dr, cg = stats_bounds(x, mean, rstd, groups)
    pc = lambda t: N._per_channel(t, cg)
    h = (x - pc(mean)) * pc(rstd)
    dz = gamma.abs() * (pc(rstd * dm) + h.abs() * (pc(dr / rstd) + 4 * U)) + 4 * U * ((gamma * h).abs() + beta.abs())
    return factor * (1.13 * dz + act_error(z, dtype)) + (half_step(dtype) + 4 * U) * y.abs() + 1e-37


def bwd_bounds(p, gamma, beta, dtype):
    dz_in = 8 * U * ((gamma * p["h"]).abs() + beta.abs())
    dslope = 1.2 * dz_in + act_error(p["z"], dtype) * 2
    ddz = p["da"].abs() * dslope + 8 * U * p["dz"].abs()
    dt = gamma.abs() * ddz + 2 * U * p["t"].abs()
    return ddz, dt


def bwd_check(ops_out, x, dy, mean, rstd, groups, gamma, beta, kind, factor, dtype, what):
    dx, dg, db = ops_out
    C = x.shape[3]
    odx, odg, odb, p = N.group_norm_act_bwd(x, dy, mean, rstd, groups, gamma, beta, kind, factor)
    ddz, dt = bwd_bounds(p, gamma, beta, dtype)
    cg = C // groups
    gm = lambda t: N._per_channel(N._group_mean(t, groups), cg)
    bound = p["r"] * (dt + gm(dt) + p["h"].abs() * gm(dt * p["h"].abs()) + K * U * (p["a1"] + p["h"].abs() * p["a2"])
                      + 8 * U * (p["t"].abs() + p["m1"].abs() + (p["h"] * p["m2"]).abs()))
    within(dx[..., :C], odx, bound + half_step(dtype) * odx.abs() + 1e-37, what + ": dx")
    check_padding(dx, C)
    if dg is not None:
        hb = p["h"].abs()
        within(dg, odg, (ddz * hb + (K + 8) * U * (p["dz"] * p["h"]).abs()).sum((0, 1, 2)) + 1e-37, what + ": dweight")
    if db is not None:
        within(db, odb, (ddz + K * U * p["dz"].abs()).sum((0, 1, 2)) + 1e-37, what + ": dbias")


SHAPES = [  # B, H, W, C, groups
    (1, 1, 1, 1, 1), (3, 1, 1, 32, 4), (2, 1, 2, 5, 5), (1, 64, 64, 32, 8), (2, 23, 23, 40, 5), (3, 9, 7, 72, 6),
    (2, 16, 16, 64, 1), (2, 8, 8, 64, 64), (4, 4, 4, 512, 8), (2, 2, 2, 1024, 32), (1, 3, 5, 1040, 2), (1, 12, 11, 33, 3),
    (2, 70, 67, 36, 9), (5, 5, 5, 100, 25), (130, 2, 2, 48, 3), (1, 128, 128, 32, 8), (1, 7, 1, 528, 1), (2, 6, 6, 2080, 13),
    (1, 200, 210, 24, 2), (17, 16, 16, 128, 32), (18, 64, 64, 64, 32), (9, 64, 60, 48, 6), (33, 20, 20, 96, 12),
    (257, 7, 7, 512, 8), (8, 4, 4, 1024, 32), (7, 23, 23, 96, 8), (3, 64, 64, 64, 8), (5, 16, 16, 64, 8), (40, 7, 5, 56, 56),
    (1, 130, 255, 100, 20), (1, 256, 255, 66, 3),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ACTS)
def test_norm_forward_and_backward(ua, dtype, shape, kind):
    B, H, W, C, G = shape
    ops = ua.ops
    x = (rnd(1, B, H, W, C) + rnd(2, C)).to(dtype)
    gamma, beta = rnd(3, C, scale=0.3, shift=1.0), rnd(4, C, scale=0.3)
    dy = rnd(5, B, H, W, C, scale=0.1).to(dtype)
    y, mean, rstd = ops.group_norm_act_fwd(place(x, dtype), C, G, gamma.cuda(), beta.cuda(), act=kind)
    assert y.shape == (B, H, W, N.pad_ch(C)) and y.dtype == dtype and mean.shape == rstd.shape == (B, G)
    x6, g6, b6 = x.double(), gamma.double(), beta.double()
    oy, omean, orstd, z = N.group_norm_act_fwd(x6, G, g6, b6, kind, float(torch.tensor(1e-5)))
    dm, dr, _ = stats_bounds(x6, omean, orstd, G)
    within(mean, omean, dm + 1e-37, "mean")
    within(rstd, orstd, dr, "rstd")
    within(y[..., :C], oy, fwd_bound(x6, oy, z, omean, orstd, g6, b6, G, dtype), "y")
    check_padding(y, C)
    m, r = omean.float(), orstd.float()
    out = ops.group_norm_act_bwd(place(x, dtype), place(dy, dtype), m.cuda(), r.cuda(), C, G, gamma.cuda(), beta.cuda(), act=kind)
    bwd_check(out, x6, dy.double(), m.double(), r.double(), G, g6, b6, kind, None, dtype, f"{shape} {kind}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per_channel", [False, True])
@pytest.mark.parametrize("shape", [(2, 9, 7, 40, 5), (3, 32, 32, 32, 8), (1, 130, 67, 64, 4), (4, 4, 4, 520, 1)])
def test_norm_with_dropout_in_views(ua, dtype, per_channel, shape):
    """Channel ranges of wider buffers in and out, dropout fused: forward equals the norm followed by the stand-alone
    dropout (bit for bit in fp32, where nothing is rounded between), the other half of the output buffer stays."""
    B, H, W, C, G = shape
    ops, Cp = ua.ops, N.pad_ch(C)
    x, dy = rnd(1, B, H, W, C).to(dtype), rnd(5, B, H, W, C, scale=0.1).to(dtype)
    gamma, beta = rnd(3, C, scale=0.3, shift=1.0), rnd(4, C, scale=0.3)
    p, seed, offset = 0.3, (5 << 40) + 77, (3 << 35) + 1
    step = torch.tensor([4], device="cuda")
    drop = ops.Drop(p, seed, offset - 4, offset_dev=step, per_channel=per_channel)
    xb = place(x, dtype, before=Cp)
    out = torch.full((B, H, W, 2 * Cp), 7.0, device="cuda", dtype=dtype)
    y, mean, rstd = ops.group_norm_act_fwd(xb, C, G, gamma.cuda(), beta.cuda(), act="silu", drop=drop, x_coff=Cp, out=out)
    assert y is out and (out[..., Cp:] == 7).all()
    factor = N.drop_factor((B, H, W, C), p, seed, offset, per_channel)
    assert torch.equal(y[..., :C].cpu() == 0, factor == 0) or dtype == torch.bfloat16
    oy, om, orr, z = N.group_norm_act_fwd(x.double(), G, gamma.double(), beta.double(), "silu", float(torch.tensor(1e-5)), factor)
    within(y[..., :C], oy, fwd_bound(x.double(), oy, z, om, orr, gamma.double(), beta.double(), G, dtype, factor), "y")
    check_padding(y, C)
    plain, _, _ = ops.group_norm_act_fwd(xb, C, G, gamma.cuda(), beta.cuda(), act="silu", x_coff=Cp)
    if dtype == torch.float32:
        assert torch.equal(ops.dropout_fwd(plain, C, drop), y[..., :Cp])
    m, r = om.float(), orr.float()
    got = ops.group_norm_act_bwd(xb, place(dy, dtype, before=16, after=32), m.cuda(), r.cuda(), C, G, gamma.cuda(), beta.cuda(),
                                 act="silu", drop=drop, x_coff=Cp, dy_coff=16)
    bwd_check(got, x.double(), dy.double(), m.double(), r.double(), G, gamma.double(), beta.double(), "silu", factor, dtype, "views")


def test_norm_without_parameters_and_with_accumulation(ua):
    ops = ua.ops
    B, H, W, C, G = 2, 6, 5, 40, 4
    x, dy = rnd(1, B, H, W, C), rnd(2, B, H, W, C)
    xb, dyb = place(x, torch.float32), place(dy, torch.float32)
    one, zero = torch.ones(C), torch.zeros(C)
    y, m, r = ops.group_norm_act_fwd(xb, C, G, act="gelu")
    y1, _, _ = ops.group_norm_act_fwd(xb, C, G, one.cuda(), zero.cuda(), act="gelu")
    assert torch.equal(y, y1)
    dx, none_w, none_b = ops.group_norm_act_bwd(xb, dyb, m, r, C, G, act="gelu")
    assert none_w is None and none_b is None
    dx1, dw, db = ops.group_norm_act_bwd(xb, dyb, m, r, C, G, one.cuda(), zero.cuda(), act="gelu")
    assert torch.equal(dx, dx1)
    w0, b0 = rnd(7, C).cuda(), rnd(8, C).cuda()
    _, aw, ab = ops.group_norm_act_bwd(xb, dyb, m, r, C, G, one.cuda(), zero.cuda(), act="gelu", dweight=w0.clone(),
                                       dbias=b0.clone(), alpha=0.5, beta=2.0)
    for got, first, new in ((aw, w0, dw), (ab, b0, db)):
        want = 0.5 * new.double() + 2 * first.double()
        within(got, want.cpu(), (4 * U * (0.5 * new.abs() + 2 * first.abs())).double().cpu() + 1e-30, "accumulated")
    only_w = ops.group_norm_act_bwd(xb, dyb, m, r, C, G, one.cuda(), None, act="gelu")
    assert torch.equal(only_w[1], dw) and only_w[2] is None


def test_norm_far_from_zero(ua):
    """A mean 10^4 standard deviations from zero costs the digits that x itself has not, and no more."""
    ops = ua.ops
    x = (rnd(1, 2, 33, 31, 32) + 1e4)
    y, mean, rstd = ops.group_norm_act_fwd(place(x, torch.float32), 32, 8)
    oy, om, orr, z = N.group_norm_act_fwd(x.double(), 8, torch.ones(32).double(), torch.zeros(32).double(), "none", float(torch.tensor(1e-5)))
    dm, dr, _ = stats_bounds(x.double(), om, orr, 8)
    within(mean, om, dm, "mean")
    within(rstd, orr, dr, "rstd")
    assert ((rstd.double().cpu() / orr - 1).abs() < 1e-5).all()
    # means are x0 + (mean of small differences), rounded once per tile and once at the end
    within(mean, om, 2 * U * om.abs() + K * U * 8, "mean")


def test_constant_groups_and_single_values(ua):
    """Variance zero: z = beta exactly, and a group of one value passes no gradient."""
    ops = ua.ops
    x = torch.full((2, 3, 3, 32), 5.25)
    beta = rnd(1, 32)
    y, mean, rstd = ops.group_norm_act_fwd(place(x, torch.float32), 32, 4, torch.ones(32).cuda(), beta.cuda())
    assert torch.equal(y.cpu(), beta.expand(2, 3, 3, 32)) and (mean == 5.25).all()
    x1, dy = rnd(2, 4, 1, 1, 48), rnd(3, 4, 1, 1, 48)
    xb = place(x1, torch.float32)
    w = rnd(4, 48).cuda()
    _, m, r = ops.group_norm_act_fwd(xb, 48, 48, w)
    dx, dw, _ = ops.group_norm_act_bwd(xb, place(dy, torch.float32), m, r, 48, 48, w)
    assert (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_stay_in_their_group(ua, bad):
    ops = ua.ops
    B, H, W, C, G = 2, 40, 20, 40, 5
    x = rnd(1, B, H, W, C)
    clean, m0, r0 = ops.group_norm_act_fwd(place(x, torch.float32), C, G, act="relu")
    x[1, 39, 19, 17] = bad                                        # group 2, the last pixel of the last image
    y, m, r = ops.group_norm_act_fwd(place(x, torch.float32), C, G, act="relu")
    hit = torch.zeros(B, H, W, N.pad_ch(C), dtype=torch.bool)
    hit[1, ..., 16:24] = True
    assert torch.equal(y.cpu()[~hit], clean.cpu()[~hit])
    assert not torch.isfinite(r[1, 2]) and not torch.isfinite(m[1, 2])
    assert torch.isnan(y.cpu()[1, ..., 16:24]).all()
    dy = rnd(3, B, H, W, C)
    dx, dw, db = ops.group_norm_act_bwd(place(x, torch.float32), place(dy, torch.float32), m, r, C, G, act="none")
    assert torch.isfinite(dx.cpu()[~hit]).all()


def test_relu_gate_is_settled_in_64_bits(ua):
    """beta chosen so that z lies within fp32 rounding of zero on both sides: the gate follows the exact sign."""
    ops = ua.ops
    H, W, C = 32, 32, 32
    x, dy = rnd(1, 1, H, W, C), torch.ones(1, H, W, C)
    gamma = rnd(2, C, scale=0.2, shift=1.0)
    mean, rstd = torch.full((1, 1), 0.1), torch.full((1, 1), 0.7)
    z0 = ((x - 0.1).double() * 0.7 * gamma.double())
    beta = -z0[0, 5, 7].float()                                  # per channel: pixel (5, 7) lands on the border
    x[0, 5, 8:20] = x[0, 5, 7] + rnd(3, 12, C) * 2.0 ** -23      # and its neighbours around it
    _, _, _, p = N.group_norm_act_bwd(x.double(), dy.double(), mean.double(), rstd.double(), 1, gamma.double(), beta.double(), "relu")
    assert int((p["z"].abs() < 1e-6).sum()) >= 8 * C
    _, _, db = ops.group_norm_act_bwd(place(x, torch.float32), place(dy, torch.float32), mean.cuda(), rstd.cuda(), C, 1,
                                      gamma.cuda(), beta.cuda(), act="relu")
    assert torch.equal(db.cpu().double(), (p["z"] > 0).double().sum((0, 1, 2)))              # counts: exact in fp32


def test_results_repeat(ua):
    ops = ua.ops
    for shape in ((7, 61, 59, 72, 6), (300, 8, 8, 64, 8), (1, 256, 256, 32, 8)):
        B, H, W, C, G = shape
        x, dy = place(rnd(1, B, H, W, C), torch.bfloat16), place(rnd(2, B, H, W, C), torch.bfloat16)
        w, b = rnd(3, C).cuda(), rnd(4, C).cuda()
        drop = ops.Drop(0.2, 9)
        runs = []
        for _ in range(3):
            y, m, r = ops.group_norm_act_fwd(x, C, G, w, b, act="gelu", drop=drop)
            runs.append((y, m, r) + ops.group_norm_act_bwd(x, dy, m, r, C, G, w, b, act="gelu", drop=drop))
        for other in runs[1:]:
            assert all(torch.equal(s, t) for s, t in zip(runs[0], other))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ACTS)
def test_sums_of_parts_that_have_not_come(ua, monkeypatch, dtype, kind):
    """Images that several workgroups share, with no patience for each other: a workgroup that looks for the others' sums
    once only forms the missing ones itself, and every bit is the same."""
    ops = ua.ops
    for B, H, W, C, G in ((3, 190, 150, 32, 8), (40, 80, 60, 48, 1), (2, 128, 128, 40, 5), (300, 33, 32, 32, 2), (1, 256, 256, 32, 32)):
        x, dy = place(rnd(1, B, H, W, C, shift=3.0), dtype), place(rnd(2, B, H, W, C), dtype)
        w, b = rnd(3, C).cuda(), rnd(4, C).cuda()
        drop = ops.Drop(0.2, 9)
        y, m, r = ops.group_norm_act_fwd(x, C, G, w, b, act=kind, drop=drop)
        want = (y, m, r) + ops.group_norm_act_bwd(x, dy, m, r, C, G, w, b, act=kind, drop=drop)
        monkeypatch.setattr(ops, "_POLLS", 0)
        for _ in range(2):
            y, m, r = ops.group_norm_act_fwd(x, C, G, w, b, act=kind, drop=drop)
            got = (y, m, r) + ops.group_norm_act_bwd(x, dy, m, r, C, G, w, b, act=kind, drop=drop)
            assert all(torch.equal(s, t) for s, t in zip(want, got)), (B, H, W, C, G)
        monkeypatch.setattr(ops, "_POLLS", -1)


def test_workgroups_that_share_an_image_run_together(ua, monkeypatch):
    """More workgroups than can run at a time, in many chunks and parts: none may wait for one that comes much later (then
    a call takes as long as their patience, 0.3 s; together they take 0.2 ms)."""
    ops = ua.ops
    B, H, W, C, G = 3, 128, 128, 1024, 1024
    gen = torch.Generator("cuda").manual_seed(1)
    x, dy = (torch.randn(B, H, W, C, device="cuda", generator=gen) for _ in range(2))
    for _ in range(3):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        y, m, r = ops.group_norm_act_fwd(x, C, G, act="relu")
        dx, _, _ = ops.group_norm_act_bwd(x, dy, m, r, C, G, act="relu")
        end.record()
        torch.cuda.synchronize()
    assert start.elapsed_time(end) < 30.0
    monkeypatch.setattr(ops, "_POLLS", 0)
    z, m2, r2 = ops.group_norm_act_fwd(x, C, G, act="relu")
    assert torch.equal(y, z) and torch.equal(m, m2) and torch.equal(r, r2)
    assert torch.equal(dx, ops.group_norm_act_bwd(x, dy, m, r, C, G, act="relu")[0])


def test_gradient_against_differences(ua):
    """<dL/dv, d> against (L(v + e d) - L(v - e d)) / 2 e for L = sum(dy * y), y from the kernel, v each input.
    The central difference is off by e^2 |L'''| / 6 (e = 2^-6, third derivatives of order 10 |d|^3 here: below 1e-3 of
    the sum's scale) and by the rounding of L, 2 L u K / e; both together stay below 1 % of |grad| |d|."""
    ops = ua.ops
    B, H, W, C, G, e = 2, 6, 5, 40, 4, 2.0 ** -6
    dt = torch.float32
    x, w, b, dy = rnd(1, B, H, W, C), rnd(2, C, scale=0.3, shift=1.0), rnd(3, C, scale=0.3), rnd(4, B, H, W, C)
    for kind in ("none", "silu", "gelu"):
        for drop in (None, ops.Drop(0.25, 3), ops.Drop(0.25, 3, per_channel=True)):
            def L(x, w, b):
                y, _, _ = ops.group_norm_act_fwd(place(x, dt, fill=0.0), C, G, w.cuda(), b.cuda(), act=kind, drop=drop)
                return (y[..., :C].double().cpu() * dy.double()).sum()
            xb = place(x, dt)
            _, m, r = ops.group_norm_act_fwd(xb, C, G, w.cuda(), b.cuda(), act=kind, drop=drop)
            grads = ops.group_norm_act_bwd(xb, place(dy, dt), m, r, C, G, w.cuda(), b.cuda(), act=kind, drop=drop)
            grads = (grads[0][..., :C].double().cpu(), grads[1].double().cpu(), grads[2].double().cpu())
            for i, (v, g) in enumerate(zip((x, w, b), grads)):
                d = torch.sign(g).float() * (0.1 if i == 0 else 1.0)      # along the gradient: nothing cancels
                args = [x, w, b]
                args[i] = v + e * d
                up = L(*args)
                args[i] = v - e * d
                diff = (up - L(*args)) / (2 * e)
                want = (g * d.double()).sum()
                assert abs(diff - want) <= 0.01 * want.abs(), (kind, i, diff, want)


# ---------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per_channel", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (2, 3, 5, 7), (1, 4, 4, 512), (3, 27, 24, 40), (2, 64, 64, 32), (1, 2, 2, 1040)])
def test_dropout(ua, dtype, per_channel, shape):
    ops = ua.ops
    B, H, W, C = shape
    Cp = N.pad_ch(C)
    x, r = rnd(1, *shape).to(dtype), rnd(2, *shape).to(dtype)
    for p, seed, offset in ((0.2, 1, 0), (0.5, (1 << 64) - 1, (1 << 64) - 2), (1e-3, 12345 << 20, 3 << 40), (0.0, 1, 0), (1.0, 1, 0),
                            (2.0 ** -17, 1, 0), (1 - 2.0 ** -17, 5, 5)):
        drop = ops.Drop(p, seed, offset, per_channel=per_channel)
        factor = N.drop_factor(shape, p, seed, offset, per_channel)
        scale = half_step(dtype) + 2 * U
        y = ops.dropout_fwd(place(x, dtype, before=16, after=16), C, drop, x_coff=16)
        want = x.double() * factor
        assert torch.equal(y[..., :C].cpu() != 0, (want != 0))
        within(y[..., :C], want, scale * want.abs(), "dropout")
        check_padding(y, C)
        assert torch.equal(ops.dropout_bwd(place(x, dtype), C, drop), y)
        out = torch.full((B, H, W, 2 * Cp), 7.0, device="cuda", dtype=dtype)
        z = ops.dropout_fwd(place(x, dtype), C, drop, residual=place(r, dtype, before=32), residual_coff=32, out=out, out_coff=Cp)
        assert (out[..., :Cp] == 7).all()
        within(z[..., Cp:Cp + C], want + r.double(), scale * (want + r.double()).abs() + 2 * U * (want.abs() + r.double().abs()), "residual")
        check_padding(z, C, Cp)


def test_dropout_in_place_and_non_finite(ua):
    ops = ua.ops
    x = rnd(1, 2, 6, 7, 64)
    x[0, 0, 0, :8] = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e38, -1e38, 1e-40])
    x[1, 5, 6] = float("nan")
    drop = ops.Drop(0.5, 3)
    keep = N.drop_factor((2, 6, 7, 64), 0.5, 3) > 0
    buf = x.cuda()
    want = ops.dropout_fwd(buf, 64, drop)
    assert (want.cpu()[~keep] == 0).all() and torch.isnan(want.cpu()[1, 5, 6][keep[1, 5, 6]]).all()
    r = rnd(2, 2, 6, 7, 64).cuda()
    both = ops.dropout_fwd(buf, 64, drop, residual=r)
    inplace = r.clone()
    assert ops.dropout_fwd(buf, 64, drop, residual=inplace, out=inplace) is inplace
    assert torch.equal(inplace.nan_to_num(nan=123.0), both.nan_to_num(nan=123.0))
    assert ops.dropout_fwd(buf, 64, drop, out=buf) is buf
    assert torch.equal(buf.nan_to_num(nan=123.0), want.nan_to_num(nan=123.0))


def test_offset_on_the_device(ua):
    ops = ua.ops
    x = rnd(1, 2, 8, 8, 32).cuda()
    for add, host in ((0, 7), (5, 2), (-3, 10), (1, (1 << 64) - 1)):
        dev = torch.tensor([add], device="cuda")
        a = ops.dropout_fwd(x, 32, ops.Drop(0.5, 9, host, offset_dev=dev))
        assert torch.equal(a, ops.dropout_fwd(x, 32, ops.Drop(0.5, 9, (host + add) % (1 << 64))))


def test_positions_beyond_32_bits(ua):
    """2^31 + 2^28 elements (element offsets and unit numbers pass 2^31, byte offsets 2^32): the last pixels of the last
    image, against the oracle at their own unit numbers; and the norm's output there from its own statistics."""
    ops = ua.ops
    B, H, W, C = 9, 2896, 2896, 32                               # 2.4e9 elements, 4.8 GB in bf16
    x = torch.empty((B, H, W, C), device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator("cuda").manual_seed(1))
    drop = ops.Drop(0.5, 77, 3)
    y = ops.dropout_fwd(x, C, drop)
    n = 1000
    first = B * H * W - n
    units = (np.arange(first, first + n, dtype=np.uint64)[:, None] * np.uint64(32) + np.arange(32, dtype=np.uint64)[None])
    keep = torch.from_numpy(N.units_kept(units, 0.5, 77, 3))
    tail_x, tail_y = x.view(-1, C)[first:].cpu(), y.view(-1, C)[first:].cpu()
    assert torch.equal(tail_y, torch.where(keep, tail_x * 2, torch.zeros_like(tail_x)))
    y, mean, rstd = ops.group_norm_act_fwd(x, C, 8, act="relu", drop=drop)
    h = (tail_x.double() - mean[-1].cpu().double().repeat_interleave(4)) * rstd[-1].cpu().double().repeat_interleave(4)
    want = torch.where(keep, h.clamp_min(0) * 2, torch.zeros_like(h))
    within(y.view(-1, C)[first:], want, (half_step(torch.bfloat16) + 8 * U) * want.abs() + 1e-37, "tail of the norm")
    assert (mean.abs() < 6 / (H * W * 4) ** 0.5).all() and ((rstd - 1).abs() < 1e-3).all()
    dx, _, _ = ops.group_norm_act_bwd(x, x, mean, rstd, C, 8, act="none")
    # dy = x = h / rstd + mean: dx = rstd (x - mean(x) - h mean(x h)) = 0 up to the roundings of terms of size |x|
    assert dx.view(-1, C)[first:].abs().max() < 2e-3


# ---------------------------------------------------------------- as a program uses them
def test_modules_and_autograd(ua):
    B, H, W, C, G = 2, 6, 5, 40, 5
    m = ua.GroupNormAct(G, C, act="silu", p=0.25).cuda()
    with torch.no_grad():
        m.weight.copy_(rnd(1, C, scale=0.3, shift=1.0))
        m.bias.copy_(rnd(2, C, scale=0.3))
    d = ua.Dropout(C, 0.5, per_channel=True)
    x = place(rnd(3, B, H, W, C), torch.float32, fill=0.0).requires_grad_()
    skip = place(rnd(4, B, H, W, C), torch.float32, after=16, fill=0.0).requires_grad_()
    torch.manual_seed(8)
    out = d(m(x), skip)
    torch.manual_seed(8)
    assert torch.equal(out, d(m(x), skip))
    assert not torch.equal(out, d(m(x), skip))
    torch.manual_seed(8)
    s1, s2 = ua.layers.fresh_drop(0.25).seed, ua.layers.fresh_drop(0.5).seed
    f1, f2 = N.drop_factor((B, H, W, C), 0.25, s1), N.drop_factor((B, H, W, C), 0.5, s2, per_channel=True)
    out.sum().backward()                                          # the gradient arrives as an expanded scalar, ones in the padding too
    x6, w6, b6 = x.detach()[..., :C].double().cpu(), m.weight.detach().double().cpu(), m.bias.detach().double().cpu()
    oy, om, orr, _ = N.group_norm_act_fwd(x6, G, w6, b6, "silu", float(torch.tensor(1e-5)), f1)
    odx, odw, odb, _ = N.group_norm_act_bwd(x6, f2, om, orr, G, w6, b6, "silu", f1)
    close = lambda a, b: torch.allclose(a.double().cpu(), b, rtol=1e-4, atol=1e-5)
    assert close(out.detach()[..., :C], oy * f2 + skip.detach()[..., :C].double().cpu())
    assert close(x.grad[..., :C], odx) and close(m.weight.grad, odw) and close(m.bias.grad, odb)
    want_skip = torch.zeros_like(skip)
    want_skip[..., :C] = 1
    assert torch.equal(skip.grad, want_skip) and (x.grad[..., C:] == 0).all()
    m.eval(), d.eval()
    with torch.no_grad():
        y = d(m(x))
    oy, _, _, _ = N.group_norm_act_fwd(x6, G, w6, b6, "silu", float(torch.tensor(1e-5)))
    assert close(y[..., :C], oy)
    # nothing is kept of the mask: x, two statistics and the parameters
    y = ua.group_norm_act(x, C, G, m.weight, m.bias, "silu", drop=ua.ops.Drop(0.5, 1))
    saved = [t for t in y.grad_fn.saved_tensors if t is not None]
    assert sum(t.numel() for t in saved) == x.numel() + 2 * C + 2 * B * G


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_block_as_a_program_runs_it(ua, dtype):
    """conv3x3 -> group norm, ReLU, dropout -> conv3x3 -> group norm, SiLU -> dropout + skip -> MSE-like gradient back
    through every operator, against the same block in float64 torch on the CPU with the oracle's masks."""
    ops = ua.ops
    B, H, W, C, G, p = 3, 16, 16, 64, 8, 0.2
    dev = "cuda"
    x, dy = rnd(1, B, H, W, C).to(dtype), rnd(2, B, H, W, C, scale=0.1).to(dtype)
    w1, w2 = (rnd(s, C, C, 3, 3, scale=0.05).to(dtype).float() for s in (3, 4))
    g1, b1, g2, b2 = rnd(5, C, scale=0.2, shift=1.0), rnd(6, C, scale=0.2), rnd(7, C, scale=0.2, shift=1.0), rnd(8, C, scale=0.2)
    d1, d2 = ops.Drop(p, 99, 0), ops.Drop(p, 99, 1)
    zero = torch.zeros(C, device=dev)
    xg = place(x, dtype)
    f1, k1 = ops.pack_conv3x3(w1.to(dev), dtype)
    f2, k2 = ops.pack_conv3x3(w2.to(dev), dtype)
    G1, B1, G2, B2 = (t.to(dev) for t in (g1, b1, g2, b2))
    u1 = ops.conv3x3_relu_fwd(xg, f1, zero, C, C, relu=False)
    a1, m1, r1 = ops.group_norm_act_fwd(u1, C, G, G1, B1, act="relu", drop=d1)
    u2 = ops.conv3x3_relu_fwd(a1, f2, zero, C, C, relu=False)
    a2, m2, r2 = ops.group_norm_act_fwd(u2, C, G, G2, B2, act="silu")
    out = ops.dropout_fwd(a2, C, d2, residual=xg)
    dyg = place(dy, dtype)
    da2 = ops.dropout_bwd(dyg, C, d2)
    du2, dg2, db2 = ops.group_norm_act_bwd(u2, da2, m2, r2, C, G, G2, B2, act="silu")
    dw2, _ = ops.conv3x3_wgrad(a1, du2, C, C)
    da1 = ops.conv3x3_dgrad(du2, k2, C, C)
    du1, dg1, db1 = ops.group_norm_act_bwd(u1, da1, m1, r1, C, G, G1, B1, act="relu", drop=d1)
    dw1, _ = ops.conv3x3_wgrad(xg, du1, C, C)
    dx = ops.dropout_fwd(ops.conv3x3_dgrad(du1, k1, C, C), C, None, residual=dyg)

    nchw = lambda t: t.double().permute(0, 3, 1, 2)
    fac = [nchw(N.drop_factor((B, H, W, C), p, 99, o)) for o in (0, 1)]
    leaves = [t.double().requires_grad_() for t in (nchw(x), w1, w2, g1, b1, g2, b2)]
    X, W1, W2, A, Bb, Cc, D = leaves
    ref = F.relu(F.group_norm(F.conv2d(X, W1, padding=1), G, A, Bb)) * fac[0]
    ref = F.silu(F.group_norm(F.conv2d(ref, W2, padding=1), G, Cc, D)) * fac[1] + X
    want = torch.autograd.grad(ref, leaves, nchw(dy))
    got = [nchw(dx.cpu()), dw1, dw2, dg1, db1, dg2, db2]
    rel = lambda a, b: ((a.double().cpu() - b).norm() / b.norm()).item()
    # bf16: each of the ten tensors stored on the way is off by at most 2^-8 of itself, the mean square of a rounding is a
    # third of that, and conv and norm pass relative errors on: 10 * 2^-8 / 3 ~ 1.3e-2.  ReLU gates that the forward
    # rounding turns (a share of ~2^-8 of the units, each with a gradient of ordinary size) add sqrt(2^-8) ~ 6e-2 behind
    # the gate.  fp32: the same with 2^-24, and a turned gate among 49,152 has probability ~1e-2 x its share 4.5e-3.
    assert rel(nchw(out.cpu()), ref.detach()) < (1.3e-2 if dtype == torch.bfloat16 else 2e-6)
    for i, (a, b) in enumerate(zip(got, want)):
        assert rel(a, b) < (8e-2 if dtype == torch.bfloat16 else 5e-6), i


def test_streams_and_graph_replay(ua):
    """Two streams at once, and a captured training step replayed with the program's eager work between: every replay has
    the mask of the counter's value at the time, and equals the eager call with that offset."""
    ops = ua.ops
    B, H, W, C, G = 4, 24, 24, 64, 8
    x, dy = rnd(1, B, H, W, C).cuda(), rnd(2, B, H, W, C).cuda()
    w, b = rnd(3, C, shift=1.0).cuda(), rnd(4, C).cuda()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def train(drop, drop2):
        y, m, r = ops.group_norm_act_fwd(x, C, G, w, b, act="silu", drop=drop)
        z = ops.dropout_fwd(y, C, drop2, residual=x)
        d = ops.dropout_bwd(dy, C, drop2)
        return (z,) + ops.group_norm_act_bwd(x, d, m, r, C, G, w, b, act="silu", drop=drop)

    def eager(n):
        return train(ops.Drop(0.3, 5, 100 + n), ops.Drop(0.3, 6, 100 + n))
    captured = ops.Drop(0.3, 5, 100, offset_dev=step), ops.Drop(0.3, 6, 100, offset_dev=step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [train(*captured) for _ in range(3)]
    on_main = [eager(0) for _ in range(3)]
    torch.cuda.synchronize()
    for a, c in zip(on_side, on_main):
        assert all(torch.equal(s, t) for s, t in zip(a, c))
    graphs = []
    for _ in range(2):                                            # two graphs share their memory pool, like two captured steps
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            out = train(*captured)
            step.add_(1)
        graphs.append((g, out))
    for n in range(6):
        g, out = graphs[n % 2]
        step.fill_(n)
        g.replay()
        torch.cuda.synchronize()
        assert step.item() == n + 1
        assert all(torch.equal(s, t) for s, t in zip(out, eager(n))), n


@pytest.mark.parametrize("dtype", DTYPES)
def test_shared_images_on_two_streams_and_in_graphs(ua, dtype):
    """Images that several workgroups share: calls on two streams at once, and captured calls whose inputs change between
    replays (what the workgroups told each other in the replay before is then wrong)."""
    ops = ua.ops
    B, H, W, C, G = 5, 120, 110, 64, 8
    inputs = [(place(rnd(i, B, H, W, C, shift=float(i)), dtype), place(rnd(10 + i, B, H, W, C), dtype)) for i in range(3)]
    w, b = rnd(3, C, shift=1.0).cuda(), rnd(4, C).cuda()
    drop = ops.Drop(0.3, 5)

    def train(x, dy):
        y, m, r = ops.group_norm_act_fwd(x, C, G, w, b, act="silu", drop=drop)
        return (y, m, r) + ops.group_norm_act_bwd(x, dy, m, r, C, G, w, b, act="silu", drop=drop)
    want = [train(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for n in range(6):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(train(*inputs[(n + k) % 3]))
    torch.cuda.synchronize()
    for k in range(2):
        for n, out in enumerate(got[k]):
            assert all(torch.equal(s, t) for s, t in zip(out, want[(n + k) % 3])), (k, n)
    x, dy = (t.clone() for t in inputs[0])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            out = train(x, dy)
        graphs.append((g, out))
    for n in range(6):
        g, out = graphs[n % 2]
        x.copy_(inputs[n % 3][0])
        dy.copy_(inputs[n % 3][1])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(out, want[n % 3])), n
        train(*inputs[(n + 1) % 3])


def test_captured_autograd_step(ua):
    """Forward and backward of the modules captured through autograd, leaves' gradients and all."""
    C, G = 64, 8
    m = ua.GroupNormAct(G, C, act="gelu", p=0.2, offset_dev=torch.zeros(1, dtype=torch.int64, device="cuda")).cuda()
    x = rnd(1, 2, 8, 8, C).cuda().requires_grad_()
    dy = rnd(2, 2, 8, 8, C).cuda()
    leaves = (x, m.weight, m.bias)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(m(x), leaves, dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    torch.manual_seed(3)
    with torch.cuda.graph(g):
        y = m(x)
        grads = torch.autograd.grad(y, leaves, dy)
    torch.manual_seed(3)
    seed = ua.layers.fresh_drop(0.2).seed
    for n in range(4):
        m.offset_dev.fill_(n)
        g.replay()
        torch.cuda.synchronize()
        e = ua.group_norm_act(x, C, G, m.weight, m.bias, "gelu", m.eps, ua.ops.Drop(0.2, seed, n))
        assert torch.equal(y, e)
        assert all(torch.equal(a, c) for a, c in zip(grads, torch.autograd.grad(e, leaves, dy)))


def test_refusals_on_the_gpu(ua):
    ops = ua.ops
    x = torch.zeros(2, 4, 4, 64, device="cuda")
    drop = ops.Drop(0.5, 1)
    w = torch.ones(40, device="cuda")
    with pytest.raises(TypeError):
        ops.dropout_fwd(x.half(), 40, drop)
    with pytest.raises(TypeError):
        ops.group_norm_act_fwd(x.double(), 40, 5)
    for bad in (x[0], x.permute(0, 3, 1, 2), x[:, :, ::2]):
        with pytest.raises(ValueError, match="contiguous"):
            ops.dropout_fwd(bad, 40, drop)
        with pytest.raises(ValueError, match="contiguous"):
            ops.group_norm_act_fwd(bad, 40, 5)
    for bad in (w[:39], w.double(), w.cpu(), torch.ones(80, device="cuda")[::2]):
        with pytest.raises(ValueError, match="weight"):
            ops.group_norm_act_fwd(x, 40, 5, bad)
    for bad in (x[:1], x.bfloat16(), x[:, :2].contiguous()):
        with pytest.raises(ValueError, match="does not go with"):
            ops.dropout_fwd(x, 40, drop, residual=bad)
        with pytest.raises(ValueError, match="does not go with"):
            ops.group_norm_act_fwd(x, 40, 5, out=bad)
        with pytest.raises(ValueError, match="does not go with"):
            ops.group_norm_act_bwd(x, bad, torch.zeros(2, 5, device="cuda"), torch.zeros(2, 5, device="cuda"), 40, 5)
    with pytest.raises(ValueError, match="statistics"):
        ops.group_norm_act_bwd(x, x.clone(), torch.zeros(2, 4, device="cuda"), torch.zeros(2, 5, device="cuda"), 40, 5)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.group_norm_act_fwd(x, 40, 5, out=x)
    with pytest.raises(RuntimeError, match="bad view"):
        ops.group_norm_act_fwd(x, 40, 5, x_coff=32)
    with pytest.raises(RuntimeError, match="bad view"):
        ops.dropout_fwd(x, 80, drop)
    with pytest.raises(RuntimeError, match="without being"):
        wide = torch.zeros(2, 4, 4, 128, device="cuda")
        ops.dropout_fwd(wide, 64, drop, out=wide, out_coff=32)
    with pytest.raises(ValueError, match="unknown activation"):
        ops.group_norm_act_fwd(x, 40, 5, act="swish")
    empty = torch.zeros(0, 4, 4, 48, device="cuda")
    y, m, r = ops.group_norm_act_fwd(empty, 40, 5, w, w)
    assert y.shape == (0, 4, 4, 48) and m.shape == (0, 5)
    dx, dw, db = ops.group_norm_act_bwd(empty, empty, m, r, 40, 5, w, w)
    assert dx.shape == (0, 4, 4, 48) and (dw == 0).all() and (db == 0).all()
    assert ops.dropout_fwd(empty, 40, drop).shape == (0, 4, 4, 48)
    torch.cuda.synchronize()


# ---------------------------------------------------------------- values whose squares pass fp32's range
LARGE = [(2, 8, 8, 64, 8), (5, 8, 8, 64, 16), (3, 9, 8, 72, 24), (2, 1, 1, 1024, 4), (1, 64, 64, 32, 8), (12, 90, 80, 32, 4), (9, 100, 96, 40, 8),
         (2, 70, 67, 36, 12), (1, 256, 255, 66, 6), (3, 256, 250, 64, 4)]      # one workgroup an image, several, the general kernels


def grouped(scales, B, C, G):
    """(B, 1, 1, C): a scale for each group, the next image's one further on."""
    s = torch.tensor([[scales[(b + g) % len(scales)] for g in range(G)] for b in range(B)], dtype=torch.float64)
    return N._per_channel(s, C // G)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", LARGE)
def test_norm_of_large_values(ua, monkeypatch, dtype, shape):
    """Finite groups whose sum of squares, or whose sum, fp32 does not hold, beside ordinary ones."""
    B, H, W, C, G = shape
    ops = ua.ops
    scale, shift = grouped([1.0, 1e18, 1e25, 2e36], B, C, G), grouped([0.0, 0.0, 1e27, 0.0, 1.0, 1e20], B, C, G)
    x = ((rnd(1, B, H, W, C) + rnd(2, C)) * scale + shift).to(dtype)
    assert torch.isfinite(x).all()
    gamma, beta = rnd(3, C, scale=0.3, shift=1.0), rnd(4, C, scale=0.3)
    y, mean, rstd = ops.group_norm_act_fwd(place(x, dtype), C, G, gamma.cuda(), beta.cuda(), act="silu")
    x6, g6, b6 = x.double(), gamma.double(), beta.double()
    oy, om, orr, z = N.group_norm_act_fwd(x6, G, g6, b6, "silu", float(torch.tensor(1e-5)))
    dm, dr, _ = stats_bounds(x6, om, orr, G)
    within(mean, om, dm + 1e-37, "mean")
    within(rstd, orr, dr, "rstd")
    within(y[..., :C], oy, fwd_bound(x6, oy, z, om, orr, g6, b6, G, dtype), "y")
    check_padding(y, C)
    monkeypatch.setattr(ops, "_POLLS", 0)
    again = ops.group_norm_act_fwd(place(x, dtype), C, G, gamma.cuda(), beta.cuda(), act="silu")
    assert all(torch.equal(s, t) for s, t in zip((y, mean, rstd), again))
    same = torch.full((B, H, W, C), 2.0 ** 100)                   # no deviations at all: z = beta
    y, mean, rstd = ops.group_norm_act_fwd(place(same, dtype), C, G, None, beta.cuda())
    assert (mean == 2.0 ** 100).all() and torch.equal(y[..., :C].float().cpu(), beta.to(dtype).float().expand(B, H, W, C))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 8, 8, 64, 8), (3, 1, 2, 64, 64), (2, 128, 128, 40, 5), (1, 256, 255, 66, 3)])
def test_relu_gate_without_deviation(ua, dtype, shape):
    """rstd = 0 (an infinite eps, or what a caller handed in): z = beta, so the gate is beta's sign."""
    B, H, W, C, G = shape
    x, dy, beta = rnd(1, B, H, W, C).to(dtype), torch.ones(B, H, W, C), rnd(2, C)
    beta[::7] = 0
    dx, dw, db = ua.ops.group_norm_act_bwd(place(x, dtype), place(dy, dtype), torch.zeros(B, G).cuda(), torch.zeros(B, G).cuda(), C, G,
                                           rnd(3, C).cuda(), beta.cuda(), act="relu")
    assert torch.equal(db.cpu(), (beta > 0).float() * (B * H * W))            # counts below 2^24: exact
    assert (dw == 0).all() and (dx == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 8, 8, 64, 8), (3, 1, 2, 64, 64), (2, 128, 128, 40, 5), (1, 256, 255, 66, 3)])
def test_relu_gate_of_groups_without_deviations(ua, dtype, shape):
    """x is the mean throughout, so z = beta: also where beta / (rstd gamma) is nothing next to the mean, in 64 bits too."""
    B, H, W, C, G = shape
    mean = torch.tensor([5.25, -5.25, 2.0 ** 60, -2.0 ** 60, 1.5e-3, 2.0 ** -70])[torch.arange(B * G) % 6].to(dtype).float().view(B, G)
    x = N._per_channel(mean, C // G).expand(B, H, W, C).contiguous()
    beta = rnd(2, C) * torch.tensor([1e-18, 1.0, 1e-30])[torch.arange(C) % 3]
    gamma = rnd(3, C)
    dy = torch.ones(B, H, W, C)
    rstd = torch.full((B, G), 1e-5).rsqrt()
    dx, dw, db = ua.ops.group_norm_act_bwd(place(x, dtype), place(dy, dtype), mean.cuda(), rstd.cuda(), C, G, gamma.cuda(), beta.cuda(),
                                           act="relu")
    assert torch.equal(db.cpu(), (beta > 0).float() * (B * H * W)) and (dw == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", LARGE)
@pytest.mark.parametrize("kind", ACTS)
def test_norm_backward_of_large_values(ua, monkeypatch, dtype, shape, kind):
    """Deviations whose squares fp32 does not hold: dx keeps all three of its terms."""
    B, H, W, C, G = shape
    ops = ua.ops
    scale, shift = grouped([1.0, 1e18, 1e25, 2e36], B, C, G), grouped([0.0, 0.0, 1e27, 0.0, 1.0, 1e20], B, C, G)
    x = ((rnd(1, B, H, W, C) + rnd(2, C)) * scale + shift).to(dtype)
    dy = rnd(5, B, H, W, C, scale=0.1).to(dtype)
    gamma, beta = rnd(3, C, scale=0.3, shift=1.0), rnd(4, C, scale=0.3)
    x6, g6, b6 = x.double(), gamma.double(), beta.double()
    _, om, orr, _ = N.group_norm_act_fwd(x6, G, g6, b6, kind, 1e-5)
    m, r = om.float(), orr.float()

    def call():
        return ops.group_norm_act_bwd(place(x, dtype), place(dy, dtype), m.cuda(), r.cuda(), C, G, gamma.cuda(), beta.cuda(), act=kind)
    out = call()
    bwd_check(out, x6, dy.double(), m.double(), r.double(), G, g6, b6, kind, None, dtype, f"{shape} {kind}")
    monkeypatch.setattr(ops, "_POLLS", 0)
    assert all(torch.equal(s, t) for s, t in zip(out, call()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p, training", [(0.5, False), (0.0, True), (0.0, False)])
def test_dropout_module_that_drops_nothing(ua, dtype, p, training):
    """Evaluation mode takes the widths that training mode takes and returns what it returns: padded channels, padding zero."""
    B, H, W, C = 2, 5, 6, 40
    d = ua.Dropout(C, p).train(training)
    x, r, dy = rnd(1, B, H, W, C).to(dtype), rnd(2, B, H, W, C).to(dtype), rnd(3, B, H, W, C).to(dtype)
    want = (x.double() + r.double()).to(dtype)
    for xa, ra in ((0, 16), (16, 0), (0, 0), (32, 16)):
        xb, rb = place(x, dtype, after=xa, fill=3.0).requires_grad_(), place(r, dtype, after=ra, fill=5.0).requires_grad_()
        y = d(xb, rb)
        assert y.shape == (B, H, W, 48) and y.dtype == dtype and torch.equal(y[..., :C].cpu(), want)
        check_padding(y, C)
        gx, gr = torch.autograd.grad(y, (xb, rb), place(dy, dtype, fill=7.0))
        for g, leaf in ((gx, xb), (gr, rb)):
            assert g.shape == leaf.shape and torch.equal(g[..., :C].cpu(), dy) and (g[..., C:] == 0).all()
    wide, narrow = place(x, dtype, after=16, fill=3.0), place(x, dtype, fill=3.0)
    y = d(wide)
    assert y.shape == (B, H, W, 48) and torch.equal(y[..., :C].cpu(), x)
    check_padding(y, C)
    assert d(narrow) is narrow
    with pytest.raises(ValueError, match="does not go with"):
        d(narrow, narrow.double())


def test_a_counter_changed_between_forward_and_backward_is_reported(ua):
    """Two forward passes with the count between them and one backward pass: the first one's mask is gone."""
    C, step = 64, torch.zeros(1, dtype=torch.int64, device="cuda")
    norm, drop = ua.GroupNormAct(8, C, p=0.5, offset_dev=step).cuda(), ua.Dropout(C, 0.5, offset_dev=step)
    for layer in (norm, drop):
        x = rnd(1, 2, 4, 4, C).cuda().requires_grad_()
        first = layer(x)
        step.add_(1)
        second = layer(x)
        torch.autograd.grad(second.sum(), x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(first.sum(), x)


@pytest.mark.parametrize("frozen", [("weight",), ("bias",), ("weight", "bias")])
def test_frozen_parameters_cost_no_sums(ua, monkeypatch, frozen):
    """Gradients that nobody asked for are not worked out; the others are the same bits."""
    ops, made = ua.ops, []
    bwd = ops.group_norm_act_bwd
    monkeypatch.setattr(ops, "group_norm_act_bwd", lambda *a, **k: made.append(bwd(*a, **k)) or made[-1])
    norm = ua.GroupNormAct(8, 64, act="silu").cuda()
    x, dy = rnd(1, 40, 16, 16, 64).cuda().requires_grad_(), rnd(2, 40, 16, 16, 64).cuda()
    every = torch.autograd.grad(norm(x), (x, norm.weight, norm.bias), dy)
    for name in frozen:
        getattr(norm, name).requires_grad_(False)
    norm(x).backward(dy)
    assert torch.equal(x.grad, every[0])
    for name, got, want in zip(("weight", "bias"), made[-1][1:], every[1:]):
        assert got is None and getattr(norm, name).grad is None if name in frozen else torch.equal(got, want)


def test_millions_of_rows_in_one_group(ua):
    """4.3 million images of one pixel with groups of more than 64 vectors: joins with a wave each, as a launch holds no more.
    The last rows against the definition, the parameters' gradients against sums in 64 bits."""
    ops, rows, C, tail = ua.ops, (1 << 22) + 100_001, 528, 1000
    x = torch.empty((rows, 1, 1, C), device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator("cuda").manual_seed(1))
    y, mean, rstd = ops.group_norm_act_fwd(x, C, 1, act="silu")
    x6 = x[-tail:].double().cpu()
    one, zero = torch.ones(C).double(), torch.zeros(C).double()
    oy, om, orr, z = N.group_norm_act_fwd(x6, 1, one, zero, "silu", float(torch.tensor(1e-5)))
    within(y[-tail:], oy, fwd_bound(x6, oy, z, om, orr, one, zero, 1, torch.bfloat16), "tail")
    dx, dw, db = ops.group_norm_act_bwd(x, y, mean, rstd, C, 1, one.float().cuda(), zero.float().cuda(), act="none")
    m, r = mean[-tail:].double().cpu(), rstd[-tail:].double().cpu()
    bwd_check((dx[-tail:], None, None), x6, y[-tail:].double().cpu(), m, r, 1, one, zero, "none", None, torch.bfloat16, "tail")
    want_w, want_b, size_w, size_b = (torch.zeros(C, device="cuda", dtype=torch.float64) for _ in range(4))
    for k in range(0, rows, 1 << 18):
        d = y[k:k + (1 << 18), 0, 0].double()
        h = (x[k:k + (1 << 18), 0, 0].double() - mean[k:k + (1 << 18)].double()) * rstd[k:k + (1 << 18)].double()
        want_w += (d * h).sum(0)
        want_b += d.sum(0)
        size_w += (d * h).abs().sum(0)
        size_b += d.abs().sum(0)
    within(dw, want_w.cpu(), ((K + 8) * U * size_w).cpu(), "dweight")
    within(db, want_b.cpu(), (K * U * size_b).cpu(), "dbias")
    del x, y, dx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape, bias", [((1, 512, 512, 96, 1), 0.0), ((2, 1024, 1024, 64, 1), 3.0), ((1, 1024, 1024, 33, 3), 1.0),
                                         ((1 << 21, 1, 1, 32, 8), 0.0), ((300, 96, 96, 32, 4), 2.0)])
def test_gradients_of_one_sign(ua, dtype, shape, bias):
    """A constant dy, as the gradient of a sum is: thousands of tiles, rows or parts add to sums without any cancellation.  The
    bounds are those of bwd_check with its K additions of 32 bits between an element and a sum; joins add in 64."""
    B, H, W, C, G = shape
    ops, gen = ua.ops, torch.Generator("cuda").manual_seed(1)
    cg = C // G
    x = torch.zeros((B, H, W, N.pad_ch(C)), device="cuda", dtype=dtype)
    x[..., :C] = torch.randn(B, H, W, C, device="cuda", generator=gen)
    dy = torch.full_like(x, 0.3)
    gamma, beta = rnd(3, C, scale=0.3, shift=1.0).cuda(), (rnd(4, C, scale=0.3) + bias).cuda()
    y, mean, rstd = ops.group_norm_act_fwd(x, C, G, gamma, beta, act="silu")
    del y
    dx, dw, db = ops.group_norm_act_bwd(x, dy, mean, rstd, C, G, gamma, beta, act="silu")
    sums = [torch.zeros(C, device="cuda", dtype=torch.float64) for _ in range(4)]       # dweight, dbias and their bounds
    step = max(1, (1 << 25) // (H * W * C))
    for k in range(0, B, step):
        b = slice(k, k + step)
        x6, dy6 = x[b, ..., :C].double(), dy[b, ..., :C].double()
        want, gw, gb, p = N.group_norm_act_bwd(x6, dy6, mean[b].double(), rstd[b].double(), G, gamma.double(), beta.double(), "silu")
        ddz, dt = bwd_bounds(p, gamma.double(), beta.double(), dtype)
        gm = lambda t: N._per_channel(N._group_mean(t, G), cg)
        bound = p["r"] * (dt + gm(dt) + p["h"].abs() * gm(dt * p["h"].abs()) + K * U * (p["a1"] + p["h"].abs() * p["a2"])
                          + 8 * U * (p["t"].abs() + p["m1"].abs() + (p["h"] * p["m2"]).abs())) + half_step(dtype) * want.abs() + 1e-37
        assert ((dx[b, ..., :C].double() - want).abs() <= bound).all()
        hb = p["h"].abs()
        for s, t in zip(sums, (gw, gb, (ddz * hb + (K + 8) * U * (p["dz"] * p["h"]).abs()).sum((0, 1, 2)),
                               (ddz + K * U * p["dz"].abs()).sum((0, 1, 2)))):
            s += t
    within(dw, sums[0].cpu(), sums[2].cpu() + 1e-37, "dweight")
    within(db, sums[1].cpu(), sums[3].cpu() + 1e-37, "dbias")
    del x, dy, dx
    ones = torch.zeros((B, H, W, N.pad_ch(C)), device="cuda", dtype=dtype)
    dy = torch.full_like(ones, 0.3)
    _, _, db = ops.group_norm_act_bwd(ones, dy, mean, rstd, C, G, gamma, beta)
    want = dy[0, 0, 0, 0].double().cpu() * (B * H * W)
    within(db, want.expand(C), K * U * want.expand(C), "dbias of a constant")
    del ones, dy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("C, G", [(512, 8), (1040, 1)])          # one workgroup; the general kernels
def test_gelu_in_fp32(ua, C, G):
    """The function and its slope by themselves: gamma = 0 makes z = beta, one image of one pixel makes dbias the slope.
    1 - Phi is fitted to 1.1e-8 or, below 1e-3, to 1.1e-5 of itself; t, the polynomial, their product and 2^x round 3 + 4 + 2 + 2
    times, 2^x's argument (z^2 / 2 log2 e, twice rounded) z^2 u; then 1 - (1 - Phi), the Gaussian's factors and one rounding each."""
    z = torch.linspace(-13, 8, C)
    zero, one = torch.zeros(C).cuda(), torch.ones(1, 1, 1, C).cuda()
    x = place(rnd(1, 1, 1, 1, C), torch.float32)
    y, m, r = ua.ops.group_norm_act_fwd(x, C, G, zero, z.cuda(), act="gelu")
    _, _, db = ua.ops.group_norm_act_bwd(x, place(one.cpu(), torch.float32), m, r, C, G, zero, z.cuda(), act="gelu")
    z = z.double()
    tail, phi, gauss = 0.5 * torch.erfc(z.abs() * 0.5 ** 0.5), 0.5 * torch.erfc(-z * 0.5 ** 0.5), torch.exp(-0.5 * z * z) / (2 * np.pi) ** 0.5
    dphi = torch.minimum(torch.tensor(1.1e-8, dtype=torch.float64), 1.1e-5 * tail) + (11 + z * z) * U * tail + U * phi
    within(y[0, 0, 0, :C], z * phi, z.abs() * dphi + U * (z * phi).abs() + 1e-37, "value")
    slope = phi + z * gauss
    within(db, slope, dphi + (z * gauss).abs() * (5 + z * z) * U + U * slope.abs() + 1e-37, "slope")


@pytest.mark.parametrize("shape", [(2, 33, 31, 32, 8), (3, 1, 2, 64, 8), (9, 100, 96, 40, 8), (1, 256, 255, 66, 3)])
def test_norm_far_from_zero_forward_and_backward(ua, shape):
    """A mean 10^4 standard deviations from zero: y is off by the mean's one rounding, U |mean| rstd, besides what it is anywhere
    (with deviations of size 1 in place of |x| in the additions: those are sums of deviations); dx, from the statistics handed on,
    by nothing else."""
    B, H, W, C, G = shape
    ops = ua.ops
    x, dy = rnd(1, B, H, W, C) + 1e4, rnd(5, B, H, W, C, scale=0.1)
    gamma, beta = rnd(3, C, scale=0.3, shift=1.0), rnd(4, C, scale=0.3)
    y, mean, rstd = ops.group_norm_act_fwd(place(x, torch.float32), C, G, gamma.cuda(), beta.cuda())
    x6, g6, b6 = x.double(), gamma.double(), beta.double()
    oy, om, orr, z = N.group_norm_act_fwd(x6, G, g6, b6, "none", float(torch.tensor(1e-5)))
    cg = C // G
    deviations = x6 - N._per_channel(om, cg)
    bound = fwd_bound(deviations, oy, z, torch.zeros_like(om), orr, g6, b6, G, torch.float32)
    within(y[..., :C], oy, bound + N._per_channel(U * om.abs() * orr, cg) * g6.abs(), "y")
    out = ops.group_norm_act_bwd(place(x, torch.float32), place(dy, torch.float32), mean, rstd, C, G, gamma.cuda(), beta.cuda(), act="silu")
    bwd_check(out, x6, dy.double(), mean.double().cpu(), rstd.double().cpu(), G, g6, b6, "silu", None, torch.float32, "backward")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("polls", [-1, 0])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_where_workgroups_share(ua, monkeypatch, dtype, polls, bad):
    """A value that is no number, in x or in dy, stays in its group and image: images of several parts, the general kernels."""
    ops = ua.ops
    monkeypatch.setattr(ops, "_POLLS", polls)
    for B, H, W, C, G in ((9, 100, 96, 40, 5), (12, 90, 80, 64, 4), (1, 256, 255, 72, 3)):
        x, dy = rnd(1, B, H, W, C).to(dtype), rnd(2, B, H, W, C).to(dtype)
        w, b = rnd(3, C, scale=0.3, shift=1.0).cuda(), rnd(4, C).cuda()
        cg, c = C // G, C // G + 1                                # group 1
        hit = torch.zeros(B, H, W, N.pad_ch(C), dtype=torch.bool)
        hit[-1, ..., cg:2 * cg] = True
        for act in ("relu", "silu"):
            def run(x, dy):
                y, m, r = ops.group_norm_act_fwd(place(x, dtype), C, G, w, b, act=act)
                return (y, m, r) + ops.group_norm_act_bwd(place(x, dtype), place(dy, dtype), m, r, C, G, w, b, act=act)
            clean = run(x, dy)
            bad_x, bad_dy = x.clone(), dy.clone()
            bad_x[-1, H - 1, W - 2, c] = bad
            bad_dy[-1, H // 2, 3, c] = bad
            y, m, r, dx, dw, db = run(bad_x, dy)
            assert torch.equal(y.cpu()[~hit], clean[0].cpu()[~hit]) and torch.isnan(y.cpu()[hit]).all()
            assert torch.equal(dx.cpu()[~hit], clean[3].cpu()[~hit])
            assert not torch.isfinite(m[-1, 1]) and not torch.isfinite(r[-1, 1]) and int(torch.isfinite(r).sum()) == B * G - 1
            dx, dw, db = run(x, bad_dy)[3:]
            assert torch.equal(dx.cpu()[~hit], clean[3].cpu()[~hit])
            for got, want in ((dw, clean[4]), (db, clean[5])):
                others = torch.arange(C) != c
                assert torch.equal(got.cpu()[others], want.cpu()[others])


def test_dropout_goes_backward_twice(ua):
    """Its node keeps no tensor unless it has a counter, so it needs no retain_graph."""
    x, drop = rnd(1, 2, 4, 4, 64).cuda().requires_grad_(), ua.ops.Drop(0.5, 1)
    y = ua.dropout(x, 64, drop)
    dy = rnd(2, 2, 4, 4, 64).cuda()
    first, = torch.autograd.grad(y, x, dy)
    again, = torch.autograd.grad(y, x, dy)
    assert torch.equal(first, again) and torch.equal(first, ua.ops.dropout_bwd(dy, 64, drop))
