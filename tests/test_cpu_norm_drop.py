"""Group norm and dropout, what needs no GPU: the generator's known answers, the oracle against torch's autograd, and
every call the library and the wrappers refuse (each is refused before anything is launched)."""
import ctypes as C

import pytest
import torch
import torch.nn.functional as F

from oracle import norm_oracle as N


@pytest.fixture(scope="module")
def ua():
    import unet_amd
    return unet_amd


def test_generator_known_answers():
    """Three vectors published with the generator."""
    kat = [((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
           ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
           ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
            (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]
    for ctr, key, want in kat:
        assert tuple(int(v) for v in N.philox4x32(ctr, key)) == want


def test_mask_statistics():
    """Rate within five standard deviations, neighbours and layers (offsets) independent to the same measure."""
    shape, p = (4, 64, 64, 64), 0.3
    n = 4 * 64 * 64 * 64
    keep = N.drop_factor(shape, p, seed=(7 << 40) + 3).flatten() > 0
    other = N.drop_factor(shape, p, seed=(7 << 40) + 3, offset=1).flatten() > 0
    sd = (n * p * (1 - p)) ** 0.5
    assert abs(int(keep.sum()) - 0.7 * n) < 5 * sd
    for a, b in ((keep[1:], keep[:-1]), (keep, other)):
        m = len(a)
        assert abs(int((a & b).sum()) - 0.49 * m) < 5 * (m * 0.49 * 0.51) ** 0.5
    maps = N.drop_factor((3, 5, 4, 40), p, seed=5, per_channel=True)
    assert torch.equal(maps, maps[:, :1, :1].expand_as(maps)) and 0 < (maps[:, 0, 0] > 0).sum() < 120


@pytest.mark.parametrize("kind", ["none", "relu", "silu", "gelu"])
def test_oracle_against_torch(kind):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 5, 3, 12, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
    b = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(2, 5, 3, 12, generator=g, dtype=torch.float64)
    factor = N.drop_factor((2, 5, 3, 12), 0.25, 11)
    f = {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[kind]
    y = f(F.group_norm(x.permute(0, 3, 1, 2), 3, w, b, 1e-5)).permute(0, 2, 3, 1) * factor
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x0, w0, b0 = x.detach(), w.detach(), b.detach()
    oy, mean, rstd, _ = N.group_norm_act_fwd(x0, 3, w0, b0, kind, 1e-5, factor)
    odx, odw, odb, _ = N.group_norm_act_bwd(x0, dy, mean, rstd, 3, w0, b0, kind, factor)
    for got, want in ((oy, y.detach()), (odx, dx), (odw, dw), (odb, db)):
        assert torch.allclose(got, want, rtol=1e-10, atol=1e-12)


# ---------------------------------------------------------------- refusals of the C entry points
A = 1 << 20          # an aligned address that nothing may touch


def _norm_fwd(L, x=A, xcs=64, xco=0, gamma=None, y=A << 4, ycs=64, yco=0, mean=A, rstd=A, B=2, H=4, W=4, Cc=40, G=5, act=1,
              eps=1e-5, drop=None, ws=A, ws_bytes=1 << 20, dt=0):
    return L.mi_group_norm_act_fwd(x, xcs, xco, gamma, None, y, ycs, yco, mean, rstd, B, H, W, Cc, G, act, eps,
                                   C.byref(drop) if drop else None, -1, ws, ws_bytes, dt, None)


def _norm_bwd(L, x=A, dy=A << 1, dx=A << 4, xcs=64, dcs=64, dco=0, mean=A, B=2, H=4, W=4, Cc=40, G=5, act=1, ws=A,
              ws_bytes=1 << 20, dt=1):
    return L.mi_group_norm_act_bwd(x, xcs, 0, dy, 64, 0, None, None, mean, A, dx, dcs, dco, None, None, 1.0, 0.0, B, H, W, Cc, G,
                                   act, None, -1, ws, ws_bytes, dt, None)


def _drop(L, x=A, xcs=64, xco=0, r=None, rcs=64, y=A << 4, ycs=64, yco=0, B=2, H=4, W=4, Cc=40, drop=None, dt=0):
    return L.mi_dropout_fwd(x, xcs, xco, r, rcs, 0, y, ycs, yco, B, H, W, Cc, C.byref(drop) if drop else None, dt, None)


def test_c_refusals(ua):
    from unet_amd._lib import Dropout
    L = ua.lib()
    nan = float("nan")
    bad_p = [Dropout(p, 1, 0, None, 0) for p in (-0.1, 1.1, nan)]
    calls = [lambda kw=kw: _norm_fwd(L, **kw) for kw in (
        dict(x=None), dict(x=A + 8), dict(y=None), dict(y=A + 4), dict(xcs=40), dict(xco=32), dict(xco=8), dict(xco=-16),
        dict(ycs=32), dict(yco=24), dict(mean=None), dict(rstd=None), dict(ws=None), dict(ws=A + 4), dict(B=-1), dict(H=0),
        dict(W=-3), dict(Cc=0), dict(G=0), dict(G=3), dict(G=-5), dict(G=80), dict(act=4), dict(act=-1), dict(eps=-1.0),
        dict(eps=nan), dict(dt=2), dict(dt=-1), dict(H=1 << 16, W=1 << 16), dict(B=1 << 20, H=1 << 10, W=1 << 10),
        dict(y=A), dict(y=A + 2 * 64 * 4), dict(y=A, yco=16, ycs=128, xcs=128), dict(y=A, ycs=128),
        dict(drop=bad_p[0]), dict(drop=bad_p[1]), dict(drop=bad_p[2]))]
    calls += [lambda kw=kw: _norm_bwd(L, **kw) for kw in (
        dict(x=None), dict(dy=None), dict(dx=None), dict(dx=A), dict(dx=A << 1), dict(mean=None), dict(ws=None), dict(xcs=32),
        dict(dco=32), dict(G=7), dict(act=9), dict(dt=3), dict(B=-2), dict(Cc=1 << 30, G=1))]
    calls += [lambda kw=kw: _drop(L, **kw) for kw in (
        dict(x=None), dict(x=A + 2), dict(y=None), dict(xcs=32), dict(xco=32), dict(ycs=56), dict(r=A + 8), dict(r=A << 6, rcs=32),
        dict(B=-1), dict(H=0), dict(Cc=-4), dict(dt=2), dict(y=A + 64 * 4), dict(y=A, ycs=80), dict(r=(A << 4) + 256),
        dict(B=1 << 20, H=1 << 10, W=1 << 10), dict(drop=bad_p[0]), dict(drop=bad_p[1]), dict(drop=bad_p[2]))]
    for i, call in enumerate(calls):
        assert call() == -1, i                                    # MI_EINVAL
        assert L.mi_last_error().decode()
    assert _norm_fwd(L, y=A << 10, B=2, H=400, W=400, ws_bytes=8) == -2 and b"workspace" in L.mi_last_error()       # MI_ESIZE
    assert _norm_bwd(L, dy=A << 9, dx=A << 10, B=300, H=40, W=40, ws_bytes=8) == -2 and b"workspace" in L.mi_last_error()


def test_more_threads_than_a_launch_holds_are_refused(ua):
    L = ua.lib()
    far = 1 << 45                                                 # behind a tensor of 2^30 pixels
    for call in (lambda: _norm_fwd(L, B=1 << 30, H=1, W=1, Cc=64, G=8, y=far, dt=1),
                 lambda: _norm_bwd(L, B=1 << 30, H=1, W=1, Cc=64, G=8, dy=far, dx=far << 1, ws_bytes=1 << 60),
                 lambda: _norm_fwd(L, B=1 << 26, H=1, W=1, Cc=640, G=1, xcs=640, ycs=640, y=far, ws_bytes=1 << 60),
                 lambda: _drop(L, B=1 << 30, H=1, W=1, Cc=256, xcs=256, ycs=256, y=far)):
        assert call() == -1 and b"too large" in L.mi_last_error()


def test_empty_batches_need_nothing(ua):
    L = ua.lib()
    assert _norm_fwd(L, B=0, x=None, y=None, mean=None, rstd=None, ws=None) == 0
    assert _drop(L, B=0, x=None, y=None) == 0
    assert L.mi_group_norm_ws_bytes(0, 4, 4, 40, 5, 0, 0) >= 0
    for bad in ((-1, 4, 4, 40, 5), (2, 0, 4, 40, 5), (2, 4, 4, 40, 3), (2, 4, 4, 0, 1), (2, 4, 4, 40, 0), (1, 1 << 16, 1 << 16, 32, 1)):
        assert L.mi_group_norm_ws_bytes(*bad, 0, 0) == 0


def test_wrapper_refusals(ua):
    ops = ua.ops
    x = torch.zeros(2, 4, 4, 48)
    for p in (-0.01, 1.01, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            ops.Drop(p, 1)
        with pytest.raises(ValueError, match="between 0 and 1"):
            ua.Dropout(40, p)
        with pytest.raises(ValueError, match="between 0 and 1"):
            ua.GroupNormAct(5, 40, p=p)
    for seed, offset in ((-1, 0), (1 << 64, 0), (0, -1), (0, 1 << 64)):
        with pytest.raises(ValueError, match="2\\^64"):
            ops.Drop(0.5, seed, offset)
    with pytest.raises(ValueError, match="offset_dev"):
        ops.Drop(0.5, 1, offset_dev=torch.zeros(1, dtype=torch.int64))          # not on the GPU
    drop = ops.Drop(0.5, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.dropout_fwd(x, 40, drop)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.group_norm_act_fwd(x, 40, 5)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.group_norm_act_bwd(x, x, torch.zeros(2, 5), torch.zeros(2, 5), 40, 5)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ua.GroupNormAct(5, 40)(x)
    for bad in ((3, 40), (0, 40), (5, 0)):
        with pytest.raises(ValueError, match="do not split"):
            ua.GroupNormAct(*bad)
    with pytest.raises(ValueError, match="unknown activation"):
        ua.GroupNormAct(5, 40, act="tanh")


def test_modules_carry_group_norms_parameters(ua):
    m, ref = ua.GroupNormAct(5, 40, act="silu", p=0.1), torch.nn.GroupNorm(5, 40)
    assert {k: v.shape for k, v in m.state_dict().items()} == {k: v.shape for k, v in ref.state_dict().items()}
    m.load_state_dict(ref.state_dict())
    assert ua.GroupNormAct(5, 40, affine=False).state_dict() == {}
    x = torch.randn(2, 4, 4, 48)
    d = ua.Dropout(40, 0.5).eval()
    assert d(x) is x and torch.equal(d(x, x), 2 * x)
    torch.manual_seed(5)
    a = [ua.layers.fresh_drop(0.5).seed for _ in range(3)]
    torch.manual_seed(5)
    assert a == [ua.layers.fresh_drop(0.5).seed for _ in range(3)] and len(set(a)) == 3


def test_dropout_module_without_drops_needs_the_kernels_for_other_widths(ua):
    d = ua.Dropout(40, 0.5).eval()
    for args in ((torch.zeros(2, 4, 4, 48), torch.zeros(2, 4, 4, 64)), (torch.zeros(2, 4, 4, 64),)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            d(*args)


def test_a_drop_is_fixed(ua):
    """Setting an attribute had no effect on what the kernels were given."""
    drop = ua.ops.Drop(0.5, 1, 2, per_channel=True)
    for name, value in (("p", 0.1), ("seed", 3), ("offset", 4), ("offset_dev", None), ("per_channel", False)):
        with pytest.raises(AttributeError):
            setattr(drop, name, value)
    assert (drop.p, drop.seed, drop.offset, drop.offset_dev, drop.per_channel) == (0.5, 1, 2, None, True)
    assert (drop._desc.p, drop._desc.seed, drop._desc.offset, drop._desc.per_channel) == (0.5, 1, 2, 1)


def test_many_rows_in_one_group_are_taken(ua):
    """5 million rows of 528 channels: refused for the workspace alone, not for joins with more threads than they run with."""
    L, far = ua.lib(), 1 << 45
    assert _norm_fwd(L, B=5_000_000, H=1, W=1, Cc=528, G=1, xcs=528, ycs=528, y=far, dt=1, ws_bytes=8) == -2
    assert L.mi_group_norm_act_bwd(A, 528, 0, far, 528, 0, None, None, A, A, far << 1, 528, 0, None, None, 1.0, 0.0, 5_000_000, 1, 1, 528, 1,
                                   1, None, -1, A, 8, 1, None) == -2


def test_refused_shapes_need_no_workspace(ua):
    """The size of a workspace is asked for before the call that would refuse the shape."""
    L, big = ua.lib(), (1 << 31) - 1
    for backward in (0, 1):
        for dt in (0, 1):
            for shape in ((1, 1, 1, big, 1), (1, 1, 1, (1 << 24) + 16, 1), (1 << 20, 1 << 10, 1 << 10, 64, 8), (big, 2, 1, 32, 4)):
                assert L.mi_group_norm_ws_bytes(*shape, backward, dt) == 0
        assert L.mi_group_norm_ws_bytes(2, 256, 255, 66, 3, backward, 2) == 0 and L.mi_group_norm_ws_bytes(2, 256, 255, 66, 3, backward, 1) > 0
