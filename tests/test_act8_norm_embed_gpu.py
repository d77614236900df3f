"""The 8-bit activation checkpoints, the RMS norm and the scaled embedding on the MI355X against their definitions in 64 bits.

Tolerances are sums of rounding errors, written at each check: a rounding to a type is off by at most half a step of it
(finfo.eps / 2 of the value), an fp32 operation by U = 2^-24, a sum of k fp32 terms by at most k U times the sum of their
magnitudes.  The checkpoint itself is exact arithmetic apart from its one rounding and is compared for equality."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops(gpu):
    from bifold_amd.hip import ops as _ops
    return _ops


@pytest.fixture(scope="module")
def L(gpu):
    from bifold_amd.hip import lib as _lib
    return _lib


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny_step(dtype):
    """Half the distance between the smallest numbers of a type."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150


def close(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), ((got - want).abs() / (bound + 1e-300)).max().item())


def make(rows, cols, dtype, seed, spread=1.0, layout="plain"):
    """(tensor on the GPU, its values in 64 bits).  layout: plain; wide = columns of a wider buffer, 16-byte aligned rows;
    off = a view whose rows start at odd addresses."""
    g = torch.Generator().manual_seed(seed)
    extra = {"plain": 0, "wide": 24, "off": 3}[layout]
    x = torch.randn(rows, cols + extra, generator=g) * spread * (1 + 6 * torch.rand(cols + extra, generator=g) ** 6)
    x = x.to(dtype)
    first = {"plain": 0, "wide": 8, "off": 1}[layout]
    return x.cuda()[:, first:first + cols] if extra else x.cuda(), x[:, first:first + cols].double()


# ------------------------------------------------------------------ the checkpoint
def kept_ref(x):
    """(q, code, values) of x [rows, cols] float64 (holding fp32 values): the definition, group by group in 64 bits."""
    rows, cols = x.shape
    groups = (cols + 31) // 32
    full = torch.zeros(rows, groups * 32, dtype=torch.float64)
    full[:, :cols] = x
    full = full.view(rows, groups, 32)
    top = full.abs().amax(2)
    fine = torch.isfinite(top) & (top < 255 * 2.0 ** 119)
    e = torch.full(top.shape, -126, dtype=torch.int64)
    safe = torch.where(fine & (top > 0), top, torch.ones_like(top))
    k = torch.frexp(safe)[1].long() - 7                         # 2^(k + 6) <= top < 2^(k + 7)
    k = torch.where(torch.round(safe / torch.exp2(k.double())) > 127, k + 1, k).clamp(min=-126)
    e = torch.where(top > 0, k, e)
    step = torch.exp2(e.double())                               # CPU: exact for whole exponents
    q = torch.where(fine[..., None], torch.round(full / step[..., None]), torch.zeros_like(full))
    val = torch.where(fine[..., None], q * step[..., None], torch.full_like(full, math.nan))
    code = torch.where(fine, e + 127, torch.full_like(e, 255))
    cut = lambda t: t.reshape(rows, -1)[:, :cols]               # noqa: E731
    return cut(q).to(torch.int8), code.to(torch.uint8), cut(val)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0)) and torch.equal(a.isnan(), b.isnan())


SHAPES = [(1, 1), (1, 32), (3, 7), (5, 33), (2, 520), (77, 768), (130, 1024), (64, 1021), (1000, 96), (3, 9000), (1, 100000)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["plain", "wide", "off"])
def test_act8_pack_and_unpack(ops, rows, cols, dtype, layout):
    x, ref = make(rows, cols, dtype, rows * 31 + cols, spread=0.7, layout=layout)
    q, code, val = kept_ref(ref)
    kept = ops.act8_pack(x)
    assert kept[0].shape == x.shape and torch.equal(kept[0].cpu(), q) and torch.equal(kept[1].cpu(), code)
    for out in TYPES:                                           # |values| < 65504: exact in every type
        assert torch.equal(ops.act8_unpack(kept, out).cpu().double(), val)
    assert ((val - ref).abs() <= ref.abs().amax() / 127).all()


def test_act8_special_groups(ops):
    x = torch.zeros(12, 40)
    x[1, 3] = math.nan
    x[2, 35] = math.inf                                         # the short last group of the row
    x[3, 5] = -math.inf
    x[4, 0], x[4, 1] = 255 * 2.0 ** 119, 1.0
    x[5, 0], x[5, 1] = 254.9 * 2.0 ** 119, 2.0 ** 120
    x[6, :32] = torch.arange(32) * 2.0 ** -149                  # subnormal numbers
    x[7, 0], x[7, 1] = 127.5, 1.0                               # rounds to 128: the next exponent
    x[8, 0], x[8, 1], x[8, 2], x[8, 3] = 127.25, 0.5, 1.5, -2.5   # ties to even
    x[9, 0] = 2.0 ** -126 * 64
    x[10, 39] = -1e-30
    x[11, 0], x[11, 1] = 1e38, 1e-38
    q, code, val = kept_ref(x.double())
    kept = ops.act8_pack(x.cuda())
    assert torch.equal(kept[1].cpu(), code)
    assert torch.equal(kept[0].cpu(), q)
    assert same(ops.act8_unpack(kept, torch.float32).cpu().double(), val)
    assert val[1].isnan()[:32].all() and not val[1].isnan()[32:].any() and val[2].isnan()[32:].all() and val[4].isnan()[:32].all()
    assert torch.isfinite(val[5]).all() and val[7, 0] == 128 and val[8, :4].tolist() == [127.0, 0.0, 2.0, -2.0]


def test_act8_empty_out_and_shape(ops, gpu):
    q, code = ops.act8_pack(torch.zeros(0, 64, device=gpu))
    assert q.shape == (0, 64) and code.shape == (0, 2) and ops.act8_unpack((q, code), torch.bfloat16).shape == (0, 64)
    x = torch.randn(2, 5, 3, 70, device=gpu)
    q, code = ops.act8_pack(x)
    assert q.shape == x.shape and code.shape == (2, 5, 3, 3)
    flat = ops.act8_pack(x.view(30, 70))
    assert torch.equal(flat[0].view_as(q), q) and torch.equal(flat[1].view_as(code), code)
    wide = torch.full((4, 100), 7.0, device=gpu)
    kept = ops.act8_pack(x.view(30, 70)[:4])
    ops.act8_unpack(kept, torch.float32, out=wide[:, 10:80])
    assert torch.equal(wide[:, 10:80], ops.act8_unpack(kept, torch.float32))
    assert (wide[:, :10] == 7).all() and (wide[:, 80:] == 7).all()
    assert (ops.act8_pack(torch.zeros(3, 64, device=gpu))[1] == 1).all()


GELUS = ["quick", "erf", "tanh"]


def act_ref(x, act):
    """(value, slope, exponent's argument, |x u'|) in 64 bits."""
    if act == "erf":
        cdf = 0.5 * torch.erfc(-x / math.sqrt(2))
        pdf = torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
        return x * cdf, cdf + x * pdf, x * x, x.abs()
    c = math.sqrt(2 / math.pi)
    u, du = (1.702 * x, torch.full_like(x, 1.702)) if act == "quick" else (2 * c * (x + 0.044715 * x ** 3),
                                                                           2 * c * (1 + 0.134145 * x * x))
    s = torch.sigmoid(u)
    return x * s, s + x * du * s * torch.sigmoid(-u), u.abs(), (x * du).abs()


def act_code(L, act):
    return {"quick": L.ACT_QUICK_GELU, "erf": L.ACT_ERF_GELU, "tanh": L.ACT_TANH_GELU}[act]


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (77, 512), (64, 1021), (33, 2048), (5, 520)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", GELUS)
@pytest.mark.parametrize("layout", ["plain", "wide"])
def test_act8_gelu(ops, L, rows, cols, dtype, act, layout):
    pre, ref = make(rows, cols, dtype, rows + cols, spread=0.8, layout=layout)
    dy, dyr = make(rows, cols, dtype, rows + cols + 1, spread=0.3, layout=layout)
    code = act_code(L, act)
    y, kept = ops.act8_gelu_fwd(pre, code)
    want, _, u, _ = act_ref(ref, act)
    # an argument of the exponential off by a few U of itself moves it by as many U times u; erfc and the products add 32 U
    # the factor of x: 1 / (1 + e) is lost where e overflows, at 2^128; erfc under 2^-126 is off by a place of 2^-149
    bound = want.abs() * (half_step(dtype) + (32 + 4 * u) * U) + tiny_step(dtype) + ref.abs() * 2.0 ** -127
    if dtype != torch.float32:
        bound = bound + ref.abs() * 2.0 ** -22                  # the 16-bit forms: erf to 1.5e-7, 1 - s in fp32
    close(y, want, bound, "y")
    q, c, val = kept_ref(ref)
    assert torch.equal(kept[0].cpu(), q) and torch.equal(kept[1].cpu(), c)
    dx = ops.act8_gelu_bwd(dy, kept, code)
    _, slope, u, xdu = act_ref(val, act)
    s_part = slope.abs() + xdu * torch.exp(-u.clamp(max=700)).clamp(max=1) if act != "erf" else slope.abs() + val.abs() * 0.4
    bound = (dyr * slope).abs() * half_step(dtype) + tiny_step(dtype)
    if dtype == torch.float32:
        bound = bound + dyr.abs() * ((64 + 8 * u) * U * s_part + 2.0 ** -60)
    else:
        bound = bound + dyr.abs() * (1 + xdu) * 2.0 ** -20      # s to 2^-21, 1 - s by subtraction, erf to 1.5e-7
    close(dx, dyr * slope, bound, "dx")
    same_place = dy.clone() if layout == "plain" else dy
    out = ops.act8_gelu_bwd(same_place, kept, code, out=same_place)
    assert out is same_place and torch.equal(out, dx)


@pytest.mark.parametrize("act", GELUS)
def test_act8_gelu_slope_against_differences(ops, L, gpu, act):
    """dpre of ones is the derivative of y: central differences of the fp32 forward at the checkpoint's own values."""
    x = torch.linspace(-6, 6, 32 * 40).view(40, 32).to(gpu)
    kept = ops.act8_pack(x)
    at = ops.act8_unpack(kept, torch.float32)
    h = 2.0 ** -6
    code = act_code(L, act)
    up, down = ops.act8_gelu_fwd(at + h, code)[0], ops.act8_gelu_fwd(at - h, code)[0]
    slope = ops.act8_gelu_bwd(torch.ones_like(at), kept, code)
    # third derivatives of the three GELUs stay under 3: h^2 / 6 * 3; the values are off by some 64 U |y|, |y| <= 6
    assert ((up - down) / (2 * h) - slope).abs().max().item() <= h * h / 2 + 2 * 6 * 64 * U / (2 * h)


def test_act8_gelu_non_finite_and_far(ops, L, gpu):
    for dtype in TYPES:
        pre = torch.zeros(2, 64, dtype=dtype, device=gpu)
        pre[0, 3] = math.inf
        pre[1, 0], pre[1, 1], pre[1, 2] = 5000.0, -5000.0, 60.0
        dy = torch.ones(2, 64, dtype=dtype, device=gpu)
        for act in GELUS:
            y, kept = ops.act8_gelu_fwd(pre, act_code(L, act))
            assert y[1, :3].tolist() == [5000.0 if dtype != torch.bfloat16 else 4992.0, 0.0, 60.0], (act, y[1, :3])
            dx = ops.act8_gelu_bwd(dy, kept, act_code(L, act))
            assert dx[0, :32].isnan().all() and not dx[0, 32:].isnan().any()      # the overflow reaches the gradient
            assert dx[1, :3].tolist() == [1.0, 0.0, 1.0]        # at 4992, -4992 and 64: the group's step is 64


# ------------------------------------------------------------------ RMS norm
NORMS = [(1, 1), (1, 64), (3, 7), (7, 255), (130, 256), (9, 257), (70, 768), (33, 1000), (66, 1024), (5, 1025), (17, 1155), (6, 2048),
         (3, 4096), (2, 4100), (4, 8192), (3, 8200), (2, 12001), (3, 16384), (2, 20001)]
PAIRS = [(torch.float32, None), (torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16),
         (torch.bfloat16, None), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float32)]


def rms_ref(x, delta, gamma, eps):
    t = x if delta is None else x + delta
    r = 1 / torch.sqrt((t * t).mean(1) + eps)
    return t, r, t * r[:, None] * gamma


def sum_error(cols):
    """U times this bounds the relative error of 1 / rms: a lane adds at most cols / 64 terms, then trees; half of it is left
    after the root."""
    return cols / 64 / 2 + 24


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("xd,dd", PAIRS)
@pytest.mark.parametrize("layout", ["plain", "wide", "off"])
def test_rmsnorm_fwd(ops, gpu, rows, cols, xd, dd, layout):
    eps = 1e-6
    x, xr = make(rows, cols, xd, rows * 7 + cols, layout=layout)
    delta, dr = make(rows, cols, dd, rows * 7 + cols + 1, spread=0.5, layout=layout) if dd else (None, None)
    gamma = 1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))
    t, r, y = rms_ref(xr, dr, gamma.double(), eps)
    size = xr.abs() + (dr.abs() if dd else 0)                   # t's rounding is relative to its terms' size
    k = sum_error(cols)
    fp32 = U * (size * r[:, None] * gamma.double().abs() * 2 + y.abs() * (k + 4))
    for od in TYPES:
        xo = torch.empty_like(x) if dd else None
        got, rstd, kept = ops.rmsnorm_fwd(x, gamma.to(gpu), od, delta=delta, x_out=xo, save_stats=True, eps=eps, checkpoint=True)
        assert got.dtype == od and got.shape == x.shape
        close(got, y, y.abs() * half_step(od) + fp32 * (1 + half_step(od)) + tiny_step(od), f"y {od}")
        # rstd: the terms' roundings move the mean square by at most 2 U |t| size per term
        close(rstd, r, r * U * (k + 2) + 2 * U * r ** 3 * (t.abs() * size).mean(1), "rstd")
        t32 = (xr.float() + dr.float()) if dd else xr.float()
        if dd:
            assert torch.equal(xo.cpu(), t32.to(xd))            # one fp32 add, one rounding
        q, code, _ = kept_ref(t32.double())
        assert torch.equal(kept[0].cpu(), q) and torch.equal(kept[1].cpu(), code)
    if dd:                                                      # in place, and not written at all
        before = x.clone()
        got2, none, no_ck = ops.rmsnorm_fwd(x, gamma.to(gpu), od, delta=delta, eps=eps, write_x=False)
        assert torch.equal(x, before) and torch.equal(got2, got) and none is None and no_ck is None
        got2, _, _ = ops.rmsnorm_fwd(x, gamma.to(gpu), od, delta=delta, eps=eps)
        assert torch.equal(x, xo) and torch.equal(got2, got)


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("xd,dd", [(torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float16, None)])
@pytest.mark.parametrize("layout", ["plain", "off"])
def test_rmsnorm_fwd_fp8(ops, gpu, rows, cols, xd, dd, layout):
    eps = 1e-6
    x, xr = make(rows, cols, xd, rows * 5 + cols, layout=layout)
    delta, dr = make(rows, cols, dd, rows * 5 + cols + 1, spread=0.5, layout=layout) if dd else (None, None)
    gamma = 1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))
    t, r, y = rms_ref(xr, dr, gamma.double(), eps)
    size = xr.abs() + (dr.abs() if dd else 0)
    fp32 = U * (size * r[:, None] * gamma.double().abs() * 2 + y.abs() * (sum_error(cols) + 8))
    xo = torch.empty_like(x) if dd else None
    y8, scale, rstd, kept = ops.rmsnorm_fwd_fp8(x, gamma.to(gpu), delta=delta, x_out=xo, save_stats=True, eps=eps, checkpoint=True)
    top = y.abs().amax(1)
    close(scale, top / 448, top / 448 * 2 * U + fp32.amax(1) / 448, "scale")
    got = y8.view(torch.float8_e4m3fn).float().cpu().double() * scale.cpu().double()[:, None]
    # e4m3: half a step is 2^-4 of the value, 2^-10 of the scale below its smallest normal number
    close(got, y, y.abs() * 2.0 ** -4 + scale.cpu().double()[:, None] * 2.0 ** -10 + 1.1 * fp32, "y8")
    y16, rstd2, kept2 = ops.rmsnorm_fwd(x, gamma.to(gpu), torch.float32, delta=delta, write_x=False, save_stats=True, eps=eps,
                                        checkpoint=True)
    assert torch.equal(rstd, rstd2) and torch.equal(kept[0], kept2[0]) and torch.equal(kept[1], kept2[1])
    assert torch.equal(scale.cpu(), y16.abs().amax(1).cpu() / torch.tensor(448.0))       # one division (a GPU tensor / number multiplies)


def test_rmsnorm_special_rows(ops, gpu):
    for cols in (64, 1000, 4096, 9000):
        x = torch.randn(4, cols, device=gpu)
        x[1] = 0
        x[2, 5] = math.nan
        x[3, cols - 1] = math.inf
        gamma = torch.ones(cols, device=gpu)
        y8, scale, rstd, kept = ops.rmsnorm_fwd_fp8(x, gamma, save_stats=True, checkpoint=True)
        y = y8.view(torch.float8_e4m3fn).float() * scale[:, None]
        assert torch.isfinite(y[0]).all() and (y[1] == 0).all() and scale[1] == 1 and y[2].isnan().all() and y[3].isnan().all()
        assert rstd[2].isnan() and rstd[3] == 0 and abs(rstd[1].item() - 1000) < 0.1
        back = ops.act8_unpack(kept, torch.float32)
        assert back[2, :32].isnan().all() and back[3, (cols - 1) // 32 * 32:].isnan().all() and torch.isfinite(back[:2]).all()
        y16, _, _ = ops.rmsnorm_fwd(x, gamma, torch.bfloat16)
        assert (y16[1] == 0).all() and y16[2].isnan().all() and y16[3, cols - 1].isnan()
        # gradients of the finite rows stay finite; dgamma shows the others
        dg = torch.empty(cols, device=gpu)
        dx = ops.rmsnorm_bwd(torch.ones(4, cols, device=gpu), kept, gamma, rstd, dg)
        assert torch.isfinite(dx[:2]).all() and dx[2].isnan().all() and dg.isnan().any()
    y8, scale, _, _ = ops.rmsnorm_fwd_fp8(torch.ones(2, 64, device=gpu), torch.full((64,), 1e-38, device=gpu))
    assert torch.isfinite(scale).all() and torch.isfinite(y8.view(torch.float8_e4m3fn).float()).all()


def rms_bwd_ref(dy, t, r, gamma, dres):
    h, b = t * r[:, None], dy * gamma
    m = (b * h).mean(1, keepdim=True)
    dx = r[:, None] * (b - h * m) + (0 if dres is None else dres)
    return dx, (dy * h).sum(0), h, b, m


@pytest.mark.parametrize("rows,cols", NORMS + [(700, 96), (5000, 64), (2100, 1100)])
@pytest.mark.parametrize("dyd,xd,rd", [(torch.float32, torch.float32, torch.float32), (torch.float16, torch.float32, torch.float16),
                                       (torch.bfloat16, "kept", torch.bfloat16), (torch.float16, "kept", torch.float32),
                                       (torch.float32, "kept", None), (torch.bfloat16, torch.bfloat16, None),
                                       (torch.float16, torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16, torch.float32),
                                       (torch.float32, torch.bfloat16, torch.bfloat16), (torch.float16, torch.bfloat16, None)])
@pytest.mark.parametrize("layout", ["plain", "off"])
def test_rmsnorm_bwd(ops, gpu, rows, cols, dyd, xd, rd, layout):
    eps = 1e-6
    src, xr = make(rows, cols, torch.float32 if xd == "kept" else xd, rows * 3 + cols, layout=layout)
    dy, dyr = make(rows, cols, dyd, rows * 3 + cols + 1, spread=0.3, layout=layout)
    dres, dr = make(rows, cols, rd, rows * 3 + cols + 2, spread=0.3, layout=layout) if rd else (None, None)
    gamma = 1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))
    g64 = gamma.double()
    _, rstd, kept = ops.rmsnorm_fwd(src, gamma.to(gpu), torch.float32, save_stats=True, eps=eps, checkpoint=True)
    if xd == "kept":
        xr = kept_ref(xr)[2]
    r = rstd.cpu().double()
    want, wg, h, b, m = rms_bwd_ref(dyr, xr, r, g64, dr)
    dg = torch.empty(cols, device=gpu)
    dx = ops.rmsnorm_bwd(dy, kept if xd == "kept" else src, gamma.to(gpu), rstd, dg, dres=dres)
    od = rd or dyd
    assert dx.dtype == od and dx.is_contiguous()
    # b: one rounding, h: one, the mean: cols / 64 + 12 of its terms' size (each with two roundings), then three operations
    bh = (b * h).abs().mean(1, keepdim=True)
    fp32 = U * r[:, None] * (5 * b.abs() + h.abs() * ((cols / 64 + 16) * bh + 5 * m.abs())) + U * (0 if dr is None else dr.abs())
    close(dx, want, want.abs() * (half_step(od) + 2 * U) + 1.01 * fp32 + tiny_step(od), "dx")
    # dgamma: a column's rows are added lane by lane (at most rows / 64 + 64 terms one after the other in every layout)
    close(dg, wg, U * (rows / 16 + 72) * (dyr * h).abs().sum(0) + 1e-30, "dgamma")
    again_g = torch.empty_like(dg)
    again = ops.rmsnorm_bwd(dy, kept if xd == "kept" else src, gamma.to(gpu), rstd, again_g, dres=dres)
    assert torch.equal(again, dx) and torch.equal(again_g, dg)                  # the same bits every time
    if layout == "plain" and dres is not None:
        into = dres.clone()
        assert ops.rmsnorm_bwd(dy, kept if xd == "kept" else src, gamma.to(gpu), rstd, dg, dres=into, out=into) is into
        assert torch.equal(into, dx)
    if layout == "plain" and dyd == od:
        into = dy.clone()
        assert ops.rmsnorm_bwd(into, kept if xd == "kept" else src, gamma.to(gpu), rstd, dg, dres=dres, out=into) is into
        assert torch.equal(into, dx)


def test_rmsnorm_bwd_against_differences(ops, gpu):
    """sum(w . y) of the fp32 forward, moved by h along a direction: the change is <dx, direction>."""
    rows, cols, h = 8, 200, 2.0 ** -9
    g = torch.Generator().manual_seed(5)
    x, w, v = (torch.randn(rows, cols, generator=g).double() for _ in range(3))
    gamma = (1 + 0.2 * torch.randn(cols, generator=g)).to(gpu)
    x = x.float().to(gpu)
    dg = torch.empty(cols, device=gpu)
    _, rstd, _ = ops.rmsnorm_fwd(x, gamma, torch.float32, save_stats=True)
    dx = ops.rmsnorm_bwd(w.float().to(gpu), x, gamma, rstd, dg)

    def f(s):
        y, _, _ = ops.rmsnorm_fwd(x + s * v.float().to(gpu), gamma, torch.float32)
        return (y.cpu().double() * w.float().double()).sum(1)

    diff = (f(h) - f(-h)) / (2 * h)
    slope = (dx.cpu().double() * v.float().double()).sum(1)
    # |d3/ds3| of a row stays under 6 |v|^3 / rms^3-ish ~ 6 * cols: h^2 / 6 of it; fp32 values: cols * 8 U / h
    assert (diff - slope).abs().max().item() <= h * h * cols + cols * 16 * U / h


def test_rmsnorm_no_rows(ops, gpu):
    x, gamma, dg = torch.zeros(0, 64, device=gpu), torch.ones(64, device=gpu), torch.full((64,), 3.0, device=gpu)
    y, rstd, kept = ops.rmsnorm_fwd(x, gamma, torch.float16, save_stats=True, checkpoint=True)
    assert y.shape == (0, 64) and rstd.shape == (0,) and kept[1].shape == (0, 2)
    assert ops.rmsnorm_bwd(x, x, gamma, rstd, dg).shape == (0, 64) and (dg == 0).all()


# ------------------------------------------------------------------ embedding
def tokens_of(kind, n, vocab, g):
    if kind == "one":
        return torch.full((n,), vocab // 2, dtype=torch.int64)
    if kind == "spread":
        return torch.randint(0, vocab, (n,), generator=g)
    if kind == "each":                                          # as few repeats as there can be, out of order
        return torch.randperm(max(n, vocab), generator=g)[:n] % vocab
    ids = (torch.exp(torch.rand(n, generator=g) * math.log(vocab)) - 1).long().clamp(0, vocab - 1)      # frequent first
    return torch.where(torch.rand(n, generator=g) < 0.5, torch.ones_like(ids).clamp(max=vocab - 1), ids)


EMBEDS = [(1, 1, 1), (1, 64, 100), (2, 7, 3), (77, 512, 49408), (300, 33, 1000), (511, 520, 50), (512, 1100, 300), (513, 16, 200),
          (700, 1030, 513), (1000, 64, 1), (1024, 2100, 90), (1025, 520, 30), (1500, 7, 40), (2000, 12, 2_100_000), (2048, 72, 70000), (2049, 72, 300), (4096, 40, 32000), (5000, 768, 511), (9000, 24, 300000), (20000, 72, 65536), (70000, 8, 600),
          (33000, 520, 20), (16601, 1024, 300), (12288, 16, 1000), (12289, 16, 600), (2100, 9, 511), (2100, 9, 512)]


@pytest.mark.parametrize("n,cols,vocab", EMBEDS)
@pytest.mark.parametrize("kind", ["one", "spread", "each", "frequent"])
@pytest.mark.parametrize("dtype", TYPES)
def test_embed_scaled(ops, gpu, n, cols, vocab, kind, dtype):
    g = torch.Generator().manual_seed(n + cols + vocab)
    ids = tokens_of(kind, n, vocab, g)
    scale = math.sqrt(cols)
    tok = ids.to(torch.int32).to(gpu)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    table = torch.randn(vocab, cols, generator=g).to(dtype)
    for od in TYPES:
        out = ops.embed_scaled_fwd(tok, table.to(gpu), scale, flag, od)
        assert torch.equal(out.cpu(), (table[ids].float() * scale).to(od))
    layout = "off" if n % 3 == 0 else "wide" if n % 3 == 1 else "plain"
    dy, dyr = make(n, cols, dtype, n, layout=layout)
    many = torch.bincount(ids, minlength=vocab).double()[:, None]
    want = torch.zeros(vocab, cols, dtype=torch.float64).index_add_(0, ids, dyr)
    size = torch.zeros(vocab, cols, dtype=torch.float64).index_add_(0, ids, dyr.abs())
    grad = ops.embed_scaled_bwd(dy, tok, vocab, scale, flag)
    bound = scale * U * (size * many + want.abs() * 2)          # a sum of `many` terms, the scale, its product
    close(grad, want * scale, bound, "grad")
    assert torch.equal(grad, ops.embed_scaled_bwd(dy, tok, vocab, scale, flag))           # the same bits every time
    assert (grad.cpu()[many[:, 0] == 0] == 0).all()
    # into a gradient that is there: rows without a token keep their bits
    base = torch.randn(vocab, cols, generator=g)
    base[::7] = math.nan
    base[ids[0]] = 1.0
    into = base.to(gpu)
    assert ops.embed_scaled_bwd(dy, tok, vocab, scale, flag, out=into, accumulate=True) is into
    quiet = many[:, 0] == 0
    assert same(into.cpu()[quiet], base[quiet])
    live = ~quiet & ~base.isnan().any(1)
    total = base.double() + want * scale
    close(into.cpu()[live], total[live], bound[live] + U * total.abs()[live] * 2, "accumulated")
    # a padding token's rows are left out, tokens outside the table too (and are reported)
    pad = int(ids[n // 2])
    wild = ids.clone()
    if n > 2:
        wild[0], wild[n - 1] = vocab + 5, -3
    keep = (wild >= 0) & (wild < vocab) & (wild != pad)
    part = torch.zeros(vocab, cols, dtype=torch.float64).index_add_(0, wild[keep], dyr[keep])
    flag.zero_()
    got = ops.embed_scaled_bwd(dy, wild.to(torch.int32).to(gpu), vocab, scale, flag, padding_idx=pad)
    close(got, part * scale, scale * U * (size * many + part.abs() * 2), "padded")
    assert (got[pad] == 0).all() and flag.item() == (1 if n > 2 else 0)
    if n > 2:
        flag.zero_()
        out = ops.embed_scaled_fwd(wild.to(torch.int32).to(gpu), table.to(gpu), scale, flag)
        assert flag.item() == 1 and torch.equal(out[0].cpu(), (table[0].float() * scale).to(dtype))


def test_embed_no_tokens(ops, gpu):
    ids = torch.zeros(0, dtype=torch.int32, device=gpu)
    assert ops.embed_scaled_fwd(ids, torch.ones(5, 8, device=gpu), 1.0).shape == (0, 8)
    grad = torch.full((5, 8), 2.0, device=gpu)
    dy = torch.zeros(0, 8, device=gpu)
    assert (ops.embed_scaled_bwd(dy, ids, 5, 1.0, out=grad, accumulate=True) == 2).all()
    assert (ops.embed_scaled_bwd(dy, ids, 5, 1.0, out=grad) == 0).all()


def test_embed_grad_against_differences(ops, gpu):
    """The lookup is linear: <grad, direction> is the exact change of <dy, out> along it."""
    g = torch.Generator().manual_seed(3)
    n, cols, vocab, scale = 900, 48, 60, 3.0
    ids = torch.randint(0, vocab, (n,), generator=g).to(torch.int32).to(gpu)
    table, v = torch.randn(vocab, cols, generator=g), torch.randn(vocab, cols, generator=g)
    dy = torch.randn(n, cols, generator=g)
    f = lambda t: (ops.embed_scaled_fwd(ids, t.to(gpu), scale).cpu().double() * dy.double()).sum()      # noqa: E731
    grad = ops.embed_scaled_bwd(dy.to(gpu), ids, vocab, scale).cpu().double()
    diff, slope = (f(table + v) - f(table - v)) / 2, (grad * v.double()).sum()
    assert abs(diff - slope).item() <= 40 * U * scale * n * cols * 4


# ------------------------------------------------------------------ large offsets, streams, graphs
def test_offsets_past_32_bits(ops, L, gpu):
    rows, cols = 1_050_000, 2080                                # 2.18e9 elements, 4.4 GB in 16 bits
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=gpu)
    for r0 in range(0, rows, 50_000):
        x[r0:r0 + 50_000].normal_()
    tail = x[-3:].clone()
    kept = ops.act8_pack(x)
    small = ops.act8_pack(tail)
    assert torch.equal(kept[0][-3:], small[0]) and torch.equal(kept[1][-3:], small[1])
    assert torch.equal(ops.act8_unpack(kept, torch.bfloat16)[-3:], ops.act8_unpack(small, torch.bfloat16))
    gamma = torch.ones(cols, device=gpu)
    y, rstd, kept2 = ops.rmsnorm_fwd(x, gamma, torch.bfloat16, save_stats=True, checkpoint=True)
    y2, r2, _ = ops.rmsnorm_fwd(tail, gamma, torch.bfloat16, save_stats=True)
    assert torch.equal(y[-3:], y2) and torch.equal(rstd[-3:], r2) and torch.equal(kept2[0][-3:], small[0])
    dg = torch.empty(cols, device=gpu)
    dx = ops.rmsnorm_bwd(y, kept2, gamma, rstd, dg)
    assert torch.equal(dx[-3:], ops.rmsnorm_bwd(y2, small, gamma, r2, dg))
    del x, kept, kept2, y, dx
    vocab, cols = 2_200_000, 1024                               # 2.25e9 elements of the table and of its gradient
    ids = torch.tensor([vocab - 1, 5, vocab - 2, vocab - 1] * 200, dtype=torch.int32, device=gpu)
    table = torch.zeros(vocab, cols, dtype=torch.bfloat16, device=gpu)
    table[-2:] = 3.0
    out = ops.embed_scaled_fwd(ids, table, 2.0)
    assert (out[0] == 6).all() and (out[1] == 0).all() and (out[2] == 6).all()
    del table
    grad = ops.embed_scaled_bwd(torch.ones(800, cols, device=gpu), ids, vocab, 0.5)
    assert (grad[-1] == 200).all() and (grad[-2] == 100).all() and (grad[5] == 100).all()
    assert (grad[6:-2].abs().amax() == 0) and (grad[:5] == 0).all()


def test_very_many_rows(ops, gpu):
    """More rows than one launch takes: what lies at and behind the seam is what a call on those rows alone gives."""
    rows, cols = (1 << 22) + 1000, 24
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(rows, cols, generator=g, device=gpu)
    delta = torch.randn(rows, cols, generator=g, device=gpu).half()
    gamma = torch.rand(cols, generator=g, device=gpu) + 0.5
    part = slice((1 << 22) - 500, rows)
    xo = torch.empty_like(x)
    y, rstd, kept = ops.rmsnorm_fwd(x, gamma, torch.float16, delta=delta, x_out=xo, save_stats=True, checkpoint=True)
    y8, scale, _, _ = ops.rmsnorm_fwd_fp8(x, gamma, delta=delta, write_x=False)
    xo2 = torch.empty_like(x[part])
    y2, r2, kept2 = ops.rmsnorm_fwd(x[part], gamma, torch.float16, delta=delta[part], x_out=xo2, save_stats=True, checkpoint=True)
    y82, scale2, _, _ = ops.rmsnorm_fwd_fp8(x[part], gamma, delta=delta[part], write_x=False)
    for a, b in ((y, y2), (rstd, r2), (kept[0], kept2[0]), (kept[1], kept2[1]), (xo, xo2), (y8, y82), (scale, scale2)):
        assert torch.equal(a[part], b)
    dg = torch.empty(cols, device=gpu)
    for dy, stream in ((y, kept), (xo, xo.bfloat16())):                       # the second mixture takes the walking kernels
        dx = ops.rmsnorm_bwd(dy, stream, gamma, rstd, dg)
        cut = (stream[0][part], stream[1][part]) if isinstance(stream, tuple) else stream[part]
        assert torch.equal(dx[part], ops.rmsnorm_bwd(dy[part], cut, gamma, rstd[part].clone(), torch.empty_like(dg)))
        assert torch.isfinite(dg).all()


def test_batched_rows(ops, gpu):
    """[batch, tokens, cols] tensors are rows of cols: the same bits as their two-dimensional views."""
    g = torch.Generator().manual_seed(8)
    x, dy = (torch.randn(3, 5, 200, generator=g).to(gpu) for _ in range(2))
    delta, gamma = torch.randn(3, 5, 200, generator=g).half().to(gpu), torch.rand(200, generator=g).to(gpu)
    y, rstd, kept = ops.rmsnorm_fwd(x, gamma, torch.float16, delta=delta, x_out=torch.empty_like(x), save_stats=True, checkpoint=True)
    y2, rstd2, kept2 = ops.rmsnorm_fwd(x.view(15, 200), gamma, torch.float16, delta=delta.view(15, 200),
                                       x_out=torch.empty(15, 200, device=gpu), save_stats=True, checkpoint=True)
    assert y.shape == x.shape and torch.equal(y.view(15, 200), y2) and torch.equal(rstd, rstd2)
    assert torch.equal(kept[0].view(15, 200), kept2[0]) and torch.equal(kept[1].view(15, 7), kept2[1])
    dg, dg2 = torch.empty(200, device=gpu), torch.empty(200, device=gpu)
    dx = ops.rmsnorm_bwd(dy, kept, gamma, rstd, dg)
    assert torch.equal(dx.view(15, 200), ops.rmsnorm_bwd(dy.view(15, 200), kept2, gamma, rstd, dg2)) and torch.equal(dg, dg2)
    ids = torch.randint(0, 40, (3, 5), generator=g).int().to(gpu)
    assert torch.equal(ops.embed_scaled_bwd(dy, ids, 40, 2.0), ops.embed_scaled_bwd(dy.view(15, 200), ids.view(15), 40, 2.0))
    one = ops.act8_pack(x[0, 0])                               # a single row
    assert torch.equal(ops.act8_unpack(one, torch.float32), ops.act8_unpack(ops.act8_pack(x), torch.float32)[0, 0])


def test_branch_that_is_the_stream(ops, gpu):
    for cols in (64, 1500, 9000):
        x = torch.randn(6, cols, device=gpu)
        want, _, _ = ops.rmsnorm_fwd(x + x, torch.ones(cols, device=gpu), torch.float32)
        double = x + x
        got, _, _ = ops.rmsnorm_fwd(x, torch.ones(cols, device=gpu), torch.float32, delta=x)      # in place
        assert torch.equal(got, want) and torch.equal(x, double)


def step(ops, L, s):
    """One pass through all of them: what a captured training step holds."""
    x = ops.embed_scaled_fwd(s["ids"], s["table"], 4.0, None, torch.float32)
    y, rstd, kept = ops.rmsnorm_fwd(x, s["gamma"], torch.float16, delta=s["delta"], save_stats=True, checkpoint=True)
    a, pre = ops.act8_gelu_fwd(y, L.ACT_TANH_GELU)
    da = ops.act8_gelu_bwd(a, pre, L.ACT_TANH_GELU)
    dg = torch.empty_like(s["gamma"])
    dx = ops.rmsnorm_bwd(da, kept, s["gamma"], rstd, dg)
    return a, dx, dg, ops.embed_scaled_bwd(dx, s["ids"], s["table"].shape[0], 4.0)


def fresh(n, vocab, cols, seed):
    g = torch.Generator().manual_seed(seed)
    return dict(ids=tokens_of("frequent", n, vocab, g).to(torch.int32).cuda(), table=torch.randn(vocab, cols, generator=g).cuda(),
                gamma=(1 + 0.1 * torch.randn(cols, generator=g)).cuda(), delta=torch.randn(n, cols, generator=g).half().cuda())


@pytest.mark.parametrize("n", [300, 1500, 3000])
def test_captured_step_replays_like_the_eager_one(ops, L, gpu, n):
    s = fresh(n, 700, 200, 1)
    step(ops, L, s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):                                      # two graphs of the same step: their workspaces are apart
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got = step(ops, L, s)
            graphs.append((graph, got))
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(2, 6):
        new = fresh(n, 700, 200, seed)
        for k in s:
            s[k].copy_(new[k])
        want = step(ops, L, s)
        for graph, got in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, got in graphs:
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_two_streams_at_once(ops, L, gpu):
    states = [fresh(4000, 900, 136, s) for s in (1, 2)]
    want = [step(ops, L, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = []
    for s, st in zip(states, streams):
        with torch.cuda.stream(st):
            got.append([step(ops, L, s) for _ in range(4)])
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        for run in runs:
            for a, b in zip(run, w):
                assert torch.equal(a, b)


# ------------------------------------------------------------------ together, as a block of a tower uses them
def test_block_from_tokens_to_table_gradient(ops, L, gpu):
    """Lookup -> RMS norm to e4m3 with the stream's checkpoint -> e4m3 product -> GELU with its checkpoint -> product; the
    backward through both checkpoints to the norm's weight and the table.  Every intermediate that is kept or rounded is taken
    as the kernels left it, and each following step is held to its own bound from there."""
    g = torch.Generator().manual_seed(11)
    n, width, hidden, vocab, scale = 640, 256, 512, 300, 16.0
    ids = tokens_of("frequent", n, vocab, g)
    tok = ids.to(torch.int32).to(gpu)
    table = (torch.randn(vocab, width, generator=g) * 0.05)
    gamma = 1 + 0.1 * torch.randn(width, generator=g)
    w1, w2 = torch.randn(hidden, width, generator=g) / 16, (torch.randn(width, hidden, generator=g) / 22).half()
    x = ops.embed_scaled_fwd(tok, table.to(gpu), scale, None, torch.float32)
    y8, sc, rstd, kept = ops.rmsnorm_fwd_fp8(x, gamma.to(gpu), save_stats=True, checkpoint=True)
    w8, wsc = ops.quantize_rows_fp8(w1.to(gpu))
    pre = ops.gemm_fp8(y8, sc, w8, wsc, out_dtype=torch.float32)
    a8 = y8.view(torch.float8_e4m3fn).float().cpu().double() * sc.cpu().double()[:, None]
    b8 = w8.view(torch.float8_e4m3fn).float().cpu().double() * wsc.cpu().double()[:, None]
    close(pre, a8 @ b8.t(), U * (width + 4) * (a8.abs() @ b8.abs().t()), "pre")
    pre16 = pre.half()
    a, kept_pre = ops.act8_gelu_fwd(pre16, L.ACT_TANH_GELU)
    out = ops.gemm(a, w2.to(gpu), out_dtype=torch.float32)
    ar = a.cpu().double()
    close(out, ar @ w2.double().t(), U * (hidden + 4) * (ar.abs() @ w2.double().abs().t()), "out")
    dout = (torch.randn(n, width, generator=g) * 0.1).half()
    da = ops.gemm(dout.to(gpu), w2.to(gpu), b_kn=True)
    dpre = ops.act8_gelu_bwd(da, kept_pre, L.ACT_TANH_GELU, out=da.clone())
    _, slope, _, xdu = act_ref(kept_ref(pre16.cpu().double())[2], "tanh")
    dar = da.cpu().double()
    close(dpre, dar * slope, (dar * slope).abs() * 2.0 ** -11 + dar.abs() * (1 + xdu) * 2.0 ** -20 + 2.0 ** -25, "dpre")
    dy = ops.gemm(dpre, w1.half().to(gpu), b_kn=True)
    dgamma = torch.empty(width, device=gpu)
    dx = ops.rmsnorm_bwd(dy, kept, gamma.to(gpu), rstd, dgamma)
    want, wg, h, b, m = rms_bwd_ref(dy.cpu().double(), kept_ref(x.cpu().double())[2], rstd.cpu().double(), gamma.double(), None)
    r = rstd.cpu().double()[:, None]
    fp32 = U * r * (5 * b.abs() + h.abs() * (20 * (b * h).abs().mean(1, keepdim=True) + 5 * m.abs()))
    close(dx, want, want.abs() * 2.0 ** -11 + 1.01 * fp32 + 2.0 ** -25, "dx")
    close(dgamma, wg, U * (n / 16 + 72) * (dy.cpu().double() * h).abs().sum(0), "dgamma")
    grad = ops.embed_scaled_bwd(dx, tok, vocab, scale)
    dxr = dx.cpu().double()
    wt = torch.zeros(vocab, width, dtype=torch.float64).index_add_(0, ids, dxr) * scale
    size = torch.zeros(vocab, width, dtype=torch.float64).index_add_(0, ids, dxr.abs()) * scale
    close(grad, wt, U * (torch.bincount(ids, minlength=vocab).double()[:, None] + 2) * size, "table gradient")


# ------------------------------------------------------------------ the LoRA towers' backward from 8-bit checkpoints
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("p_drop", [0.0, 0.25])
@pytest.mark.parametrize("policy", ["none", "mlp", "full"])
def test_lora_backward_from_checkpoints(ops, gpu, dtype, p_drop, policy):
    """`lora_checkpoint: int8` changes nothing in the forward, and its backward is the one of `native` with every kept
    activation replaced by what its checkpoint reads back as: the adapters' gradients are the same bits."""
    from bifold.losses import Losses
    from bifold.models import siglip_encoder
    from test_model_gpu import build_tiny_siglip
    T, B = 2, 2
    loss_fn = Losses.get_by_name(cfg=dict(name="bce_gaussmap", is_bimanual=True, mask_pick_heatmap=False))
    g = torch.Generator().manual_seed(77)
    sample = {"rgb": torch.randn(B, 3, 32, 32, generator=g), "rgb_context": torch.randn(B, T, 3, 32, 32, generator=g),
              "instruction": torch.randint(0, 100, (B, 64), generator=g),
              "context_attention_mask": torch.tensor([[1, 0], [1, 1]])}
    for hn in ("left_pick", "left_place", "right_pick", "right_place"):
        sample[f"{hn}_heatmap"] = torch.rand(B, 32, 32, generator=g)
    sample = {k: v.to(gpu) for k, v in sample.items()}
    seen = {}
    for how in ("native", "replaced", "int8"):
        torch.manual_seed(5)
        model = build_tiny_siglip("siglip_sequential", True, dtype, gpu, T, lora=True, r=8, lora_dropout=p_drop,
                                  lora_recompute=policy, lora_checkpoint="int8" if how == "int8" else "native")
        with torch.no_grad():
            gb = torch.Generator().manual_seed(6)
            for n, p in model.named_parameters():
                if ".lora_B." in n:
                    p.copy_(torch.randn(p.shape, generator=gb) * 0.05)
        model = model.to(gpu).train()
        torch.manual_seed(9)
        out = model(sample)
        loss, _ = loss_fn(out, sample)
        kept = 0
        for tower in model.siglip_model._saved.values():
            for S in tower["layers"]:
                for k in siglip_encoder._KEPT8:
                    kept += S[k] is not None
                    if S[k] is None:
                        continue
                    assert isinstance(S[k], tuple) == (how == "int8")
                    if how == "replaced":
                        S[k] = ops.act8_unpack(ops.act8_pack(S[k]), S[k].dtype)
        assert kept == 2 * 2 * {"none": 4, "mlp": 2, "full": 1}[policy]
        model.zero_grad()
        loss.backward()
        torch.cuda.synchronize()
        seen[how] = (loss.detach().clone(), {n: p.grad.detach().clone() for n, p in model.named_parameters()
                                             if p.requires_grad and ".lora_" in n})
    assert torch.equal(seen["int8"][0], seen["native"][0]) and len(seen["int8"][1]) == 16
    for n, gr in seen["replaced"][1].items():
        assert torch.equal(seen["int8"][1][n], gr), n
        assert torch.isfinite(gr).all() and gr.abs().max() > 0
    assert any(not torch.equal(seen["int8"][1][n], gr) for n, gr in seen["native"][1].items())


# ------------------------------------------------------------------ the erf GELU's digits far below zero
def erf_gelu_ref(x):
    """(x Phi(x), Phi(x), x phi(x)) in 64 bits; erfc keeps its digits at any x < 0."""
    cdf = 0.5 * torch.erfc(-x / math.sqrt(2))
    return x * cdf, cdf, x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


# 16-bit tensors: the exponential's argument is a product with a rounded log2(e), U |x^2| together at most; the polynomial's fit
# (13 U) and evaluation (7 U), reciprocal, exponential and products add less than 32 U; the result is rounded to the type.  An exponential under fp32's
# smallest normal number, 2^-126, may be 0, and Phi(-x) and x phi(x) are under 0.03 and 6 times it there (13 < x < 14).
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_act8_erf_gelu_of_every_16_bit_value(ops, L, gpu, dtype):
    x = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x) & (x.abs() <= 14)]
    x = torch.cat([x, torch.zeros(-len(x) % 64, dtype=dtype)]).view(-1, 64)
    y, _ = ops.act8_gelu_fwd(x.to(gpu), L.ACT_ERF_GELU)
    ref = x.double()
    want, _, _ = erf_gelu_ref(ref)
    bound = want.abs() * (half_step(dtype) + (ref * ref + 32) * U) + tiny_step(dtype)
    close(y, want, bound + torch.where(ref < -13, 2.0 ** -126, 0.0), "y")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_act8_erf_gelu_slope_of_every_kept_value(ops, L, gpu, dtype):
    """Checkpoints q 2^e as they can be: every q, steps 2^-12 to 2^-3."""
    q = torch.arange(-127, 128, dtype=torch.int8)
    q = torch.cat([q, q[:1]]).view(8, 32).repeat(10, 1).contiguous()
    code = torch.arange(115, 125, dtype=torch.uint8).repeat_interleave(8).view(-1, 1)
    at = q.double() * torch.exp2(code.double() - 127)
    slope = ops.act8_gelu_bwd(torch.ones(80, 32, dtype=dtype, device=gpu), (q.to(gpu), code.to(gpu)), L.ACT_ERF_GELU)
    _, cdf, part = erf_gelu_ref(at)
    want = cdf + part
    bound = want.abs() * half_step(dtype) + (cdf + part.abs()) * (at * at + 32) * U + tiny_step(dtype)
    close(slope, want, bound + torch.where(at < -13, 6 * 2.0 ** -126, 0.0), "slope")


# ------------------------------------------------------------------ fp16's largest numbers
@pytest.mark.parametrize("cols", [7, 32, 45, 96])
def test_finite_fp16_reads_back_finite(ops, gpu, cols):
    """65 280 (255 * 2^8) and above are kept as 64 * 2^10 = 2^16, which fp16 does not hold; a step of 2^10 is off by 2^9 at most."""
    top = torch.finfo(torch.float16).max
    x = torch.zeros(6, cols, dtype=torch.float16)
    x[0, 0], x[0, 1] = top, 1024.0
    x[1, cols - 1], x[1, 0] = -top, 3.0
    x[2, 3] = 65280.0
    x[3, 3] = 65248.0                                           # the largest number that is not kept as 2^16
    x[4, 0], x[4, cols - 1] = 65472.0, -65312.0
    x[5, 1] = math.inf
    kept = ops.act8_pack(x.to(gpu))
    back = ops.act8_unpack(kept, torch.float16).cpu()
    assert torch.isfinite(back[:5]).all() and back[5, :32].isnan().all()
    assert (back[:5].double() - x[:5].double()).abs().max() <= 512
    assert back[0, :2].tolist() == [top, 1024.0] and back[1, cols - 1] == -top and back[2, 3] == top and back[3, 3] == 65024.0
    wide = ops.act8_unpack(kept, torch.float32).cpu()           # a wider type holds what is kept
    assert wide[0, 0] == 65536.0 and wide[1, cols - 1] == -65536.0
    far = torch.zeros(1, cols)
    far[0, 0], far[0, 1] = 1e5, -1e5                            # no fp16 number: an overflow stays one
    assert ops.act8_unpack(ops.act8_pack(far.to(gpu)), torch.float16)[0, :2].tolist() == [math.inf, -math.inf]


# ------------------------------------------------------------------ outputs in the columns beside their inputs
@pytest.mark.parametrize("cols,wide", [(64, 192), (37, 120), (7, 23), (1155, 3500), (17000, 51003)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_outputs_in_columns_of_the_inputs_buffer(ops, L, gpu, cols, wide, dtype):
    """dy, dpre, the stream and the sum in one packed buffer: the same bits as apart, and the other columns untouched."""
    rows = 9
    buf = make(rows, wide, dtype, cols)[0]
    before = buf.clone()
    src, dst = buf[:, cols:2 * cols], buf[:, 2 * cols:3 * cols]
    kept = ops.act8_pack(src.contiguous())
    want = ops.act8_gelu_bwd(src.contiguous(), kept, L.ACT_TANH_GELU)
    assert ops.act8_gelu_bwd(src, kept, L.ACT_TANH_GELU, out=dst) is dst
    assert torch.equal(dst, want) and torch.equal(buf[:, :2 * cols], before[:, :2 * cols])
    assert torch.equal(buf[:, 3 * cols:], before[:, 3 * cols:])
    buf.copy_(before)
    gamma, delta = 1 + torch.rand(cols, device=gpu), buf[:, :cols]
    total = torch.empty(rows, cols, dtype=dtype, device=gpu)
    want, _, _ = ops.rmsnorm_fwd(src.contiguous(), gamma, dtype, delta=delta.contiguous(), x_out=total)
    y, _, _ = ops.rmsnorm_fwd(src, gamma, dtype, delta=delta, x_out=dst)
    assert torch.equal(y, want) and torch.equal(dst, total) and torch.equal(buf[:, :2 * cols], before[:, :2 * cols])
    assert torch.equal(buf[:, 3 * cols:], before[:, 3 * cols:])


# ------------------------------------------------------------------ the lookup's longest form on odd widths
@pytest.mark.parametrize("n,cols", [(17000, 1027), (2101, 8179)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embed_lookup_of_many_odd_rows(ops, gpu, n, cols, dtype):
    """Over 2^21 vectors of 4 (fp32) or 8 elements and no whole number of 1 024: four vectors a lane, the last workgroup's
    lanes past the end."""
    many = n * -(-cols // (4 if dtype == torch.float32 else 8))
    assert many >= 1 << 21 and many % 1024
    g = torch.Generator(device="cuda").manual_seed(n)
    table = torch.randn(777, cols, generator=g, device=gpu).to(dtype)
    ids = torch.randint(0, 777, (n,), generator=g, device=gpu, dtype=torch.int32)
    ids[n - 1] = 776
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    for od in TYPES:
        out = ops.embed_scaled_fwd(ids, table, 3.0, flag, od)
        assert torch.equal(out, (table[ids.long()].float() * 3.0).to(od))
    assert flag.item() == 0


# ------------------------------------------------------------------ each group's own error
@pytest.mark.parametrize("cols", [32, 70, 1024])
@pytest.mark.parametrize("dtype", TYPES)
def test_act8_error_of_each_group(ops, gpu, cols, dtype):
    """Rows of every magnitude: an element is off by half a step, which is at most its group's largest / 127, or 2^-127 where the
    smallest step, 2^-126, is used."""
    low, high = {torch.float32: (-149, 126), torch.bfloat16: (-133, 126), torch.float16: (-24, 14)}[dtype]
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(high - low + 1, cols, generator=g).clamp(-3, 3).double()
    x = (x * torch.exp2(torch.arange(low, high + 1).double())[:, None] / 4).to(dtype)
    q, code = ops.act8_pack(x.to(gpu))
    back = ops.act8_unpack((q, code), torch.float32).cpu().double()
    full = torch.zeros(2, x.shape[0], -(-cols // 32) * 32, dtype=torch.float64)
    full[0, :, :cols], full[1, :, :cols] = x.double(), back
    full = full.view(2, x.shape[0], -1, 32)
    top = full[0].abs().amax(2)
    half = torch.exp2(code.cpu().double() - 128)
    assert ((full[0] - full[1]).abs() <= half[..., None]).all()
    assert (half <= torch.maximum(top / 127, torch.full_like(top, 2.0 ** -127))).all()


# ------------------------------------------------------------------ how far the int8 gradients lie from the native ones
# What a kept tensor's error does to an adapter's gradient: each use multiplies the gradient by a factor made of the tensor --
# h1 in dY^T h1, x and xm through the normed rows of a LayerNorm's backward -- and moves it, relatively, by no more than the
# tensor (a stream: than what is left of it without its mean); the GELU's slope by twice that (|act''| <= 1.13 against slopes
# of some half).  Where tensors are made again from x or xm they inherit that error: `mlp` uses x twice (LayerNorm, h1) and xm
# three times (LayerNorm, slope), `full` x eight times (LayerNorm, h1, q, k, v, xm, slope).  The roundings of different tensors
# are independent, so the sum of all uses over all layers is an upper end of what they make together.
USES = {"none": {"x": 1, "h1": 1, "xm": 1, "pre": 2}, "mlp": {"x": 2, "xm": 3}, "full": {"x": 8}}


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("outlier", [0.0, 30.0])
@pytest.mark.parametrize("policy", ["none", "mlp", "full"])
def test_int8_gradients_lie_near_the_native_ones(ops, gpu, dtype, outlier, policy):
    """Relative distance of a tower's adapter gradients, int8 against native, under what the kept tensors' own errors allow; also
    with one column of the residual stream far larger than the rest (its group's step is as coarse as that column)."""
    from bifold.losses import Losses
    from test_model_gpu import build_tiny_siglip
    T, B = 2, 2
    loss_fn = Losses.get_by_name(cfg=dict(name="bce_gaussmap", is_bimanual=True, mask_pick_heatmap=False))
    g = torch.Generator().manual_seed(78)
    sample = {"rgb": torch.randn(B, 3, 32, 32, generator=g), "rgb_context": torch.randn(B, T, 3, 32, 32, generator=g),
              "instruction": torch.randint(0, 100, (B, 64), generator=g),
              "context_attention_mask": torch.tensor([[1, 0], [1, 1]])}
    for hn in ("left_pick", "left_place", "right_pick", "right_place"):
        sample[f"{hn}_heatmap"] = torch.rand(B, 32, 32, generator=g)
    sample = {k: v.to(gpu) for k, v in sample.items()}
    grads, allowed = {}, {}
    for how in ("native", "int8"):
        torch.manual_seed(5)
        model = build_tiny_siglip("siglip_sequential", True, dtype, gpu, T, lora=True, r=8, lora_dropout=0.0,
                                  lora_recompute=policy, lora_checkpoint=how)
        with torch.no_grad():
            gb = torch.Generator().manual_seed(6)
            for n, p in model.named_parameters():
                if ".lora_B." in n:
                    p.copy_(torch.randn(p.shape, generator=gb) * 0.05)
                if n.endswith("position_embedding.weight"):
                    p[:, 5] += outlier
        model = model.to(gpu).train()
        torch.manual_seed(9)
        loss, _ = loss_fn(model(sample), sample)
        if how == "native":
            for tower, kept in model.siglip_model._saved.items():
                total = 0.0
                for S in kept["layers"]:
                    for k, uses in USES[policy].items():
                        t = S[k].double()
                        off = ops.act8_unpack(ops.act8_pack(S[k]), torch.float32).double() - t
                        size = t - t.mean(-1, keepdim=True) if k in ("x", "xm") else t
                        total += uses * (off.norm() / size.norm()).item()
                allowed[tower] = total
        model.zero_grad()
        loss.backward()
        torch.cuda.synchronize()
        for tower in allowed:
            rows = [p.grad.detach().double().flatten() for n, p in model.named_parameters()
                    if p.requires_grad and ".lora_" in n and tower in n]
            assert len(rows) == 8
            grads[how, tower] = torch.cat(rows)
    for tower, most in allowed.items():
        native, int8 = grads["native", tower], grads["int8", tower]
        far = ((int8 - native).norm() / native.norm()).item()
        cos = (torch.dot(int8, native) / (int8.norm() * native.norm())).item()
        print(f"{tower} {policy} {dtype} outlier {outlier:g}: {far:.4f} of {most:.4f} allowed, cosine {cos:.6f}", flush=True)
        assert 0 < far <= most and most < 1, (tower, far, most)
        assert cos >= 1 - most * most / 2                        # what a relative distance of `most` allows, in first order
