"""Layer norm forward and backward against 64 bits.

Tolerances.  A row's sums are taken by threads of at most L elements each and
joined over lanes and warps: off by (L + 16) 2^-24 of the mean magnitude.
Each output is a short chain of fp32 operations (counted as 2^-20 of its
terms) and one rounding to its type.  A column sum over r rows is off by at
most (r + 64) 2^-24 of its sum of magnitudes, and by its terms' own errors."""
import math

import pytest
import torch

from tests import training_oracle as orc

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5


def close(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((err - tol).max()),
                           bad.nonzero()[:4].tolist())


def make(rows, cols, dtype, weight, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * (torch.rand(cols, generator=g) + 0.3)
         + offset).to(dtype)
    gamma = (torch.randn(cols, generator=g) * 0.2 + 1).to(weight)
    beta = (torch.randn(cols, generator=g) * 0.2).to(weight)
    dy = torch.randn(rows, cols, generator=g).to(dtype)
    res = torch.randn(rows, cols, generator=g).to(dtype)
    return x, gamma, beta, dy, res


def check_forward(nvlib, x, gamma, beta, xd=None, eps=EPS):
    rows, cols = x.shape
    amax = torch.empty(1, device="cuda")
    y, mean, rstd = nvlib.layernorm(x.cuda() if xd is None else xd, gamma.cuda(),
                                    None if beta is None else beta.cuda(), eps, amax_out=amax)
    wy, wm, wr = orc.layernorm(x, gamma, beta, eps)
    L = max(32, cols // 256) + 16
    size = x.double().abs().amax(1)
    em = L * 2.0 ** -24 * size
    close(mean, wm, em + 2.0 ** -24 * wm.abs(), "mean")
    # var = mean (x - mean)^2: relative 2 em^2-free error of L 2^-24, halved by the root
    close(rstd, wr, L * 2.0 ** -23 * wr + wr ** 3 * em ** 2, "rstd")
    h = (x.double() - wm[:, None]) * wr[:, None]
    g = gamma.double().abs()
    tol = (wr[:, None] * g * em[:, None] + L * 2.0 ** -22 * h.abs() * g
           + 2.0 ** -23 * (0 if beta is None else beta.double().abs()))
    close(y, wy, tol + (orc.half_step(x.dtype) + 2.0 ** -23) * wy.abs()
          + orc.least_step(x.dtype), "y")
    assert float(amax) == float(y.float().abs().max())
    return mean, rstd


def check_backward(nvlib, x, gamma, dy, res, mean, rstd, dev=None):
    rows, cols = x.shape
    xd, dyd, resd = dev or (x.cuda(), dy.cuda(), None if res is None else res.cuda())
    dx, dg, db = nvlib.layernorm_backward(dyd, xd, mean, rstd, gamma.cuda(), residual=resd)
    m, r = mean.cpu(), rstd.cpu()
    wdx, wdg, wdb = orc.layernorm_backward(dy, x, m, r, gamma, res)
    L = max(32, cols // 256) + 16
    h = (x.double() - m.double()[:, None]) * r.double()[:, None]
    u = (dy.double() * gamma.double()).abs()
    part = r.double()[:, None] * (u + u.mean(1, keepdim=True)
                                  + h.abs() * (u * h.abs()).mean(1, keepdim=True))
    tol = L * 2.0 ** -22 * part + 2.0 ** -23 * (0 if res is None else res.double().abs())
    close(dx, wdx, tol + orc.half_step(x.dtype) * wdx.abs()
          + orc.least_step(x.dtype), "dx")
    hw = orc.half_step(gamma.dtype)
    sub = orc.least_step(gamma.dtype)
    t = (dy.double() * h).abs().sum(0)
    close(dg, wdg, (rows + 64) * 2.0 ** -24 * t + 2.0 ** -22 * t + hw * wdg.abs() + sub, "dgamma")
    t = dy.double().abs().sum(0)
    close(db, wdb, (rows + 64) * 2.0 ** -24 * t + hw * wdb.abs() + sub, "dbeta")


SHAPES = [(1200, 8192), (1190, 1024), (3000, 4096), (2000, 40), (1, 1), (1, 8), (3, 7), (2, 16), (5, 64), (17, 129), (4, 256), (33, 1000), (7, 1024),
          (300, 520), (9, 4099), (2, 5120), (400, 2048), (3, 8192), (2, 8200), (2, 12288),
          (2, 16384), (3, 16392), (1, 16411), (2, 40000), (1200, 24)]


@pytest.mark.parametrize("dtype,weight", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"),
                                          ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_both_passes(nvlib, rows, cols, dtype, weight):
    x, gamma, beta, dy, res = make(rows, cols, TYPES[dtype], TYPES[weight], rows * 3 + cols)
    mean, rstd = check_forward(nvlib, x, gamma, beta if cols % 2 else None)
    check_backward(nvlib, x, gamma, dy, res if rows % 2 else None, mean, rstd)
    check_backward(nvlib, x, gamma, dy, None if rows % 2 else res, mean, rstd)
    assert nvlib.device_error() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,shift", [(8, 0), (8, 8), (3, 1)])
def test_strides(nvlib, dtype, pad, shift):
    """Rows inside a wider buffer, at aligned and odd places."""
    rows, cols = 37, 192
    x, gamma, beta, dy, res = make(rows, cols, TYPES[dtype], torch.float32, 5)

    def place(t):
        buf = torch.full((rows, cols + pad + shift), 9.0, dtype=t.dtype, device="cuda")
        buf[:, shift:shift + cols] = t.cuda()
        return buf[:, shift:shift + cols]
    px, pdy, pres = place(x), place(dy), place(res)
    mean, rstd = check_forward(nvlib, x, gamma, beta, xd=px)
    check_backward(nvlib, x, gamma, dy, res, mean, rstd, dev=(px, pdy, pres))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols,pad", [(1203, 33, 0), (1203, 33, 1), (1203, 262, 2),
                                           (901, 1027, 0), (901, 1030, 4), (640, 4098, 8),
                                           (310, 8191, 1), (5, 3, 5), (3000, 9, 2),
                                           (1100, 8190, 3), (4100, 2050, 1), (8300, 1011, 0)])
@pytest.mark.parametrize("places", [(0, 0, 0), (1, 1, 1), (6, 6, 6), (1, 2, 3)])
def test_unaligned_rows(nvlib, rows, cols, pad, places, dtype):
    """Rows of any phase of 16 bytes, the same in all arrays and not, many to a
    block; what lies around the outputs' rows stays as it was."""
    x, gamma, beta, dy, res = make(rows, cols, TYPES[dtype], torch.float32, rows + cols)

    def place(t, at):
        ld = cols + pad
        flat = torch.full((rows * ld + 16,), 77.0, dtype=t.dtype, device="cuda")
        v = flat[at:at + rows * ld].view(rows, ld)[:, :cols]
        v.copy_(t)
        return flat, v

    def around(flat, at):
        keep = flat.clone()
        keep[at:at + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = 77.0
        return bool((keep == 77.0).all())
    (_, xd), (_, dyd), (_, rd) = (place(t, at) for t, at in zip((x, dy, res), places))
    mean, rstd = check_forward(nvlib, x, gamma, beta, xd)
    check_backward(nvlib, x, gamma, dy, res, mean, rstd, (xd, dyd, rd))
    # the same through the addresses, in place: outputs at the inputs' phases
    y, _, _ = nvlib.layernorm(xd, gamma.cuda(), beta.cuda())
    dx, dg, db = nvlib.layernorm_backward(dyd, xd, mean, rstd, gamma.cuda(), residual=rd)
    ld = cols + pad
    flat, yd = place(x, places[0])
    amax = torch.empty(1, device="cuda")
    nvlib.layernorm_fwd(rows, cols, yd, ld, gamma.cuda(), beta.cuda(), x.dtype, torch.float32, EPS,
                        yd, ld, None, None, amax)
    flat2, dxd = place(dy, places[1])
    ws = torch.empty(nvlib.layernorm_bwd_workspace_bytes(rows, cols), dtype=torch.uint8,
                     device="cuda")
    dg2, db2 = torch.empty_like(dg), torch.empty_like(db)
    nvlib.layernorm_bwd(rows, cols, dxd, ld, xd, ld, mean, rstd, gamma.cuda(), rd, ld, x.dtype,
                        torch.float32, dxd, ld, dg2, db2, ws, ws.numel())
    torch.cuda.synchronize()
    # Two results of the same formula: each within its check's tolerance.
    L = max(32, cols // 256) + 16
    m, r = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    h, g = (x.double() - m) * r, gamma.double().abs()
    one = (r * g * L * 2.0 ** -24 * x.double().abs().amax(1, keepdim=True)
           + L * 2.0 ** -22 * h.abs() * g + 2.0 ** -23 * beta.double().abs()
           + (orc.half_step(x.dtype) + 2.0 ** -23) * y.double().cpu().abs() * (1 + 2.0 ** -6)
           + orc.least_step(x.dtype))
    close(yd, y.double().cpu(), 2 * one, "y in place")
    u = (dy.double() * gamma.double()).abs()
    part = r * (u + u.mean(1, keepdim=True) + h.abs() * (u * h.abs()).mean(1, keepdim=True))
    one = (L * 2.0 ** -22 * part + 2.0 ** -23 * res.double().abs()
           + orc.half_step(x.dtype) * dx.double().cpu().abs() * (1 + 2.0 ** -6)
           + orc.least_step(x.dtype))
    close(dxd, dx.double().cpu(), 2 * one, "dx in place")
    t = 2 * (rows + 70) * 2.0 ** -24
    close(dg2, dg.double().cpu(), t * (dy.double() * h).abs().sum(0), "dgamma in place")
    close(db2, db.double().cpu(), t * dy.double().abs().sum(0), "dbeta in place")
    assert float(amax) == float(yd.float().abs().max())
    assert around(flat, places[0]) and around(flat2, places[1])
    assert nvlib.device_error() == 0


def test_offset_and_outliers(nvlib):
    """A common offset far above the spread, and a first element far off: the
    statistics keep their digits."""
    x, gamma, beta, _, _ = make(20, 3000, torch.float32, torch.float32, 8, offset=1000.0)
    check_forward(nvlib, x, gamma, beta)
    x, gamma, beta, _, _ = make(20, 4096, torch.bfloat16, torch.float32, 9)
    x[:, 0] = 500.0
    check_forward(nvlib, x, gamma, beta)


def test_constant_rows_and_nan(nvlib):
    x, gamma, beta, _, _ = make(6, 512, torch.float32, torch.float32, 4)
    x[1] = 3.25
    x[2] = 0.0
    check_forward(nvlib, x, gamma, beta)
    x[4, 100] = math.nan
    x[5, 7] = math.inf
    amax = torch.empty(1, device="cuda")
    y, mean, rstd = nvlib.layernorm(x.cuda(), gamma.cuda(), beta.cuda(), EPS, amax_out=amax)
    y = y.cpu()
    assert bool(torch.isnan(y[4:]).all()) and bool(torch.isfinite(y[:4]).all())
    assert math.isnan(float(amax))


def test_in_place(nvlib):
    """y over x, dx over dy and over the residual, through the pointer-level calls."""
    for rows, cols in ((50, 640), (50, 641), (3, 20001)):
        x, gamma, beta, dy, res = make(rows, cols, torch.float32, torch.float32, cols)
        x, gamma, beta, dy, res = (t.cuda() for t in (x, gamma, beta, dy, res))
        y, mean, rstd = nvlib.layernorm(x, gamma, beta)
        xx = x.clone()
        nvlib.layernorm_fwd(rows, cols, xx, cols, gamma, beta, x.dtype, gamma.dtype, EPS, xx, cols,
                            None, None, None)
        assert torch.equal(xx, y)
        dx, dg, db = nvlib.layernorm_backward(dy, x, mean, rstd, gamma, residual=res)
        nb = nvlib.layernorm_bwd_workspace_bytes(rows, cols)
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        for over in (dy, res):
            keep = over.clone()
            g2, b2 = torch.empty_like(dg), torch.empty_like(db)
            nvlib.layernorm_bwd(rows, cols, dy, cols, x, cols, mean, rstd, gamma, res, cols,
                                x.dtype, gamma.dtype, over, cols, g2, b2, ws, nb)
            assert torch.equal(over, dx) and torch.equal(g2, dg) and torch.equal(b2, db)
            over.copy_(keep)


def test_empty(nvlib):
    gamma = torch.ones(40, device="cuda")
    x = torch.empty(0, 40, device="cuda")
    amax = torch.full((1,), 3.0, device="cuda")
    y, mean, rstd = nvlib.layernorm(x, gamma, amax_out=amax)
    assert y.shape == (0, 40) and float(amax) == 0.0
    dx, dg, db = nvlib.layernorm_backward(x, x, mean, rstd, gamma)
    assert float(dg.abs().max()) == 0.0 and float(db.abs().max()) == 0.0 and dx.shape == (0, 40)


def test_gradient_by_differences(nvlib):
    """The backward pass is the derivative of the forward pass: central
    differences of sum(y w) in 64 bits around the fp32 inputs.  With step
    2^-8 the third-order term is below 2^-16 of the terms' size here."""
    rows, cols = 3, 24
    x, gamma, beta, dy, _ = make(rows, cols, torch.float32, torch.float32, 77)
    _, mean, rstd = nvlib.layernorm(x.cuda(), gamma.cuda(), beta.cuda())
    dx, dg, db = (t.double().cpu() for t in
                  nvlib.layernorm_backward(dy.cuda(), x.cuda(), mean, rstd, gamma.cuda()))
    step = 2.0 ** -8

    def loss(a, ga, be):
        return float((orc.layernorm(a, ga, be, EPS)[0] * dy.double()).sum())
    for r, c in ((0, 0), (1, 5), (2, 23)):
        e = torch.zeros(rows, cols, dtype=torch.float64)
        e[r, c] = step
        num = (loss(x.double() + e, gamma, beta) - loss(x.double() - e, gamma, beta)) / (2 * step)
        assert abs(num - float(dx[r, c])) < 2.0 ** -10
        v = torch.zeros(cols, dtype=torch.float64)
        v[c] = step
        num = (loss(x, gamma.double() + v, beta) - loss(x, gamma.double() - v, beta)) / (2 * step)
        assert abs(num - float(dg[c])) < 2.0 ** -16
        num = (loss(x, gamma, beta.double() + v) - loss(x, gamma, beta.double() - v)) / (2 * step)
        assert abs(num - float(db[c])) < 2.0 ** -16


@pytest.mark.parametrize("rows,cols", [(700, 1024), (300, 777)])
def test_streams_and_capture(nvlib, rows, cols):
    x, gamma, beta, dy, res = (t.cuda() for t in make(rows, cols, torch.bfloat16, torch.float32, 6))
    y, mean, rstd = nvlib.layernorm(x, gamma, beta)
    want = nvlib.layernorm_backward(dy, x, mean, rstd, gamma, residual=res)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            got += [nvlib.layernorm_backward(dy, x, mean, rstd, gamma, residual=res)
                    for _ in range(3)]
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(g, want))
    amax = torch.empty(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gm, gr = nvlib.layernorm(x, gamma, beta, amax_out=amax)
        gg = nvlib.layernorm_backward(dy, x, gm, gr, gamma, residual=res)
    for k in range(2):
        x.mul_(0.5)       # the amax of the second replay is not the first one's
        gamma.mul_(0.5)
        graph.replay()
        y, mean, rstd = nvlib.layernorm(x, gamma, beta)
        want = nvlib.layernorm_backward(dy, x, mean, rstd, gamma, residual=res)
        torch.cuda.synchronize()
        assert torch.equal(gy, y) and all(torch.equal(p, q) for p, q in zip(gg, want))
        assert float(amax) == float(y.float().abs().max())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cols", [40, 100, 501, 777, 1000, 4097, 5000, 5120, 12288, 16411, 70001])
def test_constant_rows_give_beta(nvlib, cols, dtype):
    """A row of one value, whatever its digits: the mean is that value, and y is
    beta, however small eps is."""
    g = torch.Generator().manual_seed(cols)
    values = torch.cat([torch.tensor([935.1373, 0.1, -1.0 / 3.0, 1000.1]),
                        torch.rand(60, generator=g) * 1000.0]).to(TYPES[dtype])
    x = values[:, None].expand(values.numel(), cols).contiguous()
    gamma, beta = torch.randn(2, cols, generator=g)
    for eps in (1e-5, 1e-12):
        y, mean, rstd = nvlib.layernorm(x.cuda(), gamma.cuda(), beta.cuda(), eps)
        assert torch.equal(mean.cpu(), values.float())
        assert torch.equal(y.cpu(), beta.to(TYPES[dtype]).expand_as(x))


@pytest.mark.parametrize("cols", [100, 777, 1000, 5000, 5120, 12288, 20001])
@pytest.mark.parametrize("offset", [1000.0, -935.1373, 60000.0])
def test_mean_of_rows_with_an_offset(nvlib, cols, offset):
    """The mean is off by two roundings (a warp's and the row's, 2^-24 of it each)
    and by its sums of differences: chains of at most 64 additions, 2^-18 of the
    mean difference."""
    x, gamma, beta, _, _ = make(24, cols, torch.float32, torch.float32, cols, offset=offset)
    y, mean, rstd = nvlib.layernorm(x.cuda(), gamma.cuda(), beta.cuda(), EPS)
    wy, wm, wr = orc.layernorm(x, gamma, beta, EPS)
    spread = (x.double() - wm[:, None]).abs()
    em = 2.0 ** -23 * wm.abs() + 2.0 ** -18 * spread.mean(1)
    close(mean, wm, em, "mean")
    g, h = gamma.double().abs(), spread * wr[:, None]
    close(y, wy, g * ((wr * em)[:, None] + 64 * 2.0 ** -22 * h) + 2.0 ** -22 * beta.double().abs()
          + 2.0 ** -23 * wy.abs(), "y")


def test_rows_without_columns(nvlib):
    """Nothing has no mean: NaN, not what the memory held."""
    rows = 1000
    for _ in range(3):
        torch.full((rows,), 5.0, device="cuda")      # freed at once: the next ones' memory
    x, w = torch.empty(rows, 0, device="cuda"), torch.empty(0, device="cuda")
    y, mean, rstd = nvlib.layernorm(x, w)
    assert y.shape == (rows, 0)
    assert bool(torch.isnan(mean).all()) and bool(torch.isnan(rstd).all())
    dx, dg, db = nvlib.layernorm_backward(x, x, mean, rstd, w)
    assert dx.shape == (rows, 0) and dg.numel() == db.numel() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,cols,pad", [(8300, 1011, 0), (4100, 2050, 1), (1100, 8190, 3)])
def test_unaligned_rows_with_16_bit_weights(nvlib, rows, cols, pad, dtype):
    """Enough elements for the backward pass by vectors with partial ends."""
    x, gamma, beta, dy, res = make(rows, cols, TYPES[dtype], TYPES[dtype], rows - cols)

    def place(t):
        flat = torch.zeros(rows * (cols + pad) + 8, dtype=t.dtype, device="cuda")
        v = flat[1:1 + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        v.copy_(t)
        return v
    xd, dyd, rd = place(x), place(dy), place(res)
    mean, rstd = check_forward(nvlib, x, gamma, beta, xd)
    # dx is a tensor of its own: the phases agree where its rows are as long as x's
    check_backward(nvlib, x, gamma, dy, res, mean, rstd, (xd, dyd, rd))
    check_backward(nvlib, x, gamma, dy, None, mean, rstd, (xd, dyd, None))
    # and over dy, whose rows start where x's do
    dx, dg, db = nvlib.layernorm_backward(dyd, xd, mean, rstd, gamma.cuda(), residual=rd)
    ws = torch.empty(nvlib.layernorm_bwd_workspace_bytes(rows, cols), dtype=torch.uint8,
                     device="cuda")
    dg2, db2, ld = torch.empty_like(dg), torch.empty_like(db), cols + pad
    nvlib.layernorm_bwd(rows, cols, dyd, ld, xd, ld, mean, rstd, gamma.cuda(), rd, ld, x.dtype,
                        gamma.dtype, dyd, ld, dg2, db2, ws, ws.numel())
    wdx, wdg, wdb = orc.layernorm_backward(dy, x, mean.cpu(), rstd.cpu(), gamma, res)
    m, r = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    h, L = (x.double() - m) * r, max(32, cols // 256) + 16
    u = (dy.double() * gamma.double()).abs()
    part = r * (u + u.mean(1, keepdim=True) + h.abs() * (u * h.abs()).mean(1, keepdim=True))
    close(dyd, wdx, L * 2.0 ** -22 * part + 2.0 ** -23 * res.double().abs()
          + orc.half_step(x.dtype) * wdx.abs() + orc.least_step(x.dtype), "dx over dy")
    for got, want, t in ((dg2, wdg, (dy.double() * h).abs()), (db2, wdb, dy.double().abs())):
        close(got, want, ((rows + 64) * 2.0 ** -24 + 2.0 ** -22) * t.sum(0)
              + orc.half_step(gamma.dtype) * want.abs() + orc.least_step(gamma.dtype), "weights")
    assert nvlib.device_error() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2), (2, 3), (1, 7), (3, 8), (1, 9), (2, 15),
                                       (1, 17), (2, 130), (1, 705), (3, 1023), (301, 709)])
def test_ends_of_the_first_and_last_row(nvlib, rows, cols, dtype):
    """Rows that start and end anywhere in 16 bytes, also both in the same: what lies
    before the first and behind the last is not read (NaN there shows nowhere)."""
    unit = 16 // TYPES[dtype].itemsize
    for at in range(unit):
        x, gamma, beta, dy, res = make(rows, cols, TYPES[dtype], torch.float32, 7 * cols + at)

        def place(t, at):
            flat = torch.full((rows * cols + 3 * unit,), math.nan, dtype=t.dtype, device="cuda")
            v = flat[unit + at:unit + at + rows * cols].view(rows, cols)
            v.copy_(t)
            return v
        px, pdy, pres = place(x, at), place(dy, (at * 3) % unit), place(res, (at * 5 + 1) % unit)
        mean, rstd = check_forward(nvlib, x, gamma, beta, px)
        check_backward(nvlib, x, gamma, dy, res, mean, rstd, (px, pdy, pres))
        check_backward(nvlib, x, gamma, dy, None, mean, rstd, (px, place(dy, at), None))
    assert nvlib.device_error() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(149, 5003), (297, 4099), (297, 709), (1185, 131), (4737, 33)])
def test_ends_where_a_grid_would_give_them_to_one_block(nvlib, rows, cols, dtype):
    """One row more than a multiple of the blocks that fill 148 SMs."""
    x, gamma, beta, dy, res = make(rows, cols, TYPES[dtype], torch.float32, rows)

    def place(t, at):
        flat = torch.full((rows * cols + 48,), math.nan, dtype=t.dtype, device="cuda")
        v = flat[16 + at:16 + at + rows * cols].view(rows, cols)
        v.copy_(t)
        return v
    for places in ((1, 1, 1), (3, 1, 2)):
        px, pdy, pres = (place(t, at) for t, at in zip((x, dy, res), places))
        mean, rstd = check_forward(nvlib, x, gamma, beta, px)
        check_backward(nvlib, x, gamma, dy, res, mean, rstd, (px, pdy, pres))
    assert nvlib.device_error() == 0
