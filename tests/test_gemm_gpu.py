"""The product of two NVFP4 operands and its epilogues against 64 bits.

Tolerances.  Code products and scales are exact; what rounds is
- the fp32 accumulation: k / 64 tensor-core additions and the sums inside each,
  counted as (k / 64 + 8) steps of 2^-22 of the sum of magnitudes;
- S_a S_b: a few 2^-24;
- the activation: exp with 2 + 1.173 |x| steps of 2^-23 for an argument |x|
  <= 60 here, so a sigmoid is off by at most 2^-16 q (1 - q) + 2^-22;
- the output: half a step of its type, relative to a normal number, or half a
  subnormal step."""
import math

import pytest
import torch

from tests import training_oracle as orc

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def problem(m, n, k, seed):
    # amax 2688 / 2^7: with the scales of random_operand z is of order sqrt(k) / 40
    a = orc.random_operand(m, k, seed, 3.0)
    b = orc.random_operand(n, k, seed + 1, 9.0 / math.sqrt(k))
    va, vb = orc.operand_values(*a), orc.operand_values(*b)
    z = va @ vb.t()
    size = va.abs() @ vb.abs().t()
    return a, b, z, (k / 64 + 8) * 2.0 ** -22 * size + 2.0 ** -21 * z.abs()


def cuda(ts):
    return [t.cuda() for t in ts]


def act_error(z, act):
    """Error of act(z) for exact z, and its Lipschitz constant."""
    if act in ("none", "relu"):
        return 0.0, 1.0
    x = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    q = torch.sigmoid(x)
    return z.abs() * (2.0 ** -16 * q * (1 - q) + 2.0 ** -22), 1.2


def slope_error(z, act):
    if act in ("none", "relu"):
        return 0.0
    x = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    k = 1.0 if act == "silu" else 1.6 * (1 + 3 * 0.044715 * z ** 2)
    q = torch.sigmoid(x)
    dq = 2.0 ** -16 * q * (1 - q) + 2.0 ** -22
    return dq * (1 + 2 * z.abs().clamp(max=64) * k) * (z.abs() < 64)


def close(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = err > tol
    assert not bad.any(), (what, int(bad.sum()), float((err - tol).max()),
                           bad.nonzero()[:4].tolist())


SHAPES = [
    (1, 1, 32), (1, 128, 64), (1, 256, 256), (1, 130, 4096), (2, 5120, 1024), (16, 384, 512),
    (17, 129, 288), (31, 257, 2048), (33, 1000, 96), (64, 128, 512), (65, 200, 1056),
    (100, 3000, 320), (128, 128, 256), (129, 255, 544), (200, 640, 1280), (257, 4096, 512),
    (511, 2050, 768), (300, 19200, 256), (2100, 2200, 288), (700, 2047, 224), (130, 9000, 64),
    (90, 300, 4096), (128, 2000, 1024), (300, 310, 8192), (127, 6401, 480), (65, 9400, 1280),
    (66, 9500, 1280), (129, 6400, 1312),
]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(nvlib, m, n, k):
    a, b, z, tol = problem(m, n, k, m * 7 + n + k)
    d, aux = nvlib.matmul_nvfp4(*cuda(a), *cuda(b), out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert nvlib.device_error() == 0
    assert aux is None
    close(d, z, tol + orc.half_step(torch.float32) * z.abs(), "d")


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,k", [(3, 200, 1024), (50, 129, 96), (140, 333, 512),
                                   (2304, 2200, 64), (900, 1501, 96), (80, 400, 2048)])
def test_epilogue(nvlib, m, n, k, out, act):
    dtype, hs = TYPES[out], orc.half_step(TYPES[out])
    a, b, z, tol = problem(m, n, k, m + n)
    g = torch.Generator().manual_seed(k)
    bias = torch.randn(n, generator=g).to(dtype if act == "gelu" else torch.float32)
    res = torch.randn(m, n, generator=g).to(dtype)
    amax = torch.empty(1, device="cuda")
    d, aux = nvlib.matmul_nvfp4(*cuda(a), *cuda(b), bias=bias.cuda(), residual=res.cuda(),
                                activation=act, out_dtype=dtype, with_aux=True, amax_out=amax)
    z = z + bias.double()
    tol = tol + 2.0 ** -23 * (z.abs() + bias.double().abs())
    tol = tol + orc.least_step(dtype) / 2
    close(aux, z, tol + hs * z.abs(), "aux")
    own, lip = act_error(z, act)
    want = orc.act(z, act) + res.double()
    close(d, want, lip * tol + own + 2.0 ** -23 * (want.abs() + res.double().abs())
          + hs * want.abs() + orc.least_step(dtype) / 2, "d")
    assert float(amax) == float(d.float().abs().max())


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 130, 512), (40, 300, 2048), (333, 514, 256),
                                   (2500, 2177, 96), (1030, 1800, 64), (130, 200, 4096)])
def test_backward_epilogue(nvlib, m, n, k, out, act):
    dtype, hs = TYPES[out], orc.half_step(TYPES[out])
    a, b, z, tol = problem(m, n, k, m + 2 * n)
    aux = (torch.randn(m, n, generator=torch.Generator().manual_seed(k)) * 2).to(dtype)
    amax = torch.empty(1, device="cuda")
    d, dbias = nvlib.matmul_nvfp4_dact(*cuda(a), *cuda(b), aux.cuda(), activation=act,
                                       with_dbias=True, amax_out=amax)
    s = orc.act_slope(aux.double(), act)
    want = z * s
    tol = tol * s.abs() + z.abs() * slope_error(aux.double(), act) + 2.0 ** -22 * want.abs()
    close(d, want, tol + hs * want.abs() + orc.least_step(dtype) / 2, "d")
    steps = m / 64 + 40
    close(dbias, want.sum(0), tol.sum(0) + steps * 2.0 ** -24 * want.abs().sum(0), "dbias")
    assert float(amax) == float(d.float().abs().max())


def test_matches_the_casts(nvlib):
    """Operands written by the library's own row-wise cast: the product of what
    the codes stand for."""
    m, n, k = 96, 160, 512
    g = torch.Generator(device="cuda").manual_seed(1)
    ops = []
    for rows, seed in ((m, 1), (n, 2)):
        x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
        amax = torch.empty(1, device="cuda")
        nvlib.amax_bf16(x, rows * k, amax)
        bits = torch.randint(-2**31, 2**31, (rows * k // 16, 4), device="cuda", generator=g,
                             dtype=torch.int64).to(torch.int32)
        c = torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda")
        s = torch.empty(rows, k // 16, dtype=torch.uint8, device="cuda")
        nvlib.quantize_rowwise_bf16_sr(rows, k, x, amax, bits, c, s)
        ops.append((c, s, amax))
    d, _ = nvlib.matmul_nvfp4(*ops[0], *ops[1], out_dtype=torch.float32)
    va, vb = (orc.operand_values(*(t.cpu() for t in o)) for o in ops)
    z, size = va @ vb.t(), va.abs() @ vb.abs().t()
    close(d, z, (k / 64 + 8) * 2.0 ** -22 * size + 2.0 ** -21 * z.abs(), "d")


def test_weight_gradient_of_the_rht_casts(nvlib):
    """dW = dy^T x from two transposed RHT casts: the Hadamard transforms cancel
    in the product, up to the casts' own rounding (codes decoded here)."""
    tokens, fo, fi = 256, 128, 256
    g = torch.Generator(device="cuda").manual_seed(3)
    B = nvlib.hadamard16(torch.tensor([1.0, -1.0] * 8))
    ops = []
    for f in (fo, fi):
        x = torch.randn(tokens, f, device="cuda", generator=g).to(torch.bfloat16)
        amax = torch.empty(1, device="cuda")
        nvlib.amax_bf16(x, x.numel(), amax)
        c, s = nvlib.quantize_rht(x, B, amax, torch.tensor([5, 0], device="cuda"))
        ops.append((c, s, amax))
    acc = torch.randn(fo, fi, device="cuda", generator=g)
    before = acc.clone()
    d, _ = nvlib.matmul_nvfp4(*ops[0], *ops[1], residual=acc, out=acc)
    assert d.data_ptr() == acc.data_ptr()
    va, vb = (orc.operand_values(*(t.cpu() for t in o)) for o in ops)
    z, size = va @ vb.t(), va.abs() @ vb.abs().t()
    want = z + before.double().cpu()
    close(d, want, (tokens / 64 + 8) * 2.0 ** -22 * size + 2.0 ** -21 * (z.abs() + want.abs()),
          "d")


@pytest.mark.parametrize("m", [5, 200, 2200])
def test_strides_and_borders(nvlib, m):
    """Rows of D, residual and aux with wider strides: what lies between the
    rows and behind the last one stays as it was."""
    n, k = 2190 if m == 2200 else 150, 160
    a, b, z, tol = problem(m, n, k, 11)
    buf = torch.full((m + 2, n + 10), 77.0, dtype=torch.float32, device="cuda")
    out = buf[1:m + 1, 3:n + 3]
    res = torch.randn(m, n + 6, device="cuda")[:, :n]
    d, _ = nvlib.matmul_nvfp4(*cuda(a), *cuda(b), residual=res, out=out)
    want = z + res.double().cpu()
    close(d, want, tol + 2.0 ** -22 * (want.abs() + z.abs()), "d")
    out.fill_(77.0)
    assert bool((buf == 77.0).all())


@pytest.mark.parametrize("k", [32, 64, 96, 160, 256, 288, 320, 4096])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_scale_alignment(nvlib, k, shift):
    """Scales at any byte address and of any row length."""
    m, n = 20, 140
    a, b, z, tol = problem(m, n, k, k + shift)
    moved = []
    for c, s, am in (a, b):
        raw = torch.empty(s.numel() + shift, dtype=torch.uint8, device="cuda")
        t = raw[shift:].view(s.shape)
        t.copy_(s)
        moved += [c.cuda(), t, am.cuda()]
    d, _ = nvlib.matmul_nvfp4(*moved, out_dtype=torch.float32)
    close(d, z, tol + 2.0 ** -24 * z.abs(), "d")


def test_long_m(nvlib):
    """More blocks of 128 rows than a grid's second dimension holds (65535)."""
    base, times, n, k = 1000, 8389, 8, 32
    a, b, z, tol = problem(base, n, k, 17)
    rows = [t.cuda().repeat(times, 1) for t in a[:2]]
    d, _ = nvlib.matmul_nvfp4(*rows, a[2].cuda(), *cuda(b), out_dtype=torch.float32)
    d = d.view(times, base, n)
    for edge in (d.amin(0), d.amax(0)):
        close(edge, z, tol + 2.0 ** -24 * z.abs(), "d")


def test_special_values(nvlib):
    """Zero operands, a zero amax, NaN scales and infinite residuals end where
    they belong."""
    m, n, k = 33, 150, 512
    a, b, z, tol = problem(m, n, k, 5)
    # amax = 0: encode scale 1 (the cast's convention)
    d, _ = nvlib.matmul_nvfp4(a[0].cuda(), a[1].cuda(), torch.zeros(1, device="cuda"), *cuda(b),
                              out_dtype=torch.float32)
    va = orc.operand_values(a[0], a[1], 0.0)
    vb = orc.operand_values(*b)
    w, size = va @ vb.t(), va.abs() @ vb.abs().t()
    close(d, w, (k / 64 + 8) * 2.0 ** -22 * size + 2.0 ** -21 * w.abs(), "amax 0")
    # a NaN scale poisons its row alone; an infinity in the residual its element
    sa = a[1].clone()
    sa[7, 3] = 0x7F
    res = torch.zeros(m, n)
    res[2, 9], res[3, 9] = math.inf, math.nan
    amax = torch.empty(1, device="cuda")
    d, _ = nvlib.matmul_nvfp4(a[0].cuda(), sa.cuda(), a[2].cuda(), *cuda(b),
                              residual=res.cuda(), out_dtype=torch.float32, amax_out=amax)
    d = d.cpu()
    assert bool(torch.isnan(d[7]).all()) and math.isinf(float(d[2, 9])) and math.isnan(float(d[3, 9]))
    keep = torch.isfinite(d)
    assert int((~keep).sum()) == n + 2
    close(d[keep], z[keep], tol[keep] + 2.0 ** -23 * z[keep].abs(), "others")
    assert math.isnan(float(amax))
    # zero codes: exactly the bias
    bias = torch.randn(n, device="cuda")
    zero = torch.zeros_like(a[0]).cuda()
    d, _ = nvlib.matmul_nvfp4(zero, a[1].cuda(), a[2].cuda(), *cuda(b), bias=bias,
                              out_dtype=torch.float32)
    assert torch.equal(d, bias.expand(m, n))


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n", [(5, 40), (900, 1600), (900, 1601)])
def test_amax_of_odd_values(nvlib, m, n, out):
    """The amax of a lone negative maximum, of an infinity and of a NaN, whatever
    its sign and wherever it stands."""
    a, b, z, tol = problem(m, n, 64, 3)
    zero, amax = torch.zeros_like(a[0]).cuda(), torch.empty(1, device="cuda")
    for at in (0, 3, m * n - 1):
        for value in (-8.0, math.inf, -math.inf, math.nan, -math.nan):
            res = torch.full((m, n), 0.5, dtype=TYPES[out], device="cuda")
            res.view(-1)[at] = value
            nvlib.matmul_nvfp4(zero, a[1].cuda(), a[2].cuda(), *cuda(b), residual=res,
                               out_dtype=TYPES[out], amax_out=amax)
            got = float(amax)
            assert math.isnan(got) if math.isnan(value) else got == abs(value), (at, value, got)


def test_huge_activation_arguments(nvlib):
    """Arguments whose powers overflow: slopes of 0 or 1, no NaN."""
    m, n, k = 4, 130, 64
    a, b, z, tol = problem(m, n, k, 9)
    for act in ("gelu", "silu"):
        aux = torch.full((m, n), 1e30)
        aux[::2] = -1e30
        d, _ = nvlib.matmul_nvfp4_dact(*cuda(a), *cuda(b), aux.cuda(), activation=act)
        want = torch.where(aux > 0, z, torch.zeros_like(z))
        close(d, want, tol + 2.0 ** -22 * z.abs(), act)


def test_empty(nvlib):
    """No rows or no columns: nothing but the amax and the bias gradient."""
    a, b, _, _ = problem(4, 8, 64, 1)
    amax = torch.full((1,), 5.0, device="cuda")
    e = [t[:0].contiguous().cuda() for t in a[:2]] + [a[2].cuda()]
    d, _ = nvlib.matmul_nvfp4(*e, *cuda(b), amax_out=amax)
    assert d.shape == (0, 8) and float(amax) == 0.0
    d, dbias = nvlib.matmul_nvfp4_dact(*e, *cuda(b),
                                       torch.empty(0, 8, dtype=torch.bfloat16, device="cuda"),
                                       activation="gelu", with_dbias=True)
    assert d.shape == (0, 8) and torch.equal(dbias, torch.zeros(8, device="cuda"))
    e = [t[:0].contiguous().cuda() for t in b[:2]] + [b[2].cuda()]
    d, _ = nvlib.matmul_nvfp4(*cuda(a), *e)
    assert d.shape == (4, 0)


@pytest.mark.parametrize("m,n,k", [(3, 700, 4096), (700, 300, 256), (2400, 2304, 512)])
def test_repeats_and_sm_cap(nvlib, m, n, k):
    """The same bits on every call, on another stream and two calls at once; with
    a capped grid the same D, and a bias gradient added in another order; a
    captured call replays on new inputs."""
    a, b, _, _ = problem(m, n, k, 21)
    a, b = cuda(a), cuda(b)
    aux = torch.randn(m, n, device="cuda").to(torch.bfloat16)
    want, wb = nvlib.matmul_nvfp4_dact(*a, *b, aux, activation="gelu", with_dbias=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [nvlib.matmul_nvfp4_dact(*a, *b, aux, activation="gelu", with_dbias=True)
                    for _ in range(3)]
    torch.cuda.synchronize()
    for d, db in got:
        assert torch.equal(d, want) and torch.equal(db, wb)
    d = torch.empty_like(want)
    nb = nvlib.gemm_nvfp4_dact_workspace_bytes(m, n, k)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    db = torch.empty_like(wb)
    nvlib.gemm_nvfp4_dact(m, n, k, *a, *b, aux, n, "gelu", d, n, d.dtype, db, None, ws, nb,
                          sm_count=5)
    assert torch.equal(d, want)
    # fewer CTAs give a tile another accumulator, whose columns are taken in the
    # other direction: m additions of fp32 values either way
    close(db, wb.double().cpu(), (m + 40) * 2.0 ** -23 * want.double().abs().sum(0).cpu(), "dbias, capped grid")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gd, gb = nvlib.matmul_nvfp4_dact(*a, *b, aux, activation="gelu", with_dbias=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gd, want) and torch.equal(gb, wb)
    aux.neg_()
    new, nb2 = nvlib.matmul_nvfp4_dact(*a, *b, aux, activation="gelu", with_dbias=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gd, new) and torch.equal(gb, nb2)
    assert nvlib.device_error() == 0


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,n,k", [(1, 130, 512), (40, 300, 2048), (333, 514, 256),
                                   (2500, 2177, 96), (1030, 1800, 64), (130, 200, 4096)])
def test_backward_epilogue_in_f16(nvlib, m, n, k, act):
    test_backward_epilogue(nvlib, m, n, k, "f16", act)


@pytest.mark.parametrize("m", [5, 200, 2200])
def test_matrices_side_by_side(nvlib, m):
    """D, residual and aux in the same rows of one buffer are no overlap; a shifted
    residual is one, and refused."""
    n, k = 2192 if m == 2200 else 160, 160
    a, b, z, tol = problem(m, n, k, 13)
    buf = torch.randn(m, 3 * n, device="cuda")
    d, res, other = buf[:, :n], buf[:, n:2 * n], buf[:, 2 * n:].clone()
    before = res.double().cpu()
    nvlib.matmul_nvfp4(*cuda(a), *cuda(b), residual=res, out=d)
    want = z + before
    close(d, want, tol + 2.0 ** -22 * (want.abs() + z.abs()), "d")
    assert torch.equal(res.double().cpu(), before) and torch.equal(buf[:, 2 * n:], other)
    for shifted in (buf[:, 1:n + 1], buf[:, n - 1:2 * n - 1]):
        with pytest.raises(nvlib.NVFP4Error):
            nvlib.matmul_nvfp4(*cuda(a), *cuda(b), residual=shifted, out=d)
