"""AdamW against 64 bits, and its 8-bit moments bit for bit.

Tolerances of the 32-bit form: each moment is two products and a sum, each
rounded (3 steps of 2^-24 of its TERMS |beta1 m| + |(1 - beta1) g|, which may
cancel in m).  p's update passes m's error on, magnified by lr / (bias
correction * denominator), and adds a root, a quotient and two products (2^-20
of the update).  The decayed p has the factor's rounding, the product's and the
final sum's: 3 steps of 2^-24 of |p| and one of the result."""
import math

import pytest
import torch

from tests import training_oracle as orc

pytestmark = pytest.mark.gpu

H = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def close(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((err - tol).max()))


def make(sizes, param, grad, seed):
    g = torch.Generator().manual_seed(seed)
    ps = [(torch.randn(n, generator=g) * 0.05).to(param) for n in sizes]
    gs = [(torch.randn(n, generator=g) * 0.01).to(grad) for n in sizes]
    ms = [torch.randn(n, generator=g) * 0.003 for n in sizes]
    vs = [(torch.randn(n, generator=g) * 0.01) ** 2 for n in sizes]
    return ps, gs, ms, vs


def check_param(p, p0, g, m0, v, step, want, copies, amax, i):
    terms = H["beta1"] * m0.double().abs() + (1 - H["beta1"]) * g.double().abs()
    gain = H["lr"] / (1 - H["beta1"] ** step) / (
        torch.sqrt(v / (1 - H["beta2"] ** step)) + H["eps"])
    tol = (gain * terms * (3 * 2.0 ** -24 + 2.0 ** -20)
           + 2.0 ** -24 * (3 * p0.double().abs() + want.abs()))
    if p.dtype == torch.bfloat16:
        tol = tol + orc.half_step(torch.bfloat16) * want.abs() * (1 + 2.0 ** -8)
    close(p, want, tol, f"p[{i}]")
    if copies is not None:
        assert torch.equal(copies[i], p.to(torch.bfloat16))
    if amax is not None:
        top = p.to(torch.bfloat16).float().abs().max() if p.numel() else torch.zeros(())
        assert float(amax[i]) == float(top)


SIZES = [[1], [5, 3, 1000], [4096], [4097, 0, 129, 8192, 127, 128], [33] * 70, [300] * 800]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("param,grad", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"),
                                        ("bf16", "bf16"), ("bf16", "f32")])
def test_32_bit(nvlib, sizes, param, grad):
    ps, gs, ms, vs = make(sizes, TYPES[param], TYPES[grad], len(sizes))
    dp, dg, dm, dv = ([t.cuda() for t in x] for x in (ps, gs, ms, vs))
    copies = ([torch.empty(n, dtype=torch.bfloat16, device="cuda") for n in sizes]
              if param == "f32" else None)
    amax = torch.full((len(sizes),), 9.0, device="cuda")
    wds = [0.1 * (i % 3) for i in range(len(sizes))]
    scale = torch.tensor([0.5], device="cuda")
    opt = nvlib.AdamW(dp, dg, dm, dv, copies=copies, weight_decays=wds, amax_out=amax)
    opt.step(7, grad_scale=scale, **H)
    for i in range(len(sizes)):
        p, m, v = orc.adamw(ps[i], gs[i], ms[i], vs[i], step=7, wd=wds[i], grad_scale=0.5, **H)
        g = gs[i].double() * 0.5
        close(dm[i], m, 3 * 2.0 ** -24 * (0.9 * ms[i].double().abs() + 0.1 * g.abs()), "m")
        close(dv[i], v, 4 * 2.0 ** -24 * v, "v")
        check_param(dp[i], ps[i], g, ms[i], v, 7, p, copies, amax, i)


def zeros8(sizes):
    blocks = [-(-n // 128) for n in sizes]
    return ([torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes],
            [torch.zeros(b, dtype=torch.uint8, device="cuda") for b in blocks])


def f32(x):
    return x.to(torch.float32)


def expect8(x, moment, words):
    """Codes and scale bytes of fp32 values, step by step as the format says."""
    n = x.numel()
    drop, levels = (20, 8) if moment == "exp_avg" else (19, 16)
    pad = -(-n // 128) * 128 - n
    bits = torch.cat([x, torch.zeros(pad)]).abs().view(torch.int32).view(-1, 128)
    top = bits.amax(1) >> 23
    scale = torch.where(top == 255, top, (top - 7).clamp_min(1))
    inv = ((254 - scale).clamp_min(0) << 23).view(torch.float32)
    y = torch.cat([x, torch.zeros(pad)]).abs().view(-1, 128) * inv[:, None]
    low = y < 2.0 ** -6
    r = torch.cat([words, torch.zeros(pad, dtype=torch.int32)]).view(-1, 128)
    t = torch.where(low, y + 2.0 ** -6, y).view(torch.int32) + (r << (drop - 16))
    code = (t >> drop) - ((120 + low.int()) << (23 - drop))
    code = torch.where(scale[:, None] == 255, torch.zeros_like(code), code).view(-1)[:n]
    if moment == "exp_avg":
        code = code | ((x < 0).int() << 7)
    else:
        finite = (scale != 255).repeat_interleave(128)[:n]
        code = torch.where((x > 0) & finite, code.clamp_min(1), code)
    return code.to(torch.uint8), scale.to(torch.uint8)


def moment_words(n, offset, seed, counter):
    lo, hi = torch.empty(n, dtype=torch.int32), torch.empty(n, dtype=torch.int32)
    for i in range(0, n, 4):
        w = orc.philox(seed, counter, (offset + i) // 4)
        for k in range(min(4, n - i)):
            lo[i + k], hi[i + k] = w[k] & 0xFFFF, w[k] >> 16
    return lo, hi


@pytest.mark.parametrize("sizes", [[1], [128], [4, 300, 127, 4096 + 37], [513] * 40])
@pytest.mark.parametrize("grad", ["f32", "bf16"])
def test_8_bit(nvlib, sizes, grad):
    """Three steps from zero states: codes and scales bit for bit, parameters
    against 64 bits from the decoded states."""
    ps, _, _, _ = make(sizes, torch.float32, TYPES[grad], 3)
    dp = [p.cuda() for p in ps]
    (dm, ms), (dv, vs) = zeros8(sizes), zeros8(sizes)
    dg = [torch.zeros(n, dtype=TYPES[grad], device="cuda") for n in sizes]
    seed, off = 0x123456789ABCDEF, 0xFFFFFFFE
    rng = torch.tensor([seed, off], device="cuda")
    amax = torch.empty(len(sizes), device="cuda")
    opt = nvlib.AdamW(dp, dg, dm, dv, exp_avg_scales=ms, exp_avg_sq_scales=vs, amax_out=amax,
                      rng_state=rng)
    offsets = [0]
    for n in sizes:
        offsets.append(offsets[-1] + -(-n // 128) * 128)
    for step in (1, 2, 3):
        gs = make(sizes, torch.float32, TYPES[grad], 100 + step)[1]
        if sizes[-1] > 200:
            gs[-1][7] = 30.0        # an outlier pushes its block into the lowest binade
        for d, g in zip(dg, gs):
            d.copy_(g)
        before = [(p.cpu(), orc.unpack8(m.cpu(), s.cpu(), "exp_avg"),
                   orc.unpack8(v.cpu(), t.cpu(), "exp_avg_sq"))
                  for p, m, s, v, t in zip(dp, dm, ms, dv, vs)]
        opt.step(step, **H)
        torch.cuda.synchronize()
        for i, n in enumerate(sizes):
            p0, m0, v0 = before[i]
            g = f32(gs[i])
            m = f32(m0) * torch.tensor(0.9) + g * torch.tensor(1 - 0.9)
            v = f32(v0) * torch.tensor(0.95) + (g * g) * torch.tensor(1 - 0.95)
            lo, hi = moment_words(n, offsets[i], seed, off + step)
            code, scale = expect8(m, "exp_avg", lo)
            assert torch.equal(ms[i].cpu(), scale) and torch.equal(dm[i].cpu(), code), (step, i)
            code, scale = expect8(v, "exp_avg_sq", hi)
            assert torch.equal(vs[i].cpu(), scale) and torch.equal(dv[i].cpu(), code), (step, i)
            want, _, wv = orc.adamw(p0, g, m0, v0, step=step, wd=0.0, **H)
            check_param(dp[i], p0, g, m0, wv, step, want, None, amax, i)


def test_8_bit_shards_repeat_the_whole(nvlib):
    """A tensor in two pieces with their offsets: the bits of the whole."""
    n, cut = 5000, 2048
    ps, gs, _, _ = make([n], torch.float32, torch.float32, 9)
    rng = torch.tensor([11, 5], device="cuda")
    out = []
    for pieces in ([slice(0, n)], [slice(0, cut), slice(cut, n)]):
        p, g = ps[0].cuda(), gs[0].cuda()
        (m,), (ms,) = zeros8([n])
        (v,), (vs,) = zeros8([n])

        def cutb(t):
            return [t[s.start // 128:-(-s.stop // 128)] for s in pieces]

        def cute(t):
            return [t[s] for s in pieces]
        opt = nvlib.AdamW(cute(p), cute(g), cute(m), cute(v), exp_avg_scales=cutb(ms),
                          exp_avg_sq_scales=cutb(vs), offsets=[s.start for s in pieces],
                          rng_state=rng)
        for step in (1, 2):
            opt.step(step, **H)
        out.append((p, m, v, ms, vs))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_8_bit_special_values(nvlib):
    """A value that is not finite marks its block; a second moment above zero
    stays above zero; zero gradients from zero states change nothing but the decay."""
    n = 384
    p = torch.ones(n, device="cuda")
    g = torch.zeros(n, device="cuda")
    g[5] = math.inf
    g[128] = 1.0
    g[129] = 1e-12            # far below its block's lowest step
    (m,), (ms,) = zeros8([n])
    (v,), (vs,) = zeros8([n])
    amax = torch.empty(1, device="cuda")
    opt = nvlib.AdamW([p], [g], [m], [v], exp_avg_scales=[ms], exp_avg_sq_scales=[vs],
                      rng_state=torch.tensor([1, 2], device="cuda"), amax_out=amax,
                      weight_decays=[0.5])
    opt.step(1, **H)
    um, uv = (nvlib.adamw_unpack_state(c, s, k).cpu() for c, s, k in
              ((m, ms, "exp_avg"), (v, vs, "exp_avg_sq")))
    assert bool(torch.isnan(um[:128]).all()) and bool(torch.isnan(uv[:128]).all())
    assert bool(torch.isfinite(um[128:]).all()) and bool(torch.isfinite(uv[128:]).all())
    assert float(uv[129]) > 0 and bool((uv[256:] == 0).all()) and bool((um[256:] == 0).all())
    pc = p.cpu()
    assert math.isnan(float(pc[5])) and math.isnan(float(amax))
    assert bool((pc[256:] == float(torch.tensor(1.0) * torch.tensor(1 - 0.01 * 0.5))).all())


@pytest.mark.parametrize("moment", ["exp_avg", "exp_avg_sq"])
@pytest.mark.parametrize("n,shift", [(1, 0), (128, 0), (256 * 3 + 5, 0), (1000, 1)])
def test_unpack(nvlib, moment, n, shift):
    """All codes under scales from the smallest to the largest."""
    raw = (torch.arange(n + shift) * 37 % 256).to(torch.uint8)
    if moment == "exp_avg":
        raw[(raw & 127) == 127] = 0        # E4M3's NaN code is never written
    codes = raw.cuda()[shift:]
    blocks = -(-n // 128)
    scales = torch.tensor([1, 120, 127, 255, 0, 121, 3, 60] * blocks, dtype=torch.uint8)[:blocks]
    want = orc.unpack8(codes.cpu(), scales, moment)
    got = nvlib.adamw_unpack_state(codes, scales.cuda(), moment, torch.float32).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    b16 = nvlib.adamw_unpack_state(codes, scales.cuda(), moment).double().cpu()
    assert torch.equal(b16.nan_to_num(), got.float().to(torch.bfloat16).double().nan_to_num())


def test_stochastic_rounding_is_unbiased(nvlib):
    """Mean over many draws of one second moment between two codes: within 5
    standard deviations of its value."""
    n = 128 * 512
    g = torch.full((n,), math.sqrt(1.37), device="cuda")
    p = torch.zeros(n, device="cuda")
    (m,), (ms,) = zeros8([n])
    (v,), (vs,) = zeros8([n])
    opt = nvlib.AdamW([p], [g], [m], [v], exp_avg_scales=[ms], exp_avg_sq_scales=[vs],
                      rng_state=torch.tensor([77, 0], device="cuda"))
    opt.step(1, **H)
    u = nvlib.adamw_unpack_state(v, vs, "exp_avg_sq", torch.float32).double()
    want = float(torch.tensor(0.05) * (g[0].cpu() * g[0].cpu()))
    values = u.unique()
    assert values.numel() == 2 and float(values[0]) < want < float(values[1])
    sd = float(values[1] - values[0]) / 2 / math.sqrt(n)
    assert abs(float(u.mean()) - want) < 5 * sd + 2.0 ** -16 * float(values[1] - values[0])


def test_unaligned_views_and_neighbours(nvlib):
    """Tensors at odd places of flat buffers; what lies around them stays."""
    cuts = [(1, 200), (203, 777), (1001, 64)]
    flat = {k: torch.full((1100,), 2.5, device="cuda") for k in "pgmv"}
    copies = torch.full((1100,), 2.5, dtype=torch.bfloat16, device="cuda")
    ps, gs, ms, vs = make([n for _, n in cuts], torch.float32, torch.float32, 12)
    for k, seq in zip("pgmv", (ps, gs, ms, vs)):
        for (a, n), t in zip(cuts, seq):
            flat[k][a:a + n] = t.cuda()
    view = lambda t: [t[a:a + n] for a, n in cuts]  # noqa: E731
    opt = nvlib.AdamW(view(flat["p"]), view(flat["g"]), view(flat["m"]), view(flat["v"]),
                      copies=view(copies))
    opt.step(3, **H)
    for i, (a, n) in enumerate(cuts):
        p, m, v = orc.adamw(ps[i], gs[i], ms[i], vs[i], step=3, wd=0.0, **H)
        check_param(flat["p"][a:a + n], ps[i], gs[i], ms[i], v, 3, p, view(copies), None, i)
    mask = torch.ones(1100, dtype=torch.bool, device="cuda")
    for a, n in cuts:
        mask[a:a + n] = False
    for t in [*flat.values(), copies]:
        assert bool((t[mask] == 2.5).all())


@pytest.mark.parametrize("eight", [False, True])
def test_captured_step_takes_its_scalars_from_the_device(nvlib, eight):
    """A captured step replayed with new scalars, gradients and rng_state gives
    the bits of eager steps with the same."""
    sizes = [1000, 260]
    ps, _, ms, vs = make(sizes, torch.float32, torch.float32, 4)

    def build():
        p, g = [t.cuda() for t in ps], [torch.empty(n, device="cuda") for n in sizes]
        rng = torch.tensor([3, 0], device="cuda")
        if eight:
            (m, a), (v, b) = zeros8(sizes), zeros8(sizes)
            opt = nvlib.AdamW(p, g, m, v, exp_avg_scales=a, exp_avg_sq_scales=b, rng_state=rng,
                              weight_decays=[0.1, 0.0])
        else:
            m, v = [t.cuda() for t in ms], [t.cuda() for t in vs]
            opt = nvlib.AdamW(p, g, m, v, weight_decays=[0.1, 0.0])
        return opt, p, g, m, v, rng, torch.empty(3, device="cuda")
    runs = [build(), build()]
    graph = torch.cuda.CUDAGraph()
    opt, _, _, _, _, _, sc = runs[1]
    with torch.cuda.graph(graph):
        opt.step(0, lr=0.0, beta1=0.9, beta2=0.95, eps=1e-8, scalars=sc)
    for step in (1, 2, 3):
        gs = make(sizes, torch.float32, torch.float32, 50 + step)[1]
        lr = 0.01 / step
        for which, (opt, p, g, m, v, rng, sc) in enumerate(runs):
            for d, t in zip(g, gs):
                d.copy_(t)
            sc.copy_(torch.tensor([lr, 1 - 0.9 ** step, 1 - 0.95 ** step]))
            rng[1] = step
            if which:
                graph.replay()
            else:
                opt.step(0, lr=0.0, beta1=0.9, beta2=0.95, eps=1e-8, scalars=sc)
        torch.cuda.synchronize()
        for a, b in zip(runs[0][1:5], runs[1][1:5]):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    # and the device scalars mean what lr and step mean
    opt, p, g, m, v, rng, _ = build()
    for step in (1, 2, 3):
        gs = make(sizes, torch.float32, torch.float32, 50 + step)[1]
        for d, t in zip(g, gs):
            d.copy_(t)
        rng[1] = 0                         # the counter is offset + step
        opt.step(step, lr=0.01 / step, beta1=0.9, beta2=0.95, eps=1e-8)
    for x, y in zip(p, runs[0][1]):
        close(x, y.double().cpu(), 2.0 ** -18 * 0.03 + 2.0 ** -22 * x.abs().cpu(), "scalars")


def test_first_step_by_differences(nvlib):
    """From zero states the first update is lr sign(g) for gradients far above eps."""
    g = torch.tensor([3.0, -0.25, 1e-3, -2e4], device="cuda")
    p = torch.zeros(4, device="cuda")
    opt = nvlib.AdamW([p], [g], [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")])
    opt.step(1, lr=0.5, beta1=0.9, beta2=0.95, eps=1e-12)
    close(p, -0.5 * g.sign().double().cpu(), torch.full((4,), 0.5 * 2.0 ** -20), "p")


def test_refuses_a_tensor_twice(nvlib):
    """Tied weights are one parameter: two blocks would update it at once."""
    p, g, m, v = ([torch.zeros(8, device="cuda") for _ in range(2)] for _ in range(4))
    nvlib.AdamW(p, g, m, v)
    with pytest.raises(ValueError):
        nvlib.AdamW([p[0], p[0]], g, m, v)


def listed(nvlib, sizes=(300, 70), seed=21, **kw):
    """An optimizer with 32-bit moments, copies and amax, and its lists."""
    cpu = make(list(sizes), torch.float32, torch.float32, seed)
    lists = [[t.cuda() for t in x] for x in cpu]
    lists.append([torch.empty(n, dtype=torch.bfloat16, device="cuda") for n in sizes])
    amax = torch.empty(len(sizes), device="cuda")
    return nvlib.AdamW(*lists[:4], copies=lists[4], amax_out=amax, **kw), lists, amax


@pytest.mark.parametrize("which", range(6))
def test_a_tensor_with_other_memory_is_refused(nvlib, which):
    """p.data = ..., set_ and resize_ leave the tensor and take its memory away."""
    opt, lists, amax = listed(nvlib)
    t = (lists + [[amax]])[which][-1]
    opt.step(1, **H)
    keep = [x.clone() for seq in lists for x in seq]
    for change in (lambda: t.data.clone(), lambda: t.data[:t.numel() - 1],
                   lambda: torch.zeros(2 * t.numel(), dtype=t.dtype, device="cuda")[::2]):
        old = t.data
        t.data = change()
        with pytest.raises(ValueError):
            opt.step(2, **H)
        t.data = old
    n = t.numel()
    t.resize_(5 * n + 4096)
    with pytest.raises(ValueError):
        opt.step(2, **H)
    torch.cuda.synchronize()
    if which < 5:
        now = [x.flatten()[:y.numel()] for x, y in zip((x for seq in lists for x in seq), keep)]
        assert all(torch.equal(x, y) for x, y in zip(now, keep))


def test_two_steps_with_new_gradients(nvlib):
    """Gradients that are new tensors every step give the bits of an optimizer
    that was made for them; refused ones leave it as it was."""
    sizes = [300, 70, 0, 4097]
    opt, lists, amax = listed(nvlib, sizes)
    same = [[t.clone() for t in seq] for seq in lists]
    for step in (1, 2, 3):
        gs = [t.cuda() for t in make(sizes, torch.float32, torch.float32, 60 + step)[1]]
        opt.step(step, grads=gs, **H)
        nvlib.AdamW(same[0], gs, same[2], same[3], copies=same[4]).step(step, **H)
        for bad in (gs[:3], [*gs[:3], gs[3].half()], [*gs[:3], gs[3][:-1]], [*gs[:3], gs[3].cpu()],
                    [*gs[:3], torch.zeros(2 * 4097, device="cuda")[::2]], [*gs[:3], None]):
            with pytest.raises(ValueError):
                opt.step(step, grads=bad, **H)
        for k in (0, 2, 3, 4):
            assert all(torch.equal(x, y) for x, y in zip(lists[k], same[k])), (step, k)
    # without new ones the last are read again
    opt.step(4, **H)
    nvlib.AdamW(same[0], gs, same[2], same[3], copies=same[4]).step(4, **H)
    assert all(torch.equal(x, y) for x, y in zip(lists[0], same[0]))


def test_the_usual_loop_does_not_read_old_gradients(nvlib):
    """backward() after zero_grad(set_to_none=True) makes new .grad tensors."""
    ps = [torch.randn(n, device="cuda").requires_grad_() for n in (40, 7)]
    for p in ps:
        (p * p).sum().backward()
    zeros = [[torch.zeros(p.numel(), device="cuda") for p in ps] for _ in range(2)]
    opt = nvlib.AdamW(ps, [p.grad for p in ps], *zeros)
    opt.step(1, **H)
    for p in ps:
        p.grad = None
    with pytest.raises(ValueError, match="grad"):
        opt.step(2, **H)
    for p in ps:
        (3 * p).sum().backward()
    with pytest.raises(ValueError, match="grad"):
        opt.step(2, **H)
    before = [m.double().cpu() for m in zeros[0]]
    opt.step(2, grads=[p.grad for p in ps], **H)
    for m, m0 in zip(zeros[0], before):
        want = 0.9 * m0 + 0.1 * 3.0
        close(m, want, 4 * 2.0 ** -24 * (0.9 * m0.abs() + 0.3), "m")
    opt.step(3, **H)


def test_refuses_scalars_and_gradients_in_what_it_writes(nvlib):
    """amax_out is cleared, and parameters change, before they would be read."""
    opt, lists, amax = listed(nvlib)
    for kw in (dict(grad_scale=amax[1:]), dict(scalars=lists[0][0][5:8]), dict(grads=lists[2]),
               dict(grads=[lists[1][0], lists[0][0][:70]])):
        with pytest.raises(ValueError, match="overlap"):
            opt.step(1, **H, **kw)
    opt.step(1, **H)


@pytest.mark.parametrize("moment", ["exp_avg", "exp_avg_sq"])
def test_8_bit_moments_at_the_top_of_fp32_stay_finite(nvlib, moment):
    """Values whose next code would stand for 2^128: 256 codes of the largest scale
    that a block gets take the code below it."""
    n = 512
    value = 3.39e38 if moment == "exp_avg" else math.sqrt(3.39e38)
    g = torch.full((n,), value, device="cuda")
    g[::3] *= -1
    p = torch.zeros(n, device="cuda")
    (m, ms), (v, vs) = zeros8([n]), zeros8([n])
    opt = nvlib.AdamW([p], [g], m, v, exp_avg_scales=ms, exp_avg_sq_scales=vs,
                      rng_state=torch.tensor([5, 0], device="cuda"))
    opt.step(1, lr=1e-3, beta1=0.0, beta2=0.0)
    codes, scales, largest = (m, ms, 240.0) if moment == "exp_avg" else (v, vs, 248.0)
    got = nvlib.adamw_unpack_state(codes[0], scales[0], moment, torch.float32)
    sign = g.sign() if moment == "exp_avg" else torch.ones_like(g)
    assert bool((scales[0] == 247).all())
    assert torch.equal(got, sign * torch.tensor(largest * 2.0 ** 120, device="cuda"))
    # and the next step reads them: half of what was held, nothing new
    g.zero_()
    opt.step(2, lr=1e-3, beta1=0.5, beta2=0.5)
    again = nvlib.adamw_unpack_state(codes[0], scales[0], moment, torch.float32)
    assert torch.equal(again, got / 2)


@pytest.mark.parametrize("moment", ["exp_avg", "exp_avg_sq"])
@pytest.mark.parametrize("shift", [0, 1])
def test_unpack_large_scales(nvlib, moment, shift):
    """All codes under scales up to the largest finite one; a value above fp32's
    range is infinite."""
    tops = torch.tensor([126, 128, 200, 238, 239, 240, 246, 247, 248, 254], dtype=torch.uint8)
    scales = tops.repeat_interleave(2)
    raw = (torch.arange(scales.numel() * 128 + shift) % 256).to(torch.uint8)
    if moment == "exp_avg":
        raw[(raw & 127) == 127] = 0
    codes = raw.cuda()[shift:]
    want = orc.unpack8(codes.cpu(), scales, moment).float()
    got = nvlib.adamw_unpack_state(codes, scales.cuda(), moment, torch.float32).cpu()
    assert torch.equal(got, want)
    b16 = nvlib.adamw_unpack_state(codes, scales.cuda(), moment).cpu()
    assert torch.equal(b16, want.to(torch.bfloat16))


@pytest.mark.parametrize("sizes", [[1], [4, 300, 127, 4096 + 37], [513] * 40])
@pytest.mark.parametrize("param,grad", [("bf16", "bf16"), ("bf16", "f16"), ("bf16", "f32"),
                                        ("f32", "f16")])
def test_8_bit_moments_of_all_types(nvlib, sizes, param, grad):
    """The same as in fp32: two steps, codes and scales bit for bit."""
    ps = make(sizes, TYPES[param], TYPES[grad], 31)[0]
    dp, dg = [p.cuda() for p in ps], [torch.empty(n, dtype=TYPES[grad], device="cuda")
                                      for n in sizes]
    (dm, ms), (dv, vs) = zeros8(sizes), zeros8(sizes)
    copies = ([torch.empty(n, dtype=torch.bfloat16, device="cuda") for n in sizes]
              if param == "f32" else None)
    amax, rng = torch.empty(len(sizes), device="cuda"), torch.tensor([99, 7], device="cuda")
    wds = [0.1 * (i % 2) for i in range(len(sizes))]
    opt = nvlib.AdamW(dp, dg, dm, dv, exp_avg_scales=ms, exp_avg_sq_scales=vs, copies=copies,
                      amax_out=amax, rng_state=rng, weight_decays=wds)
    for step in (1, 2):
        gs = make(sizes, TYPES[param], TYPES[grad], 200 + step)[1]
        for d, g in zip(dg, gs):
            d.copy_(g)
        before = [(p.cpu(), orc.unpack8(m.cpu(), s.cpu(), "exp_avg"),
                   orc.unpack8(v.cpu(), t.cpu(), "exp_avg_sq"))
                  for p, m, s, v, t in zip(dp, dm, ms, dv, vs)]
        opt.step(step, **H)
        torch.cuda.synchronize()
        at = 0
        for i, n in enumerate(sizes):
            p0, m0, v0 = before[i]
            g = f32(gs[i])
            m = f32(m0) * torch.tensor(0.9) + g * torch.tensor(1 - 0.9)
            v = f32(v0) * torch.tensor(0.95) + (g * g) * torch.tensor(1 - 0.95)
            lo, hi = moment_words(n, at, 99, 7 + step)
            for x, words, kind, codes, scales in ((m, lo, "exp_avg", dm, ms),
                                                  (v, hi, "exp_avg_sq", dv, vs)):
                code, scale = expect8(x, kind, words)
                assert torch.equal(scales[i].cpu(), scale) and torch.equal(codes[i].cpu(), code)
            want, _, wv = orc.adamw(p0, g, m0, v0, step=step, wd=wds[i], **H)
            check_param(dp[i], p0, g, m0, wv, step, want, copies, amax, i)
            at += -(-n // 128) * 128


def test_two_threads_with_one_optimizer(nvlib):
    """Steps of two threads on one stream, each with its own new gradients: every step
    reads one thread's gradients whole (all ones or all twos; the first moment is
    then the same in every element), and none that were freed."""
    import threading
    sizes = [64] * 200
    ps = [torch.zeros(n, device="cuda") for n in sizes]
    ms, vs = ([torch.zeros(n, device="cuda") for n in sizes] for _ in range(2))
    opt = nvlib.AdamW(ps, [torch.zeros(n, device="cuda") for n in sizes], ms, vs)
    errors = []

    def work(value):
        try:
            for step in range(1, 40):
                opt.step(step, lr=0.0, beta1=0.0, beta2=0.0,
                         grads=[torch.full((n,), value, device="cuda") for n in sizes])
        except Exception as e:                # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(v,)) for v in (1.0, 2.0)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    m = torch.cat(ms)
    assert float(m[0]) in (1.0, 2.0) and bool((m == m[0]).all())
