"""The operators together, as a training step uses them: one NVFP4 MLP block
  h = norm(x);  u = gelu(h W1^T + b1);  y = u W2^T + b2 + x
forward, backward and the AdamW step on its parameters, with the casts between
them; and the tensor-level argument checks that need a device.

The step's numbers are checked stage by stage against 64 bits from the very
operands each stage read (the casts round stochastically to 4 bits, so only
then is there a tight tolerance), the chain of amax words against the tensors
they stand for, and the weights' gradients against the exact gradient of the
unquantized block by their direction.  A product with the casts' 4-bit codes
keeps most of a gradient: quantization noise of relative size e leaves a cosine
of 1 / sqrt(1 + e^2).  Here a gradient is a product of two cast operands, each
off by at most a quarter (E2M1's largest relative spacing is 1/2 with
stochastic rounding, its mean square below 1/16 where values are of their
block's size, of which every operand's norm mostly consists): e^2 < 4/16 over
the chain's four casts, so the cosine stays above 0.89; 0.8 is asked."""
import math

import pytest
import torch

from tests import training_oracle as orc

pytestmark = pytest.mark.gpu

T, H, F = 256, 256, 512          # tokens, hidden, inner


class Caster:
    """The casts of one step: row-wise along the last dimension, or transposed (RHT)."""

    def __init__(self, nv):
        self.nv, self.g = nv, torch.Generator(device="cuda").manual_seed(5)
        self.B = nv.hadamard16(torch.tensor([1.0, -1.0, -1.0, 1.0] * 4))
        self.calls = 0

    def rows(self, x, amax):
        r, c = x.shape
        bits = torch.randint(-2**31, 2**31, (r * c // 16, 4), device="cuda", generator=self.g,
                             dtype=torch.int64).to(torch.int32)
        q = torch.empty(r, c // 2, dtype=torch.uint8, device="cuda")
        s = torch.empty(r, c // 16, dtype=torch.uint8, device="cuda")
        self.nv.quantize_rowwise_bf16_sr(r, c, x, amax, bits, q, s)
        return q, s, amax

    def columns(self, x, amax):
        self.calls += 1
        rng = torch.tensor([17, self.calls], device="cuda")
        q, s = self.nv.quantize_rht(x, self.B, amax, rng)
        return q, s, amax


def word():
    return torch.empty(1, device="cuda")


def product(a, b):
    return (orc.operand_values(*(t.cpu() for t in a))
            @ orc.operand_values(*(t.cpu() for t in b)).t())


def near(got, want, rel):
    got = got.double().cpu()
    assert float((got - want).norm()) <= rel * float(want.norm())


def test_mlp_block_step(nvlib):
    nv = nvlib
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = rnd(T, H).to(torch.bfloat16)
    dy = rnd(T, H).to(torch.bfloat16)
    masters = [1 + 0.1 * rnd(H), 0.1 * rnd(H), rnd(F, H) / math.sqrt(H), 0.1 * rnd(F),
               rnd(H, F) / math.sqrt(F), 0.1 * rnd(H)]
    start = [p.clone() for p in masters]
    copies = [p.to(torch.bfloat16) for p in masters]
    gamma, beta, _, b1, _, b2 = masters
    w1, w2 = copies[2], copies[4]
    amax_w = torch.empty(6, device="cuda")
    for i, c in enumerate(copies):
        amax_w[i] = c.float().abs().max()
    cast = Caster(nv)

    # forward
    a_h, a_u = word(), word()
    h, mean, rstd = nv.layernorm(x, gamma, beta, amax_out=a_h)
    assert float(a_h) == float(h.float().abs().max())
    qh, qw1 = cast.rows(h, a_h), cast.rows(w1, amax_w[2:3])
    u, z = nv.matmul_nvfp4(*qh, *qw1, bias=b1, activation="gelu", with_aux=True, amax_out=a_u)
    assert float(a_u) == float(u.float().abs().max())
    wz = product(qh, qw1) + b1.double().cpu()
    near(z, wz, 2.0 ** -8)
    near(u, orc.act(wz, "gelu"), 2.0 ** -7)
    qu, qw2 = cast.rows(u, a_u), cast.rows(w2, amax_w[4:5])
    y, _ = nv.matmul_nvfp4(*qu, *qw2, bias=b2, residual=x)
    near(y, product(qu, qw2) + b2.double().cpu() + x.double().cpu(), 2.0 ** -8)

    # backward
    a_dy, a_dz = word(), word()
    nv.amax_bf16(dy, dy.numel(), a_dy)
    qdy, qw2t = cast.rows(dy, a_dy), cast.rows(w2.t().contiguous(), amax_w[4:5])
    dz, db1 = nv.matmul_nvfp4_dact(*qdy, *qw2t, z, activation="gelu", with_dbias=True,
                                   amax_out=a_dz)
    wdz = product(qdy, qw2t) * orc.act_slope(z.double().cpu(), "gelu")
    near(dz, wdz, 2.0 ** -8)
    near(db1, wdz.sum(0), 2.0 ** -15)
    assert float(a_dz) == float(dz.float().abs().max())
    dw2 = torch.zeros(H, F, device="cuda")
    cdy, cu = cast.columns(dy, a_dy), cast.columns(u, a_u)
    nv.matmul_nvfp4(*cdy, *cu, residual=dw2, out=dw2)
    near(dw2, product(cdy, cu), 2.0 ** -16)
    dw1 = torch.zeros(F, H, device="cuda")
    cdz, ch = cast.columns(dz, a_dz), cast.columns(h, a_h)
    nv.matmul_nvfp4(*cdz, *ch, residual=dw1, out=dw1)
    near(dw1, product(cdz, ch), 2.0 ** -16)
    qdz, qw1t = cast.rows(dz, a_dz), cast.rows(w1.t().contiguous(), amax_w[2:3])
    dh, _ = nv.matmul_nvfp4(*qdz, *qw1t)
    dx, dgamma, dbeta = nv.layernorm_backward(dh, x, mean, rstd, gamma, residual=dy)
    wdx, wdg, wdb = orc.layernorm_backward(dh.cpu(), x.cpu(), mean.cpu(), rstd.cpu(), gamma.cpu(),
                                           dy.cpu())
    near(dx, wdx, 2.0 ** -8)
    near(dgamma, wdg, 2.0 ** -15)
    near(dbeta, wdb, 2.0 ** -15)
    db2 = dy.float().sum(0)

    # the exact gradient of the block without casts
    leaf = [t.double().cpu().requires_grad_() for t in (x, gamma, beta, w1, b1, w2, b2)]
    lx, lg, lb, lw1, lb1, lw2, lb2 = leaf
    m = lx.mean(1, keepdim=True)
    lh = (lx - m) / torch.sqrt(((lx - m) ** 2).mean(1, keepdim=True) + 1e-5) * lg + lb
    out = orc.act(lh @ lw1.t() + lb1, "gelu") @ lw2.t() + lb2 + lx
    (out * dy.double().cpu()).sum().backward()
    for got, l in zip((dx, dgamma, dbeta, dw1, db1, dw2, db2), leaf):
        a, b = got.double().cpu().flatten(), l.grad.flatten()
        assert float(a @ b / (a.norm() * b.norm())) > 0.8

    # the step: both state forms move the same parameters, and the amax words
    # are those of the new copies
    grads = [dgamma, dbeta, dw1, db1, dw2, db2]
    sizes = [p.numel() for p in masters]
    rng = torch.tensor([3, 0], device="cuda")
    u8 = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")  # noqa: E731
    for eight in (False, True):
        for p, s in zip(masters, start):
            p.copy_(s)
        kw = {}
        if eight:
            kw = dict(exp_avg_scales=[u8(-(-n // 128)) for n in sizes],
                      exp_avg_sq_scales=[u8(-(-n // 128)) for n in sizes], rng_state=rng)
        new = (lambda n: u8(n)) if eight else (lambda n: torch.zeros(n, device="cuda"))
        opt = nv.AdamW(masters, grads, [new(n) for n in sizes], [new(n) for n in sizes],
                       copies=copies, weight_decays=[0, 0, 0.1, 0, 0.1, 0], amax_out=amax_w, **kw)
        opt.step(1, lr=1e-3)
        for i, (p, s) in enumerate(zip(masters, start)):
            assert torch.equal(copies[i], p.to(torch.bfloat16))
            assert float(amax_w[i]) == float(copies[i].float().abs().max())
            zero = torch.zeros(p.shape)
            want, _, _ = orc.adamw(s.cpu(), grads[i].cpu(), zero, zero, lr=1e-3, beta1=0.9,
                                   beta2=0.95, eps=1e-8, step=1, wd=(0, 0, 0.1, 0, 0.1, 0)[i])
            near(p, want, 2.0 ** -21)
        # the next step's cast reads copy and word as they are
        q = cast.rows(copies[2], amax_w[2:3])
        assert q[0].shape == (F, H // 2)
    torch.cuda.synchronize()
    assert nv.device_error() == 0


def test_tensor_level_checks(nvlib):
    nv = nvlib
    dev = dict(device="cuda")
    c = torch.zeros(4, 32, dtype=torch.uint8, **dev)
    s = torch.zeros(4, 4, dtype=torch.uint8, **dev)
    am = torch.ones(1, **dev)
    ok = (c, s, am)
    for bad in ((c[:, :24], s, am), (c.float(), s, am), (c, s[:, :3], am), (c, s, am.double()),
                (c, s.cpu(), am), (c[:, ::2], s, am), (c[0], s, am)):
        with pytest.raises(ValueError):
            nv.matmul_nvfp4(*bad, *ok)
        with pytest.raises(ValueError):
            nv.matmul_nvfp4(*ok, *bad)
    f = torch.zeros(4, 4, **dev)
    for kw in (dict(bias=torch.zeros(5, **dev)), dict(residual=f), dict(activation="tanh"),
               dict(out_dtype=torch.float64), dict(out=f.t()[:, :3]), dict(amax_out=f),
               dict(residual=f.cpu()), dict(out=torch.zeros(4, 8, **dev)[:, ::2])):
        with pytest.raises(ValueError):
            nv.matmul_nvfp4(*ok, *ok, **kw)
    with pytest.raises(ValueError):
        nv.matmul_nvfp4_dact(*ok, *ok, f[:3], activation="gelu")
    x, w = torch.zeros(4, 8, **dev), torch.ones(8, **dev)
    for args in ((x[0], w), (x.double(), w), (x, w[:7]), (x, w.to(torch.bfloat16)),
                 (x.t(), torch.ones(4, **dev)), (x, w.cpu())):
        with pytest.raises(ValueError):
            nv.layernorm(*args)
    with pytest.raises(ValueError):
        nv.layernorm(x, w, w.to(torch.float16))
    st = torch.zeros(4, **dev)
    for args in ((x[:3], x, st, st, w), (x, x, st[:3], st, w), (x, x, st, st.double(), w),
                 (x.to(torch.bfloat16), x, st, st, w)):
        with pytest.raises(ValueError):
            nv.layernorm_backward(*args)
    p = torch.zeros(200, **dev)
    u, b = torch.zeros(200, dtype=torch.uint8, **dev), torch.zeros(2, dtype=torch.uint8, **dev)
    rng = torch.tensor([1, 0], **dev)
    for kw in (dict(exp_avgs=[p[:100]]), dict(grads=[p.double()]), dict(grads=[p, p]),
               dict(copies=[p]), dict(exp_avgs=[u], exp_avg_sqs=[u]),
               dict(exp_avgs=[u], exp_avg_sqs=[u], exp_avg_scales=[b[:1]], exp_avg_sq_scales=[b],
                    rng_state=rng),
               dict(amax_out=torch.zeros(2, **dev)), dict(params=[p.half()]),
               dict(params=[p[::2]], grads=[p[:100]], exp_avgs=[p[:100]], exp_avg_sqs=[p[:100]])):
        a = dict(params=[p], grads=[p], exp_avgs=[p], exp_avg_sqs=[p])
        a.update(kw)
        with pytest.raises(ValueError):
            nv.AdamW(a.pop("params"), a.pop("grads"), a.pop("exp_avgs"), a.pop("exp_avg_sqs"), **a)
    q = torch.zeros(200, **dev)
    opt = nv.AdamW([p], [q], [q.clone()], [q.clone()])
    with pytest.raises(nv.NVFP4Error):
        opt.step(0, lr=0.1)
    with pytest.raises(ValueError):
        opt.step(1, lr=0.1, scalars=p)
    with pytest.raises(ValueError):
        nv.adamw_unpack_state(u, b[:1], "exp_avg")
