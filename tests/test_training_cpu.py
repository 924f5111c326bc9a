"""Refusals of the operators around the cast: argument checks that run before
any CUDA call (placeholder pointers, never used), and the tensor-level checks
that need no device."""
import ctypes

import pytest
import torch

OK, SHAPE, ARG, ALIGN = 0, 1, 2, 3
P = 4096        # an aligned placeholder address


def gemm(lib, m=4, n=8, k=64, A=P, SFA=P, aa=P, B=P, SFB=P, ab=P, D=P, ldd=None, out=1, bias=None,
         bt=0, res=None, ldr=None, act=0, aux=None, ldaux=None, amax=None, ws=None, nb=0):
    return lib.nvfp4_gemm(m, n, k, A, SFA, aa, B, SFB, ab, D, n if ldd is None else ldd, out, bias,
                          bt, res, n if ldr is None else ldr, act, aux,
                          n if ldaux is None else ldaux, amax, ws, nb, 0, None)


@pytest.mark.parametrize("kw,want", [
    (dict(k=48), SHAPE), (dict(k=16), SHAPE), (dict(k=0), SHAPE), (dict(m=-1), SHAPE),
    (dict(n=-8), SHAPE), (dict(ldd=7), SHAPE), (dict(res=P, ldr=7), SHAPE),
    (dict(aux=P, ldaux=7), SHAPE), (dict(m=2**31), SHAPE), (dict(k=2**31), SHAPE),
    (dict(m=2**30, n=2**30, k=32), SHAPE),
    (dict(A=None), ARG), (dict(SFA=None), ARG), (dict(aa=None), ARG), (dict(B=None), ARG),
    (dict(SFB=None), ARG), (dict(ab=None), ARG), (dict(D=None), ARG), (dict(out=3), ARG),
    (dict(out=-1), ARG), (dict(bias=P, bt=5), ARG), (dict(act=4), ARG), (dict(act=-1), ARG),
    (dict(A=P + 8), ALIGN), (dict(B=P + 8), ALIGN), (dict(D=P + 1), ALIGN),
    (dict(D=P + 2, out=0), ALIGN), (dict(res=P + 1), ALIGN), (dict(aux=P + 1), ALIGN),
    (dict(bias=P + 2), ALIGN), (dict(aa=P + 2), ALIGN), (dict(amax=P + 2), ALIGN),
    (dict(m=5000, n=512), ARG), (dict(m=5000, n=512, ws=P, nb=1024), ARG),
    (dict(m=5000, n=512, ws=P + 16, nb=1 << 20), ALIGN),
    (dict(m=0), OK), (dict(n=0), OK), (dict(m=0, A=None, D=None), OK),
])
def test_gemm_refuses(nvlib, kw, want):
    assert gemm(nvlib.load(), **kw) == want


def test_gemm_refuses_its_operands_amax_as_output(nvlib):
    """amax_out is cleared before the operands' amax are read."""
    assert gemm(nvlib.load(), amax=P, ab=P + 4) == ARG
    assert gemm(nvlib.load(), amax=P, aa=P + 4) == ARG


def test_gemm_dact_refuses(nvlib):
    lib = nvlib.load()

    def call(aux=P, ldaux=8, act=2, dbias=None, ws=None, nbytes=0, m=4, n=8, k=64, amax=None):
        return lib.nvfp4_gemm_dact(m, n, k, P, P, P, P, P, P, aux, ldaux, act, P, n, 1, dbias,
                                   amax, ws, nbytes, 0, None)
    need = lib.nvfp4_gemm_dact_workspace_bytes(4, 8, 64)
    assert need >= 8 * 4
    assert call(aux=None) == ARG
    assert call(ldaux=7) == SHAPE
    assert call(act=9) == ARG
    assert call(dbias=P) == ARG                                # no workspace
    assert call(dbias=P, ws=P, nbytes=need - 1) == ARG         # a short one
    assert call(dbias=P + 2, ws=P, nbytes=need) == ALIGN
    assert call(dbias=P, ws=P + 1, nbytes=need) == ALIGN
    assert lib.nvfp4_gemm_dact_workspace_bytes(0, 8, 64) == 0


def test_layernorm_refuses(nvlib):
    lib = nvlib.load()

    def fwd(rows=4, cols=8, x=P, ldx=8, gamma=P, beta=P, dt=1, wt=0, eps=1e-5, y=P, ldy=8, mean=P,
            rstd=P, amax=None):
        return lib.nvfp4_layernorm_fwd(rows, cols, x, ldx, gamma, beta, dt, wt, eps, y, ldy, mean,
                                       rstd, amax, None)
    assert fwd(rows=-1) == SHAPE and fwd(cols=-1) == SHAPE and fwd(cols=2**25, ldx=2**25,
                                                                    ldy=2**25) == SHAPE
    assert fwd(ldx=7) == SHAPE and fwd(ldy=7) == SHAPE
    assert fwd(x=None) == ARG and fwd(gamma=None) == ARG and fwd(y=None) == ARG
    assert fwd(dt=3) == ARG and fwd(dt=1, wt=2) == ARG and fwd(dt=0, wt=1) == ARG
    assert fwd(eps=-1.0) == ARG and fwd(eps=float("nan")) == ARG
    assert fwd(x=P + 1) == ALIGN and fwd(gamma=P + 2) == ALIGN and fwd(mean=P + 2) == ALIGN
    assert fwd(rows=0) == OK and fwd(cols=0) == OK

    need = lib.nvfp4_layernorm_bwd_workspace_bytes(4, 8)

    def bwd(rows=4, cols=8, dy=P, lddy=8, x=P, ldx=8, mean=P, rstd=P, gamma=P, res=None, ldr=8,
            dt=1, wt=0, dx=P, lddx=8, dg=P, db=P, ws=P, nb=need):
        return lib.nvfp4_layernorm_bwd(rows, cols, dy, lddy, x, ldx, mean, rstd, gamma, res, ldr,
                                       dt, wt, dx, lddx, dg, db, ws, nb, None)
    for kw in (dict(rows=-1), dict(lddy=7), dict(ldx=7), dict(lddx=7), dict(res=P, ldr=7)):
        assert bwd(**kw) == SHAPE, kw
    for kw in (dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(gamma=None),
               dict(dx=None), dict(ws=None), dict(nb=need - 1), dict(dt=7), dict(wt=2)):
        assert bwd(**kw) == ARG, kw
    for kw in (dict(dy=P + 1), dict(res=P + 1), dict(dg=P + 2), dict(ws=P + 2)):
        assert bwd(**kw) == ALIGN, kw
    assert bwd(cols=0) == OK


def test_adamw_refuses(nvlib):
    from fp4_sm120a_b200._native import AdamWTensor
    lib = nvlib.load()

    def step(count=1, pt=0, gt=0, st=0, lr=0.1, b1=0.9, b2=0.95, eps=1e-8, t=1, scale=None,
             scalars=None, amax=None, rng=None, table=True, **fields):
        base = dict(param=P, grad=P, exp_avg=P, exp_avg_sq=P, exp_avg_scale=None,
                    exp_avg_sq_scale=None, copy=None, n=10, offset=0, weight_decay=0.0)
        base.update(fields)
        arr = (AdamWTensor * 1)(AdamWTensor(**base))
        return lib.nvfp4_adamw_step(arr if table else None, count, pt, gt, st, lr, b1, b2, eps, t,
                                    scale, scalars, amax, rng, None)
    assert step(count=0) == OK and step(count=-1) == SHAPE and step(table=False) == ARG
    nan = float("nan")
    for kw in (dict(pt=2), dict(pt=-1), dict(gt=3), dict(st=2), dict(b1=1.0), dict(b1=-0.1),
               dict(b2=1.0), dict(b2=nan), dict(eps=-1.0), dict(eps=nan), dict(t=0), dict(lr=nan),
               dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None),
               dict(weight_decay=nan), dict(pt=1, copy=P),
               dict(st=1), dict(st=1, rng=P),
               dict(st=1, rng=P, exp_avg_scale=P, exp_avg_sq_scale=P, offset=64)):
        assert step(**kw) == ARG, kw
    for kw in (dict(param=P + 2), dict(grad=P + 2), dict(exp_avg=P + 1), dict(exp_avg_sq=P + 2),
               dict(copy=P + 1), dict(amax=P + 1), dict(scale=P + 2), dict(scalars=P + 2),
               dict(rng=P + 4)):
        assert step(**kw) == ALIGN, kw
    assert step(n=2**43) == SHAPE

    def unpack(codes=P, scales=P, n=4, moment=0, out=P, dt=0):
        return lib.nvfp4_adamw_unpack_state(codes, scales, n, moment, out, dt, None)
    assert unpack(n=0) == OK and unpack(moment=2) == ARG and unpack(dt=2) == ARG
    assert unpack(codes=None) == ARG and unpack(scales=None) == ARG and unpack(out=None) == ARG
    assert unpack(out=P + 2) == ALIGN


def test_descriptor_layout(nvlib):
    """The ctypes mirror has the C struct's layout (8 bytes a field)."""
    from fp4_sm120a_b200._native import AdamWTensor
    assert ctypes.sizeof(AdamWTensor) == 80
    assert AdamWTensor.n.offset == 56 and AdamWTensor.weight_decay.offset == 72


def test_tensor_level_refuses_host_tensors(nvlib):
    x, w = torch.zeros(2, 32), torch.ones(32)
    with pytest.raises(ValueError):
        nvlib.layernorm(x, w)
    with pytest.raises(ValueError):
        nvlib.matmul_nvfp4(x, x, x, x, x, x)
    with pytest.raises(ValueError):
        nvlib.adamw_unpack_state(torch.zeros(4, dtype=torch.uint8), torch.zeros(1), "exp_avg")
    with pytest.raises(ValueError):
        nvlib.AdamW([w], [w], [w], [w])
    with pytest.raises(ValueError):
        nvlib.AdamW([], [], [], [])


def test_unknown_names(nvlib):
    from fp4_sm120a_b200 import ops
    with pytest.raises(ValueError):
        ops.gemm_nvfp4(1, 1, 32, None, None, None, None, None, None, None, 1, torch.float32, None,
                       torch.float32, None, 1, "tanh", None, 1, None, None, 0, stream=0)
    with pytest.raises(ValueError):
        ops.adamw_unpack_state(None, None, 0, "momentum", None, torch.float32, stream=0)


def test_workspaces_follow_the_sizes(nvlib):
    lib = nvlib.load()
    plain, dact = lib.nvfp4_gemm_workspace_bytes, lib.nvfp4_gemm_dact_workspace_bytes
    for m in (1, 16, 17, 64, 65, 128, 129, 4099, 100000):
        for n in (1, 128, 5120):
            for k in (32, 4096):
                a, b = plain(m, n, k), dact(m, n, k)
                assert a % 256 == 0 and b % 256 == 0
                # two partial rows at least; scales: 8 bytes for 128 codes, in
                # whole blocks of 128 rows x 256 codes
                assert b - a >= 2 * 4 * n
                assert a in (0, (-(-m // 128) + -(-n // 128)) * -(-k // 256) * 2048)
    assert plain(64, 5120, 4096) == 0 and plain(128, 512, 4096) == 0
    assert plain(0, 8, 64) == dact(4, 0, 64) == 0
    assert lib.nvfp4_layernorm_bwd_workspace_bytes(10, 7) == 10 * 2 * 7 * 4
    assert lib.nvfp4_layernorm_bwd_workspace_bytes(10**6, 7) == 4 * 296 * 2 * 7 * 4
    assert lib.nvfp4_layernorm_bwd_workspace_bytes(10**6, 5120) == 296 * 2 * 5120 * 4


def test_binding_shares_the_process_libstdcxx(nvlib):
    """A second copy of the C++ runtime would crash on the first error message."""
    from fp4_sm120a_b200._native import load_binding
    x = torch.zeros(2, 32)
    with pytest.raises(TypeError, match="expected 5 arguments, got 1"):
        load_binding().layernorm(x)
    with pytest.raises(ValueError):
        load_binding().layernorm(3, x, None, 1e-5, None)
    with pytest.raises(ValueError):
        load_binding().matmul(*[x] * 6, None, None, 0, 1, None, False, None)


@pytest.mark.parametrize("rng", [torch.zeros(4, dtype=torch.int64)[::2],
                                 torch.zeros(1, dtype=torch.int64).expand(2)])
def test_adamw_refuses_a_strided_rng_state(nvlib, rng):
    """The kernel reads {seed, offset} as adjacent words."""
    w, u = torch.ones(32), torch.zeros(32, dtype=torch.uint8)
    s = torch.zeros(1, dtype=torch.uint8)
    with pytest.raises(ValueError, match="rng_state"):
        nvlib.AdamW([w], [w], [u], [u], exp_avg_scales=[s], exp_avg_sq_scales=[s], rng_state=rng)


def adamw_lists():
    z = lambda n=200, t=torch.float32: [torch.zeros(n, dtype=t) for _ in range(2)]  # noqa: E731
    return dict(params=z(), grads=z(), exp_avgs=z(t=torch.uint8), exp_avg_sqs=z(t=torch.uint8),
                exp_avg_scales=z(2, torch.uint8), exp_avg_sq_scales=z(2, torch.uint8),
                copies=z(t=torch.bfloat16), amax_out=torch.zeros(2),
                rng_state=torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("name", ["params", "exp_avgs", "exp_avg_sqs", "exp_avg_scales",
                                  "exp_avg_sq_scales", "copies"])
@pytest.mark.parametrize("how", ["twice", "views", "bytes"])
def test_adamw_refuses_lists_that_overlap(nvlib, name, how):
    """Two blocks would write the same memory at once."""
    a = adamw_lists()
    n, t = a[name][0].numel(), a[name][0].dtype
    flat = torch.zeros(2 * n, dtype=t)
    if how == "twice":
        a[name] = [flat[:n]] * 2
    elif how == "views":
        a[name] = [flat[:n], flat[n - 1:2 * n - 1]]
    else:                                     # one list's memory in another list
        other = "exp_avgs" if name != "exp_avgs" else "copies"
        raw = torch.zeros(max(n, 200) * 4, dtype=torch.uint8)
        a[name] = [raw[:n * t.itemsize].view(t), flat[:n]]
        u = a[other][0]
        a[other] = [raw[:200 * u.dtype.itemsize].view(u.dtype), a[other][1]]
    lists = [a.pop(k) for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")]
    with pytest.raises(ValueError, match="overlap|twice"):
        nvlib.AdamW(*lists, **a)


@pytest.mark.parametrize("name", ["grads", "rng_state", "amax_out"])
def test_adamw_refuses_what_it_reads_in_what_it_writes(nvlib, name):
    a = adamw_lists()
    if name == "grads":
        a["grads"] = a["params"]
    elif name == "rng_state":
        raw = torch.zeros(200, dtype=torch.uint8)
        a["exp_avgs"], a["rng_state"] = [raw, a["exp_avgs"][1]], raw[8:24].view(torch.int64)
    else:
        a["amax_out"] = a["params"][1][4:6]
    lists = [a.pop(k) for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")]
    with pytest.raises(ValueError, match="overlap"):
        nvlib.AdamW(*lists, **a)


def test_adamw_lists_side_by_side_are_no_overlap(nvlib):
    """What is left to refuse is the device."""
    a = adamw_lists()
    flat = torch.zeros(400)
    a["params"] = [flat[:200], flat[200:]]
    a["exp_avgs"][0] = a["exp_avgs"][0][:0]
    a["params"][0] = a["params"][0][:0]
    for k in ("grads", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales", "copies"):
        a[k][0] = a[k][0][:0]
    lists = [a.pop(k) for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")]
    with pytest.raises(ValueError, match="CUDA"):
        nvlib.AdamW(*lists, **a)


def test_adamw_step_refuses_scalars_in_its_amax(nvlib):
    """amax_out is cleared before grad_scale and scalars are read."""
    from fp4_sm120a_b200._native import AdamWTensor
    lib = nvlib.load()
    arr = (AdamWTensor * 3)(*[AdamWTensor(param=P, grad=P, exp_avg=P, exp_avg_sq=P, n=0)] * 3)

    def step(scale=None, scalars=None):
        return lib.nvfp4_adamw_step(arr, 3, 0, 0, 0, 0.1, 0.9, 0.95, 1e-8, 1, scale, scalars, P,
                                    None, None)
    for word in (P, P + 8):
        assert step(scale=word) == ARG
    for words in (P - 8, P, P + 8):
        assert step(scalars=words) == ARG


@pytest.mark.parametrize("offsets", [[0, -128], [0, 200], [-2**63, 0], [0, 2**63]])
def test_adamw_refuses_offsets_that_are_no_places(nvlib, offsets):
    """Random bits are numbered from 0 on, in blocks of 128."""
    a = adamw_lists()
    lists = [a.pop(k) for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")]
    with pytest.raises(ValueError, match="offsets"):
        nvlib.AdamW(*lists, offsets=offsets, **a)


@pytest.mark.parametrize("at,ldr", [(2, 64), (-2, 64), (128, 64), (62, 64), (66, 64), (0, 32),
                                    (3 * 128 + 62, 32), (-2, 2**62)])
def test_outputs_partly_over_their_inputs_are_refused(nvlib, at, ldr):
    """4 x 32 values, rows 64 apart: an input may be the output itself, or lie beside
    it in the same rows, but not shifted under it (rows read after others were written)."""
    lib, R, far = nvlib.load(), 1 << 20, 1 << 30
    over = R + at

    def bwd(dy=far, lddy=32, res=None, ldr=32):
        return lib.nvfp4_layernorm_bwd(4, 32, dy, lddy, 2 * far, 32, P, P, P, res, ldr, 1, 0, R, 64,
                                       P, P, P, 1 << 20, None)
    assert gemm(lib, m=4, n=32, D=R, ldd=64, res=over, ldr=ldr) == ARG
    assert gemm(lib, m=4, n=32, D=R, ldd=64, aux=over, ldaux=ldr) == ARG
    assert lib.nvfp4_gemm_dact(4, 32, 64, P, P, P, P, P, P, over, ldr, 2, R, 64, 1, None, None,
                               None, 0, 0, None) == ARG
    assert lib.nvfp4_layernorm_fwd(4, 32, over, ldr, P, P, 1, 0, 1e-5, R, 64, None, None, None,
                                   None) == ARG
    assert bwd(dy=over, lddy=ldr) == ARG and bwd(res=over, ldr=ldr) == ARG


def test_two_outputs_in_one_place_are_refused(nvlib):
    assert gemm(nvlib.load(), aux=P) == ARG
