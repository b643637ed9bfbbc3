"""GPU: dropout, linear_act and groupnorm_act (forward and gradients) against plain 64-bit forms."""
import importlib

import pytest
import torch

import _layers_ref as R

pytestmark = pytest.mark.gpu

ops = importlib.import_module("stable-diffusion_amd.ops")
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
dtypes = pytest.mark.parametrize("dt", list(DT))


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0, grad=False):
    g = torch.Generator().manual_seed(seed + 17 * len(shape) + sum(shape))
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda().requires_grad_(grad)


# ---- dropout --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1,), (1, 1), (1, 7), (3, 8), (2, 3, 77), (5, 333), (257, 64), (1000, 1), (2, 2, 9, 320)])
@pytest.mark.parametrize("p", [0.0, 2.0 ** -16, 0.1, 0.5, 1.0])
def test_mask_is_the_generators(shape, p):
    y = ops.dropout(torch.ones(shape, device="cuda"), p, 0x123456789ABCDEF0, 5)
    want = R.keep_scale(shape, p, 0x123456789ABCDEF0, 5)
    assert torch.equal(y.cpu(), want.float())


@dtypes
@pytest.mark.parametrize("rows,cols", [(1, 1), (4, 16), (33, 333), (130, 1280)])
@pytest.mark.parametrize("with_resid", [False, True])
def test_dropout_and_gradient(dt, rows, cols, with_resid):
    dt = DT[dt]
    x, dy = rand(rows, cols, dtype=dt, grad=True), rand(rows, cols, dtype=dt, seed=1)
    r = rand(rows, cols, dtype=dt, seed=2, grad=True) if with_resid else None
    y = ops.dropout(x, 0.3, 77, 9, resid=r)
    k = R.keep_scale((rows, cols), 0.3, 77, 9)
    ref = R.d(x) * k
    err = 2 * R.U * ref.abs()               # the scale's and the product's rounding
    if with_resid:
        err = err + R.U * (ref + R.d(r)).abs()
        ref = ref + R.d(r)
    R.check("y", y, ref, R.rounded(ref, err, dt))
    grads = torch.autograd.grad(y, [x] + ([r] if with_resid else []), dy)
    want = R.d(dy) * k
    R.check("dx", grads[0], want, R.rounded(want, 2 * R.U * want.abs(), dt))
    if with_resid:
        assert torch.equal(grads[1], dy)


def test_dropout_seed_tensor_strides_and_dropped_infinities():
    seed = torch.tensor([-5], dtype=torch.int64, device="cuda")
    x = rand(40, 50)
    a = ops.dropout(x, 0.5, seed, 1)
    assert torch.equal(a, ops.dropout(x, 0.5, -5, 1)) and torch.equal(a, ops.dropout(x, 0.5, (1 << 64) - 5, 1))
    assert not torch.equal(a, ops.dropout(x, 0.5, -5, 2)) and not torch.equal(a, ops.dropout(x, 0.5, -6, 1))
    wide = rand(40, 64)
    for v in (wide[:, 3:53], wide[::2, :50], wide.t()[:50]):              # rows apart, every other row, transposed
        assert torch.equal(ops.dropout(v, 0.5, 3), ops.dropout(v.contiguous(), 0.5, 3))
        assert torch.equal(ops.dropout(v, 0.5, 3, resid=v), ops.dropout(v.contiguous(), 0.5, 3, resid=v.contiguous()))
    one = rand(1, 50).expand(40, 50)                                       # row stride 0
    assert torch.equal(ops.dropout(one, 0.5, 3), ops.dropout(one.contiguous(), 0.5, 3))
    bad = torch.full((64, 64), float("inf"), device="cuda")
    bad[::2] = float("nan")
    y, k = ops.dropout(bad, 0.5, 11), R.keep_scale((64, 64), 0.5, 11, 0).cuda()
    assert (y[k == 0] == 0).all() and not torch.isfinite(y[k != 0]).any()


def test_dropout_numbers_rows_beyond_32_bit_products():
    """More than 2^31 eight-column groups: the rows' numbers keep counting."""
    rows = (1 << 31) + 4096
    x = torch.ones(rows, 1, dtype=torch.float16, device="cuda")
    y = ops.dropout(x, 0.5, 21, 3)
    for r0 in (0, 0x70000000 - 512, (1 << 31) - 512, rows - 1024):
        want = R.keep_scale((1024, 1), 0.5, 21, 3, row0=r0)
        assert torch.equal(y[r0:r0 + 1024].cpu(), want.half()), r0
    del x, y
    torch.cuda.empty_cache()


# ---- linear ---------------------------------------------------------------------------------------------------

LINEAR = [  # m, k, n, act, bias, resid, p
    (1, 16, 16, None, True, False, 0.0),
    (1, 1, 1, "silu", False, False, 0.0),
    (2, 320, 1280, "silu", True, False, 0.0),
    (3, 7, 5, "gelu", True, True, 0.4),
    (16, 1280, 1280, None, False, True, 0.2),
    (17, 1281, 64, "quick_gelu", True, False, 0.0),
    (65, 64, 333, None, True, True, 0.1),
    (64, 72, 136, "gelu", True, False, 0.0),
    (77, 768, 768, "quick_gelu", True, True, 0.1),
    (130, 33, 65, "silu", True, True, 0.0),
    (257, 192, 320, None, False, False, 0.5),
    (300, 2048, 64, "gelu", True, True, 0.1),
    (1000, 520, 264, "gelu", True, True, 0.1),
    (4096, 40, 24, None, True, False, 0.3),
    (31, 1000, 77, "gelu", True, True, 0.2),
    (9, 3, 1000, None, True, True, 0.5),
    (32, 4000, 17, "silu", False, True, 0.0),
    (2100, 320, 1288, "silu", True, False, 0.1),
]


def linear_case(m, k, n, act, bias, resid, p, dt, tag=""):
    dt = DT[dt]
    x, w = rand(m, k, dtype=dt, grad=True), rand(n, k, dtype=dt, seed=1, scale=k ** -0.5, grad=True)
    b = rand(n, seed=2, grad=True) if bias else None
    r = rand(m, n, dtype=dt, seed=3, grad=True) if resid else None
    dy = rand(m, n, dtype=dt, seed=4)
    y = ops.linear_act(x, w, b, act=act, resid=r, p=p, seed=99, offset=4)
    leaves = [t for t in (x, w, b, r) if t is not None]
    grads = list(torch.autograd.grad(y, leaves, dy))
    ref = R.linear_ref(x, w, b, r, dy, act, p, 99, 4, dt)
    R.check("y", y, *ref["y"])
    R.check("dx", grads.pop(0), *ref["dx"])
    R.check("dw", grads.pop(0), *ref["dw"])
    if bias:
        R.check("db", grads.pop(0), *ref["db"])
    if resid:
        assert torch.equal(grads.pop(0), dy)
    # without a graph: the same values
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, w, b, act=act, resid=r, p=p, seed=99, offset=4), y)


@dtypes
@pytest.mark.parametrize("case", LINEAR, ids=lambda c: "-".join(str(v) for v in c))
def test_linear_act_and_gradients(case, dt):
    linear_case(*case, dt)


@dtypes
def test_linear_act_long_sums(dt):
    linear_case(20000, 64, 40, "silu", True, False, 0.1, dt)       # the weight gradient's contraction is split
    linear_case(40, 9000, 48, None, True, True, 0.1, dt)           # the forward's


@dtypes
def test_linear_act_strides(dt):
    dt = DT[dt]
    xs, ws, rs = rand(50, 100, dtype=dt), rand(60, 100, dtype=dt, seed=1), rand(50, 90, dtype=dt, seed=2)
    for x, w, r in ((xs[:, 3:67], ws[:, 5:69], rs[:, 1:61]), (xs[::2, :64], ws[::3, 32:96], rs[::2, 8:28]),
                    (xs.t()[:64, :].t(), ws.t()[:64].t(), rs.t()[:60].t())):
        x, w, r = x.detach().requires_grad_(), w.detach().requires_grad_(), r.detach().requires_grad_()
        dy = rand(x.shape[0], w.shape[0] + 3, dtype=dt, seed=5)[:, 3:]
        y = ops.linear_act(x, w, act="gelu", resid=r, p=0.2, seed=1)
        g = torch.autograd.grad(y, [x, w, r], dy)
        c = [t.detach().contiguous().requires_grad_() for t in (x, w, r)]
        yc = ops.linear_act(c[0], c[1], act="gelu", resid=c[2], p=0.2, seed=1)
        gc = torch.autograd.grad(yc, c, dy.contiguous())
        ref = R.linear_ref(x, w, None, r, dy, "gelu", 0.2, 1, 0, dt)
        for name, got in (("y", y), ("y", yc), ("dx", g[0]), ("dx", gc[0]), ("dw", g[1]), ("dw", gc[1])):
            R.check(name, got, *ref[name])


def test_linear_act_leading_dimensions_partial_gradients_and_empty_batches():
    x, w, b = rand(2, 3, 5, 32, grad=True), rand(24, 32, seed=1, grad=True), rand(24, seed=2, grad=True)
    dy = rand(2, 3, 5, 24, seed=3)
    ref = R.linear_ref(x, w, b, None, dy.reshape(-1, 24), "silu", 0.3, 5, 0, torch.float32)
    for leaves, names in (([x], ["dx"]), ([w], ["dw"]), ([b], ["db"]), ([w, b], ["dw", "db"])):
        args = [t if any(t is l for l in leaves) else t.detach() for t in (x, w, b)]
        y = ops.linear_act(*args, act="silu", p=0.3, seed=5)
        R.check("y", y, *ref["y"])
        for name, g in zip(names, torch.autograd.grad(y, leaves, dy)):
            R.check(name, g, *ref[name])
    e = torch.empty(0, 4, 32, device="cuda", requires_grad=True)
    y = ops.linear_act(e, w, b, act="gelu", p=0.1, seed=1)
    assert tuple(y.shape) == (0, 4, 24)
    ge, gw, gb = torch.autograd.grad(y, [e, w, b], torch.empty_like(y))
    assert ge.shape == e.shape and not gw.any() and not gb.any()
    r = rand(2, 3, 5, 24, seed=6, grad=True)                                     # only the residual wants a gradient
    y = ops.linear_act(x.detach(), w.detach(), resid=r, act="gelu", p=0.5, seed=1)
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)
    y = ops.linear_act(x, w, p=0.0).sum()                                        # a broadcast gradient
    dx, = torch.autograd.grad(y, x)
    want = R.d(w).sum(0).expand(2, 3, 5, 32)
    R.check("dx of a sum", dx, want, R.rounded(want, 26 * R.U * R.d(w).abs().sum(0).expand_as(want), torch.float32))


@dtypes
@pytest.mark.parametrize("act", [None, "silu", "gelu", "quick_gelu"])
def test_activations_and_derivatives_over_their_range(act, dt):
    """One input, weight 1: z = x, through the whole range in which anything happens and far beyond."""
    dt = DT[dt]
    z = torch.cat([torch.linspace(-12, 12, 4001), torch.tensor([-6e4, -3e4, -1e3, -90.0, -0.0, 0.0, 90.0, 1e3, 3e4, 6e4])])
    x = z.to(dt).cuda().view(-1, 1).requires_grad_()
    w = torch.ones(1, 1, dtype=dt, device="cuda")
    y = ops.linear_act(x, w, act=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    zr = R.d(x)
    big = torch.maximum(torch.ones_like(zr), zr.abs()).clamp(max=100.0)          # beyond, the functions are 0 and z
    err = R.ACT_ERR * big + 4 * R.U * zr.abs() if act else torch.zeros_like(zr)
    ref, gref = R.act(zr, act), R.act_grad(zr, act)
    R.check("y", y, ref, R.rounded(ref, err, dt))
    R.check("dx", dx, gref, R.rounded(gref, R.ACT_ERR * big + 8 * R.U if act else 0 * big, dt) + R.half(dt) * gref.abs())


def test_infinite_and_nan_inputs_stay_where_they_are():
    x = rand(70, 24)
    x[3, 5], x[9, 0] = float("inf"), float("nan")
    w = rand(40, 24, seed=1)
    for act in (None, "silu", "gelu", "quick_gelu"):
        y = ops.linear_act(x, w, act=act)
        clean = torch.ones(70, dtype=torch.bool)
        clean[[3, 9]] = False
        assert torch.isfinite(y[clean.cuda()]).all() and torch.isnan(y[9]).all()
        z = x[3].cpu().double() @ w.cpu().double().t()
        assert torch.equal(torch.isposinf(y[3]).cpu(), torch.isposinf(z))
        if act is not None:
            assert (y[3].cpu()[torch.isneginf(z)] == 0).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("act", [None, "silu"])
def test_infinite_gradients_stay_infinite(act, dt):
    """An infinite entry of dy (or one that is infinite once scaled to the type) makes its row of dx and its column of
    dw infinite, as the formula has it, and nothing else."""
    dt = DT[dt]
    x, w = (1 + rand(5, 64).abs()).to(dt).requires_grad_(), (1 + rand(24, 64, seed=1).abs()).to(dt).requires_grad_()
    dy = rand(5, 24, seed=2).abs().to(dt)
    dy[3, 7] = float("inf")
    b = torch.zeros(24, device="cuda", requires_grad=True)
    dx, dw, db = torch.autograd.grad(ops.linear_act(x, w, b, act=act), (x, w, b), dy)
    assert torch.isposinf(dx[3]).all() and torch.isfinite(dx[[0, 1, 2, 4]]).all()
    assert torch.isposinf(dw[7]).all() and torch.isfinite(dw[:7]).all() and torch.isfinite(dw[8:]).all()
    assert torch.isposinf(db[7]) and torch.isfinite(db).sum() == 23


# ---- group norm -----------------------------------------------------------------------------------------------

GROUPNORM = [  # batch, spatial, c0, c1, groups, act, p
    (1, (1, 1), 32, 0, 32, "silu", 0.0),
    (1, (), 64, 0, 4, None, 0.0),
    (2, (8, 8), 1280, 0, 32, "silu", 0.1),
    (3, (7, 5), 96, 0, 32, "silu", 0.3),
    (2, (5, 3), 33, 0, 1, "gelu", 0.0),
    (2, (9,), 30, 0, 6, "quick_gelu", 0.2),
    (1, (16, 16), 320, 320, 32, "silu", 0.1),
    (2, (6, 7), 20, 12, 4, "silu", 0.1),
    (1, (13, 17), 7, 9, 2, None, 0.5),
    (2, (64, 64), 320, 0, 32, "silu", 0.1),
    (1, (64, 64), 640, 320, 32, "silu", 0.0),
    (1, (37, 53), 480, 0, 32, "silu", 0.0),
    (2, (100, 90), 33, 0, 11, "gelu", 0.2),
    (1, (50, 40), 2560, 0, 32, "silu", 0.1),
    (1, (40, 30), 1001, 1210, 33, "silu", 0.1),
    (1, (300, 301), 3, 0, 1, "silu", 0.0),
    (3, (30, 31), 300, 0, 300, None, 0.0),
    (1, (3, 2), 8192, 0, 1, "silu", 0.0),
]


@dtypes
@pytest.mark.parametrize("case", GROUPNORM, ids=lambda c: "-".join(str(v) for v in c))
def test_groupnorm_act_and_gradients(case, dt):
    b, sp, c0, c1, groups, act, p = case
    dt = DT[dt]
    c = c0 + c1
    x = (rand(b, *sp, c0) + rand(c0, seed=9)).to(dt).detach().requires_grad_()
    x1 = rand(b, *sp, c1, dtype=dt, seed=1, scale=2.0, grad=True) if c1 else None
    gamma, beta = (1 + rand(c, seed=2, scale=0.2)).requires_grad_(), rand(c, seed=3, scale=0.2, grad=True)
    dy = rand(b, *sp, c, dtype=dt, seed=4)
    y = ops.groupnorm_act(x, gamma, beta, 1e-5, act=act, x1=x1, groups=groups, p=p, seed=31, offset=2)
    leaves = [t for t in (x, x1, gamma, beta) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    ref = R.groupnorm_ref(x, x1, gamma, beta, dy, 1e-5, act, groups, p, 31, 2, dt)
    R.check("y", y, *ref["y"])
    names = ["dx"] + (["dx1"] if c1 else []) + ["dgamma", "dbeta"]
    for name, g in zip(names, grads):
        R.check(name, g, *ref[name])
    with torch.no_grad():
        assert torch.equal(ops.groupnorm_act(x, gamma, beta, 1e-5, act=act, x1=x1, groups=groups, p=p, seed=31, offset=2), y)


@dtypes
@pytest.mark.parametrize("hw", [(8, 8), (64, 65)])
def test_groupnorm_act_far_from_zero_partial_gradients_and_strides(hw, dt):
    dt = DT[dt]
    # a common offset of 200 spreads: the statistics may not cancel (values near it are coarse in 16 bits)
    x = (rand(2, *hw, 64, scale=0.5) + 100.0).to(dt).requires_grad_()
    gamma, beta = rand(64, seed=2).requires_grad_(), rand(64, seed=3, grad=True)
    dy = rand(2, *hw, 64, dtype=dt, seed=4)
    ref = R.groupnorm_ref(x, None, gamma, beta, dy, 1e-6, "silu", 8, 0.0, 0, 0, dt)
    for leaves, names in (([x], ["dx"]), ([gamma], ["dgamma"]), ([beta], ["dbeta"]), ([x, gamma, beta], ["dx", "dgamma", "dbeta"])):
        args = [t if any(t is l for l in leaves) else t.detach() for t in (x, gamma, beta)]
        y = ops.groupnorm_act(*args, 1e-6, groups=8)
        R.check("y", y, *ref["y"])
        for name, g in zip(names, torch.autograd.grad(y, leaves, dy)):
            R.check(name, g, *ref[name])
    nchw = x.detach().permute(0, 3, 1, 2).contiguous()
    y2 = ops.groupnorm_act(nchw.permute(0, 2, 3, 1), gamma.detach(), beta.detach(), 1e-6, groups=8)
    R.check("y", y2, *ref["y"])
    e = torch.empty(0, *hw, 64, dtype=dt, device="cuda", requires_grad=True)
    y = ops.groupnorm_act(e, gamma, beta, groups=8)
    ge, gg, gb = torch.autograd.grad(y, [e, gamma, beta], torch.empty_like(y))
    assert ge.shape == e.shape and not gg.any() and not gb.any()


@dtypes
@pytest.mark.parametrize("hot", ["first", "middle", "last"])
@pytest.mark.parametrize("b,hw,c,groups", [(2, (8, 8), 64, 8), (1, (200, 201), 64, 4), (2, (64, 65), 30, 3)])
def test_groupnorm_act_with_an_outlier(b, hw, c, groups, hot, dt):
    """One pixel is a few hundred spreads away in every channel: it makes up most of the variance, and the statistics
    may not be its rounding, whichever pixel it is."""
    dt = DT[dt]
    n = hw[0] * hw[1]
    x = rand(b, n, c)
    x[:, {"first": 0, "middle": n // 2, "last": n - 1}[hot]] += 700.0
    x = x.reshape(b, *hw, c).to(dt).requires_grad_()
    gamma, beta = rand(c, seed=2).requires_grad_(), rand(c, seed=3, grad=True)
    dy = rand(b, *hw, c, dtype=dt, seed=4)
    ref = R.groupnorm_ref(x, None, gamma, beta, dy, 1e-5, "silu", groups, 0.0, 0, 0, dt)
    y = ops.groupnorm_act(x, gamma, beta, 1e-5, groups=groups)
    R.check("y", y, *ref["y"])
    for name, g in zip(("dx", "dgamma", "dbeta"), torch.autograd.grad(y, [x, gamma, beta], dy)):
        R.check(name, g, *ref[name])


def test_groupnorm_act_equals_the_inference_kernel_where_both_apply():
    for hw in ((16, 16), (64, 64)):
        x, gamma, beta = rand(2, *hw, 320), rand(320, seed=1), rand(320, seed=2)
        ref = R.groupnorm_ref(x, None, gamma, beta, None, 1e-5, "silu", 32, 0.0, 0, 0, torch.float32)["y"]
        R.check("groupnorm", ops.groupnorm(x, gamma, beta, 1e-5, silu=True), *ref)
        R.check("groupnorm_act", ops.groupnorm_act(x, gamma, beta, 1e-5), *ref)


# ---- all of them --------------------------------------------------------------------------------------------------

def test_fused_masks_are_dropouts_own():
    x, w = rand(100, 48), rand(77, 48, seed=1)
    z = ops.linear_act(x, w)
    assert torch.equal(ops.linear_act(x, w, p=0.4, seed=8, offset=6) != 0, ops.dropout(z, 0.4, 8, 6) != 0)
    for hw in (64, 4500):
        v = rand(2, hw, 64)
        g, b = torch.ones(64, device="cuda"), torch.full((64,), 3.0, device="cuda")
        n = ops.groupnorm_act(v, g, b, act=None, groups=8)
        assert torch.equal(ops.groupnorm_act(v, g, b, act=None, groups=8, p=0.4, seed=8, offset=6) != 0,
                           ops.dropout(n, 0.4, 8, 6) != 0)


def _block(x, p, seed, params):
    """Norm + SiLU + dropout, a feed-forward with dropout inside and behind, added to its input."""
    gamma, beta, w1, b1, w2, b2 = params
    h = ops.groupnorm_act(x, gamma, beta, groups=8, p=p, seed=seed, offset=0)
    h = ops.linear_act(h, w1, b1, act="gelu", p=p, seed=seed, offset=1)
    return ops.linear_act(h, w2, b2, resid=x, p=p, seed=seed, offset=2)


def _block_params(dt=torch.float32, c=64, f=96):
    return [(1 + rand(c, seed=1, scale=0.1)).requires_grad_(), rand(c, seed=2, scale=0.1, grad=True),
            rand(f, c, seed=3, scale=c ** -0.5, dtype=dt, grad=True), rand(f, seed=4, scale=0.1, grad=True),
            rand(c, f, seed=5, scale=f ** -0.5, dtype=dt, grad=True), rand(c, seed=6, scale=0.1, grad=True)]


def _block_ref(x, p, seed, params):
    gamma, beta, w1, b1, w2, b2 = params
    b, c = x.shape[0], x.shape[-1]
    v = x.reshape(b, -1, 8, c // 8)
    v = (v - v.mean((1, 3), keepdim=True)) / torch.sqrt(v.var((1, 3), unbiased=False, keepdim=True) + 1e-5)
    h = R.act(v.reshape(x.shape) * gamma + beta, "silu") * R.keep_scale(x.shape, p, seed, 0)
    h = R.act(h @ w1.t() + b1, "gelu") * R.keep_scale(h.shape[:-1] + (w1.shape[0],), p, seed, 1)
    return x + (h @ w2.t() + b2) * R.keep_scale(x.shape, p, seed, 2)


def test_block_against_formula_and_differences():
    params, x, dy = _block_params(), rand(2, 9, 11, 64, grad=True), rand(2, 9, 11, 64, seed=7)
    y = _block(x, 0.2, 3, params)
    grads = torch.autograd.grad(y, [x] + params, dy)
    ref = [R.d(t).requires_grad_() for t in [x] + params]
    yr = _block_ref(ref[0], 0.2, 3, ref[1:])
    want = torch.autograd.grad(yr, ref, R.d(dy))
    # three layers of fp32 sums of at most 6336 terms behind one another: 1e-4 of the largest entry
    for got, w in [(y, yr.detach())] + list(zip(grads, want)):
        assert float((got.detach().double().cpu() - w).abs().max()) < 1e-4 * float(w.abs().max())
    # against central differences of the 64-bit form along a random direction: step 1e-5, third derivatives of order
    # one leave 1e-10, cancellation 1e-16 / 1e-5 of the sum's size
    with torch.no_grad():
        for i, g in enumerate(grads):
            v = torch.randn(ref[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
            moved = [[t + s * 1e-5 * v if j == i else t for j, t in enumerate(ref)] for s in (1, -1)]
            up, down = (float((_block_ref(m[0], 0.2, 3, m[1:]) * R.d(dy)).sum()) for m in moved)
            got, scale = float((g.double().cpu() * v).sum()), float((g.double().cpu() * v).abs().sum())
            assert abs(got - (up - down) / 2e-5) < 1e-4 * scale + 1e-5, i


@dtypes
def test_captured_training_step_draws_anew_on_every_replay(dt):
    """Forward and backward captured once; every replay reads the seed's new value, between eager work of its own."""
    dt = DT[dt]
    params, x, dy = _block_params(dt), rand(2, 40, 50, 64, dtype=dt, grad=True), rand(2, 40, 50, 64, dtype=dt, seed=7)
    seed = torch.tensor([1], dtype=torch.int64, device="cuda")

    def step(s):
        y = _block(x, 0.2, s, params)
        return [y.detach(), *torch.autograd.grad(y, [x] + params, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(seed)
    last = None
    for s in (1, 2, 99, 2):
        seed.fill_(s)
        g.replay()
        torch.cuda.synchronize()
        eager = step(s)
        for a, b in zip(out, eager):
            assert torch.equal(a, b), s
        assert last is None or not torch.equal(out[0], last)
        last = out[0].clone()


def test_two_graphs_and_a_second_stream_keep_to_their_own_workspaces():
    """Sizes that need workspaces (split contraction, strips), interleaved on two streams, give the eager results."""
    w = rand(64, 4096, seed=1, scale=0.02)
    xs = [rand(100, 4096, seed=s) for s in (2, 3)]
    vs = [rand(1, 70, 70, 64, seed=s) for s in (4, 5)]
    gm, bt = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")

    def work(i):
        return ops.linear_act(xs[i], w, act="silu"), ops.groupnorm_act(vs[i], gm, bt, groups=8)
    want = [work(0), work(1)]
    graphs = []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work(i)
        graphs.append((g, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = []
        for i, s in enumerate(streams):
            s2 = torch.cuda.Stream()
            with torch.cuda.stream(s2):
                eager.append(work(i))
        torch.cuda.synchronize()
        for i in (0, 1):
            for got in (graphs[i][1], eager[i]):
                for a, b in zip(got, want[i]):
                    assert torch.equal(a, b)


def test_runs_are_repeatable():
    params, x, dy = _block_params(torch.bfloat16), rand(2, 64, 64, 64, dtype=torch.bfloat16, grad=True), \
        rand(2, 64, 64, 64, dtype=torch.bfloat16, seed=7)
    first = None
    for _ in range(3):
        y = _block(x, 0.1, 5, params)
        out = [y.detach(), *torch.autograd.grad(y, [x] + params, dy)]
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(out, first))
        first = out


def test_python_refusals_on_device_tensors():
    x, w = rand(4, 8), rand(16, 8)
    for bad in (lambda: ops.dropout(x, 0.5, None), lambda: ops.dropout(x, 0.5, 1, resid=x[:2]),
                lambda: ops.dropout(x, 0.5, 1, resid=x.half()), lambda: ops.dropout(x.long(), 0.5, 1),
                lambda: ops.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64)),
                lambda: ops.linear_act(x, w.half()), lambda: ops.linear_act(x, w.t()), lambda: ops.linear_act(x, w.cpu()),
                lambda: ops.linear_act(x, w, rand(8)), lambda: ops.linear_act(x, w, rand(16).half()),
                lambda: ops.linear_act(x, w, resid=x), lambda: ops.linear_act(x, w, act="relu"),
                lambda: ops.linear_act(x[:, :0], w[:, :0]),
                lambda: ops.groupnorm_act(x, rand(8), rand(8), groups=3), lambda: ops.groupnorm_act(x, rand(4), rand(8), groups=2),
                lambda: ops.groupnorm_act(x, rand(8), rand(8), groups=2, x1=rand(3, 8)),
                lambda: ops.groupnorm_act(x[0], rand(8), rand(8), groups=2)):
        with pytest.raises(ValueError):
            bad()
    v = rand(4, 8, grad=True)
    y, = torch.autograd.grad(ops.dropout(v, 0.5, 1).sum(), v, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), v)                    # no second derivatives


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("m,k,n,act", [(1, 64, 24, "silu"), (5, 320, 640, "gelu"), (77, 768, 768, "quick_gelu"), (300, 33, 130, "silu")])
def test_small_products_lose_nothing_but_their_own_rounding(m, k, n, act, dt):
    """dx and dw of small layers with an activation are as far from 64 bits as their own rounding puts them: what dz
    loses in the tensors' type is multiplied too.  An error of the same size on top would be 1.41 times as far."""
    dt = DT[dt]
    x, w = rand(m, k, dtype=dt, grad=True), rand(n, k, dtype=dt, seed=1, scale=k ** -0.5, grad=True)
    dy = rand(m, n, dtype=dt, seed=4)
    grads = torch.autograd.grad(ops.linear_act(x, w, act=act, p=0.1, seed=99), [x, w], dy)
    ref = R.linear_ref(x, w, None, None, dy, act, 0.1, 99, 0, dt)
    for got, name in zip(grads, ("dx", "dw")):
        want = ref[name][0]
        own = float((want.to(dt).double() - want).norm())
        assert float((got.double().cpu() - want).norm()) < 1.05 * own, name


# ---- the samplers' noise dropout ------------------------------------------------------------------------------

def test_samplers_noise_dropout_by_seed():
    """``noise_dropout_seed``: the same mask on every run whatever was drawn before, another one per step and seed, and
    the one that ops.dropout gives for (seed, step)."""
    from _util import device_latent_diffusion, synth
    model = device_latent_diffusion(4, "crossattn", "fp32")
    sampler = importlib.import_module("stable-diffusion_amd").DDIMSampler(model)
    sampler.make_schedule(50, ddim_eta=0.5, verbose=False)
    x = synth.normal(11, "psd.x", (2, 4, 16, 16)).cuda()
    ctx = torch.cat([synth.normal(2, "psd.uc", (2, 77, 768)), synth.normal(1, "psd.c", (2, 77, 768))]).cuda()
    noise = synth.normal(12, "psd.noise", (2, 4, 16, 16)).cuda()

    def step(index, nz=noise, **kw):
        st = sampler._StepState(sampler, x, True)
        st.step(ctx, 20 * index + 1, index, unconditional_guidance_scale=7.5, noise_fn=lambda s: nz, **kw)
        torch.rand(3, device="cuda")
        return st.x().clone()

    def t_step(**kw):
        return model.p_sample(x, ctx[:2], torch.full((2,), 500), **kw)
    a = step(49, noise_dropout=0.5, noise_dropout_seed=7)
    assert torch.equal(a, step(49, noise_dropout=0.5, noise_dropout_seed=7))
    assert torch.equal(a, step(49, ops.dropout(noise, 0.5, 7, 49)))
    assert not torch.equal(a, step(49, noise_dropout=0.5, noise_dropout_seed=8))
    b = t_step(noise=noise, noise_dropout=0.5, noise_dropout_seed=7)
    assert torch.equal(b, t_step(noise=ops.dropout(noise, 0.5, 7, 500)))
    assert not torch.equal(ops.dropout(noise, 0.5, 7, 49), ops.dropout(noise, 0.5, 7, 500))
    lat, _ = sampler.sample(4, 2, (4, 16, 16), conditioning=ctx, eta=0.5, x_T=x, verbose=False, noise_dropout=0.3,
                            unconditional_guidance_scale=7.5, unconditional_conditioning=True,
                            noise_fn=lambda s: noise, noise_dropout_seed=1)
    again, _ = sampler.sample(4, 2, (4, 16, 16), conditioning=ctx, eta=0.5, x_T=x, verbose=False, noise_dropout=0.3,
                              unconditional_guidance_scale=7.5, unconditional_conditioning=True,
                              noise_fn=lambda s: noise, noise_dropout_seed=1)
    assert torch.equal(lat, again)


def _layer_calls():
    x, w, b, g, h = rand(6, 16, grad=True), rand(24, 16, grad=True), rand(24), rand(16), rand(16)
    return x, {"dropout": lambda: ops.dropout(x, 0.5, 3),
               "linear": lambda: ops.linear_act(x, w, b, act="gelu", p=0.25, seed=3),
               "groupnorm": lambda: ops.groupnorm_act(x.view(2, 3, 16), g, h, groups=4, p=0.25, seed=3)}


@pytest.mark.parametrize("layer", ["dropout", "linear", "groupnorm"])
def test_autograd_refuses_what_the_layers_have_not(layer):
    x, calls = _layer_calls()
    call = calls[layer]
    g, = torch.autograd.grad(call().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives"):
        g.sum().backward()
    if layer != "dropout":                                  # (dropout keeps nothing that a first pass could free)
        y = call().sum()
        y.backward()
        with pytest.raises(RuntimeError, match="second time"):
            y.backward()
        y = call().sum()
        with torch.no_grad():
            x.mul_(1.0)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        t = fw.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            if layer == "dropout":
                ops.dropout(t, 0.5, 3)
            elif layer == "linear":
                ops.linear_act(t, rand(24, 16))
            else:
                ops.groupnorm_act(t.view(2, 3, 16), rand(16), rand(16), groups=4)
    torch.cuda.synchronize()


def test_recomputation_gives_the_same_gradients():
    """Activation checkpointing runs the forward pass a second time from inside the backward pass: the masks are the
    same ones, and so are the gradients, bit by bit."""
    from torch.utils.checkpoint import checkpoint
    x, w, b = rand(20, 64, grad=True), rand(64, 64, grad=True), rand(64, grad=True)

    def block(t):
        u = ops.groupnorm_act(t.view(4, 5, 64), torch.ones_like(b), b, groups=8, p=0.3, seed=9, offset=0)
        u = ops.linear_act(u.reshape(20, 64), w, b, act="silu", p=0.3, seed=9, offset=1)
        return ops.dropout(u, 0.3, 9, offset=2, resid=t)
    want = torch.autograd.grad(block(x).square().sum(), (x, w, b))
    for reentrant in (False, True):
        got = torch.autograd.grad(checkpoint(block, x, use_reentrant=False).square().sum(), (x, w, b)) if not reentrant \
            else None
        if reentrant:
            for t in (x, w, b):
                t.grad = None
            checkpoint(block, x, use_reentrant=True).square().sum().backward()
            got = (x.grad, w.grad, b.grad)
        for g, r in zip(got, want):
            assert torch.equal(g, r)


def test_tensors_of_more_than_2_to_the_31_elements():
    """Offsets beyond 32 bits: the last rows of a large call against the formula, and a batch's last image against a
    call of its own."""
    dt, m, k, n = torch.bfloat16, (1 << 21) + 4099, 64, 1032
    x, w = torch.zeros(m, k, dtype=dt, device="cuda"), rand(n, k, dtype=dt)
    x[-5:] = rand(5, k, seed=1).to(dt)
    dy = torch.zeros(m, n, dtype=dt, device="cuda")
    dy[-5:] = rand(5, n, seed=2).to(dt)
    x.requires_grad_(), w.requires_grad_()
    b = rand(n, seed=3, grad=True)
    y = ops.linear_act(x, w, b, act="silu", p=0.3, seed=4, offset=1)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    s = R.keep_scale((5, n), 0.3, 4, 1, row0=m - 5)
    xd, wd = R.d(x[-5:]), R.d(w)
    z = xd @ wd.t() + R.d(b)
    za = xd.abs() @ wd.abs().t() + R.d(b).abs()
    ez = (k + 2) * R.U * za
    ref = s * R.act(z, "silu")
    R.check("y", y[-5:], ref, R.rounded(ref, s * (1.13 * ez + R.ACT_ERR * z.abs().clamp(min=1)) + 4 * R.U * ref.abs(), dt))
    g = R.d(dy[-5:]) * s
    dz = g * R.act_grad(z, "silu")
    edz = R.rounded(dz, 4 * R.U * dz.abs() + g.abs() * (0.86 * ez + R.ACT_ERR * z.abs().clamp(min=1)), dt)
    for name, got, want, e, rows in (("dx", dx[-5:], dz @ wd, edz @ wd.abs(), n), ("dw", dw, dz.t() @ xd, edz.t() @ xd.abs(), 5)):
        R.check(name, got, want, R.rounded(want, e + (rows + 2) * R.U * (e + want.abs() + dz.abs().sum()), dt))
    R.check("db", db, dz.sum(0), edz.sum(0) + 8 * R.U * dz.abs().sum(0))
    assert not dx[:-5].any()
    del x, w, dy, y, dx, dw

    hw, c = (1 << 21) + 77, 640
    x = torch.empty(2, hw, c, dtype=dt, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(5))
    gamma, beta = rand(c, seed=2), rand(c, seed=3)
    x.requires_grad_()
    y = ops.groupnorm_act(x, gamma, beta, groups=32)
    dx, = torch.autograd.grad(y, x, y.detach())
    one = x.detach()[1:].clone().requires_grad_()
    y1 = ops.groupnorm_act(one, gamma, beta, groups=32)
    dx1, = torch.autograd.grad(y1, one, y.detach()[1:])
    # the strips differ, so the statistics may differ by a few 2^-24 of their size, and a value by one step of bf16
    for a, r in ((y[1:], y1), (dx[1:], dx1)):
        for lo in range(0, hw, 1 << 18):
            p, q = a[:, lo:lo + (1 << 18)].detach().float(), r[:, lo:lo + (1 << 18)].detach().float()
            assert bool(((p - q).abs() <= 2.0 ** -7 * q.abs() + 1e-5).all())
    del x, y, dx, one, y1, dx1
    torch.cuda.empty_cache()


def test_groupnorm_act_of_more_slices_than_a_launch_has_blocks_in_a_row():
    """A group per channel and many samples: 2^27 slices, whose threads are more than 2^32."""
    b, c = 65535, 2048
    x = torch.empty(b, 2, c, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    gamma, beta = rand(c, seed=2).requires_grad_(), rand(c, seed=3, grad=True)
    x.requires_grad_()
    y = ops.groupnorm_act(x, gamma, beta, groups=c)
    dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), torch.ones_like(y))
    for i in (0, 1023, 30000, b - 1):
        ref = R.groupnorm_ref(x[i:i + 1], None, gamma, beta, torch.ones(1, 2, c), 1e-5, "silu", c, 0.0, 0, 0, torch.float16)
        R.check("y", y[i:i + 1], *ref["y"])
        R.check("dx", dx[i:i + 1], *ref["dx"])
    assert torch.isfinite(dg).all() and torch.isfinite(db).all()
    del x, y, dx
    torch.cuda.empty_cache()


def test_two_threads_at_once():
    """Two threads with a stream each, forward and backward, give what they give one after the other."""
    import threading

    def work(i):
        x, w, b = rand(300 + i, 256, seed=i, grad=True), rand(384, 256, seed=i, grad=True), rand(384, seed=i, grad=True)
        g, h = rand(384, seed=i + 5).requires_grad_(), rand(384, seed=i + 6, grad=True)
        u = ops.linear_act(x, w, b, act="gelu", p=0.2, seed=i, offset=0)
        u = ops.groupnorm_act(u.view(1, -1, 384), g, h, groups=12, p=0.2, seed=i, offset=1)
        u = ops.dropout(u, 0.2, i, offset=2)
        return [u] + list(torch.autograd.grad(u.square().sum(), (x, w, b, g, h)))
    want = [[t.detach().cpu() for t in work(i)] for i in range(2)]
    wrong = []

    def loop(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = [t.detach().cpu() for t in work(i)]
                    if not all(torch.equal(a, r) for a, r in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:                      # noqa: BLE001  (a thread's failure must reach the test)
            wrong.append(repr(e))
    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
