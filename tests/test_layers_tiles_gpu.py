"""GPU: every tile of linear_act's products, in each layout of the operands, whole and split, aligned and not, with 16-bit dz in
one part and in two, with one, two, three and more K-tiles and tails in all three sizes, against 64 bits.  Each case names the
tiles that it is there for, as the profiler's records have them: a plan that no longer takes them fails."""
import importlib
import math

import pytest
import torch

import _layers_ref as R

pytestmark = pytest.mark.gpu

ops = importlib.import_module("stable-diffusion_amd.ops")
_lib = importlib.import_module("stable-diffusion_amd._lib")
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}

# m, k, n, activation, tile / splits of x W^T, of dz W and of dz^T x
FP32 = [
    (25160, 80, 8, 1, "64/1", "128/1", "64/61"), (60632, 71, 9, 1, "64/1", "128/1", "64/64"),
    (72, 2768, 904, 1, "64/8", "128/10", "64/1"), (1056, 72, 2920, 0, "128/1", "64/14", "128/11"),
    (72, 3129, 2321, 0, "64/10", "64/10", "128/1"), (200, 3000, 1056, 0, "128/14", "64/1", "128/1"),
    (68, 5547, 2053, 1, "128/29", "128/11", "64/1"), (62412, 9, 81, 1, "128/1", "64/1", "64/63"),
    (9834, 1059, 67, 0, "64/3", "64/1", "128/52"), (72, 8, 8, 0, "64/1", "64/1", "64/1"),
    (72, 1392, 2568, 1, "64/3", "128/21", "128/1"), (5694, 65, 2771, 1, "128/1", "128/11", "128/23"),
]
HALF = [
    (27224, 72, 8, 1, "64/1", "128/1", "64/61"), (968, 3096, 8, 0, "64/13", "128/1", "64/8"),
    (40993, 73, 9, 1, "64/1", "128/1", "64/59"), (3645, 1703, 9, 0, "64/7", "128/1", "64/15"),
    (72, 2072, 2736, 0, "128/11", "64/11", "128/1"), (1221, 83, 5219, 1, "128/1", "64/21", "128/10"),
    (1816, 72, 4104, 1, "128/1", "64/13", "128/10"), (12616, 72, 1144, 0, "256x256/1", "64/1", "128/50"),
    (63848, 8, 136, 0, "256x256/1", "64/1", "64/63"), (49888, 8, 264, 1, "256x320/1", "64/1", "64/60"),
    (68, 3123, 5543, 0, "128/10", "64/10", "128/1"), (80, 5560, 728, 1, "64/10", "64/1", "128/1"),
    (776, 80, 5768, 1, "64/1", "128/31", "64/1"), (1448, 72, 5200, 0, "128/1", "128/21", "64/1"),
    (71, 4195, 2001, 1, "64/11", "128/11", "64/1"), (67, 4239, 2871, 0, "64/8", "128/15", "64/1"),
    (52200, 136, 136, 1, "256x256/1", "256x256/1", "64/55"), (17191, 65, 911, 0, "64/1", "64/1", "128/54"),
    (12248, 72, 1304, 1, "256x320/1", "128/4", "128/39"), (50392, 200, 136, 0, "256x256/1", "256x256/1", "64/61"),
    (50856, 136, 264, 1, "256x320/1", "256x256/1", "64/62"), (67, 9, 9, 1, "64/1", "64/1", "64/1"),
    (68, 9, 11, 0, "64/1", "64/1", "64/1"), (57176, 168, 8, 1, "64/1", "256x256/1", "64/64"),
    (54616, 208, 8, 0, "64/1", "256x256/1", "64/61"), (46088, 304, 8, 1, "64/1", "256x320/1", "64/61"),
    (55888, 264, 8, 0, "64/1", "256x320/1", "64/63"), (3128, 5848, 136, 1, "128/10", "256x320/1", "256x256/10"),
    (44048, 200, 288, 0, "256x320/1", "256x256/1", "128/63"), (68, 2289, 1857, 1, "64/12", "64/10", "128/1"),
    (72, 3176, 1832, 0, "64/8", "128/10", "128/1"), (66, 5669, 1251, 1, "64/12", "128/10", "128/1"),
    (51592, 144, 72, 1, "128/1", "256x256/1", "64/63"), (2001, 4203, 69, 1, "64/11", "64/1", "128/11"),
    (59464, 136, 72, 0, "128/1", "256x256/1", "64/62"), (72, 2376, 3472, 1, "128/8", "128/11", "256x256/1"),
    (9361, 1181, 69, 0, "64/1", "128/1", "128/49"), (144, 5616, 4488, 1, "128/6", "256x256/9", "256x256/1"),
    (72, 3752, 3216, 0, "128/8", "128/8", "256x256/1"), (44752, 264, 80, 1, "128/1", "256x320/1", "64/64"),
    (46368, 288, 72, 0, "128/1", "256x320/1", "64/61"), (160, 5512, 5656, 0, "256x256/11", "128/4", "256x256/1"),
    (200, 3488, 2320, 1, "128/6", "128/8", "256x256/1"), (200, 5960, 1448, 0, "128/10", "64/1", "256x256/1"),
    (45048, 272, 144, 0, "256x256/1", "256x320/1", "64/64"), (45112, 272, 200, 0, "256x256/1", "256x320/1", "64/47"),
    (46544, 280, 216, 1, "256x256/1", "256x320/1", "128/61"), (3704, 680, 5816, 0, "128/1", "256x256/4", "256x256/3"),
    (536, 5688, 4448, 1, "256x320/6", "128/2", "256x256/1"),
]


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 17 * len(shape) + sum(shape))
    return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g).to(dtype)


def recorded(tmp_path, run):
    """What run() returns, and the labels of its products."""
    lib = _lib.lib()
    lib.sdmi_prof_reset()
    lib.sdmi_prof_enable(1)
    try:
        out = run()
        torch.cuda.synchronize()
    finally:
        lib.sdmi_prof_enable(0)
    path = tmp_path / "prof.csv"
    assert lib.sdmi_prof_dump(str(path).encode()) == 0
    lib.sdmi_prof_reset()
    return out, [p for line in path.read_text().splitlines() for p in line.split(",") if p.startswith("linear M")]


def close(name, got, want, terms, act, dt, two):
    """A sum of ``terms`` products in fp32 is off, in units of the sums' spread s, by 0.41 sqrt(terms) u at the mean: the
    partial sums grow as the square root, each addition rounds by u / sqrt(3) of one.  Ten times that, 16 u for the epilogue and
    ACT_ERR of up to five times s for an activation; a 16-bit dz in two parts adds eps^2 / 2 of each term at most, so four
    times that of s at the very most.  Then the result's own rounding."""
    want, got = want.double(), got.detach().double()
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    s = float(want.square().mean().sqrt())
    err = 4 * math.sqrt(terms) * R.U + 16 * R.U + (5 * R.ACT_ERR if act else 0.0)
    if two:
        err += 2 * torch.finfo(dt).eps ** 2
    own = R.half(got_dtype(name, dt)) if name != "db" else R.U
    over = (got - want).abs() - (err * s + own * (want.abs() + err * s)) - torch.finfo(dt).smallest_normal
    assert float(over.max()) <= 0, (name, float(over.max()), int(over.argmax()), s)


def got_dtype(name, dt):
    return torch.float32 if name == "db" else dt


def layer(m, k, n, act, dt, p, views=(), tmp_path=None):
    """One layer forward and backward against 64 bits; views: arguments that come as unaligned views."""
    def odd(t):                                   # the same values, rows at odd addresses one element apart
        wide = torch.empty(t.shape[0], t.shape[1] + 1, dtype=t.dtype, device="cuda")
        wide[:, 1:] = t
        return wide[:, 1:]
    x, w = rand(m, k, dtype=dt), rand(n, k, dtype=dt, seed=1, scale=k ** -0.5)
    x, w = (odd(t) if name in views else t for name, t in (("x", x), ("w", w)))
    b, r, dy = rand(n, seed=2, scale=0.3), rand(m, n, dtype=dt, seed=3), rand(m, n, dtype=dt, seed=4)
    if "dy" in views:
        dy = odd(dy)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    name = "gelu" if act else None

    def run():
        y = ops.linear_act(x, w, b, act=name, resid=r, p=p, seed=99, offset=4)
        return y, torch.autograd.grad(y, leaves, dy)
    (y, (dx, dw, db, dr)), labels = recorded(tmp_path, run)
    y2, g2 = run()
    for a, c in zip((y, dx, dw, db, dr), (y2, *g2)):
        assert torch.equal(a, c)                  # and again, bit by bit
    del y2, g2
    xd, wd, g = x.detach().double(), w.detach().double(), dy.double()
    keep = ops.dropout(torch.ones(m, n, device="cuda"), p, 99, 4).double()
    keep = torch.where(keep > 0, 65536.0 / (65536 - round(p * 65536)), 0.0) if p else keep
    z = xd @ wd.t() + b.detach().double()
    close("y", y, R.act(z, name) * keep + r.detach().double(), k, act, dt, False)
    dz = g * keep * R.act_grad(z, name)
    two = bool(act) and dt != torch.float32
    close("dx", dx, dz @ wd, n, act, dt, two)
    close("dw", dw, dz.t().contiguous() @ xd, m, act, dt, two)
    close("db", db, dz.sum(0), m, act, dt, False)
    assert torch.equal(dr, dy)
    return labels


def label(m, n, k, tile, aligned, other=None):
    t, s = tile.split("/")
    return f"linear M{m} N{n} K{k} {t if 'x' in t else t + 'x' + t}{'' if aligned else 'u'}/{s}{'' if other is None else '+' + other}"


def expected(m, k, n, f, x, w, dt, views=()):
    e = torch.finfo(dt).bits // 8
    af = k * e % 16 == 0 and n % 8 == 0 and not {"x", "w"} & set(views)
    ag = n * e % 16 == 0 and k * e % 16 == 0 and k % 8 == 0
    ax, aw = ag and not {"w", "dy"} & set(views), ag and not {"x", "dy"} & set(views)
    small = lambda t, a: t if a or not t.startswith("256") else "128/" + t.split("/")[1]
    f, x, w = small(f, af), small(x, ax), small(w, aw)
    out = [label(m, n, k, f, af)]
    if x.split("/")[0] == w.split("/")[0] and not x.startswith("256") and ax == aw:
        return out + [label(n, k, m, w, aw, x.split("/")[1])]
    return out + [label(n, k, m, w, aw), label(m, k, n, x, ax)]


@pytest.mark.parametrize("case", FP32, ids=lambda c: "-".join(str(v) for v in c))
def test_tiles_fp32(case, tmp_path):
    m, k, n, act, f, x, w = case
    labels = layer(m, k, n, act, torch.float32, 0.1 if (m + k) % 3 else 0.0, tmp_path=tmp_path)
    assert labels == expected(m, k, n, f, x, w, torch.float32)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("case", HALF, ids=lambda c: "-".join(str(v) for v in c))
def test_tiles_16_bit(case, dt, tmp_path):
    m, k, n, act, f, x, w = case
    labels = layer(m, k, n, act, DT[dt], 0.1 if (m + k) % 3 else 0.0, tmp_path=tmp_path)
    assert labels == expected(m, k, n, f, x, w, DT[dt])


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("views", [("x",), ("w",), ("dy",), ("x", "w", "dy")], ids="-".join)
@pytest.mark.parametrize("case", [c for c in HALF if (c[0], c[1], c[2]) in
                                  {(50392, 200, 136), (144, 5616, 4488), (160, 5512, 5656), (3704, 680, 5816), (200, 3488, 2320)}],
                         ids=lambda c: "-".join(str(v) for v in c))
def test_large_tiles_give_way_to_unaligned_views(case, views, dt, tmp_path):
    """Sizes that take 256-wide tiles, with rows at addresses that LDS-DMA does not take: 128x128, and the same splits."""
    m, k, n, act, f, x, w = case
    labels = layer(m, k, n, act, DT[dt], 0.0 if not act else 0.1, views=views, tmp_path=tmp_path)
    # with an activation dz is the call's own memory, whatever dy's rows are
    seen = [v for v in views if v != "dy" or not act]
    assert labels == expected(m, k, n, f, x, w, DT[dt], views=seen)
