"""GPU: the layers with dropout and gradients where their accuracy is easily lost: large, small and infinite gradients in 16
bits, sizes on both sides of what a plan decides, outliers under the statistics, sums over many samples, tails of the
activations.  Against 64-bit forms, on the GPU where they are large."""
import importlib
import math

import pytest
import torch

import _layers_ref as R

pytestmark = pytest.mark.gpu

ops = importlib.import_module("stable-diffusion_amd.ops")
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
dtypes = pytest.mark.parametrize("dt", list(DT))
halves = pytest.mark.parametrize("dt", ["fp16", "bf16"])


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0, grad=False):
    g = torch.Generator().manual_seed(seed + 17 * len(shape) + sum(shape))
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda().requires_grad_(grad)


def exact_linear(x, w, bias, dy, act, p, seed, offset):
    """z, dz, dx, dw, db in 64 bits on the GPU."""
    x, w, dy = x.detach().double(), w.detach().double(), dy.double()
    z = x @ w.t()
    if bias is not None:
        z = z + bias.detach().double()
    dz = dy * R.act_grad(z, act)
    if p:
        dz = dz * R.keep_scale(dy.shape, p, seed, offset).cuda()
    return z, dz, dz @ w, dz.t().contiguous() @ x, dz.sum(0)


# ---- gradients at the ends of the types' range ----------------------------------------------------------------

@halves
@pytest.mark.parametrize("m,k,n,act,p", [(616, 768, 2000, "quick_gelu", 0.0), (2048, 320, 1280, "gelu", 0.1),
                                         (2056, 1992, 2568, "silu", 0.1), (4096, 1280, 5120, "gelu", 0.1)])
def test_large_products_lose_nothing_but_their_own_rounding(m, k, n, act, p, dt):
    """dx and dw are as far from 64 bits as their own rounding puts them at every size: a dz rounded to 16 bits would make it
    1.41 times as far.  What the fp32 sums and the two parts of dz add is below 1e-4 of the largest entries' size and so
    below 1 % of the rounding in the 2-norm."""
    dt = DT[dt]
    x, w = rand(m, k, dtype=dt, grad=True), rand(n, k, dtype=dt, seed=1, scale=k ** -0.5, grad=True)
    dy = rand(m, n, dtype=dt, seed=4)
    grads = torch.autograd.grad(ops.linear_act(x, w, act=act, p=p, seed=99), [x, w], dy)
    _, _, dx, dw, _ = exact_linear(x, w, None, dy, act, p, 99, 0)
    for name, got, want in (("dx", grads[0], dx), ("dw", grads[1], dw)):
        own = float((want.to(dt).double() - want).norm())
        assert float((got.double() - want).norm()) < 1.01 * own, name
