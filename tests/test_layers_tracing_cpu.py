"""CPU: what would record the layers with dropout and gradients without their kernels is refused, before anything else."""
import importlib

import pytest
import torch

ops = importlib.import_module("stable-diffusion_amd.ops")


def calls():
    g, h = torch.ones(8), torch.zeros(8)
    return [lambda t: ops.dropout(t, 0.5, 1), lambda t: ops.linear_act(t, torch.ones(16, 8)),
            lambda t: ops.groupnorm_act(t.view(1, 4, 8), g, h, groups=2)]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_tracing_is_refused(which):
    """A tracer would record the allocation of the result and not the launch that fills it."""
    call, x = calls()[which], torch.zeros(4, 8)
    with pytest.raises(NotImplementedError, match="trac"):
        torch.jit.trace(call, (x,), check_trace=False)
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(NotImplementedError, match="trac"):
        make_fx(call)(x)
    for how in (dict(tracing_mode="fake"), dict(pre_dispatch=True)):
        with pytest.raises(NotImplementedError, match="trac"):
            make_fx(call, **how)(x)
    with pytest.raises(ValueError, match="CPU"):          # and is over when it is over
        call(x)
