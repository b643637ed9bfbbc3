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


class Wrapper(torch.Tensor):
    """A tensor whose memory is another's: torch hands its operators to Python."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device="cuda")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} was called")


def test_tensors_without_memory_of_their_own_are_refused():
    """No address of such a tensor is any of its values': an optional one would even be taken for a missing one."""
    x, w, r, g, s = (Wrapper(t) for t in (torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, 16), torch.zeros(8),
                                         torch.zeros(1, dtype=torch.int64)))
    p = torch.zeros(4, 8)
    for call in (lambda: ops.dropout(x, 0.0, 1), lambda: ops.dropout(p, 0.5, s), lambda: ops.dropout(p, 0.5, 1, resid=x),
                 lambda: ops.linear_act(x, torch.zeros(16, 8)), lambda: ops.linear_act(p, w),
                 lambda: ops.linear_act(p, torch.zeros(16, 8), resid=r),
                 lambda: ops.linear_act(p, torch.zeros(16, 8), Wrapper(torch.zeros(16))),
                 lambda: ops.groupnorm_act(p.view(1, 4, 8), g, torch.zeros(8), groups=2),
                 lambda: ops.groupnorm_act(p.view(1, 4, 8), torch.zeros(8), g, groups=2),
                 lambda: ops.groupnorm_act(x, g, g, groups=2),
                 lambda: ops.groupnorm_act(p, torch.zeros(16), torch.zeros(16), groups=2, x1=x)):
        with pytest.raises(NotImplementedError, match="memory of its own"):
            call()
