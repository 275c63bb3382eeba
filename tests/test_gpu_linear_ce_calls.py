"""Calls of the cross entropy from hidden states and of the gradient clipping that the kernels have to refuse or count."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu

from optimus_lm_b200.ops import _ext, functional as OF


def make(T, H, V, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, device="cuda", generator=g).to(torch.bfloat16)
    w = (torch.randn(V, H, device="cuda", generator=g) * 0.05).to(torch.bfloat16)
    return x, w, torch.randint(0, V, (T,), device="cuda", generator=g)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("requires_grad", [True, False])
def test_forward_mode_of_the_loss_is_refused(grad, requires_grad):
    # no_grad does not switch forward mode off
    x, w, t = make(40, 64, 100)
    x.requires_grad_(requires_grad)
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        for a, b in ((fwad.make_dual(x, torch.ones_like(x)), w), (x, fwad.make_dual(w, torch.ones_like(w)))):
            for reduction in ("mean", "none"):
                with pytest.raises(NotImplementedError, match="forward"):
                    OF.linear_cross_entropy(a, b, t, reduction)
        # types that take the plain path have the derivative
        dual = fwad.make_dual(x.detach().float(), torch.ones(40, 64, device="cuda"))
        assert fwad.unpack_dual(OF.linear_cross_entropy(dual, w.float(), t)).tangent is not None


def test_forward_mode_of_the_clipping_is_refused():
    g = torch.ones(100, device="cuda")
    with fwad.dual_level():
        dual = fwad.make_dual(g, torch.ones_like(g))
        with pytest.raises(NotImplementedError, match="forward"):
            OF.grad_norm([torch.zeros(3, device="cuda"), dual])
        with pytest.raises(NotImplementedError, match="forward"):
            OF.clip_grad_norm_([torch.zeros(3, device="cuda"), dual], 1.0)
    assert torch.equal(g, torch.ones_like(g))


def test_frozen_head_past_the_workspace():
    # without a gradient of the weight there is no fp32 gradient of it that would have to fit: the forward makes the
    # gradient of x, and the backward only scales it
    T, H, V = 8192, 256, 20000
    x, w, t = make(T, H, V)
    x.requires_grad_()
    loss = OF.linear_cross_entropy(x, w, t, max_workspace=4 * w.numel() - 1)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dx, = torch.autograd.grad(loss, x)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - held <= 2 * x.numel() + (1 << 16)
    want, = torch.autograd.grad(OF.linear_cross_entropy(x, w, t, max_workspace=2 << 30), x)
    # one more rounding to bf16
    assert ((dx.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -16 * want.float().abs().max()).all()


# sizes whose products split their last wave and do not, every way to hold the exponentials, without gradients
COUNTED = [("mean", 300, 1000, 3000, {}, "xw"), ("sum", 512, 256, 1024, {}, "xw"), ("none", 600, 64, 500, {"max_workspace": 1}, "xw"),
           ("mean", 600, 64, 500, {"max_workspace": 4 * 64 * 500}, "xw"), ("mean", 600, 64, 500, {"max_workspace": 4 * 64 * 500}, "x"),
           ("none", 40, 64, 500, {}, "w"), ("none", 40, 64, 500, {}, "")]


@pytest.mark.parametrize("reduction,T,H,V,kw,need", COUNTED)
def test_launches_are_counted(reduction, T, H, V, kw, need):
    x, w, t = make(T, H, V)
    leaves = [v.requires_grad_() for v, n in ((x, "x"), (w, "w")) if n in need]

    def call():
        loss = OF.linear_cross_entropy(x, w, t, reduction, **kw)
        if leaves:
            torch.autograd.grad(loss, leaves, torch.ones_like(loss))
        torch.cuda.synchronize()

    call()
    proxy = _ext.enable_launch_counting()
    try:
        before = proxy.launches, proxy.by_name.get("linear_ce", 0)
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA, torch.profiler.ProfilerActivity.CPU]) as prof:
            call()
        counted = proxy.launches - before[0]
        assert proxy.by_name["linear_ce"] - before[1] == counted
    finally:
        _ext._C = proxy._mod
    seen = [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA and "olb::" in e.name]
    assert counted == len(seen) > 0, (counted, seen)
