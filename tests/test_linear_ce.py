"""Cross entropy from hidden states: the plain path against the formula in 64 bits, and what the call refuses."""
import pytest
import torch

from optimus_lm_b200.ops import functional as OF


def problem(T=37, H=16, V=50, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g, requires_grad=True)
    w = torch.randn(V, H, generator=g, requires_grad=True)
    t = torch.randint(0, V, (T,), generator=g)
    t[3], t[5], t[6] = -100, -1, V
    return x, w, t


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_plain_path(reduction):
    x, w, t = problem()
    live = (t >= 0) & (t < 50)
    logp = torch.log_softmax(x.double() @ w.double().t(), 1)
    rows = -logp[torch.arange(37), t.clamp(0, 49)] * live
    want = {"mean": rows.sum() / live.sum(), "sum": rows.sum(), "none": rows}[reduction]
    got = OF.linear_cross_entropy(x, w, t, reduction)
    assert got.dtype == torch.float32 and torch.allclose(got.double(), want, rtol=1e-5, atol=1e-5)
    v = torch.ones_like(got)
    for a, b in zip(torch.autograd.grad(got, (x, w), v), torch.autograd.grad(want, (x, w), v.double())):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


def test_shapes_and_the_shifted_form():
    x, w, _ = problem(T=24)
    labels = torch.randint(0, 50, (4, 6))
    h = x.detach().view(4, 6, 16)
    assert OF.linear_cross_entropy(h, w, labels, "none").shape == (4, 6)
    a = OF.shifted_linear_cross_entropy(h, w.detach(), labels)
    b = OF.shifted_cross_entropy_reference(h @ w.detach().t(), labels)
    assert torch.allclose(a, b, rtol=1e-5)
    assert OF.linear_cross_entropy(x[:0], w, labels.view(-1)[:0]).isnan()
    assert OF.linear_cross_entropy(x[:0], w, labels.view(-1)[:0], "sum") == 0
    assert OF.linear_cross_entropy(x[:2], w, torch.tensor([-100, -100])).isnan()


def test_refusals():
    x, w, t = problem()
    ok = dict(x=x, weight=w, targets=t)
    for change in (dict(reduction="median"), dict(weight=w[:, :8]), dict(weight=w[0]), dict(targets=t[:-1]), dict(targets=t.float()),
                   dict(targets=t.bool()), dict(weight=w[:0]), dict(targets=t.view(1, -1)), dict(max_workspace=0),
                   dict(x=x.to("meta")), dict(targets=t.to("meta"))):
        with pytest.raises(ValueError):
            OF.linear_cross_entropy(**{**ok, **change})
    with pytest.raises(ValueError):
        OF.shifted_linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError):
        OF.shifted_linear_cross_entropy(x.view(1, 37, 16), w, t.view(37, 1))


@pytest.mark.parametrize("bad", [torch.float32, torch.float64, torch.bool, torch.complex64])
def test_shifted_form_takes_integer_labels(bad):
    x, w, _ = problem(T=24)
    with pytest.raises(ValueError, match="integers"):
        OF.shifted_linear_cross_entropy(x.view(4, 6, 16), w, torch.ones(4, 6).to(bad))
    assert torch.isfinite(OF.shifted_linear_cross_entropy(x.view(4, 6, 16), w, torch.ones(4, 6, dtype=torch.int32)))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_ignored_rows_may_hold_anything(reduction, bad):
    x, w, t = problem()
    clean = x.detach().clone().requires_grad_()
    with torch.no_grad():
        x[3], x[5, 2], x[6] = bad, bad, -bad
        clean[3], clean[5], clean[6] = 0.0, 0.0, 0.0
    got, want = OF.linear_cross_entropy(x, w, t, reduction), OF.linear_cross_entropy(clean, w, t, reduction)
    assert torch.equal(got, want)
    v = torch.ones_like(got)
    for a, b in zip(torch.autograd.grad(got, (x, w), v), torch.autograd.grad(want, (clean, w), v)):
        assert torch.equal(a, b)
