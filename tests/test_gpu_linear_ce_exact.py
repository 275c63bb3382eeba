"""Cross entropy from hidden states where every logit is exact: what is left is the arithmetic behind the logits.

The hidden states have two channels that are not zero, x = (a, 1, 0, ...), the weight's rows are (b, c_v, 0, ...), all of
them small integers times powers of two, so that l_rv = a_r b + c_v is exact in fp32 in whatever order it is summed and
l_rv - l_rt = c_v - c_t is exact too, however large a b is.

Bounds, with |c_v - c_t| <= 6 and 13 columns: an exponential is off by the rounding of its exponent (2^-24 * 6 log2 e) ln 2
and of log2 e itself (1.4e-8 * 6), 2^-22 for the instruction, and the sum of 13 by 13 * 2^-24, together below 2^-19 of
the row's sum; the logarithm by 2^-22 of the loss.  A gradient's entries carry the bf16 rounding of the exponentials and the row
factor's share of the target's rounding (2^-8 p each); the target's own entry 2^-16 |d| + (2^-8)^2 |d|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

from optimus_lm_b200.ops import functional as OF

U, U32 = 2.0 ** -8, 2.0 ** -23
V = 13
WAYS = {"whole": {}, "columns": {"max_workspace": 1}, "rows": {"max_workspace": None}}


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert OF.check_status("cuda") == 0, "a kernel reported a timeout / overflow in the status word"


def problem(H, a, b, T=600, far=False):
    g = torch.Generator().manual_seed(H + T)
    x, w = torch.zeros(T, H), torch.zeros(V, H)
    x[:, 0] = a[torch.randint(0, len(a), (T,), generator=g)]
    x[:, 1] = 1.0
    w[:, 0] = b
    w[:, 1] = -torch.randint(0, 7, (V,), generator=g).float()
    t = torch.randint(0, V, (T,), generator=g)
    if far:   # a column 100 below the others, the target of some rows
        w[4, 1] = -100.0
        t[::7] = 4
    assert torch.equal(x, x.to(torch.bfloat16).float()) and torch.equal(w, w.to(torch.bfloat16).float())
    return x.cuda().to(torch.bfloat16), w.cuda().to(torch.bfloat16), t.cuda()


def check(x, w, t, reduction, way):
    kw = dict(WAYS[way])
    if way == "rows":
        kw["max_workspace"] = 4 * w.numel()
        assert 2 * 64 * x.shape[0] > 4 * w.numel()   # more than one piece
    T = x.shape[0]
    row_grad = torch.rand(T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) - 0.3 if reduction == "none" else None
    xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = OF.linear_cross_entropy(xg, wg, t, reduction, **kw)
    dx, dw = torch.autograd.grad(loss, (xg, wg), row_grad)
    xd, wd = x.double(), w.double()
    l = xd @ wd.t()
    lse = torch.logsumexp(l - l.gather(1, t[:, None]), 1)   # of the differences: the loss itself
    tol = 2.0 ** -19 + 2.0 ** -22 * lse
    want, tol = (lse, tol) if reduction == "none" else (lse.mean(), tol.mean())
    off = ((loss.double() - want).abs() / tol).max().item()
    assert off <= 1, f"loss: {off:.2f} x its bound"
    g = row_grad.double()[:, None] if reduction == "none" else torch.full((T, 1), 1.0 / T, dtype=torch.float64, device="cuda")
    p = torch.softmax(l, 1)
    onehot = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    d = g * (p - onehot)
    err = torch.where(onehot > 0, d.abs() * (2.0 ** -16 + U * U) + g.abs() * p * 2.0 ** -18, g.abs() * p * (2 * U + 2.0 ** -18))
    for name, got, e, bound in (
            ("dx", dx, d @ wd, err @ wd.abs() + 2 * (x.shape[1] + V) ** 0.5 * U32 * (d.abs() @ wd.abs())),
            ("dw", dw, d.t() @ xd, err.t() @ xd.abs() + U * (d.abs().t() @ xd.abs()) + 2 * T ** 0.5 * U32 * (d.abs().t() @ xd.abs()))):
        bound = bound + (2 if way == "rows" and name == "dx" else 1) * U * e.abs()
        off = ((got.double() - e).abs() / (bound * 1.01 + 1e-37)).max().item()
        assert off <= 1, f"{name}: {off:.2f} x its bound"
    with torch.no_grad():
        scored = OF.linear_cross_entropy(x, w, t, reduction, **kw)
    assert ((scored.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("H", [64, 512, 2048, 7168])
def test_wide_hidden_states_of_few_channels(H, way):
    # nothing to round in the logits, whatever the number of channels
    T = 3000 if way == "rows" else 600
    check(*problem(H, torch.arange(1.0, 17.0), 1.0, T), "mean", way)
    check(*problem(H, torch.arange(1.0, 17.0), 1.0, T), "none", way)

# logits of up to 992 and of 2^20 to 2^21, of both signs
LARGE = {"hundreds": (torch.cat([torch.arange(1.0, 63.0), -torch.arange(1.0, 63.0)]), 16.0),
         "millions": (torch.cat([torch.arange(1024.0, 2048.0, 8.0), -torch.arange(1024.0, 2048.0, 8.0)]), 1024.0)}


@pytest.mark.parametrize("way", ["whole", "rows"])
@pytest.mark.parametrize("size", LARGE)
@pytest.mark.parametrize("far", [False, True])
def test_large_logits(size, far, way):
    check(*problem(16, *LARGE[size], far=far), "mean", way)
    if way == "whole":
        check(*problem(16, *LARGE[size], far=far), "none", way)


@pytest.mark.parametrize("size", LARGE)
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_large_logits_computed_again(size, far, reduction):
    check(*problem(16, *LARGE[size], far=far), reduction, "columns")


@pytest.mark.parametrize("H", [64, 2048, 7168])
def test_mean_loss_of_random_hidden_states(H):
    # The signed error of the mean, which the rounding of single logits leaves and a factor on all of them does not.  A step of
    # 16 terms truncates the running sum s by less than a step of fp32 of it, the 16 products' own truncations have random
    # signs (another step): |mean error| <= 2 2^-23 mean_r sum_v p_v sum_k |s_k|, and 2^-20 of the loss for exp, sums and log.
    T, V = 64, 500
    g = torch.Generator(device="cuda").manual_seed(H)
    x = torch.randn(T, H, device="cuda", generator=g).to(torch.bfloat16)
    w = (torch.randn(V, H, device="cuda", generator=g) * (3.0 / H ** 0.5)).to(torch.bfloat16)
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    steps = torch.einsum("tkh,vkh->tvk", x.double().view(T, H // 16, 16), w.double().view(V, H // 16, 16)).cumsum(2)
    l = steps[..., -1]
    p = torch.softmax(l, 1)
    want = (torch.logsumexp(l, 1) - l.gather(1, t[:, None])[:, 0])
    bound = 2 * U32 * (p * steps.abs().sum(2)).sum(1).mean() + 2.0 ** -20 * want.mean()
    with torch.no_grad():
        off = (OF.linear_cross_entropy(x, w, t, "none").double() - want).mean().abs()
        off_mean = (OF.linear_cross_entropy(x, w, t).double() - want.mean()).abs()
    assert off <= bound and off_mean <= bound, (off.item(), off_mean.item(), bound.item())
    # the running sum's share of it, 1.4e-8 of a logit for every 16 terms, is given back: three quarters of the bias at least
    assert off <= 0.25 * 1.4e-8 * H / 16 * (p * l).sum(1).mean() + 2.0 ** -22 * want.mean(), (off.item(), want.mean().item())


@pytest.mark.parametrize("channels", [[0, 1], [0, 4000], [5, 6, 7, 2048]])
def test_channels_anywhere(channels):
    # the two channels in one product step or in two, among zeros of both signs
    x, w, t = problem(7168, torch.arange(1.0, 17.0), 1.0)
    xs, ws = torch.zeros_like(x), torch.zeros_like(w)
    xs[:, ::2] = -0.0
    xs[:, channels[-2:]], ws[:, channels[-2:]] = x[:, :2], w[:, :2]
    check(xs, ws, t, "mean", "whole")
    check(xs, ws, t, "none", "columns")
