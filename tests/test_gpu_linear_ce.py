"""Cross entropy from hidden states on the kernels, against the formula in 64 bits.

Bounds (u = 2^-8, half a step of bf16; u32 = 2^-23, a step of fp32: the tensor cores may truncate):
  logit      |dl| <= (H + 8) u32 sum_h |x w|                    H products summed in fp32
  loss row   |dloss| <= 2 max_v |dl| + 2^-18 (1 + |loss|)       softmax moves by at most the logits; exp, sums and log in
                                                                fp32 (at most 2^5 steps of it each)
  d_rv       = g (p - onehot); p is off by u p (its rounding), u p (the row factor's share of the target's rounding) and
             3 max|dl| p; the target's entry is off by 3 max|dl| |d| + u^2 |d|
  dx         u |dx| (its own rounding) + |d's error| |W|
  dw         u |dw| + |d's error|^T |X| + u |d|^T |X|           the scaled rows of X are rounded once
Gradients that go through an fp32 sum and a second bf16 rounding (several pieces, dx) have u |dx| twice.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

from optimus_lm_b200.ops import functional as OF

U, U32 = 2.0 ** -8, 2.0 ** -23


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert OF.check_status("cuda") == 0, "a kernel reported a timeout / overflow in the status word"


def make(T, H, V, *, seed=0, ignored=0.0, x_scale=1.0, w_scale=0.05, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    x = (torch.randn(T, H, device=device, generator=g) * x_scale).to(torch.bfloat16)
    w = (torch.randn(V, H, device=device, generator=g) * w_scale).to(torch.bfloat16)
    t = torch.randint(0, V, (T,), device=device, generator=g)
    if ignored:
        drop = torch.rand(T, device=device, generator=g) < ignored
        t = torch.where(drop, torch.tensor([-100, -1, V, V + 7], device=device)[torch.randint(0, 4, (T,), device=device, generator=g)], t)
    return x, w, t


def formula(x, w, t, reduction, row_grad=None):
    """(loss, dx, dw) and their bounds, in 64 bits."""
    xd, wd = x.detach().double(), w.detach().double()
    T, (V, H) = xd.shape[0], wd.shape
    live = (t >= 0) & (t < V)
    col = torch.where(live, t, torch.zeros_like(t))[:, None]
    xd = torch.where(live[:, None], xd, torch.zeros_like(xd))
    l = xd @ wd.t()
    lse = torch.logsumexp(l, 1)
    loss = torch.where(live, lse - l.gather(1, col)[:, 0], torch.zeros_like(lse))
    dl = (H + 8) * U32 * (xd.abs() @ wd.abs().t()).amax(1)
    loss_tol = torch.where(live, 2 * dl + 2.0 ** -18 * (1 + loss), torch.zeros_like(dl))
    n = int(live.sum())
    if reduction == "mean":
        g = torch.full((T,), 1.0 / max(n, 1), dtype=torch.float64, device=x.device)
    elif reduction == "sum":
        g = torch.ones(T, dtype=torch.float64, device=x.device)
    else:
        g = row_grad.double()
    g = torch.where(live, g, torch.zeros_like(g))[:, None]
    p = torch.exp(l - lse[:, None])
    onehot = torch.zeros_like(p).scatter_(1, col, 1.0)
    d = g * (p - onehot)
    # the target's entry: its own size, not p's, carries the error
    rel = 2 * U + 3 * dl[:, None] + 2.0 ** -18
    err = torch.where(onehot > 0, d.abs() * (3 * dl[:, None] + 2.0 ** -16 + U * U) + g.abs() * 3 * dl[:, None] * p, g.abs() * p * rel)
    dx, dw = d @ wd, d.t() @ xd
    sum_dx = 2 * (H + V) ** 0.5 * U32 * (d.abs() @ wd.abs())
    sum_dw = 2 * T ** 0.5 * U32 * (d.abs().t() @ xd.abs())
    bx = U * dx.abs() + err @ wd.abs() + sum_dx
    bw = U * dw.abs() + err.t() @ xd.abs() + U * (d.abs().t() @ xd.abs()) + sum_dw
    if reduction == "mean":
        out, tol = loss.sum() / n if n else torch.full((), float("nan")), loss_tol.sum() / max(n, 1)
    elif reduction == "sum":
        out, tol = loss.sum(), loss_tol.sum()
    else:
        out, tol = loss, loss_tol
    return out, dx, dw, tol, bx, bw


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    bad = off > bound * 1.01 + 1e-37
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} past their bound, worst {float((off / (bound + 1e-37)).max()):.2f} x"


# The three ways to keep the exponentials in bounds: all of them; 256 columns of the vocabulary at a time; pieces of the
# batch (of 256 rows and more), which the fp32 gradient of the weight must let through
WAYS = ["whole", "columns", "rows"]


def limit(way, w):
    return {"whole": {}, "columns": {"max_workspace": 1}, "rows": {"max_workspace": 4 * w.numel()}}[way]


def run_both(x, w, t, reduction, row_grad=None, **kw):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = OF.linear_cross_entropy(x, w, t, reduction=reduction, **kw)
    dx, dw = torch.autograd.grad(loss, (x, w), row_grad)
    assert loss.dtype == torch.float32 and dx.dtype == dw.dtype == torch.bfloat16
    return loss.detach(), dx, dw


def check(x, w, t, reduction, twice=False, **kw):
    row_grad = torch.rand(x.shape[0], device=x.device, generator=torch.Generator(device=x.device).manual_seed(5)) - 0.3 if reduction == "none" else None
    loss, dx, dw = run_both(x, w, t, reduction, row_grad, **kw)
    out, ex, ew, tol, bx, bw = formula(x, w, t, reduction, row_grad)
    assert ((loss.double() - out).abs() <= tol + 1e-37).all(), (loss, out)
    within(dx, ex, bx + (U * ex.abs() if twice else 0), "dx")
    within(dw, ew, bw, "dw")
    with torch.no_grad():
        scored = OF.linear_cross_entropy(x, w, t, reduction=reduction, **kw)
    assert ((scored.double() - out).abs() <= tol + 1e-37).all()


SIZES = [(1, 8, 1), (1, 64, 40), (2, 8, 2), (3, 72, 100), (31, 16, 63), (64, 512, 1000), (127, 128, 256), (128, 64, 257),
         (129, 200, 255), (130, 1000, 3001), (256, 256, 512), (257, 40, 65), (300, 264, 777), (513, 512, 1024),
         (700, 2048, 5000), (1100, 136, 300),
         # few rows: tiles of 224, 192, 160 and 96 columns
         (3, 16, 128256), (5, 64, 50304), (9, 24, 70001), (70, 40, 14001), (150, 16, 40000)]


@pytest.mark.parametrize("T,H,V", SIZES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_sizes(T, H, V, reduction):
    x, w, t = make(T, H, V, seed=T + H + V, ignored=0.3 if T > 2 else 0.0)
    check(x, w, t, reduction)


@pytest.mark.parametrize("T,H,V", [(700, 128, 300), (1025, 264, 777), (2000, 512, 130), (513, 72, 4001)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("way", ["columns", "rows"])
def test_pieces(T, H, V, reduction, way):
    x, w, t = make(T, H, V, seed=3, ignored=0.2)
    assert 2 * T * V > 4 * w.numel()
    check(x, w, t, reduction, twice=way == "rows", **limit(way, w))


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_logits_far_above_the_target(way, reduction):
    # rows whose target is 60 to 300 below their largest logit, between rows that are not: the flagged row blocks are
    # computed again; a target that is the largest by far, and one that is certain
    x, w, t = make(600, 128, 900, seed=9, w_scale=1.0)
    x[:] = x * 0.05
    rows = torch.tensor([0, 5, 130, 255, 256, 599], device="cuda")
    x[rows] = x[rows] * 100
    l = x.double() @ w.double().t()
    t[rows] = l[rows].argmin(1)
    x[300] = x[300] * 100
    t[300] = (x[300].double() @ w.double().t()).argmax()
    gap = (l[rows].amax(1) - l[rows].amin(1)).min()
    assert gap > 60
    check(x, w, t, reduction, twice=way == "rows", **limit(way, w))


def test_confident_rows():
    # 1 - p_target far below the rounding of p_target itself
    x, w, t = make(256, 64, 512, seed=2, w_scale=1.0)
    x = w[t].clone()
    x = (x.float() * torch.linspace(0.1, 0.6, 256, device="cuda")[:, None]).to(torch.bfloat16)
    check(x, w, t, "mean")
    check(x, w, t, "none")


@pytest.mark.parametrize("way", WAYS)
def test_no_targets_at_all(way):
    x, w, _ = make(300, 64, 100)
    kw = limit(way, w)
    t = torch.full((300,), -100, device="cuda")
    loss, dx, dw = run_both(x, w, t, "mean", **kw)
    assert loss.isnan() and not dx.any() and not dw.any()
    loss, dx, dw = run_both(x, w, t, "sum", **kw)
    assert loss == 0 and not dx.any() and not dw.any()


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_ignored_rows_may_hold_anything(way, reduction):
    x, w, t = make(400, 64, 300, seed=4)
    kw = limit(way, w)
    t[7], t[200], t[399] = -100, 300, -1
    for bad in (float("nan"), float("inf")):
        x[7], x[200, 3], x[399] = bad, bad, -bad
        check(x, w, t, reduction, twice=way == "rows", **kw)


@pytest.mark.parametrize("reduction,shape", [("mean", (0,)), ("sum", (0,)), ("none", (3, 0))])
def test_no_tokens(reduction, shape):
    x = torch.zeros(*shape, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(100, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    loss = OF.linear_cross_entropy(x, w, torch.zeros(shape, dtype=torch.long, device="cuda"), reduction)
    if reduction == "none":
        assert loss.shape == shape
    else:
        assert loss.isnan() if reduction == "mean" else loss == 0
    dx, dw = torch.autograd.grad(loss, (x, w), torch.zeros_like(loss))
    assert dx.shape == x.shape and not dw.any()


def test_shapes_strides_and_integer_types():
    x, w, t = make(6 * 40, 64, 300, seed=6, ignored=0.2)
    want = run_both(x, w, t, "mean")
    # a batch, every second position of a longer one, int32 targets, a weight inside a wider one, odd storage offsets
    wide = torch.zeros(6, 80, 64, device="cuda", dtype=torch.bfloat16)
    wide[:, ::2] = x.view(6, 40, 64)
    tw = torch.full((6, 80), 11, device="cuda", dtype=torch.int32)
    tw[:, ::2] = t.view(6, 40)
    got = run_both(wide[:, ::2], w, tw[:, ::2], "mean")
    store = torch.zeros(300, 96, device="cuda", dtype=torch.bfloat16)
    store[:, 8:72] = w
    got2 = run_both(x.view(6, 40, 64), store[:, 8:72], t.view(6, 40), "mean")
    odd = torch.zeros(300 * 64 + 3, device="cuda", dtype=torch.bfloat16)[3:].view(300, 64)
    odd.copy_(w)
    got3 = run_both(x, odd, t, "mean")
    got4 = run_both(x, w.t().contiguous().t(), t, "mean")
    for g in (got, got2, got3, got4):
        for a, b in zip(g, want):
            assert torch.equal(a.reshape(b.shape), b)
    losses = OF.linear_cross_entropy(x.view(6, 40, 64), w, t.view(6, 40), "none")
    assert losses.shape == (6, 40)
    one = OF.linear_cross_entropy(x[3], w, t[3], "none")
    assert one.shape == () and torch.allclose(one, losses.view(-1)[3], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_one_gradient_only_and_the_same_bits(way, reduction):
    x, w, t = make(520, 128, 1000, seed=8, ignored=0.1)
    kw = limit(way, w)
    g = torch.rand(520, device="cuda") if reduction == "none" else None
    _, dx, dw = run_both(x, w, t, reduction, g, **kw)
    _, dx2, dw2 = run_both(x, w, t, reduction, g, **kw)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    xg = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(OF.linear_cross_entropy(xg, w, t, reduction, **kw), xg, g)[0], dx)
    wg = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(OF.linear_cross_entropy(x, wg, t, reduction, **kw), wg, g)[0], dw)


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_backward_twice_and_scaled(way, reduction):
    x, w, t = make(520, 64, 200, seed=1)
    kw = limit(way, w)
    g = torch.rand(520, device="cuda") if reduction == "none" else None
    xg, wg = x.requires_grad_(), w.requires_grad_()
    loss = OF.linear_cross_entropy(xg, wg, t, reduction, **kw)
    first = torch.autograd.grad(loss, (xg, wg), g, retain_graph=True)
    second = torch.autograd.grad(loss, (xg, wg), g, retain_graph=True)
    quarter = torch.autograd.grad(loss, (xg, wg), g / 4 if g is not None else torch.tensor(0.25, device="cuda"))
    for a, b, c in zip(first, second, quarter):
        assert torch.equal(a, b)
        assert torch.equal((a.float() / 4).to(torch.bfloat16), c)  # a power of two moves no rounding
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, (xg, wg), g)


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_into_the_flat_gradient_buffer(way, reduction):
    x, w, t = make(520, 64, 200, seed=1)
    kw = limit(way, w)
    g = torch.ones(520, device="cuda") if reduction == "none" else None
    _, _, dw = run_both(x, w, t, reduction, g, **kw)
    w = torch.nn.Parameter(w)
    w.grad = torch.full_like(w, 7.0)  # stale: the first gradient overwrites it
    OF.enable_direct_grads([w])
    for _ in range(2):
        loss = OF.linear_cross_entropy(x, w, t, reduction, **kw)
        loss.backward(g)
    # the second one is added to the first's bf16 values in fp32 and rounded
    want = dw.float() + dw.float()
    assert ((w.grad.float() - want).abs() <= 2 * U * want.abs() + 2 * U * dw.float().abs() + 1e-30).all()


def test_shifted_matches_the_logits_path():
    B, S, H, V = 3, 130, 256, 1000
    x, w, _ = make(B * S, H, V, seed=12)
    labels = torch.randint(0, V, (B, S), device="cuda")
    labels[1, 40:60] = -100
    x = x.view(B, S, H)
    xa, wa = x.detach().requires_grad_(), w.detach().requires_grad_()
    new = OF.shifted_linear_cross_entropy(xa, wa, labels)
    new.backward()
    xb, wb = x.detach().requires_grad_(), w.detach().requires_grad_()
    old = OF.shifted_cross_entropy(OF.linear(xb, wb), labels)
    old.backward()
    # the old path rounds every logit (|l| < 4) to bf16: 2^-8 * 4 of each, softmax-weighted
    assert abs(new.item() - old.item()) < 2 * U * 4
    assert (xa.grad.float() - xb.grad.float()).norm() < 4 * U * xb.grad.float().norm()
    assert (wa.grad.float() - wb.grad.float()).norm() < 4 * U * wb.grad.float().norm()
    assert not xa.grad[:, -1].any()


def test_differences():
    x, w, t = make(40, 32, 50, seed=13, w_scale=0.3)
    loss, dx, dw = run_both(x, w, t, "sum")
    g = torch.Generator(device="cuda").manual_seed(1)
    for which, grad in (("x", dx), ("w", dw)):
        v = torch.randn(grad.shape, device="cuda", generator=g).double()
        def at(h):
            xx, ww = x.double(), w.double()
            xx, ww = (xx + h * v, ww) if which == "x" else (xx, ww + h * v)
            return torch.nn.functional.cross_entropy(xx @ ww.t(), t, reduction="sum")
        slope = (at(1e-5) - at(-1e-5)) / 2e-5
        got = (grad.double() * v).sum()
        assert (got - slope).abs() <= 4 * U * grad.double().norm() * 3


def test_streams_and_capture():
    x, w, t = make(300, 64, 500, seed=21)
    want = run_both(x, w, t, "mean")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_both(x, w, t, "mean")
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # forward and backward in two graphs with inputs that change between replays
    xs, ws, ts = x.clone().requires_grad_(), w.clone().requires_grad_(), t.clone()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for _ in range(2):
            loss = OF.linear_cross_entropy(xs, ws, ts)
            torch.autograd.grad(loss, (xs, ws))
        del loss
    torch.cuda.synchronize()
    ways = [limit(way, w) for way in WAYS]
    for kw in ways:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = OF.linear_cross_entropy(xs, ws, ts, **kw)
            dx, dw = torch.autograd.grad(loss, (xs, ws))
            loss = loss.detach()
        graphs.append(graph)
        outs.append((loss, dx, dw))
    for seed in (1, 2):
        x2, w2, t2 = make(300, 64, 500, seed=seed, ignored=0.1)
        with torch.no_grad():
            xs.copy_(x2), ws.copy_(w2), ts.copy_(t2)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (loss, dx, dw), kw in zip(outs, ways):
            for a, b in zip((loss, dx, dw), run_both(x2, w2, t2, "mean", **kw)):
                assert torch.equal(a, b)


def test_refusals():
    x, w, t = make(37, 16, 50)
    ok = dict(x=x, weight=w, targets=t)
    for change in (dict(reduction="median"), dict(weight=w[:, :8]), dict(weight=w[0]), dict(targets=t[:-1]), dict(targets=t.float()),
                   dict(targets=t > 3), dict(weight=w[:0]), dict(targets=t.view(1, -1)), dict(max_workspace=0),
                   dict(targets=t.cpu()), dict(weight=w.cpu())):
        with pytest.raises(ValueError):
            OF.linear_cross_entropy(**{**ok, **change})
    # what the kernels do not take goes the plain way
    for a, b in ((x.float(), w.float()), (x, w.float()), (x[:, :12], w[:, :12])):
        assert torch.isfinite(OF.linear_cross_entropy(a, b, t))


def test_once_differentiable():
    x, w, t = make(37, 16, 50)
    x.requires_grad_()
    loss = OF.linear_cross_entropy(x, w, t)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(loss, x, create_graph=True)


def test_many_rows_and_few_columns():
    # row blocks past the first band of tiles, and a vocabulary below one tile
    x, w, t = make(5000, 64, 50, seed=31, ignored=0.1)
    check(x, w, t, "mean")
    check(x, w, t, "none", max_workspace=1 << 18)


def test_exponentials_past_31_bits_of_elements():
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    T, H, V = 20000, 16, 128256   # 2.57e9 exponentials in one piece
    x, w, t = make(T, H, V, seed=2, w_scale=0.3)
    loss, dx, dw = run_both(x, w, t, "none", torch.ones(T, device="cuda"), max_workspace=8 << 30)
    rows = torch.cat([torch.arange(8), torch.arange(16738, 16746), torch.arange(T - 8, T)]).cuda()  # 2^31 falls into row 16743
    out, ex, _, tol, bx, _ = formula(x[rows], w, t[rows], "none", torch.ones(len(rows), device="cuda"))
    assert ((loss[rows].double() - out).abs() <= tol).all()
    within(dx[rows], ex, bx, "dx")
    cols = torch.cat([torch.arange(4), t[rows].cpu(), torch.tensor([V - 1])]).cuda()
    want, size = torch.zeros(len(cols), H, dtype=torch.float64, device="cuda"), torch.zeros(len(cols), H, dtype=torch.float64, device="cuda")
    for lo in range(0, T, 2000):
        xs, ts = x[lo:lo + 2000].double(), t[lo:lo + 2000]
        p = torch.softmax(xs @ w.double().t(), 1)[:, cols] - (ts[:, None] == cols).double()
        want += p.t() @ xs
        size += p.abs().t() @ xs.abs()
    assert ((dw[cols].double() - want).abs() <= U * want.abs() + 4 * U * size).all()


def test_more_rows_of_a_matrix_of_losses():
    x, w, t = make(4 * 50, 64, 300, seed=14, ignored=0.2)
    g = torch.rand(4, 50, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    xa, wa = x.detach().view(4, 50, 64).requires_grad_(), w.detach().requires_grad_()
    (OF.linear_cross_entropy(xa, wa, t.view(4, 50), "none") * g).sum().backward()
    _, dx, dw = run_both(x, w, t, "none", g.view(-1))
    assert torch.equal(xa.grad.view(200, 64), dx) and torch.equal(wa.grad, dw)
    # a gradient that is one number behind an expanded view
    xb, wb = x.detach().requires_grad_(), w.detach().requires_grad_()
    OF.linear_cross_entropy(xb, wb, t, "none").sum().backward()
    _, dx, dw = run_both(x, w, t, "sum")
    assert torch.equal(xb.grad, dx) and torch.equal(wb.grad, dw)


def test_two_streams_at_once():
    torch.cuda.synchronize()
    work = []
    for k in range(4):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            x, w, t = make(300 + 100 * k, 64, 500 + k, seed=40 + k)
            work.append((s, x, w, t, run_both(x, w, t, "mean")))
    torch.cuda.synchronize()
    for s, x, w, t, got in work:
        for a, b in zip(got, run_both(x, w, t, "mean")):
            assert torch.equal(a, b)


def test_status_word_read_between_forward_and_backward():
    x, w, t = make(64, 64, 100)
    x.requires_grad_()
    loss = OF.linear_cross_entropy(x, w, t)
    OF.status_word("cuda").zero_()
    assert torch.isfinite(torch.autograd.grad(loss, x)[0]).all()


@pytest.mark.parametrize("T,H,V", [(300, 1000, 3000), (512, 2048, 20000), (2500, 2048, 600), (1000, 256, 30), (40, 4096, 5000), (19000, 264, 100),
                                   (3000, 2304, 300)])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_products_whose_last_wave_is_split(T, H, V, reduction):
    # gradients of more, and of fewer, tiles than the GPU has processors, long in the vocabulary or in the batch
    x, w, t = make(T, H, V, seed=50, ignored=0.1)
    check(x, w, t, reduction)


def test_split_products_into_the_flat_gradient_buffer():
    x, w, t = make(6000, 264, 100, seed=51)
    _, _, dw = run_both(x, w, t, "mean")
    w = torch.nn.Parameter(w)
    w.grad = torch.zeros_like(w)
    OF.enable_direct_grads([w])
    for _ in range(2):
        OF.linear_cross_entropy(x, w, t).backward()
    want = dw.float() + dw.float()
    assert ((w.grad.float() - want).abs() <= 2 * U * want.abs() + 2 * U * dw.float().abs() + 1e-30).all()


@pytest.mark.parametrize("reduction,way", [("mean", "columns"), ("none", "columns"), ("mean", "rows")])
def test_memory_stays_in_bounds(reduction, way):
    T, H, V = 8192, 256, 20000   # exponentials of 328 MB
    x, w, t = make(T, H, V, seed=52)
    x.requires_grad_(), w.requires_grad_()
    bound = 4 * w.numel() - (way == "columns")   # with or without room for the fp32 gradient of the weight
    OF.linear_cross_entropy(x[:256], w, t[:256], "sum").backward()
    x.grad = w.grad = None
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    loss = OF.linear_cross_entropy(x, w, t, reduction, max_workspace=bound)
    torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
    torch.cuda.synchronize()
    peak = torch.cuda.max_memory_allocated() - held
    # the exponentials and (rows) the weight's fp32 gradient or (columns) the fp32 one of x, both gradients, scaled rows, and
    # what splits a product's last wave: at most 148 tiles of 128 x 256 in fp32 a part
    most = 2 * bound + 4 * x.numel() + 2 * (x.numel() * 2 + w.numel()) + 148 * 128 * 256 * 4 * 2 + (8 << 20)
    assert peak <= most < 2 * T * V, (peak, most)


@pytest.mark.parametrize("T,H,V", [(5, 64, 300), (300, 264, 777), (1100, 136, 301)])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_nothing_is_read_that_was_not_written(T, H, V, way, reduction):
    # workspaces come from memory that held NaN
    x, w, t = make(T, H, V, seed=60, ignored=0.2)
    g = torch.rand(T, device="cuda") if reduction == "none" else None
    want = run_both(x, w, t, reduction, g, **limit(way, w))
    sizes = [2 * T * V, 4 * V * H, 2 * V * H, 4 * T * H, 2 * T * H, 64 * T, 4 * T, 1 << 21, 1 << 24]
    for _ in range(2):
        poison = [torch.full((n // 4 + 64,), float("nan"), device="cuda") for n in sizes for _ in range(3)]
        torch.cuda.synchronize()
        del poison
        got = run_both(x, w, t, reduction, g, **limit(way, w))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
