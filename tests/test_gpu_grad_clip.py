"""Gradient norm and clipping over lists of tensors, against the formula in 64 bits.

Bounds: the norm's squares are summed in fp32 over at most 8 elements (8 roundings of 2^-24 each, relative to the sum of
positive terms) and in fp64 beyond; the root halves that and the result is rounded once: 2^-24 (8 / 2 + 1) < 2^-21.  A
scaled element carries the norm's error, the fp32 factor's (two roundings) and product's, and its own rounding.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from optimus_lm_b200.ops import functional as OF

NORM = 2.0 ** -21


def random_list(sizes, *, seed=0, fp32_every=3, shift=True, scale=1.0, device="cuda"):
    """Pieces of two buffers that start anywhere, with sentinels between them."""
    g = torch.Generator(device=device).manual_seed(seed)
    room = sum(sizes) + 80 * len(sizes) + 64
    flats = {t: torch.full((room,), 7.0, dtype=t, device=device) for t in (torch.bfloat16, torch.float32)}
    at = {t: 1 for t in flats}
    grads = []
    for k, n in enumerate(sizes):
        t = torch.float32 if fp32_every and k % fp32_every == 0 else torch.bfloat16
        lo = at[t] + (k * 7) % 13 if shift else (at[t] + 63) // 64 * 64
        grads.append(flats[t][lo:lo + n])
        at[t] = lo + n + 1
        grads[-1].copy_(torch.randn(n, device=device, generator=g) * scale)
    return grads, flats


def exact_norm(grads, norm_type):
    if norm_type == math.inf:
        return max(g.double().abs().max().item() for g in grads if g.numel())
    return math.sqrt(math.fsum(g.double().square().sum().item() for g in grads))


def check_clip(grads, max_norm, norm_type, flats=None):
    before = [g.clone() for g in grads]
    flat_before = {t: f.clone() for t, f in (flats or {}).items()}
    want = exact_norm(grads, norm_type)
    assert abs(OF.grad_norm(grads, norm_type).item() - want) <= NORM * want
    for a, b in zip(grads, before):
        assert torch.equal(a, b)
    norm = OF.clip_grad_norm_(grads, max_norm, norm_type)
    assert norm.dtype == torch.float32 and norm.dim() == 0 and abs(norm.item() - want) <= NORM * want
    factor = min(1.0, max_norm / (want + 1e-6))
    for a, b in zip(grads, before):
        e = b.double() * factor
        u = (2.0 ** -8 if b.dtype == torch.bfloat16 else 2.0 ** -24) * 1.01
        if factor == 1.0:
            assert torch.equal(a, b)
        assert ((a.double() - e).abs() <= (u + NORM + 2.0 ** -22) * e.abs() + 1e-38).all()
    for t, f in (flats or {}).items():   # nothing outside the tensors was touched
        inside = torch.zeros(f.numel(), dtype=torch.bool, device=f.device)
        for g in grads:
            if g.dtype == t and g.numel():
                lo = (g.data_ptr() - f.data_ptr()) // f.element_size()
                inside[lo:lo + g.numel()] = True
        assert torch.equal(f[~inside], flat_before[t][~inside])


LISTS = {
    "one element": [1],
    "a few": [3, 1, 8, 7, 9, 15, 16, 17],
    "around a vector and a piece": [8191, 8192, 8193, 16383, 16384, 16385, 16391, 32768, 5],
    "with empty ones": [0, 5, 0, 0, 70000, 0],
    "small table full": [11] * 250,
    "one more": [11] * 251,
    "middle table full": [9] * 800,
    "and one more": [9] * 801,
    "large table full": [3] * 2040,
    "one more than that": [3] * 2041,
    "thousands": [1 + (k * 37) % 400 for k in range(5000)],
    "large": [3_000_001, 17, 2_500_000],
}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_lists(name, norm_type):
    grads, flats = random_list(LISTS[name], seed=len(name))
    want = exact_norm(grads, norm_type)
    check_clip(grads, 0.37 * want, norm_type, flats)
    check_clip(grads, 1e9, norm_type, flats)


def test_more_pieces_than_blocks():
    grads, flats = random_list([40_000_000, 9_000_003, 11], shift=True, fp32_every=2)
    check_clip(grads, 1.0, 2.0, flats)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [1e-25, 1e-20, 3e-16, 1e18, 1e25, 1e37])
def test_values_whose_squares_leave_fp32(dtype, value):
    grads = [torch.full((1000,), value, dtype=dtype, device="cuda"), torch.zeros(5000, dtype=dtype, device="cuda"),
             torch.full((7,), -value, dtype=dtype, device="cuda")]
    want = exact_norm(grads, 2.0)
    assert abs(OF.grad_norm(grads).item() - want) <= NORM * want
    assert OF.grad_norm(grads, math.inf).item() == grads[0][0].item()


def test_many_elements_do_not_drift():
    g = torch.full((1 << 28,), 1e-3, dtype=torch.bfloat16, device="cuda")
    want = g[0].double().item() * math.sqrt(1 << 28)
    assert abs(OF.grad_norm([g]).item() - want) <= NORM * want


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_not_finite(norm_type):
    grads = [torch.ones(1000, device="cuda"), torch.ones(333, device="cuda", dtype=torch.bfloat16)]
    grads[1][332] = float("inf")
    assert OF.grad_norm(grads, norm_type).item() == math.inf
    norm = OF.clip_grad_norm_(grads, 1.0, norm_type)
    assert norm.item() == math.inf and not grads[0].any() and grads[1][332].isnan() and not grads[1][:332].any()
    grads = [torch.ones(1000, device="cuda"), torch.full((3,), float("nan"), device="cuda")]
    norm = OF.clip_grad_norm_(grads, 1.0, norm_type)
    assert norm.isnan() and all(g.isnan().all() for g in grads)


def test_zero_norm_and_zero_limit():
    grads = [torch.zeros(1000, device="cuda")]
    assert OF.clip_grad_norm_(grads, 1.0).item() == 0 and not grads[0].any()
    grads = [torch.ones(1000, device="cuda", dtype=torch.bfloat16)]
    OF.clip_grad_norm_(grads, 0.0)
    assert not grads[0].any()


def test_layouts():
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(64, 96, device="cuda", generator=g)
    rows = torch.randn(40, 50, device="cuda", generator=g).to(torch.bfloat16)
    grads = [base[:, :32], base[:, 40:91], rows.t(), torch.randn(4, 6, 8, device="cuda", generator=g).permute(2, 0, 1),
             torch.randn(33, device="cuda", generator=g)[::2], torch.tensor(3.0, device="cuda")]
    untouched = base[:, 91:].clone(), base[:, 32:40].clone()
    check_clip(grads, 1.0, 2.0)
    assert torch.equal(base[:, 91:], untouched[0]) and torch.equal(base[:, 32:40], untouched[1])


def test_more_than_31_bits_of_elements():
    free, _ = torch.cuda.mem_get_info()
    if free < 12 << 30:
        pytest.skip("needs 12 GB of free device memory")
    n = (1 << 31) + 12345
    t = torch.zeros(n + 3, dtype=torch.bfloat16, device="cuda")[3:]
    marks = [0, (1 << 30) - 1, 1 << 30, (1 << 31) - 1, 1 << 31, n - 1]
    t[marks] = 2.0
    assert OF.clip_grad_norm_([t], 1.0).item() == pytest.approx(math.sqrt(24.0), rel=NORM)
    assert torch.equal(t[marks].float(), torch.full((6,), 2 / (math.sqrt(24.0) + 1e-6), device="cuda").to(torch.bfloat16).float())
    assert int((t != 0).sum()) == 6


def test_refusals_and_other_types():
    a = torch.ones(100, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        OF.clip_grad_norm_([a, a], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        OF.clip_grad_norm_([a[:60], a[50:]], 1.0)
    with pytest.raises(ValueError, match="more than once"):
        OF.clip_grad_norm_([torch.ones(1, device="cuda").expand(5)], 1.0)
    with pytest.raises(ValueError, match="different devices"):
        OF.grad_norm([a, torch.ones(3)])
    with pytest.raises(ValueError, match="sparse"):
        OF.grad_norm([a, torch.eye(3, device="cuda").to_sparse()])
    assert torch.equal(a, torch.ones_like(a))
    assert OF.grad_norm([a, a]).item() == pytest.approx(math.sqrt(200), rel=NORM)           # twice in a norm: counted twice
    assert OF.grad_norm([torch.ones(1, device="cuda").expand(25)]).item() == 5
    half = torch.full((16,), 3.0, device="cuda", dtype=torch.float16)
    assert OF.clip_grad_norm_([half, a], 1.0).item() == pytest.approx(math.sqrt(144 + 100), rel=1e-6)
    assert half[0].item() == pytest.approx(3 / math.sqrt(244), rel=2e-3)


def test_same_bits_versions_streams_and_capture():
    grads, _ = random_list([1000, 70001, 33, 250000], seed=8)
    keep = [g.clone() for g in grads]
    a = OF.grad_norm(grads)
    assert all(torch.equal(a, OF.grad_norm(grads)) for _ in range(3))
    v = grads[0]._version
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = OF.clip_grad_norm_(grads, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and grads[0]._version > v
    want = [g.clone() for g in grads]
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n1 = OF.clip_grad_norm_(grads, 1.0)
    with torch.cuda.graph(graph2):
        n2 = OF.clip_grad_norm_(grads, 0.5)
    for _ in range(2):
        for g, k in zip(grads, keep):
            g.copy_(k)
        graph.replay()
        assert torch.equal(n1, a) and all(torch.equal(x, y) for x, y in zip(grads, want))
        graph2.replay()
        assert n2.item() == pytest.approx(1.0, rel=2 * 2.0 ** -8)
        assert OF.grad_norm(grads).item() == pytest.approx(0.5, rel=2 * 2.0 ** -8)


def test_two_calls_at_once():
    # two lists on two streams at the same time
    la, _ = random_list([900000, 17, 40000], seed=1)
    lb, _ = random_list([500000, 3, 80000], seed=2)
    wa, wb = exact_norm(la, 2.0), exact_norm(lb, 2.0)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, l in ((sa, la), (sb, lb)):
            with torch.cuda.stream(s):
                got.append(OF.grad_norm(l))
    torch.cuda.synchronize()
    for k, n in enumerate(got):
        w = wb if k % 2 else wa
        assert abs(n.item() - w) <= NORM * w


def test_norm_of_nothing_is_on_the_device():
    for dtype in (torch.float16, torch.bfloat16):
        empty = [torch.zeros(0, device="cuda", dtype=dtype)]
        assert OF.grad_norm(empty).device == OF.clip_grad_norm_(empty, 1.0).device == empty[0].device
