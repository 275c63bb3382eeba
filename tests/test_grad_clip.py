"""Gradient norm and clipping on the plain path, and what the calls refuse."""
import math

import pytest
import torch

from optimus_lm_b200.ops import functional as OF


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_plain_path(norm_type, dtype):
    g = torch.Generator().manual_seed(0)
    grads = [torch.randn(5, 7, generator=g).to(dtype), torch.randn(0).to(dtype), torch.randn(11, generator=g).to(dtype)[::2]]
    before = [x.clone() for x in grads]
    want = torch.linalg.vector_norm(torch.cat([x.double().reshape(-1) for x in grads]), norm_type)
    assert torch.allclose(OF.grad_norm(grads, norm_type).double(), want, rtol=1e-6)
    norm = OF.clip_grad_norm_(grads, 0.5, norm_type)
    assert norm.dtype == torch.float32 and torch.allclose(norm.double(), want, rtol=1e-6)
    for a, b in zip(grads, before):
        assert torch.allclose(a.double(), b.double() * (0.5 / (want + 1e-6)), rtol=2.0 ** -8 if dtype == torch.bfloat16 else 1e-6)
    again = [x.clone() for x in grads]
    OF.clip_grad_norm_(iter(grads), 100.0, norm_type)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_single_tensor_and_empty():
    assert OF.grad_norm(torch.tensor([3.0, 4.0])).item() == 5
    assert OF.grad_norm([]).item() == 0 and OF.clip_grad_norm_([], 1.0).item() == 0
    assert OF.grad_norm([torch.zeros(0)]).item() == 0 and OF.clip_grad_norm_([torch.zeros(0)], 1.0).item() == 0


def test_refusals():
    g = [torch.ones(3)]
    for bad in (1, 3.0, -math.inf, "fro"):
        with pytest.raises(ValueError):
            OF.grad_norm(g, bad)
        with pytest.raises(ValueError):
            OF.clip_grad_norm_(g, 1.0, bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            OF.clip_grad_norm_(g, bad)
    with pytest.raises(ValueError):
        OF.grad_norm([torch.ones(3), torch.ones(3, device="meta")])
    assert torch.equal(g[0], torch.ones(3))


@pytest.mark.parametrize("bad", [[None], [torch.ones(3), None], [1.0], [torch.ones(3), [torch.ones(3)]]])
def test_only_tensors(bad):
    with pytest.raises(TypeError):
        OF.grad_norm(bad)
    with pytest.raises(TypeError):
        OF.clip_grad_norm_(bad, 1.0)
    assert not isinstance(bad[0], torch.Tensor) or torch.equal(bad[0], torch.ones(3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_shared_memory_is_refused_when_scaled(dtype):
    a = torch.ones(100, dtype=dtype)
    m = torch.ones(6, 8, dtype=dtype)
    for bad in ([a, a], [a[:60], a[50:]], [a, a[3:4]], [m.t(), m[2:3]], [torch.ones(1, dtype=dtype).expand(5)],
                [torch.ones(4, dtype=dtype).as_strided((2, 3), (1, 1))]):
        for norm_type in (2.0, math.inf):
            with pytest.raises(ValueError, match="share memory|more than once"):
                OF.clip_grad_norm_(bad, 0.5, norm_type)
    assert torch.equal(a, torch.ones_like(a)) and torch.equal(m, torch.ones_like(m))
    assert OF.grad_norm([a, a]).item() == pytest.approx(math.sqrt(200), rel=1e-6)   # reading twice is no harm
    # neighbours, interleaved pieces, empty ones and a transposed matrix do not share
    base = torch.ones(4, 12, dtype=dtype)
    norm = OF.clip_grad_norm_([a[:50], a[50:], base[:, :5], base[:, 5:], a[:0], a[:0], m.t()], 0.5)
    want = 0.5 / (norm.item() + 1e-6)
    for t in (a, base, m):
        assert torch.allclose(t.float(), torch.full_like(t, want).float(), rtol=2.0 ** -10)   # a step of fp16
    # a tensor that is not dense and one that lies over it hold the same values afterwards, scaled once
    v = torch.full((10,), 2.0, dtype=dtype)
    norm = OF.clip_grad_norm_([v, v[::3]], 1.0)
    assert torch.allclose(v.float(), torch.full((10,), 2 / (norm.item() + 1e-6)), rtol=2.0 ** -10)


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_complex_and_integer_types(norm_type):
    g = torch.Generator().manual_seed(2)
    grads = [torch.complex(torch.randn(7, generator=g), torch.randn(7, generator=g)), torch.randn(5, generator=g)]
    before = [x.clone() for x in grads]
    want = torch.linalg.vector_norm(torch.cat([x.abs().double() for x in grads]), norm_type)
    assert OF.grad_norm(grads, norm_type).item() == pytest.approx(want.item(), rel=1e-6)
    OF.clip_grad_norm_(grads, 0.5, norm_type)
    for a, b in zip(grads, before):
        assert torch.allclose(a, b * (0.5 / (want.item() + 1e-6)), rtol=1e-6)
    whole = [torch.tensor([3, 4]), torch.zeros(2)]
    assert OF.grad_norm(whole, norm_type).item() == (5 if norm_type == 2 else 4)
    with pytest.raises(TypeError, match="floating"):   # whole numbers cannot be scaled
        OF.clip_grad_norm_(whole, 0.5, norm_type)
    assert whole[0].tolist() == [3, 4]
