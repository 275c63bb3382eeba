"""A rejected argument reaches Python as an exception that names the entry point and its code."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from optimus_lm_b200.ops import extension, functional as OF


def test_rejected_argument_raises():
    odd = torch.zeros(16 * 64 + 8, dtype=torch.bfloat16, device="cuda")[3:3 + 16 * 64].view(16, 64)
    rows = torch.zeros(16, device="cuda")
    with pytest.raises(RuntimeError, match="olb_ce_fwd failed with code -1"):
        extension().ce_fwd(odd, torch.zeros(16, dtype=torch.long, device="cuda"), rows, rows)
    with pytest.raises(RuntimeError, match="olb_gemm_bf16 failed with code -10"):
        OF.gemm(odd, odd, 16, 16, 64)


def test_linear_on_rows_off_the_vector_grid():
    store = torch.randn(16 * 64 + 8, device="cuda").to(torch.bfloat16)
    x = store[3:3 + 16 * 64].view(16, 64)
    w = torch.randn(32, 64, device="cuda").to(torch.bfloat16)
    assert torch.equal(OF.linear(x, w), OF.linear(x.clone(), w))
