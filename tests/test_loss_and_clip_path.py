"""Training steps through the cross entropy from hidden states and the clipping over all gradients, together."""
import pytest
import torch

from optimus_lm_b200.engine import EngineArgs, TrainEngine

TINY = {"allenai/OLMoE-1B-7B-0924--L2-SH0.125-SA0.125-SE0.125-SC0.25-SI0.25": {},
        "allenai/OLMo-1B-hf--L2": dict(hidden_size=128, intermediate_size=256, num_attention_heads=2, num_key_value_heads=2),
        "meta-llama/Llama-3.2-1B--L2": dict(hidden_size=128, intermediate_size=256, num_attention_heads=2, num_key_value_heads=1, head_dim=64),
        "deepseek-ai/DeepSeek-V3--L3-DL1-N16-K2-MI64-A4-SE1-H128-I256": {}}


def engine(choice, dtype, **kw):
    over = dict(TINY[choice], vocab_size=1000, max_position_embeddings=128)
    return TrainEngine(EngineArgs(model_choice=choice, dtype=dtype, batch_size=2, context_size=64, optimizer="pt", warmup_steps=0,
                                  lr=1e-3, min_lr=1e-3, config_overrides=over, **kw))


def steps(choice, dtype, n, **kw):
    e = engine(choice, dtype, **kw)
    g = torch.Generator().manual_seed(7)
    tokens = torch.randint(0, 1000, (2, 64), generator=g)
    out = []
    for _ in range(n):
        o = e.train_step(tokens)
        out.append((float(o.loss), float(o.grad_norm)))
    return e, out


@pytest.mark.parametrize("choice", list(TINY))
def test_cpu_steps_match_the_logits_path(choice):
    if torch.cuda.is_available():
        pytest.skip("the engine picks the GPU")
    _, a = steps(choice, "fp32", 3)
    e, b = steps(choice, "fp32", 3, use_linear_cross_entropy=True, opt_use_list_clipping=True)
    assert e.model.use_linear_cross_entropy
    for (la, na), (lb, nb) in zip(a, b):
        assert la == pytest.approx(lb, rel=1e-5) and na == pytest.approx(nb, rel=1e-4)
    ids = torch.randint(0, 1000, (2, 64))
    assert e.model(ids, labels=ids).logits is None and e.model(ids).logits.shape == (2, 64, 1000)


@pytest.mark.gpu
@pytest.mark.parametrize("choice", list(TINY))
def test_gpu_steps(choice):
    base, a = steps(choice, "bf16", 1)
    e, b = steps(choice, "bf16", 1, use_linear_cross_entropy=True, opt_use_list_clipping=True)
    # the logits path rounds every logit to bf16 (|l| < 1 with these weights); both take the same gradients onwards
    assert a[0][0] == pytest.approx(b[0][0], abs=2.0 ** -8) and a[0][1] == pytest.approx(b[0][1], rel=0.02)
    assert e.check_device_status() == 0
    # after the clipping to 1 the gradients' norm is 1 up to their rounding
    ids = torch.randint(0, 1000, (2, 64), device="cuda")
    e.model(ids, labels=ids).loss.backward()
    grads = [p.grad for p in e.model.parameters() if p.grad is not None]
    from optimus_lm_b200.ops import functional as OF
    norm = OF.clip_grad_norm_(grads, 0.25)
    want = min(0.25, norm.item() * 1.0)
    assert OF.grad_norm(grads).item() == pytest.approx(want, rel=2.0 ** -8)


@pytest.mark.gpu
def test_gpu_flat_buffer_optimizer():
    # the head's gradient goes straight into the flat buffer of the framework's own optimizer
    choice = "allenai/OLMo-1B-hf--L2"
    out = {}
    for flag in (False, True):
        over = dict(TINY[choice], vocab_size=1000, max_position_embeddings=128)
        e = TrainEngine(EngineArgs(model_choice=choice, batch_size=2, context_size=64, optimizer="unsharded", warmup_steps=0,
                                   opt_grad_acc_steps=2, config_overrides=over, use_linear_cross_entropy=flag))
        tokens = torch.randint(0, 1000, (2, 64), generator=torch.Generator().manual_seed(7))
        e.forward_backward(e.stage_inputs(tokens))
        e.forward_backward(e.stage_inputs(tokens))
        out[flag] = e.model.lm_head.weight.grad.float().clone()
        assert e.check_device_status() == 0
    assert (out[True] - out[False]).norm() < 0.02 * out[False].norm()
