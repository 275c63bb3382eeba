"""The training program's switches for the loss without logits and the clipping over lists reach what they switch."""
from types import SimpleNamespace

import pytest

import dist_train
from optimus_lm_b200.engine import EngineArgs, TrainEngine, switches_without_effect


class Reached(Exception):
    pass


@pytest.mark.parametrize("given", [False, True])
def test_loss_switch_reaches_the_model(given, monkeypatch):
    seen = {}

    def build(*args, **kw):
        seen.update(kw)
        raise Reached

    monkeypatch.setattr(dist_train, "build_model", build)
    with pytest.raises(Reached):
        dist_train.main(["--model_choice", "allenai/OLMo-1B-hf--L2"] + ["--use_linear_cross_entropy"] * given)
    assert seen.get("use_linear_cross_entropy", False) is given


TINY = dict(hidden_size=64, intermediate_size=128, num_attention_heads=1, num_key_value_heads=1, vocab_size=200, max_position_embeddings=64)


@pytest.mark.parametrize("kw,names", [
    (dict(use_linear_cross_entropy=True, opt_use_list_clipping=True, optimizer="pt"), []),
    (dict(), []),
    (dict(use_linear_cross_entropy=True, use_hf_model=True, optimizer="pt"), ["use_linear_cross_entropy"]),
    (dict(opt_use_list_clipping=True, optimizer="unsharded"), ["opt_use_list_clipping"]),
    (dict(use_linear_cross_entropy=True, opt_use_list_clipping=True, use_hf_model=True, optimizer="unsharded"),
     ["use_linear_cross_entropy", "opt_use_list_clipping"])])
def test_switches_without_effect_are_named(kw, names, recwarn):
    TrainEngine(EngineArgs(model_choice="allenai/OLMo-1B-hf--L2", dtype="fp32", batch_size=1, context_size=32, config_overrides=TINY, **kw),
                device="cpu")
    got = [str(w.message) for w in recwarn if "has no effect" in str(w.message)]
    assert len(got) == len(names) and all(n in g for n, g in zip(names, got))


@pytest.mark.parametrize("pp,model_has_it,named", [(1, True, False), (2, True, True), (1, False, True)])
def test_loss_switch_with_pipeline_stages_and_tensor_parallelism(pp, model_has_it, named):
    # a model with a tensor-parallel head does not have it
    args = EngineArgs(use_linear_cross_entropy=True)
    got = switches_without_effect(args, SimpleNamespace(use_linear_cross_entropy=model_has_it), SimpleNamespace(pipeline_parallelism=pp))
    assert bool(got) is named
