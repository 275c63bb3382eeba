"""The training program's switches for the loss without logits and the clipping over lists reach what they switch."""
import pytest
import torch

import dist_train


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
