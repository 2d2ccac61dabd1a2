"""dropout_rng is for the models that have a classifier with dropout."""

import pytest

from deepof_amd.config import Config
from deepof_amd.models import norm_kwargs


@pytest.mark.parametrize("model", ["flownets", "flownetc", "vgg16",
                                   "inception_v3"])
def test_models_without_a_classifier_refuse_its_generator(model):
    cfg = Config().apply_overrides([f"model={model}", "dropout_rng=counter"])
    with pytest.raises(ValueError, match="dropout_rng"):
        norm_kwargs(cfg)
    cfg = cfg.apply_overrides(["dropout_rng=torch"])
    assert "dropout_rng" not in norm_kwargs(cfg)


@pytest.mark.parametrize("model", ["st_single", "st_baseline"])
def test_classifiers_take_it(model):
    cfg = Config().apply_overrides([f"model={model}", "dropout_rng=counter"])
    assert norm_kwargs(cfg)["dropout_rng"] == "counter"


def test_training_refuses_it_before_it_begins(tmp_path):
    from deepof_amd.cli import main

    with pytest.raises(ValueError, match="dropout_rng"):
        main(["train", "--max-steps", "1", "dataset=synthetic", "device=cpu",
              "dropout_rng=counter", f"log_dir={tmp_path}", "run_name=r"])
