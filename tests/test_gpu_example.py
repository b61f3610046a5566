"""The example runs the objectives together with the estimator."""
import importlib.util
import os

import pytest

from conftest import ROOT


@pytest.mark.gpu
def test_boost_from_preferences(cuda):
    path = os.path.join(ROOT, "examples", "boost_from_preferences.py")
    spec = importlib.util.spec_from_file_location("boost_from_preferences", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    out = example.main(contexts=1500, features=6, actions=3, pairs=12000, rounds=12, seed=1)
    assert abs(out["reward_loss_first"] - 0.6931472) < 1e-5     # log 2: every pair even
    assert out["reward_loss_last"] < out["reward_loss_first"]
    assert out["pair_agreement"] > 0.6
    assert out["policy_loss_last"] < out["policy_loss_first"]
    assert out["value_boosted"] > out["value_uniform"]
