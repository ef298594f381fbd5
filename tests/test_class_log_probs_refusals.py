"""Calls of Garden.log_probs that are refused: host code only."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    return arboretum_amd


def booster(arb, objective=3, classes=3, **tree):
    data = arb.DMatrix(np.zeros((5, 3), np.float32), labels=np.array([0, 1, 2, 0, 1]))
    return arb.Garden({"objective": objective, "method": 1, "tree": dict(max_depth=3, labels_count=classes, **tree)}, data), data


def test_boosters_that_have_no_classes(arb):
    for objective, classes in [(0, 1), (1, 1), (3, 1)]:
        model, data = booster(arb, objective, classes)
        with pytest.raises(arb.ArboretumError, match="need a soft-max objective of two classes or more"):
            model.log_probs(data)


def test_tops(arb):
    model, data = booster(arb)
    for top in (-1, 4, 1 << 30):
        with pytest.raises(arb.ArboretumError, match="top must be 0 to the number of classes"):
            model.log_probs(data, top=top)
    for change in (dict(top=1 << 32), dict(n_rounds=1 << 32)):
        with pytest.raises(arb.ArboretumError, match="32 bits"):
            model.log_probs(data, **change)


def test_matrices_without_labels(arb):
    model, _ = booster(arb)
    with pytest.raises(arb.ArboretumError, match="labels are not set"):
        model.log_probs(arb.DMatrix(np.zeros((5, 3), np.float32)))


def test_boosters_without_trees_and_loaded_ones(arb):
    model, data = booster(arb)
    with pytest.raises(arb.ArboretumError, match="no trees" if arb.device_count() else "no HIP device"):
        model.log_probs(data)
    tree = {"nodes": [{"id": 0, "leaf": False, "left": 1, "right": 2, "threshold": 0.5, "fid": 0}], "weights": [0.1, 0.2], "depth": 2}
    text = '{"configuration": %s, "model": [%s, %s, %s]}'
    import json
    loaded = arb.load(text % (json.dumps(model.config), *[json.dumps(tree)] * 3))
    with pytest.raises(arb.ArboretumError, match="as many trees of each class"):
        loaded.log_probs(data, of_labels=False)
