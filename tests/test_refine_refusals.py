"""Boosters whose leaves cannot be refined: refused before any GPU is looked for."""
import json

import numpy as np
import pytest


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    return arboretum_amd


def model_text(trees, **tree):
    """A model of `trees` trees of two leaves each, over one feature."""
    one = {"depth": 2, "weights": [0.25, -0.5], "nodes": [
        {"id": 0, "leaf": False, "left": 1, "right": 2, "threshold": 0.5, "fid": 0},
        {"id": 1, "leaf": True, "idx": 0}, {"id": 2, "leaf": True, "idx": 1}]}
    return json.dumps({"configuration": {"objective": tree.pop("objective", 4), "method": 1, "tree": dict(max_depth=1, **tree)},
                       "model": [one] * trees})


def rows(arb, labels):
    return arb.DMatrix(np.linspace(0, 1, len(labels), dtype=np.float32)[:, None], labels=np.array(labels, np.uint8))


@pytest.mark.parametrize("trees,classes", [(6, 3), (1, 2), (7, 3)])
def test_loaded_trees_of_several_classes(arb, trees, classes):
    # a model's text does not say which class a tree is of: loaded, all of them stand for the first
    booster = arb.load(model_text(trees, labels_count=classes))
    before = [booster.tree(t)["weights"].copy() for t in range(trees)]
    with pytest.raises(arb.ArboretumError, match="as many trees of each class"):
        booster.refine_leaves(rows(arb, [0, 1, 0, 1]))
    assert all(np.array_equal(booster.tree(t)["weights"], w) for t, w in enumerate(before))


@pytest.mark.parametrize("objective", [3, 4])
def test_soft_max_of_one_class(arb, objective):
    booster = arb.load(model_text(2, objective=objective, labels_count=1))
    with pytest.raises(arb.ArboretumError, match="labels_count >= 2"):
        booster.refine_leaves(rows(arb, [0, 1, 0, 1]))


def test_a_largest_leaf_weight_below_0(arb):
    booster = arb.load(model_text(2, objective=0, labels_count=1, max_leaf_weight=-0.5))
    data = arb.DMatrix(np.zeros((4, 1), np.float32), y=np.zeros(4, np.float32))
    with pytest.raises(arb.ArboretumError, match="max_leaf_weight must not be negative"):
        booster.refine_leaves(data)
