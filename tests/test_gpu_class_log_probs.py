"""Log probabilities of a booster's classes: the booster's own path over log_probs, against the soft-max of its trees' sums in 64 bits.

The sums are those that predict() forms (the same walk), restated here as float32 additions in the order of the trees, so that they are equal bit by
bit; the bounds on what follows from them are those of the tests of log_probs with all classes in one thread: steps c = classes + 64."""
import numpy as np
import pytest
import torch

from test_gpu_log_probs import Want, close
from test_gpu_refine import make, walk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


def sums_of(model, X, classes, trees=None):
    """[rows][classes] float32, added tree by tree; trees of class k are k, k + classes, ..."""
    out = np.full((len(X), classes), np.float32(model.config["tree"].get("initial_y", 0.5)), np.float32)
    leaves = walk(model, X)
    for t in range(model.num_trees() if trees is None else trees):
        out[:, t % classes] += model.tree(t)["weights"][leaves[t]]
    return torch.from_numpy(out)


@pytest.mark.parametrize("classes,rows,rounds,top", [(2, 3000, 5, 2), (3, 3000, 7, 2), (10, 5003, 3, 3), (10, 200, 4, 10), (40, 1500, 2, 7)])
def test_against_the_soft_max_of_the_sums(arb, classes, rows, rounds, top):
    model, data, X, _, labels = make(arb, 3, rows=rows, rounds=rounds, classes=classes)
    got = model.log_probs(data, top=top)
    sums = sums_of(model, X, classes)
    want = Want(sums, torch.from_numpy(labels.astype(np.int64)), 1.0, classes + 64)
    close(torch.from_numpy(got["log_probs"]), want.log_prob, want.err_log_prob, "log_probs")
    close(torch.from_numpy(got["entropy"]), want.H, want.err_H, "entropy")
    order = want.top(top)
    assert np.array_equal(got["top"], order.numpy())
    log_p = want.log_p.gather(1, order)
    close(torch.from_numpy(got["top_log_probs"]), log_p, want.err_of(log_p, want.a.gather(1, order), want.err_L[:, None]), "top_log_probs")
    # and against the probabilities that predict() gives: float32 of the same sums' soft-max, off by half a step of it
    p = model.predict(data)
    assert np.allclose(np.exp(got["top_log_probs"].astype(np.float64)), np.take_along_axis(p, got["top"].astype(np.int64), 1), rtol=1e-5, atol=0)


def test_other_matrices_rounds_and_parts(arb):
    classes = 4
    model, data, X, _, labels = make(arb, 4, rows=2000, rounds=6, classes=classes, prebinned=False)
    plain = arb.DMatrix(X[:500])  # no labels
    got = model.log_probs(plain, top=1, of_labels=False)
    assert sorted(got) == ["entropy", "top", "top_log_probs"]
    full = model.log_probs(data, top=1)
    assert all(np.array_equal(got[k], full[k][:500]) for k in got)
    assert np.array_equal(got["top"][:, 0], np.argmax(model.predict(plain), 1))
    few = model.log_probs(data, n_rounds=2 * classes)
    want = Want(sums_of(model, X, classes, trees=2 * classes), torch.from_numpy(labels.astype(np.int64)), 1.0, classes + 64)
    close(torch.from_numpy(few["log_probs"]), want.log_prob, want.err_log_prob, "log_probs")
    with pytest.raises(arb.ArboretumError, match="labels are not set"):
        model.log_probs(plain)
    other = arb.DMatrix(X[:50], labels=np.full(50, classes, np.uint8))
    with pytest.raises(arb.ArboretumError, match="none of the booster's classes"):
        model.log_probs(other)
    # training goes on, and what was predicted stays what it was
    before = model.predict(data)
    model.log_probs(data, top=2)
    assert np.array_equal(model.predict(data), before)
    model.grow_tree()
    assert model.log_probs(data)["log_probs"].mean() > full["log_probs"].mean()
