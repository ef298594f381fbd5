"""What the tensor operators refuse, and the work memory they ask for: host code only, so nothing here reaches a GPU
(addresses are never followed: every call is refused before a kernel is launched)."""
import re

import numpy as np
import pytest

A = 1 << 20  # an address: 16-byte aligned, followed by nobody


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    return arboretum_amd


def lookup(arb, **k):
    a = dict(out=A, table=A, tokens=A, n=4, vocab=10, dim=8)
    a.update(k)
    arb.embedding(**a)


def sort(arb, **k):
    a = dict(keys=A, rows=A, tokens=A, n=4, vocab=10, work=A, work_bytes=1 << 20)
    a.update(k)
    arb.embedding_sort(**a)


def grad(arb, **k):
    a = dict(grad_table=A, grad_out=A, keys=A, rows=A, n=4, vocab=10, dim=8, work=A, work_bytes=1 << 20)
    a.update(k)
    arb.embedding_grad(**a)


def adamw(arb, **k):
    a = dict(params=[A], grads=[2 * A], exp_avgs=[3 * A], exp_avg_sqs=[4 * A], sizes=[100], step=1, lr=1e-3)
    a.update(k)
    arb.adamw(**a)


TOKENS = [
    (dict(n=-1), "bad row count"),
    (dict(bag=-1), "bad row count"),
    (dict(n=1 << 31), "below 2\\^31"),
    (dict(n=1 << 24, bag=1 << 7), "below 2\\^31"),
    (dict(vocab=0), "bad vocabulary"),
    (dict(vocab=1 << 31), "bad vocabulary"),
    (dict(token_bits=16), "32 or 64"),
    (dict(tokens=None), "null pointer"),
    (dict(tokens=A + 2), "not aligned"),
    (dict(tokens=A + 4, token_bits=64), "not aligned"),
    (dict(token_stride=-1), "bad token stride"),
    (dict(bag_stride=-4), "bad token stride"),
    (dict(status=A + 1), "not aligned"),
]


@pytest.mark.parametrize("change, says", TOKENS + [
    (dict(dtype="float64"), "element type"),
    (dict(dim=0), "bad dimension"),
    (dict(dim=1 << 24), "bad dimension"),
    (dict(out=None), "null pointer"),
    (dict(table=None), "null pointer"),
    (dict(out=A + 2), "not aligned"),
    (dict(table=A + 1, dtype="bfloat16"), "not aligned"),
    (dict(out_stride=7), "overlap"),
    (dict(table_stride=-8), "overlap"),
])
def test_embedding_refuses(arb, change, says):
    with pytest.raises(arb.ArboretumError, match=says):
        lookup(arb, **change)


@pytest.mark.parametrize("change, says", TOKENS + [
    (dict(keys=None), "null pointer"),
    (dict(rows=None), "null pointer"),
    (dict(work=None), "null pointer"),
    (dict(work=A + 8), "not aligned"),
    (dict(work_bytes=100), "too small"),
])
def test_embedding_sort_refuses(arb, change, says):
    with pytest.raises(arb.ArboretumError, match=says):
        sort(arb, **change)


@pytest.mark.parametrize("change, says", [
    (dict(n=-1), "bad row count"),
    (dict(n=1 << 24, bag=1 << 7), "below 2\\^31"),
    (dict(vocab=0), "bad vocabulary"),
    (dict(dim=0), "bad dimension"),
    (dict(dim=1 << 24), "bad dimension"),
    (dict(dtype="int8"), "element type"),
    (dict(dtype="bfloat16", grad_dtype="float16"), "float32 or of the type"),
    (dict(dtype="float32", grad_dtype="bfloat16"), "float32 or of the type"),
    (dict(grad_table=None), "null pointer"),
    (dict(grad_out=None), "null pointer"),
    (dict(keys=None), "null pointer"),
    (dict(work=None), "null pointer"),
    (dict(work=A + 4), "not aligned"),
    (dict(work_bytes=0), "too small"),
    (dict(table_stride=7), "overlap"),
    (dict(out_stride=-1), "overlap"),
    (dict(grad_table=A + 2), "not aligned"),
])
def test_embedding_grad_refuses(arb, change, says):
    with pytest.raises(arb.ArboretumError, match=says):
        grad(arb, **change)


@pytest.mark.parametrize("change, says", [
    (dict(step=0), "step counts from 1"),
    (dict(lr=-1.0), "must not be negative"),
    (dict(lr=float("nan")), "must not be negative"),
    (dict(lr=float("inf")), "finite"),
    (dict(eps=-1e-8), "must not be negative"),
    (dict(weight_decay=-0.1), "must not be negative"),
    (dict(grad_scale=float("nan")), "finite"),
    (dict(beta1=1.0), "in \\[0, 1\\)"),
    (dict(beta2=-0.1), "in \\[0, 1\\)"),
    (dict(beta2=float("nan")), "in \\[0, 1\\)"),
    (dict(sizes=[-1]), "bad tensor size"),
    (dict(sizes=[1 << 36]), "bad tensor size"),
    (dict(sizes=[100, 3]), "differ in length"),
    (dict(grads=[A, A]), "differ in length"),
    (dict(params=[0]), "null tensor"),
    (dict(exp_avg_sqs=[0]), "null tensor"),
    (dict(params=[A + 2]), "not aligned"),
    (dict(exp_avgs=[A + 2]), "not aligned"),
    (dict(grads=[A + 1], grad_dtype="bfloat16"), "not aligned"),
    (dict(exp_avgs=[A]), "overlap"),
    (dict(exp_avg_sqs=[3 * A]), "overlap"),
    (dict(dtype="float8"), "element type"),
    (dict(grad_dtype="float8"), "element type"),
    (dict(lr_device=A + 2), "not aligned"),
    (dict(step_device=A + 4), "not aligned"),
])
def test_adamw_refuses(arb, change, says):
    with pytest.raises(arb.ArboretumError, match=says):
        adamw(arb, **change)


@pytest.mark.parametrize("which", ["params", "exp_avgs", "exp_avg_sqs"])
@pytest.mark.parametrize("at", [[0, 0, 4096], [0, 396, 4096], [4096, 0, 396], [4096, 400, 0, 799], [8192, 4096, 0, 8192]])
def test_adamw_refuses_tensors_that_meet(arb, which, at):
    k = len(at)
    lists = {name: [(j + 2) * A + 65536 * i for i in range(k)] for j, name in
             enumerate(["params", "grads", "exp_avgs", "exp_avg_sqs"])}
    lists[which] = [20 * A + x for x in at]
    if 799 in at:
        lists[which][-1] = 20 * A + 796
    with pytest.raises(arb.ArboretumError, match="overlap"):
        adamw(arb, sizes=[100] * k, **lists)


def test_the_widest_row(arb):
    for call in (lookup, grad):
        with pytest.raises(arb.ArboretumError, match="bad dimension"):
            call(arb, dim=65_535 * 256 + 1)
        with pytest.raises(arb.ArboretumError, match="overlap"):  # of the right width, but too close to each other
            call(arb, dim=65_535 * 256, out_stride=-1 if call is grad else 5)


def test_nothing_to_do_is_no_error(arb):
    # no rows, no tokens, no tensors: nothing is launched
    sort(arb, n=0, keys=None, rows=None, tokens=None, work=None, work_bytes=0)
    sort(arb, bag=0, keys=None, rows=None, tokens=None, work=None, work_bytes=0)
    lookup(arb, n=0, out=None, tokens=None)
    adamw(arb, params=[], grads=[], exp_avgs=[], exp_avg_sqs=[], sizes=[])
    adamw(arb, params=[0], grads=[0], exp_avgs=[0], exp_avg_sqs=[0], sizes=[0])


def test_work_memory_grows_with_the_tokens(arb):
    assert arb.embedding_sort_bytes(0, 10) >= 0
    # pairs beside the caller's where there are two passes (vocabularies past 511)
    assert arb.embedding_sort_bytes(1 << 20, 100_000) >= 8 << 20
    assert arb.embedding_sort_bytes(1 << 20, 100) < 8 << 20
    assert arb.embedding_sort_bytes(1 << 10, 100_000, bag=1 << 10) == arb.embedding_sort_bytes(1 << 20, 100_000)
    assert arb.embedding_sort_bytes((1 << 31) - 1, 1 << 30) > 16 << 30  # no 32-bit overflow
    sizes = [arb.embedding_grad_bytes(n, 64) for n in (0, 1, 1000, 1_000_000, (1 << 31) - 1)]
    assert sizes == sorted(sizes)
    with pytest.raises(arb.ArboretumError):
        arb.embedding_sort_bytes(-1, 10)
    with pytest.raises(arb.ArboretumError):
        arb.embedding_grad_bytes(10, 0)


def test_without_a_gpu_the_operators_say_so(arb):
    if arb.device_count() > 0:
        pytest.skip("there is a GPU")
    for call in (lookup, sort, grad, adamw):
        with pytest.raises(arb.ArboretumError, match="no HIP device"):
            call(arb)


def test_leaf_tokens_and_refinement_refuse_before_any_walk(arb):
    data = arb.DMatrix(np.zeros((5, 3), np.float32), y=np.zeros(5))
    booster = arb.Garden({"objective": 0, "method": 1, "tree": {"max_depth": 3}}, data)
    says = "no trees" if arb.device_count() > 0 else "no HIP device"
    with pytest.raises(arb.ArboretumError, match=says):
        booster.leaf_tokens(data, A)
    with pytest.raises(arb.ArboretumError, match=says):
        booster.refine_leaves(data)
    with pytest.raises(arb.ArboretumError, match="token array or stride"):
        booster.leaf_tokens(data, A, stride=4)
    with pytest.raises(arb.ArboretumError, match="token array or stride"):
        booster.leaf_tokens(data, A, stride=-1)
    with pytest.raises(arb.ArboretumError, match="token array or stride"):
        booster.leaf_tokens(data, None)
    with pytest.raises(arb.ArboretumError, match="bad number of steps"):
        booster.refine_leaves(data, steps=-1)
    with pytest.raises(arb.ArboretumError, match="y is not set"):
        booster.refine_leaves(arb.DMatrix(np.zeros((5, 3), np.float32)))
    with pytest.raises(arb.ArboretumError, match="finite"):
        booster.refine_leaves(arb.DMatrix(np.zeros((5, 3), np.float32), y=np.full(5, np.inf)))
    with pytest.raises(arb.ArboretumError, match="no data matrix"):
        arb.Garden({"objective": 0}).refine_leaves()
    several = arb.Garden({"objective": 0, "tree": {"labels_count": 2}}, data)
    with pytest.raises(arb.ArboretumError, match="soft-max"):
        several.refine_leaves()


def test_every_operator_is_documented(arb):
    header = open(re.sub(r"arboretum_amd/__init__\.py$", "include/arboretum_ext.h", arb.__file__)).read()
    for name, symbol in [("embedding", "AEmbedding"), ("embedding_sort", "AEmbeddingSort"),
                         ("embedding_grad", "AEmbeddingGrad"), ("adamw", "AAdamW")]:
        assert getattr(arb, name).__doc__ and symbol in header
    assert np.dtype(np.uint64).itemsize == 8  # addresses travel as 64-bit words
