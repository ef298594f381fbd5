"""More calls that the tensor operators refuse, each of which would be answered wrongly: host code only, so nothing here
reaches a GPU (addresses are never followed: every call is refused before a kernel is launched)."""
import numpy as np
import pytest

from test_operators_host import A, adamw, grad, lookup, sort


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    return arboretum_amd


@pytest.mark.parametrize("eps", [0.0, 1e-50, 1e-46, 1e-39])
def test_adamw_refuses_an_eps_that_float32_does_not_hold(arb, eps):
    # an element whose gradient has always been 0, a table's row that no token names, would become 0 / 0
    with pytest.raises(arb.ArboretumError, match="eps must be at least 2\\^-126"):
        adamw(arb, eps=eps)


@pytest.mark.parametrize("change", [dict(lr=1e300), dict(lr=1e38), dict(lr=1e30, weight_decay=1e30), dict(eps=1e39), dict(grad_scale=-1e39),
                                    dict(grad_scale=1e300)])
def test_adamw_refuses_constants_beyond_float32(arb, change):
    # (1e38 / (1 - 0.9): the step's factor, which a moment of 0 would meet)
    with pytest.raises(arb.ArboretumError, match="beyond float32"):
        adamw(arb, **change)


def test_adamw_refuses_constants_beyond_float32_whatever_the_device_words_replace(arb):
    with pytest.raises(arb.ArboretumError, match="beyond float32"):
        adamw(arb, grad_scale=1e39, lr_device=A, step_device=A)
    with pytest.raises(arb.ArboretumError, match="eps must be at least"):
        adamw(arb, eps=0.0, lr_device=A, step_device=A)


# Sizes that a call's 32- or 64-bit words do not hold: what is left of them after dropping the upper bits would pass every check.
@pytest.mark.parametrize("call", ["embedding_sort_bytes", "embedding_grad_bytes"])
def test_work_memory_of_sizes_that_do_not_fit(arb, call):
    other = dict(vocab=10) if call == "embedding_sort_bytes" else dict(dim=8)
    for change in (dict(bag=2 ** 32 + 1), dict(bag=-2 ** 32 + 1), dict(n=2 ** 64 + 4), dict(n=-2 ** 64 + 4), {k: v + 2 ** 32 * (1 + 2 ** 32 * (k == "vocab")) for k, v in other.items()}):
        with pytest.raises(arb.ArboretumError, match="bits"):
            getattr(arb, call)(**{**dict(n=4), **other, **change})


@pytest.mark.parametrize("name,by", [("bag", 2 ** 32), ("dim", 2 ** 32), ("token_bits", 2 ** 32), ("dim", -2 ** 32), ("n", 2 ** 64), ("vocab", 2 ** 64),
                                     ("vocab", -2 ** 64), ("out_stride", 2 ** 64), ("table_stride", 2 ** 64), ("token_stride", 2 ** 64),
                                     ("bag_stride", 2 ** 64), ("bag_stride", -2 ** 65)])
def test_sizes_that_do_not_fit(arb, name, by):
    for call, takes in ((lookup, "bag dim token_bits n vocab out_stride table_stride token_stride bag_stride"),
                        (sort, "bag token_bits n vocab token_stride bag_stride"), (grad, "bag dim n vocab out_stride table_stride")):
        if name in takes.split():
            value = dict(bag=1, dim=8, token_bits=32, n=4, vocab=10, out_stride=8, table_stride=8, token_stride=1, bag_stride=1)[name]
            with pytest.raises(arb.ArboretumError, match="bits"):
                call(arb, **{name: value + by})


def test_steps_and_strides_that_do_not_fit(arb):
    with pytest.raises(arb.ArboretumError, match="64 bits"):
        adamw(arb, step=2 ** 64 + 1)
    data = arb.DMatrix(np.zeros((5, 3), np.float32), y=np.zeros(5))
    booster = arb.Garden({"objective": 0, "method": 1, "tree": {"max_depth": 3}}, data)
    with pytest.raises(arb.ArboretumError, match="32 bits"):
        booster.refine_leaves(steps=2 ** 32)
    with pytest.raises(arb.ArboretumError, match="64 bits"):
        booster.leaf_tokens(data, A, stride=2 ** 64 + 5)
    with pytest.raises(arb.ArboretumError, match="32 bits"):
        booster.leaf_tokens(data, A, n_rounds=2 ** 32 + 1)


def test_work_memory_of_less_than_nothing(arb):
    for call in (sort, grad):
        with pytest.raises(arb.ArboretumError, match="too small"):
            call(arb, work_bytes=-1)


@pytest.mark.parametrize("which", ["params", "grads", "exp_avgs", "exp_avg_sqs", "sizes"])
@pytest.mark.parametrize("value", [3.7, "100", 64.0, np.float32(8), None, [4]])
def test_adamw_refuses_lists_of_other_than_whole_numbers(arb, which, value):
    for values in ([value], np.array([value])):
        with pytest.raises(arb.ArboretumError, match="hold other than addresses and sizes"):
            adamw(arb, **{which: values})


def test_adamw_takes_lists_and_integer_arrays_alike(arb):
    # (refused for its step: after the lists)
    for kind in (list, tuple, lambda v: np.array(v, np.int64), lambda v: np.array(v, np.uint64), lambda v: [np.int64(x) for x in v],
                 lambda v: np.array(v, np.int64)[::-1][::-1]):
        lists = {name: kind([(k + 1) * A, (k + 9) * A]) for k, name in enumerate(["params", "grads", "exp_avgs", "exp_avg_sqs"])}
        with pytest.raises(arb.ArboretumError, match="step counts from 1"):
            adamw(arb, sizes=kind([100, 7]), step=0, **lists)
    with pytest.raises(arb.ArboretumError, match="step counts from 1"):
        adamw(arb, **{name: np.array([]) for name in ["params", "grads", "exp_avgs", "exp_avg_sqs", "sizes"]}, step=0)


NAMES = ["params", "grads", "exp_avgs", "exp_avg_sqs"]


def places():
    """Lists of three tensors that keep apart, 64 KB between two of them."""
    return {name: [(k + 2) * A + 65536 * i for i in range(3)] for k, name in enumerate(NAMES)}


# what is written must be apart from all else: the elements of two lists that meet would be read and written by two workgroups at once
@pytest.mark.parametrize("first,second", [(a, b) for a in NAMES for b in NAMES if a != b])
@pytest.mark.parametrize("i,j", [(0, 2), (2, 0), (1, 1)])
@pytest.mark.parametrize("by", [0, 4, 396, -396])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_adamw_refuses_tensors_of_two_lists_that_meet(arb, first, second, i, j, by, order):
    lists = places()
    lists[second][j] = lists[first][i] + by
    perm = {"rising": [0, 1, 2], "falling": [2, 1, 0], "mixed": [1, 0, 2]}[order]
    with pytest.raises(arb.ArboretumError, match="overlap"):
        adamw(arb, sizes=[100] * 3, **{name: [v[k] for k in perm] for name, v in lists.items()})


@pytest.mark.parametrize("order", [[0, 1, 2, 3], [3, 1, 0, 2], [3, 2, 1, 0]])
def test_adamw_takes_tensors_that_only_touch(arb, order):
    # parameter, gradient and states of one tensor after the other, back to back, in 16 and 32 bits; a tensor of no elements anywhere
    sizes, at, lists = [100, 7, 0, 31], 16 * A, {name: [] for name in NAMES}
    for size in sizes:
        for name, item in zip(NAMES, (2, 2, 4, 4)):
            at += -at % item
            lists[name].append(at)
            at += size * item
    lists["params"][2] = lists["exp_avgs"][0] + 4
    if arb.device_count() == 0:
        with pytest.raises(arb.ArboretumError, match="no HIP device"):
            adamw(arb, sizes=[sizes[k] for k in order], dtype="bfloat16", **{name: [v[k] for k in order] for name, v in lists.items()})


def test_adamw_takes_one_gradient_for_several_tensors(arb):
    # (gradients are only read)
    if arb.device_count() == 0:
        lists = places()
        lists["grads"] = [lists["grads"][0]] * 3
        with pytest.raises(arb.ArboretumError, match="no HIP device"):
            adamw(arb, sizes=[100] * 3, **lists)


def test_adamw_finds_one_meeting_among_many(arb):
    rng = np.random.default_rng(3)
    for trial in range(40):
        count = int(rng.integers(1, 400))
        sizes = rng.integers(0, 50, count)
        lists = {name: [] for name in NAMES}
        at = A
        slots = [(name, k) for name in NAMES for k in range(count)]
        if trial % 2:
            rng.shuffle(slots)
        for name, k in slots:
            lists[name] += [0] * (k + 1 - len(lists[name]))
            lists[name][k] = at
            at += 4 * int(sizes[k]) + 4 * int(rng.integers(0, 3))
        if arb.device_count() == 0 and sizes.any():
            with pytest.raises(arb.ArboretumError, match="no HIP device"):
                adamw(arb, sizes=sizes, **lists)
        if (sizes > 0).sum() < 2:
            continue
        one, other = rng.choice(np.flatnonzero(sizes > 0), 2, replace=False)
        a, b = rng.choice(NAMES, 2, replace=False)
        lists[a][one] = lists[b][other] + 4 * int(rng.integers(0, sizes[other]))
        with pytest.raises(arb.ArboretumError, match="overlap"):
            adamw(arb, sizes=sizes, **lists)
