"""Which calls are refused because an output meets another place of the call, and which are not because it lies between the rows of one: host code only (the calls
that are not refused end at the device, which is not there)."""
import itertools
import random

import pytest

from test_model_operators_refusals import A, keep, layer, layer_grad, logits, logits_grad, read_back, refused


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() != 0:
        pytest.skip("addresses of nothing are for machines without a device")
    return arboretum_amd


def taken(arb, call, **change):
    refused(arb, call, "no HIP device", **change)


def at(row, column, strides, item=4):
    return (row * strides[0] + column * strides[1]) * item


# 4 rows of 100 classes, neither side by side: rows further apart than their classes span, or the other way round
SPREAD = [(200, 2), (300, 3), (2, 9), (3, 13)]


@pytest.mark.parametrize("strides", SPREAD)
def test_outputs_within_logits_that_lie_apart(arb, strides):
    where = dict(row_stride=strides[0], class_stride=strides[1], logits=2 * A)
    for row, column in ((0, 0), (2, 50), (3, 99)):
        place = 2 * A + at(row, column, strides)
        refused(arb, logits, "an output and an input overlap", **where, entropy=place)
        refused(arb, logits, "an output and an input overlap", **where, status=place)
        taken(arb, logits, **where, status=place + 4)  # (what lies between two classes)
        refused(arb, logits_grad, "an output and an input overlap", grad_logits=A, status=place, **where)
    taken(arb, logits, **where, entropy=2 * A + at(3, 99, strides) + 4)
    taken(arb, logits, **where, entropy=2 * A - 16)


@pytest.mark.parametrize("strides", SPREAD)
def test_gradients_within_logits_that_lie_apart(arb, strides):
    where = dict(row_stride=strides[0], class_stride=strides[1], logits=8 * A, grad_row_stride=strides[0], grad_class_stride=strides[1])
    elements = {at(i, j, strides) for i, j in itertools.product(range(4), range(100))}
    for row, column, more in itertools.product((0, 1, -1, 2, -3, 4), (1, 0, 7, 99, -99, 100), (0, 4)):
        by = at(row, column, strides) + more
        if by == 0:
            continue
        if any(e + by in elements for e in elements):
            refused(arb, logits_grad, "an output and an input overlap", grad_logits=8 * A + by, **where)
        else:
            taken(arb, logits_grad, grad_logits=8 * A + by, **where)
    taken(arb, logits_grad, grad_logits=8 * A, **where)  # (in their place)
    # of other strides they are taken to meet wherever their ends do
    refused(arb, logits_grad, "an output and an input overlap", grad_logits=8 * A + 4, **{**where, "grad_row_stride": 100, "grad_class_stride": 1})


def test_pieces_between_rows(arb):
    # one row, or a short array, in the room that another's rows leave
    taken(arb, layer, rows=1, out=3 * A + 16 * 4, w_stride=64)
    refused(arb, layer, "an output and an input overlap", rows=1, out=3 * A + 15 * 4, w_stride=64)
    refused(arb, layer, "an output and an input overlap", rows=1, out=3 * A + 41 * 4, w_stride=64)
    taken(arb, layer, rows=1, out=3 * A + 40 * 4 + 5 * 64 * 4, w_stride=64)
    refused(arb, layer, "an output and an input overlap", rows=2, out=3 * A + 16 * 4, out_stride=70, w_stride=64)
    taken(arb, logits, row_stride=104, entropy=2 * A + 400)
    refused(arb, logits, "an output and an input overlap", row_stride=103, entropy=2 * A + 400)
    taken(arb, logits_grad, grad_row_stride=104, stats=A + 416 + 400, n=2)
    taken(arb, keep, x_stride=200, scales=3 * A + 400, codes=3 * A + 800 + 400)
    taken(arb, read_back, x_stride=200, scales=A + 400, codes=A + 800 + 400)
    refused(arb, read_back, "an output and an input overlap", x_stride=200, scales=A + 400, codes=A + 800 + 402)
    taken(arb, layer_grad, grad_x=7 * A + 16 * 4, rows=1, w_stride=32)


def test_against_every_element(arb):
    """Small calls drawn at random: an answer of `meets` where elements do, and of `taken` where none do and strides are the same or one side is a single piece."""
    rng = random.Random(3)
    for _ in range(3000):
        n, vocab = rng.randint(1, 4), rng.randint(1, 5)
        inner, outer = rng.randint(1, 4), rng.randint(1, 24)
        strides = (outer, inner) if rng.random() < 0.5 else (inner, outer)
        rows_first = strides[0] >= (vocab - 1) * strides[1] + 1
        if not rows_first and strides[1] < (n - 1) * strides[0] + 1:
            continue  # (elements of the gradient share places)
        by = rng.randint(-60, 60)
        elements = {i * strides[0] + j * strides[1] for i, j in itertools.product(range(n), range(vocab))}
        where = dict(n=n, vocab=vocab, row_stride=strides[0], class_stride=strides[1], logits=8 * A)
        meets = any(e + by in elements for e in elements) and by != 0
        (refused if meets else taken)(*((arb, logits_grad) + (("an output and an input overlap",) if meets else ())), grad_logits=8 * A + 4 * by,
                                      grad_row_stride=strides[0], grad_class_stride=strides[1], **where)
        meets = any(by + k in elements for k in range(n))
        (refused if meets else taken)(*((arb, logits) + (("an output and an input overlap",) if meets else ())), entropy=8 * A + 4 * by, top=0, **where)
