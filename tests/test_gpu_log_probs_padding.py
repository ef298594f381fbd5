"""Gradients of rows that stand for nothing: without a token, and without a part in the entropy's, they are 0 whatever their logits hold."""
import pytest
import torch

from test_gpu_log_probs import TYPES, Held, Want, close, make_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["rows", "padded", "columns", "spread"])
@pytest.mark.parametrize("n,vocab", [(9, 1), (12, 7), (70, 10), (7, 300), (5, 5000), (300, 129)])
def test_rows_of_padding_hold_anything(arb, n, vocab, layout, dtype):
    gen = torch.Generator().manual_seed(n + vocab)
    x = make_logits(gen, n, vocab, "normal", TYPES[dtype])
    tokens = torch.randint(0, vocab, (n,), generator=gen)
    none = torch.arange(n) % 3 == 1
    tokens[none] = -1
    for row, bad in zip(none.nonzero()[:, 0].tolist(), [float("nan"), float("inf"), float("-inf")] * n):
        x[row, row % vocab:] = bad
    w, h = torch.randn(n, generator=gen), torch.randn(n, generator=gen)
    fine = Want(x[~none], tokens[~none], 1.0, vocab + 64)
    for entropy in (None, torch.where(none, 0.0, h)):
        held = Held(arb, x, tokens, layout).forward()
        assert (held.log_probs.cpu()[none] == 0).all()
        for in_place in (False, True):
            got = held.backward(w, entropy, in_place=in_place)
            assert (got[none] == 0).all()
            close(got[~none], *fine.grad(w[~none], None if entropy is None else h[~none], x.dtype), "gradient")
    # with a part in the entropy's they say what they hold
    held = Held(arb, x, tokens, layout).forward()
    got = held.backward(w, h)
    broken = none & ~torch.isfinite(held.entropy.cpu()[:n])
    assert broken.any() and torch.isnan(got[broken]).all() and torch.isfinite(got[~none]).all()
