"""Every length of the list of likeliest tokens, for many rows of few classes: up to eight in one pass, stored side by side, and more in several."""
import pytest
import torch

from test_gpu_log_probs import check, make_logits, some_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


@pytest.mark.parametrize("layout", ["rows", "padded", "columns", "spread"])
@pytest.mark.parametrize("top", [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 15, 16, 17])
def test_many_rows_of_every_top(arb, top, layout):
    gen = torch.Generator().manual_seed(top)
    n, vocab = 11_000, 17
    for dtype, kind in ((torch.float32, "normal"), (torch.bfloat16, "ties"), (torch.float16, "masked")):
        check(arb, make_logits(gen, n, vocab, kind, dtype), some_tokens(gen, n, vocab), layout, scale=0.9, top=top, h=False)
