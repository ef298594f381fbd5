"""Sums of long bags, and where bags are looked up another way."""
import pytest
import torch

from test_gpu_operators import MANY, TYPES, U, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


# A bag's tokens are summed four at a time, in pairs, and such a sum joins what came before: no element takes part in more
# than two additions of pairs, bag / 4 + 1 of what came before, and six where lanes share a bag; one rounding more for
# the scale.  So a sum is off by at most (bag / 4 + 12) u of the sum of magnitudes (a chain of additions: bag u).
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,bag,dim,columns", [(70_000, 200, 1, True), (70_000, 199, 3, True), (64, 200, 512, False), (64, 203, 1100, True),
                                               (5000, 200, 16, False), (3, 2001, 1, False), (MANY // 200 + 5, 200, 1, True)])
def test_small_numbers_behind_a_large_one_are_not_lost(arb, n, bag, dim, columns, dtype):
    # 1 and then half of the last place of 1, again and again: added one at a time, each would be rounded away
    T = TYPES[dtype]
    small = U / 2 if dtype == "float32" else U
    for first in (0, bag // 2, bag - 1):
        tokens = torch.ones((bag, n) if columns else (n, bag), dtype=torch.int32, device="cuda")
        tokens[first if columns else slice(None), slice(None) if columns else first] = 0
        table = torch.full((2, dim), small, device="cuda", dtype=T)
        table[0] = 1
        out = torch.empty(n, dim, device="cuda", dtype=T)
        arb.embedding(out.data_ptr(), table.data_ptr(), tokens.data_ptr(), n, 2, dim, bag=bag, dtype=dtype,
                      token_stride=1 if columns else bag, bag_stride=n if columns else 1)
        want = torch.full((n, dim), 1 + (bag - 1) * small, dtype=torch.float64)
        within(out, want, (bag / 4 + 12) * U * want, T)


# both sides of 512 MB of tokens, and of 2^19 bags, from which on columns of scalars are read four bags a thread
@pytest.mark.parametrize("n,bag,bits", [((1 << 19) - 1, 129, 64), (1 << 19, 128, 64), ((1 << 19) + 1, 127, 64), (1 << 19, 127, 64),
                                        ((1 << 19) - 1, 257, 32), ((1 << 19) + 3, 256, 32), (1 << 19, 255, 32), ((1 << 26) + 5, 2, 32)])
def test_columns_of_scalars_on_both_sides_of_the_rule(arb, n, bag, bits):
    vocab, scale = 999, 1.5
    gen = torch.Generator(device="cuda").manual_seed(bag + bits)
    table = torch.randn(vocab, 1, generator=gen, device="cuda")
    tokens = torch.randint(-1, vocab, (bag, n), generator=gen, device="cuda", dtype=torch.int32 if bits == 32 else torch.int64)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((n + 1,), 7.0, device="cuda")
    arb.embedding(out.data_ptr(), table.data_ptr(), tokens.data_ptr(), n, vocab, 1, bag=bag, scale=scale, token_bits=bits, token_stride=1,
                  bag_stride=n, status=status.data_ptr())
    held = torch.cat([table.double() * scale, torch.zeros(1, 1, dtype=torch.float64, device="cuda")])[:, 0]
    want, mag = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2))
    for one in tokens:
        x = held[one.long()]  # (-1: the zero at the end)
        want += x
        mag += x.abs()
    within(out[:n], want.cpu(), (bag / 4 + 12) * U * mag.cpu(), torch.float32)
    assert out[n].item() == 7.0 and status.item() == 0
