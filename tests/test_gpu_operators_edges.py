"""Sums of long bags, where bags are looked up another way, and the edges of the sort's digits and launches."""
import pytest
import torch

from test_gpu_operators import MANY, TYPES, Sorted, U, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


# A bag's tokens are summed eight at a time (rows of 16 bits: four) before such a sum joins what came before; columns of scalars in fours, and
# four of these.  No element takes part in more than four additions within, bag / 8 + 1 (bag / 4 + 1) of what came before, six where lanes share
# a bag, and two roundings at the end: a sum is off by at most (bag / 8 + 14) u of the sum of magnitudes, or bag / 4 + 14 (a
# chain of additions: bag u).
def additions(bag, dtype):
    return bag / (8 if dtype == "float32" else 4) + 14


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,bag,dim,columns", [(70_000, 200, 1, True), (70_000, 199, 3, True), (64, 200, 512, False), (64, 203, 1100, True),
                                               (5000, 200, 16, False), (3, 2001, 1, False), (MANY // 200 + 5, 200, 1, True)])
def test_small_numbers_behind_a_large_one_are_not_lost(arb, n, bag, dim, columns, dtype):
    # 1 and then less than half of the last place of 1, again and again: added one at a time, each would be rounded away
    T = TYPES[dtype]
    for first, small in ((0, U / 2), (0, U / 4), (0, U / 8), (bag // 2, U / 4), (bag - 1, U / 4)):
        tokens = torch.ones((bag, n) if columns else (n, bag), dtype=torch.int32, device="cuda")
        tokens[first if columns else slice(None), slice(None) if columns else first] = 0
        table = torch.full((2, dim), small, device="cuda", dtype=T)
        table[0] = 1
        out = torch.empty(n, dim, device="cuda", dtype=T)
        arb.embedding(out.data_ptr(), table.data_ptr(), tokens.data_ptr(), n, 2, dim, bag=bag, dtype=dtype,
                      token_stride=1 if columns else bag, bag_stride=n if columns else 1)
        want = torch.full((n, dim), 1 + (bag - 1) * small, dtype=torch.float64)
        within(out, want, additions(bag, dtype) * U * want, T)


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
    within(out[:n], want.cpu(), additions(bag, "float32") * U * mag.cpu(), torch.float32)
    assert out[n].item() == 7.0 and status.item() == 0


def check_sort_and_gradient(arb, tokens, vocab, bits, columns):
    """Tokens [n][bag]: the sorted pairs, twice, and the gradient of whole numbers, which float32 sums exactly."""
    n, bag = tokens.shape
    held = (tokens.t() if columns else tokens).to(torch.int32 if bits == 32 else torch.int64).contiguous()
    s = Sorted(arb, held, n, bag, vocab, (1, n) if columns else (bag, 1), bits=bits)
    key = torch.where((tokens >= 0) & (tokens < vocab), tokens, vocab).reshape(-1)
    assert torch.equal(s.keys.long(), key.sort().values)
    pair = key * n + torch.arange(n, device="cuda").repeat_interleave(bag)
    assert torch.equal((s.keys.long() * n + s.rows.long()).sort().values, pair.sort().values)
    first = s.pairs.clone()
    s.pairs.fill_(-7)
    s.work.fill_(0x5A)
    s.call()
    assert torch.equal(s.pairs, first)
    grad_out = ((torch.arange(n, device="cuda") % 7) - 3).float()[:, None]
    got = s.grad(grad_out, torch.full((vocab, 1), float("nan"), device="cuda"))
    want = torch.zeros(vocab + 1, dtype=torch.float64, device="cuda").index_add_(0, key, grad_out[:, 0].double().repeat_interleave(bag))
    assert torch.equal(got[:, 0].double(), want[:-1])


def some_tokens(n, bag, vocab):
    """The first and the last token and none at all among others."""
    gen = torch.Generator(device="cuda").manual_seed(n + vocab)
    tokens = torch.randint(0, vocab, (n, bag), generator=gen, device="cuda")
    u = torch.rand(n, bag, generator=gen, device="cuda")
    tokens[u < 0.1] = -1
    tokens[(u > 0.1) & (u < 0.15)] = vocab - 1
    tokens[(u > 0.15) & (u < 0.2)] = 0
    return tokens


# Pairs of more than one launch, in one group of tiles (up to 262,144) and in several.  What stands for none has the key `vocab`: the largest that
# one and two digits of 9 bits hold, and the first that takes one digit more, or one bit more of each.
@pytest.mark.parametrize("vocab", [1, 255, 256, 511, 512, 262_143, 262_144, (1 << 27) - 1])
@pytest.mark.parametrize("n,bag,bits,columns", [(32_769, 1, 32, False), (40_001, 2, 64, True), (262_145, 1, 64, False), (99_991, 5, 32, True)])
def test_keys_at_the_edges_of_digits(arb, n, bag, bits, columns, vocab):
    check_sort_and_gradient(arb, some_tokens(n, bag, vocab), vocab, bits, columns)


# Pairs of one launch: where a thread takes another number of them, and where they no longer fit.
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("m", [1, 2, 63, 64, 65, 1023, 1024, 1025, 4096, 4097, 8191, 8192, 8193, 16_384, 16_385, 32_767, 32_768, 32_769])
def test_numbers_of_pairs_at_the_edges_of_launches(arb, m, bits):
    for vocab in (1, 255, 256, 511, 512, 65_535, 65_536, 50_021):
        check_sort_and_gradient(arb, some_tokens(m, 1, vocab), vocab, bits, False)


# Keys and places that together no longer fit a word of the single launch: 32,768 pairs of a vocabulary from 2^25 on take the other way.
@pytest.mark.parametrize("m,vocab", [(32_768, (1 << 25) - 1), (32_768, 1 << 25), (32_768, (1 << 25) + 255), (1024, (1 << 30) + 3), (3, (1 << 30) + 3), (2, (1 << 28) - 1)])
def test_words_of_keys_and_places_at_their_edge(arb, m, vocab):
    tokens = some_tokens(m, 1, vocab)
    held = tokens.to(torch.int32)
    s = Sorted(arb, held, m, 1, vocab, (1, 1))
    key = torch.where(tokens >= 0, tokens, vocab).reshape(-1)
    assert torch.equal(s.keys.long(), key.sort().values)
    assert torch.equal((s.keys.long() * m + s.rows.long()).sort().values, (key * m + torch.arange(m, device="cuda")).sort().values)
