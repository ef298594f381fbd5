"""Embedding lookup, its gradient and AdamW on the GPU against plain restatements in 64 bits.

Bounds.  With u = 2^-24, a sum of k values formed in float32 in any order is off by at most k u sum|x| (to first order:
k - 1 additions, and k u < 0.01 in every case here), its product with a scale by u more, and the one rounding to a result's type T
by eps_T / 2 of the value, or by half the smallest subnormal step of T.  They are written with k + 3 in the place of k + 1 for
the second-order terms.  AdamW's bound is derived at its test."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


def half_step(dtype):
    """(relative, absolute) half of a step of the type."""
    info = torch.finfo(dtype)
    return info.eps / 2, info.smallest_normal * info.eps / 2


def make_tokens(gen, n, bag, vocab, kind, bits, columns):
    """Tokens [n][bag] on the CPU as int64, and their device copy with its strides."""
    if kind == "same":
        t = torch.full((n, bag), vocab - 1)
    elif kind == "none":
        t = torch.full((n, bag), -1)
    elif kind == "skewed":
        t = (torch.rand(n, bag, generator=gen) ** 6 * vocab).long().clamp(max=vocab - 1)
    else:
        t = torch.randint(0, vocab, (n, bag), generator=gen)
    if kind == "padded":
        t[torch.rand(n, bag, generator=gen) < 0.4] = -1
        t[: max(1, n // 10)] = -1  # whole bags of nothing
    held = (t.t().contiguous() if columns else t.contiguous()).to(torch.int32 if bits == 32 else torch.int64).cuda()
    return t, held, ((1, n) if columns else (bag, 1))


def lookup_64(table, tokens, scale):
    """(result, sum of |x| times |scale|)"""
    table = torch.cat([table.double(), torch.zeros(1, table.shape[1], dtype=torch.float64)])
    t = torch.where((tokens >= 0) & (tokens < len(table) - 1), tokens, len(table) - 1)
    out = torch.zeros(tokens.shape[0], table.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for j in range(tokens.shape[1]):
        out += table[t[:, j]]
        mag += table[t[:, j]].abs()
    return out * scale, mag * abs(scale)


def grad_64(grad_out, tokens, vocab, scale):
    """(result, sum of |x| times |scale|, terms)"""
    n, bag = tokens.shape
    t = torch.where((tokens >= 0) & (tokens < vocab), tokens, vocab).reshape(-1)
    rows = torch.arange(n).repeat_interleave(bag)
    out = torch.zeros(vocab + 1, grad_out.shape[1], dtype=torch.float64)
    out.index_add_(0, t, grad_out.double()[rows])
    mag = torch.zeros_like(out).index_add_(0, t, grad_out.double().abs()[rows])
    terms = torch.bincount(t, minlength=vocab + 1)[:, None].double()
    return out[:-1] * scale, mag[:-1] * abs(scale), terms[:-1]


def within(got, want, sum_error, dtype):
    rel, step = half_step(dtype)
    bound = sum_error + rel * (want.abs() + sum_error) + step
    off = (got.double().cpu() - want).abs()
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert worst <= 0, "off by %g more than the bound" % worst


class Sorted:
    """embedding_sort of device tokens."""

    def __init__(self, arb, held, n, bag, vocab, strides, status=None, bits=32, stream=None):
        self.pairs = torch.full((2, max(1, n * bag)), -7, dtype=torch.int32, device="cuda")
        size = arb.embedding_sort_bytes(n, vocab, bag=bag)
        self.work = torch.full((max(16, size),), 0xA5, dtype=torch.uint8, device="cuda")
        self.keys, self.rows = self.pairs[0], self.pairs[1]
        self.n, self.bag, self.vocab = n, bag, vocab
        self.arb = arb
        self.call = lambda stream=None: arb.embedding_sort(
            self.keys.data_ptr(), self.rows.data_ptr(), held.data_ptr(), n, vocab, self.work.data_ptr(), size, bag=bag,
            token_bits=bits, token_stride=strides[0], bag_stride=strides[1],
            status=None if status is None else status.data_ptr(), stream=stream)
        self.call(stream)

    def grad(self, grad_out, grad_table, scale=1.0, accumulate=False, stream=None, out_stride=None):
        dim = grad_out.shape[1]
        size = self.arb.embedding_grad_bytes(self.n, dim, bag=self.bag)
        self.grad_work = torch.full((max(16, size),), 0xA5, dtype=torch.uint8, device="cuda")
        name = {v: k for k, v in TYPES.items()}
        self.call_grad = lambda stream=None: self.arb.embedding_grad(
            grad_table.data_ptr(), grad_out.data_ptr(), self.keys.data_ptr(), self.rows.data_ptr(), self.n, self.vocab, dim,
            self.grad_work.data_ptr(), size, bag=self.bag, scale=scale, dtype=name[grad_out.dtype],
            grad_dtype=name[grad_table.dtype], accumulate=accumulate, table_stride=grad_table.stride(0),
            out_stride=grad_out.stride(0) if out_stride is None else out_stride, stream=stream)
        self.call_grad(stream)
        return grad_table


# n, bag, vocab, dim, tokens, bits, columns
SHAPES = [
    (1, 1, 1, 1, "any", 32, False),
    (1, 1, 7, 4096, "any", 64, False),
    (3, 1, 1000, 771, "any", 32, False),
    (64, 1, 511, 64, "any", 32, False),       # the largest key of one digit
    (65, 1, 512, 63, "padded", 32, False),    # ... and of two
    (257, 3, 1000, 65, "padded", 64, True),
    (1000, 7, 300, 5, "skewed", 32, True),
    (1000, 7, 300, 8, "skewed", 32, False),
    (4096, 1, 50021, 16, "any", 32, False),   # a whole tile of the sort
    (4097, 1, 262143, 3, "any", 32, False),   # one pair more, the largest key of two digits
    (5000, 1, 262144, 2, "any", 32, False),   # three digits
    (9000, 20, 5120, 1, "any", 32, True),     # leaf weights
    (9000, 20, 5120, 1, "padded", 32, False),
    (3000, 33, 77, 2, "same", 32, True),
    (20000, 1, 9, 31, "skewed", 32, False),
    (333, 5, 40, 260, "same", 32, False),
    (100, 4, 12, 129, "none", 32, False),
    (70001, 2, 3, 1, "skewed", 64, False),
    (30011, 4, 11, 12, "skewed", 32, True),
    (10, 200, 51200, 1, "any", 32, False),
    (0, 3, 10, 6, "any", 32, False),
    (6, 0, 10, 6, "any", 32, False),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,bag,vocab,dim,kind,bits,columns", SHAPES)
def test_lookup_and_gradient(arb, n, bag, vocab, dim, kind, bits, columns, dtype):
    gen = torch.Generator().manual_seed(n * 31 + bag * 7 + vocab + dim)
    tokens, held, strides = make_tokens(gen, n, bag, vocab, kind, bits, columns)
    T = TYPES[dtype]
    table = torch.randn(vocab, dim, generator=gen).to(T)
    scale = 1.7
    out = torch.full((n, dim), float("nan"), dtype=T, device="cuda")
    arb.embedding(out.data_ptr(), table.cuda().data_ptr(), held.data_ptr(), n, vocab, dim, bag=bag, scale=scale, dtype=dtype,
                  token_bits=bits, token_stride=strides[0], bag_stride=strides[1])
    scale = float(np.float32(scale))
    want, mag = lookup_64(table, tokens, scale)
    within(out, want, (bag + 3) * U * mag, T)

    s = Sorted(arb, held, n, bag, vocab, strides, bits=bits)
    m = n * bag
    keys, rows = s.keys[:m].cpu().long(), s.rows[:m].cpu().long()
    flat = torch.where(tokens >= 0, tokens, vocab).reshape(-1)
    assert torch.equal(keys, flat.sort().values)
    if m:  # every pair is there once
        all_pairs = flat * n + torch.arange(n).repeat_interleave(bag)
        assert torch.equal((keys * n + rows).sort().values, all_pairs.sort().values)
    grad_out = torch.randn(n, dim, generator=gen).to(T)
    want, mag, terms = grad_64(grad_out, tokens, vocab, scale)
    for O in {torch.float32, T}:
        got = s.grad(grad_out.cuda(), torch.full((vocab, dim), float("nan"), dtype=O, device="cuda"), scale=1.7)
        within(got, want, (terms + 3) * U * mag, O)
        again = s.grad(grad_out.cuda(), torch.full((vocab, dim), 5.0, dtype=O, device="cuda"), scale=1.7)
        assert torch.equal(got, again)  # no order of atomics decides a sum
        old = torch.randn(vocab, dim, generator=gen).to(O)
        got = s.grad(grad_out.cuda(), old.cuda(), scale=1.7, accumulate=True)
        total = want + old.double()
        within(got, total, (terms + 3) * U * mag + 2 * U * (want.abs() + old.double().abs()), O)
        untouched = terms[:, 0] == 0
        assert torch.equal(got.cpu()[untouched], old[untouched])


def test_gradient_is_the_difference_quotient_of_the_lookup(arb):
    # the lookup is linear in the table, so a quotient of any step is the derivative: with whole numbers and powers of two
    # both sides are exact
    gen = torch.Generator().manual_seed(5)
    n, bag, vocab, dim, scale = 50, 6, 30, 5, 0.5
    tokens, held, strides = make_tokens(gen, n, bag, vocab, "padded", 32, False)
    table = torch.randint(-8, 9, (vocab, dim), generator=gen).float()
    weight = torch.randint(-4, 5, (n, dim), generator=gen).float()

    def loss(t):
        out = torch.empty(n, dim, device="cuda")
        arb.embedding(out.data_ptr(), t.data_ptr(), held.data_ptr(), n, vocab, dim, bag=bag, scale=scale)
        return (out.cpu().double() * weight.double()).sum().item()

    grad = Sorted(arb, held, n, bag, vocab, strides).grad(weight.cuda(), torch.empty(vocab, dim, device="cuda"), scale=scale).cpu()
    for v, d in [(0, 0), (7, 4), (29, 2), (13, 1)]:
        up, down = table.clone(), table.clone()
        up[v, d] += 2
        down[v, d] -= 2
        assert (loss(up.cuda()) - loss(down.cuda())) / 4 == grad[v, d].item()


@pytest.mark.parametrize("bits", [32, 64])
def test_tokens_outside_the_table_are_reported_and_read_nothing(arb, bits):
    big = 2 ** 31 - 1 if bits == 32 else 2 ** 40
    n, vocab, dim = 6, 5, 8
    tokens = torch.tensor([0, 4, 5, -1, -2, big])[:, None]
    held = tokens.to(torch.int32 if bits == 32 else torch.int64).cuda()
    table = torch.arange(vocab * dim).reshape(vocab, dim).float()
    for use, want_status in [(6, 1), (2, 0)]:
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full((use, dim), 9.0, device="cuda")
        arb.embedding(out.data_ptr(), table.cuda().data_ptr(), held.data_ptr(), use, vocab, dim, token_bits=bits,
                      status=status.data_ptr())
        assert status.item() == want_status
        assert torch.equal(out.cpu().double(), lookup_64(table, tokens[:use], 1.0)[0])
        status.zero_()
        s = Sorted(arb, held, use, 1, vocab, (1, 1), status=status, bits=bits)
        assert status.item() == want_status
        assert s.keys.cpu().tolist() == ([0, 4, 5, 5, 5, 5] if use == 6 else [0, 4])
    # -1 alone is no error
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    Sorted(arb, torch.full((9,), -1, dtype=torch.int32, device="cuda"), 9, 1, 4, (1, 1), status=status)
    assert status.item() == 0


def test_pairs_that_are_not_of_a_sort_read_nothing_outside(arb):
    # keys and rows of a caller's making: rows outside grad_out add nothing, keys outside the table reach nothing
    n, vocab, dim = 4, 3, 5
    s = Sorted(arb, torch.tensor([0, 1, 1, 2], dtype=torch.int32, device="cuda"), n, 1, vocab, (1, 1))
    s.rows.copy_(torch.tensor([0, 4, 2, -1], dtype=torch.int32))
    s.keys.copy_(torch.tensor([0, 1, 1, 1000], dtype=torch.int32))
    g = torch.arange(n * dim).reshape(n, dim).float()
    got = s.grad(g.cuda(), torch.full((vocab, dim), 3.0, device="cuda")).cpu()
    assert torch.equal(got, torch.stack([g[0], g[2], torch.zeros(dim)]))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,pad,first", [(8, 0, 0), (8, 5, 1), (64, 3, 3), (771, 1, 1), (1, 2, 1), (16, 16, 0)])
def test_strides_and_starts_of_any_alignment(arb, dtype, dim, pad, first):
    # rows `dim + pad` apart, from element `first` on; what lies between the rows stays as it was
    T, n, bag, vocab = TYPES[dtype], 37, 3, 50
    gen = torch.Generator().manual_seed(dim + pad)
    tokens, held, strides = make_tokens(gen, n, bag, vocab, "padded", 32, False)
    width = dim + pad

    def spread(values, fill):
        buffer = torch.full((values.shape[0] * width + first,), fill, dtype=T)
        view = buffer[first:].reshape(-1, width)[:, :dim]
        view.copy_(values)
        buffer = buffer.cuda()
        return buffer, buffer[first:].reshape(-1, width)

    table = torch.randn(vocab, dim, generator=gen).to(T)
    _, wide_table = spread(table, float("nan"))
    out_buffer, wide_out = spread(torch.zeros(n, dim, dtype=T), 7.0)
    arb.embedding(wide_out.data_ptr(), wide_table.data_ptr(), held.data_ptr(), n, vocab, dim, bag=bag, dtype=dtype, out_stride=width,
                  table_stride=width)
    want, mag = lookup_64(table, tokens, 1.0)
    within(wide_out[:, :dim], want, (bag + 3) * U * mag, T)
    assert (wide_out[:, dim:] == 7).all() and (out_buffer[:first] == 7).all()

    grad_out = torch.randn(n, dim, generator=gen).to(T)
    _, wide_grad = spread(grad_out, float("nan"))
    s = Sorted(arb, held, n, bag, vocab, strides)
    into_buffer, into = spread(torch.zeros(vocab, dim, dtype=T), 7.0)
    s.grad(wide_grad[:, :dim], into[:, :dim])
    want, mag, terms = grad_64(grad_out, tokens, vocab, 1.0)
    within(into[:, :dim], want, (terms + 3) * U * mag, T)
    assert (into[:, dim:] == 7).all() and (into_buffer[:first] == 7).all()


def test_gradient_of_a_broadcast_output(arb):
    # every bag has the same gradient row: a stride of 0
    n, vocab, dim = 500, 20, 33
    gen = torch.Generator().manual_seed(1)
    tokens, held, strides = make_tokens(gen, n, 1, vocab, "any", 32, False)
    row = torch.randn(1, dim, generator=gen)
    got = Sorted(arb, held, n, 1, vocab, strides).grad(row.cuda(), torch.empty(vocab, dim, device="cuda"), out_stride=0)
    want, mag, terms = grad_64(row.expand(n, dim), tokens, vocab, 1.0)
    within(got, want, (terms + 3) * U * mag, torch.float32)


def test_infinities_and_nan_stay_in_their_rows(arb):
    n, vocab, dim = 8, 6, 70
    table = torch.ones(vocab, dim)
    table[1, 5], table[2, 6], table[3] = float("inf"), float("nan"), float("nan")
    tokens = torch.tensor([[0, 1], [0, 2], [0, -1], [-1, -1], [4, 5], [1, 1], [0, 0], [5, 5]])
    held = tokens.to(torch.int32).cuda()
    out = torch.empty(n, dim, device="cuda")
    arb.embedding(out.data_ptr(), table.cuda().data_ptr(), held.data_ptr(), n, vocab, dim, bag=2)
    want = lookup_64(table, tokens, 1.0)[0].float()
    assert torch.equal(out.cpu().nan_to_num(nan=77.0), want.nan_to_num(nan=77.0))  # (row 3 of the table is named by nobody)
    grad_out = torch.ones(n, dim)
    grad_out[3] = float("nan")  # a bag without tokens
    grad_out[4, 0] = float("-inf")
    got = Sorted(arb, held, n, 2, vocab, (2, 1)).grad(grad_out.cuda(), torch.empty(vocab, dim, device="cuda")).cpu()
    want = grad_64(torch.where(torch.isnan(grad_out), 0.0, grad_out), tokens, vocab, 1.0)[0].float()
    assert torch.equal(got, want)


def test_offsets_beyond_32_bits(arb):
    # a table of 2^31 and more elements, rows of its end and of its start
    vocab, dim = 33_000, 65_537
    table = torch.empty(vocab, dim, dtype=torch.bfloat16, device="cuda")
    named = torch.tensor([0, 1, 16_384, 32_767, 32_768, vocab - 1])
    for v in named.tolist():
        table[v] = (torch.arange(dim, device="cuda") + 7 * v) % 251
    out = torch.empty(len(named), dim, dtype=torch.bfloat16, device="cuda")
    held = named.to(torch.int32).cuda()
    arb.embedding(out.data_ptr(), table.data_ptr(), held.data_ptr(), len(named), vocab, dim, dtype="bfloat16")
    assert torch.equal(out, table[named.cuda()])
    grad = torch.full((vocab, dim), 3.0, dtype=torch.bfloat16, device="cuda")
    Sorted(arb, held, len(named), 1, vocab, (1, 1)).grad(out, grad)
    assert torch.equal(grad[named.cuda()], out)
    grad[named.cuda()] = 0
    assert not grad.any()


# ---- AdamW

def adamw_64(p, g, m, v, step, lr, beta1, beta2, eps, decay, grad_scale):
    """(p, m, v) and their bounds.  With u = 2^-24 for each operation and each constant rounded to float32: m takes two products, two constants,
    the product with grad_scale and one sum: 5 u of beta1 |m| + (1 - beta1) |g|.  v takes twice the error of g, and so on: 8 u of its value.  The step
    U = step_size m / (sqrt(v) / root + eps) carries m's error, half of v's, and six roundings and three constants: 13 u |U| beside
    step_size dm / denominator.  p: its product with a constant (2 u |p|) and the difference (u (|p| + |U|)), then its type's rounding."""
    g = float(np.float32(grad_scale)) * g.double()
    p, m, v = p.double(), m.double(), v.double()
    dm = 5 * U * (beta1 * m.abs() + (1 - beta1) * g.abs())
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    den = v.sqrt() / (1 - beta2 ** step) ** 0.5 + eps
    size = lr / (1 - beta1 ** step)
    upd = size * m / den
    new = p * (1 - lr * decay) - upd
    dp = size * dm / den + 13 * U * upd.abs() + 2 * U * p.abs() + U * (p.abs() + upd.abs())
    return (new, m, v), (1.01 * dp, 1.01 * dm, 1.01 * 8 * U * v)


def make_tensors(gen, sizes, dtype, grad_dtype, first=0):
    """Tensors packed back to back in one buffer each, from element `first` on."""
    total = sum(sizes) + first
    p = torch.randn(total, generator=gen).to(dtype)
    g = (torch.randn(total, generator=gen) * 0.1).to(grad_dtype)
    m = torch.randn(total, generator=gen) * 0.05
    v = torch.rand(total, generator=gen) * 0.01
    at = np.concatenate([[0], np.cumsum(sizes)[:-1]]).astype(np.int64) + first
    return p, g, m, v, at


HYPER = dict(beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.1, grad_scale=0.5)


def run_adamw(arb, tensors, at, sizes, step=3, lr=0.01, dtype="float32", grad_dtype=None, order=None, **more):
    lists = [t.data_ptr() + at * t.element_size() for t in tensors]
    sizes = np.asarray(sizes, np.int64)
    if order is not None:
        lists, sizes = [x[order] for x in lists], sizes[order]
    arb.adamw(*lists, sizes, step, lr, dtype=dtype, grad_dtype=grad_dtype, **{**HYPER, **more})


@pytest.mark.parametrize("grad_dtype", list(TYPES))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sizes,first", [([1], 0), ([1], 1), ([5, 3, 0, 1023], 1), ([8192, 8193, 1, 4], 0), ([100_003, 7], 3),
                                         ([17] * 300, 0), ([64] * 88, 0), ([64] * 89 + [20_000], 2)])
def test_adamw(arb, dtype, grad_dtype, sizes, first):
    gen = torch.Generator().manual_seed(len(sizes) + first)
    P, G = TYPES[dtype], TYPES[grad_dtype]
    *host, at = make_tensors(gen, sizes, P, G, first)
    dev = [t.cuda() for t in host]
    run_adamw(arb, dev, at, sizes, dtype=dtype, grad_dtype=grad_dtype)
    (p, m, v), (dp, dm, dv) = adamw_64(*host, 3, 0.01, 0.9, 0.99, 1e-6, 0.1, 0.5)
    within(dev[0][first:], p[first:], dp[first:], P)
    for got, want, bound in ((dev[2], m, dm), (dev[3], v, dv)):
        assert ((got.cpu().double() - want).abs()[first:] <= bound[first:] + 2.0 ** -149).all()
    for got, was in zip(dev, host):  # the gradients, and what is in front of the tensors
        assert torch.equal(got.cpu()[:first], was[:first])
    assert torch.equal(dev[1].cpu(), host[1])


def test_adamw_in_any_order_of_the_list_with_gaps_left_alone(arb):
    gen = torch.Generator().manual_seed(3)
    sizes = [33, 9000, 1, 250]
    *host, at = make_tensors(gen, [s + 5 for s in sizes], torch.float32, torch.float32)
    forth = [t.cuda() for t in host]
    run_adamw(arb, forth, at, sizes)
    back = [t.cuda() for t in host]
    run_adamw(arb, back, at, sizes, order=np.array([2, 0, 3, 1]))
    gap = torch.ones(len(host[0]), dtype=torch.bool)
    for a, s in zip(at, sizes):
        gap[a:a + s] = False
    for a, b, was in zip(forth, back, host):
        assert torch.equal(a, b)
        assert torch.equal(a.cpu()[gap], was[gap])
    assert not torch.equal(forth[0].cpu()[~gap], host[0][~gap])


def test_adamw_first_step_and_plain_cases(arb):
    # from zero states the first step moves by lr against the sign of the gradient, less eps; a zero gradient moves nothing
    g = torch.tensor([0.5, -2.0, 0.0, 1e-3])
    p = torch.zeros(4, device="cuda")
    m, v = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    arb.adamw([p.data_ptr()], [g.cuda().data_ptr()], [m.data_ptr()], [v.data_ptr()], [4], 1, 0.25, weight_decay=0.0, eps=1e-12)
    assert torch.allclose(p.cpu(), -0.25 * g.sign(), rtol=1e-5, atol=0)
    # weight decay alone
    p = torch.tensor([1.0, -2.0], device="cuda")
    z = [torch.zeros(2, device="cuda") for _ in range(3)]
    arb.adamw([p.data_ptr()], [z[0].data_ptr()], [z[1].data_ptr()], [z[2].data_ptr()], [2], 1, 0.5, weight_decay=0.5)
    assert p.cpu().tolist() == [0.75, -1.5]


def test_adamw_passes_infinities_on(arb):
    p = torch.ones(5, device="cuda")
    g = torch.tensor([1.0, float("nan"), float("inf"), 0.0, 1.0], device="cuda")
    m, v = torch.zeros(5, device="cuda"), torch.zeros(5, device="cuda")
    arb.adamw([p.data_ptr()], [g.data_ptr()], [m.data_ptr()], [v.data_ptr()], [5], 1, 0.1)
    assert torch.isfinite(p).cpu().tolist() == [True, False, False, True, True]


def test_adamw_reads_step_and_rate_from_the_device(arb):
    gen = torch.Generator().manual_seed(9)
    sizes = [9000, 55]
    *host, at = make_tensors(gen, sizes, torch.float32, torch.float32)
    for step, lr in [(1, 0.5), (7, 0.01), (100_000, 1e-4)]:
        lr = float(np.float32(lr))
        a, b, c = ([t.cuda() for t in host] for _ in range(3))
        step_d, lr_d = torch.tensor([step], device="cuda"), torch.tensor([lr], device="cuda")
        run_adamw(arb, a, at, sizes, step=step, lr=lr)
        run_adamw(arb, b, at, sizes, step=1, lr=9.0, step_device=step_d.data_ptr(), lr_device=lr_d.data_ptr())
        run_adamw(arb, c, at, sizes, step=1, lr=lr, step_device=step_d.data_ptr())
        # (powers in 64 bits on the host and on the GPU may differ in their last place, a constant then by one float32 rounding)
        want, bound = adamw_64(*host, step, lr, 0.9, 0.99, 1e-6, 0.1, 0.5)
        for got in (a, b, c):
            within(got[0], want[0], bound[0], torch.float32)


# ---- how the operators run together

class Model:
    """Embeddings trained towards targets: lookup, squared error, gradient, step."""

    def __init__(self, arb, seed, n=700, bag=3, vocab=400, dim=24):
        gen = torch.Generator().manual_seed(seed)
        self.arb, self.shape = arb, (n, bag, vocab, dim)
        self.tokens, self.held, strides = make_tokens(gen, n, bag, vocab, "padded", 32, False)
        self.table = torch.randn(vocab, dim, generator=gen).cuda()
        self.target = torch.randn(n, dim, generator=gen).cuda()
        self.m, self.v = torch.zeros_like(self.table), torch.zeros_like(self.table)
        self.out, self.grad_out, self.grad = torch.empty(n, dim, device="cuda"), torch.empty(n, dim, device="cuda"), torch.empty_like(self.table)
        self.step = torch.zeros(1, dtype=torch.int64, device="cuda")
        self.pairs = torch.empty(2, n * bag, dtype=torch.int32, device="cuda")
        size = max(arb.embedding_sort_bytes(n, vocab, bag=bag), arb.embedding_grad_bytes(n, dim, bag=bag))
        self.work = torch.empty(size, dtype=torch.uint8, device="cuda")

    def train_step(self, stream):
        arb, (n, bag, vocab, dim) = self.arb, self.shape
        work, size = self.work.data_ptr(), self.work.numel()
        self.step += 1
        arb.embedding(self.out.data_ptr(), self.table.data_ptr(), self.held.data_ptr(), n, vocab, dim, bag=bag, scale=0.5, stream=stream)
        torch.sub(self.out, self.target, out=self.grad_out)
        arb.embedding_sort(self.pairs[0].data_ptr(), self.pairs[1].data_ptr(), self.held.data_ptr(), n, vocab, work, size, bag=bag,
                           stream=stream)
        arb.embedding_grad(self.grad.data_ptr(), self.grad_out.data_ptr(), self.pairs[0].data_ptr(), self.pairs[1].data_ptr(), n,
                           vocab, dim, work, size, bag=bag, scale=0.5, stream=stream)
        arb.adamw([self.table.data_ptr()], [self.grad.data_ptr()], [self.m.data_ptr()], [self.v.data_ptr()], [vocab * dim], 1,
                  0.05, weight_decay=0.0, step_device=self.step.data_ptr(), stream=stream)

    def results(self):
        return [t.clone() for t in (self.out, self.grad, self.table, self.m, self.v)]


def test_a_training_run(arb):
    # gradients of every step against autograd in 64 bits
    model = Model(arb, 1)
    n, bag, vocab, dim = model.shape
    for _ in range(5):
        before = model.table.cpu()
        model.train_step(None)
        table = before.double().requires_grad_()
        t = torch.where(model.tokens >= 0, model.tokens, vocab)
        out = 0.5 * torch.cat([table, torch.zeros(1, dim, dtype=torch.float64)])[t].sum(1)
        (0.5 * (out - model.target.cpu().double()) ** 2).sum().backward()
        # k terms of grad_out, each off by the lookup's error and the difference's rounding
        _, mag = lookup_64(before, model.tokens, 0.5)
        one = (bag + 3) * U * mag + 2 * U * (out.detach().abs() + model.target.cpu().double().abs()) + U * out.detach().abs()
        error, _, _ = grad_64(one, model.tokens, vocab, 0.5)
        _, size, terms = grad_64((out.detach() - model.target.cpu().double()), model.tokens, vocab, 0.5)
        within(model.grad, table.grad, 1.01 * error + (terms + 3) * U * size, torch.float32)


def test_captured_and_replayed_beside_another(arb):
    # two models captured into two graphs, replayed in turn with eager work of a third between: each as if it ran alone
    stream = torch.cuda.Stream()
    alone = []
    for seed in (1, 2):
        model = Model(arb, seed)
        runs = []
        for _ in range(4):
            model.train_step(None)
            runs.append(model.results())
        alone.append(runs)
    third = Model(arb, 3)
    third.train_step(None)
    torch.cuda.synchronize()
    models, graphs = [], []
    for seed in (1, 2):
        model = Model(arb, seed)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            model.train_step(torch.cuda.current_stream().cuda_stream)
        models.append(model)
        graphs.append(graph)
    for k in range(4):
        for model, graph, runs in zip(models, graphs, alone):
            graph.replay()
            third.train_step(None)
            torch.cuda.synchronize()
            for got, want in zip(model.results(), runs[k]):
                assert torch.equal(got, want), k


def test_two_streams_at_once(arb):
    # two models on two streams, nothing waited for in between
    want = []
    for seed in (1, 2):
        model = Model(arb, seed)
        for _ in range(6):
            model.train_step(None)
        want.append(model.results())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    models = [Model(arb, 1), Model(arb, 2)]
    torch.cuda.synchronize()
    for _ in range(6):
        for model, stream in zip(models, streams):
            with torch.cuda.stream(stream):
                model.train_step(stream.cuda_stream)
    torch.cuda.synchronize()
    for model, w in zip(models, want):
        for a, b in zip(model.results(), w):
            assert torch.equal(a, b)


MANY = 1 << 27  # tokens, column by column, from which on rows of one element are looked up four bags a thread


@pytest.mark.parametrize("kind,bits,dtype", [("leaves", 32, "float32"), ("leaves", 64, "float16"), ("wide", 32, "bfloat16"),
                                             ("padded", 32, "float32"), ("padded", 64, "float32")])
def test_scalar_embeddings_of_many_columns(arb, kind, bits, dtype):
    bag, T = 13, TYPES[dtype]
    n = MANY // bag + 1027
    vocab = 13 * 1500
    gen = torch.Generator(device="cuda").manual_seed(bits)
    piece = {"leaves": 256, "wide": 1500, "padded": 1024}[kind]
    stride = n + 3
    held = torch.full((bag, stride), 1 << 30, dtype=torch.int32 if bits == 32 else torch.int64, device="cuda")
    for j in range(bag):
        held[j, :n] = torch.randint(0, piece, (n,), generator=gen, device="cuda") + j * 1500
        if kind == "padded":
            held[j, :n][torch.rand(n, generator=gen, device="cuda") < 0.3] = -1
    if kind == "padded":
        held[4, :n] = -1
        held[:, 5000:8000] = -1
    table = torch.randn(vocab, 1, generator=gen, device="cuda").to(T)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((n + 1, 2), 9.0, device="cuda", dtype=T)
    arb.embedding(out.data_ptr(), table.data_ptr(), held.data_ptr(), n, vocab, 1, bag=bag, scale=0.75, dtype=dtype, token_bits=bits,
                  token_stride=1, bag_stride=stride, out_stride=2, status=status.data_ptr())
    want, mag = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2))
    for j in range(bag):
        t = held[j, :n].long()
        x = torch.where(t >= 0, table.double()[t.clamp(min=0), 0], 0.0) * 0.75
        want += x
        mag += x.abs()
    within(out[:n, 0], want.cpu(), (bag + 3) * U * mag.cpu(), T)
    assert (out[:, 1] == 9).all() and (out[n] == 9).all() and status.item() == 0


def test_scalar_embeddings_report_a_wrong_token_in_any_column(arb):
    bag, vocab = 9, 2304
    n = MANY // bag + 1
    held = torch.arange(bag, dtype=torch.int32, device="cuda")[:, None].repeat(1, n) * 256
    table = torch.ones(vocab, 1, device="cuda")
    for column, row, token in [(0, 0, vocab), (8, n - 1, -2), (3, 77_777, 2 ** 31 - 1)]:
        right = held[column, row].item()
        held[column, row] = token
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.empty(n, device="cuda")
        arb.embedding(out.data_ptr(), table.data_ptr(), held.data_ptr(), n, vocab, 1, bag=bag, token_stride=1, bag_stride=n,
                      status=status.data_ptr())
        held[column, row] = right
        want = torch.full((n,), 9.0, device="cuda")
        want[row] = 8.0
        assert torch.equal(out, want) and status.item() == 1


def test_gradients_of_many_pairs_the_tokens_out_of_order(arb):
    # more pairs than one launch sorts: several tiles and groups of tiles, one, two and three digits
    for n, bag, vocab, dim in [(300_000, 3, 400, 1), (33_000, 1, 100_000, 9), (150_000, 2, 300_000, 2), (300_000, 1, 70, 3)]:
        gen = torch.Generator(device="cuda").manual_seed(vocab)
        tokens = (torch.rand(n, bag, generator=gen, device="cuda") ** 2 * vocab).long()
        tokens[torch.rand(n, bag, generator=gen, device="cuda") < 0.1] = -1
        for strides, held in (((bag, 1), tokens.to(torch.int32)), ((1, n), tokens.t().to(torch.int32).contiguous()),
                              ((bag + 1, 1), torch.cat([tokens, tokens[:, :1]], 1).to(torch.int32))):
            s = Sorted(arb, held, n, bag, vocab, strides)
            key = torch.where(tokens >= 0, tokens, vocab).reshape(-1)
            assert torch.equal(s.keys.long(), key.sort().values)
            pair = key * n + torch.arange(n, device="cuda").repeat_interleave(bag)
            assert torch.equal((s.keys.long() * n + s.rows.long()).sort().values, pair.sort().values)
            g = torch.randn(n, dim, generator=gen, device="cuda")
            got = s.grad(g, torch.full((vocab, dim), float("nan"), device="cuda"))
            rows = torch.arange(n, device="cuda").repeat_interleave(bag)
            want = torch.zeros(vocab + 1, dim, dtype=torch.float64, device="cuda").index_add_(0, key, g.double()[rows])
            mag = torch.zeros(vocab + 1, dim, dtype=torch.float64, device="cuda").index_add_(0, key, g.double().abs()[rows])
            # sums are formed in parts (a lane's share of a chunk, chunks of a run): no part and no joining of parts takes more
            # than 20,000 additions one after the other
            terms = torch.bincount(key, minlength=vocab + 1)[:-1, None].clamp(max=20_000).cpu()
            within(got, want[:-1].cpu(), (terms + 3) * U * mag[:-1].cpu(), torch.float32)
            assert torch.equal(got, s.grad(g, torch.empty(vocab, dim, device="cuda")))


def test_more_rows_than_one_launch_takes(arb):
    n, vocab, dim = (1 << 30) + 7, 1000, 16  # two lanes a row
    gen = torch.Generator(device="cuda").manual_seed(11)
    held = torch.randint(0, vocab, (n,), generator=gen, device="cuda", dtype=torch.int32)
    table = torch.randn(vocab, dim, generator=gen, device="cuda").half()
    out = torch.empty(n, dim, dtype=torch.float16, device="cuda")
    arb.embedding(out.data_ptr(), table.data_ptr(), held.data_ptr(), n, vocab, dim, dtype="float16")
    for i in range(0, n, 1 << 23):  # (torch's own gather takes a workgroup per index, which a launch counts with 32 bits)
        assert torch.equal(out[i:i + (1 << 23)], table[held[i:i + (1 << 23)].long()])


def test_one_bag_of_very_many_tokens(arb):
    # a single row of the result: all lanes of one group walk the bag
    bag, vocab = 5_000_003, 8
    held = (torch.arange(bag, device="cuda") % vocab).to(torch.int32)
    table = torch.tensor([1.0, -1.0, 2.0, -2.0, 0.5, -0.5, 0.25, -0.25], device="cuda")[:, None].contiguous()
    out = torch.empty(1, device="cuda")
    arb.embedding(out.data_ptr(), table.data_ptr(), held.data_ptr(), 1, vocab, 1, bag=bag)
    assert out.item() == 2.0  # (whole quarters: every sum is exact) 5,000,003 = 8 * 625,000 + 3
    s = Sorted(arb, held, 1, bag, vocab, (bag, 1))
    got = s.grad(torch.ones(1, 1, device="cuda"), torch.empty(vocab, 1, device="cuda"))
    assert got[:, 0].tolist() == [625_001.0] * 3 + [625_000.0] * 5


@pytest.mark.parametrize("beta1,beta2", [(0.0, 0.0), (0.0, 0.999), (0.9, 0.0), (0.95, 0.9999)])
def test_adamw_with_other_betas(arb, beta1, beta2):
    gen = torch.Generator().manual_seed(2)
    *host, at = make_tensors(gen, [3000], torch.float32, torch.float32)
    for step in (1, 2, 1000):
        for on_device in (False, True):
            dev = [t.cuda() for t in host]
            step_d = torch.tensor([step], device="cuda")
            more = dict(step=1, step_device=step_d.data_ptr()) if on_device else dict(step=step)
            run_adamw(arb, dev, at, [3000], beta1=beta1, beta2=beta2, **more)
            want, bound = adamw_64(*host, step, 0.01, beta1, beta2, 1e-6, 0.1, 0.5)
            within(dev[0], want[0], bound[0], torch.float32)
            for k in (1, 2):
                assert ((dev[k + 1].cpu().double() - want[k]).abs() <= bound[k] + 2.0 ** -149).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [9, 64, 260, 1100])
@pytest.mark.parametrize("m", [2, 31, 63, 64, 65, 256, 511, 512, 513])
def test_gradient_of_few_pairs(arb, m, dim, dtype):
    # runs of every length within and across the chunks that one workgroup holds
    gen = torch.Generator().manual_seed(m + dim)
    T = TYPES[dtype]
    for lengths in ([m], [1] * m, [m // 2, m - m // 2], [1, m - 1], [m - 1, 1], [3] * (m // 3) + [m % 3]):
        tokens = torch.repeat_interleave(torch.arange(len(lengths)) * 2, torch.tensor(lengths))[torch.randperm(m, generator=gen)]
        vocab = 2 * len(lengths) + 1
        held = tokens.to(torch.int32).cuda()
        grad_out = torch.randn(m, dim, generator=gen).to(T)
        s = Sorted(arb, held, m, 1, vocab, (1, 1))
        got = s.grad(grad_out.cuda(), torch.full((vocab, dim), float("nan"), dtype=T, device="cuda"))
        want, mag, terms = grad_64(grad_out, tokens[:, None], vocab, 1.0)
        within(got, want, (terms + 3) * U * mag, T)
        old = torch.randn(vocab, dim, generator=gen).to(T)
        got = s.grad(grad_out.cuda(), old.cuda(), accumulate=True)
        within(got, want + old.double(), (terms + 3) * U * mag + 2 * U * (want.abs() + old.double().abs()), T)


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("m", [4095, 4096, 4097, 16_384, 16_385, 32_769, 65_535, 65_536, 65_537, 131_072, 131_073, 262_144, 262_145])
def test_order_of_pairs_where_the_tiles_change(arb, m, bits):
    # both sides of every number of pairs from which on the sort takes other tiles or other launches
    gen = torch.Generator(device="cuda").manual_seed(m)
    for vocab in (300, 40_000, 300_000, 2 ** 31 - 1):
        tokens = torch.randint(0, vocab, (m,), generator=gen, device="cuda")
        tokens[torch.rand(m, generator=gen, device="cuda") < 0.2] = vocab // 2
        tokens[torch.rand(m, generator=gen, device="cuda") < 0.1] = -1
        s = Sorted(arb, tokens.to(torch.int32 if bits == 32 else torch.int64), m, 1, vocab, (1, 1), bits=bits)
        key = torch.where(tokens >= 0, tokens, vocab)
        assert torch.equal(s.keys.long(), key.sort().values)
        # every pair once, and pairs of a token in the same order from call to call
        pair = key * m + torch.arange(m, device="cuda")
        assert torch.equal((s.keys.long() * m + s.rows.long()).sort().values, pair.sort().values)
        first = s.pairs.clone()
        s.pairs.fill_(-7)
        s.call()
        assert torch.equal(s.pairs, first)


def test_few_pairs_of_a_table_of_a_billion_rows(arb):
    # more rows of zeros than one launch of large workgroups counts
    vocab, dim = (1 << 30) + 7, 9
    named = torch.tensor([vocab - 1, 0, 1 << 29, 0])
    grad_out = torch.arange(1, 1 + 4 * dim).reshape(4, dim).half().cuda()
    s = Sorted(arb, named.to(torch.int32).cuda(), 4, 1, vocab, (1, 1))
    got = s.grad(grad_out, torch.full((vocab, dim), float("nan"), dtype=torch.float16, device="cuda"))
    assert torch.equal(got[vocab - 1], grad_out[0]) and torch.equal(got[1 << 29], grad_out[2])
    assert torch.equal(got[0], grad_out[1] + grad_out[3])  # (whole numbers: exact)
    for row in (vocab - 1, 0, 1 << 29):
        got[row] = 0
    for i in range(0, vocab, 1 << 26):  # (a NaN counts)
        assert torch.count_nonzero(got[i:i + (1 << 26)]).item() == 0
    again = s.grad(grad_out, got, accumulate=True)
    assert torch.equal(again[vocab - 1], grad_out[0]) and torch.equal(again[0], grad_out[1] + grad_out[3])
