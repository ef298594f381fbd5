"""Log probabilities, entropies, likeliest tokens and the gradient of logits on the GPU against a plain restatement in 64 bits.

Bounds, with u = 2^-24, a_j = scale (x_j - max x), L = log sum exp a, p = softmax, E|a| = sum p |a|.  An exponent in powers of two is a
difference, a product and a constant of two roundings: off by 4 u |a|; its power by 2 u more.  Maxima that move on the way add
distances that end to end are |a|, and two roundings each.  A sum of c steps adds c u.  Steps: an element in 64 of a row and 64 for the joins
(a wave shares a row at least), or all of a row that one thread reads.  So
  err(L) = u (4 E|a| + c + 4 + 2 |L|),   err(log_prob) = u (3 |a_t| + |log_prob|) + err(L)
  err(H) = err(L) + u (4 E[a^2] + (c + 16) E|a|) + E|a| err(S) + 4 u (|L| + H),   err(S) the part of err(L) that S is off by
  err(p) / p = u (3 |a| + 2 |L| + 4 |log p| + 4) + err(L)   (a difference, a constant of two roundings, L in powers of two, their sum)
and the gradient's terms with these and a rounding for each operation.  A result's type adds half its step."""
import itertools

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
INF = float("inf")


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


def half_step(dtype):
    info = torch.finfo(dtype)
    return info.eps / 2, info.smallest_normal * info.eps / 2


def make_logits(gen, n, vocab, kind, dtype):
    if kind == "normal":
        x = 3 * torch.randn(n, vocab, generator=gen)
    elif kind == "ties":
        x = torch.randint(-3, 4, (n, vocab), generator=gen).float()
    elif kind == "rising":
        x = torch.arange(vocab).float().expand(n, vocab) * (20.0 / vocab) - 5.0
    elif kind == "falling":
        x = 5.0 - torch.arange(vocab).float().expand(n, vocab) * (20.0 / vocab)
    elif kind == "constant":
        x = torch.full((n, vocab), -7.25)
    elif kind == "masked":
        x = 3 * torch.randn(n, vocab, generator=gen)
        x[torch.rand(n, vocab, generator=gen) < 0.6] = -INF
        x[::3] = -INF  # rows of nothing
        x[1::3, 0] = 0.0
    elif kind == "one":
        x = torch.full((n, vocab), -INF)
        x[torch.arange(n), torch.randint(0, vocab, (n,), generator=gen)] = 2.5
    elif kind == "lowest":  # masks of the type's lowest value
        x = 3 * torch.randn(n, vocab, generator=gen)
        x[torch.rand(n, vocab, generator=gen) < 0.5] = torch.finfo(dtype).min
        x[::2] = torch.finfo(dtype).min
    return x.to(dtype)


class Want:
    """The same in 64 bits, and how far off each may be."""

    def __init__(self, x, tokens, scale, chain):
        self.x, self.tokens, self.scale = x.double(), tokens, scale
        n, vocab = x.shape
        most = self.x.amax(1, keepdim=True)
        nothing = (most == -INF)[:, 0]
        base = torch.where(most == -INF, 0.0, most)
        self.a = scale * (self.x - base)
        e = torch.exp(self.a)
        s = e.sum(1)
        self.L = torch.where(nothing, 0.0, torch.log(s))
        self.log_p = self.a - self.L[:, None]
        self.p = torch.exp(self.log_p)
        fa = torch.where(self.p > 0, self.a.abs(), 0.0)
        self.mean_a = (self.p * fa).sum(1)
        self.H = torch.where(nothing, 0.0, self.L + self.mean_a)
        err_s = U * (4 * self.mean_a + chain + 4)
        self.err_L = err_s + 2 * U * self.L.abs()
        self.err_H = self.err_L + U * (4 * (self.p * fa * fa).sum(1) + (chain + 16) * self.mean_a) + self.mean_a * err_s + 4 * U * (self.L.abs() + self.H)
        self.nothing, self.most = nothing, most[:, 0]
        named = tokens >= 0
        t = tokens.clamp(min=0, max=vocab - 1)[:, None]
        self.named = named & (tokens < vocab)
        self.log_prob = torch.where(self.named, self.log_p.gather(1, t)[:, 0], 0.0)
        self.err_log_prob = self.err_of(self.log_prob, torch.where(self.named, self.a.gather(1, t)[:, 0], 0.0))

    def err_of(self, log_p, a, err_L=None):
        err_L = self.err_L if err_L is None else err_L
        return torch.where(torch.isfinite(log_p), U * (3 * a.abs() + log_p.abs()) + err_L, 0.0)

    def top(self, k):
        x = self.x.numpy()
        order = np.stack([np.lexsort((np.arange(x.shape[1]), -row)) for row in x])[:, :k] if k else np.zeros((len(x), 0), int)
        return torch.from_numpy(order)

    def grad(self, w, h, dtype):
        """(gradient, bound) for upstream gradients w and h (or None)"""
        w = torch.where(self.named, w.double(), 0.0)[:, None]
        hit = torch.zeros_like(self.p)
        hit[self.named, self.tokens[self.named]] = 1
        log_p, a = torch.where(self.p > 0, self.log_p, 0.0), torch.where(self.p > 0, self.a, 0.0)
        err_lp = U * (3 * a.abs() + 2 * self.L[:, None].abs() + log_p.abs()) + self.err_L[:, None]
        rel = err_lp + U * (3 * log_p.abs() + 4)
        p = torch.where(self.nothing[:, None], 0.0, self.p)
        hit = torch.where(self.nothing[:, None], 0.0, hit)
        g, err = w * (hit - p), w.abs() * (p * rel + 3 * U * (hit - p).abs())
        if h is not None:
            h = h.double()[:, None]
            g = g - h * p * (log_p + self.H[:, None])
            size = log_p.abs() + self.H[:, None]
            err = err + h.abs() * p * (rel * size + err_lp + self.err_H[:, None] + 4 * U * size)
        g, err = self.scale * g, self.scale * (err + 4 * U * g.abs())
        err = err + 3e-38  # (a probability below float32's normal numbers may be 0)
        rel, step = half_step(dtype)
        return g, err + rel * (g.abs() + err) + step


def close(got, want, bound, what):
    got, want, bound = got.double().cpu(), want.expand(got.shape), bound.expand(got.shape)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(off <= bound) & ~same
    assert not bad.any(), "%s: %d off, the worst %g where %g is allowed" % (what, bad.sum(), off[bad].max(), bound[bad][off[bad].argmax()])


class Held:
    """Logits on the device with room between rows, or class by class, and what the calls write."""

    def __init__(self, arb, x, tokens, layout, bits=32, scale=1.0, top=0, status=None):
        self.arb, (self.n, self.vocab) = arb, x.shape
        self.scale, self.top, self.status = scale, top, status
        if layout == "rows":
            self.buffer, self.strides, first = x.contiguous().reshape(-1), (self.vocab, 1), 0
        elif layout == "padded":
            wide = torch.full((self.n, self.vocab + 3), float("nan"), dtype=x.dtype)
            wide[:, :self.vocab] = x
            first = 1
            self.buffer = torch.cat([torch.full((1,), float("nan"), dtype=x.dtype), wide.reshape(-1)])
            self.strides = (self.vocab + 3, 1)
        elif layout == "columns":
            self.buffer, self.strides, first = x.t().contiguous().reshape(-1), (1, self.n), 0
        else:  # neither side by side
            wide = torch.full((self.n, self.vocab, 2), float("nan"), dtype=x.dtype)
            wide[:, :, 0] = x
            self.buffer, self.strides, first = wide.reshape(-1), (2 * self.vocab, 2), 0
        self.buffer = self.buffer.cuda()
        self.at = self.buffer.data_ptr() + first * self.buffer.element_size()
        self.first = first
        self.dtype = {v: k for k, v in TYPES.items()}[x.dtype]
        self.tokens = None if tokens is None else tokens.to(torch.int32 if bits == 32 else torch.int64).cuda()
        self.bits = bits
        n = max(self.n, 1)
        self.log_probs = torch.full((n,), 99.0, device="cuda")
        self.entropy = torch.full((n,), 99.0, device="cuda")
        self.stats = torch.full((n, 2), 99.0, device="cuda")
        self.top_tokens = torch.full((n, max(top, 1)), -99, device="cuda", dtype=torch.int32)
        self.top_log_probs = torch.full((n, max(top, 1)), 99.0, device="cuda")
        self.size = arb.log_probs_bytes(self.n, self.vocab, top=top)
        self.work = torch.full((max(16, self.size),), 0xA5, dtype=torch.uint8, device="cuda")

    def common(self, stream):
        return dict(scale=self.scale, dtype=self.dtype, token_bits=self.bits, row_stride=self.strides[0], class_stride=self.strides[1],
                    status=None if self.status is None else self.status.data_ptr(), stream=stream)

    def forward(self, stream=None, entropy=True, stats=True):
        t = None if self.tokens is None else self.tokens.data_ptr()
        self.arb.log_probs(None if t is None else self.log_probs.data_ptr(), self.at, t, self.n, self.vocab, self.work.data_ptr(), self.size,
                           entropy=self.entropy.data_ptr() if entropy else None, stats=self.stats.data_ptr() if stats else None, top=self.top,
                           top_tokens=self.top_tokens.data_ptr() if self.top else None, top_log_probs=self.top_log_probs.data_ptr() if self.top else None,
                           **self.common(stream))
        return self

    def backward(self, w, h, stream=None, in_place=False):
        self.w, self.h = w.cuda(), None if h is None else h.cuda()
        self.grad = self.buffer if in_place else torch.full_like(self.buffer, 7.0)
        at = self.grad.data_ptr() + self.first * self.grad.element_size()
        self.arb.log_probs_grad(at, self.w.data_ptr(), self.at, self.tokens.data_ptr(), self.stats.data_ptr(), self.n, self.vocab,
                                grad_entropy=None if h is None else self.h.data_ptr(), entropy=None if h is None else self.entropy.data_ptr(),
                                **self.common(stream))
        return self.grad_rows()

    def grad_rows(self):
        view = self.grad.cpu()[self.first:]
        return torch.as_strided(view, (self.n, self.vocab), self.strides) if self.n else view.reshape(0, self.vocab)


def check(arb, x, tokens, layout, scale=1.0, top=0, bits=32, h=True):
    n, vocab = x.shape
    scale = float(np.float32(scale))
    chain = vocab + 64 if layout in ("columns", "spread") or vocab <= 128 else vocab / 64 + 64
    want = Want(x, tokens, scale, chain)
    held = Held(arb, x, tokens, layout, bits=bits, scale=scale, top=top).forward()
    close(held.log_probs[:n], want.log_prob, want.err_log_prob, "log_probs")
    close(held.entropy[:n], want.H, want.err_H, "entropy")
    assert torch.equal(held.stats[:n, 0].cpu().double(), want.most)
    close(held.stats[:n, 1], want.L, want.err_L, "stats")
    if top:
        order = want.top(top)
        assert torch.equal(held.top_tokens.cpu().long(), order)
        log_p = want.log_p.gather(1, order)
        close(held.top_log_probs, log_p, want.err_of(log_p, torch.where(torch.isfinite(log_p), want.a.gather(1, order), 0.0), want.err_L[:, None]), "top_log_probs")
    gen = torch.Generator().manual_seed(n + vocab)
    w = torch.randn(n, generator=gen)
    for hh in (None, torch.randn(n, generator=gen)) if h else (None,):
        got = held.backward(w, hh)
        g, bound = want.grad(w, hh, x.dtype)
        close(got, g, bound, "gradient")
        if layout == "padded":
            rest = held.grad.cpu()
            assert (rest[0] == 7) and (rest[1:].reshape(n, vocab + 3)[:, vocab:] == 7).all()
        if layout == "spread":
            assert (held.grad.cpu().reshape(n, vocab, 2)[:, :, 1] == 7).all()
    got = held.backward(w, None)
    in_place = held.backward(w, None, in_place=True)
    assert torch.equal(got, in_place) or torch.equal(got.nan_to_num(77.0), in_place.nan_to_num(77.0))


def some_tokens(gen, n, vocab):
    t = torch.randint(0, vocab, (n,), generator=gen)
    t[torch.rand(n, generator=gen) < 0.2] = -1
    return t


SIZES = [(1, 1, 1), (5, 2, 2), (3, 10, 3), (300, 10, 10), (7, 31, 9), (64, 32, 4), (65, 33, 33), (9, 64, 64), (5, 65, 20), (11, 300, 5), (257, 511, 1),
         (4, 2047, 64), (3, 2048, 7), (3, 2049, 64), (6, 5000, 20), (2, 8191, 5), (300, 8193, 5), (260, 16_400, 64), (1, 50_021, 20), (33, 50_021, 5), (1, 131_072, 64),
         (2, 131_075, 0), (257, 4096, 0)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,vocab,top", SIZES)
def test_rows(arb, n, vocab, top, dtype):
    gen = torch.Generator().manual_seed(n * 1000 + vocab)
    x = make_logits(gen, n, vocab, "normal", TYPES[dtype])
    check(arb, x, some_tokens(gen, n, vocab), "rows", scale=0.7, top=top, h=n * vocab < 1 << 20)


@pytest.mark.parametrize("kind", ["ties", "rising", "falling", "constant", "masked", "one", "lowest"])
@pytest.mark.parametrize("n,vocab,top", [(7, 3, 3), (9, 32, 17), (8, 40, 40), (6, 700, 64), (4, 3000, 9), (300, 5001, 20), (3, 40_007, 64)])
@pytest.mark.parametrize("layout", ["rows", "columns"])
def test_values_that_tie_rise_or_are_masked(arb, n, vocab, top, kind, layout):
    gen = torch.Generator().manual_seed(vocab)
    dtype = [torch.float32, torch.bfloat16, torch.float16][(vocab + len(kind)) % 3]
    x = make_logits(gen, n, vocab, kind, dtype)
    check(arb, x, some_tokens(gen, n, vocab), layout, scale=1.6 if kind != "lowest" else 1.0, top=top)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["padded", "columns", "spread"])
@pytest.mark.parametrize("n,vocab,top", [(5, 3, 2), (70, 10, 3), (1000, 10, 3), (300, 33, 12), (20, 129, 64), (3, 2500, 5)])
def test_strides_and_starts_of_any_alignment(arb, n, vocab, top, layout, dtype):
    gen = torch.Generator().manual_seed(n + 7 * vocab)
    x = make_logits(gen, n, vocab, "normal", TYPES[dtype])
    check(arb, x, some_tokens(gen, n, vocab), layout, scale=1.3, top=top, bits=64)


# many rows of few classes: a thread a row, and top in passes of eight
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["rows", "padded", "columns", "spread"])
@pytest.mark.parametrize("n,vocab,top", [(40, 1, 1), (500, 4, 3), (2600, 10, 8), (5200, 16, 10), (18_000, 61, 9), (9000, 128, 2), (4200, 127, 0)])
def test_many_rows_of_few_classes(arb, n, vocab, top, layout, dtype):
    gen = torch.Generator().manual_seed(n + vocab)
    x = make_logits(gen, n, vocab, "normal", TYPES[dtype])
    check(arb, x, some_tokens(gen, n, vocab), layout, scale=1.1, top=top)


@pytest.mark.parametrize("kind", ["ties", "rising", "falling", "constant", "masked", "one", "lowest"])
@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("n,vocab,top", [(2000, 7, 5), (6000, 17, 11)])
def test_many_rows_that_tie_rise_or_are_masked(arb, n, vocab, top, kind, layout):
    gen = torch.Generator().manual_seed(vocab + n)
    dtype = [torch.float32, torch.bfloat16, torch.float16][(vocab + len(kind)) % 3]
    x = make_logits(gen, n, vocab, kind, dtype)
    check(arb, x, some_tokens(gen, n, vocab), layout, scale=0.8 if kind != "lowest" else 1.0, top=top)


# few rows class by class: teams whose loads lie apart, rows in parts, gradients whose classes are shared out
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["columns", "spread"])
@pytest.mark.parametrize("n,vocab,top", [(1, 2000, 64), (2, 40_007, 20), (260, 2049, 3), (10, 16_385, 0), (3, 131, 9)])
def test_few_rows_class_by_class(arb, n, vocab, top, layout, dtype):
    gen = torch.Generator().manual_seed(n + vocab)
    x = make_logits(gen, n, vocab, "normal", TYPES[dtype])
    check(arb, x, some_tokens(gen, n, vocab), layout, scale=0.9, top=top)


@pytest.mark.parametrize("n,vocab", [(5, 12), (4, 600), (6, 3000), (300, 9000), (2, 30_000), (3000, 12), (9000, 50)])
@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_rows_with_a_nan_or_plus_infinity_say_so_and_others_do_not(arb, n, vocab, bad):
    gen = torch.Generator().manual_seed(vocab)
    x = make_logits(gen, n, vocab, "normal", torch.float32)
    x[1, vocab // 2] = bad
    if n > 4:
        x[4] = -INF
        x[4, vocab - 1] = bad
    tokens = torch.randint(0, vocab, (n,), generator=gen)
    top = 6
    held = Held(arb, x, tokens, "rows", top=top).forward()
    w = torch.randn(n, generator=gen)
    grad = held.backward(w, w)
    broken = torch.zeros(n, dtype=torch.bool)
    broken[[1, 4] if n > 4 else [1]] = True
    for out in (held.log_probs, held.entropy, held.top_log_probs, grad):
        out = out.cpu().reshape(n, -1)
        assert torch.isnan(out[broken]).all() and torch.isfinite(out[~broken]).all()
    assert (held.top_tokens.cpu()[broken] == -1).all()
    fine = Want(x[~broken], tokens[~broken], 1.0, vocab + 64)
    close(held.log_probs.cpu()[~broken], fine.log_prob, fine.err_log_prob, "log_probs")
    assert torch.equal(held.top_tokens.cpu().long()[~broken], fine.top(top))


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("layout", ["rows", "columns"])
def test_tokens_outside_are_reported_and_count_as_none(arb, bits, layout):
    vocab = 50
    big = 2 ** 31 - 1 if bits == 32 else 2 ** 40
    tokens = torch.tensor([0, 49, -1, 50, -2, big])
    x = make_logits(torch.Generator().manual_seed(1), 6, vocab, "normal", torch.float32)
    for use, told in [(6, 1), (3, 0)]:
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        held = Held(arb, x[:use], tokens[:use], layout, bits=bits, status=status).forward()
        assert status.item() == told
        assert (held.log_probs.cpu()[2:] == 0).all() and (held.log_probs.cpu()[:2] < 0).all()
        status.zero_()
        w = torch.ones(use)
        w[2:] = float("nan")  # what a row without a token is given plays no part
        grad = held.backward(w, None)
        assert status.item() == told
        assert (grad[2:] == 0).all() and (grad[:2] != 0).all()


def test_no_tokens_no_rows_and_single_outputs(arb):
    x = make_logits(torch.Generator().manual_seed(1), 40, 3001, "normal", torch.bfloat16)
    full = Held(arb, x, torch.zeros(40, dtype=torch.long), "rows", top=4).forward()
    only = Held(arb, x, None, "rows", top=4).forward(entropy=False, stats=False)
    assert torch.equal(only.top_tokens, full.top_tokens) and torch.equal(only.top_log_probs, full.top_log_probs)
    assert (only.log_probs == 99).all() and (only.entropy == 99).all() and (only.stats == 99).all()
    entropy = Held(arb, x, None, "rows").forward(stats=False)
    assert torch.equal(entropy.entropy, full.entropy)
    Held(arb, x, None, "rows").forward(entropy=False, stats=False)
    Held(arb, x[:0], torch.zeros(0, dtype=torch.long), "rows", top=4).forward()
    got = Held(arb, x[:0], torch.zeros(0, dtype=torch.long), "rows")
    got.backward(torch.zeros(0), None)
    assert not got.grad.numel()


def test_gradient_against_differences(arb):
    # central differences of the definition in 64 bits: off by step^2 / 6 of a third derivative, which for these (scale 1.5, values of at
    # most a few) is below 40: 7e-10 at a step of 1e-5, beside 1e-16 * 40 / 1e-5 for the rounding
    gen = torch.Generator().manual_seed(4)
    n, vocab, scale = 4, 37, 1.5
    x = make_logits(gen, n, vocab, "normal", torch.float32)
    tokens = torch.tensor([3, -1, 36, 0])
    w, h = torch.randn(n, generator=gen), torch.randn(n, generator=gen)
    held = Held(arb, x, tokens, "rows", scale=scale).forward()
    grad = held.backward(w, h).double()

    def loss(y):
        log_p = torch.log_softmax(scale * y, 1)
        named = torch.where(tokens >= 0, log_p.gather(1, tokens.clamp(min=0)[:, None])[:, 0], 0.0)
        return (w.double() * named - h.double() * (log_p.exp() * log_p).sum(1)).sum()

    bound = Want(x, tokens, scale, vocab + 64).grad(w, h, torch.float32)[1]
    for i, j in itertools.product(range(n), [0, 3, 17, 36]):
        up, down = x.double(), x.double()
        up[i, j] += 1e-5
        down[i, j] -= 1e-5
        assert abs((loss(up) - loss(down)) / 2e-5 - grad[i, j]) <= bound[i, j] + 1e-9 + 1e-9


def test_results_are_the_same_from_run_to_run(arb):
    x = make_logits(torch.Generator().manual_seed(1), 3, 100_003, "normal", torch.bfloat16)
    tokens = torch.tensor([1, 2, 3])
    a, b = (Held(arb, x, tokens, "rows", top=64).forward() for _ in range(2))
    assert torch.equal(a.log_probs, b.log_probs) and torch.equal(a.entropy, b.entropy) and torch.equal(a.top_tokens, b.top_tokens)


def test_offsets_beyond_32_bits(arb):
    # rows 1.2 G elements apart, and classes as far apart
    far, vocab = 1_200_000_001, 3000
    buffer = torch.zeros(2 * far + vocab, dtype=torch.bfloat16, device="cuda")
    x = make_logits(torch.Generator().manual_seed(1), 3, vocab, "normal", torch.bfloat16)
    for r in range(3):
        buffer[r * far:r * far + vocab] = x[r].cuda()
    near = Held(arb, x, torch.tensor([5, 2999, 7]), "rows", top=5).forward()
    distant = Held(arb, x, torch.tensor([5, 2999, 7]), "rows", top=5)
    distant.buffer, distant.at, distant.strides = buffer, buffer.data_ptr(), (far, 1)
    distant.forward()
    for name in ("log_probs", "entropy", "top_tokens", "top_log_probs", "stats"):
        assert torch.equal(getattr(near, name), getattr(distant, name))
    w = torch.ones(3)
    want = near.backward(w, None)
    distant.w = w.cuda()
    arb.log_probs_grad(distant.at, distant.w.data_ptr(), distant.at, distant.tokens.data_ptr(), distant.stats.data_ptr(), 3, vocab, **distant.common(None))
    assert torch.equal(torch.stack([buffer[r * far:r * far + vocab] for r in range(3)]).cpu(), want)
    y = make_logits(torch.Generator().manual_seed(2), 5, 3, "normal", torch.bfloat16)
    for c in range(3):
        buffer[c * far:c * far + 5] = y[:, c].cuda()
    near = Held(arb, y, torch.tensor([0, 1, 2, 0, 1]), "columns", top=3).forward()
    distant = Held(arb, y, torch.tensor([0, 1, 2, 0, 1]), "columns", top=3)
    distant.buffer, distant.at, distant.strides = buffer, buffer.data_ptr(), (1, far)
    distant.forward()
    for name in ("log_probs", "entropy", "top_tokens", "top_log_probs", "stats"):
        assert torch.equal(getattr(near, name), getattr(distant, name))


def test_captured_replayed_and_on_two_streams(arb):
    gen = torch.Generator().manual_seed(1)
    cases = [(3, 60_000, 20), (400, 2500, 5)]
    helds = [Held(arb, make_logits(gen, n, v, "normal", torch.bfloat16), torch.randint(0, v, (n,), generator=gen), "rows", top=k) for n, v, k in cases]
    w = [torch.randn(n, generator=gen) for n, _, _ in cases]
    for held, ww in zip(helds, w):
        held.forward()
        held.backward(ww, None)  # (kernels are loaded before they are captured)
    torch.cuda.synchronize()
    graphs = []
    for held in helds:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s = torch.cuda.current_stream().cuda_stream
            held.forward(s)
            arb.log_probs_grad(held.grad.data_ptr(), held.w.data_ptr(), held.at, held.tokens.data_ptr(), held.stats.data_ptr(), held.n, held.vocab,
                               **held.common(s))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round in range(3):
        wants = []
        for held, (n, v, k) in zip(helds, cases):
            x = make_logits(torch.Generator().manual_seed(10 * round + v), n, v, "normal", torch.bfloat16)
            held.buffer.copy_(x.reshape(-1))
            eager = Held(arb, x, held.tokens.cpu(), "rows", top=k).forward()
            eager.backward(held.w.cpu(), None)
            wants.append(eager)
            for out in (held.log_probs, held.entropy, held.top_log_probs, held.grad):
                out.fill_(55.0)
            held.work.fill_(0x5A)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for held, eager in zip(helds, wants):
            for name in ("log_probs", "entropy", "top_tokens", "top_log_probs", "grad"):
                assert torch.equal(getattr(held, name), getattr(eager, name)), (round, name)
