"""The gradient of gated layers in float16 where d_gate and d_up, which the products take in 16 bits, lie beyond float16 or below its normal numbers,
against the formulas in 64 bits.

Bounds, with u = 2^-24 and M the greatest finite magnitude of d_gate and d_up: each of them is off by 24 u (1 + g^2) of the terms that its slope is a sum of, by half a
step (2^-11 of it), and by 2^-25 M where they are taken as they are (1 <= M < 65504: half of float16's least step), by 2^-39 M where they are taken times a power of
two that brings M to 2^14 or more.  A sum of k products in float32 adds (2 k + 8) u of their magnitudes, the result half a step of its own."""
import pytest
import torch

from test_gpu_gated import U, act_64, close, spread

pytestmark = pytest.mark.gpu

T = torch.float16


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


def draw(gen, rows, dim, hidden, regime):
    """grad_out, x, w_gate, w_up, gate, up; the last two are inputs of the gradient by themselves, and need not be products"""
    normal = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    about = lambda size, *s: size * (0.5 + torch.rand(*s, generator=gen))  # noqa: E731
    sign = lambda *s: torch.randint(0, 2, s, generator=gen) * 2.0 - 1.0  # noqa: E731
    if regime == "below":  # d_gate of 2^-28, whose sums over rows of one sign are numbers of float16
        y, x, u, g = about(2.0 ** -20, rows, hidden), about(1.0, rows, dim), about(2.0 ** -8, rows, hidden), about(1.0, rows, hidden)
        wg, wu = 8 * normal(hidden, dim), 8 * normal(hidden, dim)
    else:
        y, u = about(2.0 ** 11, rows, hidden) * sign(rows, hidden), about(64.0, rows, hidden) * sign(rows, hidden)
        g, x = normal(rows, hidden), 2.0 ** -12 * normal(rows, dim)
        wg, wu = 2.0 ** -10 * normal(hidden, dim), 2.0 ** -10 * normal(hidden, dim)
        if regime == "a row beyond":
            y[1:], u[1:] = normal(rows - 1, hidden), normal(rows - 1, hidden)
        elif regime == "ordinary":
            y, u = normal(rows, hidden), normal(rows, hidden)
    return tuple(v.to(T) for v in (y, x, wg, wu, g, u))


class Gradient:
    def __init__(self, arb, rows, dim, hidden, activation="silu", kept="as is", pad=0, first=0):
        self.arb, self.rows, self.dim, self.hidden, self.activation, self.eight = arb, rows, dim, hidden, activation, kept == "8 bits"
        self.pad, self.first = pad, first
        self.size = arb.gated_grad_bytes(rows, dim, hidden, dtype="float16")
        self.work = torch.full((self.size,), 0xA5, dtype=torch.uint8, device="cuda")
        self.grad_x_buffer, self.grad_x, _ = spread(torch.zeros(rows, dim, dtype=T), pad, first, 7.0)
        self.grad_w = [spread(torch.zeros(hidden, dim, dtype=T), pad, first, 7.0) for _ in range(2)]

    def put(self, y, x, wg, wu, g, u):
        self.host = [v.double() for v in (y, x, wg, wu, g, u)]
        held = [spread(v, self.pad, self.first, float("nan")) for v in (y, x, wg, wu)]
        self.on_device = [h[1] for h in held]
        if self.eight:
            self.kept, self.scales = [], []
            for k, v in enumerate((g, u)):
                codes = torch.empty(self.rows, self.hidden, dtype=torch.int8, device="cuda")
                scales = torch.empty(self.rows, (self.hidden + 63) // 64, device="cuda")
                v = v.cuda()
                self.arb.activation_checkpoint(codes.data_ptr(), scales.data_ptr(), v.data_ptr(), self.rows, self.hidden, dtype="float16")
                self.kept.append(codes)
                self.scales.append(scales)
                self.host[4 + k] = (codes.float() * scales.repeat_interleave(64, 1)[:, :self.hidden]).double().cpu()
            self.kept_stride = self.hidden
        else:
            held = [spread(v, self.pad, self.first, float("nan")) for v in (g, u)]
            self.kept, self.kept_stride = [h[1] for h in held], self.hidden + self.pad
        return self

    def run(self, stream=None, grad_x=True, grad_w=True):
        y, x, wg, wu = self.on_device
        scales = dict(gate_scales=self.scales[0].data_ptr(), up_scales=self.scales[1].data_ptr()) if self.eight else {}
        self.arb.gated_grad(self.grad_x.data_ptr() if grad_x else None, self.grad_w[0][1].data_ptr() if grad_w else None,
                            self.grad_w[1][1].data_ptr() if grad_w else None, y.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), self.rows, self.dim,
                            self.hidden, self.work.data_ptr(), self.size, self.kept[0].data_ptr(), self.kept[1].data_ptr(), activation=self.activation,
                            dtype="float16", grad_x_stride=self.dim + self.pad, grad_w_stride=self.dim + self.pad, grad_out_stride=self.hidden + self.pad,
                            kept_stride=self.kept_stride, x_stride=self.dim + self.pad, w_stride=self.dim + self.pad, stream=stream, **scales)
        return self

    def results(self):
        return [v[:, :self.dim].clone() for v in (self.grad_x, self.grad_w[0][1], self.grad_w[1][1])]

    def check(self, grad_x=True, grad_w=True, rows=slice(None)):
        y, x, wg, wu, g, u = self.host
        act, slope, size = act_64(self.activation, g)
        dg, du = y * u * slope, y * act
        most = max(torch.where(torch.isfinite(d), d.abs(), 0.0).max() for d in (dg, du))
        least = (2.0 ** -25 if 1 <= most < 65504 else 2.0 ** -39) * most
        own = 24 * U * (1 + g * g)
        edg, edu = own * (y * u).abs() * size, own * (y * act).abs()
        edg, edu = edg + 2.0 ** -11 * (dg.abs() + edg) + least, edu + 2.0 ** -11 * (du.abs() + edu) + least
        if grad_x:
            err = edg[rows] @ wg.abs() + edu[rows] @ wu.abs()
            err += (4 * self.hidden + 8) * U * (dg[rows].abs() @ wg.abs() + du[rows].abs() @ wu.abs() + err)
            close(self.grad_x[rows, :self.dim], dg[rows] @ wg + du[rows] @ wu, err, T, "grad_x")
        if grad_w:
            for (_, got, _), d, ed, what in zip(self.grad_w, (dg, du), (edg, edu), ("grad_w_gate", "grad_w_up")):
                err = ed.t() @ x.abs()
                err += (2 * self.rows + 8) * U * (d.abs().t() @ x.abs() + err)
                close(got[:, :self.dim], d.t() @ x, err, T, what)
        return self


# both products at once, their shares joined by one thread and by eight, one after the other, in large tiles, in copies of rows that begin anywhere
SIZES = [(40, 64, 64, 0, 0), (3, 8, 7, 0, 0), (5000, 64, 40, 0, 0), (300, 771, 205, 0, 0), (130, 65, 131, 1, 1), (200, 136, 72, 8, 8), (257, 72, 136, 3, 1), (4000, 136, 2100, 0, 0)]


@pytest.mark.parametrize("regime", ["beyond", "below", "a row beyond", "ordinary"])
@pytest.mark.parametrize("rows,dim,hidden,pad,first", SIZES)
def test_factors_beyond_float16(arb, rows, dim, hidden, pad, first, regime):
    gen = torch.Generator().manual_seed(rows + dim)
    for kept in ("as is", "8 bits"):
        gradient = Gradient(arb, rows, dim, hidden, ["silu", "gelu"][rows % 2], kept, pad, first)
        gradient.put(*draw(gen, rows, dim, hidden, regime)).run().check()


@pytest.mark.parametrize("regime", ["beyond", "below"])
def test_one_of_the_gradients(arb, regime):
    gradient = Gradient(arb, 150, 72, 100).put(*draw(torch.Generator().manual_seed(1), 150, 72, 100, regime))
    gradient.run(grad_w=False).check(grad_w=False).run(grad_x=False).check()


def test_a_row_of_infinities_leaves_the_others_as_they_are(arb):
    for bad in (float("inf"), float("nan")):
        for regime in ("beyond", "below", "ordinary"):
            values = draw(torch.Generator().manual_seed(2), 60, 48, 80, regime)
            values[0][7, 3] = bad
            gradient = Gradient(arb, 60, 48, 80).put(*values).run()
            gradient.check(grad_w=False, rows=slice(0, 7)).check(grad_w=False, rows=slice(8, 60))
            assert not torch.isfinite(gradient.grad_x[7]).any()
            others = [k for k in range(80) if k != 3]  # (and the weights of the other hidden columns)
            assert torch.isfinite(gradient.grad_w[0][1][others]).all() and not torch.isfinite(gradient.grad_w[1][1][3]).any()


def test_nothing_to_pass_on(arb):
    values = draw(torch.Generator().manual_seed(3), 50, 24, 30, "ordinary")
    values[0].zero_()
    gradient = Gradient(arb, 50, 24, 30).put(*values).run()
    assert all((v == 0).all() for v in gradient.results())


def test_replays_find_the_range_of_their_own_inputs(arb):
    rows, dim, hidden = 300, 64, 96
    regimes = ["ordinary", "beyond", "below", "ordinary", "below"]
    gradient = Gradient(arb, rows, dim, hidden).put(*draw(torch.Generator().manual_seed(0), rows, dim, hidden, "ordinary")).run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gradient.run(torch.cuda.current_stream().cuda_stream)
    for seed, regime in enumerate(regimes):
        values = draw(torch.Generator().manual_seed(seed), rows, dim, hidden, regime)
        eager = Gradient(arb, rows, dim, hidden).put(*values).run()
        for to, value in zip(gradient.on_device + gradient.kept, values):
            to.copy_(value)
        gradient.host = eager.host
        gradient.work.fill_(0x5A)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        gradient.check()
        assert all(torch.equal(a, b) for a, b in zip(gradient.results(), eager.results())), regime
