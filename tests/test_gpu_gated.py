"""Gated layers, their gradients and activations kept in 8 bits on the GPU against plain restatements in 64 bits.

Bounds, with u = 2^-24.  A sum of k products formed in float32 is off by at most (2 k + 8) u times the sum of their magnitudes (a
rounding for the product, where float32 does not hold it, and one for the sum).  act has a slope of at most 1.13, so
act(g) is off by 1.2 times what g is off by, and by its own 16 u (1 + g^2) |act(g)| (an exponential or erfc at a rounded argument: g^2 is the
condition of both tails).  The gradient is compared with one formed from the gate and up that the layer kept, which are its inputs: d_gate and
d_up are off by their own float32 roundings, 24 u (1 + g^2) of the terms that their slopes are sums of, and by half a step of the type they are rounded to;
products pass that on.  What is kept in 8 bits is off by half a scale.  A result adds half a step of its type."""
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
    info = torch.finfo(dtype)
    return info.eps / 2, info.smallest_normal * info.eps / 2


def close(got, want, err, dtype, what):
    rel, step = half_step(dtype)
    got, want, err = got.cpu(), want.cpu(), err.cpu()
    bound = err + rel * (want.abs() + err) + step
    off = (got.double().cpu() - want).abs()
    # (rounding to nearest takes what is beyond the type's greatest number by half a step or more to infinity: 1.1e5 is no number of float16)
    beyond = torch.isinf(got.double().cpu()) & (got.double().cpu().sign() == want.sign()) & ((want.abs() + err) * (1 + rel) >= torch.finfo(dtype).max)
    bad = ~(off <= bound) & ~beyond
    assert not bad.any(), "%s: %d off, the worst %g where %g is allowed" % (what, bad.sum(), off[bad].max(), bound[bad][off[bad].argmax()])


def act_64(name, g):
    """act(g), its slope, and the sum of the magnitudes that the slope is formed from"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s), s + (g * s * (1 - s)).abs()
    phi = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)  # (ndtr forms 1 + erf: 0 at -12.5 instead of 3.7e-36)
    bell = torch.exp(-g * g / 2) / (2 * np.pi) ** 0.5
    return g * phi, phi + g * bell, phi + (g * bell).abs()


def spread(values, pad, first, fill):
    """The values in rows `pad` elements further apart, from element `first` on: (buffer, view on the device, stride)"""
    rows, width = values.shape
    buffer = torch.full((first + rows * (width + pad),), fill, dtype=values.dtype)
    buffer[first:].reshape(rows, width + pad)[:, :width] = values
    buffer = buffer.cuda()
    return buffer, buffer[first:].reshape(rows, width + pad), width + pad


class Layer:
    def __init__(self, arb, rows, dim, hidden, dtype, activation="silu", kept="as is", pad=0, first=0, seed=0, x=None, stream=None, size=1.0):
        self.arb, self.rows, self.dim, self.hidden, self.dtype = arb, rows, dim, hidden, dtype
        self.T, self.activation, self.pad, self.first, self.eight = TYPES[dtype], activation, pad, first, kept == "8 bits"
        gen = torch.Generator().manual_seed(seed + rows + 31 * dim + 1009 * hidden)
        self.x = (size * torch.randn(rows, dim, generator=gen) if x is None else x).to(self.T)
        self.wg, self.wu = ((torch.randn(hidden, dim, generator=gen) * dim ** -0.5).to(self.T) for _ in range(2))
        self.grad_out = torch.randn(rows, hidden, generator=gen).to(self.T)
        put = lambda v, fill=float("nan"): spread(v, pad, first, fill)[1:]  # noqa: E731
        self.d_x, self.x_stride = put(self.x)
        self.d_wg, self.w_stride = put(self.wg)
        self.d_wu, _ = put(self.wu)
        self.d_grad, self.grad_out_stride = put(self.grad_out)
        zeros = lambda r, w: torch.zeros(r, w, dtype=self.T)  # noqa: E731
        self.out_buffer, self.out, self.out_stride = spread(zeros(rows, hidden), pad, first, 7.0)
        groups = (hidden + 63) // 64
        self.scales = torch.full((2, max(rows, 1), groups), -5.0, device="cuda")
        if self.eight:
            kinds = torch.zeros(rows, hidden, dtype=torch.int8)
            self.gate_buffer, self.gate, self.kept_stride = spread(kinds, pad, first, 77)
            self.up_buffer, self.up, _ = spread(kinds, pad, first, 77)
        elif kept == "as is":
            self.gate_buffer, self.gate, self.kept_stride = spread(zeros(rows, hidden), pad, first, 7.0)
            self.up_buffer, self.up, _ = spread(zeros(rows, hidden), pad, first, 7.0)
        else:
            self.gate = self.up = None
            self.kept_stride = None
        self.size = max(arb.gated_bytes(rows, dim, hidden, dtype=dtype), arb.gated_grad_bytes(rows, dim, hidden, dtype=dtype))
        self.work = torch.full((max(16, self.size),), 0xA5, dtype=torch.uint8, device="cuda")
        self.grad_x_buffer, self.grad_x, self.grad_x_stride = spread(zeros(rows, dim), pad, first, 7.0)
        self.grad_wg_buffer, self.grad_wg, self.grad_w_stride = spread(zeros(hidden, dim), pad, first, 7.0)
        self.grad_wu_buffer, self.grad_wu, _ = spread(zeros(hidden, dim), pad, first, 7.0)

    def common(self, stream):
        at = lambda v: None if v is None else v.data_ptr()  # noqa: E731
        return dict(gate=at(self.gate), up=at(self.up), gate_scales=self.scales[0].data_ptr() if self.eight else None,
                    up_scales=self.scales[1].data_ptr() if self.eight else None, activation=self.activation, dtype=self.dtype,
                    kept_stride=self.kept_stride, x_stride=self.x_stride, w_stride=self.w_stride, stream=stream)

    def forward(self, stream=None):
        self.arb.gated(self.out.data_ptr(), self.d_x.data_ptr(), self.d_wg.data_ptr(), self.d_wu.data_ptr(), self.rows, self.dim, self.hidden,
                       self.work.data_ptr(), self.size, out_stride=self.out_stride, **self.common(stream))
        return self

    def backward(self, stream=None, grad_x=True, grad_w=True):
        self.arb.gated_grad(self.grad_x.data_ptr() if grad_x else None, self.grad_wg.data_ptr() if grad_w else None,
                            self.grad_wu.data_ptr() if grad_w else None, self.d_grad.data_ptr(), self.d_x.data_ptr(), self.d_wg.data_ptr(),
                            self.d_wu.data_ptr(), self.rows, self.dim, self.hidden, self.work.data_ptr(), self.size,
                            grad_x_stride=self.grad_x_stride, grad_w_stride=self.grad_w_stride, grad_out_stride=self.grad_out_stride, **self.common(stream))
        return self

    def products(self):
        x, wg, wu = self.x.double(), self.wg.double(), self.wu.double()
        per = (2 * self.dim + 8) * U
        return x @ wg.t(), x @ wu.t(), per * (x.abs() @ wg.abs().t()), per * (x.abs() @ wu.abs().t())

    def kept_values(self):
        """gate and up as the layer kept them"""
        out = []
        for k, v in enumerate((self.gate, self.up)):
            v = v[:, :self.hidden].cpu()
            if self.eight:
                scale = self.scales[k][:self.rows].cpu().repeat_interleave(64, 1)[:, :self.hidden]
                v = v.float() * scale
            out.append(v.double())
        return out

    def check_forward(self):
        g, u, eg, eu = self.products()
        act = act_64(self.activation, g)[0]
        ea = 1.2 * eg + 16 * U * (1 + g * g) * act.abs()
        close(self.out[:, :self.hidden], act * u, u.abs() * ea + act.abs() * eu + ea * eu + 2 * U * (act * u).abs(), self.T, "out")
        if self.gate is not None:
            for k, (got, want, err) in enumerate(zip(self.kept_values(), (g, u), (eg, eu))):
                if self.eight:
                    got, want, err = got.cpu(), want.cpu(), err.cpu()
                    for c in range(0, self.hidden, 64):
                        most = want[:, c:c + 64].abs().max(1).values + err[:, c:c + 64].max(1).values
                        scale = self.scales[k][:self.rows, c // 64].double().cpu()
                        off_scale = err[:, c:c + 64].max(1).values / 127 + 2 * U * most
                        assert ((scale - want[:, c:c + 64].abs().max(1).values / 127).abs() <= off_scale).all()
                        bound = 0.5 * scale[:, None] * (1 + 8 * U) + err[:, c:c + 64] + 4 * U * want[:, c:c + 64].abs()
                        assert ((got[:, c:c + 64] - want[:, c:c + 64]).abs() <= bound).all()
                else:
                    close(got, want, err, self.T, "kept")
        return self

    def check_backward(self, grad_x=True, grad_w=True):
        if self.rows:
            g, u = self.kept_values()
        else:
            g = u = torch.zeros(0, self.hidden, dtype=torch.float64)
        y, x, wg, wu = (v.double() for v in (self.grad_out, self.x, self.wg, self.wu))
        act, slope, size = act_64(self.activation, g)
        rel, step = half_step(self.T)
        own = 24 * U * (1 + g * g)
        dg, du = y * u * slope, y * act
        edg, edu = own * (y * u).abs() * size, own * (y * act).abs()
        edg, edu = edg + rel * (dg.abs() + edg) + step, edu + rel * (du.abs() + edu) + step
        if grad_x:
            want = dg @ wg + du @ wu
            err = edg @ wg.abs() + edu @ wu.abs()
            err += (4 * self.hidden + 8) * U * (dg.abs() @ wg.abs() + du.abs() @ wu.abs() + err)
            close(self.grad_x[:, :self.dim], want, err, self.T, "grad_x")
        if grad_w:
            for got, d, ed, what in ((self.grad_wg, dg, edg, "grad_w_gate"), (self.grad_wu, du, edu, "grad_w_up")):
                err = ed.t() @ x.abs()
                err += (2 * self.rows + 8) * U * (d.abs().t() @ x.abs() + err)
                close(got[:, :self.dim], d.t() @ x, err, self.T, what)
        return self

    def check_margins(self):
        """What lies between and before the rows stays as it was."""
        every = [(self.out_buffer, self.hidden), (self.grad_x_buffer, self.dim), (self.grad_wg_buffer, self.dim), (self.grad_wu_buffer, self.dim)]
        if self.gate is not None:
            every += [(self.gate_buffer, self.hidden), (self.up_buffer, self.hidden)]
        for buffer, width in every:
            fill = 77 if buffer.dtype == torch.int8 else 7
            assert (buffer[:self.first] == fill).all()
            assert (buffer[self.first:].reshape(-1, width + self.pad)[:, width:] == fill).all()


# rows, dim, hidden
SIZES = [(1, 1, 1), (1, 16, 64), (1, 4096, 100), (2, 33, 65), (3, 8, 7), (5, 64, 64), (15, 100, 30), (16, 128, 128), (17, 520, 257), (31, 7, 300),
         (33, 1000, 63), (64, 64, 64), (65, 129, 127), (127, 96, 512), (128, 128, 128), (129, 200, 129), (130, 771, 205), (257, 72, 136), (300, 16, 16), (513, 40, 24),
         (1000, 5, 3), (2500, 24, 70), (5000, 64, 40), (256, 256, 256), (511, 520, 520)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", SIZES)
def test_layer_and_gradient(arb, rows, dim, hidden, dtype):
    which = (rows + dim + hidden) % 2
    layer = Layer(arb, rows, dim, hidden, dtype, activation=["silu", "gelu"][which]).forward().check_forward()
    layer.backward().check_backward()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kept", ["as is", "no"])
@pytest.mark.parametrize("rows,dim,hidden,pad,first", [(1, 4095, 33, 0, 0), (16, 1027, 40, 0, 0), (7, 1024, 50, 1, 0), (9, 2048, 31, 0, 1), (16, 513, 17, 2, 1), (3, 130, 16, 0, 0),
                                                        (5, 4097, 70, 3, 3), (17, 1027, 40, 0, 0), (2, 1, 300, 0, 0), (4, 5, 259, 0, 1),
                                                        (16, 7, 131, 0, 0), (1, 771, 1000, 0, 0), (3, 9, 15, 2, 5), (1, 256, 129, 1, 3)])
def test_few_rows_that_begin_anywhere(arb, rows, dim, hidden, pad, first, kept, dtype):
    layer = Layer(arb, rows, dim, hidden, dtype, kept=kept, pad=pad, first=first).forward().check_forward()
    if kept != "no":
        layer.backward().check_backward()
    layer.check_margins()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows,dim,hidden", [(1, 40, 200), (3, 8, 7), (70, 64, 64), (130, 96, 129), (257, 30, 320), (5, 512, 1024)])
def test_kept_in_8_bits(arb, rows, dim, hidden, activation, dtype):
    layer = Layer(arb, rows, dim, hidden, dtype, activation=activation, kept="8 bits").forward().check_forward()
    layer.backward().check_backward()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kept", ["as is", "8 bits", "no"])
@pytest.mark.parametrize("rows,dim,hidden,pad,first", [(1, 24, 40, 3, 1), (6, 24, 40, 3, 1), (130, 65, 131, 1, 1), (40, 64, 128, 8, 0), (200, 136, 72, 8, 8),
                                                        (300, 64, 192, 5, 3), (260, 128, 256, 64, 0)])
def test_strides_and_starts_of_any_alignment(arb, rows, dim, hidden, pad, first, kept, dtype):
    layer = Layer(arb, rows, dim, hidden, dtype, kept=kept, pad=pad, first=first, activation="gelu").forward().check_forward()
    if kept != "no":
        layer.backward().check_backward()
    layer.check_margins()


def test_weights_that_share_a_matrix_and_a_broadcast_row(arb):
    # rows of x all the same one (a stride of 0), gate and up the halves of one matrix
    rows, dim, hidden = 70, 48, 96
    layer = Layer(arb, rows, dim, hidden, "float32", x=torch.randn(1, dim, generator=torch.Generator().manual_seed(3)).expand(rows, dim).contiguous())
    both = torch.cat([layer.wg, layer.wu]).cuda()
    layer.d_wg, layer.d_wu = both[:hidden], both[hidden:]
    layer.d_x, layer.x_stride = layer.x[:1].cuda(), 0
    layer.forward().check_forward().backward().check_backward()
    row = layer.grad_out[:1].cuda()
    layer.grad_out = layer.grad_out[:1].expand(rows, hidden).contiguous()
    layer.d_grad, layer.grad_out_stride = row, 0
    layer.backward().check_backward()


def test_parts_of_the_gradient_and_no_rows(arb):
    layer = Layer(arb, 50, 40, 72, "bfloat16").forward()
    layer.backward(grad_w=False).check_backward(grad_w=False)
    assert (layer.grad_wg == 0).all() and (layer.grad_wu == 0).all()
    layer.grad_x.fill_(3)
    layer.backward(grad_x=False).check_backward(grad_x=False)
    assert (layer.grad_x == 3).all()
    empty = Layer(arb, 0, 40, 72, "bfloat16").forward()
    empty.grad_wg.fill_(3)
    empty.grad_wu.fill_(3)
    empty.backward()
    assert (empty.grad_wg == 0).all() and (empty.grad_wu == 0).all()


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_gates(arb, activation, dtype):
    # gates of hundreds on both sides: the activation is the identity, or nothing
    layer = Layer(arb, 40, 64, 64, dtype, activation=activation, size=60.0).forward().check_forward()
    layer.backward().check_backward()


@pytest.mark.parametrize("rows", [7, 5000])
@pytest.mark.parametrize("activation,most", [("silu", 80.0), ("gelu", 12.5)])
def test_activations_over_their_range(arb, activation, most, rows):
    # one product with 1 is exact: gates from end to end of what normal numbers of float32 tell from the identity and from nothing, by the kernels for few rows
    # and for many
    x = torch.linspace(-most, most, rows, dtype=torch.float32)[:, None].cuda()
    one = torch.ones(1, 1, device="cuda")
    out, gate, up, dx = (torch.full_like(x, 7) for _ in range(4))
    dw = torch.empty(2, 1, 1, device="cuda")
    grad = torch.ones_like(x)
    work = torch.empty(max(arb.gated_bytes(rows, 1, 1), arb.gated_grad_bytes(rows, 1, 1)), dtype=torch.uint8, device="cuda")
    kept = dict(gate=gate.data_ptr(), up=up.data_ptr(), activation=activation)
    both = (x.data_ptr(), one.data_ptr(), one.data_ptr(), rows, 1, 1, work.data_ptr(), work.numel())
    arb.gated(out.data_ptr(), *both, **kept)
    arb.gated_grad(dx.data_ptr(), dw[0].data_ptr(), dw[1].data_ptr(), grad.data_ptr(), *both, **kept)
    torch.cuda.synchronize()
    g = x.double().cpu()
    act, slope, slope_sum = act_64(activation, g)
    close(out, act * g, 18 * U * (1 + g * g) * (act * g).abs(), torch.float32, "out")
    want = g * slope + act
    close(dx, want, 24 * U * (1 + g * g) * (g.abs() * slope_sum + act.abs()), torch.float32, "grad_x")


def test_infinities_and_nan_stay_in_their_rows(arb):
    rows, dim, hidden = 140, 70, 90
    for kept in ("as is", "8 bits"):
        good = Layer(arb, rows, dim, hidden, "bfloat16", kept=kept).forward().backward()
        layer = Layer(arb, rows, dim, hidden, "bfloat16", kept=kept)
        for row, value in ((3, float("nan")), (77, float("inf")), (139, float("-inf"))):
            layer.d_x[row, 5] = value
        layer.forward().backward()
        bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
        bad[[3, 77, 139]] = True
        assert torch.equal(layer.out[~bad], good.out[~bad]) and torch.equal(layer.grad_x[~bad], good.grad_x[~bad])
        assert torch.isnan(layer.out[3]).all() and not torch.isfinite(layer.out[bad]).all(1).any()
        assert torch.isnan(layer.grad_wg[:, 5]).all()  # every weight of that column has met them
        if kept == "8 bits":
            assert torch.isnan(layer.scales[0][bad]).all() and torch.isfinite(layer.scales[:, ~bad]).all()


def test_gradient_against_differences(arb):
    # central differences along a direction, the layer in 64 bits: a step of 1e-4 is off by 1e-8 / 6 of a third derivative (below 100 times the direction's
    # size here), beside the bounds of the gradient's elements along the direction, all within 1e-4 of its size
    for activation in ("silu", "gelu"):
        layer = Layer(arb, 9, 13, 21, "float32", activation=activation).forward().backward()
        gen = torch.Generator().manual_seed(8)
        x, wg, wu, y = (v.double() for v in (layer.x, layer.wg, layer.wu, layer.grad_out))
        grads = [layer.grad_x[:, :13], layer.grad_wg[:, :13], layer.grad_wu[:, :13]]
        for which in range(3):
            d = torch.randn([x, wg, wu][which].shape, generator=gen, dtype=torch.float64)
            d /= d.norm()

            def loss(step):
                args = [x, wg, wu]
                args[which] = args[which] + step * d
                return (act_64(activation, args[0] @ args[1].t())[0] * (args[0] @ args[2].t()) * y).sum()

            want = (loss(1e-4) - loss(-1e-4)) / 2e-4
            got = (grads[which].double().cpu() * d).sum()
            assert abs(want - got) <= 1e-6 + 1e-4 * grads[which].double().cpu().norm()


def test_results_are_the_same_from_run_to_run(arb):
    layer = Layer(arb, 3000, 72, 60, "bfloat16").forward().backward()
    first = [v.clone() for v in (layer.out, layer.grad_x, layer.grad_wg, layer.grad_wu)]
    layer.work.fill_(0x3C)
    layer.forward().backward()
    assert all(torch.equal(a, b) for a, b in zip(first, (layer.out, layer.grad_x, layer.grad_wg, layer.grad_wu)))


def test_offsets_beyond_32_bits(arb):
    # rows 1.2 G elements apart, on every side
    far, rows, dim, hidden = 1_200_000_000, 3, 64, 64
    layer = Layer(arb, rows, dim, hidden, "bfloat16").forward().backward()
    buffer = torch.zeros(2 * far + 4096, dtype=torch.bfloat16, device="cuda")

    def distant(values, at):
        view = torch.as_strided(buffer, values.shape, (far, 1), at)
        view.copy_(values)
        return view

    other = Layer(arb, rows, dim, hidden, "bfloat16")
    other.d_x, other.x_stride = distant(layer.x, 0), far
    other.d_grad, other.grad_out_stride = distant(layer.grad_out, 512), far
    other.out, other.out_stride = distant(torch.zeros(rows, hidden), 1024), far
    other.gate, other.up, other.kept_stride = distant(torch.zeros(rows, hidden), 1536), distant(torch.zeros(rows, hidden), 2048), far
    other.grad_x, other.grad_x_stride = distant(torch.zeros(rows, dim), 2560), far
    other.forward().backward()
    for name in ("out", "gate", "up", "grad_x", "grad_wg", "grad_wu"):
        assert torch.equal(getattr(other, name), getattr(layer, name)), name


def test_captured_replayed_and_on_two_streams(arb):
    layers = [Layer(arb, 200, 72, 130, "bfloat16", kept="8 bits"), Layer(arb, 2000, 64, 40, "float16"), Layer(arb, 1, 256, 512, "bfloat16")]
    for layer in layers:
        layer.forward().backward()
    torch.cuda.synchronize()
    graphs = []
    for layer in layers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s = torch.cuda.current_stream().cuda_stream
            layer.forward(s)
            layer.backward(s)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in layers]
    for round in range(3):
        wants = []
        for layer in layers:
            other = Layer(arb, layer.rows, layer.dim, layer.hidden, layer.dtype, kept="8 bits" if layer.eight else "as is", seed=round + 1).forward().backward()
            layer.d_x.copy_(other.d_x)
            layer.d_wg.copy_(other.d_wg)
            layer.d_wu.copy_(other.d_wu)
            layer.d_grad.copy_(other.d_grad)
            for out in (layer.out, layer.grad_x, layer.grad_wg, layer.grad_wu):
                out.fill_(9.0)
            layer.work.fill_(0x5A)
            wants.append(other)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for layer, other in zip(layers, wants):
            for name in ("out", "grad_x", "grad_wg", "grad_wu"):
                assert torch.equal(getattr(layer, name), getattr(other, name)), (round, name)


# ---- activations in 8 bits by themselves

def kept_by_hand(x):
    """codes and scales: every operation is one of float32, correctly rounded, so they are equal bit by bit"""
    x = x.float().numpy()
    rows, dim = x.shape
    codes, scales = np.zeros((rows, dim), np.int8), np.zeros((rows, (dim + 63) // 64), np.float32)
    for c in range(0, dim, 64):
        part = x[:, c:c + 64]
        scale = np.maximum(np.abs(part).max(1) / np.float32(127), np.float32(2.0 ** -100))
        scales[:, c // 64] = scale
        codes[:, c:c + 64] = np.rint(part / scale[:, None])
    return codes, scales


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim,pad,first", [(1, 1, 0, 0), (3, 64, 0, 0), (5, 63, 1, 1), (7, 65, 0, 0), (40, 771, 0, 0), (33, 128, 8, 8), (1000, 100, 3, 1), (200, 4096, 0, 0),
                                                 (9, 2047, 5, 2), (70_001, 8, 0, 0)])
def test_activations_kept_and_read_back(arb, rows, dim, pad, first, dtype):
    T = TYPES[dtype]
    gen = torch.Generator().manual_seed(rows + dim)
    x = (torch.randn(rows, dim, generator=gen) * torch.exp(2 * torch.randn(1, dim, generator=gen))).to(T)
    x[0] = 0
    _, held, stride = spread(x, pad, first, float("nan"))
    groups = (dim + 63) // 64
    codes, scales = torch.full((rows * dim + 1,), 99, dtype=torch.int8, device="cuda"), torch.full((rows * groups + 1,), 99.0, device="cuda")
    arb.activation_checkpoint(codes.data_ptr(), scales.data_ptr(), held.data_ptr(), rows, dim, dtype=dtype, x_stride=stride)
    want_codes, want_scales = kept_by_hand(x)
    assert np.array_equal(codes[:-1].cpu().numpy().reshape(rows, dim), want_codes) and codes[-1] == 99
    assert np.array_equal(scales[:-1].cpu().numpy().reshape(rows, groups), want_scales) and scales[-1] == 99
    buffer, back, stride = spread(torch.zeros(rows, dim, dtype=T), pad, first, 7.0)
    arb.activation_restore(back.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, dim, dtype=dtype, x_stride=stride)
    want = (torch.from_numpy(want_codes).float() * torch.from_numpy(want_scales).repeat_interleave(64, 1)[:, :dim]).to(T)
    assert torch.equal(back[:, :dim].cpu(), want)
    assert (buffer[:first] == 7).all() and (back[:, dim:] == 7).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_extreme_activations(arb, dtype):
    T = TYPES[dtype]
    info = torch.finfo(T)
    rows, dim = 7, 130
    x = torch.ones(rows, dim).to(T)
    x[0], x[1], x[2] = info.max, info.smallest_normal, info.min
    x[3, 70], x[4, 0], x[5, 129] = float("nan"), float("inf"), float("-inf")
    x[6, ::2] = -1e-30 if dtype != "float16" else -6e-8
    held = x.cuda()
    codes, scales, back = torch.empty(rows, dim, dtype=torch.int8, device="cuda"), torch.empty(rows, 3, device="cuda"), torch.empty_like(held)
    arb.activation_checkpoint(codes.data_ptr(), scales.data_ptr(), held.data_ptr(), rows, dim, dtype=dtype)
    arb.activation_restore(back.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, dim, dtype=dtype)
    back, x = back.cpu().double(), x.double()
    broken = torch.zeros(rows, dim, dtype=torch.bool)
    broken[3, 64:128] = broken[4, :64] = broken[5, 128:] = True
    assert torch.isnan(back[broken]).all() and torch.isfinite(back[~broken]).all()
    rel, step = half_step(T)
    most = torch.where(torch.isfinite(x), x.abs(), 0.0)
    for c in range(0, dim, 64):
        part = slice(c, min(dim, c + 64))
        scale = (most[:, part].max(1, keepdim=True).values / 127).clamp(min=2.0 ** -100)
        off = (back[:, part] - x[:, part]).abs()
        bound = 0.5 * scale * (1 + 8 * U) + (rel + 4 * U) * x[:, part].abs() + step
        assert (off <= bound)[~broken[:, part]].all()


def test_a_layer_of_leaf_embeddings_from_lookup_to_step(arb):
    """The operators in a row, as a model over leaves uses them: lookup, a gated layer whose activations are kept in 8 bits, logits, log
    probabilities, and all gradients down to the table, compared with the same in 64 bits.  Every stage is held to its own bound elsewhere; here
    the roundings of 8 bits (0.6 % of the kept values each, three of them meet in a gradient) and of bfloat16 (0.2 % on each of about eight
    stages) add up to less than 5 % of a gradient's norm."""
    gen = torch.Generator().manual_seed(6)
    n, bag, vocab, dim, hidden, classes = 700, 5, 90, 48, 200, 11
    tokens = torch.randint(0, vocab, (n, bag), generator=gen)
    labels = torch.randint(0, classes, (n,), generator=gen)
    labels[::9] = -1
    T = torch.bfloat16
    table = torch.randn(vocab, dim, generator=gen).to(T).cuda()
    wg, wu = ((torch.randn(hidden, dim, generator=gen) * dim ** -0.5).to(T).cuda() for _ in range(2))
    head = (torch.randn(classes, hidden, generator=gen) * hidden ** -0.5).to(T).cuda()
    held, label = tokens.to(torch.int32).cuda(), labels.to(torch.int32).cuda()
    new = lambda *s, t=T: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731

    def at(v):
        return v.data_ptr()

    x = new(n, dim)
    arb.embedding(at(x), at(table), at(held), n, vocab, dim, bag=bag, scale=0.4, dtype="bfloat16")
    x_codes, x_scales = new(n, dim, t=torch.int8), new(n, 1, t=torch.float32)
    arb.activation_checkpoint(at(x_codes), at(x_scales), at(x), n, dim, dtype="bfloat16")
    size = max(arb.gated_bytes(n, dim, hidden, dtype="bfloat16"), arb.gated_grad_bytes(n, dim, hidden, dtype="bfloat16"), arb.embedding_sort_bytes(n, vocab, bag=bag),
               arb.embedding_grad_bytes(n, dim, bag=bag), arb.log_probs_bytes(n, classes))
    work = new(size, t=torch.uint8)
    kept, scales, out = new(2, n, hidden, t=torch.int8), new(2, n, 4, t=torch.float32), new(n, hidden)
    more = dict(gate=at(kept[0]), up=at(kept[1]), gate_scales=at(scales[0]), up_scales=at(scales[1]), dtype="bfloat16")
    arb.gated(at(out), at(x), at(wg), at(wu), n, dim, hidden, at(work), size, **more)
    logits = out @ head.t()
    lp, stats = new(n, t=torch.float32), new(n, 2, t=torch.float32)
    arb.log_probs(at(lp), at(logits), at(label), n, classes, at(work), size, stats=at(stats), dtype="bfloat16")
    weight = torch.full((n,), -1.0, device="cuda")
    arb.log_probs_grad(at(logits), at(weight), at(logits), at(label), at(stats), n, classes, dtype="bfloat16")
    grad_head, grad_out = logits.t() @ out, logits @ head
    arb.activation_restore(at(x), at(x_codes), at(x_scales), n, dim, dtype="bfloat16")
    grad_x, grad_wg, grad_wu = new(n, dim), new(hidden, dim), new(hidden, dim)
    arb.gated_grad(at(grad_x), at(grad_wg), at(grad_wu), at(grad_out), at(x), at(wg), at(wu), n, dim, hidden, at(work), size, **more)
    keys, rows = new(n * bag, t=torch.int32), new(n * bag, t=torch.int32)
    arb.embedding_sort(at(keys), at(rows), at(held), n, vocab, at(work), size, bag=bag)
    grad_table = new(vocab, dim, t=torch.float32)
    arb.embedding_grad(at(grad_table), at(grad_x), at(keys), at(rows), n, vocab, dim, at(work), size, bag=bag, scale=0.4, dtype="bfloat16")

    p = [v.double().cpu().requires_grad_() for v in (table, wg, wu, head)]
    x64 = 0.4 * p[0][tokens].sum(1)
    g, u = x64 @ p[1].t(), x64 @ p[2].t()
    log_p = torch.log_softmax((g * torch.sigmoid(g) * u) @ p[3].t(), 1)
    named = labels >= 0
    loss = -log_p[named, labels[named]].sum()
    loss.backward()
    for got, want in zip((grad_table, grad_wg, grad_wu, grad_head), p):
        got = got.double().cpu()
        assert (got - want.grad).norm() <= 0.05 * want.grad.norm()
    assert abs(-lp.double().sum().item() - loss.item()) <= 0.02 * loss.item() and (lp[~named.cuda()] == 0).all()


class OnDevice(Layer):
    """The same, its restatement in 64 bits on the GPU."""

    def __init__(self, *args, **more):
        super().__init__(*args, **more)
        self.x, self.wg, self.wu, self.grad_out = (v.cuda() for v in (self.x, self.wg, self.wu, self.grad_out))

    def kept_values(self):
        out = []
        for k, v in enumerate((self.gate, self.up)):
            v = v[:, :self.hidden]
            if self.eight:
                v = v.float() * self.scales[k][:self.rows].repeat_interleave(64, 1)[:, :self.hidden]
            out.append(v.double())
        return out


@pytest.mark.parametrize("rows,dim,hidden,dtype,pad,first,kept", [
    (4000, 136, 2100, "bfloat16", 0, 0, "no"), (4000, 136, 2100, "float16", 8, 8, "as is"), (4100, 129, 1999, "bfloat16", 0, 0, "as is"),
    (1030, 3600, 4100, "bfloat16", 0, 0, "as is"), (1001, 3601, 4099, "float16", 3, 1, "as is"), (3001, 132, 2300, "float32", 0, 0, "as is"),
    (260, 7000, 7200, "bfloat16", 0, 0, "as is"), (300, 3700, 3500, "float32", 1, 1, "as is"), (3000, 72, 2200, "bfloat16", 0, 0, "8 bits")])
def test_sizes_that_fill_the_chip(arb, rows, dim, hidden, dtype, pad, first, kept):
    layer = OnDevice(arb, rows, dim, hidden, dtype, kept=kept, pad=pad, first=first, activation="gelu" if rows % 2 else "silu").forward()
    layer.check_forward()
    if kept != "no":
        layer.backward().check_backward()
    layer.check_margins()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,dim,hidden", [(3, 515, 200), (16, 77, 129), (40, 515, 70), (450, 65, 70)])
def test_weights_that_begin_differently(arb, rows, dim, hidden, dtype):
    layer = Layer(arb, rows, dim, hidden, dtype)
    wu_buffer, layer.d_wu, _ = spread(layer.wu, 0, 3, float("nan"))
    layer.forward().check_forward().backward().check_backward()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,dim,hidden", [(5, 48, 70), (300, 64, 128)])
def test_gate_beside_up_in_one_matrix(arb, rows, dim, hidden, dtype):
    alone, beside = (Layer(arb, rows, dim, hidden, dtype) for _ in range(2))
    kept = torch.full((rows, 2 * hidden + 1), 7.0, dtype=TYPES[dtype], device="cuda")
    grads = torch.full((hidden, 2 * dim + 3), 7.0, dtype=TYPES[dtype], device="cuda")
    beside.gate, beside.up, beside.kept_stride = kept[:, :hidden], kept[:, hidden:2 * hidden], 2 * hidden + 1
    beside.grad_wg, beside.grad_wu, beside.grad_w_stride = grads[:, :dim], grads[:, dim:2 * dim], 2 * dim + 3
    for layer in (alone, beside):
        layer.forward().backward()
    for name in ("out", "gate", "up", "grad_x", "grad_wg", "grad_wu"):
        assert torch.equal(getattr(alone, name), getattr(beside, name)), name
    assert (kept[:, 2 * hidden:] == 7).all() and (grads[:, 2 * dim:] == 7).all()
