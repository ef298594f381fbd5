"""Calls of log_probs, gated and activation_checkpoint, and of their gradients, that are refused: host code only, so nothing here reaches
a GPU (addresses are never followed: every call is refused before a kernel is launched)."""
import pytest

A = 1 << 20


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    return arboretum_amd


def logits(arb, **change):
    a = dict(log_probs=A, logits=2 * A, tokens=3 * A, n=4, vocab=100, work=4 * A, work_bytes=1 << 20, entropy=5 * A, stats=6 * A, top=3,
             top_tokens=7 * A, top_log_probs=8 * A)
    a.update(change)
    arb.log_probs(**a)


def logits_grad(arb, **change):
    a = dict(grad_logits=A, grad_log_probs=2 * A, logits=3 * A, tokens=4 * A, stats=5 * A, n=4, vocab=100)
    a.update(change)
    arb.log_probs_grad(**a)


def keep(arb, **change):
    a = dict(codes=A, scales=2 * A, x=3 * A, rows=4, dim=100)
    a.update(change)
    arb.activation_checkpoint(**a)


def read_back(arb, **change):
    a = dict(x=A, codes=2 * A, scales=3 * A, rows=4, dim=100)
    a.update(change)
    arb.activation_restore(**a)


def layer(arb, **change):
    a = dict(out=A, x=2 * A, w_gate=3 * A, w_up=4 * A, rows=5, dim=16, hidden=24, work=5 * A, work_bytes=1 << 20)
    a.update(change)
    arb.gated(**a)


def layer_grad(arb, **change):
    a = dict(grad_x=A, grad_w_gate=2 * A, grad_w_up=3 * A, grad_out=4 * A, x=5 * A, w_gate=6 * A, w_up=7 * A, rows=5, dim=16, hidden=24,
             work=8 * A, work_bytes=1 << 30, gate=9 * A, up=10 * A)
    a.update(change)
    arb.gated_grad(**a)


CALLS = [logits, logits_grad, keep, read_back, layer, layer_grad]


def refused(arb, call, match, **change):
    with pytest.raises(arb.ArboretumError, match=match):
        call(arb, **change)


def test_the_calls_as_they_stand_reach_the_device(arb):
    if arb.device_count() == 0:
        for call in CALLS:
            refused(arb, call, "no HIP device")


@pytest.mark.parametrize("call,names", [
    (logits, "logits work top_tokens top_log_probs"), (logits_grad, "grad_logits logits stats"), (keep, "codes scales x"),
    (read_back, "codes scales x"), (layer, "out x w_gate w_up"), (layer_grad, "grad_out x w_gate w_up work")])
def test_null_pointers(arb, call, names):
    for name in names.split():
        change = {name: None}
        if name == "work" and call is logits:
            change.update(vocab=100_000)
        refused(arb, call, "null pointer argument", **change)


@pytest.mark.parametrize("call,names", [
    (logits, "log_probs logits tokens entropy top_tokens top_log_probs"), (logits_grad, "grad_logits grad_log_probs logits tokens"),
    (keep, "scales x"), (read_back, "scales x"), (layer, "out x w_gate w_up"), (layer_grad, "grad_x grad_w_gate grad_w_up grad_out x w_gate w_up gate up")])
def test_pointers_that_are_not_aligned_to_their_elements(arb, call, names):
    for name in names.split():
        refused(arb, call, "not aligned", **{name: A + 2})
    for name, by in [("stats", 4)] if call in (logits, logits_grad) else []:
        refused(arb, call, "not aligned", **{name: A + by})
    if call in (logits, logits_grad):
        refused(arb, call, "not aligned", tokens=A + 4, token_bits=64)
        refused(arb, call, "not aligned", status=A + 2)
    if call in (layer, layer_grad):
        scales = dict(gate=A, up=A, gate_scales=A, up_scales=A)
        refused(arb, call, "not aligned", **{**scales, "gate_scales": A + 2})
        refused(arb, call, "not aligned", **{**scales, "up_scales": A + 2})
        refused(arb, call, "not aligned", dtype="bfloat16", x=A + 1)
        refused(arb, call, "not aligned", gate=A + 2, up=A)


def test_work_memory(arb):
    need = arb.log_probs_bytes(4, 100_000, top=3)
    assert need > 0
    refused(arb, logits, "too small: %d bytes" % need, vocab=100_000, work_bytes=need - 1)
    refused(arb, logits, "too small", vocab=100_000, work_bytes=-1)
    refused(arb, logits, "work is not aligned", vocab=100_000, work=A + 8)
    need = arb.gated_grad_bytes(5, 16, 24)
    refused(arb, layer_grad, "too small: %d bytes" % need, work_bytes=need - 1)
    refused(arb, layer_grad, "work is not aligned", work=A + 8)


@pytest.mark.parametrize("call", CALLS)
def test_unknown_names(arb, call):
    refused(arb, call, "element type", dtype="float64")
    refused(arb, call, "element type", dtype=None)
    if call in (layer, layer_grad):
        refused(arb, call, "activation", activation="tanh")
        refused(arb, call, "activation", activation=0)


@pytest.mark.parametrize("call,name,values,match", [
    (logits, "n", [-1, 1 << 31], "bad number of rows"), (logits_grad, "n", [-1, 1 << 31], "bad number of rows"),
    (logits, "vocab", [-1, 0, 1 << 31], "bad number of classes"), (logits_grad, "vocab", [-1, 0, 1 << 31], "bad number of classes"),
    (logits, "top", [-1, 65], "top must be"), (logits, "token_bits", [16, 0, -32], "32 or 64"), (logits_grad, "token_bits", [8], "32 or 64"),
    (logits, "row_stride", [-1], "negative"), (logits, "class_stride", [-1], "negative"), (logits, "row_stride", [1 << 62], "too large"),
    (logits_grad, "grad_row_stride", [-1], "negative"), (logits_grad, "grad_class_stride", [1 << 61], "too large"),
    (logits, "scale", [0.0, -1.0, float("nan"), float("inf"), 1e-40, 1e39, 3.3e38], "scale must be"),
    (logits_grad, "scale", [0.0, -1.0, float("nan"), float("inf")], "scale must be"),
    (keep, "rows", [-1, 1 << 31], "bad number of rows"), (keep, "dim", [0, -1, (1 << 24) + 1], "bad dimension"), (keep, "x_stride", [-1, 1 << 31], "stride"),
    (read_back, "rows", [-1, 1 << 31], "bad number of rows"), (read_back, "dim", [0], "bad dimension"), (read_back, "x_stride", [99], "overlap"),
    (layer, "rows", [-1, 1 << 31], "bad number of rows"), (layer, "dim", [0, -5, (1 << 24) + 1], "bad dimension"),
    (layer, "hidden", [0, (1 << 24) + 1], "bad hidden dimension"), (layer, "out_stride", [23, -1, 1 << 31], "bad stride of out"),
    (layer, "x_stride", [-1], "bad stride of x"), (layer, "w_stride", [-1], "bad stride of the weights"),
    (layer_grad, "rows", [-1, 1 << 31], "bad number of rows"), (layer_grad, "dim", [0], "bad dimension"), (layer_grad, "hidden", [0], "bad hidden"),
    (layer_grad, "grad_x_stride", [15, -1], "bad stride of grad_x"), (layer_grad, "grad_w_stride", [15], "bad stride of the weights' gradients"),
    (layer_grad, "kept_stride", [23], "bad stride of gate and up"), (layer_grad, "grad_out_stride", [-1], "bad stride of grad_out")])
def test_sizes_and_strides(arb, call, name, values, match):
    for value in values:
        refused(arb, call, match, **{name: value})


@pytest.mark.parametrize("call,words,long_words", [
    (logits, "top token_bits", "n vocab row_stride class_stride"), (logits_grad, "token_bits", "n vocab row_stride class_stride grad_row_stride grad_class_stride"),
    (keep, "dim", "rows x_stride"), (read_back, "dim", "rows x_stride"), (layer, "dim hidden", "rows out_stride kept_stride x_stride w_stride"),
    (layer_grad, "dim hidden", "rows grad_x_stride grad_w_stride grad_out_stride kept_stride x_stride w_stride")])
def test_integers_that_their_words_do_not_hold(arb, call, words, long_words):
    for names, bits in ((words, 32), (long_words, 64)):
        for name in names.split():
            for by in (1 << bits, -(1 << bits)):
                refused(arb, call, "does not fit into %d bits" % bits, **{name: 16 + by})


@pytest.mark.parametrize("name", ["log_probs_bytes", "gated_bytes", "gated_grad_bytes"])
def test_work_memory_of_sizes_that_are_refused(arb, name):
    sizes = dict(n=4, vocab=100) if name == "log_probs_bytes" else dict(rows=4, dim=8, hidden=8)
    for key, bits in [("n", 64), ("vocab", 64)] if name == "log_probs_bytes" else [("rows", 64), ("dim", 32), ("hidden", 32)]:
        for value in (-1, (1 << bits) + 4):
            with pytest.raises(arb.ArboretumError):
                getattr(arb, name)(**{**sizes, key: value})


def test_what_goes_together(arb):
    refused(arb, logits, "tokens and log_probs go together", tokens=None)
    refused(arb, logits, "tokens and log_probs go together", log_probs=None)
    refused(arb, logits, "more than there are classes", vocab=2)
    refused(arb, logits_grad, "tokens and grad_log_probs go together", tokens=None)
    refused(arb, logits_grad, "tokens and grad_log_probs go together", grad_log_probs=None)
    refused(arb, logits_grad, "entropy go together", grad_entropy=A)
    refused(arb, logits_grad, "entropy go together", entropy=A)
    refused(arb, logits_grad, "rows of the gradient overlap", grad_row_stride=99)
    refused(arb, logits_grad, "rows of the gradient overlap", grad_row_stride=0)
    refused(arb, logits_grad, "rows of the gradient overlap", grad_class_stride=0)
    refused(arb, logits_grad, "rows of the gradient overlap", grad_row_stride=2, grad_class_stride=2)
    refused(arb, logits_grad, "rows of the gradient overlap", grad_row_stride=1, grad_class_stride=3)
    refused(arb, logits_grad, "has their strides", grad_logits=3 * A, grad_row_stride=101)
    for call in (layer, layer_grad):
        refused(arb, call, "gate and up go together", gate=A, up=None)
        refused(arb, call, "gate and up go together", gate=A, up=A, gate_scales=A)
    refused(arb, layer, "scales without", gate_scales=A, up_scales=A)
    refused(arb, layer_grad, "null pointer", gate=None, up=None)
    refused(arb, layer_grad, "both weights go together", grad_w_gate=None)


def test_calls_of_nothing_need_no_device(arb):
    logits(arb, n=0, logits=None, tokens=None, log_probs=None, work=None, work_bytes=0, entropy=None, stats=None, top_tokens=None, top_log_probs=None)
    logits(arb, tokens=None, log_probs=None, entropy=None, stats=None, top=0)
    logits_grad(arb, n=0)
    keep(arb, rows=0, x=None, codes=None, scales=None)
    read_back(arb, rows=0, x=None, codes=None, scales=None)
    layer(arb, rows=0, x=None, out=None)
    layer_grad(arb, grad_x=None, grad_w_gate=None, grad_w_up=None)


def test_work_memory_of_ordinary_sizes(arb):
    assert arb.log_probs_bytes(0, 100) == 0 and arb.log_probs_bytes(1, 100, top=5) == 0 and arb.log_probs_bytes(4096, 131_072, top=20) == 0
    assert arb.log_probs_bytes(1, 131_072, top=20) < 1 << 20
    # both rounded factors, rows apart by whole tiles, and shares of the products of at most a few outputs
    assert 2 * 8192 * 16384 * 2 <= arb.gated_grad_bytes(8192, 4096, 16384, dtype="bfloat16") < 3 * 8192 * 16384 * 2


def test_outputs_that_meet_inputs_or_each_other(arb):
    for name in ("logits", "tokens"):
        refused(arb, logits, "an output and an input overlap", **{name: 5 * A})
    refused(arb, logits, "two outputs overlap", entropy=A + 12)
    refused(arb, logits, "two outputs overlap", top_tokens=8 * A - 44)
    refused(arb, logits, "an output and an input overlap", logits=2 * A, log_probs=2 * A + 1596)
    refused(arb, logits, "an output and an input overlap", logits=2 * A, row_stride=1, class_stride=4, log_probs=2 * A + 1584)
    refused(arb, logits, "an output and an input overlap", status=3 * A + 4)
    refused(arb, logits_grad, "an output and an input overlap", grad_logits=3 * A + 400)
    for name in ("tokens", "stats", "grad_log_probs"):
        refused(arb, logits_grad, "an output and an input overlap", **{name: A + 4 * 392})
    refused(arb, keep, "an output and an input overlap", codes=3 * A + 1596)
    refused(arb, keep, "two outputs overlap", codes=2 * A + 28)
    refused(arb, read_back, "an output and an input overlap", x=2 * A - 1596)
    for name in ("x", "w_gate", "w_up"):
        refused(arb, layer, "an output and an input overlap", **{name: A})
    refused(arb, layer, "two outputs overlap", gate=9 * A, up=9 * A)
    refused(arb, layer, "two outputs overlap", gate=9 * A, up=A + 476)
    refused(arb, layer, "two outputs overlap", gate=9 * A, up=10 * A, gate_scales=11 * A, up_scales=11 * A + 16)
    for name in ("grad_out", "x", "w_gate", "w_up", "gate", "up"):
        for output in (A, 2 * A, 3 * A, 8 * A):
            refused(arb, layer_grad, "an output and an input overlap", **{name: output})
    refused(arb, layer_grad, "two outputs overlap", grad_w_gate=3 * A)


def test_rows_that_lie_between_each_other_do_not_meet(arb):
    # the columns of one matrix: gate beside up, a result beside its input
    if arb.device_count() == 0:
        for call, change in [
                (layer, dict(gate=9 * A, up=9 * A + 96, kept_stride=48)),
                (layer, dict(out=2 * A + 64, out_stride=40, x_stride=40)),
                (layer_grad, dict(grad_w_gate=2 * A, grad_w_up=2 * A + 64, grad_w_stride=32)),
                (layer_grad, dict(x=A + 64, x_stride=32, grad_x_stride=32)),
                (logits_grad, dict(grad_logits=3 * A + 400, row_stride=200)),
                (logits_grad, dict(grad_logits=3 * A + 16, row_stride=1, class_stride=8)),
                (keep, dict(codes=3 * A + 400 * 4)),
                (read_back, dict(codes=A + 400 * 4))]:
            refused(arb, call, "no HIP device", **change)
        refused(arb, layer, "two outputs overlap", gate=9 * A, up=9 * A + 92, kept_stride=48)
        refused(arb, layer, "two outputs overlap", gate=9 * A, up=9 * A + 100, kept_stride=48)
