"""The operators of a model on top of embeddings as cases that can be timed: its gated layers, what they keep for the
backward pass, and the log probabilities that it answers with and learns from.

  log_probs   of the given token of each row of logits, with the entropy of the row and its `top` likeliest tokens
  loss        the same without the top, and the gradient of the logits: a training step's end
  gated       act(x Wg^T) * (x Wu^T)
  step        the same with its gradients; what the backward pass needs is kept as it is, or in 8 bits
  checkpoint  activations kept in 8 bits, a scale for every 64 values of a row, and read back

A token of -1 stands for none.  `own` chooses between the plain form in elementary torch operations and this package's
entry points."""
import math

import torch

own = False

GROUP = 64  # values of a row that share a scale


def _logits(name, kind, n, vocab, dtype, **more):
    case = {"name": name, "kind": kind, "n": n, "vocab": vocab, "dtype": dtype, "order": "rows", "top": 0, "padding": 0.0,
            "masked": 0.0, "scale": 1.0, "entropy_weight": 0.0}
    case.update(more)
    return case


def _layer(name, kind, rows, dim, hidden, dtype, **more):
    case = {"name": name, "kind": kind, "rows": rows, "dim": dim, "hidden": hidden, "dtype": dtype, "activation": "silu",
            "kept": "as is"}
    case.update(more)
    return case


def listed():
    return [
        # The next token of one sequence, its entropy and the twenty likeliest: an answer's log probabilities.
        _logits("log_probs_token", "log_probs", 1, 131_072, "bfloat16", top=20),
        # The log probabilities of a million rows under ten classes, as a booster holds its scores: class by class.
        _logits("log_probs_classes", "log_probs", 1_000_003, 10, "float32", order="columns", top=3),
        # Short padded sequences scored at a temperature, a vocabulary that divides nothing, a fifth of it ruled out.
        _logits("log_probs_ragged", "log_probs", 777, 50_021, "float16", top=5, padding=0.2, masked=0.2, scale=1 / 0.7),
        # A training batch's loss over a large vocabulary.
        _logits("loss_batch", "loss", 4_096, 131_072, "bfloat16"),
        # Odd sizes, padding, and an entropy that takes part in the loss.
        _logits("loss_ragged", "loss", 777, 50_021, "float16", padding=0.2, scale=1.3, entropy_weight=0.01),
        # A model that answers row by row: the weights are read for one row.
        _layer("gated_token", "gated", 1, 4_096, 16_384, "bfloat16"),
        # A whole batch.
        _layer("gated_batch", "gated", 8_192, 4_096, 16_384, "bfloat16"),
        # Sizes that divide nothing, rows that begin anywhere.
        _layer("gated_ragged", "gated", 1_003, 771, 2_055, "float16", activation="gelu"),
        # A training step of a large layer.
        _layer("step_batch", "step", 4_096, 4_096, 16_384, "bfloat16"),
        # A layer over the leaf vectors of a hundred thousand rows, its activations kept in 8 bits.
        _layer("step_leaf_vectors", "step", 100_003, 64, 256, "bfloat16", kept="8 bits"),
        # The activations of a batch, kept and read back.
        {"name": "checkpoint_batch", "kind": "checkpoint", "rows": 65_536, "dim": 4_096, "dtype": "bfloat16"},
        # Those of a small one, of an odd width.
        {"name": "checkpoint_ragged", "kind": "checkpoint", "rows": 1_003, "dim": 771, "dtype": "float16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["log_probs", "log_probs", "loss", "gated", "gated", "step", "step", "checkpoint"])
    if kind == "checkpoint":
        dim = _log(rng, 16, 16_384)
        return {"kind": kind, "rows": min(_log(rng, 1, 300_000), (1 << 28) // dim), "dim": dim,
                "dtype": rng.choice(["bfloat16", "float16"])}
    if kind in ("log_probs", "loss"):
        if rng.random() < 0.3:  # classes
            vocab, order, dtype = _log(rng, 2, 100), rng.choice(["rows", "columns"]), "float32"
            n = min(_log(rng, 100, 2_000_000), (1 << 27) // vocab)
        else:
            vocab, order, dtype = _log(rng, 1_000, 200_000), "rows", rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
            n = min(_log(rng, 1, 8_192), (1 << 28) // vocab)
        case = {"kind": kind, "n": n, "vocab": vocab, "dtype": dtype, "order": order, "padding": rng.choice([0.0, 0.3]),
                "masked": rng.choice([0.0, 0.0, 0.5]), "scale": rng.choice([1.0, 0.6, 1.7]), "top": 0, "entropy_weight": 0.0}
        if kind == "log_probs":
            case["top"] = min(rng.choice([0, 1, 5, 20, 64]), max(1, vocab // 2))
        else:
            case["entropy_weight"] = rng.choice([0.0, 0.02])
        return case
    if rng.random() < 0.3:  # a small layer over many rows
        dim, hidden, rows = _log(rng, 8, 512), _log(rng, 8, 1_024), _log(rng, 1_000, 200_000)
    else:
        dim, hidden, rows = _log(rng, 64, 8_192), _log(rng, 64, 16_384), _log(rng, 1, 8_192)
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    most = 1.5e12 if dtype != "float32" else 1.5e11
    if kind == "step":
        most /= 3
    rows = max(1, min(rows, int(most / (4.0 * dim * hidden))))
    return {"kind": kind, "rows": rows, "dim": dim, "hidden": hidden, "dtype": dtype, "activation": rng.choice(["silu", "gelu"]),
            "kept": "8 bits" if kind == "step" and dtype != "float32" and rng.random() < 0.5 else "as is"}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["kind"] == "checkpoint":
        # some columns of a layer's activations are much larger than others
        x = normal(case["rows"], case["dim"]).mul_(torch.exp(0.7 * normal(case["dim"])))
        return {"case": case, "x": x.to(dtype)}
    if case["kind"] in ("gated", "step"):
        rows, dim, hidden = case["rows"], case["dim"], case["hidden"]
        state = {"case": case, "x": normal(rows, dim).to(dtype), "w_gate": (normal(hidden, dim) / math.sqrt(dim)).to(dtype),
                 "w_up": (normal(hidden, dim) / math.sqrt(dim)).to(dtype)}
        if case["kind"] == "step":
            state["grad_out"] = normal(rows, hidden).to(dtype)
        return state
    n, vocab = case["n"], case["vocab"]
    tokens = torch.randint(0, vocab, (n,), generator=gen, device="cuda", dtype=torch.int32)
    # a model favours some tokens: those given, and a few more of each row
    logits = normal(n, vocab).mul_(2.0)
    logits.scatter_add_(1, tokens[:, None].long(), 4.0 * torch.rand(n, 1, generator=gen, device="cuda"))
    for _ in range(3):
        some = torch.randint(0, vocab, (n, 1), generator=gen, device="cuda")
        logits.scatter_add_(1, some, 6.0 * torch.rand(n, 1, generator=gen, device="cuda"))
    if case["masked"] > 0:  # tokens that an answer may not hold, the same for all rows
        out = torch.rand(vocab, generator=gen, device="cuda") < case["masked"]
        out[0] = False
        tokens = torch.where(out[tokens.long()], 0, tokens)
        logits[:, out] = -math.inf
    if case["padding"] > 0:
        tokens = torch.where(torch.rand(n, generator=gen, device="cuda") < case["padding"], -1, tokens)
    logits = logits.to(dtype)
    state = {"case": case, "logits": logits.t().contiguous() if case["order"] == "columns" else logits, "tokens": tokens}
    if case["kind"] == "loss":
        # the mean over the rows that count, scaled up where 16 bits have few exponents
        weight = (65_536.0 if case["dtype"] == "float16" else 1.0) / n
        state["grad_log_probs"] = torch.where(tokens >= 0, -weight / (1.0 - case["padding"]), 0.0)
        if case["entropy_weight"] > 0:
            state["grad_entropy"] = torch.full((n,), -case["entropy_weight"] * weight, device="cuda")
    return state


# ---- the plain forms

def _activation(name, g):
    """act(g) and its derivative"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1.0 + g * (1.0 - s))
    phi = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _quantised(x):
    """codes [rows][groups][GROUP] and scales [rows][groups] of what is kept in 8 bits"""
    rows, dim = x.shape
    groups = (dim + GROUP - 1) // GROUP
    if dim % GROUP:
        x = torch.cat([x, x.new_zeros(rows, groups * GROUP - dim)], 1)
    x = x.reshape(rows, groups, GROUP)
    scale = x.abs().amax(2) / 127.0
    codes = torch.round(x / torch.where(scale > 0, scale, 1.0)[..., None])
    return codes.to(torch.int8), scale


def _restored(codes, scale, dim):
    return (codes.float() * scale[..., None]).reshape(codes.shape[0], -1)[:, :dim]


def _plain_checkpoint(state):
    x = state["x"]
    codes, scale = _quantised(x.float())
    return {"x": _restored(codes, scale, x.shape[1]).to(x.dtype), "scales": scale}


def _plain_gated(state):
    x = state["x"].float()
    g, u = x @ state["w_gate"].float().t(), x @ state["w_up"].float().t()
    return (_activation(state["case"]["activation"], g)[0] * u).to(state["x"].dtype)


def _plain_step(state):
    case, dtype = state["case"], state["x"].dtype
    x, w_gate, w_up, grad = state["x"].float(), state["w_gate"].float(), state["w_up"].float(), state["grad_out"].float()
    g, u = x @ w_gate.t(), x @ w_up.t()
    out = (_activation(case["activation"], g)[0] * u).to(dtype)
    if case["kept"] == "8 bits":
        kept_x, kept_g, kept_u = _quantised(x), _quantised(g), _quantised(u)
        x, g, u = _restored(*kept_x, case["dim"]), _restored(*kept_g, case["hidden"]), _restored(*kept_u, case["hidden"])
    a, slope = _activation(case["activation"], g)
    dg, du = grad * u * slope, grad * a
    return {"out": out, "grad_x": (dg @ w_gate + du @ w_up).to(dtype), "grad_w_gate": (dg.t() @ x).to(dtype),
            "grad_w_up": (du.t() @ x).to(dtype)}


def _plain_log_probs(state):
    case, tokens = state["case"], state["tokens"].long()
    columns = case["order"] == "columns"
    x = state["logits"].t() if columns else state["logits"]
    z = x.float() * case["scale"]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1)
    rest = torch.log(total)
    given = z.gather(1, tokens.clamp(min=0)[:, None])[:, 0] - rest
    out = {"log_probs": torch.where(tokens >= 0, given, 0.0),
           "entropy": rest - (e * torch.where(e > 0, z, 0.0)).sum(1) / total}
    if case["top"]:
        # in order of the logits, equal ones by their index: as one whole number
        bits = (x.float() + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + (case["vocab"] - 1 - torch.arange(case["vocab"], device="cuda"))
        top = torch.topk(key, case["top"], dim=1).indices
        out["top"] = top.to(torch.int32)
        out["top_log_probs"] = z.gather(1, top) - rest[:, None]
    if case["kind"] == "loss":
        p = e / total[:, None]
        grad = -p * state["grad_log_probs"][:, None]
        grad.scatter_add_(1, tokens.clamp(min=0)[:, None], state["grad_log_probs"][:, None])
        if case["entropy_weight"] > 0:
            log_p = torch.where(p > 0, z - rest[:, None], 0.0)
            grad -= state["grad_entropy"][:, None] * p * (log_p + out["entropy"][:, None])
        grad = (grad * case["scale"]).to(x.dtype)
        out["grad"] = grad.t().contiguous() if columns else grad
    return out


# ---- the package's entry points

def _own_checkpoint(state):
    import arboretum_amd as arb
    case, x = state["case"], state["x"]
    rows, dim = x.shape
    stream = torch.cuda.current_stream().cuda_stream
    codes = torch.empty(rows, dim, device="cuda", dtype=torch.int8)
    scales = torch.empty(rows, (dim + GROUP - 1) // GROUP, device="cuda")
    arb.activation_checkpoint(codes.data_ptr(), scales.data_ptr(), x.data_ptr(), rows, dim, dtype=case["dtype"], stream=stream)
    back = torch.empty_like(x)
    arb.activation_restore(back.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, dim, dtype=case["dtype"], stream=stream)
    return {"x": back, "scales": scales}


def _work(state, size):
    """Work memory, kept from step to step."""
    if "work" not in state:
        state["work"] = torch.empty(max(size, 16), device="cuda", dtype=torch.uint8)
    return state["work"]


def _own_gated(state):
    import arboretum_amd as arb
    case, x = state["case"], state["x"]
    rows, dim, hidden = case["rows"], case["dim"], case["hidden"]
    work = _work(state, arb.gated_bytes(rows, dim, hidden, dtype=case["dtype"]))
    out = torch.empty(rows, hidden, device="cuda", dtype=x.dtype)
    arb.gated(out.data_ptr(), x.data_ptr(), state["w_gate"].data_ptr(), state["w_up"].data_ptr(), rows, dim, hidden, work.data_ptr(),
              work.numel(), activation=case["activation"], dtype=case["dtype"], stream=torch.cuda.current_stream().cuda_stream)
    return out


def _own_step(state):
    import arboretum_amd as arb
    case, x = state["case"], state["x"]
    rows, dim, hidden, eight = case["rows"], case["dim"], case["hidden"], case["kept"] == "8 bits"
    stream = torch.cuda.current_stream().cuda_stream
    more = {"activation": case["activation"], "dtype": case["dtype"], "stream": stream}
    work = _work(state, max(arb.gated_bytes(rows, dim, hidden, dtype=case["dtype"]),
                            arb.gated_grad_bytes(rows, dim, hidden, dtype=case["dtype"])))
    w_gate, w_up = state["w_gate"].data_ptr(), state["w_up"].data_ptr()
    kept = torch.empty(2, rows, hidden, device="cuda", dtype=torch.int8 if eight else x.dtype)
    held = {"gate": kept[0].data_ptr(), "up": kept[1].data_ptr()}
    if eight:
        scales = torch.empty(2, rows, (hidden + GROUP - 1) // GROUP, device="cuda")
        held.update(gate_scales=scales[0].data_ptr(), up_scales=scales[1].data_ptr())
        codes = torch.empty(rows, dim, device="cuda", dtype=torch.int8)
        x_scales = torch.empty(rows, (dim + GROUP - 1) // GROUP, device="cuda")
        arb.activation_checkpoint(codes.data_ptr(), x_scales.data_ptr(), x.data_ptr(), rows, dim, dtype=case["dtype"], stream=stream)
    out = torch.empty(rows, hidden, device="cuda", dtype=x.dtype)
    arb.gated(out.data_ptr(), x.data_ptr(), w_gate, w_up, rows, dim, hidden, work.data_ptr(), work.numel(), **held, **more)
    if eight:
        x = torch.empty_like(x)
        arb.activation_restore(x.data_ptr(), codes.data_ptr(), x_scales.data_ptr(), rows, dim, dtype=case["dtype"], stream=stream)
    grad_x, grad_w = torch.empty_like(x), torch.empty(2, hidden, dim, device="cuda", dtype=x.dtype)
    arb.gated_grad(grad_x.data_ptr(), grad_w[0].data_ptr(), grad_w[1].data_ptr(), state["grad_out"].data_ptr(), x.data_ptr(), w_gate,
                   w_up, rows, dim, hidden, work.data_ptr(), work.numel(), **held, **more)
    return {"out": out, "grad_x": grad_x, "grad_w_gate": grad_w[0], "grad_w_up": grad_w[1]}


def _own_log_probs(state):
    import arboretum_amd as arb
    case, logits, tokens = state["case"], state["logits"], state["tokens"]
    n, vocab, top, columns = case["n"], case["vocab"], case["top"], case["order"] == "columns"
    more = {"scale": case["scale"], "dtype": case["dtype"], "stream": torch.cuda.current_stream().cuda_stream}
    if columns:
        more.update(row_stride=1, class_stride=n)
    work = _work(state, arb.log_probs_bytes(n, vocab, top=top))
    out = {"log_probs": torch.empty(n, device="cuda"), "entropy": torch.empty(n, device="cuda")}
    held = dict(more)
    if top:
        out["top"] = torch.empty(n, top, device="cuda", dtype=torch.int32)
        out["top_log_probs"] = torch.empty(n, top, device="cuda")
        held.update(top=top, top_tokens=out["top"].data_ptr(), top_log_probs=out["top_log_probs"].data_ptr())
    if case["kind"] == "loss":
        stats = torch.empty(n, 2, device="cuda")
        held["stats"] = stats.data_ptr()
    arb.log_probs(out["log_probs"].data_ptr(), logits.data_ptr(), tokens.data_ptr(), n, vocab, work.data_ptr(), work.numel(),
                  entropy=out["entropy"].data_ptr(), **held)
    if case["kind"] == "loss":
        if case["entropy_weight"] > 0:
            more.update(grad_entropy=state["grad_entropy"].data_ptr(), entropy=out["entropy"].data_ptr())
        out["grad"] = torch.empty_like(logits)
        arb.log_probs_grad(out["grad"].data_ptr(), state["grad_log_probs"].data_ptr(), logits.data_ptr(), tokens.data_ptr(),
                           stats.data_ptr(), n, vocab, **more)
    return out


_PLAIN = {"log_probs": _plain_log_probs, "loss": _plain_log_probs, "gated": _plain_gated, "step": _plain_step,
          "checkpoint": _plain_checkpoint}
_OWN = {"log_probs": _own_log_probs, "loss": _own_log_probs, "gated": _own_gated, "step": _own_step, "checkpoint": _own_checkpoint}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---- what a pass cannot do without, and its result in 64 bits

def work(case):
    item = 4 if case["dtype"] == "float32" else 2
    kind = case["kind"]
    if kind == "checkpoint":
        every = case["rows"] * case["dim"]
        return {"bytes": every * 2 * (item + 1 + 4 / GROUP), "flops": 5 * every}
    if kind in ("gated", "step"):
        rows, dim, hidden = case["rows"], case["dim"], case["hidden"]
        moved, flops = (rows * dim + 2 * hidden * dim + rows * hidden) * item, 4.0 * rows * dim * hidden
        if kind == "step":  # and the output's gradient read, those of input and weights written
            moved, flops = moved + (rows * hidden + rows * dim + 2 * hidden * dim) * item, 3 * flops
        return {"bytes": moved, "flops": flops}
    every = case["n"] * case["vocab"]
    moved, flops = every * item + case["n"] * (12 + 8 * case["top"]), 6 * every
    if kind == "loss":  # (the logits once, their gradients once)
        moved, flops = moved + every * item, 2 * flops
    return {"bytes": moved, "flops": flops}


def _kept_64(v):
    """What 8 bits keep of v: the scale is held in 32 bits."""
    out = torch.empty_like(v)
    for c in range(0, v.shape[1], GROUP):
        part = v[:, c:c + GROUP]
        scale = (part.abs().max(1, keepdim=True).values / 127).float().double()
        out[:, c:c + GROUP] = torch.nan_to_num(part / scale).round() * scale
    return out


def _exact_layer(case, state):
    x, w_gate, w_up = state["x"].double(), state["w_gate"].double(), state["w_up"].double()
    g, u = torch.mm(x, w_gate.t()), torch.mm(x, w_up.t())

    def act(v):
        if case["activation"] == "silu":
            return v / (1 + torch.exp(-v))
        return v * torch.special.ndtr(v)

    out = act(g) * u
    if case["kind"] == "gated":
        return out
    if case["kept"] == "8 bits":
        x, g, u = _kept_64(x), _kept_64(g), _kept_64(u)
    if case["activation"] == "silu":
        slope = (1 + torch.exp(-g) * (1 + g)) / (1 + torch.exp(-g)) ** 2
    else:
        slope = torch.special.ndtr(g) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    grad = state["grad_out"].double()
    du = grad * act(g)
    dg = grad * u * slope
    return {"out": out, "grad_x": torch.mm(dg, w_gate) + torch.mm(du, w_up), "grad_w_gate": torch.mm(x.t(), dg).t(),
            "grad_w_up": torch.mm(x.t(), du).t()}


def _exact_logits(case, state):
    columns, k, loss = case["order"] == "columns", case["top"], case["kind"] == "loss"
    parts, at = [], max(1, (1 << 26) // case["vocab"])
    for r in range(0, case["n"], at):
        rows = (state["logits"][:, r:r + at].t() if columns else state["logits"][r:r + at]).double()
        token = state["tokens"][r:r + at].long()
        log_p = torch.log_softmax(rows * case["scale"], 1)
        p = torch.exp(log_p)
        finite = torch.where(p > 0, log_p, 0.0)
        entropy = -(p * finite).sum(1)
        named = token >= 0
        one = torch.zeros_like(token, dtype=torch.float64)
        one[named] = log_p[named, token[named]]
        part = {"log_probs": one, "entropy": entropy}
        if k:
            part["top_log_probs"] = torch.sort(log_p, 1, descending=True).values[:, :k]
        if loss:
            weight = state["grad_log_probs"][r:r + at].double()
            hit = torch.zeros_like(p)
            hit[named, token[named]] = 1
            grad = weight[:, None] * (hit - p)
            if case["entropy_weight"] > 0:
                grad = grad - state["grad_entropy"][r:r + at].double()[:, None] * p * (finite + entropy[:, None])
            part["grad"] = grad * case["scale"]
        parts.append(part)
    out = {name: torch.cat([part[name] for part in parts]) for name in parts[0]}
    if loss and columns:
        out["grad"] = out["grad"].t().contiguous()
    if k:
        out["top"] = None
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "checkpoint":
        x = state["x"].double()
        scales = torch.stack([x[:, c:c + GROUP].abs().max(1).values / 127 for c in range(0, case["dim"], GROUP)], 1)
        return {"x": _kept_64(x), "scales": scales}
    return (_exact_layer if case["kind"] in ("gated", "step") else _exact_logits)(case, state)
