"""The operators for embeddings over tokens as cases that can be timed: a table of embeddings looked up, its gradient, and
the optimizer's step over the tables.

  lookup  out[i] = scale * (sum of table[token] over the bag of tokens of row i).  A bag of one is a model's input
          embedding; a bag of one leaf per tree is how the rows of a data matrix meet the leaves of a booster.
  grad    the gradient of the table: grad[v] = scale * (sum of grad_out[i] over the tokens of all bags that are v).
  adamw   one AdamW step over a list of tensors, its two states in 32 bits.

A token of -1 stands for none.  `own` chooses between the plain form in elementary torch operations and this package's
entry points."""
import math

import numpy as np
import torch

own = False

BETA1, BETA2, EPS = 0.9, 0.999, 1e-8


def _lookup(name, n, bag, vocab, dim, dtype, **more):
    case = {"name": name, "kind": "lookup", "n": n, "bag": bag, "vocab": vocab, "dim": dim, "dtype": dtype,
            "order": "rows", "leaves": 0, "padding": 0.0, "scale": 1.0}
    case.update(more)
    return case


def _grad(name, n, bag, vocab, dim, dtype, grad_dtype, **more):
    case = _lookup(name, n, bag, vocab, dim, dtype, **more)
    case.update(kind="grad", grad_dtype=grad_dtype)
    return case


def listed():
    return [
        # A model that answers token by token looks up the last one: latency is all there is.
        _lookup("lookup_token", 1, 1, 32_000, 4096, "bfloat16", scale=64.0),
        # The input embedding of a batch of long sequences.
        _lookup("lookup_batch", 65_536, 1, 131_072, 4096, "bfloat16"),
        # A ragged batch: padded positions, a width and a vocabulary that divide nothing.
        _lookup("lookup_ragged", 5_003, 1, 50_021, 771, "float16", padding=0.2, scale=27.77),
        # A million rows against the leaves of 200 trees of depth 8, as the trees hand them out (tree by tree).
        _lookup("lookup_leaves", 1_000_003, 200, 200 * 256, 1, "float32", order="columns", leaves=256),
        # Leaf embeddings of a hundred trees for a model on top of the booster, tokens row by row.
        _lookup("lookup_leaf_vectors", 100_003, 100, 100 * 64, 16, "bfloat16", leaves=64),
        # The gradient of a small table of categories.
        _grad("grad_small", 64, 1, 1_000, 64, "float32", "float32"),
        # A training batch: gradients in 16 bits, the table's gradient kept in 32.
        _grad("grad_batch", 32_768, 1, 65_536, 4096, "bfloat16", "float32", scale=64.0),
        # Short padded sequences, odd sizes, gradients in 16 bits throughout.
        _grad("grad_ragged", 5_003, 1, 50_021, 771, "float16", "float16", padding=0.2, scale=2.5),
        # Leaf weights: half a million rows, a hundred trees, a few thousand rows to a leaf.
        _grad("grad_leaves", 500_009, 100, 100 * 256, 1, "float32", "float32", order="columns", leaves=256),
        # The leaf tables of ten classes.
        {"name": "adamw_tables", "kind": "adamw", "tensors": 10, "largest": 6_400, "spread": 0.0, "align": 64,
         "dtype": "float32", "grad_dtype": "float32", "decay": 0.0, "grad_scale": 1.0},
        # The tensors of a model trained in 32 bits: matrices and vectors of many sizes, back to back in one buffer.
        {"name": "adamw_many", "kind": "adamw", "tensors": 300, "largest": 2_000_000, "spread": 3.0, "align": 1,
         "dtype": "float32", "grad_dtype": "float32", "decay": 0.01, "grad_scale": 0.25},
        # Large matrices held and differentiated in 16 bits.
        {"name": "adamw_16bit", "kind": "adamw", "tensors": 16, "largest": 16_777_216, "spread": 0.5, "align": 64,
         "dtype": "bfloat16", "grad_dtype": "bfloat16", "decay": 0.1, "grad_scale": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lookup", "lookup", "grad", "grad", "adamw"])
    if kind == "adamw":
        tensors = _log(rng, 1, 400)
        dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
        return {"kind": kind, "tensors": tensors, "largest": min(_log(rng, 100, 16_777_216), 150_000_000 // tensors),
                "spread": rng.choice([0.0, 0.5, 3.0]), "align": rng.choice([1, 64]), "dtype": dtype,
                "grad_dtype": rng.choice([dtype, "bfloat16"]), "decay": rng.choice([0.0, 0.1]),
                "grad_scale": rng.choice([1.0, 0.125])}
    of = rng.choice(["text", "text", "leaves", "categories"])
    if of == "text":  # one token a row
        bag, leaves, order = 1, 0, "rows"
        vocab, dim = _log(rng, 1_000, 131_072), _log(rng, 64, 8_192)
        n = min(_log(rng, 1, 65_536), (1 << 27) // dim)
        if kind == "grad":
            vocab = min(vocab, (1 << 27) // dim)
        dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    else:
        leaves = rng.choice([8, 64, 256]) if of == "leaves" else 0
        bag = _log(rng, 2, 200)
        vocab = bag * leaves if leaves else _log(rng, 1_000, 200_000)
        dim = rng.choice([1, 1, 1, 3, 8, 16, 33])
        n = min(_log(rng, 100, 1_000_003), 48_000_000 // (bag * dim))
        order = rng.choice(["rows", "columns"])
        dtype = "float32" if dim == 1 else rng.choice(["float32", "bfloat16"])
    case = {"kind": kind, "n": max(1, n), "bag": bag, "vocab": vocab, "dim": dim, "dtype": dtype, "order": order,
            "leaves": leaves, "padding": 0.0 if leaves else rng.choice([0.0, 0.3]), "scale": rng.choice([1.0, 0.37])}
    if kind == "grad":
        case["grad_dtype"] = rng.choice(["float32", dtype])
    return case


def _tokens(case, gen):
    """Tokens [n][bag], or [bag][n] where they come column by column."""
    n, bag, vocab = case["n"], case["bag"], case["vocab"]
    u = torch.rand((bag, n) if case["order"] == "columns" else (n, bag), generator=gen, device="cuda")
    if case["leaves"]:  # some leaves hold many more rows than others
        first = torch.arange(bag, device="cuda", dtype=torch.int32) * case["leaves"]
        leaf = (u * u * case["leaves"]).to(torch.int32).clamp_(max=case["leaves"] - 1)
        return leaf + (first[:, None] if case["order"] == "columns" else first)
    # the frequency of a token falls with its rank, and the ranks lie scattered over the table
    rank = ((vocab + 1.0) ** u.double() - 1.0).long().clamp_(max=vocab - 1)
    step = next(s for s in (7919, 7907, 7901) if vocab % s)
    tokens = ((rank * step + 13) % vocab).to(torch.int32)
    if case["padding"] > 0:
        tokens[torch.rand(tokens.shape, generator=gen, device="cuda") < case["padding"]] = -1
    return tokens


def _sizes(case):
    """(elements of each tensor, where each begins in the buffer, elements of the buffer)"""
    share = np.modf(0.5 + 0.6180339887498949 * np.arange(case["tensors"]))[0] ** case["spread"]
    sizes = np.maximum(1, np.round(case["largest"] * share)).astype(np.int64)
    room = (sizes + case["align"] - 1) // case["align"] * case["align"]
    ends = np.cumsum(room)
    return sizes, ends - room, int(ends[-1])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    if case["kind"] == "adamw":
        sizes, begins, total = _sizes(case)
        real = torch.zeros(total, device="cuda")  # room between two tensors holds zeros and stays as it is
        mark = torch.zeros(total + 1, device="cuda", dtype=torch.int32)
        mark[torch.from_numpy(begins).cuda()] += 1
        mark.index_add_(0, torch.from_numpy(begins + sizes).cuda(), torch.full((len(sizes),), -1, device="cuda", dtype=torch.int32))
        real.copy_(torch.cumsum(mark[:-1], 0) > 0)
        noise = lambda s: torch.randn(total, generator=gen, device="cuda").mul_(s).mul_(real)  # noqa: E731
        buffers = {"p": noise(0.5).to(dtype), "g": noise(0.01).to(getattr(torch, case["grad_dtype"])), "m": noise(0.003),
                   "v": noise(0.01).square_()}
        # a program keeps the addresses of its tensors as it keeps the tensors
        at = {k: b.data_ptr() + begins * b.element_size() for k, b in buffers.items()}
        return {"case": case, **buffers, "at": at, "sizes": sizes, "lr": 1e-3, "step": 10}
    state = {"case": case, "tokens": _tokens(case, gen)}
    if case["kind"] == "lookup":
        state["table"] = torch.randn(case["vocab"], case["dim"], generator=gen, device="cuda").to(dtype)
    else:
        state["grad_out"] = torch.randn(case["n"], case["dim"], generator=gen, device="cuda").to(dtype)
    return state


# ---- the plain forms

def _plain_lookup(state):
    case, table = state["case"], state["table"]
    tokens = state["tokens"].long()
    if case["padding"] > 0:
        rows = torch.where((tokens >= 0)[..., None], table[tokens.clamp(min=0)].float(), 0.0)
    else:
        rows = table[tokens].float()
    return (rows.sum(0 if case["order"] == "columns" else 1) * case["scale"]).to(table.dtype)


def _plain_grad(state):
    case, grad_out = state["case"], state["grad_out"]
    tokens = state["tokens"].long()
    if case["padding"] > 0:
        tokens = torch.where(tokens >= 0, tokens, case["vocab"])
    rows = grad_out.float().unsqueeze(0 if case["order"] == "columns" else 1).expand(*tokens.shape, -1)
    grad = torch.zeros(case["vocab"] + 1, case["dim"], device="cuda")
    grad.index_add_(0, tokens.reshape(-1), rows.reshape(-1, case["dim"]))
    return (grad[:-1] * case["scale"]).to(getattr(torch, case["grad_dtype"]))


def _plain_adamw(state):
    case, m, v = state["case"], state["m"], state["v"]
    state["step"] += 1
    step, lr = state["step"], state["lr"]
    g = state["g"].float() * case["grad_scale"]
    p = state["p"].float() * (1.0 - lr * case["decay"])
    m.mul_(BETA1).add_(g * (1.0 - BETA1))
    v.mul_(BETA2).add_(g * g * (1.0 - BETA2))
    p -= lr / (1.0 - BETA1 ** step) * m / (v.sqrt() / math.sqrt(1.0 - BETA2 ** step) + EPS)
    state["p"].copy_(p)
    return {"p": state["p"], "m": m, "v": v}


# ---- the package's entry points

def _own_lookup(state):
    import arboretum_amd as arb
    case, table, tokens = state["case"], state["table"], state["tokens"]
    n, bag, dim = case["n"], case["bag"], case["dim"]
    out = torch.empty(n, dim, device="cuda", dtype=table.dtype)
    strides = (1, n) if case["order"] == "columns" else (bag, 1)
    arb.embedding(out.data_ptr(), table.data_ptr(), tokens.data_ptr(), n, case["vocab"], dim, bag=bag, scale=case["scale"],
                  dtype=case["dtype"], token_stride=strides[0], bag_stride=strides[1],
                  stream=torch.cuda.current_stream().cuda_stream)
    return out


def _own_grad(state):
    import arboretum_amd as arb
    case, grad_out, tokens = state["case"], state["grad_out"], state["tokens"]
    n, bag, vocab, dim = case["n"], case["bag"], case["vocab"], case["dim"]
    stream = torch.cuda.current_stream().cuda_stream
    if "work" not in state:  # kept from step to step
        size = max(arb.embedding_sort_bytes(n, vocab, bag=bag), arb.embedding_grad_bytes(n, dim, bag=bag))
        state["work"] = torch.empty(size, device="cuda", dtype=torch.uint8)
        state["order"] = torch.empty(2, n * bag, device="cuda", dtype=torch.int32)
    work, order = state["work"], state["order"]
    keys, rows = order.data_ptr(), order.data_ptr() + 4 * n * bag
    strides = (1, n) if case["order"] == "columns" else (bag, 1)
    arb.embedding_sort(keys, rows, tokens.data_ptr(), n, vocab, work.data_ptr(), work.numel(), bag=bag,
                       token_stride=strides[0], bag_stride=strides[1], stream=stream)
    grad = torch.empty(vocab, dim, device="cuda", dtype=getattr(torch, case["grad_dtype"]))
    arb.embedding_grad(grad.data_ptr(), grad_out.data_ptr(), keys, rows, n, vocab, dim, work.data_ptr(), work.numel(),
                       bag=bag, scale=case["scale"], dtype=case["dtype"], grad_dtype=case["grad_dtype"], stream=stream)
    return grad


def _own_adamw(state):
    import arboretum_amd as arb
    case, at = state["case"], state["at"]
    state["step"] += 1
    arb.adamw(at["p"], at["g"], at["m"], at["v"], state["sizes"], state["step"], state["lr"], beta1=BETA1, beta2=BETA2,
              eps=EPS, weight_decay=case["decay"], grad_scale=case["grad_scale"], dtype=case["dtype"],
              grad_dtype=case["grad_dtype"], stream=torch.cuda.current_stream().cuda_stream)
    return {"p": state["p"], "m": state["m"], "v": state["v"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"lookup": _own_lookup, "grad": _own_grad, "adamw": _own_adamw}[kind](state)
    return {"lookup": _plain_lookup, "grad": _plain_grad, "adamw": _plain_adamw}[kind](state)


# ---- what a pass cannot do without, and its result in 64 bits

def _bytes_of(dtype):
    return 4 if dtype == "float32" else 2


def work(case):
    if case["kind"] == "adamw":
        total = int(_sizes(case)[0].sum())
        return {"bytes": total * (2 * _bytes_of(case["dtype"]) + _bytes_of(case["grad_dtype"]) + 16), "flops": 15 * total}
    m, vocab, dim, item = case["n"] * case["bag"], case["vocab"], case["dim"], _bytes_of(case["dtype"])
    found = m * (1.0 - case["padding"])
    if case["kind"] == "grad":
        moved = 4 * m + case["n"] * dim * item + vocab * dim * _bytes_of(case["grad_dtype"])
    else:
        if case["leaves"]:
            distinct = min(m, vocab)
        else:  # rows of the table that some token names, on average
            share = np.diff(np.log1p(np.arange(vocab + 1))) / math.log1p(vocab)
            distinct = float(np.sum(-np.expm1(found * np.log1p(-share))))
        moved = 4 * m + case["n"] * dim * item + distinct * dim * item
    return {"bytes": moved, "flops": found * dim + case["n"] * dim}


def _exact_lookup(case, state):
    table = state["table"].double()
    tokens = state["tokens"] if case["order"] == "columns" else state["tokens"].t()
    out = torch.zeros(case["n"], case["dim"], device="cuda", dtype=torch.float64)
    for one in tokens:
        named = torch.nonzero(one >= 0)[:, 0]
        out[named] += table[one[named].long()]
    return out * case["scale"]


def _exact_grad(case, state):
    # tokens in order, the sums of all that come before, and the difference between the ends of each run
    tokens = (state["tokens"].t() if case["order"] == "columns" else state["tokens"]).reshape(-1)
    named = torch.nonzero(tokens >= 0)[:, 0]
    ordered, at = torch.sort(tokens[named].long())
    row = torch.div(named[at], case["bag"], rounding_mode="floor")
    ends = torch.searchsorted(ordered, torch.arange(case["vocab"] + 1, device="cuda"))
    out = torch.empty(case["vocab"], case["dim"], device="cuda", dtype=torch.float64)
    for c in range(0, case["dim"], 64):
        sums = torch.cumsum(state["grad_out"][:, c:c + 64].double()[row], 0)
        sums = torch.cat([torch.zeros_like(sums[:1]), sums])
        out[:, c:c + 64] = sums[ends[1:]] - sums[ends[:-1]]
    return out * case["scale"]


def _exact_adamw(case, state):
    p, g, m, v = (state[k].double() for k in "pgmv")
    t = state["step"] + 1
    g = case["grad_scale"] * g
    m = m + (1.0 - BETA1) * (g - m)
    v = v + (1.0 - BETA2) * (g * g - v)
    m_hat, v_hat = m / (1.0 - BETA1 ** t), v / (1.0 - BETA2 ** t)
    return {"p": p - state["lr"] * (case["decay"] * p + m_hat / (torch.sqrt(v_hat) + EPS)), "m": m, "v": v}


def exact(case, seed):
    state = prepare(case, seed)
    return {"lookup": _exact_lookup, "grad": _exact_grad, "adamw": _exact_adamw}[case["kind"]](case, state)
