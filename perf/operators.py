"""Layer norm, dropout and the two joined with a residual sum: cases to time and to compare.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end)
or, with ``own`` set, through the calls a user of graphsage_amd makes.  ``exact`` is the definition in 64 bits.

A case names the operator (``layer_norm``, ``dropout``, ``dropout_add_layer_norm``), what is done with it
(``train``: forward and gradients; otherwise the forward alone), the table (``rows`` x ``cols``, ``dtype``) and,
where they mean something, the drop rate ``p``, whether there is a ``residual``, whether the sum is returned too
(``return_sum``) and whether the weights are kept in fp32 beside 16-bit activations (``fp32_weights``).
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, train, rows, cols, dtype, p=0.0, residual=False, return_sum=False, fp32_weights=False):
    return {"name": name, "op": op, "train": train, "rows": rows, "cols": cols, "dtype": dtype, "p": p,
            "residual": residual, "return_sum": return_sum, "fp32_weights": fp32_weights}


def listed():
    return [
        # one node's hidden row normalised while serving it: nothing but latency
        _case("ln_one_row", "layer_norm", False, 1, 256, "fp32"),
        # the hidden rows of a batch of pairs with their negatives (7 x 1024) in a wide 16-bit encoder
        _case("ln_batch_rows", "layer_norm", False, 7168, 1024, "bf16", fp32_weights=True),
        # a hidden layer of the 64-wide encoder over ten million nodes, forward and backward
        _case("ln_train_10m_nodes", "layer_norm", True, 10_000_000, 64, "fp32"),
        # the same step on odd sizes: rows that start at every alignment
        _case("ln_train_odd", "layer_norm", True, 99_991, 257, "fp16"),
        # long rows in 16 bits, weights in 32
        _case("ln_train_wide", "layer_norm", True, 16_384, 4096, "bf16", fp32_weights=True),
        # the activations of one small batch
        _case("dropout_batch", "dropout", False, 1024, 64, "fp32", p=0.3),
        # a hidden layer of the 128-wide encoder over a million nodes
        _case("dropout_train_1m_nodes", "dropout", True, 1_000_000, 128, "fp32", p=0.3),
        # a large 16-bit table whose rows are odd
        _case("dropout_train_odd", "dropout", True, 1_000_003, 129, "bf16", p=0.1),
        # hidden layer with its residual, 128 wide, a million nodes
        _case("joined_train_1m_nodes", "dropout_add_layer_norm", True, 1_000_000, 128, "fp32", p=0.3, residual=True),
        # the first hidden layer of the 256-wide encoder: its input has another width, so no residual
        _case("joined_train_first_layer", "dropout_add_layer_norm", True, 1_000_000, 256, "fp32", p=0.3),
        # long 16-bit rows, the sum carried on to the next layer
        _case("joined_train_wide_sum", "dropout_add_layer_norm", True, 8191, 5120, "bf16", p=0.1, residual=True,
              return_sum=True),
        # serving a few rows: no dropout, the sum carried on
        _case("joined_few_rows", "dropout_add_layer_norm", False, 33, 1000, "fp16", residual=True, return_sum=True),
    ]


def draw(rng):
    op = rng.choice(["layer_norm", "dropout", "dropout_add_layer_norm"])
    train = rng.random() < 0.6
    # a norm over a handful of columns cancels to nothing; dropout does not care
    least = 1.0 if op == "dropout" else 8.0
    cols = int(round(math.exp(rng.uniform(math.log(least), math.log(16384.0)))))
    most = min(4_000_000, (1 << 27) // cols)                     # up to 134 M elements
    rows = int(round(math.exp(rng.uniform(0.0, math.log(most)))))
    if op == "layer_norm":
        p, residual = 0.0, False
    elif op == "dropout":
        p, residual = rng.choice([0.1, 0.3, 0.5, round(rng.uniform(0.01, 0.95), 3)]), False
    else:
        p = rng.choice([0.0, 0.1, 0.3, round(rng.uniform(0.01, 0.9), 3)])
        residual = rng.random() < 0.8
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    return {"op": op, "train": train, "rows": rows, "cols": cols, "dtype": dtype, "p": p, "residual": residual,
            "return_sum": op == "dropout_add_layer_norm" and rng.random() < 0.4,
            "fp32_weights": dtype != "fp32" and op != "dropout" and rng.random() < 0.5}


def work(case):
    n, size = case["rows"] * case["cols"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "dropout":
        return {"bytes": (4 if case["train"] else 2) * n * size, "flops": (2 if case["train"] else 1) * n}
    # tables in and out: x, y; with gradients g and dx; with a residual itself and its gradient; the returned sum
    # and its gradient.  Parameters: weight and bias, and their gradients.
    tables = 2 + int(case["residual"]) + int(case["return_sum"])
    flops = 8 + 2 * int(case["residual"])
    params = 2 * case["cols"]
    if case["train"]:
        tables, params, flops = 2 * tables, 2 * params, flops + 14
    wsize = 4 if case["fp32_weights"] else size
    return {"bytes": tables * n * size + params * wsize, "flops": flops * n}


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    shape, dtype, train = (case["rows"], case["cols"]), DTYPES[case["dtype"]], case["train"]

    def normal(*size):
        return torch.randn(*size, generator=gen, device=dev)

    state = {"case": case, "seed": int(torch.randint(0, 1 << 62, (1,), generator=gen, device=dev).item())}
    # activations: columns of unlike scale around unlike means; behind a ReLU where dropout follows one
    scale = 0.5 + torch.rand(shape[1], generator=gen, device=dev)
    x = normal(*shape).mul_(scale).add_(0.5 * normal(shape[1]))
    if case["op"] != "layer_norm":
        x = x.relu_()
    leaves = [x.to(dtype)]
    if case["residual"]:
        leaves.append(normal(*shape).to(dtype))
    if case["op"] != "dropout":
        wdtype = torch.float32 if case["fp32_weights"] else dtype
        leaves.append((1.0 + 0.1 * normal(shape[1])).to(wdtype))
        leaves.append((0.1 * normal(shape[1])).to(wdtype))
    if train:
        for leaf in leaves:
            leaf.requires_grad_(True)
        state["grads"] = [normal(*shape).to(dtype) for _ in range(2 if case["return_sum"] else 1)]
    state["leaves"] = leaves
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------- the framework's calls
def _run_own(state):
    import graphsage_amd as gs
    case, leaves = state["case"], state["leaves"]
    x = leaves[0]
    if case["op"] == "layer_norm":
        outs = [gs.layer_norm(x, leaves[1], leaves[2], eps=EPS)]
    elif case["op"] == "dropout":
        outs = [gs.dropout(x, p=case["p"], seed=state["seed"])]
    else:
        out = gs.dropout_add_layer_norm(x, leaves[1] if case["residual"] else None, leaves[-2], leaves[-1],
                                        p=case["p"], eps=EPS, seed=state["seed"], return_sum=case["return_sum"])
        outs = list(out) if case["return_sum"] else [out]
    if not case["train"]:
        return outs
    return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, state["grads"]))


# ---------------------------------------------------------------------------------------------- the plain form
_LOW = 0xFFFFFFFF


def _keep(n, seed, p, device):
    """1 where element i of n is kept: a 32-bit counter hash of (seed, i), its upper 24 bits against p."""
    i = torch.arange(n, dtype=torch.int64, device=device)
    h = ((i & _LOW) * 0x9E3779B1) & _LOW
    h ^= seed & _LOW
    h ^= ((i >> 32) * 0x85EBCA77 + (seed >> 32)) & _LOW
    h ^= h >> 16
    h = (h * 0x85EBCA6B) & _LOW
    h ^= h >> 13
    h = (h * 0xC2B2AE35) & _LOW
    h ^= h >> 16
    border = torch.tensor(p, dtype=torch.float32).item()
    return (h >> 8) >= math.ceil(border * (1 << 24))


@torch.no_grad()
def _run_plain(state):
    case, leaves = state["case"], state["leaves"]
    dtype = DTYPES[case["dtype"]]
    x = leaves[0].float()
    keep = None
    if case["p"] > 0.0:
        keep = _keep(x.numel(), state["seed"], case["p"], x.device).view(x.shape)

    def drop(t):
        return t if keep is None else torch.where(keep, t / (1.0 - case["p"]), torch.zeros((), device=t.device))

    if case["op"] == "dropout":
        outs = [drop(x).to(dtype)]
        if case["train"]:
            outs.append(drop(state["grads"][0].float()).to(dtype))
        return outs
    z = drop(x)
    if case["residual"]:
        z = z + leaves[1].float()
    weight, bias = leaves[-2].float(), leaves[-1].float()
    centred = z - z.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    hat = centred * rstd
    outs = [(hat * weight + bias).to(dtype)]
    if case["return_sum"]:
        outs.append(z.to(dtype))
    if not case["train"]:
        return outs
    g = state["grads"][0].float()
    a = g * weight
    dz = rstd * (a - a.mean(1, keepdim=True) - hat * (a * hat).mean(1, keepdim=True))
    if case["return_sum"]:
        dz = dz + state["grads"][1].float()
    outs.append(drop(dz).to(dtype))
    if case["residual"]:
        outs.append(dz.to(dtype))
    outs.append((g * hat).sum(0, dtype=torch.float64).to(leaves[-2].dtype))
    outs.append(g.sum(0, dtype=torch.float64).to(leaves[-1].dtype))
    return outs


# ----------------------------------------------------------------------------------- the definition in 64 bits
def _mix(h, shift, factor):
    return ((h ^ (h >> shift)) * factor) % (1 << 32)


def _kept(first, count, seed, p, device):
    index = torch.arange(first, first + count, dtype=torch.int64, device=device)
    high, low = index // (1 << 32), index % (1 << 32)
    key = (high * 0x85EBCA77 + seed // (1 << 32)) % (1 << 32)
    word = (low * 0x9E3779B1) % (1 << 32)
    word = word ^ key ^ (seed % (1 << 32))
    word = _mix(_mix(word, 16, 0x85EBCA6B), 13, 0xC2B2AE35)
    word = word ^ (word >> 16)
    # the drop rate is a 32-bit number; so is the draw, of which 24 bits count
    rate = torch.tensor(p, dtype=torch.float32, device=device).double()
    return (word // 256).double() / (1 << 24) >= rate


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    leaves = [t.detach() for t in state["leaves"]]
    rows, cols = case["rows"], case["cols"]
    grads = state.get("grads", [])
    x, dev = leaves[0], leaves[0].device
    train, normed = case["train"], case["op"] != "dropout"

    def table():
        return torch.empty(rows, cols, dtype=torch.float64, device=dev)

    y, total = table(), table() if case["return_sum"] else None
    dx, dres = (table() if train else None), (table() if train and case["residual"] else None)
    dw = torch.zeros(cols, dtype=torch.float64, device=dev)
    db = torch.zeros(cols, dtype=torch.float64, device=dev)
    step = max(1, (1 << 25) // cols)
    for r0 in range(0, rows, step):
        part = slice(r0, min(rows, r0 + step))
        z = x[part].double()
        factor = torch.ones_like(z)
        if case["p"] > 0.0:
            kept = _kept(r0 * cols, z.numel(), state["seed"], case["p"], dev).view_as(z)
            factor = kept.double() / (1.0 - case["p"])
        z = z * factor
        if not normed:
            y[part] = z
            if train:
                dx[part] = grads[0][part].double() * factor
            continue
        if case["residual"]:
            z += leaves[1][part].double()
        if total is not None:
            total[part] = z
        mean = z.sum(1, keepdim=True) / cols
        var = ((z - mean) ** 2).sum(1, keepdim=True) / cols
        sigma = (var + EPS).sqrt()
        hat = (z - mean) / sigma
        y[part] = leaves[-1].double() + leaves[-2].double() * hat
        if not train:
            continue
        g = grads[0][part].double()
        dw += (g * hat).sum(0)
        db += g.sum(0)
        a = g * leaves[-2].double()
        dz = (a - (a.sum(1, keepdim=True) + hat * (a * hat).sum(1, keepdim=True)) / cols) / sigma
        if total is not None:
            dz += grads[1][part].double()
        dx[part] = dz * factor
        if dres is not None:
            dres[part] = dz
    outs = [y] + ([total] if total is not None else [])
    if train:
        outs += [dx] + ([dres] if dres is not None else []) + ([dw, db] if normed else [])
    return outs
