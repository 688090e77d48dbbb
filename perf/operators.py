"""Measured cases of the typed projections, the adapted projection and the 8-bit embedding table.

Rows are nodes or edges of a typed graph (or requests against it), ``types`` the id of each row's
type, -1 where the type is unknown:

    typed      y[r] = x[r] W[t] + b[t], zero rows for unknown types; its gradients
    adapted    y[r] = x[r] W + b + scale (x[r] A[t]) B[t], the shared part alone for unknown types; its
               gradients
    table      rows quantised to 8 bits as they are written (one scale per row and group of columns),
               read back, and read by the edge operators
"""
import math

import torch

own = False  # False: the plain forms; True: this package's kernels

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
CODES = {"int8": (torch.int8, 127.0), "float8_e4m3": (torch.float8_e4m3fn, 448.0)}
SMALLEST_SCALE = 2.0 ** -90  # of a group of the 8-bit table


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a handful of nodes of a typed graph asked for at once, at the default width of 100
        {"name": "typed_request", "op": "typed", "train": False, "dtype": "float32", "rows": 48,
         "types": 7, "inputs": 100, "outputs": 100},
        # every node of a graph of 169 343 nodes through the projection of its type
        {"name": "typed_nodes", "op": "typed", "train": False, "dtype": "float32",
         "rows": 169_343, "types": 40, "inputs": 128, "outputs": 128},
        # a training step over a batch of typed edges: many small types, odd widths
        {"name": "typed_train_ragged", "op": "typed", "train": True, "dtype": "float32",
         "rows": 100_003, "types": 301, "inputs": 100, "outputs": 71},
        # a training step over all nodes of a graph of 2 449 029 nodes
        {"name": "typed_train_nodes", "op": "typed", "train": True, "dtype": "bfloat16",
         "rows": 2_449_029, "types": 16, "inputs": 128, "outputs": 128},
        # requests that come one row each, nearly every one with an adapter of its own
        {"name": "adapted_request", "op": "adapted", "train": False, "dtype": "bfloat16",
         "rows": 33, "types": 64, "inputs": 512, "outputs": 512, "rank": 16},
        # every node through the shared projection and its type's correction
        {"name": "adapted_nodes", "op": "adapted", "train": False, "dtype": "float32",
         "rows": 169_343, "types": 237, "inputs": 128, "outputs": 128, "rank": 8},
        # training adapters alone beside a frozen projection: many types, odd rank
        {"name": "adapted_train_frozen", "op": "adapted", "train": True, "frozen": True,
         "dtype": "float32", "rows": 30_011, "types": 500, "inputs": 100, "outputs": 100,
         "rank": 5},
        # training the shared projection and its adapters together
        {"name": "adapted_train", "op": "adapted", "train": True, "frozen": False,
         "dtype": "bfloat16", "rows": 1_000_000, "types": 64, "inputs": 128, "outputs": 128,
         "rank": 16},
        # a few updated rows written into an 8-bit table and read back
        {"name": "table_request", "op": "table", "dtype": "bfloat16", "codes": "float8_e4m3",
         "table_rows": 2_708, "rows": 17, "width": 100, "group": 32},
        # a third of the nodes written and read back
        {"name": "table_rows", "op": "table", "dtype": "float32", "codes": "int8",
         "table_rows": 1_000_000, "rows": 333_333, "width": 128, "group": 64},
        # element-wise edge features out of the 8-bit table
        {"name": "edges_hadamard", "op": "edges", "method": "Hadamard", "codes": "float8_e4m3",
         "table_rows": 169_343, "rows": 1_200_000, "width": 100, "group": 64},
        # link scores of many candidate edges out of the 8-bit table
        {"name": "edges_cosine", "op": "edges", "method": "CosineSimilarity", "codes": "int8",
         "table_rows": 2_449_029, "rows": 8_000_000, "width": 128, "group": 128},
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["typed", "typed", "adapted", "adapted", "table", "edges"])
    if op == "typed":
        inputs, outputs = spread(8, 512), spread(8, 512)
        return {"op": op, "train": rng.random() < 0.5, "dtype": rng.choice(sorted(DTYPES)),
                "rows": spread(1, min(2_000_000, 300_000_000 // (inputs + outputs))),
                "types": spread(1, 400), "inputs": inputs, "outputs": outputs}
    if op == "adapted":
        inputs, outputs = spread(16, 512), spread(16, 512)
        train = rng.random() < 0.5
        case = {"op": op, "train": train, "dtype": rng.choice(sorted(DTYPES)),
                "rows": spread(1, min(800_000, 150_000_000 // (inputs + outputs))),
                "types": spread(1, 400), "inputs": inputs, "outputs": outputs,
                "rank": spread(1, 64)}
        if train:
            case["frozen"] = rng.random() < 0.5
        return case
    width = spread(8, 512)
    case = {"op": op, "codes": rng.choice(sorted(CODES)),
            "table_rows": spread(1_000, min(2_500_000, 300_000_000 // width)),
            "width": width, "group": rng.choice([16, 32, 64, 128])}
    if op == "table":
        case["dtype"] = rng.choice(sorted(DTYPES))
        case["rows"] = spread(1, case["table_rows"])
    else:
        case["method"] = rng.choice(["Hadamard", "AbsoluteL1", "Concatenate", "L2Distance",
                                     "CosineSimilarity"])
        case["rows"] = spread(1, min(5_000_000, 400_000_000 // width))
    return case


def work(case):
    rows = case["rows"]
    if case["op"] in ("typed", "adapted"):
        size = 2 if case["dtype"] == "bfloat16" else 4
        k, n, r = case["inputs"], case["outputs"], case.get("rank", 0)
        used = min(case["types"], rows)
        if case["op"] == "typed":
            weights, flops = used * (k * n + n), 2 * rows * k * n
        else:
            weights, flops = k * n + n + used * r * (k + n), 2 * rows * (k * n + r * (k + n))
        nbytes = rows * (k + n) * size + weights * size + rows * 4
        if case["train"]:
            nbytes += rows * (k + n) * size  # the gradients that come in and go out
            if case.get("frozen"):
                # no product for the shared weight's gradient
                nbytes += used * r * (k + n) * size
                flops = flops * 3 - 2 * rows * k * n
            else:
                nbytes += weights * size
                flops *= 3
        return {"bytes": nbytes, "flops": flops}
    d = case["width"]
    row = d + 4 * -(-d // case["group"])  # codes and scales of one row
    if case["op"] == "table":
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": rows * (2 * d * size + 2 * row + 8), "flops": 4 * rows * d}
    width = {"Concatenate": 2 * d, "CosineSimilarity": 1, "L2Distance": 1}.get(case["method"], d)
    reads = min(2 * rows, case["table_rows"])  # a row that several edges share is read once
    return {"bytes": reads * row + rows * (8 + 4 * width),
            "flops": rows * d * (10 if width == 1 else 3)}


# ------------------------------------------------------------------------------------ inputs
def _types(case, gen):
    """Type ids of the rows: a few common types and a long tail, 1 in 64 rows unknown."""
    count = case["types"]
    share = 1.0 / torch.arange(1, count + 1, device="cuda", dtype=torch.float64)
    edges = torch.cumsum(share / share.sum(), 0)
    u = torch.rand(case["rows"], device="cuda", dtype=torch.float64, generator=gen)
    ids = torch.searchsorted(edges, u).clamp_(max=count - 1)
    # the common types' ids lie anywhere among the ids
    ids = torch.randperm(count, device="cuda", generator=gen)[ids]
    ids[torch.rand(case["rows"], device="cuda", generator=gen) < 1 / 64] = -1
    return ids.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(scale).to(dtype)

    state = {"case": case}
    rows = case["rows"]
    if case["op"] in ("typed", "adapted"):
        dtype, k, n = DTYPES[case["dtype"]], case["inputs"], case["outputs"]
        state["types"] = _types(case, gen)
        state["x"] = normal(rows, k, scale=0.3, dtype=dtype)
        if case["op"] == "typed":
            state["weight"] = normal(case["types"], k, n, scale=k ** -0.5, dtype=dtype)
            state["bias"] = normal(case["types"], n, scale=0.1, dtype=dtype)
        else:
            r = case["rank"]
            state["weight"] = normal(k, n, scale=k ** -0.5, dtype=dtype)
            state["bias"] = normal(n, scale=0.1, dtype=dtype)
            state["down"] = normal(case["types"], k, r, scale=k ** -0.5, dtype=dtype)
            state["up"] = normal(case["types"], r, n, scale=r ** -0.5, dtype=dtype)
            state["scale"] = 2.0 / r
        if case["train"]:
            state["dy"] = normal(rows, n, scale=0.01, dtype=dtype)
        return state
    d, table_rows = case["width"], case["table_rows"]
    code_type, largest = CODES[case["codes"]]
    # a stored table as it is kept: codes in rows padded to 16 bytes, one scale per group
    values = normal(table_rows, d, scale=0.25)
    padded = torch.zeros(table_rows, (d + 15) // 16 * 16, device="cuda")
    padded[:, :d] = values.clamp_(-1, 1).mul_(largest)
    padded = padded.round_() if case["codes"] == "int8" else padded
    state["codes"] = padded.to(code_type)
    state["scales"] = torch.rand(table_rows, -(-d // case["group"]), device="cuda",
                                 generator=gen).add_(0.5).div_(largest)
    if case["op"] == "table":
        state["values"] = normal(rows, d, scale=0.3, dtype=DTYPES[case["dtype"]])
        state["at"] = torch.randperm(table_rows, device="cuda", generator=gen)[:rows]
    else:
        for name in ("sources", "destinations"):
            state[name] = torch.randint(0, table_rows, (rows,), device="cuda", generator=gen,
                                        dtype=torch.int32)
    return state


# ---------------------------------------------------------------------------- this package's
def _run_own(s):
    import embiggen_amd as E

    case = s["case"]
    if case["op"] in ("typed", "adapted"):
        train = case["train"]
        names = ["x", "weight", "bias"] if case["op"] == "typed" else [
            "x", "weight", "bias", "down", "up"]
        wanted = ["x", "down", "up"] if case.get("frozen") else names
        t = {name: s[name].detach().requires_grad_(train and name in wanted) for name in names}
        if case["op"] == "typed":
            y = E.typed_projection(t["x"], t["weight"], s["types"], bias=t["bias"])
        else:
            y = E.adapted_projection(t["x"], t["weight"], t["down"], t["up"], s["types"],
                                     bias=t["bias"], scale=s["scale"])
        if not train:
            return {"y": y}
        grads = torch.autograd.grad(y, [t[name] for name in wanted], s["dy"])
        return {"y": y.detach(), **{"d_" + name: g for name, g in zip(wanted, grads)}}
    table = E.QuantizedTable(s["codes"], s["scales"], embedding_size=case["width"],
                             group_size=case["group"])
    if case["op"] == "table":
        table.write(s["values"], s["at"])
        return table.read(s["at"], dtype=s["values"].dtype)
    return E.edge_embedding(table, s["sources"], s["destinations"], case["method"])


# -------------------------------------------------------------------------------- plain forms
def _sorted_by_type(s, count):
    order = torch.argsort(s["types"], stable=True)
    counts = torch.bincount(s["types"] + 1, minlength=count + 1).tolist()
    return order, counts  # the unknown rows come first


def _plain_typed(s):
    case = s["case"]
    order, counts = _sorted_by_type(s, case["types"])
    x, w, b = s["x"].float()[order], s["weight"].float(), s["bias"].float()
    y = torch.zeros(case["rows"], case["outputs"], device="cuda")
    xs, ys = x.split(counts), y.split(counts)
    if not case["train"]:
        for t in range(case["types"]):
            torch.addmm(b[t], xs[t + 1], w[t], out=ys[t + 1])
        return {"y": torch.empty_like(y).index_copy_(0, order, y).to(s["x"].dtype)}
    dy = s["dy"].float()[order]
    dx, dw, db = torch.zeros_like(x), torch.empty_like(w), torch.empty_like(b)
    dxs, dys = dx.split(counts), dy.split(counts)
    for t in range(case["types"]):
        torch.addmm(b[t], xs[t + 1], w[t], out=ys[t + 1])
        torch.mm(dys[t + 1], w[t].t(), out=dxs[t + 1])
        torch.mm(xs[t + 1].t(), dys[t + 1], out=dw[t])
        torch.sum(dys[t + 1], 0, out=db[t])
    out = {"y": torch.empty_like(y).index_copy_(0, order, y),
           "d_x": torch.empty_like(dx).index_copy_(0, order, dx), "d_weight": dw, "d_bias": db}
    return {name: v.to(s["x"].dtype) for name, v in out.items()}


def _plain_adapted(s):
    case = s["case"]
    order, counts = _sorted_by_type(s, case["types"])
    x, w, b = s["x"].float()[order], s["weight"].float(), s["bias"].float()
    down, up, scale = s["down"].float(), s["up"].float(), s["scale"]
    y = torch.addmm(b, x, w)
    xs, ys = x.split(counts), y.split(counts)
    if not case["train"]:
        for t in range(case["types"]):
            ys[t + 1].addmm_(xs[t + 1] @ down[t], up[t], alpha=scale)
        return {"y": torch.empty_like(y).index_copy_(0, order, y).to(s["x"].dtype)}
    dy = s["dy"].float()[order]
    dx, d_down, d_up = dy @ w.t(), torch.empty_like(down), torch.empty_like(up)
    dxs, dys = dx.split(counts), dy.split(counts)
    for t in range(case["types"]):
        low, back = xs[t + 1] @ down[t], (dys[t + 1] @ up[t].t()) * scale
        ys[t + 1].addmm_(low, up[t], alpha=scale)
        dxs[t + 1].addmm_(back, down[t].t())
        torch.mm(xs[t + 1].t(), back, out=d_down[t])
        torch.mm((low * scale).t(), dys[t + 1], out=d_up[t])
    out = {"y": torch.empty_like(y).index_copy_(0, order, y),
           "d_x": torch.empty_like(dx).index_copy_(0, order, dx), "d_down": d_down, "d_up": d_up}
    if not case["frozen"]:
        out.update(d_weight=x.t() @ dy, d_bias=dy.sum(0))
    return {name: v.to(s["x"].dtype) for name, v in out.items()}


def _values(codes, scales, case):
    """The float32 values of gathered rows of the table."""
    d, group = case["width"], case["group"]
    return codes[:, :d].float() * scales.repeat_interleave(group, 1)[:, :d]


def _plain_table(s):
    case = s["case"]
    d, group, rows = case["width"], case["group"], case["rows"]
    code_type, largest = CODES[case["codes"]]
    groups = -(-d // group)
    v = torch.zeros(rows, groups * group, device="cuda")
    v[:, :d] = s["values"].float()
    v = v.view(rows, groups, group)
    scales = (v.abs().amax(2) / largest).clamp_(min=SMALLEST_SCALE)
    quotient = v.double() / scales.double().unsqueeze(2)  # rounded once: borders lie between codes
    quotient = quotient.view(rows, -1)[:, :d]
    if case["codes"] == "int8":
        codes = quotient.round().to(code_type)
    else:
        # the nearest of the format's values, ties to the even one
        step = torch.exp2(torch.floor(torch.log2(quotient.abs().clamp_(min=2.0 ** -6))) - 3)
        codes = ((quotient / step).round() * step).float().to(code_type)
    s["codes"].view(torch.uint8)[s["at"], :d] = codes.view(torch.uint8)
    s["scales"][s["at"]] = scales
    codes = s["codes"].view(torch.uint8)[s["at"]].view(code_type)
    return _values(codes, s["scales"][s["at"]], case).to(s["values"].dtype)


def _plain_edges(s):
    case = s["case"]
    rows = []
    for name in ("sources", "destinations"):
        codes = s["codes"].view(torch.uint8)[s[name].long()].view(s["codes"].dtype)
        rows.append(_values(codes, s["scales"][s[name].long()], case))
    a, b = rows
    method = case["method"]
    if method == "Hadamard":
        return a * b
    if method == "AbsoluteL1":
        return (a - b).abs()
    if method == "Concatenate":
        return torch.cat([a, b], 1)
    if method == "L2Distance":
        return (a - b).square().sum(1, keepdim=True).sqrt()
    norm = (a.square().sum(1).sqrt() * b.square().sum(1).sqrt()).clamp(min=1e-6)
    return ((a * b).sum(1) / norm).unsqueeze(1)


def run(state):
    if own:
        return _run_own(state)
    return {"typed": _plain_typed, "adapted": _plain_adapted, "table": _plain_table,
            "edges": _plain_edges}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------- exact
def _exact_projection(s):
    """Row by row definitions in 64 bits, the rows of one type at a time."""
    case = s["case"]
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    typed, train = case["op"] == "typed", case["train"]
    rows, ids = case["rows"], s["types"].long()
    dy = s["dy"].double() if train else None
    if typed:
        out = {"y": x.new_zeros(rows, case["outputs"])}
        if train:
            out.update(d_x=torch.zeros_like(x), d_weight=torch.zeros_like(w),
                       d_bias=torch.zeros_like(b))
    else:
        down, up, scale = s["down"].double(), s["up"].double(), s["scale"]
        out = {"y": x @ w + b}
        if train:
            out.update(d_x=dy @ w.T, d_down=torch.zeros_like(down), d_up=torch.zeros_like(up))
            if not case["frozen"]:
                out.update(d_weight=x.T @ dy, d_bias=dy.sum(0))
    for t in torch.unique(ids[ids >= 0]).tolist():
        at = (ids == t).nonzero().squeeze(1)
        xt, dyt = x[at], dy[at] if train else None
        if typed:
            out["y"][at] = xt @ w[t] + b[t]
            if train:
                out["d_x"][at] = dyt @ w[t].T
                out["d_weight"][t] = xt.T @ dyt
                out["d_bias"][t] = dyt.sum(0)
        else:
            both = down[t] @ up[t] * scale
            out["y"][at] += xt @ both
            if train:
                out["d_x"][at] += dyt @ both.T
                d_both = xt.T @ dyt * scale
                out["d_down"][t] = d_both @ up[t].T
                out["d_up"][t] = down[t].T @ d_both
    return out


def _exact_rows(codes, scales, case):
    d, group = case["width"], case["group"]
    group_of = torch.arange(d, device=codes.device) // group
    return codes[:, :d].to(torch.float32).double() * scales.double()[:, group_of]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("typed", "adapted"):
        return _exact_projection(s)
    d, group = case["width"], case["group"]
    largest = CODES[case["codes"]][1]
    if case["op"] == "table":
        v, parts = s["values"].double(), []
        for first in range(0, d, group):
            part = v[:, first:first + group]
            # a stored scale is a float32 number
            scale = (part.abs().amax(1, keepdim=True) / largest).float().double()
            scale = scale.clamp(min=SMALLEST_SCALE)
            if case["codes"] == "int8":
                code = torch.round(part / scale)
            else:
                mantissa, exponent = torch.frexp(part / scale)  # mantissa in [0.5, 1)
                bits = torch.full_like(part, 4.0) - (-5.0 - exponent).clamp(min=0)
                code = torch.ldexp(torch.round(torch.ldexp(mantissa, bits)), exponent - bits)
            parts.append(code * scale)
        return torch.cat(parts, 1)
    out = []
    for first in range(0, case["rows"], 1 << 20):  # in slices: 64 bits take room
        a, b = (_exact_rows(s["codes"].view(torch.uint8)[at].view(s["codes"].dtype),
                            s["scales"][at], case)
                for at in (s[name][first:first + (1 << 20)].long()
                           for name in ("sources", "destinations")))
        if case["method"] == "Hadamard":
            out.append(a * b)
        elif case["method"] == "AbsoluteL1":
            out.append(abs(a - b))
        elif case["method"] == "Concatenate":
            out.append(torch.hstack([a, b]))
        elif case["method"] == "L2Distance":
            out.append(torch.linalg.vector_norm(a - b, dim=1)[:, None])
        else:
            norms = torch.linalg.vector_norm(a, dim=1) * torch.linalg.vector_norm(b, dim=1)
            out.append(((a * b).sum(1) / norms.clamp(min=1e-6))[:, None])
    return torch.cat(out)
