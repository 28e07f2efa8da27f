"""Cases, plain forms and 64-bit values of the scaled 8-bit and the expert-grouped matrix products.

Five operators in four kinds of case, picked by case["op"]:

  linear_i8    x [M,K] (fp16 / bf16) is rounded to 8-bit integers with one scale per token and multiplied with 8-bit
               weights [N,K] that carry one scale per output channel: quantize_rows, then gemm_i8
  gemm_i8      the product alone, on integers that are there already
  grouped      c[t] = a[t] b[e]^T for the rows t of expert e, rows sorted by expert, ragged sizes: grouped_gemm
  grouped_i8   the same on 8-bit integers with a scale per token and per (expert, channel): grouped_gemm_i8
  backward     both gradients of `grouped`: da[t] = dc[t] b[e] and db[e] = sum over the rows of e of dc[t]^T a[t]
               (grouped_gemm_dgrad, grouped_gemm_wgrad)
"""
import torch

own = False   # True: run() calls the framework's operators; False: elementary torch operations in 32 bits

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One generated token through one projection of a model whose weights are held in 8 bits: latency.
        {"name": "linear_i8 one token", "op": "linear_i8", "rows": 1, "n": 4096, "k": 4096, "x": "fp16", "out": "fp16"},
        # A serving batch of a few dozen tokens, a wide projection: the weights stream from memory once.
        {"name": "linear_i8 decode batch", "op": "linear_i8", "rows": 48, "n": 14336, "k": 4096, "x": "bf16", "out": "bf16"},
        # Odd sizes and an fp32 result: a short prompt into a head that is no multiple of anything.
        {"name": "gemm_i8 odd sizes", "op": "gemm_i8", "rows": 777, "n": 1001, "k": 2064, "x": "fp16", "out": "fp32"},
        # Prompt processing at the framework's headline GEMM size.
        {"name": "linear_i8 prompt", "op": "linear_i8", "rows": 8192, "n": 8192, "k": 8192, "x": "fp16", "out": "fp16"},
        # A few generated tokens, each sent to some of many experts: most experts get a row or none.
        {"name": "grouped decode", "op": "grouped", "rows": 64, "n": 2048, "k": 2048, "experts": 64, "idle": 14, "skew": 0.5, "tail": 0, "x": "bf16"},
        # A short prompt: ragged groups, empty experts, an odd output width, rows behind the last group.
        {"name": "grouped ragged", "op": "grouped", "rows": 1333, "n": 1001, "k": 776, "experts": 9, "idle": 2, "skew": 0.4, "tail": 11, "x": "fp16"},
        # Prompt processing: a few hundred rows per expert and more.
        {"name": "grouped prompt", "op": "grouped", "rows": 16384, "n": 4096, "k": 2048, "experts": 32, "idle": 0, "skew": 0.2, "tail": 0, "x": "bf16"},
        # The first two again with experts held in 8 bits.
        {"name": "grouped_i8 decode", "op": "grouped_i8", "rows": 96, "n": 2048, "k": 4096, "experts": 32, "idle": 3, "skew": 0.5, "tail": 0, "x": "fp16", "out": "fp16"},
        {"name": "grouped_i8 prompt", "op": "grouped_i8", "rows": 8192, "n": 4096, "k": 4096, "experts": 16, "idle": 1, "skew": 0.2, "tail": 0, "x": "bf16", "out": "bf16"},
        # Training on a small batch: ragged groups with one expert that got no row, whose gradient is zero.
        {"name": "backward ragged", "op": "backward", "rows": 1333, "n": 1000, "k": 776, "experts": 9, "idle": 1, "skew": 0.4, "tail": 11, "x": "fp16"},
        # A training step's batch.
        {"name": "backward batch", "op": "backward", "rows": 16384, "n": 4096, "k": 2048, "experts": 16, "idle": 0, "skew": 0.2, "tail": 0, "x": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["linear_i8", "gemm_i8", "grouped", "grouped_i8", "backward"])
    x = rng.choice(["fp16", "bf16"])
    if op in ("linear_i8", "gemm_i8"):
        rows, n, k = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 4, 512) * 16
        return {"op": op, "rows": rows, "n": n, "k": k, "x": x, "out": rng.choice(["fp16", "bf16", "fp32"])}
    experts = _log(rng, 1, 128)
    rows, n, k = _log(rng, 1, 16384), _log(rng, 8, 512) * 8, _log(rng, 4, 256) * 16
    while experts * n * k > 1 << 28:
        experts = (experts + 1) // 2
    while rows * n * k > 1 << 36:
        rows = (rows + 1) // 2
    if op != "backward" and rng.random() < 0.3:
        n += rng.randrange(1, 8)   # output rows that are no multiple of 16 bytes
    case = {"op": op, "rows": rows, "n": n, "k": k, "experts": experts, "idle": rng.randrange(experts) // 3,
            "skew": rng.choice([0.0, 0.2, 0.4]), "tail": rng.choice([0, 0, 5, 64]), "x": x}
    if op == "grouped_i8":
        case["out"] = rng.choice(["fp16", "bf16", "fp32"])
    return case


def _sizes(case):
    """Rows of each expert before the seed shuffles them: the first experts get more, `idle` of them none."""
    live = case["experts"] - case["idle"]
    share = [(i + 1.0) ** -case["skew"] for i in range(live)]
    total = sum(share)
    edge, acc = [0], 0.0
    for s in share:
        acc += s
        edge.append(int(round(case["rows"] * acc / total)))
    edge[-1] = case["rows"]
    return [b - a for a, b in zip(edge, edge[1:])] + [0] * case["idle"]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def scales(*shape):
        return (torch.rand(*shape, generator=g, device=DEV) + 0.5) * 0.01

    def ints(*shape):
        # in pieces: a whole expert stack in fp32 would be large
        out = torch.empty(shape, dtype=torch.int8, device=DEV)
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 27):
            part = flat[i:i + (1 << 27)]
            part.copy_((normal(part.numel()) * 40).round_().clamp_(-127, 127))
        return out

    op, rows, n, k = case["op"], case["rows"], case["n"], case["k"]
    dtype = TYPES[case["x"]]
    s = {"op": op, "rows": rows, "n": n, "k": k}
    if op in ("linear_i8", "gemm_i8"):
        s["b"], s["scale_b"] = ints(n, k), scales(n)
        s["c"] = torch.empty(rows, n, dtype=TYPES[case["out"]], device=DEV)
        if op == "linear_i8":
            x = normal(rows, k)
            x[:, torch.randint(k, (max(1, k // 128),), generator=g, device=DEV)] *= 6   # outlier channels, as activations have them
            s["x"] = x.to(dtype)
            s["q"] = torch.empty(rows, k, dtype=torch.int8, device=DEV)       # kept by a serving program, like c
            s["scale_a"] = torch.empty(rows, device=DEV)
        else:
            s["q"], s["scale_a"] = ints(rows, k), scales(rows)
        return s
    sizes = torch.tensor(_sizes(case), device=DEV)
    sizes = sizes[torch.randperm(case["experts"], generator=g, device=DEV)]
    offsets = torch.zeros(case["experts"] + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = sizes.cumsum(0)
    s["offsets"], s["most"] = offsets, max(_sizes(case))
    total = rows + case["tail"]     # rows behind the last group are left as they are
    if op == "grouped":
        s["a"] = normal(total, k).to(dtype)
        s["b"] = torch.stack([(normal(n, k) * k ** -0.5).to(dtype) for _ in range(case["experts"])])
        s["c"] = normal(total, n).to(dtype)
    elif op == "grouped_i8":
        s["q"], s["scale_a"] = ints(total, k), scales(total)
        s["b"], s["scale_b"] = ints(case["experts"], n, k), scales(case["experts"], n)
        s["c"] = normal(total, n).to(TYPES[case["out"]])
    else:
        s["a"] = normal(total, k).to(dtype)
        s["b"] = torch.stack([(normal(n, k) * k ** -0.5).to(dtype) for _ in range(case["experts"])])
        s["dc"] = normal(total, n).to(dtype)
        s["da"] = normal(total, k).to(dtype)
        s["db"] = torch.empty(case["experts"], n, k, dtype=dtype, device=DEV)
    return s


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _run_own(s):
    from tiledcuda_b200 import ops

    if s["op"] == "linear_i8":
        ops.quantize_rows(s["x"], s["q"], s["scale_a"])
        ops.gemm_i8(s["q"], s["b"], s["scale_a"], s["scale_b"], s["c"])
        return {"c": s["c"], "scale_a": s["scale_a"]}
    if s["op"] == "gemm_i8":
        ops.gemm_i8(s["q"], s["b"], s["scale_a"], s["scale_b"], s["c"])
        return {"c": s["c"]}
    if s["op"] == "grouped":
        ops.grouped_gemm(s["a"], s["b"], s["offsets"], s["c"])
        return {"c": s["c"]}
    if s["op"] == "grouped_i8":
        ops.grouped_gemm_i8(s["q"], s["b"], s["scale_a"], s["scale_b"], s["offsets"], s["c"])
        return {"c": s["c"]}
    ops.grouped_gemm_dgrad(s["dc"], s["b"], s["offsets"], s["da"])
    ops.grouped_gemm_wgrad(s["dc"], s["a"], s["offsets"], s["db"])
    return {"da": s["da"], "db": s["db"]}


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _rows_of_groups(s):
    """Row numbers [E, most] of each group, padded, and which of them are real."""
    first, last = s["offsets"][:-1].long(), s["offsets"][1:].long()
    at = first[:, None] + torch.arange(s["most"], device=DEV)
    return at.clamp(max=max(0, s["rows"] - 1)), at < last[:, None]


def _padded(t, at, real):
    return t.float()[at] * real[:, :, None]


def _run_plain(s):
    op = s["op"]
    if op in ("linear_i8", "gemm_i8"):
        out = {}
        q, scale = s["q"], s["scale_a"]
        if op == "linear_i8":
            x = s["x"].float()
            scale = (x.abs().amax(1) / 127).clamp(min=torch.finfo(torch.float32).tiny)
            q = (x.double() / scale.double()[:, None]).round()   # 64 bits: quotients next to a half have to round the right way
            out["scale_a"] = scale
        c = q.float() @ s["b"].float().t()
        out["c"] = (c * scale[:, None] * s["scale_b"][None, :]).to(s["c"].dtype)
        return out
    at, real = _rows_of_groups(s)
    if op == "backward":
        dc = _padded(s["dc"], at, real)
        s["da"][at[real]] = torch.bmm(dc, s["b"].float())[real].to(s["da"].dtype)
        db = torch.bmm(dc.transpose(1, 2), _padded(s["a"], at, real))
        return {"da": s["da"], "db": db.to(s["db"].dtype)}
    if op == "grouped":
        c = torch.bmm(_padded(s["a"], at, real), s["b"].float().transpose(1, 2))
    else:
        c = torch.bmm(_padded(s["q"], at, real), s["b"].float().transpose(1, 2))
        c = c * s["scale_a"][at][:, :, None] * s["scale_b"][:, None, :]
    s["c"][at[real]] = c[real].to(s["c"].dtype)
    return {"c": s["c"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op, rows = case["op"], case["rows"]
    if op in ("linear_i8", "gemm_i8"):
        out = {}
        if op == "linear_i8":
            x = s["x"].double()
            scale = torch.div(x.abs().max(dim=1).values.float(), 127.0)
            scale = torch.maximum(scale, torch.full_like(scale, 2.0 ** -126)).double()
            a = torch.round(x / scale.unsqueeze(1))
            out["scale_a"] = x.abs().max(dim=1).values / 127
        else:
            a, scale = s["q"].double(), s["scale_a"].double()
        out["c"] = torch.einsum("mk,nk->mn", a, s["b"].double()) * torch.outer(scale, s["scale_b"].double())
        return out
    edges = s["offsets"].tolist()
    groups = [(e, i, j) for e, (i, j) in enumerate(zip(edges, edges[1:]))]
    if op == "backward":
        da, db = s["da"].double(), torch.zeros(s["db"].shape, dtype=torch.float64, device=DEV)
        for e, i, j in groups:
            dc = s["dc"][i:j].double()
            da[i:j] = dc @ s["b"][e].double()
            db[e] = dc.t() @ s["a"][i:j].double()
        return {"da": da, "db": db}
    c = s["c"].double()
    for e, i, j in groups:
        a = (s["a"] if op == "grouped" else s["q"])[i:j].double()
        c[i:j] = a @ s["b"][e].double().t()
        if op == "grouped_i8":
            c[i:j] *= torch.outer(s["scale_a"][i:j].double(), s["scale_b"][e].double())
    return {"c": c}


def work(case):
    """One pass: inputs once (of the experts, those that have rows), outputs once."""
    op, rows, n, k = case["op"], case["rows"], case["n"], case["k"]
    flops = 2.0 * rows * n * k
    if op in ("linear_i8", "gemm_i8"):
        out = TYPES[case["out"]].itemsize
        a = (2 if op == "linear_i8" else 1) * rows * k + 4 * rows
        return {"bytes": float(a + n * k + 4 * n + out * rows * n), "flops": flops}
    live, experts = sum(x > 0 for x in _sizes(case)), case["experts"]
    if op == "grouped":
        return {"bytes": 2.0 * (rows * k + live * n * k + rows * n), "flops": flops}
    if op == "grouped_i8":
        return {"bytes": float(rows * (k + 4) + live * n * (k + 4) + TYPES[case["out"]].itemsize * rows * n), "flops": flops}
    # dc, a and the weights in, both gradients out
    return {"bytes": 2.0 * (rows * n + rows * k + live * n * k + rows * k + experts * n * k), "flops": 2 * flops}
