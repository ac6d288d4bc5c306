"""Products with 8-bit and 16-bit weights and what an expert layer needs around
them, as cases that can be timed:

quantise   rows (or 128 x 128 blocks) into e4m3 with a scale for each 128
           channels, rows taken through an index list or in order;
linear     y = x W^T, e4m3 with scales or 16-bit, plain or gated
           (silu(gate) * up);
grouped    the same with a weight matrix for each expert, the rows of x
           ordered by expert or read through an index list;
route      k experts for each token with their weights, and the order by
           expert that `grouped` takes (or that order for experts given);
combine    the experts' rows back to their tokens, weighted and added.

`own` False computes them with elementary torch operations; True calls the
library (rabbit_b200.capi). A block of 128 channels x has the scale
s = fp32(max|x| / 448) and holds e4m3(x / s), rounded to nearest even.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
      "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
BLOCK = 128


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one token's hidden row of the OLMoE-shaped model: all latency
        dict(name="quantise 1x2048 f32", op="quantise", dtype="f32", rows=1, cols=2048, of=0,
             block=1),
        # a long prompt's rows, two experts each, taken through the routing's list
        dict(name="quantise 16384x4096 bf16 listed", op="quantise", dtype="bf16", rows=16384,
             cols=4096, of=8191, block=1),
        # a decode step's projection of the Mixtral-shaped model: the weights' bytes
        dict(name="linear 1x4096x4096 e4m3", op="linear", dtype="e4m3", out="f32", rows=1,
             n_in=4096, n_out=4096, gated=False),
        # gate and up of a Mixtral-shaped dense block over a long prompt, an odd number of tokens
        dict(name="linear 8191x4096x14336 e4m3 gated", op="linear", dtype="e4m3", out="bf16",
             rows=8191, n_in=4096, n_out=14336, gated=True),
        # the OLMoE-shaped model's decode step: 8 of 64 experts, a row each
        dict(name="grouped 1 token of 64 bf16 gated", op="grouped", dtype="bf16", out="f32",
             tokens=1, k=8, experts=64, n_in=2048, n_out=1024, gated=True, listed=True, dropped=0,
             idle=0),
        # a decode batch of 64 through the Mixtral-shaped down projection, rows in order
        dict(name="grouped 64 tokens of 8 e4m3", op="grouped", dtype="e4m3", out="bf16", tokens=64,
             k=2, experts=8, n_in=14336, n_out=4096, gated=False, listed=False, dropped=3, idle=0),
        # a long chunk over the DeepSeek-shaped experts: ragged, some without a row
        dict(name="grouped 4099 tokens of 64 e4m3 gated", op="grouped", dtype="e4m3", out="bf16",
             tokens=4099, k=6, experts=64, n_in=2048, n_out=1408, gated=True, listed=True,
             dropped=0, idle=3),
        # a long prompt through the Mixtral-shaped experts in 16 bits: the most operations
        dict(name="grouped 8192 tokens of 8 f16 gated", op="grouped", dtype="f16", out="f16",
             tokens=8192, k=2, experts=8, n_in=4096, n_out=14336, gated=True, listed=True,
             dropped=0, idle=0),
        # the Mixtral-shaped router's scores of one token
        dict(name="route 1 of 8", op="route", tokens=1, k=2, experts=8, over_all=False, masked=0,
             given=False),
        # a long chunk over the DeepSeek-shaped router, a few experts off for some tokens
        dict(name="route 8191 of 64", op="route", tokens=8191, k=6, experts=64, over_all=True,
             masked=5, given=False),
        # one token's eight experts of the OLMoE-shaped model added to its row
        dict(name="combine 1x8x2048 f32", op="combine", dtype="f32", out="f32", tokens=1, k=8,
             cols=2048, dropped=0, base=True),
        # a long prompt's two experts each added to its rows
        dict(name="combine 8191x2x4096 bf16", op="combine", dtype="bf16", out="bf16", tokens=8191,
             k=2, cols=4096, dropped=100, base=True),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantise", "linear", "linear", "grouped", "grouped", "route", "combine"])
    if op == "quantise":
        rows, cols = log_int(rng, 1, 16384), log_int(rng, 100, 6144)
        block = rng.choice([1, 1, BLOCK])
        of = rng.choice([0, log_int(rng, 1, 8192)]) if block == 1 else 0
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=rows, cols=cols, of=of,
                    block=block)
    if op == "route":
        experts = log_int(rng, 4, 256)
        return dict(op=op, tokens=log_int(rng, 1, 8192), k=rng.randint(1, min(8, experts)),
                    experts=experts, over_all=rng.random() < .5,
                    masked=rng.choice([0, experts // 8, experts]), given=rng.random() < .25)
    if op == "combine":
        tokens, k = log_int(rng, 1, 8192), rng.randint(1, 8)
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]),
                    out=rng.choice(["f32", "f16", "bf16"]), tokens=tokens, k=k,
                    cols=log_int(rng, 64, 6144), dropped=rng.choice([0, tokens * k // 9]),
                    base=rng.random() < .7)
    n_in, n_out = log_int(rng, 128, 14336), log_int(rng, 128, 14336)
    both = dict(dtype=rng.choice(["e4m3", "e4m3", "f16", "bf16"]),
                out=rng.choice(["f32", "f16", "bf16", "bf16"]), n_in=n_in, n_out=n_out,
                gated=rng.random() < .5)
    if op == "linear":
        most = int(1.9e12 / (4.0 * n_in * n_out))
        return dict(op=op, rows=log_int(rng, 1, max(1, min(8192, most))), **both)
    experts = log_int(rng, 2, 128)
    while 2 * experts * n_in * n_out > 1 << 30:
        experts = max(1, experts // 2)
        both["n_in"] = n_in = max(128, n_in * 3 // 4)
    k = rng.randint(1, min(8, experts))
    most = int(1.9e12 / (4.0 * k * n_in * n_out))
    tokens = log_int(rng, 1, max(1, min(8192, most)))
    return dict(op=op, tokens=tokens, k=k, experts=experts, listed=rng.random() < .5,
                dropped=rng.choice([0, tokens * k // 7]), idle=rng.choice([0, experts // 4]), **both)


# ----------------------------------------------------------------- inputs --
def padded(n, dtype):
    """Elements between rows of n: 16 bytes' multiple, as the products take them."""
    unit = 16 // SIZE[dtype]
    return -(-n // unit) * unit


def group_sizes(case):
    """Rows of each expert, uneven, `idle` experts without any and `dropped`
    pairs with no expert. They go by the case alone."""
    r = random.Random("%(tokens)d %(k)d %(experts)d %(idle)d" % case)
    E, picks = case["experts"], []
    live = r.sample(range(E), max(1, E - case["idle"]))
    if case["tokens"] <= 64 and len(live) >= case["k"]:
        for _ in range(case["tokens"]):
            picks += r.sample(live, case["k"])
    else:
        weight = [0.3 + r.random() ** 2 for _ in live]
        picks = r.choices(live, weight, k=case["tokens"] * case["k"])
    picks = picks[:max(0, len(picks) - case["dropped"])]
    sizes = [0] * E
    for e in picks:
        sizes[e] += 1
    return sizes


def normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def activations(gen, rows, cols):
    """Rows with a few heavy channels, as hidden states have them."""
    heavy = 1 + 3 * torch.rand(cols, generator=gen, device="cuda").pow(8)
    return normal(gen, rows, cols) * heavy


def to_e4m3(t):
    """t (64 bits) to the nearest e4m3 value, ties to even, held at +-448."""
    _, exponent = torch.frexp(t)
    step = torch.ldexp(torch.ones_like(t), exponent.clamp(min=-5) - 4)
    return (torch.round(t / step) * step).clamp(-448, 448)


def quantised(x, block):
    """e4m3 values (f32) of x [..., rows, cols] and their fp32 scales, one for
    each `block` rows and 128 channels; the division and its rounding in 64 bits."""
    rows, cols = x.shape[-2:]
    x = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK, 0, -rows % block))
    x = x.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, block))  # [.., row, in, col, in]
    s = (x.abs().amax((-3, -1)) / 448).float()
    t = s.double()[..., :, None, :, None]
    q = torch.where(t > 0, to_e4m3(x / torch.where(t > 0, t, 1.0)), 0.0)
    return q.flatten(-2).flatten(-3, -2)[..., :rows, :cols].float(), s


def weights(gen, case, s):
    """One matrix, or gate and up, for each expert: w [experts, 1 or 2, n_out, stride]
    and, in e4m3, scale [experts, 1 or 2, n_out / 128, n_in / 128]."""
    E, G, N, K = case.get("experts", 1), 1 + case["gated"], case["n_out"], case["n_in"]
    stride, dt = padded(K, case["dtype"]), DT[case["dtype"]]
    s["w"] = torch.zeros(E, G, N, stride, dtype=dt, device="cuda")
    e4m3 = case["dtype"] == "e4m3"
    if e4m3:
        s["ws"] = torch.empty(E, G, -(-N // BLOCK), -(-K // BLOCK), device="cuda")
    for e in range(E):
        for g in range(G):
            w = normal(gen, N, K) * (0.5 + torch.rand(N, 1, generator=gen, device="cuda")) / math.sqrt(K)
            if e4m3:
                w, s["ws"][e, g] = quantised(w, BLOCK)
            s["w"][e, g, :, :K] = w.to(dt)


def rows_in(gen, case, rows, s):
    """x [rows, stride] and, in e4m3, its scales."""
    K = case["n_in"]
    s["x"] = torch.zeros(rows, padded(K, case["dtype"]), dtype=DT[case["dtype"]], device="cuda")
    x = activations(gen, rows, K)
    if case["dtype"] == "e4m3":
        x, s["xs"] = quantised(x, 1)
    s["x"][:, :K] = x.to(s["x"].dtype)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case=case)
    op = case["op"]
    if op == "quantise":
        R, C = case["rows"], case["cols"]
        s["x"] = activations(gen, case["of"] or R, C).to(DT[case["dtype"]])
        if case["of"]:
            s["rows"] = torch.randint(case["of"], (R,), generator=gen, device="cuda").int()
        s["q"] = torch.zeros(R, padded(C, "e4m3"), dtype=torch.float8_e4m3fn, device="cuda")
        s["scale"] = torch.zeros(-(-R // case["block"]), -(-C // BLOCK), device="cuda")
        return s
    if op == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        skew = normal(gen, E)
        score = normal(gen, T, E) + 0.7 * skew
        score = (score * 64).round() / 64  # 16-bit routers give equal scores now and then
        off = torch.rand(T, E, generator=gen, device="cuda").argsort(-1) < case["masked"]
        some = torch.rand(T, 1, generator=gen, device="cuda") < 0.3
        s["score"] = torch.where(off & some, -math.inf, score)
        s["ids"] = torch.zeros(T, k, dtype=torch.int32, device="cuda")
        if case["given"]:
            s["ids"] = s["score"].topk(k).indices.int()
            s["ids"][torch.rand(T, k, generator=gen, device="cuda") < 0.1] = -1  # padding
        s["weights"] = torch.zeros(T, k, device="cuda")
        s["offsets"] = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        s["rows"] = torch.zeros(T * k, dtype=torch.int32, device="cuda")
        s["place"] = torch.zeros(T, k, dtype=torch.int32, device="cuda")
        return s
    if op == "combine":
        T, k, C = case["tokens"], case["k"], case["cols"]
        s["y"] = normal(gen, T * k, C).to(DT[case["dtype"]])
        s["place"] = torch.randperm(T * k, generator=gen, device="cuda").int()
        s["place"] = torch.where(s["place"] < T * k - case["dropped"], s["place"], -1).view(T, k)
        s["weights"] = normal(gen, T, k).softmax(-1)
        s["base"] = normal(gen, T, C).to(DT[case["out"]]) if case["base"] else None
        s["out"] = torch.zeros(T, C, dtype=DT[case["out"]], device="cuda")
        return s
    weights(gen, case, s)
    if op == "linear":
        rows = case["rows"]
        rows_in(gen, case, rows, s)
    else:
        sizes, rows = group_sizes(case), case["tokens"] * case["k"]
        ends = torch.tensor([0] + sizes).cumsum(0)
        s["offsets"], s["most"] = ends.int().cuda(), max(1, max(sizes))
        rows_in(gen, case, case["tokens"] if case["listed"] else rows, s)
        if case["listed"]:
            pair = torch.randperm(rows, generator=gen, device="cuda") // case["k"]
            s["rows"] = torch.where(torch.arange(rows, device="cuda") < sum(sizes), pair, -1).int()
    s["y"] = torch.zeros(rows, case["n_out"], dtype=DT[case["out"]], device="cuda")
    if own:
        from rabbit_b200 import capi
        s["linear"] = capi.Linear(library_dtype(case["dtype"]), case["n_out"], case["n_in"],
                                  s["w"].data_ptr(), n_experts=case.get("experts", 1),
                                  gated=case["gated"], w_stride=s["w"].shape[-1],
                                  d_scale=s["ws"].data_ptr() if "ws" in s else 0)
    return s


def library_dtype(dtype):
    from rabbit_b200 import capi
    return {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16, "e4m3": capi.E4M3}[dtype]


# ------------------------------------------------------------ plain forms --
def dequantised(q, scale, block):
    """Values times their block's scale, in 32 bits; q [..., rows, cols]."""
    s = scale.repeat_interleave(block, -2)[..., :q.shape[-2], :]
    return q.float() * s.repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]


def plain_operands(s):
    K = s["case"]["n_in"]
    x, w = s["x"][:, :K], s["w"][..., :K]
    if s["case"]["dtype"] == "e4m3":
        return dequantised(x, s["xs"], 1), dequantised(w, s["ws"], BLOCK)
    return x.float(), w.float()


def product(x, w):
    """x [.., rows, K], w [.., 1 or 2, N, K]: the product, or silu(gate) * up."""
    y = x @ w[..., 0, :, :].transpose(-1, -2)
    if w.shape[-3] == 1:
        return y
    return y / (1 + torch.exp(-y)) * (x @ w[..., 1, :, :].transpose(-1, -2))


def plain_grouped(s):
    case, x_w = s["case"], plain_operands(s)
    rows, start = case["tokens"] * case["k"], s["offsets"][:-1].long()
    at = start[:, None] + torch.arange(s["most"], device="cuda")  # [expert, row of it]
    real = at < s["offsets"][1:, None]
    at = torch.where(real, at, rows)  # the padding reads row 0 and goes to one row more
    source = s["rows"].clamp(min=0).long() if case["listed"] else torch.arange(rows, device="cuda")
    source = torch.nn.functional.pad(source, (0, 1))
    y = product(x_w[0][source[at]], x_w[1])
    out = torch.zeros(rows + 1, case["n_out"], dtype=s["y"].dtype, device="cuda")
    out[at] = y.to(out.dtype)
    out[rows] = 0
    return out[:rows]


def plain_route(s):
    case, E, k = s["case"], s["case"]["experts"], s["case"]["k"]
    if case["given"]:
        ids, found = s["ids"].long(), {}
    else:
        score, order = s["score"].sort(dim=-1, descending=True, stable=True)  # equal: lowest id first
        top, total = score[:, :1], score if case["over_all"] else score[:, :k]
        e = torch.where(total > -math.inf, torch.exp(total - torch.where(top > -math.inf, top, 0.0)), 0.0)
        real = score[:, :k] > -math.inf
        weight = torch.where(real, e[:, :k] / e.sum(-1, keepdim=True).clamp(min=1e-30), 0.0)
        ids = torch.where(real, order[:, :k], -1)
        found = {"ids": ids.int(), "weights": weight}
    flat = torch.where(ids < 0, E, ids).flatten()
    by_expert, pair = flat.sort(stable=True)
    live = by_expert < E
    place = torch.empty_like(pair)
    place[pair] = torch.where(live, torch.arange(pair.numel(), device="cuda"), -1)
    ends = (by_expert[:, None] < torch.arange(E + 1, device="cuda")).sum(0)
    return {**found, "offsets": ends.int(), "rows": torch.where(live, pair // k, -1).int(),
            "place": place.view(ids.shape).int()}


def plain_combine(s):
    place = s["place"].long()
    y = torch.where((place < 0)[..., None], 0.0, s["y"].float()[place.clamp(min=0)])
    out = (s["weights"][..., None] * y).sum(1)
    if s["base"] is not None:
        out = s["base"].float() + out
    return out.to(s["out"].dtype)


# -------------------------------------------------------------------- run --
def run(s):
    case, op = s["case"], s["case"]["op"]
    if not own:
        if op == "quantise":
            x = s["x"][s["rows"].long()] if case["of"] else s["x"]
            q, scale = quantised(x, case["block"])
            return {"q": q.to(torch.float8_e4m3fn), "scale": scale}
        if op == "linear":
            x, w = plain_operands(s)
            return product(x, w[0]).to(s["y"].dtype)
        return {"grouped": plain_grouped, "route": plain_route, "combine": plain_combine}[op](s)
    from rabbit_b200 import capi
    stream = torch.cuda.current_stream().cuda_stream
    if op == "quantise":
        capi.f8_quantise_dev(library_dtype(case["dtype"]), s["x"].data_ptr(), s["q"].data_ptr(),
                             s["scale"].data_ptr(), case["rows"], case["cols"],
                             q_stride=s["q"].shape[1], block_rows=case["block"],
                             d_rows=s["rows"].data_ptr() if case["of"] else 0,
                             x_rows=s["x"].shape[0], stream=stream)
        return {"q": s["q"][:, :case["cols"]], "scale": s["scale"]}
    if op == "route":
        given = case["given"]
        capi.experts_route_dev(0 if given else s["score"].data_ptr(), case["tokens"],
                               case["experts"], case["k"], s["ids"].data_ptr(),
                               0 if given else s["weights"].data_ptr(), s["offsets"].data_ptr(),
                               s["rows"].data_ptr(), s["place"].data_ptr(),
                               over_all=case["over_all"], stream=stream)
        found = {} if given else {"ids": s["ids"], "weights": s["weights"]}
        return {**found, "offsets": s["offsets"], "rows": s["rows"], "place": s["place"]}
    if op == "combine":
        capi.experts_combine_dev(library_dtype(case["dtype"]), s["y"].data_ptr(), s["y"].shape[0],
                                 s["place"].data_ptr(), s["weights"].data_ptr(), case["tokens"],
                                 case["k"], case["cols"], library_dtype(case["out"]),
                                 s["out"].data_ptr(),
                                 d_base=s["base"].data_ptr() if case["base"] else 0, stream=stream)
        return s["out"]
    scales = dict(d_x_scale=s["xs"].data_ptr()) if "xs" in s else {}
    if op == "linear":
        s["linear"].apply_dev(s["x"].data_ptr(), library_dtype(case["out"]), s["y"].data_ptr(),
                              case["rows"], x_stride=s["x"].shape[1], stream=stream, **scales)
    else:
        s["linear"].grouped_dev(s["x"].data_ptr(), s["x"].shape[0], s["offsets"].data_ptr(),
                                library_dtype(case["out"]), s["y"].data_ptr(), s["y"].shape[0],
                                d_rows=s["rows"].data_ptr() if case["listed"] else 0,
                                x_stride=s["x"].shape[1], stream=stream, **scales)
    return s["y"]


# ------------------------------------------------------------------- work --
def work(case):
    op = case["op"]
    if op == "quantise":
        R, C = case["rows"], case["cols"]
        read = min(R, case["of"]) if case["of"] else R
        blocks = -(-R // case["block"]) * -(-C // BLOCK)
        return dict(bytes=read * C * SIZE[case["dtype"]] + R * C + 4 * blocks + 4 * R * bool(case["of"]),
                    flops=3 * R * C)
    if op == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        scores = 0 if case["given"] else 4 * T * E + 4 * T * k
        return dict(bytes=scores + 4 * (3 * T * k + E + 1), flops=0 if case["given"] else 3 * T * E)
    if op == "combine":
        T, k, C = case["tokens"], case["k"], case["cols"]
        rows = T * k - case["dropped"]
        return dict(bytes=rows * C * SIZE[case["dtype"]] + T * C * SIZE[case["out"]] * (1 + case["base"])
                    + 8 * T * k, flops=2 * rows * C)
    sizes = [case["rows"]] if op == "linear" else group_sizes(case)
    rows, G, N, K = sum(sizes), 1 + case["gated"], case["n_out"], case["n_in"]
    live, size = sum(n > 0 for n in sizes), SIZE[case["dtype"]]
    read = min(rows, case["tokens"]) if case.get("listed") else rows
    scales = 4 * -(-K // BLOCK) * (read + live * G * -(-N // BLOCK)) if size == 1 else 0
    return dict(bytes=read * K * size + live * G * N * K * size + scales + rows * N * SIZE[case["out"]],
                flops=2.0 * rows * K * N * G)


# ------------------------------------------------------------------ exact --
def exact_codes(x, s):
    """The e4m3 values nearest to x / s: the 127 that are not negative, searched."""
    held = torch.arange(127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    t = torch.where(s > 0, x.abs() / torch.where(s > 0, s, 1.0), 0.0)
    up = torch.searchsorted(held, t.contiguous()).clamp(1, 126)
    low, high = held[up - 1], held[up]
    mid = (low + high) / 2
    above = (t > mid) | ((t == mid) & (up % 2 == 0))
    return torch.where(above, high, low) * torch.where(x < 0, -1.0, 1.0)


def exact_quantise(s):
    case, b = s["case"], s["case"]["block"]
    x = s["x"].double()
    if case["of"]:
        x = x.index_select(0, s["rows"].long())
    q = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    scale = torch.empty(-(-case["rows"] // b), -(-case["cols"] // BLOCK), dtype=torch.float64, device="cuda")
    for j in range(scale.shape[1]):
        part = x[:, j * BLOCK:(j + 1) * BLOCK]
        top = part.abs().max(1).values
        if b > 1:
            top = torch.stack([t.max() for t in top.split(b)])
        scale[:, j] = (top / 448.0).to(torch.float32).double()
        q[:, j * BLOCK:(j + 1) * BLOCK] = exact_codes(
            part, scale[:, j].repeat_interleave(b)[:case["rows"], None])
    return {"q": q, "scale": scale}


def exact_product(s, x, xs, e):
    """Rows x of expert e in 64 bits, block by block of the channels."""
    K, y = s["case"]["n_in"], []
    for g in range(s["w"].shape[1]):
        if xs is None:
            y.append(x[:, :K].double() @ s["w"][e, g, :, :K].double().T)
            continue
        block = torch.arange(K, device="cuda") // BLOCK
        ws = s["ws"][e, g][torch.arange(s["case"]["n_out"], device="cuda") // BLOCK].double()
        y.append((x[:, :K].double() * xs.double()[:, block])
                 @ (s["w"][e, g, :, :K].double() * ws[:, block]).T)
    return y[0] if len(y) == 1 else y[0] * torch.sigmoid(y[0]) * y[1]


def exact_route(s):
    case, E, k = s["case"], s["case"]["experts"], s["case"]["k"]
    T, weight = case["tokens"], None
    if case["given"]:
        ids = s["ids"].long()
    else:
        left, ids = s["score"].double().clone(), []
        weight = torch.zeros(T, k, dtype=torch.float64, device="cuda")
        for j in range(k):  # the first of the largest that are left, k times
            top = left.max(-1, keepdim=True).values
            first = (left == top).to(torch.uint8).argmax(-1, keepdim=True)
            ids.append(torch.where(top > -math.inf, first, -1))
            left.scatter_(1, first, -math.inf)
        ids = torch.cat(ids, 1)
        picked = torch.where(ids >= 0, s["score"].double().gather(1, ids.clamp(min=0)), -math.inf)
        total = torch.logsumexp(s["score"].double() if case["over_all"] else picked, -1, keepdim=True)
        weight = torch.where(ids >= 0, torch.exp(picked - total), 0.0)
    pairs = sorted((e, p) for p, e in enumerate(ids.flatten().tolist()) if e >= 0)
    place, rows, ends = [-1] * (T * k), [-1] * (T * k), [0] * (E + 1)
    for at, (e, p) in enumerate(pairs):
        place[p], rows[at] = at, p // k
        ends[e + 1] += 1
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    found = {} if case["given"] else {"ids": ids.int(), "weights": weight}
    return {**found, "offsets": whole(ends).cumsum(0).int(), "rows": whole(rows),
            "place": whole(place).view(T, k)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        return exact_quantise(s)
    if case["op"] == "route":
        return exact_route(s)
    if case["op"] == "combine":
        out = torch.zeros(case["tokens"], case["cols"], dtype=torch.float64, device="cuda")
        if case["base"]:
            out += s["base"].double()
        for j in range(case["k"]):
            t = (s["place"][:, j] >= 0).nonzero()[:, 0]
            out[t] += s["weights"][t, j, None].double() * s["y"][s["place"][t, j].long()].double()
        return out
    if case["op"] == "linear":
        return exact_product(s, s["x"], s.get("xs"), 0)
    out = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    ends = s["offsets"].tolist()
    for e in range(case["experts"]):
        a, b = ends[e], ends[e + 1]
        if b > a:
            at = s["rows"][a:b].long() if case["listed"] else torch.arange(a, b, device="cuda")
            out[a:b] = exact_product(s, s["x"][at], s["xs"][at] if "xs" in s else None, e)
    return out
