"""The cache-side operators of a decoding engine, as cases that can be timed:

rope       rotary positions of query / key rows (interleaved or half pairs,
           part of the head, scaled for long contexts);
append     keys and values written into a paged cache of 4-bit groups, the
           keys rotated on the way; returned are the rows as the cache then
           holds them;
attention  queries against that cache, one token a sequence or many.

`own` False computes them with elementary torch operations; True calls the
library (rabbit_b200.capi). The 4-bit format, for 32 consecutive channels x of
one (token, head): scale s = bf16(max|x| / 7), code = rint(x / s), held as
code * s (s = 0: all zero).
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one token of the OLMoE-shaped model (16 heads x 128, fp32, the
        # reference's interleaved pairs): the smallest call, all latency
        dict(name="rope 1x16x128 f32", op="rope", dtype="f32", tokens=1, heads=16, head_dim=128,
             rot=128, layout="interleaved", scaling="none", factor=1.0, far=256),
        # query and key heads of a fused projection (32 + 8 heads, half of
        # each head rotated), a 256-token chunk far into a scaled context
        dict(name="rope 257x40x128 half part", op="rope", dtype="bf16", tokens=257, heads=40,
             head_dim=128, rot=64, layout="half", scaling="yarn", factor=32.0, far=131072),
        # a long prompt's queries at once
        dict(name="rope 16384x32x128 bf16", op="rope", dtype="bf16", tokens=16384, heads=32,
             head_dim=128, rot=128, layout="half", scaling="bands", factor=8.0, far=32768),
        # the OLMoE-shaped model's token into its cache (16 KV heads, fp32)
        dict(name="append 1x16x128 f32", op="append", dtype="f32", tokens=1, kv_heads=16,
             head_dim=128, page=16, rot=128, layout="interleaved", scaling="none", factor=1.0,
             far=256, skipped=0),
        # a decode step of 64 sequences, a few of them padding
        dict(name="append 64x8x128 bf16", op="append", dtype="bf16", tokens=64, kv_heads=8,
             head_dim=128, page=64, rot=128, layout="half", scaling="linear", factor=4.0,
             far=16384, skipped=5),
        # a long prompt: an odd number of tokens, a head of two and a half groups
        dict(name="append 8191x8x80 f16", op="append", dtype="f16", tokens=8191, kv_heads=8,
             head_dim=80, page=32, rot=32, layout="half", scaling="ntk", factor=2.0, far=65536,
             skipped=0),
        # the OLMoE-shaped model's decode step at the end of its 256-token window
        dict(name="attention 1x255 f32 mha", op="attention", dtype="f32", seqs=1, q_len=1, ctx=255,
             heads=16, kv_heads=16, head_dim=128, page=16, window=0, empty=0, pad=0),
        # a Mixtral-shaped decode batch, ragged, two sequences not yet begun
        # and padded rows behind the last
        dict(name="attention 64x4096 bf16", op="attention", dtype="bf16", seqs=64, q_len=1,
             ctx=4096, heads=32, kv_heads=8, head_dim=128, page=64, window=0, empty=2, pad=3),
        # one long conversation, the split over positions carries it
        dict(name="attention 1x131072 bf16", op="attention", dtype="bf16", seqs=1, q_len=1,
             ctx=131072, heads=32, kv_heads=8, head_dim=128, page=64, window=0, empty=0, pad=0),
        # drafted tokens checked four at a time within a window, 48 query heads, fp32
        dict(name="attention 16x4 draft f32", op="attention", dtype="f32", seqs=16, q_len=4,
             ctx=5000, heads=48, kv_heads=8, head_dim=128, page=32, window=2048, empty=0, pad=0),
        # a 256-token prefill chunk behind 4096 cached positions
        dict(name="attention 256 chunk bf16", op="attention", dtype="bf16", seqs=1, q_len=256,
             ctx=4352, heads=32, kv_heads=8, head_dim=128, page=64, window=0, empty=0, pad=0),
        # a large decode batch: the most bytes
        dict(name="attention 128x8192 f16", op="attention", dtype="f16", seqs=128, q_len=1,
             ctx=8192, heads=32, kv_heads=8, head_dim=128, page=128, window=0, empty=0, pad=0),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw_scaling(rng):
    s = rng.choice(["none", "linear", "ntk", "bands", "yarn"])
    return dict(scaling=s, factor=1.0 if s == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    hd = rng.choice([32, 64, 80, 96, 128, 128, 128, 256])
    layout = rng.choice(["interleaved", "half"])
    rot = rng.choice([hd, hd, hd // 2])
    if op == "rope":
        heads = rng.choice([1, 3, 8, 16, 20, 32, 40, 48])
        most = 16384 * 32 * 128 * 2 // (heads * hd * (4 if dtype == "f32" else 2))
        return dict(op=op, dtype=dtype, tokens=log_int(rng, 1, min(16384, most)), heads=heads,
                    head_dim=hd, rot=rot, layout=layout, far=log_int(rng, 16400, 1 << 20),
                    **draw_scaling(rng))
    if op == "append":
        tokens = log_int(rng, 1, 8191)
        return dict(op=op, dtype=dtype, tokens=tokens, kv_heads=rng.choice([1, 2, 4, 5, 8, 16]),
                    head_dim=hd, page=rng.choice([16, 32, 64, 128]), rot=rot, layout=layout,
                    far=log_int(rng, 16400, 1 << 20), skipped=rng.choice([0, 0, tokens // 5]),
                    **draw_scaling(rng))
    kvh = rng.choice([1, 2, 4, 8, 16])
    heads = kvh * rng.choice([1, 2, 3, 4, 6, 7, 8, 16])
    q_len = rng.choice([1, 1, 1, 2, 5, log_int(rng, 8, 256)])
    ctx = log_int(rng, q_len, 65536)
    seqs = log_int(rng, 1, 128)
    # within half the largest listed case's cache and the listed chunk's products
    while seqs > 1 and (seqs * ctx * kvh * hd > 1 << 29 or seqs * q_len * ctx * heads * hd > 1 << 32):
        seqs //= 2
    while ctx > q_len and (ctx * kvh * hd > 1 << 29 or q_len * ctx * heads * hd > 1 << 32):
        ctx = max(q_len, ctx // 2)
    return dict(op=op, dtype=dtype, seqs=seqs, q_len=q_len, ctx=ctx, heads=heads, kv_heads=kvh,
                head_dim=hd, page=rng.choice([16, 32, 64, 128]),
                window=rng.choice([0, 0, 1 + ctx // 3]), empty=seqs // 8 if rng.random() < .3 else 0,
                pad=rng.choice([0, 0, 2]))


# ----------------------------------------------------------------- inputs --
def original_ctx(case):
    return 4096


def kv_lens(case):
    """The sequences' lengths: a batch is ragged, `empty` of it not begun, the
    first one at full length. They go by the case alone."""
    r = random.Random("%(seqs)d %(ctx)d %(q_len)d %(heads)d" % case)
    lens = [case["ctx"]]
    for _ in range(case["seqs"] - 1):
        lens.append(max(case["q_len"], int(case["ctx"] * r.uniform(0.15, 1.0))))
    for i in range(case["empty"]):
        lens[-1 - 3 * i if 3 * i < case["seqs"] - 1 else -1] = 0
    return lens


def q_lens(case):
    """One token a sequence, or up to q_len, the first sequence all of it; a
    sequence that has not begun asks one token over nothing."""
    r = random.Random("q %(seqs)d %(ctx)d %(q_len)d %(heads)d" % case)
    first = [case["q_len"]]
    rest = [r.randint((case["q_len"] + 1) // 2, case["q_len"]) for _ in range(case["seqs"] - 1)]
    return [q if n else 1 for q, n in zip(first + rest, kv_lens(case))]


def normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def quantised(x):
    """Codes (f32 whole numbers) and bf16 scales of x [..., head_dim]; the
    division and its rounding in 64 bits."""
    hd = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -hd % GROUP)).unflatten(-1, (-1, GROUP))
    s = (x.abs().amax(-1).float() / 7).bfloat16()
    t = s.double().unsqueeze(-1)
    q = torch.where(t > 0, torch.round(x / torch.where(t > 0, t, 1.0)), 0.0)
    return q.clamp(-8, 7).float().flatten(-2)[..., :hd], s


def rope_turns(case, device):
    """Rotations per position of each pair (64 bits), and the magnitude."""
    n, base, fac, ctx = case["rot"], 10000.0, case["factor"], original_ctx(case)
    i = torch.arange(n // 2, dtype=torch.float64, device=device)
    if case["scaling"] == "ntk":
        base = base * fac ** (n / (n - 2.0))
    f = base ** (-2.0 * i / n)
    mag = 1.0
    if case["scaling"] == "linear":
        f = f / fac
    elif case["scaling"] == "bands":  # by the wavelength's share of the first context
        smooth = ((ctx * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = (1 - smooth) * f / fac + smooth * f
    elif case["scaling"] == "yarn":
        def dim(turns):
            return n * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), n - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / fac * ramp
        mag = 0.1 * math.log(fac) + 1.0
    return f, mag


def library_rope(case):
    from rabbit_b200 import capi
    return capi.Rope(case["head_dim"], rot_dim=case["rot"],
                     layout={"interleaved": capi.ROPE_INTERLEAVED, "half": capi.ROPE_HALF}[case["layout"]],
                     scaling={"none": capi.ROPE_SCALE_NONE, "linear": capi.ROPE_SCALE_LINEAR,
                              "ntk": capi.ROPE_SCALE_NTK, "bands": capi.ROPE_SCALE_BANDS,
                              "yarn": capi.ROPE_SCALE_YARN}[case["scaling"]],
                     base=10000.0, factor=case["factor"], original_ctx=original_ctx(case),
                     low=1.0, high={"bands": 4.0, "yarn": 32.0}.get(case["scaling"], 0.0))


def library_dtype(dtype):
    from rabbit_b200 import capi
    return {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}[dtype]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = DT[case["dtype"]]
    s = dict(case=case)
    if case["op"] in ("rope", "append"):
        T, hd = case["tokens"], case["head_dim"]
        heads = case["heads"] if case["op"] == "rope" else case["kv_heads"]
        # a run of positions that ends at the far end of the context
        end = int(torch.randint(max(T, case["far"] - 64), case["far"] + 1, (1,), generator=gen,
                                device="cuda"))
        s["pos"] = torch.arange(end - T, end, dtype=torch.int32, device="cuda")
        heavy = 1 + 3 * torch.rand(heads, hd, generator=gen, device="cuda").pow(8)
        s["x"] = (normal(gen, T, heads, hd) * heavy).to(dt)
        if case["op"] == "rope":
            if own:
                s["rope"], s["dt"] = library_rope(case), library_dtype(dt)
                s["y"] = torch.empty_like(s["x"])
            return s
        s["v"] = normal(gen, T, heads, hd).to(dt)
        pages = -(-T // case["page"]) + 3
        order = torch.randperm(pages, generator=gen, device="cuda")
        t = torch.arange(T, device="cuda")
        slots = order[t // case["page"]] * case["page"] + t % case["page"]
        gone = torch.randperm(T, generator=gen, device="cuda")[:case["skipped"]]
        s["slots"] = slots.index_fill(0, gone, -1)
        if own:
            from rabbit_b200 import capi
            s["rope"], s["dt"] = library_rope(case), library_dtype(dt)
            s["kv"] = capi.Kv4(n_layers=1, n_kv_heads=heads, head_dim=hd, page_size=case["page"],
                               n_pages=pages)
            s["k_held"] = torch.zeros(T, heads, hd, device="cuda")
            s["v_held"] = torch.zeros(T, heads, hd, device="cuda")
        return s

    # attention: a filled cache, its page table in no order, and the queries
    page, nkv, hd, heads = case["page"], case["kv_heads"], case["head_dim"], case["heads"]
    lens, qs = kv_lens(case), q_lens(case)
    wide = max(1, -(-max(lens) // page))
    used = sum(-(-n // page) for n in lens)
    pages = used + 1
    order = torch.randperm(pages, generator=gen, device="cuda")
    need = torch.tensor([-(-n // page) for n in lens], device="cuda")
    first = torch.cumsum(need, 0) - need
    at = first[:, None] + torch.arange(wide, device="cuda")
    real = torch.arange(wide, device="cuda") < need[:, None]
    s["table"] = torch.where(real, order[at.clamp(max=pages - 1)], 0).int()
    s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    start = [0]
    for q in qs:
        start.append(start[-1] + q)
    s["q_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    rows = start[-1] + case["pad"]
    s["q"] = normal(gen, rows, heads, hd).to(dt)
    heavy = 1 + 3 * torch.rand(nkv, hd, generator=gen, device="cuda").pow(8)
    if own:
        from rabbit_b200 import capi
        s["dt"] = library_dtype(dt)
        s["kv"] = capi.Kv4(n_layers=1, n_kv_heads=nkv, head_dim=hd, page_size=page, n_pages=pages)
        s["scratch"] = capi.Kv4Scratch(s["kv"])
        s["batch"] = capi.Kv4Batch(n_seqs=len(lens), d_kv_len=s["kv_len"].data_ptr(),
                                   d_page_table=s["table"].data_ptr(), max_pages=wide,
                                   d_q_start=s["q_start"].data_ptr(), max_q_len=max(qs))
        s["out"] = torch.zeros_like(s["q"])
    else:
        s["codes"] = [torch.empty(pages * page, nkv, hd, dtype=torch.int8, device="cuda") for _ in "kv"]
        s["scales"] = [torch.empty(pages * page, nkv, -(-hd // GROUP), dtype=torch.bfloat16,
                                   device="cuda") for _ in "kv"]
    step = max(1, (1 << 25) // (page * nkv * hd)) * page
    for a in range(0, pages * page, step):
        n = min(step, pages * page - a)
        k, v = normal(gen, n, nkv, hd) * heavy, normal(gen, n, nkv, hd)
        if own:
            slots = torch.arange(a, a + n, device="cuda")
            s["kv"].append_dev(0, library_dtype(torch.float32), k.data_ptr(), v.data_ptr(),
                               slots.data_ptr(), n,
                               stream=torch.cuda.current_stream().cuda_stream)
        else:
            for i, x in enumerate((k, v)):
                q, sc = quantised(x)
                s["codes"][i][a:a + n] = q.to(torch.int8)
                s["scales"][i][a:a + n] = sc
    return s


# ------------------------------------------------------------ plain forms --
def pairs(case, x):
    """The two halves of the rotated pairs of x [..., head_dim], and the rest."""
    r = x[..., :case["rot"]]
    if case["layout"] == "half":
        a, b = r.chunk(2, -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
    return a, b, x[..., case["rot"]:]


def joined(case, a, b, rest):
    both = torch.cat([a, b], -1) if case["layout"] == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([both, rest], -1)


def rotated(case, x, pos):
    """x [T, heads, head_dim] rotated, in x's own precision; angles in 64 bits."""
    f, mag = rope_turns(case, x.device)
    angle = pos.double()[:, None, None] * f
    c, n = (mag * torch.cos(angle)).to(x.dtype), (mag * torch.sin(angle)).to(x.dtype)
    a, b, rest = pairs(case, x)
    return joined(case, a * c - b * n, b * c + a * n, rest)


def plain_append(s):
    case, keep = s["case"], s["slots"] >= 0
    out = []
    for x in (rotated(case, s["x"].double(), s["pos"]), s["v"]):
        q, sc = quantised(x)
        held = q * sc.float().repeat_interleave(GROUP, -1)[..., :case["head_dim"]]
        out.append(torch.where(keep[:, None, None], held, 0.0))
    return {"k": out[0], "v": out[1]}


def plain_attention(s):
    case = s["case"]
    page, nkv, hd, heads = case["page"], case["kv_heads"], case["head_dim"], case["heads"]
    G, n_seq, wide = heads // nkv, case["seqs"], s["table"].shape[1] * case["page"]
    p = torch.arange(wide, device="cuda")
    slot = s["table"].long()[:, p // page] * page + p % page

    def cached(i):  # [seq, position, kv head, channel]
        sc = s["scales"][i][slot].float().repeat_interleave(GROUP, -1)[..., :hd]
        return s["codes"][i][slot].float() * sc

    # the queries laid out by sequence, padded to the longest
    q_len = s["q_start"].diff()
    qi = torch.arange(case["q_len"], device="cuda")
    row = (s["q_start"][:-1, None] + qi).clamp(max=s["q"].shape[0] - 1).long()
    real = qi < q_len[:, None]
    q = s["q"].float()[row].view(n_seq, case["q_len"], nkv, G, hd)
    at = s["kv_len"][:, None] - q_len[:, None] + qi  # [seq, query]
    seen = (p <= at[..., None]) & (p < s["kv_len"][:, None, None])
    if case["window"]:
        seen &= p > at[..., None] - case["window"]
    seen = seen[:, None, :, None, :]
    score = torch.einsum("sqngd,spnd->snqgp", q, cached(0)) / math.sqrt(hd)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    total = e.sum(-1).permute(0, 2, 1, 3).unsqueeze(-1)
    o = torch.einsum("snqgp,spnd->sqngd", e, cached(1))
    o = torch.where(total > 0, o / total, 0.0).reshape(n_seq, case["q_len"], heads, hd)
    rows = s["q"].shape[0]  # the padding goes to one row more
    out = torch.zeros(rows + 1, heads, hd, dtype=s["q"].dtype, device="cuda")
    out[torch.where(real, row, rows)] = o.to(out.dtype)
    return out[:rows]


# -------------------------------------------------------------------- run --
def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "rope":
            return rotated(case, s["x"].float(), s["pos"]).to(s["x"].dtype)
        return plain_append(s) if case["op"] == "append" else plain_attention(s)
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "rope":
        s["rope"].apply_dev(s["dt"], s["x"].data_ptr(), s["y"].data_ptr(), s["pos"].data_ptr(),
                            case["tokens"], case["heads"], stream=stream)
        return s["y"]
    if case["op"] == "append":
        s["kv"].append_dev(0, s["dt"], s["x"].data_ptr(), s["v"].data_ptr(), s["slots"].data_ptr(),
                           case["tokens"], rope=s["rope"], d_positions=s["pos"].data_ptr(),
                           stream=stream)
        s["kv"].read_dev(0, library_dtype(torch.float32), s["slots"].data_ptr(), case["tokens"],
                         s["k_held"].data_ptr(), s["v_held"].data_ptr(), stream=stream)
        return {"k": s["k_held"], "v": s["v_held"]}
    s["kv"].attention_dev(0, s["scratch"], s["dt"], s["q"].data_ptr(), s["out"].data_ptr(),
                          s["q"].shape[0], case["heads"], s["batch"], window=case["window"],
                          stream=stream)
    return s["out"]


# ------------------------------------------------------------------- work --
def visible(case):
    """(positions that some query sees, (query, position) pairs) over the batch."""
    some = each = 0
    for n, q in zip(kv_lens(case), q_lens(case)):
        low = high = None
        for i in range(q):
            at = n - q + i
            a = max(0, at - case["window"] + 1) if case["window"] else 0
            if at >= a and n:
                each += at + 1 - a
                low = a if low is None else min(low, a)
                high = at + 1
        some += 0 if low is None else high - low
    return some, each


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    hd = case["head_dim"]
    row = hd / 2 + 2 * -(-hd // GROUP)  # a cached row of one head
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return dict(bytes=2 * n * hd * size + 4 * case["tokens"], flops=3 * n * case["rot"])
    if case["op"] == "append":
        n = (case["tokens"] - case["skipped"]) * case["kv_heads"]
        return dict(bytes=2 * n * hd * size + 2 * n * row + 2 * n * hd * 4 + 12 * case["tokens"],
                    flops=n * (3 * case["rot"] + 2 * 3 * hd))
    some, each = visible(case)
    rows = sum(q_lens(case))
    return dict(bytes=2 * some * case["kv_heads"] * row + 2 * rows * case["heads"] * hd * size,
                flops=4 * each * case["heads"] * hd)


# ------------------------------------------------------------------ exact --
def exact_rope(case, x, pos):
    """Every pair's rotation as a complex product, all in 64 bits."""
    n, ctx, out = case["rot"], float(original_ctx(case)), x.double().clone()
    pos = pos.double()
    for i in range(n // 2):
        base = 10000.0
        if case["scaling"] == "ntk":
            base *= math.pow(case["factor"], n / (n - 2))
        freq, mag = math.pow(base, -2 * i / n), 1.0
        if case["scaling"] == "linear":
            freq /= case["factor"]
        if case["scaling"] == "bands":
            wave = 2 * math.pi / freq
            if wave > ctx:
                freq /= case["factor"]
            elif wave > ctx / 4:
                keep = (ctx / wave - 1) / 3
                freq = keep * freq + (1 - keep) * freq / case["factor"]
        if case["scaling"] == "yarn":
            lo, hi = (n * math.log(ctx / (r * 2 * math.pi)) / (2 * math.log(10000.0)) for r in (32, 1))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), n - 1)
            t = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            freq, mag = freq * (1 - t) + freq / case["factor"] * t, 1 + math.log(case["factor"]) / 10
        a, b = (i, i + n // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., a].double(), x[..., b].double())
        z = z * torch.polar(torch.full_like(pos, mag), pos * freq)[:, None]
        out[..., a], out[..., b] = z.real, z.imag
    return out


def exact_held(x):
    """x [..., head_dim] as groups of 4-bit codes stand for it."""
    out = torch.zeros_like(x)
    for c in range(0, x.shape[-1], GROUP):
        g = x[..., c:c + GROUP]
        s = (g.abs().max(-1, keepdim=True).values.float() / 7).to(torch.bfloat16).double()
        q = torch.where(s == 0, 0.0, (g / s).round())
        out[..., c:c + GROUP] = q * s
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return exact_rope(case, s["x"], s["pos"])
    if case["op"] == "append":
        k, v = exact_held(exact_rope(case, s["x"], s["pos"])), exact_held(s["v"].double())
        k[s["slots"] < 0], v[s["slots"] < 0] = 0, 0
        return {"k": k, "v": v}
    page, hd, G = case["page"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = torch.arange(hd, device="cuda") // GROUP
    row = 0
    for i, (n, q) in enumerate(zip(kv_lens(case), q_lens(case))):
        if n:
            p = torch.arange(n, device="cuda")
            slot = s["table"][i, p // page].long() * page + p % page
            k, v = (c[slot].double() * sc[slot].double()[..., group]
                    for c, sc in zip(s["codes"], s["scales"]))
            at = torch.arange(n - q, n, device="cuda")[:, None]
            hidden = (p > at) | ((p <= at - case["window"]) if case["window"] else (p < 0))
            for h in range(case["heads"]):
                z = s["q"][row:row + q, h].double() @ k[:, h // G].T / hd ** 0.5
                w = z.masked_fill(hidden, -math.inf).softmax(-1).nan_to_num(0.0)
                out[row:row + q, h] = w @ v[:, h // G]
        row += q
    return out
