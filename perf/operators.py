"""Cases of the operators between a layer's q / k / v projections and its output projection: the rotation of queries and
keys by their positions, the per-head norm of queries and keys fused with that rotation and with the write into the
paged cache, and attention over the paged cache with an optional sliding window and sink tokens.

`own` selects what `run` calls: the framework's operators, or their plain form (elementary torch operations in 32 bits,
angles in 64). Head counts are those of this repository's layer (40 query heads over 8 key heads of 128 channels: q
5120 rows, k and v 1024) beside generic ones; 4096 rows and up to 16 verified tokens are its benchmark's sizes.
"""

import math
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    def rope(name, T, heads, kv_heads, dim, rot, **more):
        return dict({"name": name, "op": "rope", "T": T, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
                     "interleaved": False, "scaling": "none", "factor": 1.0, "dtype": "bf16", "far": 4096}, **more)

    def norm(name, T, heads, kv_heads, dim, rot, **more):
        return dict(rope(name, T, heads, kv_heads, dim, rot), **dict({"op": "norm", "into": "bf16", "page": 64}, **more))

    def attn(name, B, new, past, **more):
        return dict({"name": name, "op": "attn", "B": B, "new_min": new[0], "new": new[1], "past_min": past[0], "past": past[1],
                     "heads": 40, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "sinks": 0, "dtype": "bf16"}, **more)

    return [
        # one new token far into a long context, rotated with frequencies stretched for it: latency
        rope("rope 1 token", 1, 40, 8, 128, 128, far=900000, scaling="yarn", factor=32.0),
        # a prompt chunk of a model that rotates a quarter of each head in adjacent pairs
        rope("rope prompt", 8191, 24, 4, 256, 64, interleaved=True, dtype="fp16", far=131072, scaling="linear", factor=4.0),
        # the decode step of a batch: the stacked projection's fp32 rows into queries and the cache
        norm("norm+rope decode", 33, 40, 8, 128, 128, dtype="fp32", far=30000),
        # the benchmark's prefill chunk
        norm("norm+rope prefill", 4096, 40, 8, 128, 128, far=16384),
        # the first tokens of one conversation: the smallest call, latency only
        attn("decode 1 x 700", 1, (1, 1), (699, 699)),
        # one long context: all of the GPU for one sequence
        attn("decode 1 x 128k", 1, (1, 1), (131071, 131071)),
        # a serving batch of ragged long contexts: cache bandwidth
        attn("decode 16 x 32k", 16, (1, 1), (20000, 32767), page=16),
        # a large batch that keeps a window and the first tokens of each conversation
        attn("decode 64, window 4096", 64, (1, 1), (1000, 30000), window=4096, sinks=4, dtype="fp16", heads=32, page=32),
        # speculative verification of up to 16 tokens for a ragged batch
        attn("verify 16 x 16", 16, (1, 16), (500, 9000)),
        # fresh prompts of different lengths with a window of 1024 and 64 sink tokens
        attn("prefill 4, window 1024", 4, (1500, 8001), (0, 0), window=1024, sinks=64),
        # the next chunk of a long prompt; the wide heads of the larger layers
        attn("chunk 512 at 24k", 1, (512, 512), (24000, 24000), heads=24, kv_heads=4, dim=256),
        # a whole prompt: tensor-core throughput
        attn("prefill 8192", 1, (8192, 8192), (0, 0)),
    ]


MOST_SCORES = 40 * 8192 * 8192  # of the largest listed case: what the plain form holds at once


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["rope", "norm", "attn", "attn", "attn"])
    heads, kv_heads, dim = rng.choice([(40, 8, 128), (32, 8, 128), (24, 4, 256), (16, 16, 64), (12, 1, 128), (64, 8, 64), (7, 7, 128)])
    if kind != "attn":
        c = {"op": kind, "T": log(1, 8191), "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": dim // rng.choice([1, 1, 2, 4]),
             "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "factor": 1.0,
             "dtype": rng.choice(["bf16", "fp16", "fp32"]) if kind == "rope" else rng.choice(["bf16", "fp32"]), "far": log(8192, 1 << 20)}
        if c["scaling"] != "none":
            c["factor"] = float(rng.choice([2, 4, 8, 32]))
        if kind == "norm":
            c["into"] = rng.choice(["bf16", "fp16"])
            c["page"] = rng.choice([16, 32, 64, 128])
        return c
    most = max(work(x)["flops"] for x in listed())
    bytes_ = max(work(x)["bytes"] for x in listed())
    while True:
        phase = rng.choice(["decode", "verify", "prefill", "chunk"])
        c = {"op": "attn", "B": log(1, 96) if phase in ("decode", "verify") else log(1, 12)}
        new = {"decode": 1, "verify": rng.randint(2, 16), "prefill": log(17, 8192), "chunk": log(17, 2048)}[phase]
        past = 0 if phase == "prefill" else log(1, 65536)
        c["new_min"], c["new"] = (new, new) if rng.random() < 0.3 else (max(1, rng.randint(new // 4, new)), new)
        c["past_min"], c["past"] = (past, past) if rng.random() < 0.3 else (rng.randint(past // 4, past), past)
        c |= {"heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128])}
        c |= {"window": 0, "sinks": 0, "dtype": rng.choice(["bf16", "fp16"])}
        if rng.random() < 0.5:
            c["window"], c["sinks"] = log(100, 8192), rng.choice([0, 1, 4, 64, 130])
        w = work(c)
        if c["B"] * c["new"] * heads * (c["new"] + c["past"]) <= MOST_SCORES and w["flops"] <= most and w["bytes"] <= bytes_ \
                and c["B"] * (c["new"] + c["past"]) * kv_heads * dim <= 16 * 32768 * 1024:
            return c


def lengths(case):
    """New tokens and tokens in the cache (the new ones among them) of each sequence: spread evenly, in mixed order."""
    B = case["B"]
    at = [(b * 37 % B) / max(B - 1, 1) if B > 1 and math.gcd(37, B) == 1 else (b / max(B - 1, 1)) for b in range(B)]
    new = [case["new"] - int(x * (case["new"] - case["new_min"])) for x in at]
    past = [case["past_min"] + int(x * (case["past"] - case["past_min"])) for x in at]
    return new, [n + p for n, p in zip(new, past)]


def seen_pairs(new, kv, window, sinks):
    """(query, key) pairs that the mask leaves, and keys that at least one query of the sequence sees."""
    pairs = keys = 0
    first = kv - new
    for p in range(first, kv):
        low = max(0, p - window + 1) if window else 0
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, first - window + 1) if window else 0
    keys = kv - low + min(sinks, low)
    return pairs, keys


def work(case):
    D, Hq, Hk = case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "attn":
        pairs = keys = 0
        new, kv = lengths(case)
        for n, k in zip(new, kv):
            a, b = seen_pairs(n, k, case["window"], case["sinks"])
            pairs, keys = pairs + a, keys + b
        return {"bytes": 2 * (2 * sum(new) * Hq * D + 2 * keys * Hk * D), "flops": 4 * pairs * Hq * D}
    size = 4 if case["dtype"] == "fp32" else 2
    T, rows = case["T"], Hq + Hk
    if case["op"] == "rope":
        return {"bytes": 2 * T * rows * D * size + 8 * T, "flops": 3 * T * rows * case["rot"]}
    rows += Hk  # v goes into the cache as it is
    return {"bytes": T * rows * D * (size + 2) + 16 * T, "flops": T * (Hq + Hk) * (5 * D + 3 * case["rot"])}


def rotary_arguments(case):
    return {"base": 1e6, "interleaved": case["interleaved"], "scaling": case["scaling"], "factor": case["factor"], "original_len": 32768}


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    D, Hq, Hk = case["dim"], case["heads"], case["kv_heads"]
    s = {"case": case}
    if own:
        if "qwen3-27b-5090_b200" not in sys.path:
            sys.path.insert(0, "qwen3-27b-5090_b200")
        from q27b200 import attention, rotary
    if case["op"] != "attn":
        T, dt = case["T"], DTYPES[case["dtype"]]
        far = case["far"]
        # positions of a batch's tokens: runs of consecutive ones, up to the context's end
        start = torch.randint(0, max(1, far - T), (1,), generator=g, device="cuda")
        s["positions"] = start + torch.arange(T, device="cuda") if T > 64 else torch.randint(0, far, (T,), generator=g, device="cuda")
        qkv = normal(T, (Hq + 2 * Hk) * D, dtype=dt, std=1.5)  # the stacked projection's rows
        s["q"] = qkv[:, :Hq * D].unflatten(1, (Hq, D))
        s["k"] = qkv[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
        s["v"] = qkv[:, (Hq + Hk) * D:].unflatten(1, (Hk, D))
        if case["op"] == "norm":
            page, into = case["page"], DTYPES[case["into"]]
            pages = (T + page - 1) // page + 3
            s["k_cache"], s["v_cache"] = normal(pages, Hk, page, D, dtype=into), normal(pages, Hk, page, D, dtype=into)
            s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:T]
            s["q_weight"], s["k_weight"] = (normal(D, dtype=torch.bfloat16, std=0.2) for _ in range(2))
        if own:
            s["rotary"] = rotary.Rotary(case["rot"], **rotary_arguments(case))
            if case["op"] == "norm":
                s["cache"] = attention.KvCache(s["k_cache"], s["v_cache"])
        return s
    dt, page, B = DTYPES[case["dtype"]], case["page"], case["B"]
    new, kv = lengths(case)
    T, width = sum(new), (max(kv) + page - 1) // page
    s["q"] = normal(T, Hq, D, dtype=dt, std=1.5)
    need = [(k + page - 1) // page for k in kv]
    pages = sum(need) + 1
    s["k_cache"] = torch.empty(pages, Hk, page, D, dtype=dt, device="cuda").normal_(generator=g)
    s["v_cache"] = torch.empty(pages, Hk, page, D, dtype=dt, device="cuda").normal_(generator=g)
    free = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    owner = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(need, device="cuda"))
    at = torch.cat([torch.arange(n, device="cuda") for n in need])
    table[owner, at] = free[:len(at)]
    if case["window"]:  # pages that no query can see any more have been given back
        first = torch.tensor([k - n - case["window"] + 1 for n, k in zip(new, kv)], device="cuda")[:, None]
        place = torch.arange(width, device="cuda")[None, :] * page
        table[(place + page <= first) & (place >= case["sinks"])] = -1
    s["table"] = table
    s["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["q_begin"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    s["max_new"], s["max_kv"] = max(new), max(kv)
    if own:
        s["cache"] = attention.KvCache(s["k_cache"], s["v_cache"])
        s["attention"] = attention.Attention(Hq, Hk, D, window=case["window"] or None, sinks=case["sinks"])
    return s


def run(s):
    c = s["case"]
    if own:
        from q27b200 import rotary
        if c["op"] == "rope":
            return rotary.rope(s["rotary"], s["positions"], s["q"], s["k"])
        if c["op"] == "norm":
            q = rotary.qk_norm_rope(s["rotary"], s["positions"], s["q"], s["k"], s["q_weight"], s["k_weight"], eps=EPS, v=s["v"],
                                    cache=s["cache"], slots=s["slots"])
            return q, s["k_cache"], s["v_cache"]
        if c["new"] == 1:
            return s["attention"](s["q"], s["cache"], s["table"], s["kv_lens"], max_kv=s["max_kv"])
        return s["attention"](s["q"], s["cache"], s["table"], s["kv_lens"], s["q_begin"], max_new=s["max_new"], max_kv=s["max_kv"])
    if c["op"] == "rope":
        return plain_rope(c, s["positions"], s["q"].float()).to(s["q"].dtype), plain_rope(c, s["positions"], s["k"].float()).to(s["k"].dtype)
    if c["op"] == "norm":
        page, into = c["page"], s["k_cache"].dtype
        q = plain_rope(c, s["positions"], plain_norm(s["q"].float(), s["q_weight"])).to(into)
        k = plain_rope(c, s["positions"], plain_norm(s["k"].float(), s["k_weight"])).to(into)
        s["k_cache"][s["slots"] // page, :, s["slots"] % page] = k
        s["v_cache"][s["slots"] // page, :, s["slots"] % page] = s["v"].to(into)
        return q, s["k_cache"], s["v_cache"]
    return plain_attention(c, s)


# ---- plain forms ----------------------------------------------------------------------------------------------------


def plain_frequencies(c):
    """Radians per position of each rotated pair, fp64, and the factor on cos and sin. linear: positions divided by the
    factor; ntk: the base raised so that the slowest pair turns that much slower; yarn (Peng et al. 2023): pairs that turn
    less than once over the original context are divided, those that turn more than 32 times are kept, a ramp between,
    and the logits' temperature goes into cos and sin as 0.1 ln(factor) + 1."""
    a, rot = rotary_arguments(c), c["rot"]
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot
    base, f = a["base"], a["factor"]
    if a["scaling"] == "ntk":
        base = base * f ** (rot / (rot - 2))
    w = torch.exp(-i * math.log(base))
    if a["scaling"] == "linear":
        w = w / f
    if a["scaling"] == "yarn":
        turns = a["original_len"] * w / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return w * keep + w / f * (1 - keep), 0.1 * math.log(f) + 1
    return w, 1.0


def plain_rope(c, positions, x):
    w, amplitude = plain_frequencies(c)
    angle = positions.double()[:, None, None] * w
    cos, sin = (torch.cos(angle) * amplitude).float(), (torch.sin(angle) * amplitude).float()
    rot = c["rot"]
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def plain_norm(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + weight.float())


def plain_attention(c, s):
    B, Hq, Hk, D, page = c["B"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    n, L, G = s["max_new"], s["table"].shape[1] * page, Hq // Hk
    q_begin, kv_lens = s["q_begin"].long(), s["kv_lens"].long()
    T = s["q"].shape[0]
    i = torch.arange(n, device="cuda")
    rows = (q_begin[:-1, None] + i).clamp(max=T - 1)
    q = s["q"][rows].float().unflatten(2, (Hk, G)).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * n, D)
    table = s["table"].long().clamp(min=0)
    k = s["k_cache"][table].permute(0, 2, 1, 3, 4).reshape(B, Hk, L, D).float()
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5).view(B, Hk, G, n, L)
    del k
    at = (kv_lens - (q_begin[1:] - q_begin[:-1]))[:, None, None] + i[None, :, None]
    j = torch.arange(L, device="cuda")
    see = j <= at
    if c["window"]:
        see &= (j > at - c["window"]) | (j < c["sinks"])
    see = see[:, None, None]
    p.masked_fill_(~see, -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    v = s["v_cache"][table].permute(0, 2, 1, 3, 4).reshape(B, Hk, L, D).float()
    o = torch.matmul(p.view(B, Hk, G * n, L), v).view(B, Hk, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(q_begin, t, right=True) - 1
    return o[b, t - q_begin[b]].to(s["q"].dtype)


# ---- the definition in 64 bits, written apart -----------------------------------------------------------------------


def exact(case, seed):
    global own
    mine, own = own, False
    s = prepare(case, seed)
    own = mine
    if case["op"] == "attn":
        return exact_attention(case, s)
    q, k = s["q"].double(), s["k"].double()
    if case["op"] == "rope":
        return exact_rotation(case, s["positions"], q), exact_rotation(case, s["positions"], k)
    q, k = (x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True).pow(2) / case["dim"] + EPS).sqrt() * (w.double() + 1)
            for x, w in ((q, s["q_weight"]), (k, s["k_weight"])))
    kc, vc = s["k_cache"].double().transpose(1, 2).flatten(0, 1), s["v_cache"].double().transpose(1, 2).flatten(0, 1)
    kc[s["slots"]] = exact_rotation(case, s["positions"], k)
    vc[s["slots"]] = s["v"].double()
    shape = (-1, case["page"])
    return exact_rotation(case, s["positions"], q), kc.unflatten(0, shape).transpose(1, 2), vc.unflatten(0, shape).transpose(1, 2)


def exact_rotation(case, positions, x):
    rot, f, a = case["rot"], case["factor"], rotary_arguments(case)
    amplitude, speed = 1.0, []
    for pair in range(rot // 2):
        base = a["base"] * f ** (rot / (rot - 2)) if case["scaling"] == "ntk" else a["base"]
        w = base ** (-2 * pair / rot)
        if case["scaling"] == "linear":
            w /= f
        if case["scaling"] == "yarn":
            ramp = min(1.0, max(0.0, (a["original_len"] * w / math.tau - 1) / 31))
            w, amplitude = w * (ramp + (1 - ramp) / f), 1 + math.log(f) / 10
        speed.append(w)
    turn = positions[:, None].double() * torch.tensor(speed, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(turn, amplitude), turn)[:, None]
    head = x[..., :rot]
    z = head.unflatten(-1, (-1, 2)) if case["interleaved"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    z = z if case["interleaved"] else z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), x[..., rot:]], -1)


def exact_attention(case, s):
    new, kv = lengths(case)
    Hk, G, D, page = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (n, length) in enumerate(zip(new, kv)):
        slot = torch.arange(length, device="cuda")
        where = s["table"][b].long()[slot // page].clamp(min=0), slot % page
        position = torch.arange(length - n, length, device="cuda")
        behind = position[:, None] - slot[None, :]
        hidden = behind < 0
        if case["window"]:
            hidden |= (behind >= case["window"]) & (slot >= case["sinks"])
        for h in range(Hk):
            key, value = s["k_cache"][where[0], h, where[1]].double(), s["v_cache"][where[0], h, where[1]].double()
            for g in range(G):
                score = s["q"][begin:begin + n, h * G + g].double() @ key.T / math.sqrt(D)
                score[hidden] = -math.inf
                out[begin:begin + n, h * G + g] = torch.softmax(score, -1) @ value
        begin += n
    return out
