"""What a step over a 4-bit paged K/V cache costs: the page plan, the store and the attention, case by case.

A step runs three operators in a row: `page_plan` turns request lengths into pages, positions and cache slots;
`qk_rope_store_kv4` normalises and rotates queries and keys and writes keys and values as 4-bit codes (read back here
by `kv4_rows` as the values they stand for); `attention_kv4` attends over the pages.  With `own` false, `run` computes
them from elementary torch operations; with `own` true it makes the framework's calls.

The cache format: 16 consecutive channels of a head share one E4M3 scale s, an element is an E2M1 code c
(0, .5, 1, 1.5, 2, 3, 4, 6 with a sign, element 2i in the low nibble of byte i), and the value is c * s * scale with
one fp32 scale for keys and one for values:  s = e4m3(min(448, max|z| / (6 scale))),  c = e2m1(z / (scale * s)), both
rounded to nearest, ties to even; a block whose s is zero has zero codes.
"""
import math
import random

import torch

own = False

EPS = 1e-5                                  # of the per-head norms
QK_SCALE_FACTOR = 5.4730064863875           # multiplies head_dim ** -0.5 in the layer's attention
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 64 requests: a token each, a page only where one starts
        {"name": "plan-decode-64", "op": "plan", "batch": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 1, "ctx_hi": 16384,
         "page": 64, "max_pages": 512, "pad": 0, "lens": 11},
        # a continuous batch of chunks and decode tokens, small pages, the token buffers padded as a captured graph has them
        {"name": "plan-chunks-256", "op": "plan", "batch": 256, "new_lo": 1, "new_hi": 1024, "ctx_lo": 0, "ctx_hi": 8192,
         "page": 16, "max_pages": 1024, "pad": 777, "lens": 12},
        # one-token pages (the reference layer's own page size), every new token takes a page
        {"name": "plan-page1-1000", "op": "plan", "batch": 1000, "new_lo": 1, "new_hi": 500, "ctx_lo": 0, "ctx_hi": 700,
         "page": 1, "max_pages": 1200, "pad": 0, "lens": 13},
        # a verify block of a few tokens through the store: latency
        {"name": "store-decode-8", "op": "store", "tokens": 8, "hq": 32, "hkv": 8, "dim": 128, "theta": 1e6,
         "scale": 1.0, "far": 100000},
        # the native shard's short chunk: head_dim 64, no rotation, a scale that is not a power of two
        {"name": "store-native-753", "op": "store", "tokens": 753, "hq": 16, "hkv": 2, "dim": 64, "theta": 0.0,
         "scale": 0.37, "far": 80000},
        # the whole prefill of the benchmark's layer
        {"name": "store-prefill-16384", "op": "store", "tokens": 16384, "hq": 32, "hkv": 8, "dim": 128, "theta": 1e6,
         "scale": 0.5, "far": 30000},
        # a decode step of one request: too little work for the machine, latency counts
        {"name": "attn-decode-1x4096", "op": "attn", "batch": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 4095,
         "ctx_hi": 4095, "hq": 32, "hkv": 8, "dim": 128, "page": 64, "window": 0, "gate": False, "lens": 21},
        # a decode step of 64 requests of very different lengths: bandwidth and balance
        {"name": "attn-decode-64xragged", "op": "attn", "batch": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 1000,
         "ctx_hi": 32768, "hq": 32, "hkv": 8, "dim": 128, "page": 64, "window": 0, "gate": True, "lens": 22},
        # the native shard decoding over a long context in one-token pages
        {"name": "attn-decode-4x80000", "op": "attn", "batch": 4, "new_lo": 1, "new_hi": 1, "ctx_lo": 80000,
         "ctx_hi": 80000, "hq": 16, "hkv": 2, "dim": 64, "page": 1, "window": 0, "gate": True, "lens": 23},
        # verify blocks of 8 tokens
        {"name": "attn-verify-16x8", "op": "attn", "batch": 16, "new_lo": 8, "new_hi": 8, "ctx_lo": 500, "ctx_hi": 8192,
         "hq": 32, "hkv": 8, "dim": 128, "page": 64, "window": 0, "gate": False, "lens": 24},
        # the native shard's short chunk after a long context, one-token pages, sliding window on
        {"name": "attn-chunk-753-window", "op": "attn", "batch": 4, "new_lo": 500, "new_hi": 753, "ctx_lo": 60000,
         "ctx_hi": 80000, "hq": 16, "hkv": 2, "dim": 64, "page": 1, "window": 8192, "gate": True, "lens": 25},
        # the whole prefill of the benchmark's layer
        {"name": "attn-prefill-4x4096", "op": "attn", "batch": 4, "new_lo": 4096, "new_hi": 4096, "ctx_lo": 0,
         "ctx_hi": 0, "hq": 32, "hkv": 8, "dim": 128, "page": 64, "window": 0, "gate": True, "lens": 26},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(("plan", "store", "store", "attn", "attn", "attn"))
    if kind == "plan":
        batch = _log(rng, 1, 2000)
        new_hi = _log(rng, 1, max(1, 200000 // batch))
        page = rng.choice((1, 16, 32, 64, 100))
        ctx_hi = _log(rng, 1, 16384 if page > 1 else 1000)
        pages = (ctx_hi + new_hi + page - 1) // page
        return {"op": "plan", "batch": batch, "new_lo": min(rng.choice((0, 1)), new_hi), "new_hi": new_hi, "ctx_lo": 0,
                "ctx_hi": ctx_hi, "page": page, "max_pages": pages + rng.randrange(40), "pad": rng.choice((0, 5, 300)),
                "lens": rng.randrange(1 << 20)}
    hq, hkv = rng.choice(((32, 8), (16, 2), (8, 2), (8, 8), (24, 4), (10, 2), (16, 1), (28, 4)))
    dim = rng.choice((64, 128))
    if kind == "store":
        return {"op": "store", "tokens": _log(rng, 1, 16384), "hq": hq, "hkv": hkv, "dim": dim,
                "theta": rng.choice((0.0, 1e4, 1e6)), "scale": rng.choice((1.0, 0.5, 0.37, 0.0123)),
                "far": _log(rng, 1, 500000)}
    case = {"op": "attn", "batch": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 0, "ctx_hi": 0, "hq": hq, "hkv": hkv,
            "dim": dim, "page": rng.choice((1, 16, 64, 48, 128)), "window": rng.choice((0, 0, 0, 1, 333, 4096)),
            "gate": rng.random() < 0.5, "lens": rng.randrange(1 << 20)}
    form = rng.choice(("decode", "decode", "verify", "chunk", "prefill"))
    if form == "decode":
        case["batch"] = _log(rng, 1, 256)
        case["ctx_hi"] = _log(rng, 1, min(100000, 250000 // case["batch"]))
    elif form == "verify":
        case["batch"] = _log(rng, 1, 32)
        case["new_hi"] = _log(rng, 2, 32)
        case["ctx_hi"] = _log(rng, 1, min(50000, 100000 // case["batch"]))
    elif form == "chunk":
        case["batch"] = rng.randrange(1, 5)
        case["new_hi"] = _log(rng, 33, 800)
        case["ctx_hi"] = _log(rng, 1, 40000 // case["batch"])
    else:
        case["batch"] = rng.randrange(1, 5)
        case["new_hi"] = _log(rng, 100, 4096)
        case["new_lo"] = case["new_hi"] // 2
    return case


def _lengths(case):
    """(new tokens, cached tokens) of each request; the first request has the longest of both."""
    rng = random.Random(case["lens"])
    new, ctx = [case["new_hi"]], [case["ctx_hi"]]
    for _ in range(case["batch"] - 1):
        new.append(rng.randint(case["new_lo"], case["new_hi"]))
        ctx.append(min(case["ctx_hi"], max(case["ctx_lo"], _log(rng, case["ctx_lo"] + 1, case["ctx_hi"] + 1) - 1)))
    return new, ctx


def _visible(first, n, window):
    """Visible (query, key) pairs of n queries at positions first .. first + n - 1."""
    total = n * first + n * (n + 1) // 2
    if window:
        for i in range(max(0, window - first), n):          # a query that sees more than the window loses the rest
            total -= first + i + 1 - window
    return total


def work(case):
    if case["op"] == "plan":
        new, ctx = _lengths(case)
        page = case["page"]
        taken = sum(-(-(c + n) // page) - -(-c // page) for n, c in zip(new, ctx))
        return {"bytes": 12 * case["batch"] + 8 * taken + 16 * (sum(new) + case["pad"]), "flops": 0}
    d, hq, hkv = case["dim"], case["hq"], case["hkv"]
    if case["op"] == "store":
        # rows in, queries and codes out, codes in again and the values they stand for out
        per = (hq + 2 * hkv) * d * 2 + hq * d * 2 + 2 * (2 * hkv * d * 9 // 16) + 2 * hkv * d * 2 + 16
        return {"bytes": per * case["tokens"], "flops": 20 * (hq + 2 * hkv) * d * case["tokens"]}
    new, ctx = _lengths(case)
    keys = sum((min(c + n, case["window"] + n - 1) if case["window"] else c + n) for n, c in zip(new, ctx) if n)
    pairs = sum(_visible(c, n, case["window"]) for n, c in zip(new, ctx))
    rows = sum(new) * hq * d
    return {"bytes": keys * hkv * d * 9 // 8 + rows * 2 * (3 if case["gate"] else 2), "flops": 4 * hq * d * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _quantise(z, scale):
    """Codes u8 [..., D / 2] and block scales e4m3 [..., D / 16] of z (fp64), by the definition."""
    shape = z.shape
    z = z.reshape(*shape[:-1], shape[-1] // 16, 16)
    want = (z.abs().amax(-1) / (6.0 * scale)).clamp(max=448.0)
    # E4M3 to nearest even without passing through fp32: multiples of 2^(e - 3), subnormals of 2^-9
    step = torch.exp2(torch.floor(torch.log2(want.clamp(min=2.0 ** -6))).clamp(min=-6.0) - 3.0)
    s = torch.round(want / step) * step
    c = (s * scale).unsqueeze(-1)
    mag = torch.where(c > 0, z.abs() / c, torch.zeros_like(z))
    code = torch.zeros_like(mag, dtype=torch.uint8)
    for border, up_on_tie in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):
        code += (mag >= border) if up_on_tie else (mag > border)
    code = torch.where(z < 0, code + 8, code) * (c > 0)
    code = code.reshape(*shape[:-1], shape[-1] // 2, 2)
    packed = (code[..., 0] | (code[..., 1] << 4)).to(torch.uint8)
    return packed, s.float().to(torch.float8_e4m3fn)


def _dequantise(packed, sf, dtype=torch.float32):
    """code * block scale (without the tensor scale)."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=dtype, device=packed.device)
    lo, hi = grid[(packed & 15).int()], grid[(packed >> 4).int()]
    v = torch.stack([lo, hi], -1).reshape(*packed.shape[:-1], packed.shape[-1] // 16 * 2, 16)
    return (v * sf.to(dtype).unsqueeze(-1)).reshape(*packed.shape[:-1], packed.shape[-1] * 2)


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "plan":
        return _prepare_plan(case, g)
    if case["op"] == "store":
        return _prepare_store(case, g)
    return _prepare_attn(case, g)


def _prepare_plan(case, g):
    new, ctx = _lengths(case)
    batch, page = case["batch"], case["page"]
    have = [-(-c // page) for c in ctx]
    need = [-(-(c + n) // page) for n, c in zip(new, ctx)]
    total = sum(need) + 64
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    used = sum(have)
    table = torch.full((batch, case["max_pages"]), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(case["max_pages"], device="cuda")
    have_t = torch.tensor(have, device="cuda")
    held = col < have_t.unsqueeze(1)
    table[held] = ids[:used]
    head = int(torch.randint(0, 60, (1,), generator=g, device="cuda"))
    free = torch.cat([torch.full((head,), -7, dtype=torch.int32, device="cuda"), ids[used:]])
    return {"op": "plan", "new": torch.tensor(new, dtype=torch.int32, device="cuda"),
            "seq": torch.tensor(ctx, dtype=torch.int32, device="cuda"), "table": table, "free": free,
            "head": torch.tensor([head], dtype=torch.int32, device="cuda"), "page": page,
            "tokens": sum(new) + case["pad"], "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_store(case, g):
    t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
    # one projection row: queries, keys, values and the gate columns, which the store does not read; a few large channels
    spread = torch.exp(0.5 * torch.randn((2 * hq + 2 * hkv) * d, generator=g, device="cuda"))
    qkv = (torch.randn((t, spread.numel()), generator=g, device="cuda") * spread).to(torch.bfloat16)
    rows = t + t // 2 + 64
    loc = torch.randperm(rows, generator=g, device="cuda")[:t]
    inv = None
    if case["theta"]:
        inv = 1.0 / (case["theta"] ** (torch.arange(0, d, 2, dtype=torch.float32, device="cuda") / d))
    scale = torch.tensor(case["scale"], dtype=torch.float32, device="cuda")
    byte = {"dtype": torch.uint8, "device": "cuda"}
    return {"op": "store", "qkv": qkv, "pos": torch.randint(0, case["far"] + 1, (t,), generator=g, device="cuda"),
            "loc": loc, "inv": inv, "scale": scale, "hq": hq, "hkv": hkv, "dim": d,
            "k": torch.zeros((rows, hkv, d // 2), **byte), "v": torch.zeros((rows, hkv, d // 2), **byte),
            "ks": torch.zeros((rows, hkv, d // 16), **byte).view(torch.float8_e4m3fn),
            "vs": torch.zeros((rows, hkv, d // 16), **byte).view(torch.float8_e4m3fn),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_attn(case, g):
    new, ctx = _lengths(case)
    hq, hkv, d, page = case["hq"], case["hkv"], case["dim"], case["page"]
    need = [-(-(c + n) // page) for n, c in zip(new, ctx)]
    total = sum(need)
    table = torch.full((case["batch"], max(need)), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(max(need), device="cuda") < torch.tensor(need, device="cuda").unsqueeze(1)
    table[held] = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    k_scale, v_scale = 0.5, 0.37
    state = {"op": "attn", "new": new, "ctx": ctx, "hq": hq, "hkv": hkv, "dim": d, "page": page,
             "window": case["window"], "scale": d ** -0.5 * QK_SCALE_FACTOR, "table": table,
             "ks": torch.tensor(k_scale, device="cuda"), "vs": torch.tensor(v_scale, device="cuda")}
    rows = total * page
    for name, scale in (("k", k_scale), ("v", v_scale)):
        codes = torch.empty((rows, hkv, d // 2), dtype=torch.uint8, device="cuda")
        sf = torch.empty((rows, hkv, d // 16), dtype=torch.float8_e4m3fn, device="cuda")
        for at in range(0, rows, 1 << 17):
            n = min(1 << 17, rows - at)
            z = torch.randn((n, hkv, d), generator=g, device="cuda").to(torch.bfloat16).double()
            codes[at:at + n], sf[at:at + n] = _quantise(z, scale)
        state[name], state[name + "f"] = codes.view(total, page, hkv, d // 2), sf.view(total, page, hkv, d // 16)
    tokens = sum(new)
    state["q"] = torch.randn((tokens, hq, d), generator=g, device="cuda").to(torch.bfloat16)
    # the layer's projection rows hold the gate after the queries, keys and values
    wide = torch.randn((tokens, (2 * hq + 2 * hkv) * d), generator=g, device="cuda").to(torch.bfloat16)
    state["gate"] = wide[:, (hq + 2 * hkv) * d:] if case["gate"] else None
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    state["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    state["seq"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    state["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "store": _plain_store, "attn": _plain_attn}[state["op"]](state)


def _run_own(s):
    from muse_spark_open_challenge_b200 import ops
    if s["op"] == "plan":
        cu, positions, cache_loc, head = ops.page_plan(s["new"], s["seq"], s["table"], s["free"], s["head"], s["page"],
                                                       s["tokens"], status=s["status"])
        return s["table"], cu, positions, cache_loc, head
    if s["op"] == "store":
        q = ops.qk_rope_store_kv4(s["qkv"], s["pos"], s["loc"], s["inv"], s["scale"], s["scale"], s["k"], s["ks"],
                                  s["v"], s["vs"], s["hq"], s["hkv"], s["dim"], status=s["status"])
        return (q, ops.kv4_rows(s["k"], s["ks"], s["scale"], s["loc"], status=s["status"]),
                ops.kv4_rows(s["v"], s["vs"], s["scale"], s["loc"], status=s["status"]))
    return ops.attention_kv4(s["q"], s["k"], s["kf"], s["v"], s["vf"], s["table"], s["seq"], s["cu"], s["ks"], s["vs"],
                             s["scale"], len(s["new"]), max(s["new"]), s["hq"], s["hkv"], s["dim"], s["page"],
                             s["window"], gate=s["gate"], status=s["status"])


def _plain_plan(s):
    new, seq, page, table = s["new"].long(), s["seq"].long(), s["page"], s["table"]
    have = (seq + page - 1) // page
    take = (seq + new + page - 1) // page - have
    before = torch.cumsum(take, 0) - take
    col = torch.arange(table.shape[1], device=table.device)
    fresh = (col >= have.unsqueeze(1)) & (col < (have + take).unsqueeze(1))
    source = s["head"].long() + before.unsqueeze(1) + (col - have.unsqueeze(1))
    table.copy_(torch.where(fresh, s["free"][source.clamp(0, s["free"].numel() - 1)], table))
    cu = torch.zeros(new.numel() + 1, dtype=torch.int64, device=table.device)
    cu[1:] = torch.cumsum(new, 0)
    t = torch.arange(s["tokens"], device=table.device)
    req = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = req < new.numel()
    req = req.clamp(max=new.numel() - 1)
    positions = torch.where(live, seq[req] + t - cu[req], torch.zeros_like(t))
    slot = table[req, positions // page].long() * page + positions % page
    cache_loc = torch.where(live, slot, torch.full_like(t, -1))
    return table, cu.int(), positions, cache_loc, s["head"] + take.sum().int()


def _plain_store(s):
    hq, hkv, d, t = s["hq"], s["hkv"], s["dim"], s["qkv"].shape[0]
    x = s["qkv"][:, :(hq + 2 * hkv) * d].reshape(t, hq + 2 * hkv, d)
    qk = x[:, :hq + hkv].double()                            # 64 bits: codes turn on values next to a border
    qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    if s["inv"] is not None:
        angle = s["pos"].double().unsqueeze(1) * s["inv"].double()
        cos, sin = torch.cos(angle).unsqueeze(1), torch.sin(angle).unsqueeze(1)
        even, odd = qk[..., 0::2], qk[..., 1::2]
        qk = torch.stack([even * cos - odd * sin, even * sin + odd * cos], -1).reshape(qk.shape)
    out = [qk[:, :hq].float().to(torch.bfloat16)]
    scale = s["scale"].double()
    for z, codes, sf in ((qk[:, hq:], s["k"], s["ks"]), (x[:, hq + hkv:].double(), s["v"], s["vs"])):
        new_codes, new_sf = _quantise(z, scale)
        codes[s["loc"]] = new_codes
        sf.view(torch.uint8)[s["loc"]] = new_sf.view(torch.uint8)
        values = _dequantise(codes[s["loc"]], sf.view(torch.uint8)[s["loc"]].view(torch.float8_e4m3fn)) * s["scale"]
        out.append(values.to(torch.bfloat16))
    return tuple(out)


def _plain_attn(s):
    hq, hkv, d, page, window = s["hq"], s["hkv"], s["dim"], s["page"], s["window"]
    group = hq // hkv
    out = torch.empty((s["q"].shape[0], hq * d), dtype=torch.bfloat16, device="cuda")
    at = 0
    for b, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        if n == 0:
            continue
        low = max(0, c - window + 1) if window else 0
        p = torch.arange(low, c + n, device="cuda")
        row = s["table"][b, p // page].long() * page + p % page
        k = _dequantise(s["k"].view(-1, hkv, d // 2)[row], s["kf"].view(-1, hkv, d // 16)[row]) * s["ks"]
        v = _dequantise(s["v"].view(-1, hkv, d // 2)[row], s["vf"].view(-1, hkv, d // 16)[row]) * s["vs"]
        k, v = k.transpose(0, 1), v.transpose(0, 1)          # [hkv, keys, d]
        step = max(1, (1 << 28) // (hq * p.numel()))
        for i in range(0, n, step):
            m = min(step, n - i)
            q = s["q"][at + i:at + i + m].float().reshape(m, hkv, group, d).transpose(0, 1).reshape(hkv, m * group, d)
            score = torch.matmul(q, k.transpose(1, 2)) * s["scale"]
            score = score.view(hkv, m, group, -1)
            mine = (c + i + torch.arange(m, device="cuda")).view(1, m, 1, 1)
            hidden = p > mine
            if window:
                hidden |= p <= mine - window
            score.masked_fill_(hidden, -math.inf)
            e = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.matmul((e / e.sum(-1, keepdim=True)).view(hkv, m * group, -1), v)
            o = o.view(hkv, m, group, d).transpose(0, 1).reshape(m, hq, d)
            if s["gate"] is not None:
                o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS)
                o = o * torch.sigmoid(s["gate"][at + i:at + i + m].float()).view(m, hq, d)
            out[at + i:at + i + m] = o.reshape(m, hq * d).to(torch.bfloat16)
        at += n
    return out


# ------------------------------------------------------------------------------------------------ the exact values
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] == "store":
        return _exact_store(s)
    return _exact_attn(s)


def _exact_plan(s):
    """Request by request on the host, as the definition reads."""
    new, seq, free, head = s["new"].tolist(), s["seq"].tolist(), s["free"].tolist(), s["head"].item()
    table, page = s["table"].tolist(), s["page"]
    cu, positions, slots = [0], [], []
    for b, (n, c) in enumerate(zip(new, seq)):
        for i in range(-(-c // page), -(-(c + n) // page)):
            table[b][i] = free[head]
            head += 1
        cu.append(cu[-1] + n)
        positions += range(c, c + n)
        slots += [table[b][p // page] * page + p % page for p in range(c, c + n)]
    pad = s["tokens"] - len(positions)
    make = lambda v, t: torch.tensor(v, dtype=t, device="cuda")     # noqa: E731
    return (make(table, torch.int32), make(cu, torch.int32), make(positions + [0] * pad, torch.int64),
            make(slots + [-1] * pad, torch.int64), make([head], torch.int32))


def _exact_store(s):
    """The values of the definition: nearest grid point by distance, blocks one power of two at a time."""
    hq, hkv, d = s["hq"], s["hkv"], s["dim"]
    scale = s["scale"].double()
    scales = torch.arange(0, 127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()   # finite E4M3 >= 0
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")

    def nearest(x, points):
        """Index of the nearest of the ascending points, the even index on a tie."""
        i = torch.searchsorted(points, x.contiguous()).clamp(1, points.numel() - 1)
        down, up = x - points[i - 1], points[i] - x
        lower = (down < up) | ((down == up) & ((i - 1) % 2 == 0))
        return torch.where(lower, i - 1, i)

    parts = []
    for first, count, norm in ((0, hq, True), (hq, hkv, True), (hq + hkv, hkv, False)):
        z = s["qkv"][:, first * d:(first + count) * d].double().view(-1, count, d)
        if norm:
            z = z * (z.square().sum(-1, keepdim=True) / d + EPS).rsqrt()
            if s["inv"] is not None:
                turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                                   torch.outer(s["pos"].double(), s["inv"].double()))
                z = torch.view_as_real(torch.view_as_complex(z.view(-1, count, d // 2, 2)) * turn.unsqueeze(1))
                z = z.reshape(-1, count, d)
        parts.append(z)
    out = [parts[0]]
    for z in parts[1:]:
        blocks = z.reshape(-1, 16)
        values = torch.empty_like(blocks)
        for at in range(0, blocks.shape[0], 1 << 20):
            x = blocks[at:at + (1 << 20)]
            sf = scales[nearest((x.abs().amax(1) / 6.0 / scale).clamp(max=448.0), scales)].unsqueeze(1)
            unit = torch.where(sf > 0, sf * scale, torch.ones_like(sf))
            mag = grid[nearest((x.abs() / unit).clamp(max=6.0), grid)]
            values[at:at + (1 << 20)] = torch.where(sf > 0, torch.copysign(mag, x) * unit, torch.zeros_like(x))
        out.append(values.view(z.shape))
    return tuple(out)


def _exact_attn(s):
    hq, hkv, d = s["hq"], s["hkv"], s["dim"]
    if sum(_visible(c, n, 0) for n, c in zip(s["new"], s["ctx"])) * hq * d > 1 << 41:
        return None
    first = [0]
    for n in s["new"]:
        first.append(first[-1] + n)
    out = torch.zeros((first[-1], hq, d), dtype=torch.float64, device="cuda")
    for b, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        place = torch.arange(c + n, device="cuda")
        page, inside = torch.div(place, s["page"], rounding_mode="floor"), place % s["page"]
        where = s["table"][b].long()[page]
        for h in range(hkv):
            key = _dequantise(s["k"][where, inside, h], s["kf"][where, inside, h], torch.float64) * s["ks"].double()
            val = _dequantise(s["v"][where, inside, h], s["vf"][where, inside, h], torch.float64) * s["vs"].double()
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                for i in range(0, n, 1024):
                    m = min(1024, n - i)
                    rows = slice(first[b] + i, first[b] + i + m)
                    score = s["q"][rows, g].double() @ key.T * s["scale"]
                    at = c + i + torch.arange(m, device="cuda").unsqueeze(1)
                    seen = place <= at
                    if s["window"]:
                        seen &= place > at - s["window"]
                    out[rows, g] = torch.softmax(score.where(seen, -math.inf), -1) @ val
    if s["gate"] is not None:
        out = out * (out.square().mean(-1, keepdim=True) + EPS).rsqrt()
        out = out / (1.0 + torch.exp(-s["gate"].double().reshape(out.shape)))
    return out.reshape(first[-1], hq * d)
