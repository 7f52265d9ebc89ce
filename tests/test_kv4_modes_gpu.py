"""Attention over the 4-bit K/V cache where a call is large enough for its other modes: decode steps whose CTAs take
several KV heads at once, and long contexts behind many query rows, cut into key slices that are joined afterwards.
Every head, channel, query row and cache row has data of its own, and each test asserts from the sizes that its mode is
the one that runs."""
import random

import pytest
import torch

from oracle import kv4_ref as K

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from muse_spark_open_challenge_b200 import ops as _ops
    return _ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check(ops, new, ctx, hq, hkv, d, page, window, gated, seed, sample=None, width=None, hole=None, max_q=None):
    """One call on random codes and scales (values of deviation near 1/2) against the oracle, for the requests in `sample`
    (None: all); `hole` is a (request, page) whose table entry is missing."""
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-(c + n) // page) for n, c in zip(new, ctx)]
    ids = list(range(sum(need) + 3))
    rng.shuffle(ids)
    table = torch.full((len(new), width or max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[:n], dtype=torch.int32)
        del ids[:n]
    if hole:
        table[hole] = -1
    pages = sum(need) + 3
    shape = (pages, page, hkv)
    cache = []
    for _ in range(2):
        cache.append(torch.randint(0, 256, (*shape, d // 2), dtype=torch.uint8, generator=g, device="cuda"))
        cache.append(torch.exp2(-1.75 + 0.3 * torch.randn((*shape, d // 16), generator=g, device="cuda")).to(FP8))
    t, cols = sum(new), hq * d
    q = torch.randn((t, hq + 1, d), generator=g, device="cuda").to(torch.bfloat16)[:, :hq]
    gate = torch.randn((t, cols + 8), generator=g, device="cuda").to(torch.bfloat16)[:, :cols] if gated else None
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    out = torch.full((t + 2, cols), 7.0, dtype=torch.bfloat16, device="cuda")
    half, status = torch.tensor(0.5, device="cuda"), i32([0])
    ops.attention_kv4(q, *cache, table.cuda(), i32(ctx), i32(cu), half, half, 0.3, len(new), max_q or max(new), hq, hkv, d,
                      page, window, gate=gate, out=out[:t], status=status)
    assert int(status) == (-6 if hole else 0) and (out[t:] == 7).all()
    for b in range(len(new)) if sample is None else sample:
        if new[b] == 0:
            continue
        mine = table[b, :need[b]]
        at = torch.where(mine >= 0, mine, 0).cuda().long()
        rows = [K.dequantise(cache[i][at].flatten(0, 1).cpu(), cache[i + 1][at].flatten(0, 1).cpu(), 0.5) for i in (0, 2)]
        here = torch.where(mine >= 0, torch.arange(need[b]), -1)[None]      # the same pages, in order
        part = slice(cu[b], cu[b + 1])
        want, bound = K.attend(q[part].cpu(), *rows, here, [ctx[b]], [0, new[b]], 0.3, page, window,
                               None if gate is None else gate[part].cpu())
        worst = ((out[part].cpu().double() - want).abs() - bound).max()
        assert worst <= 0, f"request {b}: beyond the bound by {float(worst)}"
    return out[:t]


# ------------------------------------------------------------------------------------------------ heads taken together
def takes_heads_together(new, ctx, hq, hkv, d, window):
    """(heads of a CTA, whether the call takes them together): at least eight key tiles a worker."""
    slim = d == 64 or max(new) * (hq // hkv) <= 8
    warps, ctas = (8, 2) if slim else (4, 3)
    heads = 1
    while heads < warps and hkv % (2 * heads) == 0:
        heads *= 2
    tile, tiles = 32 * warps // heads, 0
    for n, c in zip(new, ctx):
        if n:
            first = max(0, c - window + 1) // tile if window else 0
            tiles += max(1, -(-(c + n) // tile) - first) * (hkv // heads)
    return heads, tiles >= 8 * ctas * torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("hq,hkv,d,batch,new_hi,ctx_lo,ctx_hi,page,window,gated,heads", [
    (32, 8, 128, 64, 1, 400, 3000, 16, 0, False, 8),          # a decode step of ragged requests
    (32, 8, 128, 50, 4, 1200, 3000, 64, 0, True, 4),          # two column blocks, four warps, two groups of heads
    (8, 4, 64, 170, 1, 500, 2500, 1, 0, True, 4),             # two warps a head
    (16, 2, 64, 130, 2, 500, 6000, 64, 0, False, 2),          # four warps a head, two column blocks
    (16, 16, 64, 90, 1, 200, 3000, 48, 700, False, 8),        # two groups, a window in front
    (6, 6, 128, 70, 1, 1000, 4000, 24, 0, True, 2),           # three groups
    (24, 8, 128, 120, 2, 100, 3000, 16, 1000, True, 8),       # a window and several tokens
])
def test_attention_decode_with_heads_taken_together(ops, hq, hkv, d, batch, new_hi, ctx_lo, ctx_hi, page, window, gated, heads):
    rng = random.Random(batch + d)
    new = [rng.choice([0, 1, new_hi, new_hi, new_hi, new_hi]) for _ in range(batch)]
    ctx = [rng.randint(ctx_lo, ctx_hi) for _ in range(batch)]
    new[1], ctx[1], ctx[2], new[2] = new_hi, ctx_hi, 0, 1
    assert max(new) * (hq // hkv) <= 16 and takes_heads_together(new, ctx, hq, hkv, d, window) == (heads, True)
    sample = [0, 1, 2, 3, batch - 1] + rng.sample(range(4, batch - 1), 6)
    first = check(ops, new, ctx, hq, hkv, d, page, window, gated, batch, sample)
    assert torch.equal(first, check(ops, new, ctx, hq, hkv, d, page, window, gated, batch, []))      # bit for bit


# ------------------------------------------------------------------------------------------------ key slices
def slices(ops, new, ctx, hq, hkv, width, page, window):
    """Key tiles of each (block, slice) as (first sub-tile's, second sub-tile's)."""
    from muse_spark_open_challenge_b200 import _lib
    splits = _lib.lib().msl_attention_split_plan(len(new), max(new), hq, hkv, width, page, window)
    tq, found = 128 // (hq // hkv), []
    for n, c in zip(new, ctx):
        for q0 in range(0, n, 2 * tq):
            begin = max(0, c + q0 - window + 1) // 128 if window else 0
            tiles = []
            for s in range(2):
                rows = max(0, min(tq, n - q0 - s * tq))
                tiles.append(max(1, (c + q0 + s * tq + rows - 1) // 128 + 1 - begin) if rows else 0)
            chunk = -(-max(tiles) // splits)
            found += [tuple(max(0, min(x, (k + 1) * chunk) - k * chunk) for x in tiles) for k in range(splits)]
    return splits, found


@pytest.mark.parametrize("hq,hkv,d,new,ctx,page,width,window,gated,empty", [
    (8, 2, 64, [150, 40, 257], [6000, 100, 3000], 64, None, 0, False, "both"),
    (8, 2, 128, [300], [4000], 1, None, 0, True, ""),
    (6, 2, 128, [200, 383], [5000, 129], 48, None, 2500, True, ""),
    (2, 2, 64, [256, 256, 30], [2432, 0, 5], 64, 80, 0, True, "both one"),
    (16, 2, 64, [200, 3, 0], [7000, 6000, 50], 1, None, 4096, True, ""),
    (1, 1, 128, [256, 1], [2432, 4000], 128, 40, 0, False, "one"),
    (128, 1, 64, [7, 2], [9000, 300], 16, None, 0, True, "both"),
])
def test_attention_prefill_in_key_slices(ops, hq, hkv, d, new, ctx, page, width, window, gated, empty):
    assert max(new) * (hq // hkv) > 128
    wide = width or max(-(-(c + n) // page) for n, c in zip(new, ctx))
    splits, found = slices(ops, new, ctx, hq, hkv, wide, page, window)
    assert splits > 1
    if "both" in empty:
        assert (0, 0) in found
    if "one" in empty:
        assert any(a == 0 < b for a, b in found)
    first = check(ops, new, ctx, hq, hkv, d, page, window, gated, d + hq, width=width)
    assert torch.equal(first, check(ops, new, ctx, hq, hkv, d, page, window, gated, d + hq, [], width=width))


@pytest.mark.parametrize("gated", [False, True])
def test_attention_key_slices_with_a_missing_page(ops, gated):
    """A hole inside a slice, and a slice that sees nothing but the hole."""
    new, ctx = [200, 140], [3000, 700]
    assert slices(ops, new, ctx, 8, 2, 13, 256, 0)[0] > 1
    check(ops, new, ctx, 8, 2, 64, 256, 0, gated, 5, hole=(0, 1))
    check(ops, new, ctx, 8, 2, 64, 256, 0, gated, 6, hole=(1, 0))
