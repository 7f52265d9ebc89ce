"""The operators of the 4-bit K/V cache on the GPU against their 64-bit restatement (oracle/kv4_ref.py): plan and store
exactly, attention within a bound derived from its roundings; masks that leave little or nothing, pages of any size,
ragged and empty requests, pitches, garbage in hidden places, capture, other streams, and the layer over such a cache."""
import dataclasses
import math
import random

import pytest
import torch

from conftest import to_device
from oracle import kv4_ref as K

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from muse_spark_open_challenge_b200 import ops as _ops
    return _ops


@pytest.fixture
def status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ page plan
def run_plan(ops, new, seq, table, free, head, page, tokens, status):
    dev = i32(table)
    cu, pos, loc, out = ops.page_plan(i32(new), i32(seq), dev, i32(free), i32([head]), page, tokens, status=status)
    return dev.tolist(), cu.tolist(), pos.tolist(), loc.tolist(), int(out)


def plan_case(rng, batch, new_hi, ctx_hi, page, spare=3):
    new = [rng.randint(0, new_hi) for _ in range(batch)]
    seq = [rng.randint(0, ctx_hi) for _ in range(batch)]
    need = [-(-(c + n) // page) for n, c in zip(new, seq)]
    ids = list(range(sum(need) + spare))
    rng.shuffle(ids)
    table = [[-1] * (max(need) + 2) for _ in range(batch)]
    for row, c in zip(table, seq):
        for i in range(-(-c // page)):
            row[i] = ids.pop()
    return new, seq, table, ids


@pytest.mark.parametrize("batch,new_hi,ctx_hi,page,pad", [
    (1, 1, 0, 64, 0), (1, 5000, 77, 16, 9), (3, 0, 50, 16, 4), (64, 1, 3000, 64, 0), (255, 9, 40, 1, 0), (256, 9, 40, 7, 1),
    (257, 70, 300, 100, 300), (1000, 20, 100, 16, 0), (2100, 3, 5, 2, 0)])
def test_page_plan(ops, status, batch, new_hi, ctx_hi, page, pad):
    rng = random.Random(batch * 31 + page)
    new, seq, table, ids = plan_case(rng, batch, new_hi, ctx_hi, page)
    free, head = [-5, -6] + ids, 2
    tokens = sum(new) + pad
    want = K.plan(new, seq, table, free, head, page, tokens)
    assert run_plan(ops, new, seq, table, free, head, page, tokens, status) == want[:5]
    assert int(status) == 0 and not want[5]


@pytest.mark.parametrize("what", ["free list ends", "empty free list", "head past the list", "table row ends",
                                  "too many tokens", "negative lengths", "held page missing"])
def test_page_plan_reports(ops, status, what):
    new, seq, table, free, head, tokens = [5, 40, 3], [3, 16, 30], [[0, -1, -1, -1], [1, -1, -1, -1], [2, 3, -1, -1]], \
        [10, 11, 12, 13, 14], 0, 48
    if what == "free list ends":
        free = free[:2]
    elif what == "empty free list":
        free = []
    elif what == "head past the list":
        head = 6
    elif what == "table row ends":
        new[1], tokens = 90, 98
        free = list(range(10, 30))
    elif what == "too many tokens":
        tokens = 20
    elif what == "negative lengths":
        new[0], seq[2] = -4, -1
    else:
        table[2][1] = -1
    want = K.plan(new, seq, table, free, head, 16, tokens)
    got = run_plan(ops, new, seq, table, free, head, 16, tokens, status)
    assert want[5] and int(status) == -6
    assert got == want[:5]


# ------------------------------------------------------------------------------------------------ store
def empty_cache(rows, hkv, d, fill=0xEE):
    return [torch.full((rows, hkv, w), fill, dtype=torch.uint8, device="cuda") for w in (d // 2, d // 16) * 2]


def run_store(ops, qkv, pos, loc, inv, scales, cache, hq, hkv, d, status=None):
    k, ks, v, vs = cache
    return ops.qk_rope_store_kv4(qkv, pos, loc, inv, scales[0], scales[1], k, ks.view(FP8), v, vs.view(FP8), hq, hkv, d,
                                 status=status)


def check_store(q, cache, loc, qkv, pos, inv, scales, hq, hkv, d):
    zq, zk, zv = K.store(qkv.cpu(), pos.cpu(), None if inv is None else inv.cpu(), hq, hkv, d)
    for z, codes, sf, scale in ((zk, cache[0], cache[1], scales[0]), (zv, cache[2], cache[3], scales[1])):
        want_codes, want_sf = K.quantise(z, scale.cpu())
        assert torch.equal(sf[loc].cpu(), want_sf.view(torch.uint8))
        assert torch.equal(codes[loc].cpu(), want_codes)
    # Half a bf16 step of a value formed in fp32.  The value e cos - o sin may cancel, so its error counts against the
    # pair: in half steps (2^-24 each) at most 12 in the norm's factor (the sum of squares 12 deep, halved by the
    # root, the root itself 2 ulp and more), 1 in e = x r, 1 in the cosine, 2 in product and difference: 16 * 2^-24
    # (|e| + |o|) in all, and |e| + |o| <= sqrt(2) |pair|, which the rotation keeps.
    pair = zq.reshape(*zq.shape[:-1], -1, 2).norm(dim=-1).repeat_interleave(2, -1)
    slack = 16 * 2 ** -24 * 2 ** 0.5 * pair
    assert ((q.cpu().double() - zq).abs() <= (zq.abs() + slack) * 2 ** -8 + slack + 1e-38).all()


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 2, 64), (3, 1, 64), (7, 7, 128), (5, 1, 128), (1, 1, 64)])
@pytest.mark.parametrize("tokens,theta,scale", [(1, 1e6, 1.0), (37, 0.0, 0.37), (300, 1e4, 0.0123)])
def test_store(ops, status, hq, hkv, d, tokens, theta, scale):
    g = torch.Generator(device="cuda").manual_seed(tokens + hq)
    wide = torch.randn((tokens, (2 * hq + 2 * hkv) * d + 8), generator=g, device="cuda")
    qkv = (wide * torch.exp(torch.randn(wide.shape[1], generator=g, device="cuda"))).to(torch.bfloat16)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
    loc = torch.randperm(tokens + 50, generator=g, device="cuda")[:tokens]
    inv = (theta ** (-torch.arange(0, d, 2, device="cuda") / d)).float() if theta else None
    scales = [torch.tensor(scale, device="cuda"), torch.tensor(2.0 * scale, device="cuda")]
    cache = empty_cache(tokens + 50, hkv, d)
    q = run_store(ops, qkv, pos, loc, inv, scales, cache, hq, hkv, d, status)
    assert int(status) == 0
    check_store(q, cache, loc, qkv, pos, inv, scales, hq, hkv, d)
    kept = torch.ones(tokens + 50, dtype=torch.bool, device="cuda")
    kept[loc] = False
    assert all((c[kept] == 0xEE).all() for c in cache)                 # no other row is touched
    for codes, sf, s in ((cache[0], cache[1], scales[0]), (cache[2], cache[3], scales[1])):
        want = K.dequantise(codes[loc].cpu(), sf[loc].cpu(), s.cpu())
        for dtype, half in ((torch.float32, 2 ** -24), (torch.bfloat16, 2 ** -8 + 2 ** -23)):
            got = ops.kv4_rows(codes, sf, s, loc, dtype=dtype, status=status)
            assert got.dtype == dtype and ((got.cpu().double() - want).abs() <= want.abs() * half).all()
    assert int(status) == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [1e-6, 1e-3])
def test_store_blocks_whose_scale_saturates(ops, status, d, scale):
    """A cache scale far too small for the keys: block scales stop at 448, and what is left inside the grid has rotation
    partners thousands of units larger, whose fp32 error reaches over a border."""
    t, hq, hkv = 2000, 8, 8
    g = torch.Generator(device="cuda").manual_seed(d)
    qkv = torch.randn((t, (2 * hq + 2 * hkv) * d), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 1 << 20, (t,), generator=g, device="cuda")
    loc = torch.randperm(t, generator=g, device="cuda")
    inv = (1e4 ** (-torch.arange(0, d, 2, device="cuda") / d)).float()
    keys = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d // 2, 2)      # half of the pairs nearly cancel: e cos - o sin
    angle = pos[:, None].double() * inv.double()
    cancel = keys[..., 0].double() * (angle.cos() / angle.sin())[:, None]
    some = (cancel.abs() < 4) & (torch.rand(cancel.shape, generator=g, device="cuda") < 0.5)
    keys[..., 1] = torch.where(some, cancel.to(torch.bfloat16), keys[..., 1])
    scales = [torch.tensor(scale, device="cuda"), torch.tensor(scale, device="cuda")]
    cache = empty_cache(t, hkv, d)
    q = run_store(ops, qkv, pos, loc, inv, scales, cache, hq, hkv, d, status)
    assert int(status) == 0
    check_store(q, cache, loc, qkv, pos, inv, scales, hq, hkv, d)


def test_store_ties_zeros_and_values_without_a_code(ops, status):
    """V is stored without a norm: exact ties, all-zero blocks, values beyond the format, infinities and NaN."""
    hq = hkv = 1
    d = 64
    v = torch.zeros((6, d))
    v[0, :16] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -0.0])
    v[0, 16:32] = v[0, :16] * 1.125
    v[1] = 1e30
    v[1, 3] = -1e30
    v[2] = torch.linspace(-6.375, 6.375, 64)            # 6.375 / 6 = 1.0625 lies half way between two scales
    v[3] = 2.0 ** -12
    v[3, 20] = 2.0 ** -7
    v[4, 0], v[4, 1], v[4, 2] = float("inf"), float("-inf"), 1.0
    v[5, 16:] = float("nan")
    qkv = torch.cat([torch.ones((6, 2 * d)), v], 1).to(torch.bfloat16).cuda()
    one = torch.ones((), device="cuda")
    cache = empty_cache(6, hkv, d)
    loc = torch.arange(6, device="cuda")
    run_store(ops, qkv, loc, loc, None, [one, one], cache, hq, hkv, d, status)
    want_codes, want_sf = K.quantise(qkv[:4, None, 2 * d:].cpu().double(), 1.0)
    assert torch.equal(cache[2][:4].cpu(), want_codes) and torch.equal(cache[3][:4].cpu(), want_sf.view(torch.uint8))
    odd = ops.kv4_rows(cache[2], cache[3], one, loc[4:], dtype=torch.float32)[:, 0].cpu()
    assert odd[0, :3].tolist() == [2688.0, -2688.0, 0.0] and (odd[0, 3:] == 0).all()
    assert (odd[1, :16] == 0).all() and (odd[1, 16:].abs() == 2688.0).all() and int(status) == 0


def test_store_skips_padding_and_reports_rows_beyond_the_cache(ops, status):
    hq, hkv, d = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn((5, 8 * d), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.arange(5, device="cuda")
    one = torch.ones((), device="cuda")
    cache = empty_cache(8, hkv, d)
    run_store(ops, qkv, pos, torch.tensor([-1, 3, -7, 0, -1], device="cuda"), None, [one, one], cache, hq, hkv, d, status)
    assert int(status) == 0
    assert [(c == 0xEE).all(-1).all(-1).tolist() for c in cache] == [[False, True, True, False] + [True] * 4] * 4
    run_store(ops, qkv, pos, torch.tensor([-1, 8, 1, 9, 7], device="cuda"), None, [one, one], cache, hq, hkv, d, status)
    assert int(status) == -6 and (cache[0][2] == 0xEE).all() and not (cache[0][7] == 0xEE).all()
    status.zero_()
    got = ops.kv4_rows(cache[0], cache[1], one, torch.tensor([-1, 8, 7], device="cuda"), status=status)
    assert int(status) == -6 and (got[:2] == 0).all() and (got[2] != 0).any()
    assert ops.kv4_rows(cache[0], cache[1], one, pos[:0]).shape == (0, hkv, d)


# ------------------------------------------------------------------------------------------------ attention
def paged(rng, new, ctx, page, hkv, d, seed, spare=2):
    """Random cache rows behind a scattered page table, the unused rows and tails full of NaN scales."""
    need = [-(-(c + n) // page) for n, c in zip(new, ctx)]
    total = sum(need) + spare
    ids = list(range(total))
    rng.shuffle(ids)
    width = max(max(need), 1) + 1
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    g = torch.Generator().manual_seed(seed)
    cache = [torch.full((total * page, hkv, w), 0xFF, dtype=torch.uint8) for w in (d // 2, d // 16) * 2]
    for b, (n, c) in enumerate(zip(new, ctx)):
        for i in range(need[b]):
            table[b, i] = ids.pop()
        p = torch.arange(c + n)
        rows = table[b].long()[p // page] * page + p % page
        for which in (0, 2):
            z = torch.randn((c + n, hkv, d), generator=g).double()
            cache[which][rows], sf = K.quantise(z, 0.5)
            cache[which + 1][rows] = sf.view(torch.uint8)
    return table, cache


def run_attention(ops, q, cache, table, ctx, cu, max_q, hq, hkv, d, page, window, scale, gate=None, out=None, status=None,
                  scales=None):
    k, ks, v, vs = [c.cuda() for c in cache]
    half = torch.tensor(0.5, device="cuda")
    return ops.attention_kv4(q, k, ks.view(FP8), v, vs.view(FP8), table.cuda(), i32(ctx), i32(cu), *(scales or (half, half)),
                             scale, len(ctx), max_q, hq, hkv, d, page, window, gate=gate, out=out, status=status)


def check_attention(ops, status, new, ctx, hq, hkv, d, page, window, gated, seed=0, scale=0.3, spoil=None):
    rng = random.Random(seed)
    table, cache = paged(rng, new, ctx, page, hkv, d, seed)
    if spoil is not None:
        spoil(table, cache)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = sum(new)
    wide = torch.randn((t, hq + 1, d), generator=g, device="cuda").to(torch.bfloat16)
    q = wide[:, :hq]                                                # a pitch of one head more
    gate = torch.randn((t, hq * d + 8), generator=g, device="cuda").to(torch.bfloat16)[:, :hq * d] if gated else None
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    out = torch.full((t + 3, hq * d + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    run_attention(ops, q, cache, table, ctx, cu, max(max(new), 1), hq, hkv, d, page, window, scale, gate,
                  out[:t, :hq * d], status)
    assert (out[t:] == 7).all() and (out[:, hq * d:] == 7).all()
    rows = [K.dequantise(cache[i], cache[i + 1], 0.5) for i in (0, 2)]
    want, bound = K.attend(q.cpu(), *rows, table, ctx, cu, scale, page, window, None if gate is None else gate.cpu())
    got = out[:t, :hq * d].cpu().double()
    worst = ((got - want).abs() - bound).max() if t else torch.zeros(())
    assert worst <= 0, f"beyond the bound by {float(worst)}"
    return got


HEADS = [(32, 8, 128), (16, 2, 64), (8, 8, 64), (7, 1, 128), (10, 2, 64), (12, 4, 128), (16, 1, 128), (40, 1, 64)]


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("page,window,gated", [(64, 0, False), (1, 0, True), (24, 100, True)])
def test_attention_decode(ops, status, hq, hkv, d, page, window, gated):
    check_attention(ops, status, [1] * 5, [0, 15, 200, 1, 700], hq, hkv, d, page, window, gated, seed=hq + page)
    assert int(status) == 0


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("new,ctx,page,window", [
    ([8, 3, 0, 5], [130, 0, 9, 255], 16, 0), ([1, 20, 2], [400, 0, 31], 64, 33), ([33], [0], 100, 1), ([70, 64], [90, 0], 1, 0)])
def test_attention_short_blocks(ops, status, hq, hkv, d, new, ctx, page, window):
    check_attention(ops, status, new, ctx, hq, hkv, d, page, window, True, seed=hq + page)
    assert int(status) == 0


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 2, 64), (5, 1, 128), (6, 2, 64)])
@pytest.mark.parametrize("new,ctx,page,window,gated", [
    ([300], [0], 64, 0, True), ([257, 1, 129], [40, 300, 0], 64, 0, False), ([200, 383], [500, 129], 48, 130, True),
    ([140, 0, 0], [1000, 4, 0], 1, 0, True), ([513], [255], 128, 1, False)])
def test_attention_prefill(ops, status, hq, hkv, d, new, ctx, page, window, gated):
    check_attention(ops, status, new, ctx, hq, hkv, d, page, window, gated, seed=hq + page)
    assert int(status) == 0


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 9], [150, 3, 200]])
def test_attention_hides_keys_without_a_page_and_zeroes_rows_that_see_nothing(ops, status, new):
    ctx = [100, 0, 64]

    def spoil(table, cache):
        table[0, 2] = -3                      # a hole inside a long context
        table[1, :] = -1                      # request 1 has no page at all
        table[2, 1] = 1 << 20                 # beyond the cache
    got = check_attention(ops, status, new, ctx, 8, 2, 64, 16, 0, False, spoil=spoil)
    assert int(status) == -6
    first = sum(new[:1])
    assert (got[first:first + new[1]] == 0).all() and (got[:first] != 0).any()


@pytest.mark.parametrize("new,longest", [([2, 1], 2), ([150, 20], 150)])
def test_attention_page_table_too_short(ops, status, new, longest):
    """Keys past max_pages pages are hidden and reported; nothing is read beyond the table's rows."""
    table, cache = paged(random.Random(0), new, [50, 40], 16, 2, 64, 0)
    short = table[:, :2].contiguous()
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn((sum(new), 4, 64), generator=g, device="cuda").to(torch.bfloat16)
    cu = [0, new[0], sum(new)]
    got = run_attention(ops, q, cache, short, [50, 40], cu, longest, 4, 2, 64, 16, 0, 0.3, status=status)
    rows = [K.dequantise(cache[i], cache[i + 1], 0.5) for i in (0, 2)]
    want, bound = K.attend(q.cpu(), *rows, short, [50, 40], cu, 0.3, 16, 0)
    assert ((got.cpu().double() - want).abs() <= bound).all() and int(status) == -6


@pytest.mark.parametrize("new", [[3, 1], [130, 60]])
def test_attention_nan_scales_of_a_later_key_do_not_reach_earlier_rows(ops, status, new):
    """The scale bytes of the block's last key are NaN codes: rows before it must not notice."""
    ctx = [70, 10]
    table, cache = paged(random.Random(2), new, ctx, 16, 2, 128, 2)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn((sum(new), 8, 128), generator=g, device="cuda").to(torch.bfloat16)
    args = (table, ctx, [0, new[0], sum(new)], max(new), 8, 2, 128, 16, 0, 0.2)
    clean = run_attention(ops, q, cache, *args, status=status)
    at = ctx[0] + new[0] - 1
    row = int(table[0, at // 16]) * 16 + at % 16
    for i in (1, 3):
        cache[i][row] = 0x7F
    got = run_attention(ops, q, cache, *args, status=status)
    assert torch.equal(got[:new[0] - 1], clean[:new[0] - 1]) and torch.equal(got[new[0]:], clean[new[0]:])
    assert torch.isfinite(got.float()).all() and not torch.equal(got, clean) and int(status) == 0


@pytest.mark.parametrize("new", [[1, 1], [150, 150]])
@pytest.mark.parametrize("factor", [1e-30, 1e-6, 1.0, 1e4, 1e30])
def test_attention_query_magnitudes(ops, status, new, factor):
    """bf16 queries of any size: the softmax scale makes up for it, so the results agree."""
    ctx, hq, hkv, d = [200, 90], 4, 2, 64
    table, cache = paged(random.Random(3), new, ctx, 16, hkv, d, 3)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = (torch.randn((sum(new), hq, d), generator=g, device="cuda") * factor).to(torch.bfloat16)
    cu = [0, new[0], sum(new)]
    got = run_attention(ops, q, cache, table, ctx, cu, max(new), hq, hkv, d, 16, 0, 0.3 / factor, status=status)
    rows = [K.dequantise(cache[i], cache[i + 1], 0.5) for i in (0, 2)]
    want, bound = K.attend(q.cpu(), *rows, table, ctx, cu, 0.3 / factor, 16, 0)
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("new", [[1, 1], [150, 150]])
def test_attention_nan_query_stays_in_its_row(ops, new):
    ctx, hq, hkv, d = [200, 90], 4, 2, 64
    table, cache = paged(random.Random(4), new, ctx, 16, hkv, d, 4)
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn((sum(new), hq, d), generator=g, device="cuda").to(torch.bfloat16)
    args = (table, ctx, [0, new[0], sum(new)], max(new), hq, hkv, d, 16, 0, 0.3)
    clean = run_attention(ops, q, cache, *args).view(-1, hq, d)
    q[0, 1, 5] = float("nan")
    got = run_attention(ops, q, cache, *args).view(-1, hq, d)
    assert torch.isnan(got[0, 1].float()).all()
    keep = torch.ones(sum(new), hq, dtype=torch.bool)
    keep[0, 1] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("batch,ctx_hi", [(1, 30000), (70, 900), (300, 40), (2, 5)])
def test_attention_many_workers_and_ragged_batches(ops, status, batch, ctx_hi):
    """Work items cut over many workers, and many items within one; both against the oracle, and bit-repeatable."""
    rng = random.Random(batch)
    ctx = [rng.randint(0, ctx_hi) for _ in range(batch)]
    ctx[0] = ctx_hi
    first = check_attention(ops, status, [1] * batch, ctx, 8, 2, 64, 16, 0, False, seed=batch)
    again = check_attention(ops, status, [1] * batch, ctx, 8, 2, 64, 16, 0, False, seed=batch)
    assert torch.equal(first, again) and int(status) == 0


@pytest.mark.parametrize("batch,hq,hkv,d,new_hi,ctx_hi,window", [
    (90, 16, 8, 64, 12, 300, 0),      # several whole (request, KV head) pairs in one block's range of key tiles
    (400, 8, 2, 64, 9, 40, 0),        # one key tile each
    (3, 16, 2, 128, 16, 9000, 0),     # one pair over many blocks
    (70, 16, 4, 128, 32, 1500, 200),  # ranges that end inside pairs, a window in front
    (4, 128, 1, 64, 1, 600, 0),       # one token fills the block of rows
    (3, 100, 1, 128, 1, 700, 64),
])
def test_attention_blocks_of_rows_share_the_key_tiles(ops, status, batch, hq, hkv, d, new_hi, ctx_hi, window):
    rng = random.Random(batch)
    new = [rng.choice([0, 1, rng.randint(1, new_hi)]) for _ in range(batch)]
    new[1] = new_hi                   # 17 to 128 rows a KV head
    ctx = [rng.randint(0, ctx_hi) for _ in range(batch)]
    check_attention(ops, status, new, ctx, hq, hkv, d, 16, window, batch % 20 == 0, seed=batch)
    assert int(status) == 0


@pytest.mark.parametrize("batch,new", [(300, 1), (300, 4), (3, 24), (2, 150)])
def test_attention_small_weights_behind_dominating_keys(ops, status, batch, new):
    """Eight keys take nearly all the weight and have no value; each of 2000 others weighs 1.37 * 2^-22 of one of them.
    P carries 2^6, so such a weight is 1.37 * 2^-16 and rounded by at most 2^-25, below 2^-9 of it; fp32 sums and
    exponentials are good to 2^-13, and bf16 adds 2^-8."""
    hq, hkv, d, page, ctx = 8, 2, 64, 16, 2000
    pages = -(-(ctx + new) // page)
    k = torch.zeros((pages * page, hkv, d // 2), dtype=torch.uint8)
    v = torch.full_like(k, 0x22)                                    # ones
    sf = torch.full((pages * page, hkv, d // 16), 0x38, dtype=torch.uint8)
    k[0:256:32] = 0x22
    v[0:256:32] = 0
    q = torch.ones((batch * new, hq, d), dtype=torch.bfloat16, device="cuda")
    one = torch.tensor(1.0, device="cuda")
    table = torch.arange(pages, dtype=torch.int32).repeat(batch, 1)
    scale = math.log(2 ** 22 / 1.37) / d
    got = run_attention(ops, q, (k, sf, v, sf), table, [ctx] * batch, [new * b for b in range(batch + 1)], new, hq, hkv, d,
                        page, 0, scale, status=status, scales=(one, one))
    assert int(status) == 0
    others = (ctx + 1 - 8 + torch.arange(new).double()) * 1.37 * 2 ** -22
    want = (others / (8 + others)).repeat(batch)[:, None]
    assert ((got.cpu().double() - want).abs() <= want * (2 ** -8 + 2 ** -9 + 2 ** -12)).all()


@pytest.mark.parametrize("longest", [1, 12, 90])
def test_attention_captured_once_serves_other_lengths_beside_another_stream(ops, longest):
    """A captured call reads its lengths on the device, and calls on two streams at once do not share a workspace."""
    hq, hkv, d, page, batch = 8, 2, 64, 16, 6
    rng = random.Random(longest)
    steps = [([rng.randint(0, longest) for _ in range(batch)], [rng.randint(0, 1500) for _ in range(batch)]) for _ in range(3)]
    table, cache = paged(rng, [longest] * batch, [1500] * batch, page, hkv, d, longest)
    k, ks, v, vs = [c.cuda() for c in cache]
    half = torch.tensor(0.5, device="cuda")
    t = longest * batch
    q = torch.randn((t, hq, d), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    table_gpu, ctx, cu = table.cuda(), i32([0] * batch), i32([0] * (batch + 1))

    def call(ctx, cu, out):
        ops.attention_kv4(q, k, ks.view(FP8), v, vs.view(FP8), table_gpu, ctx, cu, half, half, 0.3, batch, longest, hq, hkv,
                          d, page, 0, out=out)
    outs = [torch.full((t, hq * d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    call(ctx, cu, outs[0])                                          # (with nothing to do)
    torch.cuda.synchronize()
    assert (outs[0] == 7).all()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        call(ctx, cu, outs[0])
    rows = [K.dequantise(cache[i], cache[i + 1], 0.5) for i in (0, 2)]
    lengths = []
    for new, past in steps:
        sums = [sum(new[:b]) for b in range(batch + 1)]
        lengths.append((i32(past), i32(sums), past, sums))
    torch.cuda.synchronize()
    for i, (past_gpu, sums_gpu, _, _) in enumerate(lengths):
        ctx.copy_(past_gpu), cu.copy_(sums_gpu)
        outs[0].fill_(7.0)
        other = lengths[i - 1]
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(4):
            graph.replay()
            with torch.cuda.stream(side):
                call(other[0], other[1], outs[1])
        torch.cuda.synchronize()
        for out, (_, _, past, sums) in ((outs[0], lengths[i]), (outs[1], other)):
            n = sums[-1]                                            # rows behind it stay as they were
            want, bound = K.attend(q[:n].cpu(), *rows, table, past, sums, 0.3, page, 0)
            assert ((out[:n].cpu().double() - want).abs() <= bound).all()
        assert (outs[0][lengths[i][3][-1]:] == 7).all()


@pytest.mark.parametrize("new", [1, 140])
def test_attention_offsets_beyond_32_bits(ops, status, new):
    """Cache rows whose byte offset passes 2^32 (keys and values share one buffer to save memory)."""
    hq, hkv, d, page = 8, 8, 128, 64
    rows = (1 << 23) + 4 * page
    codes = torch.zeros((rows, hkv, d // 2), dtype=torch.uint8, device="cuda")
    sf = torch.zeros((rows, hkv, d // 16), dtype=torch.uint8, device="cuda")
    g = torch.Generator().manual_seed(5)
    ctx = 180 - new
    pages = [rows // page - 1, 3, rows // page - 2]
    z = torch.randn((180, hkv, d), generator=g).double()
    c, s = K.quantise(z, 0.5)
    p = torch.arange(180)
    at = torch.tensor(pages)[p // page] * page + p % page
    codes[at.cuda()], sf[at.cuda()] = c.cuda(), s.view(torch.uint8).cuda()
    q = torch.randn((new, hq, d), generator=g).to(torch.bfloat16).cuda()
    half = torch.tensor(0.5, device="cuda")
    got = ops.attention_kv4(q, codes, sf.view(FP8), codes, sf.view(FP8), i32([pages]), i32([ctx]), i32([0, new]), half, half,
                            0.2, 1, new, hq, hkv, d, page, 0, status=status)
    small = K.dequantise(c, s, 0.5)                          # the same 180 rows behind an identity table
    want, bound = K.attend(q.cpu(), small, small, torch.arange(3, dtype=torch.int32)[None], [ctx], [0, new], 0.2, page, 0)
    assert ((got.cpu().double() - want).abs() <= bound).all() and int(status) == 0
    back = ops.kv4_rows(codes, sf, half, at.cuda(), dtype=torch.float32, status=status)
    assert torch.equal(back.cpu().double(), small)


# ------------------------------------------------------------------------------------------------ together
def step_tensors(seed=7, hq=8, hkv=2, d=64, page=16):
    new, ctx = [1, 9, 0, 40], [70, 0, 5, 33]
    rng = random.Random(seed)
    need = [-(-(c + n) // page) for n, c in zip(new, ctx)]
    table, cache = paged(rng, [0] * 4, ctx, page, hkv, d, seed, spare=sum(need))
    width = max(need) + 1
    table = torch.cat([table, torch.full((4, max(0, width - table.shape[1])), -1, dtype=torch.int32)], 1)
    used = set(table[table >= 0].tolist())
    free = [i for i in range(cache[0].shape[0] // page) if i not in used]
    rng.shuffle(free)
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn((54, (2 * hq + 2 * hkv) * d), generator=g, device="cuda").to(torch.bfloat16)
    return new, ctx, table, cache, free, qkv


def test_plan_store_attend_as_a_step(ops, status):
    """The three operators in a row, on a padded token buffer, eagerly, then captured once and replayed with other
    lengths of the same batch: each replay equals the eager step and the oracle."""
    hq, hkv, d, page = 8, 2, 64, 16
    new, ctx, table, cache, free, qkv = step_tensors()
    inv = (1e4 ** (-torch.arange(0, d, 2, device="cuda") / d)).float()
    half = torch.tensor(0.5, device="cuda")
    dev = {"new": i32(new), "ctx": i32(ctx), "table": table.cuda(), "free": i32(free), "head": i32([0]),
           "cache": [c.cuda() for c in cache]}
    k, ks, v, vs = dev["cache"]
    kv = (k, ks.view(FP8), v, vs.view(FP8))

    def step():
        cu, pos, loc, head = ops.page_plan(dev["new"], dev["ctx"], dev["table"], dev["free"], dev["head"], page, 54,
                                           status=status)
        q = ops.qk_rope_store_kv4(qkv, pos, loc, inv, half, half, *kv, hq, hkv, d, status=status)
        out = torch.zeros((54, hq * d), dtype=torch.bfloat16, device="cuda")
        ops.attention_kv4(q, *kv, dev["table"], dev["ctx"], cu, half, half, 0.3, 4, 54, hq, hkv, d, page, 0,
                          gate=qkv[:, (hq + 2 * hkv) * d:], out=out, status=status)
        return q, cu, loc, head, out

    def check(new, ctx, got):
        q, cu, loc, head, out = [x.clone() for x in got]
        want = K.plan(new, ctx, table.tolist(), free, 0, page, 54)
        assert cu.tolist() == want[1] and loc.tolist() == want[3] and int(head) == want[4]
        assert dev["table"].tolist() == want[0]
        live = sum(new)
        _, zk, zv = K.store(qkv.cpu(), torch.tensor(want[2]), inv.cpu(), hq, hkv, d)
        rows = [c.clone() for c in cache]
        at = torch.tensor(want[3][:live])
        rows[0][at], s = K.quantise(zk[:live], 0.5)
        rows[1][at] = s.view(torch.uint8)
        rows[2][at], s = K.quantise(zv[:live], 0.5)
        rows[3][at] = s.view(torch.uint8)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev["cache"], rows))
        values = [K.dequantise(rows[i], rows[i + 1], 0.5) for i in (0, 2)]
        o, bound = K.attend(q.cpu()[:live], *values, torch.tensor(want[0]), ctx, want[1], 0.3, page, 0,
                            qkv[:live, (hq + 2 * hkv) * d:].cpu())
        assert ((out[:live].cpu().double() - o).abs() <= bound).all() and (out[live:] == 0).all()
        assert int(status) == 0

    def reset():
        dev["table"].copy_(table)
        for a, b in zip(dev["cache"], cache):
            a.copy_(b)

    check(new, ctx, step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        reset()
        check(new, ctx, step())                               # on another stream
    torch.cuda.current_stream().wait_stream(side)
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for other in ([1, 9, 0, 40], [3, 2, 30, 1], [0, 0, 1, 0]):
        reset()
        dev["new"].copy_(i32(other))
        graph.replay()
        torch.cuda.synchronize()
        check(other, ctx, captured)


def test_wrappers_refuse(ops):
    from muse_spark_open_challenge_b200._lib import MslError
    hq, hkv, d = 8, 2, 64
    one = torch.ones((), device="cuda")
    c = empty_cache(32, hkv, d)
    ks, vs = c[1].view(FP8), c[3].view(FP8)
    q = torch.zeros((2, hq, d), dtype=torch.bfloat16, device="cuda")
    good = dict(q=q, k_cache=c[0], k_sf=ks, v_cache=c[2], v_sf=vs, page_table=i32([[0, 1]]), seq_lens=i32([0]),
                cu_seqlens_q=i32([0, 2]), k_scale=one, v_scale=one, softmax_scale=0.1, batch=1, max_q_len=2, hq=hq, hkv=hkv,
                head_dim=d, page_size=16, window=0)
    torch.cuda.synchronize()
    for change in (dict(q=q.float()), dict(q=q[:, :4]), dict(q=q.transpose(0, 1)), dict(k_sf=ks[:, :, :2]), dict(k_sf=ks.cpu()),
                   dict(v_cache=c[2][:16], v_sf=vs[:16]), dict(page_table=i32([0, 1])), dict(page_table=i32([[0, 1], [2, 3]])[:, :1]),
                   dict(seq_lens=torch.zeros(1, device="cuda").long()), dict(cu_seqlens_q=i32([0, 1, 2])),
                   dict(k_scale=torch.ones(2, device="cuda")), dict(k_scale=one.double()), dict(hq=7), dict(head_dim=32),
                   dict(page_size=0), dict(window=-1), dict(batch=0), dict(max_q_len=0),
                   dict(gate=torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda")),
                   dict(out=torch.zeros((2, hq * d), device="cuda")), dict(status=torch.zeros(1, device="cuda"))):
        with pytest.raises(MslError):
            ops.attention_kv4(**{**good, **change})
    with pytest.raises(MslError):
        ops.kv4_rows(c[0], ks, one, i32([0]))
    with pytest.raises(MslError):
        ops.kv4_rows(c[0], ks, one, torch.zeros(1, device="cuda").long(), dtype=torch.float16)
    qkv = torch.zeros((2, 12 * d), dtype=torch.bfloat16, device="cuda")
    at = torch.zeros(2, dtype=torch.int64, device="cuda")
    store = dict(qkv=qkv, positions=at, cache_loc=at - 1, inv_freq=None, k_scale=one, v_scale=one, k_cache=c[0], k_sf=ks,
                 v_cache=c[2], v_sf=vs, hq=hq, hkv=hkv, head_dim=d)
    for change in (dict(qkv=qkv[:, :-1]), dict(positions=at.int()), dict(cache_loc=at[:1]), dict(inv_freq=torch.ones(8, device="cuda")),
                   dict(k_cache=c[0].transpose(0, 1)), dict(head_dim=128), dict(qkv=qkv.t())):
        with pytest.raises(MslError):
            ops.qk_rope_store_kv4(**{**store, **change})
    lens = i32([1, 1])
    plan = dict(new_lens=lens, seq_lens=lens, page_table=i32([[0, 1], [2, 3]]), free_pages=i32([4, 5]), free_head=i32([0]),
                page_size=16, tokens=2)
    for change in (dict(seq_lens=i32([1])), dict(page_table=i32([[0, 1]])), dict(free_head=i32([0, 0])), dict(page_size=0),
                   dict(tokens=-1), dict(new_lens=lens.long())):
        with pytest.raises((MslError, RuntimeError)):
            ops.page_plan(**{**plan, **change})


# ------------------------------------------------------------------------------------------------ the layer
@pytest.mark.parametrize("lens,ctxs,page", [([1, 1, 1], [40, 0, 130], 16), ([90, 150], [64, 5], 64)])
def test_layer_over_a_4_bit_cache(ops, lens, ctxs, page):
    """`layer.kernel_fn` with the codes and block scales in `data`: the attention stage equals the three operators
    called in a row on the same projection, new rows land in the cache, and the layer runs on and replays."""
    from muse_spark_open_challenge_b200 import layer, synth
    shape = dataclasses.replace(synth.MID, hidden=512, hq=8, hkv=2, n_experts=16, local_experts=16, moe_width=512, inter=256,
                                shared_inter=256)
    st = layer.prepare(to_device(synth.make_weights(shape, seed=1), "cuda"))
    data = synth.make_input(shape, lens, ctxs, seed=2, page=page, kv_scale=0.5)
    data.update(synth.kv4_cache(shape, data["k_cache"].shape[0], page, seed=3))
    data = to_device(data, "cuda")
    before = {k: data[k].view(torch.uint8).clone() for k in ("k_cache", "k_cache_sf", "v_cache", "v_cache_sf")}
    stage = layer.attention_stage(data, st)
    qkv = ops.gemm(data["attn_input"], st["qkv_gate"], status=st["status"])
    inv = layer._inv_freq(st, shape.rope_theta, shape.head_dim)
    names = ("k_cache", "k_cache_sf", "v_cache", "v_cache_sf")
    flat = [before[n].view(-1, *before[n].shape[2:]).clone() for n in names]
    q = run_store(ops, qkv, data["positions"], data["cache_loc"], inv, (data["k_scale"], data["v_scale"]), flat, shape.hq,
                  shape.hkv, shape.head_dim)
    for n, f in zip(names, flat):
        assert torch.equal(data[n].view(torch.uint8).view(f.shape), f) and not torch.equal(f, before[n].view(f.shape))
    cfg = data["config"]
    rows = [K.dequantise(flat[i].cpu(), flat[i + 1].cpu(), 0.5) for i in (0, 2)]
    want, bound = K.attend(q.cpu(), *rows, data["page_table"].cpu(), ctxs, data["cu_seqlens_q"].tolist(),
                           cfg["sm_scale"] * cfg["qk_scale_factor"], page, 0,
                           qkv[:, (shape.hq + 2 * shape.hkv) * shape.head_dim:].cpu())
    assert ((stage.cpu().double() - want).abs() <= bound).all()
    hidden, stream, ids = [x.clone() for x in layer.kernel_fn(data, st)]
    layer.check_status(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.kernel_fn(data, st)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], hidden) and torch.equal(out[1], stream) and torch.equal(out[2], ids)
    layer.check_status(st)
    from muse_spark_open_challenge_b200._lib import MslError
    with pytest.raises(MslError):
        layer.attention_stage(data, st, after_store=lambda: None)


def test_stack_over_4_bit_caches_chains_its_layers(ops):
    from muse_spark_open_challenge_b200 import layer, stack, synth
    shape = dataclasses.replace(synth.MID, hidden=512, hq=8, hkv=2, n_experts=16, local_experts=16, moe_width=512, inter=256,
                                shared_inter=256)
    states = stack.prepare_stack([to_device(synth.make_weights(shape, seed=i), "cuda") for i in range(2)])
    step = to_device(synth.make_input(shape, [5, 1], [20, 33], seed=2, page=16, kv_scale=0.5), "cuda")
    pages = step["k_cache"].shape[0]
    caches = [to_device(synth.kv4_cache(shape, pages, 16, seed=i), "cuda") for i in range(2)]
    for name in ("k_cache", "v_cache"):
        step.pop(name)
        step[name + "s"] = [c[name].clone() for c in caches]
        step[name + "_sfs"] = [c[name + "_sf"].clone() for c in caches]
    hidden, stream, ids = stack.forward(step, states)
    carry = (None, None)
    for i, st in enumerate(states):
        data = {k: v for k, v in step.items() if not k.endswith(("_caches", "_sfs"))}
        data.update(caches[i])
        if i:
            data["attn_input"], data["stream"] = carry
        h, s, e = layer.kernel_fn(data, st)
        carry = (h, s)
        layer.check_status(st)
        assert torch.equal(e, ids[i])
    assert torch.equal(h, hidden) and torch.equal(s, stream)


# ------------------------------------------------------------------------------------------------ odd numbers
@pytest.mark.parametrize("new", [[1, 1], [4, 2], [20, 9], [150, 150]])
def test_attention_zero_query_rows_under_small_scales(ops, status, new):
    """A row of zeros weighs all visible keys alike, also where softmax_scale * k_scale over the power of two that the
    row was scaled by is below the smallest fp32 number."""
    ctx, hq, hkv, d, page = [200, 90], 8, 2, 64, 16
    table, cache = paged(random.Random(6), new, ctx, page, hkv, d, 6)
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn((sum(new), hq, d), generator=g, device="cuda").to(torch.bfloat16)
    q[0, 1] = 0
    q[-1] = 0
    cu = [0, new[0], sum(new)]
    k_scale, v_scale = torch.tensor(1e-8, device="cuda"), torch.tensor(0.5, device="cuda")
    got = run_attention(ops, q, cache, table, ctx, cu, max(new), hq, hkv, d, page, 0, 0.125, status=status,
                        scales=(k_scale, v_scale))
    rows = [K.dequantise(cache[i], cache[i + 1], s.cpu()) for i, s in ((0, k_scale), (2, v_scale))]
    want, bound = K.attend(q.cpu(), *rows, table, ctx, cu, 0.125, page, 0)
    assert ((got.cpu().double() - want).abs() <= bound).all() and int(status) == 0


def test_rows_whose_scale_is_a_nan_code_read_as_448(ops, status):
    """... as in the attention, which must not spread a NaN."""
    codes, sf = empty_cache(4, 2, 64, fill=0x5A)[:2]
    sf.fill_(0x30)
    sf[1, 0, 2], sf[2, 1, 0], sf[3] = 0x7F, 0xFF, 0x7E
    half = torch.tensor(0.5, device="cuda")
    got = ops.kv4_rows(codes, sf, half, torch.arange(4, device="cuda"), dtype=torch.float32, status=status)
    assert torch.equal(got.cpu().double(), K.dequantise(codes.cpu(), sf.cpu(), 0.5)) and int(status) == 0


@pytest.mark.parametrize("new,longest", [([3, 1], 2), ([1, 9], 8), ([2, 150, 20], 140)])
def test_attention_reports_a_request_longer_than_max_q_len(ops, status, new, longest):
    """Rows up to max_q_len are right, the ones behind them are left as they are, and the status says so."""
    ctx, hq, hkv, d, page = [40, 200, 7][:len(new)], 8, 2, 64, 16
    table, cache = paged(random.Random(8), new, ctx, page, hkv, d, 8)
    t = sum(new)
    q = torch.randn((t, hq, d), generator=torch.Generator(device="cuda").manual_seed(8), device="cuda").to(torch.bfloat16)
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    out = torch.full((t, hq * d), 7.0, dtype=torch.bfloat16, device="cuda")
    run_attention(ops, q, cache, table, ctx, cu, longest, hq, hkv, d, page, 0, 0.3, out=out, status=status)
    assert int(status) == -6
    rows = [K.dequantise(cache[i], cache[i + 1], 0.5) for i in (0, 2)]
    want, bound = K.attend(q.cpu(), *rows, table, ctx, cu, 0.3, page, 0)
    for b, n in enumerate(new):
        at = slice(cu[b], cu[b] + min(n, longest))
        assert ((out[at].cpu().double() - want[at]).abs() <= bound[at]).all()
        assert (out[at.stop:cu[b + 1]] == 7).all()
    status.zero_()
    run_attention(ops, q, cache, table, ctx, cu, max(new), hq, hkv, d, page, 0, 0.3, out=out, status=status)
    assert int(status) == 0


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (4, 4, 128)])
@pytest.mark.parametrize("far", [0, 900, 1 << 18])
def test_store_turns_queries_as_the_fp8_store_does(ops, status, hq, hkv, d, far):
    """The two stores agree on norm, pairs and direction; the angle is an fp32 product in the FP8 one (off by half a step,
    2^-24 of it) and a 64-bit one here.  Beside that: half an E4M3 step (2^-4, or 2^-10 among the subnormals) and half a
    bf16 one, and 2^-19 of the pair for the norms, sines and cosines formed in fp32 on both sides."""
    t = 60
    g = torch.Generator(device="cuda").manual_seed(far + d)
    qkv = torch.randn((t, (hq + 2 * hkv) * d), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, far + 1, (t,), generator=g, device="cuda")
    loc = torch.arange(t, device="cuda")
    inv = (1e4 ** (-torch.arange(0, d, 2, device="cuda") / d)).float()
    one = torch.ones((), device="cuda")
    k, v = (torch.zeros((t, hkv, d), device="cuda").to(FP8) for _ in range(2))
    theirs = ops.qk_rope_store(qkv, pos, loc, inv, one, one, k, v, hq, hkv, d, status=status).double()
    mine = run_store(ops, qkv, pos, loc, inv, [one, one], empty_cache(t, hkv, d), hq, hkv, d, status).double()
    pair = mine.view(t, hq, d // 2, 2).norm(dim=-1)
    turn = (pos.double()[:, None] * inv.double() * 2 ** -24).unsqueeze(1)
    slack = (pair * (turn + 2 ** -19 + 2 ** -8)).repeat_interleave(2, -1)
    bound = slack + (mine.abs() + slack) * 2 ** -4 + 2 ** -10
    assert ((mine - theirs).abs() <= bound).all() and int(status) == 0


@pytest.mark.parametrize("power", [-100, -8, 100])
def test_store_values_and_scale_times_a_power_of_two(ops, status, power):
    """V and its scale times the same power of two have the same codes and block scales, to the ends of the range that
    the interface gives for scales; with a single one they saturate or vanish."""
    t, hq, hkv, d = 50, 2, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn((t, (2 * hq + 2 * hkv) * d), generator=g, device="cuda").to(torch.bfloat16)
    qkv[3, (hq + hkv) * d:] = 0
    loc = torch.arange(t, device="cuda")
    one, scale = torch.ones((), device="cuda"), torch.tensor(2.0 ** power, device="cuda")
    far = qkv.clone()
    far[:, (hq + hkv) * d:] *= 2.0 ** power
    first, second = empty_cache(t, hkv, d), empty_cache(t, hkv, d)
    run_store(ops, qkv, loc, loc, None, [one, one], first, hq, hkv, d, status)
    run_store(ops, far, loc, loc, None, [scale, scale], second, hq, hkv, d, status)
    assert torch.equal(first[2], second[2]) and torch.equal(first[3], second[3]) and int(status) == 0
    _, keys, _ = K.store(qkv.cpu(), loc.cpu(), None, hq, hkv, d)
    want = K.quantise(keys, 2.0 ** power)
    assert torch.equal(second[0].cpu(), want[0]) and torch.equal(second[1].cpu(), want[1].view(torch.uint8))


def test_captured_step_that_moves_its_lengths_on(ops, status):
    """A decode step captured once, with the free list's head and the cached lengths moved on at its end, replayed for one
    token after another: pages, slots and lengths are those of the steps one by one, and every step's attention is right."""
    hq, hkv, d, page, batch = 8, 2, 64, 4, 3
    seq, new = [5, 0, 8], [1, 1, 0]
    table = [[7, 3, -1, -1, -1], [-1] * 5, [0, 11, -1, -1, -1]]
    free, head = [9, 2, 10, 1, 8, 4, 6, 5], 0
    g = torch.Generator(device="cuda").manual_seed(12)
    steps = torch.randn((7, 3, (hq + 2 * hkv) * d), generator=g, device="cuda").to(torch.bfloat16)
    half = torch.tensor(0.5, device="cuda")
    cache = empty_cache(12 * page, hkv, d, fill=0)
    for c, fill in zip(cache, (0x31, 0x38, 0x52, 0x30)):
        c.fill_(fill)
    k, ks, v, vs = cache
    kv = (k, ks.view(FP8), v, vs.view(FP8))
    dev = {"new": i32(new), "seq": i32(seq), "table": i32(table), "free": i32(free), "head": i32([head]), "qkv": steps[0].clone()}

    def step():
        cu, pos, loc, after = ops.page_plan(dev["new"], dev["seq"], dev["table"], dev["free"], dev["head"], page, 3,
                                            status=status)
        q = ops.qk_rope_store_kv4(dev["qkv"], pos, loc, None, half, half, *kv, hq, hkv, d, status=status)
        out = ops.attention_kv4(q, *kv, dev["table"], dev["seq"], cu, half, half, 0.3, batch, 1, hq, hkv, d, page, 0,
                                status=status)
        dev["head"].copy_(after)
        dev["seq"].add_(dev["new"])
        return q, out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    start = {n: x.clone() for n, x in dev.items()}
    before = [c.clone() for c in cache]
    with torch.cuda.stream(side):                             # a first call outside the capture, taken back
        step()
    torch.cuda.current_stream().wait_stream(side)
    for n, x in start.items():
        dev[n].copy_(x)
    for c, b in zip(cache, before):
        c.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = step()
    for qkv in steps:
        dev["qkv"].copy_(qkv)
        graph.replay()
        table, cu, _, loc, head, bad = K.plan(new, seq, table, free, head, page, 3)
        rows = [K.dequantise(cache[i].cpu(), cache[i + 1].cpu(), 0.5) for i in (0, 2)]
        want, bound = K.attend(q.cpu()[:2], *rows, torch.tensor(table), seq, cu, 0.3, page, 0)
        assert ((out[:2].cpu().double() - want).abs() <= bound).all()
        seq = [c + n for c, n in zip(seq, new)]
        assert not bad and dev["table"].tolist() == table and dev["seq"].tolist() == seq and dev["head"].tolist() == [head]
        check_store(q[:2], cache, torch.tensor(loc[:2], device="cuda"), qkv[:2], torch.zeros(2), None, (half, half), hq, hkv, d)
    assert head == 3 and int(status) == 0
