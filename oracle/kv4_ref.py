"""TEST INFRASTRUCTURE ONLY: the operators of the 4-bit K/V cache, restated in 64 bits on the CPU.

Format: 16 channels share an E4M3 scale s, an element is an E2M1 code c (element 2i in the low nibble of byte i) and
stands for c * s * scale; s = e4m3(min(448, max|z| / (6 scale))), c = e2m1(z / (s * scale)), to nearest, ties to even.
The reference caches FP8 only (muse_prefill_layer/reference.py:181-191); masks, norms and the gate follow its
attention block (reference.py:356-410).
"""
from __future__ import annotations

import torch

from oracle.nvfp4_ref import E2M1_GRID

FP8 = torch.float8_e4m3fn
EPS = 1e-5
GRID = torch.tensor(E2M1_GRID, dtype=torch.float64)
SCALES = torch.arange(127, dtype=torch.uint8).view(FP8).double()       # the finite E4M3 values >= 0, ascending


def nearest(x, points):
    """Index of the nearest of ascending `points`, the even index on a tie; x beyond the last takes the last."""
    hi = torch.searchsorted(points, x.contiguous()).clamp(1, len(points) - 1)
    lo = hi - 1
    below, above = x - points[lo], points[hi] - x
    take_lo = (below < above) | ((below == above) & (lo % 2 == 0))
    return torch.where(take_lo, lo, hi)


def quantise(z, scale):
    """(codes u8 [..., D / 2], scales e4m3 [..., D / 16]) of fp64 z [..., D]."""
    scale = float(scale)
    blocks = z.double().reshape(*z.shape[:-1], z.shape[-1] // 16, 16)
    s_idx = nearest((blocks.abs().amax(-1) / (6.0 * scale)).clamp(max=448.0), SCALES)
    unit = (SCALES[s_idx] * scale).unsqueeze(-1)
    code = nearest((blocks.abs() / unit.where(unit > 0, torch.ones(()).double())).clamp(max=6.0), GRID)
    code = torch.where(unit > 0, code + 8 * (blocks < 0), torch.zeros_like(code)).reshape(*z.shape[:-1], z.shape[-1] // 2, 2)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), s_idx.to(torch.uint8).view(FP8)


def dequantise(codes, scales, scale):
    """fp64 [..., D]; a NaN scale byte reads as 448."""
    s = scales.view(FP8).double().nan_to_num(nan=448.0) * float(scale)
    c = torch.stack([codes & 15, codes >> 4], -1).long().flatten(-2)
    v = torch.where(c >= 8, -GRID[c % 8], GRID[c % 8])
    return (v.reshape(*s.shape, 16) * s.unsqueeze(-1)).flatten(-2)


def store(qkv, positions, inv_freq, hq, hkv, d):
    """(q, k, v) in fp64 [T, heads, D] as they are before rounding."""
    x = qkv[:, :(hq + 2 * hkv) * d].double().reshape(-1, hq + 2 * hkv, d)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    qk = qk / (qk.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    if inv_freq is not None:
        angle = positions.double()[:, None] * inv_freq.double()
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        e, o = qk[..., 0::2], qk[..., 1::2]
        qk = torch.stack([e * cos - o * sin, e * sin + o * cos], -1).flatten(-2)
    return qk[:, :hq], qk[:, hq:], v


def attend(q, k_rows, v_rows, page_table, seq_lens, cu, softmax_scale, page, window, gate=None):
    """Attention over fp64 cache rows [rows, hkv, D].  Returns (out fp64 [T, hq * D], an elementwise bound of the error
    that rounding P to fp16, the fp32 sums and the final rounding to bf16 can make).

    Rounding P moves each term by at most half an fp16 step, 2^-11 of it, or 2^-25 below 2^-14 (P's largest value is at
    least 1 and l at least that, so the latter adds at most 2^-25 sum|v|); the fp32 scores, exponentials and sums are
    good to 2^-13 of a term as long as the scores stay below 2^8 in log2 units; bf16 adds half a step, 2^-8."""
    t, hq, d = q.shape
    hkv = k_rows.shape[1]
    out, bound = torch.zeros((t, hq, d)).double(), torch.zeros((t, hq, d)).double()
    for b in range(len(seq_lens)):
        first, n, past = int(cu[b]), int(cu[b + 1] - cu[b]), int(seq_lens[b])
        for h in range(hq):
            kv = h // (hq // hkv)
            keys = torch.arange(past + n)
            idx = (keys // page).clamp(max=page_table.shape[1] - 1)
            pages = page_table[b].long()[idx]
            pages = torch.where(keys // page < page_table.shape[1], pages, torch.full_like(pages, -1))
            rows = pages * page + keys % page
            held = (pages >= 0) & (rows < k_rows.shape[0])
            rows = rows.where(held, torch.zeros_like(rows))
            pos = past + torch.arange(n)[:, None]
            seen = (keys <= pos) & held
            if window:
                seen &= keys > pos - window
            kk, vv = k_rows[rows, kv], v_rows[rows, kv]
            vv = vv.where(seen.any(0)[:, None], torch.zeros_like(vv))
            s = (q[first:first + n, h].double() @ kk.T * softmax_scale).masked_fill(~seen, float("-inf"))
            p = torch.softmax(s, -1).nan_to_num(0.0)                 # a row that sees nothing is zero
            out[first:first + n, h] = p @ vv
            bound[first:first + n, h] = p @ vv.abs() * (2.0 ** -11 + 2.0 ** -13) + 2.0 ** -25 * seen.double() @ vv.abs()
    if gate is not None:
        r = (out.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        # d(o r) = r do - o r^3 mean(o do), and r rms(o) <= 1
        bound = r * (bound + out.abs() * r * bound.pow(2).mean(-1, keepdim=True).sqrt())
        sig = torch.sigmoid(gate.double()).reshape(t, hq, d)
        out, bound = out * r * sig, bound * sig + 2.0 ** -20 * (out * r * sig).abs()
    out, bound = out.flatten(1), bound.flatten(1)
    return out, bound + 2.0 ** -8 * (out.abs() + bound) + 1e-38


def plan(new_lens, seq_lens, page_table, free_pages, free_head, page, tokens):
    """(page table, cu, positions, cache_loc, free head, anything wrong) by the definition, lists in and out."""
    table, head, bad = [list(r) for r in page_table], free_head, False
    width = len(table[0])
    cu, positions, loc = [0], [], []
    for b, (n, c) in enumerate(zip(new_lens, seq_lens)):
        bad |= n < 0 or c < 0
        n, c = max(n, 0), max(c, 0)
        bad |= -(-(c + n) // page) > width
        for i in range(min(-(-c // page), width), min(-(-(c + n) // page), width)):
            if 0 <= head < len(free_pages):
                table[b][i] = free_pages[head]
                head += 1
            else:
                table[b][i], bad = -1, True
        for pos in range(c, c + n):
            have = table[b][pos // page] if pos // page < width else -1
            bad |= have < 0
            positions.append(pos)
            loc.append(have * page + pos % page if have >= 0 else -1)
        cu.append(min(cu[-1] + n, tokens))
    bad |= len(positions) > tokens
    pad = tokens - len(positions)
    return table, cu, (positions + [0] * pad)[:tokens], (loc + [-1] * pad)[:tokens], head, bad
