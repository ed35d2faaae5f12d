"""The 8-bit cache in plain torch, 64 bits, on the CPU: what the kernels of quant_cache.cu and attention_q8.cu are compared with."""
import math

import torch

LEAST = 2.0 ** -110


def quantize(x):
    """Whole numbers (float64) and scales of rows [..., hd] of float64 values."""
    most = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    small = most < LEAST
    inv = torch.where(bad | small, torch.zeros_like(most), 127.0 / most.clamp_min(LEAST))
    codes = torch.round(torch.where(bad[..., None], torch.zeros_like(x), x) * inv[..., None])
    scale = torch.where(small, torch.zeros_like(most), most / 127.0)
    return codes, torch.where(bad, torch.full_like(most, math.nan), scale)


def rotate(x, cos, sin, paired=False):
    """[T, heads, hd] turned by [T, rd / 2] tables: channel j with j + rd / 2.  ``paired``: the two stand side by side in x."""
    half = cos.shape[1]
    if not half:
        return x
    if paired:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], dim=-1)


def row_index(positions, req, table, page_size):
    """Page (-1: none) and place of every token."""
    pages, slots = [], []
    for p, r in zip(positions.tolist(), req.tolist()):
        b = p // page_size if p >= 0 else -1
        pages.append(int(table[r, b]) if 0 <= b < table.shape[1] and 0 <= r < table.shape[0] else -1)
        slots.append(p % page_size if p >= 0 else 0)
    return torch.tensor(pages, dtype=torch.long), torch.tensor(slots, dtype=torch.long)


def attention(q, k, v, ks, vs, cu_q, q_start, kv_len, table, scale, window=0, chunk=0, sink=None):
    """(out, sum of p |v|, largest scale * sum of |q| * 1280 ks of a key, largest p vs of a key times the sum of its channel's numbers) of
    every (token, head, channel), float64.  q [T, nh, hd] and the pages as the kernels get them, moved to the CPU."""
    T, nh, hd = q.shape
    num_pages, nkv, page, _ = k.shape
    G = nh // nkv
    out = torch.zeros(T, nh, hd, dtype=torch.float64)
    mass = torch.zeros_like(out)
    score_abs = torch.zeros(T, nh, 1, dtype=torch.float64)
    least = torch.zeros_like(out)
    for r in range(len(q_start)):
        for t in range(int(cu_q[r]), int(cu_q[r + 1])):
            pos = int(q_start[r]) + t - int(cu_q[r])
            lo = max(0, pos - window + 1) if window else 0
            if chunk:
                lo = max(lo, pos - pos % chunk)
            keys = torch.arange(lo, min(pos + 1, int(kv_len[r])))
            blk = keys // page
            pid = torch.where(blk < table.shape[1], table[r][blk.clamp_max(table.shape[1] - 1)].long(), torch.full_like(blk, -1))
            ok = (pid >= 0) & (pid < num_pages)
            keys, pid = keys[ok], pid[ok]
            if not len(keys):
                continue
            slot = keys % page
            for g in range(nkv):
                kk = k[pid, g, slot].double() * ks[pid, g, slot].double()[:, None]
                vv = v[pid, g, slot].double() * vs[pid, g, slot].double()[:, None]
                qq = q[t, g * G:(g + 1) * G].double()
                s = qq @ kk.t() * scale
                m = s.amax(-1, keepdim=True)
                e = torch.exp(s - m)
                total = e.sum(-1, keepdim=True)
                if sink is not None:
                    total = total + torch.exp(sink[g * G:(g + 1) * G].double()[:, None] - m)
                p = e / total
                out[t, g * G:(g + 1) * G] = p @ vv
                mass[t, g * G:(g + 1) * G] = p @ vv.abs()
                score_abs[t, g * G:(g + 1) * G, 0] = qq.abs().sum(-1) * 1280 * ks[pid, g, slot].double().max() * scale
                w = (p * vs[pid, g, slot].double()).amax(-1, keepdim=True)
                least[t, g * G:(g + 1) * G] = w * v[pid, g, slot].double().abs().sum(0)
    return out, mass, score_abs, least


def attention_bound(out, mass, score_abs, least, hd):
    """What the kernels may be off by:
      the result's rounding to bfloat16, 2^-8 of it;
      the weights', p vs in float16: 2^-11 of each, so of sum p |v|, and where that is less than its smallest step, 2^-25 of the largest weight;
      a score's: hd / 16 products of sixteen terms added in the matrix units, where a key's numbers stand 1152 too high (below 1280), each
      sum cut at 2^-23 of the magnitudes so far, and two steps for what comes off and the factors; as an exponent it is in weights
      and denominator;
      2^-16 for exponentials, and sums of the longest lists tested here in float32."""
    u = 2.0 ** -8
    ds = (hd / 16 + 2) * 2.0 ** -23 * score_abs
    return u * out.abs() + (1 + u) * ((2.0 ** -11 + 2 * torch.expm1(2 * ds) + 2.0 ** -16) * mass + 2.0 ** -25 * least) + 1e-30
