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


class Exact:
    """What :func:`attention` returns, float64 [T, heads, channels] each (or one number a row)."""

    def __init__(self, T, nh, hd):
        def zeros(n):
            return torch.zeros(T, nh, n, dtype=torch.float64)
        self.out = zeros(hd)       # sum of p v
        self.mass = zeros(hd)      # sum of p |v|
        self.raised = zeros(1)     # scale * sum |q| * 1280 times the largest scale of a key
        self.scores = zeros(1)     # scale * the largest sum |q k|
        self.coarse = zeros(1)     # scale * sum |q| times the largest scale of a key of the request
        self.least = zeros(hd)     # the largest p vs times the sum of the channel's numbers
        self.least_v = zeros(hd)   # the largest p times the largest vs of the request, times the sum of the channel's numbers
        self.most_v = zeros(1)     # the largest vs of the request


def attention(q, k, v, ks, vs, cu_q, q_start, kv_len, table, scale, window=0, chunk=0, sink=None):
    """The definition, key by key.  q [T, nh, hd] and the pages as the kernels get them, moved to the CPU."""
    T, nh, hd = q.shape
    num_pages, nkv, page, _ = k.shape
    G = nh // nkv
    e = Exact(T, nh, hd)
    for r in range(len(q_start)):
        whole = torch.arange(int(kv_len[r]))
        held = table[r][(whole // page).clamp_max(table.shape[1] - 1)].long()
        whole, held = whole[held >= 0], held[held >= 0]
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
                heads = slice(g * G, (g + 1) * G)
                key_s, value_s = ks[pid, g, slot].double(), vs[pid, g, slot].double()
                numbers = v[pid, g, slot].double()
                kk, vv = k[pid, g, slot].double() * key_s[:, None], numbers * value_s[:, None]
                qq = q[t, heads].double()
                s = qq @ kk.t() * scale
                m = s.amax(-1, keepdim=True)
                x = torch.exp(s - m)
                total = x.sum(-1, keepdim=True)
                if sink is not None:
                    total = total + torch.exp(sink[heads].double()[:, None] - m)
                p = x / total
                most_k, most_v = (z[held, g, whole % page].double().nan_to_num(0, 0, 0).max() for z in (ks, vs))
                e.out[t, heads], e.mass[t, heads] = p @ vv, p @ vv.abs()
                size = qq.abs().sum(-1, keepdim=True) * scale
                e.raised[t, heads], e.coarse[t, heads] = size * 1280 * key_s.max(), size * most_k
                e.scores[t, heads] = (qq.abs() @ kk.abs().t()).amax(-1, keepdim=True) * scale
                e.least[t, heads] = (p * value_s).amax(-1, keepdim=True) * numbers.abs().sum(0)
                e.least_v[t, heads] = p.amax(-1, keepdim=True) * most_v * numbers.abs().sum(0)
                e.most_v[t, heads] = most_v
    return e


def attention_bound(e, hd, wide=None):
    """What the kernels may be off by:
      the result's rounding to bfloat16, 2^-8 of it;
      the weights', p vs in float16: 2^-11 of each, so of sum p |v|, and where that is less than its smallest step, 2^-25 of the largest weight;
      a score's: hd / 16 products of sixteen terms added in the matrix units, where a key's numbers stand 1152 too high (below 1280), each
      sum cut at 2^-23 of the magnitudes so far, and two steps for what comes off and the factors; as an exponent it is in weights
      and denominator;
      2^-16 for exponentials, and sums of the longest lists tested here in float32.
    ``wide`` [T]: rows of the tcgen05 kernel, where keys and values are rounded to float16 too (their scale, then the product), as multiples of
    a power of two that is less than twice the largest scale of the 64 keys beside them: 2^-10 of sum |q k|, and where that is less than
    float16's smallest step, 2^-25 of twice that scale for every channel, and of a number of 127 at most for the scale; of values 2^-10 of
    sum p |v|, and as much of twice theirs; the weights are multiples of p times it."""
    u = 2.0 ** -8

    def bound(ds, rounding, small):
        return u * e.out.abs() + (1 + u) * ((rounding + 2 * torch.expm1(2 * ds) + 2.0 ** -16) * e.mass + small) + 1e-30
    sums = (hd / 16 + 2) * 2.0 ** -23
    tol = bound(sums * e.raised, 2.0 ** -11, 2.0 ** -25 * e.least)
    if wide is not None and wide.any():
        more = bound((sums + 2.0 ** -10) * e.scores + 128 * 2.0 ** -24 * e.coarse, 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -20,
                     2.0 ** -24 * (e.least_v + 128 * e.most_v))
        tol = torch.where(wide[:, None, None], more, tol)
    return tol
