"""What the 8-bit cache of keys and values and the log probabilities of given tokens are measured on.

Four kinds of case, each one call or two of a program that serves a model:

``write``    a step's keys and values go into the cache: rotation of the queries and keys, every (token, kv head) row of a key or a
             value as whole numbers of -127 to 127 with one float32 scale, written to the page of its position; then what was
             written is read back, as bfloat16.
``read``     the keys and values of whole requests read back from their pages as bfloat16 (a request handed to another cache, or
             looked at).
``attend``   causal attention of a step's tokens over the cache: ``decode`` requests with ``step`` tokens each (one, or the few of a
             draft that is checked) at contexts of ``shortest`` to ``longest`` tokens, and, where ``portion`` > 0, that many tokens of
             one more request's prompt, which stands at position ``at``.
``logprob``  log probabilities of given tokens under a step's logits: of the token itself, its rank, the entropy of its
             distribution, and the ``top`` most probable tokens (ties: the lowest id first).

Everything follows from the seed.  Keys have a few channels that are much larger than the others, as keys of a trained model have;
pages lie in the pool in random order, and what lies behind a request's last token is left over from others.
"""
import math
import random

import torch

own = False

# (query heads, kv heads, head size)
HEADS = {"8b": (32, 8, 128), "7b": (28, 4, 128), "14b": (40, 8, 128)}
MORE_HEADS = {"even64": (16, 16, 64), "seven64": (14, 2, 64), "three96": (12, 4, 96), "two256": (16, 8, 256), "one128": (8, 1, 128),
              "five80": (10, 2, 80)}
ALL_HEADS = {**HEADS, **MORE_HEADS}
MOST = 127.0


def _write(name, heads, tokens, requests, at, page=16):
    return {"name": name, "kind": "write", "heads": heads, "tokens": tokens, "requests": requests, "at": at, "page": page}


def _read(name, heads, requests, shortest, longest, page=16):
    return {"name": name, "kind": "read", "heads": heads, "requests": requests, "shortest": shortest, "longest": longest, "page": page}


def _attend(name, heads, decode=0, shortest=0, longest=0, step=1, portion=0, at=0, page=16):
    return {"name": name, "kind": "attend", "heads": heads, "decode": decode, "shortest": shortest, "longest": longest, "step": step,
            "portion": portion, "at": at, "page": page}


def _logprob(name, rows, vocab, top):
    return {"name": name, "kind": "logprob", "rows": rows, "vocab": vocab, "top": top}


def listed():
    return [
        # a decode step of eight requests: one row of keys and of values a request and kv head
        _write("write_8", "8b", 8, 8, 8191),
        # a prompt's keys and values
        _write("write_2048", "8b", 2048, 1, 0),
        # a chat's history read back
        _read("read_701", "8b", 1, 701, 701),
        # eight long requests, moved to another cache
        _read("read_8x8192", "8b", 8, 8192, 8192),
        # a chat with one user: one token, a short history
        _attend("chat_token", "8b", decode=1, shortest=701, longest=701),
        # eight requests deep in their contexts
        _attend("decode_8x8192", "8b", decode=8, shortest=8192, longest=8192),
        # a busy server: many requests at contexts of all lengths decode while one more joins with a piece of its prompt
        _attend("serve_mixed", "7b", decode=31, shortest=512, longest=4096, portion=617, at=512),
        # an ordinary prompt, whole
        _attend("prompt_2048", "8b", portion=2048),
        # a later piece of a long document's prompt
        _attend("long_prompt_piece", "14b", portion=2048, at=13312),
        # a chat that shows how sure the model was of its token, with five alternatives
        _logprob("logprob_1", 1, 128256, 5),
        # a server's batch, each request with the most alternatives
        _logprob("logprob_32", 32, 152064, 20),
        # a text scored: every token's log probability, and what the model would have said
        _logprob("score_1024", 1024, 128256, 1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    """Seconds, roughly: what keeps a drawn case within the listed ones."""
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 4e14


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        del case["name"]
        if _cost(case) <= most:
            return case


def _draw(rng):
    kind = rng.random()
    heads = rng.choice(sorted(HEADS) * 3 + sorted(MORE_HEADS))
    page = rng.choice([16, 16, 16, 8, 32, 64, 24])
    if kind < 0.15:
        n = _log(rng, 1, 4096)
        requests = min(n, rng.choice([1, n, _log(rng, 1, 16)]))
        return _write("", heads, n, min(requests, 256), rng.choice([0, _log(rng, 1, 100000)]), page)
    if kind < 0.3:
        requests = _log(rng, 1, 16)
        longest = _log(rng, 1, max(1, 65536 // requests))
        return _read("", heads, requests, (longest + 2) // 3, longest, page)
    if kind < 0.5:       # decode
        n = _log(rng, 1, 64)
        longest = _log(rng, 16, min(65536, 262144 // n))
        return _attend("", heads, decode=n, shortest=longest // 8 + 8, longest=max(longest, longest // 8 + 8), step=rng.choice([1, 1, 1, 2, 5]),
                       page=page)
    if kind < 0.62:      # a prompt, or a later piece of one
        return _attend("", heads, portion=_log(rng, 2, 2048), at=rng.choice([0, 0, _log(rng, 1, 13312)]), page=page)
    if kind < 0.75:      # both
        n = _log(rng, 2, 48)
        longest = _log(rng, 64, min(4096, 70000 // n))
        return _attend("", heads, decode=n, shortest=longest // 8 + 1, longest=longest, portion=_log(rng, 17, 1500),
                       at=rng.choice([0, _log(rng, 1, 4096)]), page=page)
    return _logprob("", _log(rng, 1, 1024), rng.choice([32000, 128256, 152064, 50021, _log(rng, 1000, 160000)]), rng.choice([0, 1, 5, 5, 20]))


# ------------------------------------------------------------------------------------------------ sizes of a case
def _segments(case):
    """(tokens, position of the first, length after the step) of every request: a matter of the case, not of the seed."""
    if case["kind"] == "write":
        n, r = case["tokens"], case["requests"]
        lens = [n // r + (i < n % r) for i in range(r)]
        return [(m, case["at"], case["at"] + m) for m in lens]
    rng = random.Random(case["longest"] * 31 + case.get("decode", 0) + case.get("requests", 0))
    count = case["decode"] if case["kind"] == "attend" else case["requests"]
    lens = [max(rng.randint(case["shortest"], case["longest"]), case.get("step", 1)) for _ in range(count)]
    if case["kind"] == "read":
        return [(m, 0, m) for m in lens]
    got = [(case["step"], m - case["step"], m) for m in lens]
    if case["portion"]:
        got.append((case["portion"], case["at"], case["at"] + case["portion"]))
    return got


def work(case):
    if case["kind"] == "logprob":
        rows, top = case["rows"], case["top"]
        return {"bytes": rows * (4 * case["vocab"] + 4 + 12 + 8 * top), "flops": 4 * rows * case["vocab"]}
    nh, nkv, hd = ALL_HEADS[case["heads"]]
    row = hd + 4                                    # a cached row and its scale
    segs = _segments(case)
    tokens = sum(n for n, _, _ in segs)
    if case["kind"] == "write":
        # the projection's rows and the table of cosines and sines in, the queries, the rows and what is read back out
        return {"bytes": tokens * ((nh + 2 * nkv) * hd * 4 + hd * 4 + nh * hd * 2 + 2 * nkv * row + 4 * nkv * hd),
                "flops": tokens * (nh + 2 * nkv) * hd * 4}
    if case["kind"] == "read":
        return {"bytes": tokens * nkv * 2 * (row + 2 * hd), "flops": tokens * nkv * 2 * hd}
    seen = sum(n * at + n * (n + 1) // 2 for n, at, _ in segs)
    return {"bytes": sum(total for _, _, total in segs) * nkv * 2 * row + tokens * nh * hd * 4, "flops": 4 * seen * nh * hd}


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.empty(shape, device="cuda").normal_(0.0, 1.0, generator=gen)


def _pool(gen, pages, nkv, page, hd, loud):
    """Rows of whole numbers and their scales, as the cache holds them: [pages, kv heads, page, head size] and without the last."""
    spread = torch.ones(hd, device="cuda")
    if loud:
        spread[torch.randint(0, hd, (max(1, hd // 32),), generator=gen, device="cuda")] = 6.0
    codes = torch.empty((pages, nkv, page, hd), dtype=torch.int8, device="cuda")
    scales = torch.empty((pages, nkv, page), dtype=torch.float32, device="cuda")
    for a in range(0, pages, 1024):
        x = _normal(gen, min(1024, pages - a), nkv, page, hd) * spread
        x = x * torch.exp(0.4 * _normal(gen, *x.shape[:3], 1))           # some tokens louder than others
        most = x.abs().amax(-1)
        codes[a:a + 1024] = torch.round(x * (MOST / most)[..., None]).to(torch.int8)
        scales[a:a + 1024] = most / MOST
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    state = {"case": case, "kind": case["kind"]}
    if case["kind"] == "logprob":
        rows, vocab = case["rows"], case["vocab"]
        # some distributions sharp and some flat; a text's tokens are mostly likely ones
        logits = _normal(gen, rows, vocab) * torch.empty(rows, 1, device="cuda").uniform_(0.8, 3.5, generator=gen)
        likely = logits.argmax(-1)
        other = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        pick = torch.rand(rows, generator=gen, device="cuda") < 0.5
        state["logits"], state["targets"] = logits, torch.where(pick, likely, other).to(torch.int32)
        return state
    nh, nkv, hd = ALL_HEADS[case["heads"]]
    page = case["page"]
    segs = _segments(case)
    lens = torch.tensor([n for n, _, _ in segs])
    starts = torch.tensor([a for _, a, _ in segs])
    totals = torch.tensor([t for _, _, t in segs])
    R, T = len(segs), int(lens.sum())
    blocks = -(-totals // page)
    W = int(blocks.max())
    req = torch.repeat_interleave(torch.arange(R), lens)
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
    pos = torch.arange(T) - cu[:-1][req] + starts[req]
    # pages are held where something is read or written; other places of a table hold no page
    first = starts // page if case["kind"] == "write" else torch.zeros_like(starts)
    held = (torch.arange(W)[None] < blocks[:, None]) & (torch.arange(W)[None] >= first[:, None])
    count = int(held.sum())
    pages = count + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed * 31 + 1))[:count]
    table = torch.full((R, W), -1)
    table[held] = order
    state.update(nh=nh, nkv=nkv, hd=hd, R=R, T=T, pages=pages, h_len=lens.tolist(), h_start=starts.tolist(), h_total=totals.tolist(),
                 req=req.to("cuda", torch.int32), pos=pos.to("cuda", torch.int32), cu=cu.to("cuda", torch.int32),
                 start=starts.to("cuda", torch.int32), total=totals.to("cuda", torch.int32), table=table.to("cuda", torch.int32))
    if case["kind"] == "write":
        state["k"] = torch.zeros((pages, nkv, page, hd), dtype=torch.int8, device="cuda")
        state["v"] = torch.zeros_like(state["k"])
        state["k_scale"] = torch.zeros((pages, nkv, page), device="cuda")
        state["v_scale"] = torch.zeros_like(state["k_scale"])
        x = _normal(gen, T, nh + 2 * nkv, hd)
        loud = torch.randint(0, hd, (max(1, hd // 32),), generator=gen, device="cuda")
        x[:, nh:nh + nkv, loud] *= 6.0
        state["qkv"] = x.reshape(T, -1)
        inv = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        angle = state["pos"].double()[:, None] * inv
        state["turns"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        return state
    state["k"], state["k_scale"] = _pool(gen, pages, nkv, page, hd, True)
    state["v"], state["v_scale"] = _pool(gen, pages, nkv, page, hd, False)
    if case["kind"] == "attend":
        state["q"] = _normal(gen, T, nh * hd).to(torch.bfloat16)
        state["scale"] = hd ** -0.5
    return state


# ------------------------------------------------------------------------------------------------ the calls
def run(state):
    return _OWN[state["kind"]](state) if own else _PLAIN[state["kind"]](state)


def _pages(s):
    from blackwellllm_b200.kernels import ops
    return ops.QuantPages(s["k"], s["v"], s["k_scale"], s["v_scale"])


def _own_write(s):
    from blackwellllm_b200.kernels import ops
    pages = _pages(s)
    q = ops.quant_append(s["qkv"], s["pos"], s["req"], s["table"], pages, s["nh"], table=s["turns"])
    k, v = ops.quant_read(pages, s["pos"], s["req"], s["table"])
    return {"q": q, "k": k, "v": v}


def _own_read(s):
    from blackwellllm_b200.kernels import ops
    k, v = ops.quant_read(_pages(s), s["pos"], s["req"], s["table"])
    return {"k": k, "v": v}


def _own_attend(s):
    from blackwellllm_b200.engine.batch import StepBatch
    from blackwellllm_b200.kernels import ops
    batch = StepBatch(T=s["T"], R=s["R"], token_ids=s["pos"], positions=s["pos"], req_of_token=s["req"], cu_q=s["cu"], q_start=s["start"],
                      kv_len=s["total"], state_slot=s["start"], logit_rows=s["start"], block_tables={0: s["table"]},
                      h_q_start=s["h_start"], h_q_len=s["h_len"], h_kv_len=s["h_total"])
    return ops.quant_attention(s["q"], _pages(s), batch, s["table"], s["nh"], s["scale"])


def _own_logprob(s):
    from blackwellllm_b200.kernels import ops
    got = ops.token_log_probs(s["logits"], s["targets"], s["case"]["top"])
    return {"log_prob": got.log_prob, "entropy": got.entropy, "rank": got.rank, "top_ids": got.top_ids, "top_log_probs": got.top_log_probs}


# ------------------------------------------------------------------------------------------------ the plain forms
def _where(s):
    """Page and place in it of every token of the step."""
    page = s["case"]["page"]
    return s["table"][s["req"].long(), (s["pos"] // page).long()].long(), (s["pos"] % page).long()


def _plain_read(s):
    page, slot = _where(s)
    k = s["k"][page, :, slot].float() * s["k_scale"][page, :, slot][..., None]
    v = s["v"][page, :, slot].float() * s["v_scale"][page, :, slot][..., None]
    return {"k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16)}


def _held(x):
    """Whole numbers and scale of rows [..., head size]."""
    most = x.abs().amax(-1)
    codes = torch.round(x * torch.where(most > 0, MOST / most, 0.0)[..., None]).to(torch.int8)
    return codes, most / MOST


def _plain_write(s):
    nh, nkv, hd = s["nh"], s["nkv"], s["hd"]
    x = s["qkv"].view(s["T"], nh + 2 * nkv, hd)
    cos, sin = s["turns"].chunk(2, dim=1)
    a, b = x[:, :nh + nkv].chunk(2, dim=-1)
    turned = torch.cat([a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]], dim=-1)
    page, slot = _where(s)
    s["k"][page, :, slot], s["k_scale"][page, :, slot] = _held(turned[:, nh:])
    s["v"][page, :, slot], s["v_scale"][page, :, slot] = _held(x[:, nh + nkv:])
    return {"q": turned[:, :nh].to(torch.bfloat16).reshape(s["T"], nh * hd), **_plain_read(s)}


def _attend_group(s, r0, r1):
    """Attention of requests r0 to r1 - 1, which have the same number of tokens."""
    nh, nkv, hd = s["nh"], s["nkv"], s["hd"]
    n, G, page = s["h_len"][r0], nh // nkv, s["case"]["page"]
    W = -(-max(s["h_total"][r0:r1]) // page)
    table = s["table"][r0:r1, :W].long().clamp_min(0)

    def gathered(codes, scales):
        x = codes[table].float() * scales[table][..., None]                     # [requests, W, kv heads, page, head size]
        return x.permute(0, 2, 1, 3, 4).reshape(r1 - r0, nkv, W * page, hd)
    k, v = gathered(s["k"], s["k_scale"]), gathered(s["v"], s["v_scale"])
    t0 = sum(s["h_len"][:r0])
    q = s["q"][t0:t0 + n * (r1 - r0)].float().view(r1 - r0, n, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(r1 - r0, nkv, G * n, hd)
    scores = (q @ k.transpose(-1, -2)) * s["scale"]
    at = s["start"][r0:r1, None].long() + torch.arange(n, device="cuda")
    hidden = torch.arange(W * page, device="cuda")[None, None] > at[..., None]  # [requests, n, keys]
    scores = scores.view(r1 - r0, nkv, G, n, W * page).masked_fill_(hidden[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    total = p.sum(-1, keepdim=True)
    # places behind a request's last token have weight 0
    v = v.masked_fill((torch.arange(W * page, device="cuda")[None] >= s["total"][r0:r1, None])[:, None, :, None], 0.0)
    o = (p.view(r1 - r0, nkv, G * n, W * page) @ v).view(r1 - r0, nkv, G, n, hd) / total
    return o.permute(0, 3, 1, 2, 4).reshape(-1, nh * hd).to(torch.bfloat16)


def _plain_attend(s):
    decode = s["case"]["decode"]
    groups = [_attend_group(s, a, b) for a, b in ((0, decode), (decode, s["R"])) if b > a]
    return torch.cat(groups) if len(groups) > 1 else groups[0]


def _plain_logprob(s):
    x, top = s["logits"], s["case"]["top"]
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    z = e.sum(-1)
    log_z = z.log()
    entropy = log_z - (e * d).sum(-1) / z
    at = s["targets"].long()[:, None]
    mine = x.gather(-1, at)
    before = (x > mine) | ((x == mine) & (torch.arange(x.shape[1], device="cuda") < at))
    log_prob = d.gather(-1, at)[:, 0] - log_z
    value, ids = torch.sort(d, dim=-1, descending=True, stable=True)
    return {"log_prob": log_prob, "entropy": entropy, "rank": before.sum(-1).to(torch.int32), "top_ids": ids[:, :top].to(torch.int32),
            "top_log_probs": value[:, :top] - log_z[:, None]}


_OWN = {"write": _own_write, "read": _own_read, "attend": _own_attend, "logprob": _own_logprob}
_PLAIN = {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "logprob": _plain_logprob}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s)


def _exact_rows(codes, scales, s):
    """The cached rows of every token of the step [tokens, kv heads, head size]."""
    page = s["case"]["page"]
    flat = s["table"].long()[s["req"].long(), (s["pos"] // page).long()] * page + s["pos"].long() % page
    rows = codes.transpose(1, 2).reshape(-1, s["nkv"], s["hd"])[flat].double()
    return rows * scales.transpose(1, 2).reshape(-1, s["nkv"])[flat].double().unsqueeze(-1)


def _exact_read(s):
    return {"k": _exact_rows(s["k"], s["k_scale"], s), "v": _exact_rows(s["v"], s["v_scale"], s)}


def _exact_write(s):
    T, nh, nkv, hd = s["T"], s["nh"], s["nkv"], s["hd"]
    x = s["qkv"].double().view(T, nh + 2 * nkv, hd)
    half = hd // 2
    pairs = torch.complex(x[:, :nh + nkv, :half], x[:, :nh + nkv, half:])
    turns = torch.complex(s["turns"][:, :half].double(), s["turns"][:, half:].double())[:, None]
    turned = torch.view_as_real(pairs * turns).transpose(-1, -2).reshape(T, nh + nkv, hd)

    def read_back(rows):
        step = rows.abs().amax(-1, keepdim=True) / 127
        return torch.where(step > 0, torch.round(rows / step) * step, torch.zeros_like(rows))
    return {"q": turned[:, :nh].reshape(T, nh * hd), "k": read_back(turned[:, nh:]), "v": read_back(x[:, nh + nkv:])}


def _exact_attend(s):
    nh, nkv, hd, page = s["nh"], s["nkv"], s["hd"], s["case"]["page"]
    out, t0 = torch.empty(s["T"], nh, hd, dtype=torch.float64, device="cuda"), 0
    for r, (n, at, total) in enumerate(zip(s["h_len"], s["h_start"], s["h_total"])):
        ids = s["table"][r, :-(-total // page)].long()
        seen = torch.arange(total, device="cuda")[None] <= at + torch.arange(n, device="cuda")[:, None]
        for g in range(nkv):
            k = (s["k"][ids, g].double() * s["k_scale"][ids, g, :, None].double()).reshape(-1, hd)[:total]
            v = (s["v"][ids, g].double() * s["v_scale"][ids, g, :, None].double()).reshape(-1, hd)[:total]
            for h in range(g * (nh // nkv), (g + 1) * (nh // nkv)):
                q = s["q"][t0:t0 + n, h * hd:(h + 1) * hd].double()
                p = torch.softmax(torch.where(seen, (q @ k.t()) * s["scale"], -math.inf), dim=-1)
                out[t0:t0 + n, h] = p @ v
        t0 += n
    return out.view(s["T"], nh * hd)


def _exact_logprob(s):
    top = s["case"]["top"]
    parts = []
    for row, target in zip(s["logits"], s["targets"].tolist()):
        x = row.double()
        lp = x - torch.logsumexp(x, 0)
        order = torch.sort(x, descending=True, stable=True).indices[:top]
        rank = ((x > x[target]).sum() + (x[:target] == x[target]).sum()).to(torch.int32)
        parts.append((lp[target], -(lp.exp() * lp).sum(), rank, order.to(torch.int32), lp[order]))
    return {k: torch.stack([p[i] for p in parts]) for i, k in enumerate(("log_prob", "entropy", "rank", "top_ids", "top_log_probs"))}


_EXACT = {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "logprob": _exact_logprob}
