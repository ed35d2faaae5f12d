"""The 8-bit cache and the log probabilities through the engine: models whose keys and values are written, attended and read back in 8 bits,
and the distributions that generated and given tokens come from, against the plain implementation in 64 bits.

The bound on logits over an 8-bit cache has two parts.  ``tiny.TOL`` times the largest logit covers the engine's bfloat16 arithmetic, as
in the tests of the plain cache.  That arithmetic also makes some numbers round to the other neighbour, which moves a cached number by one
step where rounding itself moves it by at most half a step: so twice what quantisation as a whole does to the plain implementation's logits."""
import math

import pytest
import torch

import tiny
from plain_model import (load_plain_weights, plain_attention, plain_config, plain_embedding, plain_inv_freq, plain_linear, plain_logits,
                         plain_rmsnorm, plain_rope, plain_swiglu)
from plain_quant import quantize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LENGTHS = {"llama": 90, "qwen": 70, "llama3": 50, "partial": 100}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = str(tmp_path_factory.mktemp("models"))
    return {(n, d): tiny.make_folder(n, d, root) for n in tiny.CONFIGS for d in ("float32", "bfloat16")}


def make(folder, dtype="bfloat16", ctx=256, batch=4, **kw):
    from blackwellllm_b200 import BlackwellEngine, InferenceConfig
    return BlackwellEngine(folder, InferenceConfig(max_context_length=ctx, max_batch_size=batch), dtype=dtype, **kw)


def quant_logits(raw, weights, ids):
    """The plain implementation with every key row (rotated) and value row a scale and whole numbers."""
    c = plain_config(raw)
    W = {k: v.double() for k, v in weights.items()}
    x = plain_embedding(W["model.embed_tokens.weight"], ids)
    T, pos, inv = len(ids), torch.arange(len(ids)), plain_inv_freq(c["hd"], c["theta"], c["scaling"], c["rd"])

    def rows(t):
        codes, scale = quantize(t)
        return codes * scale[..., None]

    for i in range(c["L"]):
        p = f"model.layers.{i}."
        h = plain_rmsnorm(x, W[p + "input_layernorm.weight"], c["eps"])
        q, k, v = (plain_linear(h, W[p + f"self_attn.{n}_proj.weight"], W.get(p + f"self_attn.{n}_proj.bias") if c["bias"] else None)
                   .view(T, -1, c["hd"]) for n in "qkv")
        o = plain_attention(plain_rope(q, pos, inv), rows(plain_rope(k, pos, inv)), rows(v)).reshape(T, -1)
        x = x + plain_linear(o, W[p + "self_attn.o_proj.weight"])
        h = plain_rmsnorm(x, W[p + "post_attention_layernorm.weight"], c["eps"])
        x = x + plain_linear(plain_swiglu(plain_linear(h, W[p + "mlp.gate_proj.weight"]), plain_linear(h, W[p + "mlp.up_proj.weight"])),
                             W[p + "mlp.down_proj.weight"])
    x = plain_rmsnorm(x, W["model.norm.weight"], c["eps"])
    return plain_linear(x, W["model.embed_tokens.weight"] if c["tie"] else W["lm_head.weight"])


def oracle(raw, folder, ids):
    """Logits over the 8-bit cache, and the bound on the engine's."""
    W = load_plain_weights(folder)
    want, plain = quant_logits(raw, W, ids), plain_logits(raw, W, ids)
    return want, tiny.TOL["bfloat16"] * float(want.abs().max()) + 2.0 * float((want - plain).abs().max())


def check(got, want, bound):
    got = got.double().cpu()
    assert bool(torch.isfinite(got).all())
    assert float((got - want).abs().max()) <= bound, (float((got - want).abs().max()), bound)


@pytest.mark.parametrize("cuts", ["whole", "pieces", "one_by_one"])
@pytest.mark.parametrize("name", list(tiny.CONFIGS))
def test_logits_wherever_a_prompt_is_cut(folders, name, cuts):
    """All at once, in portions of odd sizes (1 to 40 rows), or a token at a time (recorded and replayed)."""
    from blackwellllm_b200 import StepEntry
    raw, _, page = tiny.CONFIGS[name]
    n = LENGTHS[name]
    ids = tiny.prompt(n, raw["vocab_size"], 21)
    want, bound = oracle(raw, folders[(name, "bfloat16")], ids)
    eng = make(folders[(name, "bfloat16")], page_size=page, kv_dtype="int8").engine
    sizes = {"whole": [n], "pieces": [1, 2, 5, 17, 3, 16], "one_by_one": [1] * n}[cuts]
    if cuts == "pieces":
        sizes.append(n - sum(sizes))
    at = 0
    for m in sizes:
        got = eng.step([StepEntry("a", ids[at:at + m], list(range(m)))])
        check(got, want[at:at + m], bound)
        at += m
    if cuts == "one_by_one":
        assert eng.graph_kernel_count(1) > 0


@pytest.mark.parametrize("heads, kv, hd", [(4, 2, 64), (6, 2, 128), (4, 1, 192)])
def test_logits_of_wider_heads(tmp_path, heads, kv, hd):
    """Heads whose prompts the tensor-memory kernel takes: a prompt, a portion behind it, and tokens one by one."""
    from blackwellllm_b200 import StepEntry
    from blackwellllm_b200.weights.random_init import write_random_model
    raw = dict(tiny.TINY_LLAMA, hidden_size=128, num_attention_heads=heads, num_key_value_heads=kv, head_dim=hd)
    write_random_model(str(tmp_path), raw, dtype="bfloat16", seed=3, std=0.05)
    ids = tiny.prompt(190, raw["vocab_size"], 8)
    want, bound = oracle(raw, str(tmp_path), ids)
    eng = make(str(tmp_path), page_size=16, kv_dtype="int8").engine
    at = 0
    for m in (100, 1, 1, 1, 1, 1, 66, 17, 1, 1):
        check(eng.step([StepEntry("a", ids[at:at + m], list(range(m)))]), want[at:at + m], bound)
        at += m
    assert at == 190


def test_mixed_steps_and_many_prompts(folders):
    """A step of prompts of every length beside decoding requests; rows of one request never reach another's."""
    from blackwellllm_b200 import StepEntry
    raw, _, page = tiny.CONFIGS["llama"]
    folder = folders[("llama", "bfloat16")]
    texts = {r: tiny.prompt(n, raw["vocab_size"], 50 + n) for r, n in (("a", 60), ("b", 9), ("c", 33), ("d", 2))}
    ref = {r: oracle(raw, folder, t) for r, t in texts.items()}
    eng = make(folder, page_size=page, kv_dtype="int8").engine
    at = dict.fromkeys(texts, 0)
    for portions in ({"a": 40, "b": 1}, {"b": 1, "c": 20, "a": 1}, {"a": 18, "b": 6, "d": 1, "c": 12}, {"d": 1, "c": 1, "b": 1, "a": 1}):
        got = eng.step([StepEntry(r, texts[r][at[r]:at[r] + n], list(range(n))) for r, n in portions.items()])
        row = 0
        for r, n in portions.items():
            want, bound = ref[r]
            check(got[row:row + n], want[at[r]:at[r] + n], bound)
            at[r], row = at[r] + n, row + n
    assert at == {r: len(t) for r, t in texts.items()}


@pytest.mark.parametrize("name", ["llama", "qwen", "partial"])
def test_the_first_layers_cached_rows(folders, name):
    """Of the first layer, whose input is exact, the keys and values read back stand within half a step of the plain ones and what the
    norm's rounding to bfloat16 (half a step of 2^-8, through the absolute weights) can move them and the largest of their row by."""
    from blackwellllm_b200 import StepEntry
    raw, _, page = tiny.CONFIGS[name]
    folder = folders[(name, "bfloat16")]
    ids = tiny.prompt(61, raw["vocab_size"], 5)
    c, W = plain_config(raw), {k: v.double() for k, v in load_plain_weights(folder).items()}
    p = "model.layers.0."
    h = plain_rmsnorm(plain_embedding(W["model.embed_tokens.weight"], ids), W[p + "input_layernorm.weight"], c["eps"])
    inv, pos = plain_inv_freq(c["hd"], c["theta"], c["scaling"], c["rd"]), torch.arange(61)
    eng = make(folder, page_size=page, kv_dtype="int8").engine
    at = 0
    for m in (30, 1, 1, 9, 20):     # the projection's ways for few tokens and for many
        eng.step([StepEntry("a", ids[at:at + m], [])])
        at += m
    got = eng.cached_kv("a", 0)
    half = c["rd"] // 2
    for n, have in zip("kv", got):
        w, b = W[p + f"self_attn.{n}_proj.weight"], W.get(p + f"self_attn.{n}_proj.bias") if c["bias"] else None
        x = plain_linear(h, w, b).view(61, c["nkv"], c["hd"])
        off = (h.abs() @ w.abs().T * (2.0 ** -8 + 2.0 ** -16)).view(61, c["nkv"], c["hd"])
        if n == "k":
            x = plain_rope(x, pos, inv)
            pair = off[..., :half] + off[..., half:2 * half]
            off = torch.cat([pair, pair, off[..., 2 * half:]], dim=-1)
        most = x.abs().amax(-1, keepdim=True) + off.amax(-1, keepdim=True)
        bound = off + most / 254.0 * (1 + 1e-5) + (most + off) * 2.0 ** -8       # (the last: read back in bfloat16)
        assert have.dtype == torch.bfloat16 and have.shape == x.shape
        assert bool(((have.double().cpu() - x).abs() <= bound).all())
    again = eng.cached_kv("a", 0, 17, 44)
    assert torch.equal(again[0], got[0][17:44]) and torch.equal(again[1], got[1][17:44])


def test_a_sequence_goes_back_and_on(folders):
    """Rewound and continued otherwise: the scales of the rows behind are those of the new tokens."""
    raw, _, page = tiny.CONFIGS["qwen"]
    folder = folders[("qwen", "bfloat16")]
    llm = make(folder, page_size=page, kv_dtype="int8")
    one, two = tiny.prompt(50, raw["vocab_size"], 1), tiny.prompt(50, raw["vocab_size"], 2)
    llm.prefill(one, 0, 0.0, 1.0)
    ids = one[:29] + two[:20]
    llm.prefill(two[:20], 29, 0.0, 1.0)
    want, bound = oracle(raw, folder, ids)
    check(llm._last_logits[0], want[-1], bound)


def test_a_batch_decoded_step_by_step(folders):
    """forward_batch, with the tokens given and taken from the step before: every token is the oracle's best within the bound."""
    from blackwellllm_b200 import DecodeRequest, FROM_LAST
    raw, _, page = tiny.CONFIGS["llama"]
    folder = folders[("llama", "bfloat16")]
    llm = make(folder, page_size=page, kv_dtype="int8")
    texts = {s: tiny.prompt(n, raw["vocab_size"], 90 + n) for s, n in ((3, 19), (1, 40))}
    for s, t in texts.items():
        t.append(llm.prefill(t, 0, 0.0, 1.0, seq_id=s))
    for step in range(12):
        last = {s: t[-1] for s, t in texts.items()}
        got = llm.forward_batch([DecodeRequest(seq_id=s, token_id=last[s] if step < 6 else FROM_LAST, pos=len(t) - 1) for s, t in texts.items()])
        for s, tok in zip(texts, got):
            texts[s].append(tok)
    for s, t in texts.items():
        want, bound = oracle(raw, folder, t)
        for i in range(len(t) - 13, len(t) - 1):
            assert float(want[i].max() - want[i, t[i + 1]]) <= 2 * bound


def test_generation_under_preemption_with_log_probabilities(folders):
    """Few pages: requests are sent back and recomputed.  Every generated token has its log probability, and what score() says of the same
    text agrees: both differ from the plain implementation's logits by the bound, a log probability from logits by twice their difference."""
    from blackwellllm_b200 import SamplingParams
    raw, _, _ = tiny.CONFIGS["llama"]
    folder = folders[("llama", "bfloat16")]
    llm = make(folder, page_size=8, num_pages=14, kv_dtype="int8", ctx=96)
    prompts = [tiny.prompt(n, raw["vocab_size"], 60 + n) for n in (20, 31, 12)]
    params = [SamplingParams(temperature=0.0, max_new_tokens=40, ignore_eos=True, logprobs=3),
              SamplingParams(temperature=0.8, max_new_tokens=40, ignore_eos=True, logprobs=0, repetition_penalty=1.3),
              SamplingParams(temperature=0.0, max_new_tokens=40, ignore_eos=True)]
    res = llm.generate(prompts, params)
    assert sum(r.preemptions for r in res) > 0 and res[2].logprobs is None
    for r, p in zip(res[:2], params):
        text = r.prompt_token_ids + r.token_ids
        want, bound = oracle(raw, folder, text)
        lp = torch.log_softmax(want, -1)
        scored = llm.score(text, top=3)
        assert [s.token_id for s in scored] == text[1:] and len(r.logprobs) == len(r.token_ids) == 40
        for i, s in enumerate(scored):
            assert abs(s.log_prob - float(lp[i, text[i + 1]])) <= 2 * bound and len(s.top) == 3
        for i, e in enumerate(r.logprobs):
            at = len(r.prompt_token_ids) - 1 + i
            assert e.token_id == text[at + 1] and len(e.top) == p.logprobs
            assert abs(e.log_prob - float(lp[at, e.token_id])) <= 2 * bound
            if p.temperature == 0.0:
                assert e.rank == 0 and e.top[0] == (e.token_id, pytest.approx(e.log_prob, abs=1e-6))
    assert llm.engine.cache.free_pages() == [14]


@pytest.mark.parametrize("name", ["llama", "partial"])
def test_log_probabilities_against_the_plain_distribution(folders, name):
    """float32: log probabilities and entropy of generated tokens, sampled ones under a repetition penalty among them, and of a scored text.
    A logit is off by at most ``bound``; a log probability by twice that.  Entropy is a mean of -ln p under p: it moves by twice the bound
    and by what the change of p, a factor of at most e^(2 bound), makes of every term."""
    from blackwellllm_b200 import SamplingParams
    raw, _, page = tiny.CONFIGS[name]
    folder = folders[(name, "float32")]
    W, V = load_plain_weights(folder), raw["vocab_size"]
    llm = make(folder, "float32", page_size=page)
    prompts = [tiny.prompt(n, V, 70 + n) for n in (5, 33)]
    params = [SamplingParams(temperature=0.0, max_new_tokens=12, ignore_eos=True, logprobs=5),
              SamplingParams(temperature=1.2, top_p=0.95, max_new_tokens=12, ignore_eos=True, logprobs=2, repetition_penalty=1.5)]
    for r, p in zip(llm.generate(prompts, params), params):
        text = r.prompt_token_ids + r.token_ids
        lg = plain_logits(raw, W, text)
        lp = torch.log_softmax(lg, -1)
        bound = tiny.TOL["float32"] * float(lg.abs().max()) + 1e-5
        entries = [(len(r.prompt_token_ids) - 1 + i, e, p.logprobs) for i, e in enumerate(r.logprobs)]
        assert len(entries) == 12
        entries += [(i, e, 4) for i, e in enumerate(llm.score(text, top=4))]
        for at, e, top in entries:
            row = lp[at]
            assert e.token_id == text[at + 1] and abs(e.log_prob - float(row[e.token_id])) <= 2 * bound
            entropy = float(-(row.exp() * row).sum())
            assert abs(e.entropy - entropy) <= 2 * bound + (math.exp(2 * bound) - 1) * (entropy + 2 * bound)
            before = int((row > row[e.token_id] + 4 * bound).sum()), int((row > row[e.token_id] - 4 * bound).sum())
            assert before[0] <= e.rank <= before[1]
            assert len(e.top) == top and len({t for t, _ in e.top}) == top
            best = torch.sort(row, descending=True).values
            for k, (t, v) in enumerate(e.top):
                assert abs(v - float(row[t])) <= 2 * bound and abs(v - float(best[k])) <= 2 * bound


def test_a_text_is_scored_beside_running_requests(folders):
    """Scoring takes a slot and pages for itself, gives them back, and leaves what others generate as it was."""
    from blackwellllm_b200 import EngineError, SamplingParams
    raw, _, page = tiny.CONFIGS["qwen"]
    V = raw["vocab_size"]
    llm = make(folders[("qwen", "bfloat16")], page_size=page, kv_dtype="int8", max_batch_tokens=24)
    params = SamplingParams(temperature=0.0, max_new_tokens=12, ignore_eos=True, logprobs=1)
    prompts = [tiny.prompt(n, V, 80 + n) for n in (11, 26)]
    alone = llm.generate(prompts, params)
    text = tiny.prompt(75, V, 3)
    whole = llm.score(text, top=2)
    rids = [llm.add_request(p, params) for p in prompts]
    done, rounds = {}, 0
    while llm.scheduler.has_work():
        for r in llm.step():
            done[r.request_id] = r
        rounds += 1
        if rounds % 3 == 0:
            assert llm.score(text, top=2) == whole
    assert [done[r].token_ids for r in rids] == [r.token_ids for r in alone]
    assert [[e.token_id for e in done[r].logprobs] for r in rids] == [r.token_ids for r in alone]
    assert llm.score([]) == [] and llm.score(text[:1]) == []
    for bad, top in (([1, V], 0), ([-1, 1], 0), ([1, 2], 33), ([1, 2], -1), ([1] * 257, 0)):
        with pytest.raises(EngineError):
            llm.score(bad, top)
    assert llm.engine.cache.free_pages() == [g.num_pages for g in llm.engine.cache.groups] and not llm.engine.cache.live


def test_half_the_bytes_hold_more_pages(folders):
    """Without a number of pages the pool takes a share of the free memory: over 8 bits at most the share of the plain one, with the pages
    that twice channels + 4 bytes a row make of it."""
    from blackwellllm_b200.engine.engine import Engine, EngineOptions
    raw, _, _ = tiny.CONFIGS["llama"]
    kw = dict(page_size=16, kv_fraction=1e-4, max_requests=2)
    plain = Engine.from_config(raw, options=EngineOptions(**kw)).cache.groups[0].num_pages
    quant = Engine.from_config(raw, options=EngineOptions(kv_dtype="int8", **kw)).cache.groups[0].num_pages
    hd = raw["head_dim"]
    assert quant / plain == pytest.approx(2 * hd / (hd + 4), rel=0.1)


def test_a_prompt_whose_attention_gave_up_is_an_error(folders):
    """The status set as a wait that gives up sets it: the step's rows are no numbers and its caller hears of it, in every call that takes
    prompts; afterwards all is as before."""
    from blackwellllm_b200 import EngineError, SamplingParams
    from blackwellllm_b200.kernels.build import load_library
    raw, _, page = tiny.CONFIGS["llama"]
    llm = make(folders[("llama", "bfloat16")], page_size=page, kv_dtype="int8")
    ids, params = tiny.prompt(50, raw["vocab_size"], 4), SamplingParams(temperature=0.0, max_new_tokens=6, ignore_eos=True)
    want, scored = llm.generate(ids, params)[0].token_ids, llm.score(ids)
    hd = llm.engine.cache.groups[0].request.head_dim
    give_up = load_library("attention_q8_tc", {"HEAD_DIM": hd}).bw_attention_q8_tc_give_up
    for call in (lambda: llm.generate(ids, params), lambda: llm.prefill(ids, 0, 0.0, 1.0), lambda: llm.score(ids)):
        assert give_up(39) == 0
        with pytest.raises(EngineError, match="gave up"):
            call()
    while llm.scheduler.has_work():
        for r in llm.step():
            assert r.token_ids == want
    assert llm.score(ids) == scored and llm.generate(ids, params)[0].token_ids == want
