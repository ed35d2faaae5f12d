"""The 8-bit cache and the log probabilities of generated tokens without a GPU: what options, models and the cache manager make of them."""
import contextlib
import ctypes

import pytest
import torch

import tiny
import tiny_fuvevik
import tiny_gafulix
import tiny_vubotar
import tiny_zanivik
import tiny_zigipel
import tiny_zogulorn
from blackwellllm_b200 import cli
from blackwellllm_b200.cache.manager import CacheManager
from blackwellllm_b200.config.registry import parse_config
from blackwellllm_b200.engine.engine import Engine, EngineError, EngineOptions, StepEntry
from blackwellllm_b200.kernels import ops
from blackwellllm_b200.kernels.build import load_library
from blackwellllm_b200.models.decoder import DecoderModel
from blackwellllm_b200.parts.base import BuildContext, FixedStateRequest, PagedKVRequest
from blackwellllm_b200.sampling.params import SamplingParams

CPU = torch.device("cpu")


@pytest.mark.parametrize("name", list(tiny.CONFIGS))
def test_the_dense_models_keep_their_keys_and_values_in_8_bits(name):
    cfg = parse_config(tiny.CONFIGS[name][0])
    plain = DecoderModel(cfg, BuildContext(CPU, torch.bfloat16)).cache_requests()
    model, _ = Engine._model(cfg, BuildContext(CPU, torch.bfloat16, quant_cache=True))
    quant = model.cache_requests()
    assert len(quant) == len(plain) > 0 and all(r.quantized for r in quant) and not any(r.quantized for r in plain)
    for a, b in zip(quant, plain):
        assert (a.num_kv_heads, a.head_dim, a.window) == (b.num_kv_heads, b.head_dim, b.window)
        assert a.page_bytes(16, 2) == 2 * 16 * a.num_kv_heads * (a.head_dim + 4)
        assert b.page_bytes(16, 2) == 2 * 16 * b.num_kv_heads * b.head_dim * 2


@pytest.mark.parametrize("module", [tiny_fuvevik, tiny_gafulix, tiny_vubotar, tiny_zanivik, tiny_zigipel, tiny_zogulorn])
def test_a_design_whose_layers_keep_something_else_is_refused_where_it_is_built(module):
    """Head norms, latent keys, gates, soft caps and the like have no form over 8 bits: an error, never a cache in the wrong type."""
    refused = 0
    for raw, _ in module.CONFIGS.values():
        cfg = parse_config(raw)
        try:
            model, _ = Engine._model(cfg, BuildContext(CPU, torch.bfloat16, quant_cache=True))
        except (EngineError, ops.KernelError) as e:
            refused += 1
            assert "8-bit cache" in str(e) or "kv_dtype" in str(e)
        else:
            assert all(r.quantized for e in model.cache_requests() for r in (e if isinstance(e, tuple) else (e,)) if isinstance(r, PagedKVRequest))
    assert refused


def test_options():
    cfg = parse_config(tiny.TINY_LLAMA)
    with pytest.raises(EngineError, match="kv_dtype must be"):
        Engine._build(cfg, EngineOptions(kv_dtype="int4"))
    with pytest.raises(EngineError, match="bfloat16"):
        Engine._build(cfg, EngineOptions(kv_dtype="int8", dtype="float32"))
    with pytest.raises(ops.KernelError, match="float32"):
        DecoderModel(cfg, BuildContext(CPU, torch.float32, quant_cache=True))
    ap = cli.build_parser()
    assert ap.parse_args([]).kv_dtype == "model" and ap.parse_args(["--kv-dtype", "int8"]).kv_dtype == "int8"
    with pytest.raises(SystemExit):
        ap.parse_args(["--kv-dtype", "int4"])


def test_head_sizes_and_groups_that_the_kernels_do_not_take():
    for hd, group in ((24, 1), (272, 1), (0, 1), (64, 17)):
        with pytest.raises(ops.KernelError, match="8-bit cache"):
            ops.check_quant_supported(hd, group)
    raw = dict(tiny.TINY_LLAMA, num_attention_heads=34, num_key_value_heads=2)
    with pytest.raises(ops.KernelError):
        DecoderModel(parse_config(raw), BuildContext(CPU, torch.bfloat16, quant_cache=True))


def test_operands_on_the_host_are_refused():
    """There is no CPU path: an error, and nothing is written."""
    pages = ops.QuantPages(torch.zeros(3, 2, 8, 16, dtype=torch.int8), torch.zeros(3, 2, 8, 16, dtype=torch.int8), torch.zeros(3, 2, 8), torch.zeros(3, 2, 8))
    table, one = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ops.KernelError):
        ops.quant_append(torch.ones(1, 6 * 16), one, one, table, pages, 2)
    with pytest.raises(ops.KernelError):
        ops.quant_read(pages, one, one, table)
    with pytest.raises(ops.KernelError):
        ops.token_log_probs(torch.zeros(1, 9), one)
    assert not pages.k.any() and not pages.v_scale.any()


def entry(lib, name, res=ctypes.c_int):
    fn = getattr(load_library(lib, {"HEAD_DIM": 64} if "attention" in lib else None), name)
    fn.restype = res
    return fn


def ints(*values):
    return (ctypes.c_int * len(values))(*values)


def test_what_the_entry_points_refuse_before_they_touch_the_device():
    """Sizes and segments that no kernel takes come back as error codes (-1: bad argument, -2: not supported)."""
    p, ll, f = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_float
    at = [p(1 << 20)] * 9       # never followed
    need = ll(0)
    deal = entry("attention_q8", "bw_attention_q8_deal")
    for lens, starts, nh, nkv, page in (((-1,), (0,), 4, 2, 16), ((1,), (-1,), 4, 2, 16), ((1,), (0x7fffffff,), 4, 2, 16), ((1,), (0,), 5, 2, 16),
                                        ((1,), (0,), 0, 2, 16), ((1,), (0,), 4, 0, 16), ((1,), (0,), 4, 2, 0)):
        assert deal(at[0], at[0], ints(*lens), ints(*starts), 1, nh, nkv, page, 0, 0, 4096, None, ctypes.byref(need), None) == -1
    room = entry("attention_q8_tc", "bw_attention_q8_tc_room", ll)
    for lens, starts, G, nkv in (((-1,), (0,), 4, 2), ((40,), (-1,), 4, 2), ((40,), (0x7fffffe0,), 4, 2), ((40,), (0,), 0, 2), ((40,), (0,), 4, 0)):
        assert room(ints(*lens), ints(*starts), 1, 16, G, nkv, 0, 0) == -1
    assert room(ints(0x7ffffff), ints(0), 1, 16, 16, 2, 0, 0) == -2
    attend = entry("attention_q8", "bw_attention_q8")
    for lens, starts, nh, nkv, page, pages, blocks in (((1,), (-5,), 4, 2, 16, 9, 9), ((-1,), (5,), 4, 2, 16, 9, 9), ((1,), (5,), 3, 2, 16, 9, 9),
                                                       ((1,), (5,), 4, 2, 0, 9, 9), ((1,), (5,), 4, 2, 16, 0, 9), ((1,), (5,), 4, 2, 16, 9, 0)):
        assert attend(*at, p(1 << 20), blocks, ints(*lens), ints(*starts), 1, nh, nkv, page, pages, 0, 0, 0, f(0.1), None, None, ll(0),
                      ctypes.byref(need), None, None) == -1
    assert attend(*at, p(1 << 20), 9, ints(1), ints(5), 1, 4, 2, 1 << 16, 1 << 16, 0, 0, 0, f(0.1), None, None, ll(0), ctypes.byref(need), None, None) == -2
    append = entry("quant_cache", "bw_quant_append")
    good = dict(planes=1, rd=0, nh=2, tokens=1, requests=1, blocks=1, page=16, pages=4, nkv=2, hd=64, type=0)
    for name, value, code in (("planes", 0, -1), ("rd", 3, -1), ("rd", 66, -1), ("rd", 8, -1), ("nh", -1, -1), ("tokens", -1, -1), ("requests", 0, -1),
                              ("blocks", 0, -1), ("page", 0, -1), ("pages", 0, -1), ("nkv", 0, -1), ("hd", 24, -1), ("hd", 272, -1),
                              ("tokens", 0x7fffffff, -2), ("type", 7, -2)):
        a = dict(good, **{name: value})
        assert append(at[0], a["type"], a["planes"], ll(0), None, a["rd"], 0, at[0], a["nh"], *at[:7], a["tokens"], a["requests"], a["blocks"], a["page"],
                      a["pages"], a["nkv"], a["hd"], 1, None) == code, (name, value)
    read = entry("quant_cache", "bw_quant_read")
    assert read(*at, 7, 1, 1, 1, 16, 4, 2, 64, None) == -2 and read(*at, 0, 1, 1, 1, 16, 4, 2, 40, None) == -1
    assert read(*at[:7], p((1 << 20) + 8), at[0], 0, 1, 1, 1, 16, 4, 2, 64, None) == -1
    probs = entry("token_probs", "bw_token_probs")
    for V, top, ld in ((0, 0, 8), (8, 9, 8), (8, 33, 8), (8, -1, 8), (8, 0, 7), ((1 << 30) + 1, 0, 1 << 31)):
        assert probs(*at[:7], 1, V, top, ll(ld), None) == -1
    assert probs(None, *at[:6], 1, 8, 0, ll(8), None) == -1 and probs(*at[:5], None, None, 1, 8, 1, ll(8), None) == -1


def test_pools():
    """Numbers and scales of a group lie in two tensors, each layer has its own part of both, and another group keeps its type."""
    a, b = PagedKVRequest(2, 16, None, quantized=True), PagedKVRequest(2, 16, None)
    cache = CacheManager([a, b, a], 8, 5, 2, dtype=torch.bfloat16, device=CPU)
    assert len(cache.groups) == 2 and [v.group for v in cache.views] == [0, 1, 0]
    one, plain, two = cache.views
    assert plain.quant is None and plain.k_pages.dtype == torch.bfloat16 and cache.groups[1].scales is None
    for v in (one, two):
        assert v.quant.k is v.k_pages and v.quant.v is v.v_pages
        for t in (v.quant.k, v.quant.v):
            assert t.dtype == torch.int8 and t.shape == (5, 2, 8, 16) and t.is_contiguous()
        for t in (v.quant.k_scale, v.quant.v_scale):
            assert t.dtype == torch.float32 and t.shape == (5, 2, 8) and t.is_contiguous()
    parts = [t for v in (one, two) for t in (v.quant.k, v.quant.v, v.quant.k_scale, v.quant.v_scale)]
    for i, t in enumerate(parts):
        t.fill_(i + 1)
    assert all(bool((t == i + 1).all()) for i, t in enumerate(parts))
    kept = CacheManager([a], 8, 5, 2, device=None)
    assert kept.views[0].quant is None and kept.views[0].k_pages is None


def test_how_many_log_probabilities_may_be_asked_for():
    assert SamplingParams().logprobs is None
    for n in (0, 1, 32):
        assert SamplingParams(logprobs=n).logprobs == n
    for n in (-1, 33):
        with pytest.raises(ValueError, match="logprobs"):
            SamplingParams(logprobs=n)
    with pytest.raises(TypeError):
        SamplingParams(logprobs=2.5)


class PagesOnly:
    """A stand-in model that owns pages and computes nothing."""

    def __init__(self, vocab):
        self.vocab, self.blocks = vocab, []

    def cache_requests(self):
        return [PagedKVRequest(2, 16, None), PagedKVRequest(2, 16, 16), None]

    def forward(self, batch, views):
        return torch.zeros((len(batch.logit_rows), self.vocab), dtype=torch.float32)


def test_cached_rows_are_read_by_position(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    cfg = parse_config(tiny.TINY_LLAMA)
    eng = Engine(cfg, PagesOnly(cfg.vocab_size), EngineOptions(dtype="float32", page_size=8, num_pages=12, max_requests=3,
                                                               cuda_graphs=False, device="cpu"))
    eng.step([StepEntry("b", [1] * 3, []), StepEntry("a", [1] * 29, [])])
    for v in eng.cache.views[:2]:
        v.k_pages.copy_(torch.randn(v.k_pages.shape))
        v.v_pages.copy_(torch.randn(v.v_pages.shape))
    for layer in (0, 1):
        v, table = eng.cache.views[layer], eng.cache.block_table("a", layer)
        k, val = eng.cached_kv("a", layer)
        assert k.shape == val.shape == (29, 2, 16)
        for p in range(29):
            page = table[p // 8]
            assert torch.equal(k[p], v.k_pages[page, :, p % 8] if page >= 0 else torch.zeros(2, 16))
            assert torch.equal(val[p], v.v_pages[page, :, p % 8] if page >= 0 else torch.zeros(2, 16))
        some = eng.cached_kv("a", layer, 7, 18)
        assert torch.equal(some[0], k[7:18]) and torch.equal(some[1], val[7:18])
    assert -1 in eng.cache.block_table("a", 1)
    assert eng.cached_kv("b", 0, 3)[0].shape == (0, 2, 16)
    with pytest.raises(EngineError, match="not live"):
        eng.cached_kv("c", 0)
    for layer in (-1, 2, 3):
        with pytest.raises(EngineError, match="owns no pages"):
            eng.cached_kv("a", layer)
    for start, stop in ((-1, 2), (5, 4), (0, 30)):
        with pytest.raises(EngineError, match="positions"):
            eng.cached_kv("a", 0, start, stop)


def test_cached_rows_end_before_a_token_that_is_only_reserved(monkeypatch):
    """A step prepared ahead makes its requests longer by a token that nobody has computed: no row of it is read until the step is
    launched, and none once it is cancelled, rolled back or its request is freed."""
    class Graph:
        def replay(self):
            pass

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", lambda graph: contextlib.nullcontext())
    cfg = parse_config(tiny.TINY_LLAMA)
    eng = Engine(cfg, PagesOnly(cfg.vocab_size), EngineOptions(dtype="float32", page_size=8, num_pages=12, max_requests=3, device="cpu", graph_after=1))

    def rows():
        return [eng.cached_kv(r, layer)[0].shape[0] for r in ("a", "b") for layer in (0, 1)]

    eng.step([StepEntry("a", [1] * 5, []), StepEntry("b", [1] * 8, [])])
    eng.step([StepEntry("a", [1], [0]), StepEntry("b", [1], [0])])       # recorded: from here on steps are prepared ahead
    assert rows() == [6, 6, 9, 9]
    prep = eng.prepare_decode_ahead(["a", "b"])
    assert prep is not None and [eng.cache.length(r) for r in ("a", "b")] == [7, 10]
    assert rows() == [6, 6, 9, 9]
    with pytest.raises(EngineError, match="positions"):
        eng.cached_kv("a", 0, 0, 7)
    eng.launch_prepared(prep, [1, 2])
    assert rows() == [7, 7, 10, 10]
    prep = eng.prepare_decode_ahead(["a", "b"])
    assert rows() == [7, 7, 10, 10]
    eng.cancel_prepared(prep)
    assert rows() == [7, 7, 10, 10] and [eng.cache.length(r) for r in ("a", "b")] == [7, 10]
    # rolled back to a position before it, or freed and begun again, while the step is still prepared
    eng.prepare_decode_ahead(["a", "b"])
    eng.cache.truncate("a", 4)
    eng.end_request("b")
    eng.step([StepEntry("b", [1] * 3, [])])
    assert rows() == [4, 4, 3, 3]


@pytest.mark.parametrize("lens", [(1 << 24,), (1 << 23, 1 << 23), (1, 1 << 24)])
def test_more_rows_of_queries_than_32_bits_count_are_refused(lens):
    """2^24 tokens of 256 heads are 2^32 rows: places in the queries and outputs would wrap."""
    room = entry("attention_q8_tc", "bw_attention_q8_tc_room", ctypes.c_longlong)
    starts = [0] * len(lens)
    assert room(ints(*lens), ints(*starts), len(lens), 16, 16, 16, 0, 0) == -2
    few = [n >> 4 for n in lens]
    assert room(ints(*few), ints(*starts), len(lens), 16, 16, 16, 0, 0) > 0


def scratch_of(lens, nkv, nh, bound=0):
    """Floats of scratch that a call asks for (nothing is launched: it has none), for requests of one token each at these lengths."""
    attend = entry("attention_q8", "bw_attention_q8")
    p, ll, at = ctypes.c_void_p, ctypes.c_longlong, [ctypes.c_void_p(1 << 20)] * 9
    need, R = ll(0), len(lens)
    code = attend(*at, p(1 << 20), 9, ints(*[1] * R), ints(*[n - 1 for n in lens]), R, nh, nkv, 16, 1 << 10, 0, 0, bound, ctypes.c_float(0.1), None, None,
                  ll(0), ctypes.byref(need), None, None)
    assert code == -11
    return need.value


def test_a_long_request_beside_many_short_ones_is_divided():
    """However many requests there are, one that is far longer than its share of the GPU is several blocks' work (and is joined from scratch): at the
    lengths of the call, and in a step that is captured for lengths to come."""
    deal = entry("attention_q8", "bw_attention_q8_deal")
    for count in (40, 100, 200, 700):
        assert scratch_of([131072] + [500] * (count - 1), 8, 32) > 0
        need = ctypes.c_longlong(0)
        assert deal(None, None, ints(*[1] * count), ints(*[0] * count), count, 32, 8, 16, 0, 0, 131072, None, ctypes.byref(need), None) == 0
        assert need.value >= 4 * count


def test_scratch_is_a_matter_of_the_slices_that_there_are():
    """Not of as many for each request as the longest has: a slice is 16 rows of 64 channels and two numbers, and as many as four times the blocks
    of a GPU (at most 32 an SM) beside one a request and kv head are room enough for any step."""
    for nkv, nh in ((1, 8), (2, 8), (8, 32)):
        for count in (20, 51, 256):
            for longest in (30000, 131072, 1000000):
                for lens in ([longest] + [300] * (count - 1), [300] * (count - 1) + [longest], [longest >> (i % 12) for i in range(count)]):
                    need = scratch_of(lens, nkv, nh)
                    assert need <= 16 * 66 * 4 * (148 * 32 + count * nkv) + 6 * (148 * 32 + count)


def test_cached_rows_of_a_layer_that_owns_a_state_beside_its_pages(monkeypatch):
    class PagesAndState(PagesOnly):
        def cache_requests(self):
            pages, state = PagedKVRequest(2, 16, None), FixedStateRequest((3,), torch.float32)
            return [(pages, state), (state, pages), (state,), (pages, pages)]

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    cfg = parse_config(tiny.TINY_LLAMA)
    eng = Engine(cfg, PagesAndState(cfg.vocab_size), EngineOptions(dtype="float32", page_size=8, num_pages=12, max_requests=3,
                                                                   cuda_graphs=False, device="cpu"))
    eng.step([StepEntry("a", [1] * 11, [])])
    table = eng.cache.block_table("a", 0)
    for layer, place in ((0, 0), (1, 1)):
        v = eng.cache.views[layer][place]
        v.k_pages.copy_(torch.randn(v.k_pages.shape))
        k, val = eng.cached_kv("a", layer)
        assert k.shape == val.shape == (11, 2, 16)
        assert all(torch.equal(k[p], v.k_pages[table[p // 8], :, p % 8]) for p in range(11)) and not val.any()
    with pytest.raises(EngineError, match="owns no pages"):
        eng.cached_kv("a", 2)
    with pytest.raises(EngineError, match="more than one"):
        eng.cached_kv("a", 3)


class Rule(PagesOnly):
    """After a token t at position p comes (t + p) % vocab, over a cache in 8 bits that nobody writes."""

    def cache_requests(self):
        return [PagedKVRequest(2, 16, None, quantized=True)]

    def forward(self, batch, views):
        out = torch.zeros((len(batch.logit_rows), self.vocab), dtype=torch.float32)
        for i, t in enumerate(batch.logit_rows.tolist()):
            out[i, (int(batch.token_ids[t]) + int(batch.positions[t])) % self.vocab] = 1.0
        return out


def test_a_prompt_whose_attention_gave_up_is_an_error_and_computed_again(monkeypatch):
    """The status is looked at with the tokens of a step that had a portion of a prompt, never for steps of single tokens; the requests of such
    a step wait again, and what they generate then is what they would have."""
    import dataclasses

    from blackwellllm_b200 import BlackwellEngine, InferenceConfig
    from blackwellllm_b200.engine import llm as llm_module

    class Best:
        def __init__(self, device):
            pass

        def sample_async(self, logits, *a):
            return logits.argmax(dim=1)

        def sample(self, logits, *a):
            return logits.argmax(dim=1).tolist()

    def from_config(raw, seed=0, std=0.02, options=None):
        cfg = parse_config(raw)
        return Engine(cfg, Rule(cfg.vocab_size), dataclasses.replace(options, device="cpu", cuda_graphs=False))

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(llm_module.Engine, "from_config", staticmethod(from_config))
    monkeypatch.setattr(llm_module, "Sampler", Best)
    answers, asked = [], []
    monkeypatch.setattr(ops, "attention_q8_status", lambda: asked.append(1) or (answers.pop(0) if answers else 0))
    llm = BlackwellEngine(None, InferenceConfig(max_context_length=96, max_batch_size=3), config=tiny.CONFIGS["llama"][0], page_size=8, max_batch_tokens=16)
    prompts = [[3, 4, 5], list(range(10, 40)), [9, 8]]
    params = SamplingParams(temperature=0.0, max_new_tokens=5, ignore_eos=True)
    want = [r.token_ids for r in llm.generate(prompts, params)]
    portions = len(asked)
    assert 0 < portions < 6
    for bad in range(portions):
        answers[:] = [0] * bad + [39]
        rids = [llm.add_request(p, params) for p in prompts]
        done, failed = {}, 0
        while llm.scheduler.has_work():
            try:
                done.update((r.request_id, r.token_ids) for r in llm.step())
            except EngineError as e:
                assert "gave up" in str(e)
                failed += 1
        assert failed == 1 and [done[r] for r in rids] == want
        llm.engine.cache.check_invariants()
    asked.clear()
    first = llm.prefill([1, 2, 3], 0, 0.0, 1.0)
    assert len(asked) == 1 and llm.forward(first, 3, 0.0, 1.0) == (first + 3) % llm.vocab_size and len(asked) == 1
    answers[:] = [39]
    with pytest.raises(EngineError, match="gave up"):
        llm.prefill([4, 5, 6], 4, 0.0, 1.0)
    assert llm.engine.cache.length(("seq", 0)) == 4 and llm.prefill([4, 5, 6], 4, 0.0, 1.0) == (6 + 6) % llm.vocab_size
    assert llm.prefill([1, 2, 3], 0, 0.0, 1.0) == first
