"""The 8-bit cache on the GPU: rows written and read back, and attention over them, against a plain 64-bit implementation."""
import math
import random

import pytest
import torch

from blackwellllm_b200.engine.batch import StepBatch
from blackwellllm_b200.kernels import ops
from plain_quant import attention, attention_bound, quantize, rotate, row_index

pytestmark = pytest.mark.gpu


def _cuda(t, dtype=None):
    return t.to("cuda", dtype) if dtype else t.cuda()


class Case:
    """Requests with segments (tokens, first position, length) over a pool whose pages lie in random order."""

    def __init__(self, segments, nkv, hd, page, seed, gone=(), extra=3):
        g = torch.Generator().manual_seed(seed)
        self.segments, self.nkv, self.hd, self.page = segments, nkv, hd, page
        R = len(segments)
        blocks = [-(-total // page) for _, _, total in segments]
        count = sum(blocks)
        self.num_pages = count + extra
        order = torch.randperm(self.num_pages, generator=g)[:count].tolist()
        self.table = torch.full((R, max(blocks + [1]) + 1), -1, dtype=torch.int32)
        for r, n in enumerate(blocks):
            for b in range(n):
                self.table[r, b] = order.pop()
        for r, b in gone:
            self.table[r, b] = -1
        lens = torch.tensor([n for n, _, _ in segments])
        self.cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
        self.T = int(self.cu[-1])
        self.req = torch.repeat_interleave(torch.arange(R), lens)
        self.start = torch.tensor([a for _, a, _ in segments])
        self.total = torch.tensor([t for _, _, t in segments])
        self.pos = torch.arange(self.T) - self.cu[:-1][self.req] + self.start[self.req]
        self.gen = g

    def fill(self, loud=True):
        """A pool full of rows: what the segments' requests hold, and leftovers."""
        shape = (self.num_pages, self.nkv, self.page, self.hd)
        got = []
        for which in range(2):
            x = torch.randn(shape, generator=self.gen, dtype=torch.float64)
            if loud and which == 0:
                x[..., ::7] *= 5.0
            codes, scale = quantize(x * torch.exp(torch.randn(shape[:3] + (1,), generator=self.gen, dtype=torch.float64)))
            got += [codes.to(torch.int8), scale.float()]
        self.k, self.k_scale, self.v, self.v_scale = got
        return self

    def empty(self):
        shape = (self.num_pages, self.nkv, self.page, self.hd)
        self.k, self.v = torch.full(shape, 77, dtype=torch.int8), torch.full(shape, -77, dtype=torch.int8)
        self.k_scale, self.v_scale = torch.full(shape[:3], 3.0), torch.full(shape[:3], 5.0)
        return self

    def pages(self):
        return ops.QuantPages(self.k.cuda(), self.v.cuda(), self.k_scale.cuda(), self.v_scale.cuda())

    def batch(self, bound=None):
        i32 = torch.int32
        z = self.start.to("cuda", i32)
        return StepBatch(T=self.T, R=len(self.segments), token_ids=self.pos.to("cuda", i32), positions=self.pos.to("cuda", i32),
                         req_of_token=self.req.to("cuda", i32), cu_q=self.cu.to("cuda", i32), q_start=z, kv_len=self.total.to("cuda", i32),
                         state_slot=z, logit_rows=z, block_tables={0: self.table.cuda()}, h_q_start=self.start.tolist(),
                         h_q_len=[n for n, _, _ in self.segments], h_kv_len=self.total.tolist(), static_bound=bound)

    def check_attention(self, nh, window=0, chunk=0, sink=None, scale=None, bound=None, pages=None):
        q = torch.randn(self.T, nh * self.hd, generator=self.gen).to(torch.bfloat16)
        scale = self.hd ** -0.5 if scale is None else scale
        b = self.batch(bound)
        got = ops.quant_attention(q.cuda(), pages or self.pages(), b, b.block_tables[0], nh, scale, window or None, chunk or None,
                                  None if sink is None else sink.cuda())
        e = attention(q.view(self.T, nh, self.hd), self.k, self.v, self.k_scale, self.v_scale, self.cu, self.start, self.total, self.table, scale,
                      window, chunk, sink)
        want = e.out
        lens = torch.tensor([n for n, _, _ in self.segments])
        wide = (lens * (nh // self.nkv) > ops.QUANT_FEW_ROWS)[self.req]
        tol = attention_bound(e, self.hd, wide)
        got = got.cpu().double().view_as(want)
        assert ops.attention_q8_status() == 0
        assert torch.isfinite(got).all()
        over = ((got - want).abs() / tol).max().item()
        assert over <= 1.0, f"error {over:.2f} times the bound"
        # the bound of a row supposes that all roundings of its scores go the same way; together the rows are off by what independent ones
        # make: the result's 2^-8 / sqrt(12) of it and, of what is averaged, the weights' and in wide rows the values' and the scores' (2^-11
        # of a score's terms each); a quarter more than the first
        assert (got - want).norm() <= 1.25 * 2.0 ** -7 / math.sqrt(12) * want.norm() + 1e-30
        return got


# ------------------------------------------------------------------------------------------------ writing and reading back
@pytest.mark.parametrize("hd,rd,page", [(128, 128, 16), (64, 64, 8), (64, 32, 16), (80, 80, 24), (256, 64, 16), (16, 16, 1), (96, 12, 5),
                                        (128, 0, 64), (144, 6, 16)])
@pytest.mark.parametrize("source", ["float32", "bfloat16", "planes", "paired"])
def test_append_then_read(hd, rd, page, source):
    nh, nkv = 6, 2
    c = Case([(5, 3, 8), (1, 40, 41), (0, 0, 1), (17, 0, 17)], nkv, hd, page, seed=hd * 100 + rd + page, gone=[(0, 4 // page)]).empty()
    width = (nh + 2 * nkv) * hd
    x = torch.randn(c.T, width, generator=c.gen)
    x[:, ::11] *= 9.0
    planes = None
    if source == "bfloat16":
        x = x.to(torch.bfloat16).float()
    if source == "planes":
        planes = torch.randn(3, c.T, width, generator=c.gen)
        x = (planes[0] + planes[1]) + planes[2]
    angle = torch.rand(c.T, rd // 2, generator=c.gen, dtype=torch.float64) * 6
    turns = torch.cat([angle.cos(), angle.sin()], dim=1).float() if rd else None
    pages, table = c.pages(), c.table.cuda()
    pos, req = _cuda(c.pos, torch.int32), _cuda(c.req, torch.int32)
    fed = planes.cuda() if planes is not None else x.cuda().to(torch.bfloat16) if source == "bfloat16" else x.cuda()
    q = ops.quant_append(fed, pos, req, table, pages, nh, table=None if turns is None else turns.cuda(), paired=source == "paired")
    heads = x.double().view(c.T, nh + 2 * nkv, hd)
    cos, sin = (turns.double().chunk(2, dim=1) if rd else (torch.zeros(c.T, 0), torch.zeros(c.T, 0)))
    turned = rotate(heads[:, :nh + nkv], cos, sin, paired=source == "paired")
    # a rotated channel is two products and a sum in float32: 2^-22 of the magnitudes; then one rounding to bfloat16
    size = rotate(heads[:, :nh + nkv].abs(), cos.abs(), -sin.abs(), paired=source == "paired").abs() + turned.abs()
    want_q = turned[:, :nh]
    err = (q.cpu().double().view_as(want_q) - want_q).abs()
    assert (err <= 2.0 ** -8 * want_q.abs() + 2.0 ** -21 * size[:, :nh]).all()
    page_of, slot = row_index(c.pos, c.req, c.table, page)
    held = page_of >= 0
    assert not held.all() and held.any()
    for name, rows, rough in (("k", turned[:, nh:], size[:, nh:]), ("v", heads[:, nh + nkv:], heads[:, nh + nkv:].abs())):
        codes, scale = getattr(pages, name).cpu(), getattr(pages, name + "_scale").cpu().double()
        _, want_s = quantize(rows)
        got_s = scale[page_of[held], :, slot[held]]
        # the largest magnitude is off by what the rotation is off, the division by half a step
        slack = 2.0 ** -21 * rough.amax(-1)
        assert ((got_s - want_s[held]).abs() <= 2.0 ** -24 * want_s[held] + slack[held] / 127).all()
        got = codes[page_of[held], :, slot[held]].double() * got_s[..., None]
        # a number is within half a scale of the value; the factor, the product and the scale are each rounded (127 steps of 2^-24, in scales)
        assert ((got - rows[held]).abs() <= 0.5 * (1 + 2.0 ** -14) * got_s[..., None] + 2 * slack[held][..., None]).all()
        # what no token of the step owns is as it was
        mark = torch.ones(codes.shape[0], codes.shape[2], dtype=torch.bool)
        mark[page_of[held], slot[held]] = False
        left = codes.transpose(1, 2)[mark]
        assert (left == (77 if name == "k" else -77)).all()
        assert (scale.transpose(1, 2)[mark] == (3.0 if name == "k" else 5.0)).all()
    # read back: the number times its scale, one rounding
    for dtype, u in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8)):
        for got, name in zip(ops.quant_read(pages, pos, req, table, dtype), ("k", "v")):
            codes, scale = getattr(pages, name).cpu().double(), getattr(pages, name + "_scale").cpu().double()
            want = torch.zeros(c.T, nkv, hd, dtype=torch.float64)
            want[held] = codes[page_of[held], :, slot[held]] * scale[page_of[held], :, slot[held]][..., None]
            # (float32: the product itself is rounded once; bfloat16: that and the rounding to it)
            assert ((got.cpu().double() - want).abs() <= (u + 2.0 ** -24) * want.abs()).all()


def test_append_without_writing():
    c = Case([(3, 0, 3)], 2, 64, 16, seed=1).empty()
    pages = c.pages()
    x = torch.randn(3, (4 + 4) * 64, generator=c.gen).cuda()
    q = ops.quant_append(x, _cuda(c.pos, torch.int32), _cuda(c.req, torch.int32), c.table.cuda(), pages, 4, append=False)
    assert torch.equal(q, x[:, :256].to(torch.bfloat16))
    assert (pages.k == 77).all() and (pages.v == -77).all() and (pages.k_scale == 3).all() and (pages.v_scale == 5).all()


def test_rows_at_the_ends_of_the_range():
    """Zeros, tiny and huge rows, infinities and NaN: nothing overflows, and what is no number stays none."""
    hd, nh, nkv = 64, 1, 1
    x = torch.ones(8, hd)
    x[0] = 0.0
    x[1] = 1e-40
    x[2] = 2.0 ** -109
    x[3] = 3.3e38
    x[4, 5] = math.inf
    x[5, 63] = math.nan
    x[6] = -0.0
    x[7, 1:] = 1e-30
    c = Case([(8, 0, 8)], nkv, hd, 4, seed=2).empty()
    pages = c.pages()
    rows = torch.cat([torch.zeros(8, hd), x, x.flip(0)], dim=1).cuda()
    pos, req, table = _cuda(c.pos, torch.int32), _cuda(c.req, torch.int32), c.table.cuda()
    ops.quant_append(rows, pos, req, table, pages, nh)
    k, v = (t.cpu()[:, 0] for t in ops.quant_read(pages, pos, req, table, torch.float32))
    for got, want in ((k, x), (v, x.flip(0))):
        for a, b in zip(got, want):
            if not torch.isfinite(b).all():
                assert torch.isnan(a).all()
            else:
                most = b.abs().max().item()
                # (tiny rows are zeros; else half a scale, and the product's rounding)
                tol = 2.0 ** -110 if most < 2.0 ** -110 else most / 127 * 0.5 * (1 + 2.0 ** -20)
                assert torch.isfinite(a).all() and (a.double() - b.double()).abs().max().item() <= tol


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("hd", [128, 64, 80, 256, 16, 96])
@pytest.mark.parametrize("nh,nkv,page", [(8, 2, 16), (7, 1, 8), (16, 1, 24), (3, 3, 64), (10, 2, 1)])
def test_attention_few_queries(hd, nh, nkv, page):
    segs = [(1, 0, 1), (1, 15, 16), (1, 63, 64), (1, 64, 65), (1, 300, 301), (0, 5, 5), (2 if nh // nkv <= 8 else 1, 130, 132 if nh // nkv <= 8 else 131)]
    Case(segs, nkv, hd, page, seed=hd + nh + page).fill().check_attention(nh)


@pytest.mark.parametrize("hd", [128, 64, 80, 256, 192, 16, 48, 96, 144, 208])
@pytest.mark.parametrize("nh,nkv,page", [(8, 2, 16), (7, 1, 8), (16, 1, 24), (4, 4, 64)])
def test_attention_portions(hd, nh, nkv, page):
    segs = [(37, 0, 37), (1, 70, 71), (19, 111, 130), (130, 5, 135), (3, 200, 203)]
    Case(segs, nkv, hd, page, seed=hd * 3 + nh + page).fill().check_attention(nh)


@pytest.mark.parametrize("window,chunk", [(1, 0), (17, 0), (64, 0), (100, 0), (0, 32), (50, 64), (0, 1)])
def test_attention_windows_and_chunks(window, chunk):
    segs = [(1, 299, 300), (40, 90, 130), (2, 63, 65), (25, 0, 25)]
    c = Case(segs, 2, 64, 16, seed=window * 7 + chunk).fill()
    c.check_attention(6, window, chunk)
    c.check_attention(6, window, chunk, bound=512)


def test_attention_sink():
    c = Case([(1, 99, 100), (30, 10, 40), (1, 0, 1)], 2, 128, 16, seed=5).fill()
    c.check_attention(8, sink=torch.linspace(-3, 6, 8))


@pytest.mark.parametrize("count", [33, 40])
def test_attention_more_portions_than_one_launch_takes(count):
    Case([(18 + i % 3, i, 18 + i % 3 + i) for i in range(count)], 1, 64, 16, seed=count).fill().check_attention(2)


@pytest.mark.parametrize("keys", [700, 5001, 30001])
def test_attention_slices_are_joined_in_order(keys):
    """One request, long: many slices, joined in a cluster or through memory; the same inputs give the same bits."""
    c = Case([(1, keys - 1, keys)], 1, 128, 16, seed=keys).fill()
    b, pages = c.batch(), c.pages()
    q = torch.randn(1, 4 * 128, generator=c.gen).to(torch.bfloat16).cuda()
    outs = [ops.quant_attention(q, pages, b, b.block_tables[0], 4, 0.088) for _ in range(5)]
    assert all(torch.equal(o, outs[0]) for o in outs)
    c.check_attention(4)


def test_attention_pages_that_are_gone():
    """Keys whose pages are not held are not seen; a row that sees none is zeros, in both kernels."""
    c = Case([(1, 40, 41), (20, 12, 32), (1, 20, 21), (18, 0, 18)], 2, 64, 16, seed=11,
             gone=[(0, 1), (1, 0), (2, 0), (2, 1), (3, 0), (3, 1)]).fill()
    got = c.check_attention(6)
    # (positions 12 to 15 of the second request see its first page alone, which is gone)
    empty = torch.zeros(c.T, dtype=torch.bool)
    empty[1:5] = empty[21:] = True
    assert (got[empty] == 0).all() and (got[~empty] != 0).any(-1).all()


def test_attention_leaves_out_what_is_no_number_where_it_is_not_seen():
    """Scales that are NaN behind a request's last token, in other requests' pages and in a later token of the same tile."""
    c = Case([(1, 20, 21), (30, 0, 30)], 1, 64, 16, seed=13).fill()
    page = c.page
    free = [p for p in range(c.num_pages) if p not in c.table.tolist()[0] + c.table.tolist()[1]]
    c.k_scale[free], c.v_scale[free] = math.nan, math.nan
    for r, total in ((0, 21), (1, 30)):
        last = int(c.table[r, (total - 1) // page])
        c.k_scale[last, :, total % page:] = math.nan
        c.v_scale[last, :, total % page:] = math.inf
    c.check_attention(4)
    # a key of position 25 is no number: the tokens before it do not see that, the ones from it on do
    p25 = int(c.table[1, 25 // page])
    c.k_scale[p25, :, 25 % page] = math.nan
    c.v_scale[p25, :, 25 % page] = math.nan
    b = c.batch()
    q = torch.randn(c.T, 4 * 64, generator=c.gen).to(torch.bfloat16).cuda()
    got = ops.quant_attention(q, c.pages(), b, b.block_tables[0], 4, 0.125).float()
    assert torch.isfinite(got[:26]).all() and torch.isnan(got[26:]).all()


def test_attention_in_a_graph_of_any_length():
    """A captured decode step replays with other lengths, on the bound that it was captured for."""
    c = Case([(1, 700, 701), (1, 3, 4), (1, 64, 65)], 2, 128, 16, seed=17).fill()
    b = c.batch(bound=1024)
    pages = c.pages()
    q = torch.zeros(c.T, 8 * 128, dtype=torch.bfloat16, device="cuda")
    ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.088)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.088)
    for starts in ([700, 3, 64], [0, 250, 1], [63, 64, 63]):
        starts = [min(s, int(t) - 1) for s, t in zip(starts, c.total)]
        b.q_start.copy_(torch.tensor(starts)); b.kv_len.copy_(torch.tensor(starts) + 1)
        fresh = torch.randn(c.T, 8 * 128, generator=c.gen).to(torch.bfloat16)
        q.copy_(fresh)
        graph.replay()
        e = attention(fresh.view(3, 8, 128), c.k, c.v, c.k_scale, c.v_scale, c.cu, starts, [s + 1 for s in starts], c.table, 0.088)
        assert ((out.cpu().double().view_as(e.out) - e.out).abs() <= attention_bound(e, 128)).all()


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("count,nkv,group,window,bound", [(70, 1, 4, 0, 2048), (33, 2, 6, 300, 2048), (9, 2, 16, 0, 2048), (40, 1, 8, 0, 256)])
def test_attention_in_a_graph_of_many_lengths(count, nkv, group, window, bound, shared):
    """A captured step deals its blocks out by the lengths of the replay: many requests, one or two tokens or none each, short and long ones
    (longer than the bound, too: such a request gets longer slices)."""
    longest = 1500
    g = torch.Generator().manual_seed(count)
    lens = torch.randint(0, 3 if 2 * group <= 16 else 2, (count,), generator=g)
    lens[:3] = 1
    c = Case([(int(n), longest - int(n), longest) for n in lens], nkv, 64, 16, seed=count).fill()
    b, pages, nh = c.batch(bound), c.pages(), nkv * group
    q = torch.zeros(c.T, nh * 64, dtype=torch.bfloat16, device="cuda")
    ops.quant_attention(q, pages, b, b.block_tables[0], nh, 0.125, window or None)
    ops.quant_attention_deal(b, nh, nkv, 64, 16, window or None)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dealt = ops.quant_attention_deal(b, nh, nkv, 64, 16, window or None) if shared else None
        out, again = (ops.quant_attention(q, pages, b, b.block_tables[0], nh, 0.125, window or None, dealt=dealt) for _ in range(2))
    for step in range(4):
        ends = torch.randint(2, 60, (count,), generator=g)
        if step == 1:
            ends[1], ends[-1] = longest, 1100
        elif step == 2:
            ends[:] = 900
        elif step == 3:
            ends[:] = 2
        starts = ends - lens
        b.q_start.copy_(starts); b.kv_len.copy_(ends)
        fresh = torch.randn(c.T, nh * 64, generator=c.gen).to(torch.bfloat16)
        q.copy_(fresh)
        out.fill_(float("nan")); again.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, again)
        e = attention(fresh.view(-1, nh, 64), c.k, c.v, c.k_scale, c.v_scale, c.cu, starts.tolist(), ends.tolist(), c.table, 0.125, window)
        assert ((out.cpu().double().view_as(e.out) - e.out).abs() <= attention_bound(e, 64)).all()


def test_a_division_goes_with_its_step():
    """How keys are divided is not taken from another step or for other sizes; a step whose lengths the host knows has none."""
    c = Case([(1, 700, 701)] * 3, 2, 64, 16, seed=1).fill()
    b, other, pages = c.batch(4096), c.batch(4096), c.pages()
    q = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device="cuda")
    assert ops.quant_attention_deal(c.batch(), 8, 2, 64, 16) is None
    dealt = ops.quant_attention_deal(b, 8, 2, 64, 16)
    assert dealt is not None
    ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.125, dealt=dealt)
    for batch, nh, window in ((other, 8, None), (b, 4, None), (b, 8, 128)):
        with pytest.raises(ops.KernelError, match="another step"):
            ops.quant_attention(q[:, :nh * 64].contiguous(), pages, batch, batch.block_tables[0], nh, 0.125, window, dealt=dealt)
    b.h_q_len = [1, 1, 0]
    with pytest.raises(ops.KernelError):
        ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.125, dealt=dealt)
    with pytest.raises(ops.KernelError):
        ops.quant_attention_deal(other, 7, 2, 64, 16)


def test_a_scale_that_is_not_positive():
    c = Case([(1, 3, 4), (20, 0, 20)], 2, 64, 16, seed=1).fill()
    b, pages = c.batch(), c.pages()
    q = torch.zeros(21, 4 * 64, dtype=torch.bfloat16, device="cuda")
    for scale in (0.0, -0.125, math.nan):
        with pytest.raises(ops.KernelError, match="positive"):
            ops.quant_attention(q, pages, b, b.block_tables[0], 4, scale)


def test_refusals():
    c = Case([(1, 3, 4)], 2, 64, 16, seed=1).fill()
    pages, b = c.pages(), c.batch()
    table = b.block_tables[0]
    q = torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ops.KernelError):
        ops.quant_attention(q.float(), pages, b, table, 4, 0.1)
    with pytest.raises(ops.KernelError):
        ops.quant_attention(q, pages, b, table, 3, 0.1)
    with pytest.raises(ops.KernelError):
        ops.quant_attention(torch.zeros(2, 4 * 64, dtype=torch.bfloat16, device="cuda"), pages, b, table, 4, 0.1)
    with pytest.raises(ops.KernelError):
        ops.quant_attention(q, ops.QuantPages(pages.k, pages.v, pages.k_scale[:, :1], pages.v_scale), b, table, 4, 0.1)
    with pytest.raises(ops.KernelError):
        ops.quant_attention(q, ops.QuantPages(pages.k.float(), pages.v, pages.k_scale, pages.v_scale), b, table, 4, 0.1)
    with pytest.raises(ops.KernelError):
        ops.quant_attention(q, pages, b, table, 4, 0.1, sink=torch.zeros(3, device="cuda"))
    with pytest.raises(ops.KernelError):      # 34 query heads to a kv head
        ops.quant_attention(torch.zeros(1, 34 * 64, dtype=torch.bfloat16, device="cuda"), pages, b, table, 34, 0.1)
    x = torch.zeros(1, 8 * 64, device="cuda")
    with pytest.raises(ops.KernelError):
        ops.quant_append(x[:, :-1].contiguous(), b.positions, b.req_of_token, table, pages, 4)
    with pytest.raises(ops.KernelError):
        ops.quant_append(x, b.positions, b.req_of_token, table, pages, 4, table=torch.zeros(1, 63, device="cuda"))
    with pytest.raises(ops.KernelError):
        ops.quant_append(x.half(), b.positions, b.req_of_token, table, pages, 4)
    with pytest.raises(ops.KernelError):
        ops.quant_read(pages, b.positions, b.req_of_token[:0], table)
    with pytest.raises(ops.KernelError):
        ops.quant_read(pages, b.positions, b.req_of_token, table, torch.float16)


def test_operands_that_do_not_fit_are_named_and_nothing_is_written():
    """Every operand by itself wrong in type, place, shape, order or length: an error that is ours, and pages as they were."""
    c = Case([(1, 3, 4), (20, 0, 20)], 2, 64, 16, seed=1).fill()
    pages, b = c.pages(), c.batch()
    table, nh = b.block_tables[0], 4
    before = [t.clone() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    q = torch.zeros(21, nh * 64, dtype=torch.bfloat16, device="cuda")
    x = torch.ones(21, 8 * 64, device="cuda")
    turns = torch.zeros(21, 64, device="cuda")

    def wrong(t):
        out = [t.double() if t.dtype == torch.float32 else t.float(), t.cpu(), t.flatten()]
        if t.dim() > 1 and t.shape[-1] > 1:
            out.append(t.transpose(-1, -2).contiguous().transpose(-1, -2))      # the same numbers in another order
        return out

    parts = [pages.k, pages.v, pages.k_scale, pages.v_scale]
    tries = []
    for i, t in enumerate(parts):
        for w in wrong(t) + [t[:, :1].contiguous(), t[:-1]]:
            bad = ops.QuantPages(*[w if j == i else p for j, p in enumerate(parts)])
            tries += [lambda bad=bad: ops.quant_append(x, b.positions, b.req_of_token, table, bad, nh),
                      lambda bad=bad: ops.quant_read(bad, b.positions, b.req_of_token, table),
                      lambda bad=bad: ops.quant_attention(q, bad, b, table, nh, 0.1)]
    for w in wrong(table):
        tries += [lambda w=w: ops.quant_append(x, b.positions, b.req_of_token, w, pages, nh), lambda w=w: ops.quant_read(pages, b.positions, b.req_of_token, w),
                  lambda w=w: ops.quant_attention(q, pages, b, w, nh, 0.1)]
    tries.append(lambda: ops.quant_attention(q, pages, b, table[:1], nh, 0.1))
    for w in (b.positions.long(), b.positions.cpu(), b.positions[:-1], b.positions.repeat_interleave(2)[::2]):
        tries += [lambda w=w: ops.quant_append(x, w, b.req_of_token, table, pages, nh), lambda w=w: ops.quant_append(x, b.positions, w, table, pages, nh),
                  lambda w=w: ops.quant_read(pages, w, b.req_of_token, table), lambda w=w: ops.quant_read(pages, b.positions, w, table)]
    for w in wrong(x)[:2] + [x.flatten(), x.t().contiguous().t(), x[:, :-64].contiguous(), x[None, None], x[None].to(torch.bfloat16), x[None][:0],
                             torch.ones(2, 21, 8 * 64 + 8, device="cuda")[:, :, :8 * 64]]:
        tries.append(lambda w=w: ops.quant_append(w, b.positions, b.req_of_token, table, pages, nh))
    for w in (turns.double(), turns.cpu(), turns[:-1], turns[:, :-1].contiguous(), torch.zeros(21, 66, device="cuda"), turns.t().contiguous().t()):
        tries.append(lambda w=w: ops.quant_append(x, b.positions, b.req_of_token, table, pages, nh, table=w))
    for w in wrong(q) + [q[:-1], q[:, :-64].contiguous()]:
        tries.append(lambda w=w: ops.quant_attention(w, pages, b, table, nh, 0.1))
    for name in ("cu_q", "q_start", "kv_len"):
        for w in (getattr(b, name).long(), getattr(b, name).cpu(), getattr(b, name)[:1]):
            other = c.batch()
            setattr(other, name, w)
            tries.append(lambda other=other: ops.quant_attention(q, pages, other, table, nh, 0.1))
    for name, w in (("h_q_len", [1]), ("h_q_len", [1, 19]), ("h_q_len", [-1, 22]), ("h_q_len", [1, 2 ** 40]), ("h_q_start", [3]), ("h_q_start", [-3, 0]),
                    ("h_q_start", [3, 2 ** 31 - 30]), ("T", 20), ("R", 3)):
        other = c.batch()
        setattr(other, name, w)
        tries.append(lambda other=other: ops.quant_attention(q, pages, other, table, nh, 0.1))
    for sink in (torch.zeros(nh, device="cuda").double(), torch.zeros(nh), torch.zeros(nh + 1, device="cuda"), torch.zeros(2 * nh, device="cuda")[::2]):
        tries.append(lambda sink=sink: ops.quant_attention(q, pages, b, table, nh, 0.1, sink=sink))
    for i, t in enumerate(tries):
        with pytest.raises(ops.KernelError):
            t()
            pytest.fail(f"call {i} was taken")
    assert all(torch.equal(a, t) for a, t in zip(before, parts))
    # lengths as a tuple are as good as a list, and a batch without tokens has no rows
    b.h_q_len, b.h_q_start = tuple(b.h_q_len), tuple(b.h_q_start)
    assert ops.quant_attention(q, pages, b, table, nh, 0.1).shape == q.shape
    none = Case([(0, 5, 5)], 2, 64, 16, seed=2).fill()
    nb, np_ = none.batch(), none.pages()
    assert ops.quant_attention(q[:0], np_, nb, nb.block_tables[0], nh, 0.1).shape == (0, nh * 64)
    assert ops.quant_append(x[:0], nb.positions, nb.req_of_token, nb.block_tables[0], np_, nh).shape == (0, nh * 64)
    assert ops.quant_read(np_, nb.positions, nb.req_of_token, nb.block_tables[0])[0].shape == (0, 2, 64)


def test_calls_on_two_streams_at_once_and_two_recorded_steps():
    """Scratch is a call's own: decoding requests whose slices join through memory and portions of prompts, side by side on two streams, and
    two graphs replayed in turn and side by side, give what each gives by itself."""
    cases = [Case([(1, 9000, 9001), (1, 40, 41), (70, 300, 370)], 2, 64, 16, seed=s).fill() for s in (1, 2)]
    work = []
    for c in cases:
        b = c.batch()
        q = torch.randn(c.T, 8 * 64, generator=c.gen).to(torch.bfloat16).cuda()
        work.append((q, c.pages(), b, b.block_tables[0]))

    def run(i):
        q, pages, b, table = work[i]
        return ops.quant_attention(q, pages, b, table, 8, 0.125)

    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    # recorded: the same steps with their lengths left to the device
    steps = []
    for c in cases:
        d = Case([(1, 9000, 9001), (1, 40, 41), (1, 700, 701)], 2, 64, 16, seed=c.T).fill()
        b = d.batch(bound=16384)
        q = torch.randn(d.T, 8 * 64, generator=d.gen).to(torch.bfloat16).cuda()
        pages = d.pages()
        alone = ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.125)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.125)
        steps.append((graph, out, alone, (q, pages, b)))
    for _ in range(10):
        for s, (graph, out, _, _) in zip(streams, steps):
            with torch.cuda.stream(s):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, alone) for _, out, alone, _ in steps)
    assert ops.attention_q8_status() == 0


def scales_far_apart(c, kind):
    """The case's value rows again: ``tiny`` from what is barely written on, ``zeros`` rows of nothing beside loud ones, ``wide`` everything,
    ``spread`` as far apart as portions of prompts take it."""
    lo, hi = {"tiny": (-117, -95), "zeros": (29, 31), "wide": (-117, 95), "spread": (-60, 39)}[kind]
    draws = torch.rand(c.v_scale.shape, generator=c.gen)
    c.v_scale = torch.exp2(lo + 0.02 + (hi - lo) * draws).float()
    if kind == "zeros":
        empty = torch.rand(c.v_scale.shape, generator=c.gen) < 0.7
        c.v_scale[empty], c.v[empty] = 0.0, 0
        # a request's first keys as well, so that a slice begins with them
        for r in range(len(c.segments)):
            first = int(c.table[r, 0])
            c.v_scale[first], c.v[first] = 0.0, 0
    return c


def check_scales(c, nh, counts=-102):
    """As ``check_attention`` with nothing absolute in the bound, but for scales that count as 2^``counts`` in the reference of a row's weights."""
    hd = c.hd
    q = torch.randn(c.T, nh * hd, generator=c.gen).to(torch.bfloat16)
    b = c.batch()
    got = ops.quant_attention(q.cuda(), c.pages(), b, b.block_tables[0], nh, hd ** -0.5).cpu().double().view(c.T, nh, hd)
    e = attention(q.view(c.T, nh, hd), c.k, c.v, c.k_scale, c.v_scale, c.cu, c.start, c.total, c.table, hd ** -0.5)
    # a weight is within 2^-25 of the largest, p times a scale of at least that: p is at most 1, and the numbers of a channel as many as
    # keys, at most 127 each
    low = 2.0 ** -25 * 2.0 ** counts * 127 * (c.pos + 1).double()[:, None, None]
    tol = attention_bound(e, hd) - 1e-30 + 1.01 * low
    over = ((got - e.out).abs() / tol).max().item()
    assert torch.isfinite(got).all() and over <= 1.0, f"error {over:.2f} times the bound"
    assert ops.attention_q8_status() == 0


@pytest.mark.parametrize("kind", ["tiny", "zeros", "wide"])
@pytest.mark.parametrize("hd,nh,nkv,page", [(128, 8, 2, 16), (64, 7, 1, 8), (80, 16, 1, 24)])
def test_value_scales_far_apart(kind, hd, nh, nkv, page):
    """A few rows a request, one slice and many: what a scale of 2^-117 leaves, rows of zeros that keep their share, and both beside large ones."""
    segs = [(1, 40, 41), (1, 699, 700), (1, 0, 1), (2 if nh // nkv <= 8 else 1, 30, 32 if nh // nkv <= 8 else 31)]
    check_scales(scales_far_apart(Case(segs, nkv, hd, page, seed=hd + len(kind)).fill(), kind), nh)
    check_scales(scales_far_apart(Case([(1, 9000, 9001)], nkv, hd, page, seed=hd + 1).fill(), kind), nh)


@pytest.mark.parametrize("kind", ["plain", "tiny", "zeros", "spread"])
@pytest.mark.parametrize("hd,nh,nkv,page", [(128, 8, 2, 16), (64, 7, 1, 8), (256, 4, 1, 24), (96, 6, 2, 16)])
def test_portions_keep_what_the_bound_of_a_few_rows_grants(kind, hd, nh, nkv, page):
    """Portions of prompts round weights and results alone: they are within the bound without anything for keys and values, whatever their scales."""
    c = Case([(70, 0, 70), (41, 160, 201), (1, 99, 100), (130, 600, 730)], nkv, hd, page, seed=hd * 5 + len(kind)).fill()
    # (scales of 0 count as 2^-60 there, others as they are)
    check_scales(c if kind == "plain" else scales_far_apart(c, kind), nh, -60 if kind == "zeros" else -1000)


@pytest.mark.parametrize("hd,nh,nkv", [(128, 8, 2), (64, 6, 1), (192, 2, 1)])
@pytest.mark.parametrize("louder", [2.0 ** 14, 2.0 ** 20, 2.0 ** 30])
def test_a_later_token_leaves_the_rows_before_it_alone(hd, nh, nkv, louder):
    """Prompts whose tokens from some position on, in the tile of rows that do not see them, are far louder, or no numbers: the rows before
    have the same bits, and those of the same prompt cut there within the bound."""
    n, at = 230, 141
    c = Case([(n, 0, n)], nkv, hd, 16, seed=hd).fill()
    q = torch.randn(n, nh * hd, generator=c.gen).to(torch.bfloat16).cuda()
    b = c.batch()
    quiet = ops.quant_attention(q, c.pages(), b, b.block_tables[0], nh, 0.1)
    page, slot = row_index(c.pos, c.req, c.table, c.page)
    for factor in (louder, math.nan):
        for scales in (c.k_scale, c.v_scale):
            scales[page[at:], :, slot[at:]] *= factor
        loud = ops.quant_attention(q, c.pages(), b, b.block_tables[0], nh, 0.1)
        assert torch.equal(loud[:at], quiet[:at])
        if factor == louder:
            # (rows that see the loud keys have scores of up to 2^40: exponentials of their float32 errors have no bound, and there is none for them)
            e = attention(q.cpu().view(n, nh, hd), c.k, c.v, c.k_scale, c.v_scale, c.cu, c.start, c.total, c.table, 0.1)
            assert ((loud.cpu().double().view_as(e.out) - e.out).abs() <= attention_bound(e, hd))[:at].all()
            cut = Case([(at, 0, at)], nkv, hd, 16, seed=hd)
            cut.k, cut.v, cut.k_scale, cut.v_scale, cut.table = c.k, c.v, c.k_scale, c.v_scale, c.table
            cb = cut.batch()
            alone = ops.quant_attention(q[:at].contiguous(), cut.pages(), cb, cb.block_tables[0], nh, 0.1)
            assert ((alone.cpu().double().view(at, nh, hd) - e.out[:at]).abs() <= attention_bound(e, hd)[:at]).all()
        else:
            assert torch.isnan(loud[at:]).all()
    assert ops.attention_q8_status() == 0


def test_after_a_wait_gave_up_rows_are_no_numbers():
    """With the status set, as a wait that gives up sets it, nothing passes for a result: whole items and such as several blocks share (joined
    from parts) are NaN until the status has been read; requests of few rows are another kernel's."""
    from blackwellllm_b200.kernels.build import load_library
    c = Case([(200, 0, 200), (1, 40, 41), (70, 3000, 3070)], 2, 64, 16, seed=3).fill()
    b, pages = c.batch(), c.pages()
    q = torch.randn(c.T, 4 * 64, generator=c.gen).to(torch.bfloat16).cuda()
    want = ops.quant_attention(q, pages, b, b.block_tables[0], 4, 0.125)
    assert ops.attention_q8_status() == 0 and torch.isfinite(want).all()
    assert load_library("attention_q8_tc", {"HEAD_DIM": 64}).bw_attention_q8_tc_give_up(39) == 0
    for _ in range(2):
        got = ops.quant_attention(q, pages, b, b.block_tables[0], 4, 0.125)
        assert torch.isnan(got[:200]).all() and torch.isnan(got[201:]).all() and torch.equal(got[200], want[200])
    assert ops.attention_q8_status() == 39 and ops.attention_q8_status() == 0
    assert torch.equal(ops.quant_attention(q, pages, b, b.block_tables[0], 4, 0.125), want)


def test_a_long_request_beside_two_hundred_short_ones():
    """Slices dealt out on the device for a call of its own too, more of them than run at once: at the call's lengths, repeated on two streams, and
    replayed at others (all short, the long one elsewhere, one longer than the bound)."""
    lens = [21 + i % 7 for i in range(200)]
    lens[37], lens[150] = 9001, 700
    c = Case([(1, n - 1, n) for n in lens], 4, 64, 16, seed=12).fill()
    got = c.check_attention(8)
    b, pages = c.batch(), c.pages()
    q = torch.randn(c.T, 8 * 64, generator=c.gen).to(torch.bfloat16).cuda()
    want = ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.125)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.125))
    torch.cuda.synchronize()
    assert got.shape[0] == 200 and all(torch.equal(o, want) for o in outs)
    b = c.batch(bound=4096)
    ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.125)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dealt = ops.quant_attention_deal(b, 8, 4, 64, 16)
        out = ops.quant_attention(q, pages, b, b.block_tables[0], 8, 0.125, dealt=dealt)
    assert dealt is not None
    for long37, long150 in ((9001, 700), (20, 20), (3, 699), (5000, 1)):
        ends = [min(n, 20) for n in lens]
        ends[37], ends[150] = long37, long150
        starts = [n - 1 for n in ends]
        b.q_start.copy_(torch.tensor(starts)); b.kv_len.copy_(torch.tensor(ends))
        out.fill_(float("nan"))
        graph.replay()
        e = attention(q.cpu().view(200, 8, 64), c.k, c.v, c.k_scale, c.v_scale, c.cu, starts, ends, c.table, 0.125)
        assert ((out.cpu().double().view_as(e.out) - e.out).abs() <= attention_bound(e, 64)).all()
