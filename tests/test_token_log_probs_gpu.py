"""Log probability, rank, entropy and alternatives of given tokens against the definition in 64 bits."""
import math

import pytest
import torch

from blackwellllm_b200.kernels import ops

pytestmark = pytest.mark.gpu


def plain(row, target, top):
    """(log prob, entropy, rank, ids, log probs) of one float32 row, 64 bits, on the CPU."""
    x = row.double()
    nan = math.nan
    if torch.isnan(x).any() or (x == math.inf).any() or not (x > -math.inf).any():
        return nan, nan, -1, [-1] * top, [nan] * top
    # (differences to the largest, its own term beside the sum: x - logsumexp(x) would lose 7e-15 of a largest logit of 40)
    best = int(x.argmax())
    d = x - x[best]
    e = d.exp()
    e[best] = 0.0
    lp = d - math.log1p(e.sum().item())
    p = lp.exp()
    entropy = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum().item()
    order = torch.sort(x, descending=True, stable=True).indices
    ids = order[:top].tolist()
    if not 0 <= target < len(x):
        return nan, entropy, -1, ids, lp[ids].tolist()
    rank = int((x > x[target]).sum() + (x[:target] == x[target]).sum())
    return lp[target].item(), entropy, rank, ids, lp[ids].tolist()


def check(logits, targets, top):
    got = ops.token_log_probs(logits, torch.tensor(targets, dtype=torch.int32, device="cuda"), top)
    host = logits.cpu()
    for r, t in enumerate(targets):
        lp, entropy, rank, ids, lps = plain(host[r], t, top)
        assert got.rank[r].item() == rank
        assert got.top_ids[r].tolist() == ids
        x = host[r][torch.isfinite(host[r])].double()
        span = (x.max() - x.min()).clamp_max(200).item() if len(x) else 0.0
        # A term e^d, d a float32 difference: d and its product with log2 e are each off by 2^-24 of themselves, the exponential by 2^-22; the terms
        # that count have d within the span.  Sums of n terms in threads of at most 512 and trees of 2^-24 a step, so 2^-15 of z at the
        # very most; for the log probability that is absolute, and its own value is rounded once more.
        loose = 2.0 ** -22 * (4 + span) + 520 * 2.0 ** -24
        for a, b in [(got.log_prob[r].item(), lp)] + list(zip(got.top_log_probs[r].tolist(), lps)):
            if math.isnan(b) or math.isinf(b):
                assert (math.isnan(a) and math.isnan(b)) or a == b
            else:
                # of a sharp distribution 1 - p counts: what is off is off by that much of it
                sharp = min(1.0, 2 * -math.expm1(max(lps[0], -700.0))) if lps else 1.0
                assert abs(a - b) <= loose * max(sharp, 0.0) + 2.0 ** -22 * abs(b), (r, a, b)
        a = got.entropy[r].item()
        if math.isnan(entropy):
            assert math.isnan(a)
        else:
            # two sums, each off by `loose` of itself; |w| / (1 + z) is at most the entropy, and so is log(1 + z)
            assert abs(a - entropy) <= 4 * loose * max(entropy, 2.0 ** -40) + 1e-30, (r, a, entropy)
    return got


@pytest.mark.parametrize("V", [1, 2, 3, 31, 33, 512, 2047, 2049, 8192, 8195, 32003, 65536, 128256, 152064])
@pytest.mark.parametrize("R", [1, 3, 37])
def test_against_64_bits(R, V):
    g = torch.Generator().manual_seed(V * 100 + R)
    x = torch.randn(R, V, generator=g) * torch.rand(R, 1, generator=g) * 5
    targets = [[int(torch.randint(0, V, (1,), generator=g)), int(x[r].argmax()), 0, V - 1][r % 4] for r in range(R)]
    for top in sorted({0, 1, min(5, V), min(32, V)}):
        check(x.cuda(), targets, top)


def test_many_rows_are_a_block_each():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(400, 9001, generator=g)
    check(x.cuda(), torch.randint(0, 9001, (400,), generator=g).tolist(), 20)


@pytest.mark.parametrize("V", [4096, 60001])
def test_ties_go_to_the_lowest_id(V):
    g = torch.Generator().manual_seed(V)
    x = torch.zeros(6, V)
    x[1] = torch.randint(0, 3, (V,), generator=g).float()
    x[2] = torch.randn(V, generator=g).to(torch.bfloat16).float().clamp_max(1.0)
    x[3, ::2] = -0.0                                     # equal to 0, not below it
    x[4] = torch.arange(V).float() / 64                  # the best tokens last
    x[5] = -x[4]
    check(x.cuda(), [V // 2, 7, V - 1, 8, V - 3, 5], 32)


@pytest.mark.parametrize("rows", [6, 301])
@pytest.mark.parametrize("V", [152064, 9001])
def test_alternatives_wherever_the_best_stand(rows, V):
    """Rows in order, of one value, of few values, and with all the large ones in the elements of a few threads: lists of many candidates."""
    g = torch.Generator().manual_seed(rows + V)
    x = torch.randn(rows, V, generator=g)
    x[0] = torch.linspace(-3, 3, V)
    x[1] = torch.linspace(3, -3, V)
    x[2] = 0.25
    x[3] = torch.randint(0, 3, (V,), generator=g).float()
    four = torch.arange(V) // 4
    x[4] = torch.where(four % 512 < 224, x[4] + 50, x[4])       # seven warps of a block, where a block has the row
    x[5] = torch.where(four % 512 == 77, x[5] + 50, x[5])
    for top in (2, 7, 8, 9, 20, 32):
        target = torch.arange(rows, dtype=torch.int32) % V
        got = ops.token_log_probs(x.cuda(), target.cuda(), top)
        again = ops.token_log_probs(x.cuda(), target.cuda(), top)
        for r in range(6):
            order = torch.sort(x[r].double(), descending=True, stable=True).indices
            assert got.top_ids[r].tolist() == order[:top].tolist(), r
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    check(x[:6].cuda(), [0, 1, 2, 3, 4, 5], 32)


def test_masked_and_broken_rows():
    V = 5003
    g = torch.Generator().manual_seed(1)
    x = torch.randn(9, V, generator=g)
    x[0, 10:] = -math.inf                                # ten tokens are left, twelve asked for
    x[1] = -math.inf
    x[2, 77] = math.inf
    x[3, 4000] = math.nan
    x[4, :] = -math.inf
    x[4, 4999] = 3.0                                     # one token is certain
    x[5, 1:] = -3.0e38
    x[6] = -math.inf
    x[6, [5, 4000]] = torch.tensor([-1.0e30, 2.0])
    x[7, 12] = -math.nan
    targets = [10, 3, 77, 0, 4999, 0, 5, 1, -1]
    got = check(x.cuda(), targets, 12)
    assert got.log_prob[4].item() == 0 and got.entropy[4].item() == 0 and got.log_prob[0].item() == -math.inf
    got = check(x.cuda(), [V, 1, 2, 3, 0, 4, 4000, 8, 2 ** 31 - 1], 0)
    assert got.top_ids.shape == (9, 0)


def test_sharp_rows_keep_their_bits():
    """The most probable token's log probability and the entropy where everything else together has 1e-3 to 1e-12 of the mass."""
    V = 128256
    x = torch.zeros(5, V)
    for r, gap in enumerate((19.0, 24.0, 30.0, 36.0, 40.0)):
        x[r, 100 + r] = gap
    got = check(x.cuda(), [100 + r for r in range(5)], 2)
    assert (got.log_prob < 0).all() and (got.entropy > 0).all()


def test_rows_apart_unaligned_and_the_same_bits():
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(7, 3 + 20000 + 5, generator=g).cuda()
    for first in (0, 1, 2, 3, 4):
        x = wide[:, first:first + 20000]
        got = check(x, [0, 19999, 5, 6, 7, 8, 9], 5)
        again = ops.token_log_probs(x, torch.tensor([0, 19999, 5, 6, 7, 8, 9], dtype=torch.int32, device="cuda"), 5)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_in_a_graph_and_on_another_stream():
    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, 30000, generator=g).cuda()
    t = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    want = ops.token_log_probs(x, t, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.token_log_probs(x, t, 5)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.token_log_probs(x, t, 5)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, other, got):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals():
    x = torch.zeros(2, 40, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    for logits, target, top in [(x.double(), t, 0), (x, t.long(), 0), (x, t[:1], 0), (x, t, 33), (x, t, -1), (x[:, :20], t, 21),
                                (x.t(), torch.zeros(40, dtype=torch.int32, device="cuda"), 0), (x[0], t, 0), (x.cpu(), t, 0),
                                (x[:1].expand(2, 40), t, 0)]:
        with pytest.raises(ops.KernelError):
            ops.token_log_probs(logits, target, top)
    assert ops.token_log_probs(x[:0], t[:0], 5).top_ids.shape == (0, 5)
