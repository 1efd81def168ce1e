"""route_experts against its definition in float64 (oracle/mxfp4.py)."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as ref

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def _check(logits, topk, bias=None, weights_dtype=torch.float32, **kw):
    from ferry_b200 import expert_ops
    sel, w = expert_ops.route_experts(logits.to(DEV), topk, bias=None if bias is None else bias.to(DEV),
                                      weights_dtype=weights_dtype, **kw)
    norm = kw.pop('norm_topk_prob', True)
    want_sel, want_w = ref.route(logits.double().numpy(), topk, bias=None if bias is None else bias.double().numpy(),
                                 norm=norm, **kw)
    np.testing.assert_array_equal(sel.cpu().numpy(), want_sel)
    # formed in float64, rounded once: half a step of the weights' type
    # (a subnormal's half step is absolute)
    f = torch.finfo(weights_dtype)
    got = w.double().cpu().numpy()
    np.testing.assert_allclose(got, want_w, rtol=f.eps / 2 * (1 + 1e-6), atol=f.smallest_normal * f.eps)
    assert sel.dtype == torch.int64 and w.dtype == weights_dtype
    return sel, w


def _logits(tokens, experts, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(tokens, experts, generator=g).mul_(1.5).to(dtype)


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('tokens,experts,topk,groups,kept,group_score', [
    (1, 1, 1, 1, 1, 'max'), (1, 64, 6, 1, 1, 'max'), (5, 33, 33 - 1, 1, 1, 'max'), (64, 128, 8, 1, 1, 'max'),
    (3, 160, 6, 8, 3, 'max'), (130, 256, 8, 8, 4, 'top2'), (17, 96, 4, 3, 2, 'top2'),
    (9, 1024, 32, 1, 1, 'max'), (7, 1024, 16, 32, 5, 'top2'), (6, 60, 10, 20, 4, 'max'), (4, 32, 1, 32, 1, 'max'),
    (2, 2, 2, 1, 1, 'max'), (5, 21, 3, 7, 7, 'top2'),
])
def test_matches_definition(tokens, experts, topk, groups, kept, group_score, score, dtype):
    x = _logits(tokens, experts, experts + topk, TYPES[dtype])
    bias = 0.3 * torch.randn(experts, generator=torch.Generator().manual_seed(3))
    kw = dict(score=score, n_group=groups, topk_group=kept, group_score=group_score)
    _check(x, topk, **kw)
    _check(x, topk, bias, norm_topk_prob=False, scaling=2.5, **kw)
    _check(x, topk, bias, weights_dtype=torch.bfloat16, **kw)
    _check(x, topk, weights_dtype=torch.float16, norm_topk_prob=False, scaling=0.5, **kw)


def test_ties_go_to_the_lower_id():
    x = torch.zeros(4, 64)
    x[1, ::2] = 1.0
    x[2, 63] = 2.0
    for score in ('softmax', 'sigmoid'):
        sel, _ = _check(x, 8, score=score)
        assert sel[0].tolist() == list(range(8)) and sel[2].tolist() == [63] + list(range(7))
        sel, _ = _check(x, 4, score=score, n_group=8, topk_group=2, group_score='top2')
        assert sel[0].tolist() == [0, 1, 2, 3]
    _check(_logits(300, 128, 9).mul(2).round().div(2), 8, score='sigmoid', bias=torch.zeros(128))


def test_scores_that_float32_cannot_tell_apart():
    """sigmoid(20 + i * 2^-10) differ by about 2e-12: one float32, but 64 bits
    order them."""
    x = (20 + torch.arange(64) * 2.0 ** -10)[torch.randperm(64, generator=torch.Generator().manual_seed(0))]
    _check(x.view(1, -1), 8, score='sigmoid')
    _check(x.view(1, -1), 8, score='sigmoid', n_group=8, topk_group=4, group_score='top2')


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_masked_and_infinite_logits(score):
    inf, nan = float('inf'), float('nan')
    x = _logits(7, 32, 1)
    x[0, 3:] = -inf           # three experts left of the topk 4
    x[1, :] = -inf            # none left
    x[2, 5] = nan
    x[3, :16] = -inf
    x[4, :] = torch.finfo(torch.float32).min
    x[5, 7] = torch.finfo(torch.float32).max
    x[6, 9] = inf
    if score == 'softmax':    # exp(inf - inf) is not a number: the whole row
        from ferry_b200 import expert_ops
        sel, w = expert_ops.route_experts(x[6:].to(DEV), 4, weights_dtype=torch.float32)
        assert sel.tolist() == [[0, 1, 2, 3]] and bool(w.isnan().all())
        x = x[:6]
    for groups, kept in ((1, 1), (4, 2)):
        _check(x, 4, score=score, n_group=groups, topk_group=kept)
        _check(x, 4, score=score, n_group=groups, topk_group=kept, norm_topk_prob=False,
               bias=torch.linspace(-1, 1, 32))
    if score == 'softmax':
        _, w = _check(x[1:2], 4)
        assert bool((w == 0).all())


def test_strides_streams_and_empty():
    from ferry_b200 import expert_ops
    wide = _logits(50, 200, 2).to(DEV)
    part = wide[3:40, 11:139]
    want = expert_ops.route_experts(part.contiguous(), 8)
    for x in (part, part.t().contiguous().t()):
        got = expert_ops.route_experts(x, 8)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = expert_ops.route_experts(wide[:1, :128].expand(6, 128), 8)
    assert bool((got[0] == got[0][0]).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = expert_ops.route_experts(part, 8)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    sel, w = expert_ops.route_experts(wide[:0], 8)
    assert sel.shape == (0, 8) and w.shape == (0, 8)


def test_graph_capture():
    from ferry_b200 import expert_ops
    x = _logits(40, 128, 4).to(DEV)
    expert_ops.route_experts(x, 8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sel, w = expert_ops.route_experts(x, 8)
    x.copy_(_logits(40, 128, 5))
    g.replay()
    want = expert_ops.route_experts(x, 8)
    assert torch.equal(sel, want[0]) and torch.equal(w, want[1])


def test_feeds_the_runtime():
    """OffloadRuntime.execute on a grouped sigmoid router's choices, against the
    oracle runtime given the same."""
    from ferry_b200 import expert_ops
    from ferry_b200.model import ModelSpec
    from ferry_b200.quota import Topology
    from ferry_b200.runtime import OffloadRuntime
    from ferry_b200.workload import cpu_pool
    from oracle.layer import OracleRuntime
    from tests.tolerance import assert_bf16_close
    spec = ModelSpec('qwen3_moe', (0, 1), 32, 4, 256, 128)
    pool = cpu_pool(spec, 2, 0).pin_memory()
    topo = Topology.uniform(1, 32)
    rt = OffloadRuntime(spec, pool, [40], 'ferry', topo, sync_fetch=True)
    orc = OracleRuntime(spec, pool, [40], 'ferry', topo.masks, topo.seconds, topo.lut)
    g = torch.Generator().manual_seed(0)
    for layer in (0, 1, 0):
        x = torch.randn(19, 256, generator=g).to(torch.bfloat16)
        sel, w = expert_ops.route_experts(_logits(19, 32, layer).to(DEV), 4, score='sigmoid', n_group=8,
                                          topk_group=4, group_score='top2', scaling=2.5)
        got = rt.execute(layer, x.to(DEV), sel, w, None)
        rt.check()
        want, _, _ = orc.execute(layer, [x], [sel.cpu()], [w.cpu()])
        assert_bf16_close(got.cpu(), want[0])
    rt.close()


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('groups,kept,group_score', [(1, 1, 'max'), (8, 3, 'max'), (8, 4, 'top2')])
def test_close_keys(score, groups, kept, group_score):
    """Keys a few to a few thousand units of float32 apart, with and without a
    bias that brings different scores together: the 64-bit order decides."""
    g = torch.Generator().manual_seed(groups)
    kw = dict(score=score, n_group=groups, topk_group=kept, group_score=group_score)
    for spread in (2.0 ** -24, 2.0 ** -21, 2.0 ** -18, 2.0 ** -14, 2.0 ** -10):
        x = 1 + spread * torch.randint(-64, 64, (40, 128), generator=g).float()
        _check(x, 8, **kw)
        bias = torch.randn(128, generator=g)
        score_of = torch.softmax if score == 'softmax' else (lambda t, d: torch.sigmoid(t))
        y = torch.randn(1, 128, generator=g)
        close = 3 - score_of(y.double(), 1)[0].float() + spread * torch.randint(-64, 64, (128,), generator=g).float()
        _check(y.expand(3, 128).contiguous(), 8, bias=close, **kw)
        _check(torch.randn(40, 128, generator=g), 8, bias=bias * spread, **kw)


def test_ties_across_the_border():
    """More equal logits than places, equal logits under different biases, and
    scores far below the largest."""
    x = torch.full((5, 128), -1.0)
    x[1, 3::7] = 2.0
    x[2, :4] = torch.tensor([5.0, 4.0, 3.0, 2.0])
    x[3, 100:] = -100.0
    x[4, 10:] = -200.0
    for score in ('softmax', 'sigmoid'):
        for topk in (1, 8, 17, 32):
            _check(x, topk, score=score)
            _check(x, topk, score=score, bias=torch.arange(128).remainder(3).float() * 0.25)


def _close_worths(tokens, size, seed):
    """Logits of four experts in two groups, and biases (size, -size) in each, such
    that the two groups' sums of keys lie a few float32 steps of `size` apart, for
    softmax scores (the logits are log s with sum s = 1) and for sigmoid scores."""
    g = np.random.default_rng(seed)
    s = g.uniform(0.2, 0.8, (tokens, 4))
    apart = g.uniform(-1, 1, tokens) * np.minimum(4 * size * 2.0 ** -24, 0.1)
    soft = s.copy()
    soft[:, 2:] *= ((soft[:, :2].sum(1) + apart) / soft[:, 2:].sum(1))[:, None]
    s[:, 3] = np.clip(s[:, 0] + s[:, 1] - s[:, 2] + apart, 0.01, 0.99)
    bias = torch.tensor([size, -size, size, -size], dtype=torch.float32)
    return {'softmax': torch.from_numpy(np.log(soft)).float(),
            'sigmoid': torch.from_numpy(np.log(s / (1 - s))).float()}, bias


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('size', [1.0, 64.0, 256.0, 1e4, 1e6])
def test_group_sums_of_biases_that_cancel(size, score):
    """The two largest keys of a group may be far larger than their sum, and are
    rounded at their own size."""
    logits, bias = _close_worths(600, size, int(size))
    kw = dict(score=score, n_group=2, topk_group=1, group_score='top2')
    _check(logits[score], 2, bias=bias, **kw)
    wide = torch.cat((logits[score], _logits(600, 28, 1)), 1)  # of 16 groups, 5 stay
    _check(wide, 6, bias=torch.cat((bias, torch.zeros(28))), score=score, n_group=16, topk_group=5, group_score='top2')


def test_group_sums_that_float32_orders_the_other_way():
    """Worths of 0.7950212 and 0.7950132; float32 has 0.7949829 and 0.7950440."""
    x = torch.tensor([[-0.33179307, -0.50137854, -1.0042144, 0.10770209]])
    sel, _ = _check(x, 2, bias=torch.tensor([1000.0, -1000.0, 1000.0, -1000.0]), score='sigmoid', n_group=2,
                    topk_group=1, group_score='top2')
    assert sel.tolist() == [[0, 1]]


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_group_sum_that_is_not_a_number(score):
    """+inf and -inf biases in one group: its worth is NaN and ranks last, whichever
    lanes hold the two."""
    inf = float('inf')
    for experts, groups in ((8, 4), (64, 8), (32, 16)):
        size = experts // groups
        for one in (0, groups - 1):
            bias = torch.zeros(experts)
            bias[one * size:(one + 1) * size] = -inf
            for at in (0, size - 1):
                b = bias.clone()
                b[one * size + at] = inf
                for kept in (1, 2, groups - 1):
                    with np.errstate(invalid='ignore'):
                        _check(_logits(20, experts, experts), 2, bias=b, score=score, n_group=groups, topk_group=kept,
                               group_score='top2')


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('experts', [1024, 256, 40])
def test_many_ties_and_one_that_is_not(score, experts):
    """Rows of equal logits, and such rows with one that is a step of float32 above or
    below, in the first, the last and a middle place."""
    one = 0.75
    x = torch.full((7, experts), one)
    for i, (at, to) in enumerate([(0, 1.0), (0, 0.0), (experts - 1, 1.0), (experts - 1, 0.0), (experts // 2 + 1, 1.0),
                                  (experts // 2 + 1, 0.0)]):
        x[i, at] = torch.nextafter(torch.tensor(one), torch.tensor(to))
    for topk in (1, 8, 32):
        sel, _ = _check(x, topk, score=score)
        assert sel[6].tolist() == list(range(topk))
        _check(x, topk, score=score, bias=torch.linspace(0, 1, 4).repeat(experts // 4).float())
    _check(x, 4, score=score, n_group=4, topk_group=2, group_score='top2')
