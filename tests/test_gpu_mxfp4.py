"""MXFP4 rows and the routed experts over them against their definitions in
float64 (oracle/mxfp4.py)."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as ref

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
BF16 = torch.bfloat16
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def _values(rows, width, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g)
    if dtype != torch.float16:  # magnitudes over the whole range of a block scale
        x = x * torch.exp2(torch.randint(-60, 60, (rows, width // 32, 1), generator=g).float()).expand(
            -1, -1, 32).reshape(rows, width)
    return x.to(dtype)


def _check_quantize(x):
    from ferry_b200 import expert_ops
    codes, scales = expert_ops.quantize_mxfp4(x.to(DEV))
    want_codes, want_scales = ref.quantize(x.double().numpy())
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    np.testing.assert_array_equal(codes.cpu().numpy(), want_codes)
    return codes, scales


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('rows,width', [(1, 32), (3, 64), (7, 96), (129, 1408), (2, 4096), (1, 98304)])
def test_quantize_is_exact(rows, width, dtype):
    x = _values(rows, width, TYPES[dtype])
    codes, scales = _check_quantize(x)
    from ferry_b200 import expert_ops
    want = ref.dequantize(codes.cpu().numpy(), scales.cpu().numpy())
    for out in (torch.bfloat16, torch.float32):  # both hold every such value
        got = expert_ops.dequantize_mxfp4(codes, scales, out)
        np.testing.assert_array_equal(got.double().cpu().numpy(), want)
    got = expert_ops.dequantize_mxfp4(codes, scales, torch.float16)
    np.testing.assert_array_equal(got.cpu().numpy(), torch.from_numpy(want).to(torch.float16).numpy())


def test_quantize_borders():
    """Every midpoint between two codes, its neighbours and the values past the
    largest code, at scales from the smallest to the largest."""
    mids = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.9])
    vals = np.concatenate([mids, np.nextafter(mids.astype(np.float32), np.float32(9)),
                           np.nextafter(mids.astype(np.float32), np.float32(-9))])
    vals = np.concatenate([vals, -vals])
    vals = np.resize(vals, (len(vals) + 30) // 31 * 31).reshape(-1, 31)
    vals = np.concatenate([vals, np.full((len(vals), 1), 4.0)], 1).astype(np.float32)  # the scale's own value
    rows = [vals * np.float32(2.0 ** e) for e in (-126, -100, -20, 0, 17, 100, 124)]
    x = torch.from_numpy(np.concatenate(rows)).reshape(-1, 32)
    _check_quantize(x)
    _check_quantize(x.reshape(1, -1))
    _check_quantize(x[:60].to(BF16))


def test_quantize_special_blocks():
    inf, nan = float('inf'), float('nan')
    x = torch.zeros(9, 64)
    x[1, 3] = inf
    x[2, 40] = -inf
    x[3, 5] = nan
    x[4] = -0.0
    x[5] = torch.finfo(torch.float32).smallest_normal / 4   # subnormals
    x[6] = torch.finfo(torch.float32).tiny * 0 + 1e-45
    x[7] = torch.finfo(torch.float32).max
    x[8, 0], x[8, 1] = 1e30, 1e-30
    codes, scales = _check_quantize(x)
    from ferry_b200 import expert_ops
    got = expert_ops.dequantize_mxfp4(codes, scales, torch.float32).cpu()
    assert bool(got[1, :32].isnan().all()) and not bool(got[1, 32:].isnan().any())
    assert bool(got[3, :32].isnan().all()) and bool(got[2, 32:].isnan().all())
    assert bool((got[4] == 0).all()) and bool(got[4].signbit().all())


def test_every_code_and_scale_reads_back():
    from ferry_b200 import expert_ops
    codes = torch.arange(256, dtype=torch.uint8).repeat(16).view(256, 16)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1)
    want = ref.dequantize(codes.numpy(), scales.numpy())
    got = expert_ops.dequantize_mxfp4(codes.to(DEV), scales.to(DEV), torch.float32).cpu()
    with np.errstate(over='ignore'):
        np.testing.assert_array_equal(got.numpy(), want.astype(np.float32))
    got = expert_ops.dequantize_mxfp4(codes.to(DEV), scales.to(DEV)).cpu()
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), torch.from_numpy(want).float().to(BF16).nan_to_num(7.0, 8.0, 9.0))


def test_quantize_views():
    """Rows cut out of wider ones, misaligned starts, outputs inside expert rows."""
    from ferry_b200 import expert_ops
    from ferry_b200.model import mxfp4_parts
    for dtype in (BF16, torch.float32):
        wide = _values(12, 512, dtype, 3).to(DEV)
        for part in (wide[:, 3:67], wide[2:9, 8:200], wide.t()[:96].t(), wide[:1, 5:37].expand(4, 32),
                     wide.view(3, 4, 512)[:, 1:3, 64:128]):
            want = ref.quantize(part.double().cpu().numpy())
            codes, scales = expert_ops.quantize_mxfp4(part)
            np.testing.assert_array_equal(codes.cpu().numpy(), want[0])
            np.testing.assert_array_equal(scales.cpu().numpy(), want[1])
        rows = torch.full((12, 5 + 512 // 32 * 17), 7, dtype=torch.uint8, device=DEV)
        for cut in (0, 1, 4):  # 4-byte aligned and not
            body = rows[:, cut:cut + 512 // 32 * 17]
            rows.fill_(7)
            expert_ops.quantize_mxfp4(wide, out=mxfp4_parts(body))
            want = ref.quantize(wide.double().cpu().numpy())
            np.testing.assert_array_equal(body.cpu().numpy(), np.concatenate(want, 1))
            assert bool((rows[:, :cut] == 7).all()) and bool((rows[:, cut + 512 // 32 * 17:] == 7).all())
            frame = torch.zeros(12, 515, dtype=dtype, device=DEV)
            expert_ops.dequantize_mxfp4(*mxfp4_parts(body), dtype, out=frame[:, cut and 3:(cut and 3) + 512])
            np.testing.assert_array_equal(frame[:, cut and 3:(cut and 3) + 512].double().cpu().numpy(),
                                          ref.dequantize(*want))
    codes, scales = expert_ops.quantize_mxfp4(torch.zeros(0, 64, device=DEV))
    assert codes.shape == (0, 32) and scales.shape == (0, 2)
    assert expert_ops.dequantize_mxfp4(codes, scales).shape == (0, 64)


def test_pack_expert():
    from ferry_b200.model import mxfp4_parts, mxfp4_row_bytes, pack_expert, pack_expert_mxfp4
    g = torch.Generator(device=DEV).manual_seed(1)
    gate, up = (torch.randn(96, 128, generator=g, device=DEV) * 0.02 for _ in range(2))
    down = torch.randn(128, 96, generator=g, device=DEV) * 0.02
    row = pack_expert_mxfp4(gate, up, down)
    assert row.shape == (mxfp4_row_bytes(128, 96),)
    want = ref.quantize(pack_expert(gate, up, down).double().cpu().numpy())
    for got, w in zip(mxfp4_parts(row), want):
        np.testing.assert_array_equal(got.cpu().numpy(), w)


# ---------------------------------------------------------------------------
# the experts

def _layer(sizes, hidden, inter, slots, tokens, topk, seed=0, low=110, high=122):
    """CPU tensors of a layer: random codes, scale bytes in [low, high]."""
    g = torch.Generator().manual_seed(seed)
    n = 3 * hidden * inter
    cache = torch.randint(0, 256, (slots, n // 32 * 17), generator=g, dtype=torch.uint8)
    cache[:, n // 2:] = torch.randint(low, high + 1, (slots, n // 32), generator=g, dtype=torch.uint8)
    x = torch.randn(tokens, hidden, generator=g).to(BF16)
    w = torch.rand(tokens, topk, generator=g)
    starts = torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int64)
    routes = int(starts[-1])
    return dict(cache=cache, x=x, w=w, slots=torch.randint(0, slots, (len(sizes),), generator=g), starts=starts,
                rows=torch.randint(0, tokens, (routes,), generator=g),
                cols=torch.randint(0, topk, (routes,), generator=g), hidden=hidden, inter=inter)


def _run(d, **kw):
    from ferry_b200 import expert_ops
    t = [d[k].to(DEV) for k in ('cache', 'x', 'w', 'slots', 'starts', 'rows', 'cols')]
    return expert_ops.execute_experts_mxfp4(*t, d['hidden'], d['inter'], **kw)


def _want(d):
    """(values, bound): the definition in float64 and how far a kernel may be
    from it that holds x and the activation as two e4m3 parts (x exactly, the
    activation within 2^-9 of its value, both within 2^-21 of the largest value
    of their block of 32 where that is more), sums in float32, rounds the result
    to bf16 (2^-8 of the value) and takes exp with the error that CUDA's
    documentation gives for __expf (2 + 1.173 |x| units of 2^-23, three more for
    the sum and the quotient, one for the product)."""
    def largest(v):
        b = np.abs(v).reshape(v.shape[0], -1, 32).max(2, keepdims=True)
        return np.broadcast_to(b, b.shape[:2] + (32,)).reshape(v.shape)
    H, I = d['hidden'], d['inter']
    x, w = d['x'].double().numpy(), d['w'].double().numpy()
    n = 3 * H * I
    out, bound = np.zeros((len(d['rows']), H)), np.zeros((len(d['rows']), H))
    u24 = 2.0 ** -24
    for g, slot in enumerate(d['slots'].tolist()):
        a, b = int(d['starts'][g]), int(d['starts'][g + 1])
        if a == b:
            continue
        row = d['cache'][slot].numpy()
        gate, up, down = np.split(ref.dequantize(row[:n // 2], row[n // 2:]), 3)
        gate, up, down = gate.reshape(I, H).T, up.reshape(I, H).T, down.reshape(H, I).T
        xs = x[d['rows'][a:b].numpy()]
        gt, u = xs @ gate, xs @ up
        silu = gt / (1 + np.exp(-gt))
        act = silu * u
        # a float32 sum of 2 H products (exact): 2 H - 1 roundings at most
        dx = np.where(np.abs(xs) < 2.0 ** -13 * largest(xs), 2.0 ** -21 * largest(xs), 0.0)
        dg, du = ((2 * H * u24 * (np.abs(xs) + dx) + dx) @ np.abs(m) for m in (gate, up))
        dact = 1.1 * dg * (np.abs(u) + du) + np.abs(silu) * du + (8 + 1.173 * np.abs(gt)) * 2.0 ** -23 * np.abs(act)
        dact = dact + 2.0 ** -9 * (np.abs(act) + dact) + 2.0 ** -21 * largest(np.abs(act) + dact)
        y = act @ down
        wt = w[d['rows'][a:b].numpy(), d['cols'][a:b].numpy()][:, None]
        dy = (dact + 2 * I * u24 * (np.abs(act) + dact)) @ np.abs(down)
        out[a:b] = y * wt
        bound[a:b] = np.abs(wt) * (dy + u24 * (np.abs(y) + dy))
        bound[a:b] += 2.0 ** -8 * (np.abs(out[a:b]) + bound[a:b])
    return out, bound


def _assert_close(got, d, keep=slice(None)):
    want, bound = _want(d)
    err = np.abs(got.double().cpu().numpy() - want)[keep]
    assert np.isfinite(err).all()
    worst = np.max(err / np.maximum(bound[keep], 1e-300)) if err.size else 0.0
    assert worst <= 1.0, f'{worst:.2f} times the bound'


CASES = [
    # sizes, hidden, inter, slots, tokens, topk
    ([1], 128, 128, 1, 1, 1),
    ([1, 0, 2], 256, 128, 3, 5, 2),
    ([0, 3, 16, 17, 0, 32, 33], 384, 256, 4, 40, 4),
    ([64, 65, 127, 128, 129], 128, 384, 5, 200, 3),
    ([300, 1, 257], 512, 128, 2, 300, 2),
    ([1] * 40, 128, 256, 40, 7, 8),
    ([1, 7, 15, 40], 2048, 768, 4, 16, 8),
    ([5, 2], 2048, 1408, 2, 6, 6),
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: f'H{c[1]}_I{c[2]}_n{sum(c[0])}')
def test_experts_match_definition(case):
    d = _layer(*case)
    _assert_close(_run(d), d)


@pytest.mark.parametrize('case', [
    # enough groups that an item has two tiles of weight rows: narrow, middling and wide
    # sub-groups, an odd number of down tiles, scale rows of 4, 8 and 16-byte multiples
    ([1, 0, 3, 2] * 50, 128, 128, 5, 9, 4),
    ([5, 17, 33, 0, 40] * 10, 384, 512, 6, 50, 4),
    ([20, 60, 113] * 17, 384, 384, 4, 120, 8),
    ([1, 250, 48, 49, 64] * 10, 512, 512, 3, 90, 6),
    ([16] * 60, 640, 384, 2, 30, 3),
    ([30, 12, 33, 49] * 10, 256, 512, 3, 40, 4),
    ([64, 65, 20, 48, 1] * 10, 384, 512, 3, 70, 6),
], ids=lambda c: f'H{c[1]}_I{c[2]}_n{sum(c[0])}')
def test_experts_of_many_groups(case):
    d = _layer(*case)
    got = _run(d)
    _assert_close(got, d)
    assert torch.equal(got, _run(d))


@pytest.mark.parametrize('case', [
    # more groups than a block of the table's kernel has threads, with and without an
    # order by size; the widest rows either way; one group of many sub-groups
    ([1, 0, 20, 2, 0, 33] * 70, 128, 128, 3, 9, 4),
    ([0] * 300 + [2, 0, 1], 128, 256, 2, 5, 2),
    ([3], 65536, 128, 1, 3, 2),
    ([2, 1], 128, 65536, 2, 3, 2),
    ([4001], 128, 128, 1, 500, 8),
], ids=lambda c: f'G{len(c[0])}_H{c[1]}_I{c[2]}')
def test_experts_at_the_edges(case):
    d = _layer(*case)
    _assert_close(_run(d), d)


def test_bad_slots_among_many_groups():
    d = _layer([1, 0, 20, 2, 0, 33] * 70, 128, 128, 3, 9, 4)
    good = _run(d)
    slots = d['slots'].clone()
    slots[[2, 3, 417]] = torch.tensor([3, -1, 2 ** 40])
    slots[1] = 77  # of an empty group: not looked at
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = _run(dict(d, slots=slots), err=err)
    bad = torch.zeros(len(d['rows']), dtype=torch.bool)
    for g in (2, 3):
        bad[d['starts'][g]:d['starts'][g + 1]] = True
    bad[d['starts'][417]:d['starts'][418]] = True
    assert int(err) == 4 and bool(got[bad.to(DEV)].isnan().all())
    assert torch.equal(got[~bad.to(DEV)], good[~bad.to(DEV)])


def test_output_over_the_input():
    """out may be the rows that input was: they are read before any is written."""
    d = _layer([5, 60, 3], 256, 128, 3, 68, 1)
    d['rows'] = torch.randperm(68, generator=torch.Generator().manual_seed(1))
    d['cols'] = torch.zeros(68, dtype=torch.int64)
    want = _run(d)
    t = {k: d[k].to(DEV) for k in ('cache', 'x', 'w', 'slots', 'starts', 'rows', 'cols')}
    from ferry_b200 import expert_ops
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = expert_ops.execute_experts_mxfp4(t['cache'], t['x'], t['w'], t['slots'], t['starts'], t['rows'], t['cols'],
                                           256, 128, out=t['x'], err=err)
    assert got.data_ptr() == t['x'].data_ptr() and torch.equal(got, want) and int(err) == 0


def test_experts_weight_types_and_layout():
    from ferry_b200 import expert_ops
    d = _layer([9, 30, 2], 256, 256, 3, 20, 4)
    base = _run(d)
    for dtype in (BF16, torch.float16):
        e = dict(d, w=d['w'].to(dtype))
        _assert_close(_run(e), e)
    # strided and misaligned inputs, strided index tensors
    wide = torch.zeros(20, 300, dtype=BF16, device=DEV)
    for off in (0, 8, 3):
        x = wide[:, off:off + 256]
        x.copy_(d['x'])
        t = {k: d[k].to(DEV) for k in ('cache', 'w', 'slots', 'starts')}
        two = torch.stack((d['rows'], d['cols']), 1).to(DEV)
        got = expert_ops.execute_experts_mxfp4(t['cache'], x, t['w'], t['slots'], t['starts'], two[:, 0], two[:, 1],
                                               256, 256)
        assert torch.equal(got, base)
    assert torch.equal(_run(d), base)  # the same bits every time


def test_experts_scales_of_every_size():
    """Scale bytes above 128 (large blocks) take two multiplies; byte 0 and the
    smallest products vanish; byte 255 is NaN."""
    d = _layer([3, 20], 128, 128, 2, 8, 2, low=126, high=131)
    d['x'] = (d['x'].float() * 2.0 ** -12).to(BF16)
    _assert_close(_run(d), d)
    d = _layer([4], 128, 128, 1, 8, 2)
    n = 3 * 128 * 128
    d['cache'][0, n // 2 + 5] = 255   # one block of one gate row
    got = _run(d)
    assert bool(got.isnan().all())    # every output column sums over that activation
    d = _layer([4], 128, 128, 1, 8, 2)
    d['cache'][0, n // 2:] = 0
    assert bool((_run(d) == 0).all())


def test_experts_rows_of_no_group_stay():
    d = _layer([3, 0, 18], 128, 128, 2, 8, 2)
    more = 12
    d['rows'] = torch.cat((torch.zeros(4, dtype=torch.int64), d['rows'], torch.full((more - 4,), 10 ** 12)))
    d['cols'] = torch.cat((torch.zeros(4, dtype=torch.int64), d['cols'], torch.full((more - 4,), -5)))
    d['starts'] = d['starts'] + 4
    out = torch.full((len(d['rows']), 128), 3.0, dtype=BF16, device=DEV)
    got = _run(d, out=out)
    assert got is out
    assert bool((out[:4] == 3).all()) and bool((out[25:] == 3).all())
    _assert_close(out, d, slice(4, 25))
    # no group has a route
    d['starts'][:] = 4
    out.fill_(3.0)
    assert bool((_run(d, out=out) == 3).all())


def test_experts_device_errors():
    from ferry_b200._lib import FerrybError
    d = _layer([5, 6], 128, 128, 2, 8, 2)
    good = _run(d)
    for key, at, value in (('rows', 2, 8), ('rows', 7, -1), ('cols', 3, 2), ('cols', 3, -1), ('slots', 1, 2),
                           ('slots', 0, -1)):
        e = dict(d, **{key: d[key].clone()})
        e[key][at] = value
        with pytest.raises(FerrybError, match='out of range'):
            _run(e)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = _run(e, err=err)
        assert int(err) == 4
        bad = torch.zeros(11, dtype=torch.bool)
        if key == 'slots':
            bad[:5] = at == 0
            bad[5:] = at == 1
        else:
            bad[at] = True
        assert bool(got[bad.to(DEV)].isnan().all())
        assert torch.equal(got[~bad.to(DEV)], good[~bad.to(DEV)])
    for starts in ([0, 7, 5], [-1, 5, 11], [0, 5, 12], [5, 0, 11]):
        e = dict(d, starts=torch.tensor(starts))
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.full((11, 128), 3.0, dtype=BF16, device=DEV)
        _run(e, err=err, out=out)
        assert int(err) == 4 and bool((out == 3).all())
    assert torch.equal(_run(d), good)


def test_experts_overlapping_calls_and_graphs():
    """Two streams at once, and two captured graphs replayed against eager."""
    from ferry_b200 import expert_ops
    ds = [_layer([30, 1, 200], 256, 128, 3, 64, 4, seed=1), _layer([5, 130], 128, 256, 2, 64, 4, seed=2)]
    want = [_run(d) for d in ds]
    dev = [[d[k].to(DEV) for k in ('cache', 'x', 'w', 'slots', 'starts', 'rows', 'cols')] for d in ds]
    errs = [torch.zeros(1, dtype=torch.int32, device=DEV) for _ in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(expert_ops.execute_experts_mxfp4(*dev[i], ds[i]['hidden'], ds[i]['inter'], err=errs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i]) and int(errs[i]) == 0
    graphs, caught = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            caught.append(expert_ops.execute_experts_mxfp4(*dev[i], ds[i]['hidden'], ds[i]['inter'], err=errs[i]))
        graphs.append(g)
    for _ in range(2):
        for i in range(2):
            caught[i].zero_()
            with torch.cuda.stream(streams[i]):
                streams[i].wait_stream(torch.cuda.current_stream())
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(caught[i], want[i]) and int(errs[i]) == 0


def test_experts_empty_calls():
    d = _layer([2], 128, 128, 1, 4, 2)
    for e in (dict(d, rows=d['rows'][:0], cols=d['cols'][:0], starts=torch.zeros(2, dtype=torch.int64)),
              dict(d, rows=d['rows'][:0], cols=d['cols'][:0], slots=d['slots'][:0], starts=d['starts'][:1])):
        assert _run(e).shape == (0, 128)


def test_agrees_with_bf16_experts():
    """The same weights through execute_experts, whose bf16 gate, up and
    product roundings add three half steps to this operator's two."""
    from ferry_b200 import expert_ops
    from ferry_b200.model import mxfp4_parts
    d = _layer([4, 20], 256, 128, 2, 32, 4)
    rows = d['cache'].to(DEV)
    wide = expert_ops.dequantize_mxfp4(*mxfp4_parts(rows))
    w = d['w'].to(BF16)
    r, c = d['rows'].to(DEV), d['cols'].to(DEV)
    cut = d['starts'].tolist()
    old = torch.cat(expert_ops.execute_experts(wide, d['x'].to(DEV), w.to(DEV), d['slots'].tolist(),
                                               [r[a:b] for a, b in zip(cut, cut[1:])],
                                               [c[a:b] for a, b in zip(cut, cut[1:])], 256, 128)).float()
    new = _run(dict(d, w=w)).float()
    assert float((old - new).norm() / new.norm()) < 5 * 2.0 ** -8


def test_routed_layer_over_fetched_rows():
    """The operators as a serving layer uses them: a pool of quantised experts
    in pinned memory, the router's choices, the layout, the fetch, the experts
    and the weighted sum per token; against float64 on the same rows."""
    from ferry_b200 import expert_ops
    from ferry_b200.layout import LayoutBuffers
    from ferry_b200.model import mxfp4_parts, mxfp4_row_bytes
    T, E, K, H, I = 21, 16, 4, 256, 128
    g = torch.Generator(device=DEV).manual_seed(5)
    pool = torch.empty(E, mxfp4_row_bytes(H, I), dtype=torch.uint8).pin_memory()
    packed = torch.empty(pool.shape, dtype=torch.uint8, device=DEV)
    expert_ops.quantize_mxfp4(torch.randn(E, 3 * H * I, generator=g, device=DEV) * 0.05, out=mxfp4_parts(packed))
    pool.copy_(packed)
    x = torch.randn(T, H, generator=g, device=DEV).to(BF16)
    logits = torch.randn(T, E, generator=g, device=DEV)
    selected, weights = expert_ops.route_experts(logits, K, score='sigmoid', n_group=4, topk_group=2,
                                                 group_score='top2', bias=torch.linspace(0, .2, E, device=DEV),
                                                 weights_dtype=torch.float32)
    buf = LayoutBuffers(1, T, K, E, 0, DEV, fused=False)
    buf.run(selected.to(torch.uint8), torch.zeros(T, K, dtype=torch.int32, device=DEV))
    cache = torch.zeros_like(packed)
    slots = torch.randperm(E, generator=g, device=DEV)
    engine = expert_ops.H2DEngine(cache, pool)
    engine.fetch(slots.tolist(), list(range(E)))
    engine.wait_device(slots.tolist())
    out = expert_ops.execute_experts_mxfp4(cache, x, weights, slots, buf.starts, buf.rows, buf.cols, H, I)
    y = expert_ops.scatter_returned(out, buf.rows, T)
    d = dict(cache=pool, x=x.cpu(), w=weights.cpu(), slots=torch.arange(E), starts=buf.starts.cpu(),
             rows=buf.rows.cpu(), cols=buf.cols.cpu(), hidden=H, inter=I)
    _assert_close(out, d)
    want, bound = _want(d)
    total, slack = np.zeros((T, H)), np.zeros((T, H))
    np.add.at(total, d['rows'].numpy(), want)
    np.add.at(slack, d['rows'].numpy(), bound)
    # K float32 additions and one rounding to bf16 on top
    mag = np.zeros((T, H))
    np.add.at(mag, d['rows'].numpy(), np.abs(want) + bound)
    slack += K * 2.0 ** -24 * mag
    slack += 2.0 ** -8 * (np.abs(total) + slack)
    assert bool((np.abs(y.double().cpu().numpy() - total) <= slack).all())
    engine.close()


NARROW = ([1, 0, 20, 2, 33], 256, 128, 3, 40, 4)          # hi and lo parts side by side
WIDE = ([300, 64, 113], 128, 256, 2, 120, 4)              # one after the other
LONG_SCALES = ([40, 3, 90], 512, 512, 2, 60, 4)           # scale rows that go through TMA


def _assert_only_nan(d, bad, good):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = _run(d, err=err)
    bad = bad.to(DEV)
    assert int(err) == 0 and bool(bad.any()) and not bool(bad.all())
    assert bool(got[bad].isnan().all())
    assert torch.equal(got[~bad], good[~bad])


@pytest.mark.parametrize('case', [NARROW, WIDE, LONG_SCALES], ids=['narrow', 'wide', 'long'])
def test_a_row_that_is_not_finite_is_nan_and_leaves_the_others(case):
    """Infinities and NaN in inputs and routing weights, activations that overflow: the
    routes concerned are NaN in every column, their neighbours in a tile the same bits."""
    inf, nan = float('inf'), float('nan')
    d = _layer(*case)
    good = _run(d)
    assert bool(good.isfinite().all())
    row, col = int(d['rows'][len(d['rows']) // 2]), int(d['cols'][len(d['rows']) // 2])
    for at in (0, 31, 77, d['hidden'] - 1):
        for value in (inf, -inf, nan):
            x = d['x'].clone()
            x[row, at] = value
            _assert_only_nan(dict(d, x=x), d['rows'] == row, good)
    for value in (inf, -inf, nan):
        w = d['w'].clone()
        w[row, col] = value
        _assert_only_nan(dict(d, w=w), (d['rows'] == row) & (d['cols'] == col), good)
    # finite inputs: gate and up near 2^90, their product beyond float32
    x = d['x'].clone()
    x[row] = (x[row].float() * 2.0 ** 95).to(BF16)
    _assert_only_nan(dict(d, x=x), d['rows'] == row, good)
    # a finite activation times a finite weight
    x[row] = (d['x'][row].float() * 2.0 ** 40).to(BF16)
    w = d['w'].clone()
    w[row] = 2.0 ** 120
    _assert_only_nan(dict(d, x=x, w=w), d['rows'] == row, good)


@pytest.mark.parametrize('case', [NARROW, WIDE, LONG_SCALES], ids=['narrow', 'wide', 'long'])
@pytest.mark.parametrize('low,high,power', [(62, 66, 60), (190, 194, -70), (40, 200, -80), (5, 9, 118), (120, 134, 0)])
def test_experts_of_far_scales(case, low, high, power):
    """Scale bytes far from 127, alike and mixed in a row, under inputs that bring gate and
    up back near 1 (or below)."""
    d = _layer(*case, low=low, high=high)
    d['x'] = (d['x'].float() * 2.0 ** power).to(BF16)
    _assert_close(_run(d), d)


@pytest.mark.parametrize('case', [NARROW, WIDE], ids=['narrow', 'wide'])
def test_columns_far_apart_in_a_block(case):
    """Blocks of 32 whose values span 2^20: held to 2^-21 of the largest below 2^-13 of it."""
    d = _layer(*case)
    g = torch.Generator().manual_seed(9)
    d['x'] = (d['x'].float() * torch.exp2(-torch.randint(0, 21, d['x'].shape, generator=g).float())).to(BF16)
    d['w'] = d['w'] * torch.exp2(-torch.randint(0, 60, d['w'].shape, generator=g).float())
    _assert_close(_run(d), d)
