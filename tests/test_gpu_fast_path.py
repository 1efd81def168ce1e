"""The short way into the operators (csrc/expert_ops_fast.cpp) and the Python
one around it: the same bits, and what the short way leaves is answered all
the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
BF16 = torch.bfloat16


@pytest.fixture
def taken(monkeypatch):
    """Which calls the extension answered."""
    from ferry_b200 import _lib
    real, seen = _lib.fast(), {}

    def wrap(name):
        def f(*args):
            out = getattr(real, name)(*args)
            seen[name] = out is not None
            return out
        return staticmethod(f)
    names = ('route_experts', 'quantize_mxfp4', 'dequantize_mxfp4', 'execute_experts_mxfp4')
    monkeypatch.setattr(_lib, '_fast', type('Watched', (), {n: wrap(n) for n in names}))
    return seen


def _both(monkeypatch, f):
    from ferry_b200 import _lib
    short = f()
    with monkeypatch.context() as m:
        m.setattr(_lib, '_fast', _lib._NoFast)
        long = f()
    return short, long


@pytest.mark.parametrize('dtype', [BF16, torch.float16, torch.float32], ids=str)
def test_route(taken, monkeypatch, dtype):
    from ferry_b200 import expert_ops
    wide = torch.randn(9, 80, device=DEV).to(dtype)
    for x in (wide, wide[:, 8:72], wide[:1, :1], wide[::2, :64]):
        bias = torch.randn(x.shape[1], device=DEV)
        for kw in (dict(), dict(score='sigmoid', bias=bias, weights_dtype=torch.float32, norm_topk_prob=False,
                                scaling=2.5)):
            (a, v), (b, w) = _both(monkeypatch, lambda: expert_ops.route_experts(x, 1, **kw))
            assert taken['route_experts'] and torch.equal(a, b) and torch.equal(v, w)
            assert a.shape == b.shape and v.dtype == w.dtype
    sel, w = expert_ops.route_experts(wide.t(), 3)  # columns adjacent: copied first
    assert not taken['route_experts']
    want = expert_ops.route_experts(wide.t().contiguous(), 3)
    assert torch.equal(sel, want[0]) and torch.equal(w, want[1])


@pytest.mark.parametrize('dtype', [BF16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize('shape', [(32,), (1, 64), (5, 96), (2, 3, 32)], ids=str)
def test_quantize(taken, monkeypatch, dtype, shape):
    from ferry_b200 import expert_ops
    x = torch.randn(shape, device=DEV).to(dtype)
    (c, s), (d, t) = _both(monkeypatch, lambda: expert_ops.quantize_mxfp4(x))
    assert taken['quantize_mxfp4'] and torch.equal(c, d) and torch.equal(s, t)
    y, z = _both(monkeypatch, lambda: expert_ops.dequantize_mxfp4(c, s, dtype))
    assert taken['dequantize_mxfp4'] and y.dtype == dtype and torch.equal(y, z) and y.shape == x.shape
    wide = torch.randn(4, 160, device=DEV).to(dtype)
    (c, s), (d, t) = _both(monkeypatch, lambda: expert_ops.quantize_mxfp4(wide[:, 32:96]))
    assert taken['quantize_mxfp4'] and torch.equal(c, d) and torch.equal(s, t)
    (c, s), (d, t) = _both(monkeypatch, lambda: expert_ops.quantize_mxfp4(wide.t()[:64, :].t()))
    assert torch.equal(c, d) and torch.equal(s, t)
    (c, s), _ = _both(monkeypatch, lambda: expert_ops.quantize_mxfp4(wide.reshape(160, 4).t()))
    assert not taken['quantize_mxfp4'] and c.shape == (4, 80)
    with pytest.raises(RuntimeError, match='multiple of 32'):
        expert_ops.quantize_mxfp4(wide[:, :48])


def test_experts(taken, monkeypatch):
    from ferry_b200 import expert_ops
    from ferry_b200.model import mxfp4_row_bytes
    H, I, slots = 256, 128, 3
    cache = torch.randint(0, 256, (slots, mxfp4_row_bytes(H, I)), dtype=torch.uint8, device=DEV)
    cache[:, 3 * H * I // 2:] = 118
    x = torch.randn(7, H, device=DEV).to(BF16)
    w = torch.rand(7, 4, device=DEV)
    ids = lambda *v: torch.tensor(v, device=DEV)
    t = [cache, x, w, ids(2, 0), ids(0, 3, 5), ids(0, 6, 2, 2, 1), ids(0, 1, 3, 3, 2)]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    a, b = _both(monkeypatch, lambda: expert_ops.execute_experts_mxfp4(*t, H, I, err=err))
    assert taken['execute_experts_mxfp4'] and torch.equal(a, b) and int(err) == 0
    out = torch.empty(5, H, dtype=BF16, device=DEV)
    assert expert_ops.execute_experts_mxfp4(*t, H, I, err=err, out=out).data_ptr() == out.data_ptr()
    assert taken['execute_experts_mxfp4'] and torch.equal(out, a)
    assert torch.equal(expert_ops.execute_experts_mxfp4(*t, H, I), a)  # waits, and raises on errors
    assert not taken['execute_experts_mxfp4']
    for i, bad in ((0, cache[:, :-1]), (1, x.float()), (2, w[:5]), (3, t[3].int()), (4, t[4][:2]), (6, t[6][:4])):
        with pytest.raises(RuntimeError):
            expert_ops.execute_experts_mxfp4(*t[:i], bad, *t[i + 1:], H, I, err=err)
    t[5] = ids(0, 7, 2, 2, 1)  # no such row
    got = expert_ops.execute_experts_mxfp4(*t, H, I, err=err)
    assert int(err) == 4 and bool(got[1].isnan().all()) and torch.equal(got[0], a[0])


def test_streams_and_graphs(taken):
    """Launched on the current stream, and capturable."""
    from ferry_b200 import expert_ops
    x = torch.randn(33, 128, device=DEV)
    want = expert_ops.route_experts(x, 8)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        y = x * 1
        got = expert_ops.route_experts(y, 8)
    side.synchronize()
    assert taken['route_experts'] and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c, s = expert_ops.quantize_mxfp4(x)
        back = expert_ops.dequantize_mxfp4(c, s, torch.float32)
    x.mul_(3)
    g.replay()
    assert torch.equal(back, expert_ops.dequantize_mxfp4(*expert_ops.quantize_mxfp4(x), torch.float32))


def test_offsets_beyond_32_bits(taken):
    """Rows further than 2^32 elements apart, and a cache slot that starts beyond 4 GiB."""
    from ferry_b200 import expert_ops
    from ferry_b200.model import mxfp4_row_bytes
    far = 2 ** 32 + 64
    x = torch.empty(far + 64, dtype=BF16, device=DEV).as_strided((2, 64), (far, 1))
    x.copy_(torch.randn(2, 64))
    near = x.contiguous()
    for got, want in zip(expert_ops.route_experts(x, 4), expert_ops.route_experts(near, 4)):
        assert torch.equal(got, want)
    codes, scales = expert_ops.quantize_mxfp4(x)
    assert taken['route_experts'] and taken['quantize_mxfp4']
    for got, want in zip((codes, scales), expert_ops.quantize_mxfp4(near)):
        assert torch.equal(got, want)
    expert_ops.dequantize_mxfp4(codes, scales, BF16, out=x)
    assert torch.equal(x, expert_ops.dequantize_mxfp4(codes, scales))
    del x
    H, I = 2048, 1408
    size = mxfp4_row_bytes(H, I)
    slots = 2 ** 32 // size + 3
    cache = torch.empty(slots, size, dtype=torch.uint8, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    cache[0] = torch.randint(0, 256, (size,), generator=g, dtype=torch.uint8, device=DEV)
    cache[0, 3 * H * I // 2:] = 117
    cache[-1] = cache[0]
    y = torch.randn(3, H, device=DEV).to(BF16)
    w = torch.rand(3, 1, device=DEV)
    rows, cols = torch.arange(3, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    starts, err = torch.tensor([0, 3], device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    a, b = (expert_ops.execute_experts_mxfp4(cache, y, w, torch.tensor([s], device=DEV), starts, rows, cols, H, I,
                                             err=err) for s in (0, slots - 1))
    assert int(err) == 0 and torch.equal(a, b) and bool((a != 0).any())


def test_back_to_back_calls_see_each_other():
    """A chain in which each launch reads what the one before it wrote, far longer
    than the launch queue's overlap."""
    from ferry_b200 import expert_ops
    x = torch.randn(64, 4096, device=DEV)
    want = expert_ops.dequantize_mxfp4(*expert_ops.quantize_mxfp4(x), torch.float32)
    y = x
    for _ in range(50):
        y = expert_ops.dequantize_mxfp4(*expert_ops.quantize_mxfp4(y), torch.float32)  # quantised values stay
    assert torch.equal(y, want)
    for _ in range(50):
        y = y * -1                        # a kernel of torch between
        c, s = expert_ops.quantize_mxfp4(y)
        y = expert_ops.dequantize_mxfp4(c, s, torch.float32)
        sel, w = expert_ops.route_experts(y[:, :128], 2)
    assert torch.equal(y, want)
    assert torch.equal(sel, expert_ops.route_experts(want[:, :128].contiguous(), 2)[0])


def test_output_at_an_odd_element_is_refused(taken):
    """Before anything is launched, by the short way too."""
    from ferry_b200 import expert_ops
    from ferry_b200.model import mxfp4_row_bytes
    H, I = 128, 128
    cache = torch.full((1, mxfp4_row_bytes(H, I)), 118, dtype=torch.uint8, device=DEV)
    x, w = torch.randn(3, H, device=DEV).to(BF16), torch.rand(3, 1, device=DEV)
    ids = lambda *v: torch.tensor(v, device=DEV)
    args = (cache, x, w, ids(0), ids(0, 3), ids(0, 1, 2), ids(0, 0, 0), H, I)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    buf = torch.full((3 * H + 4,), 7.0, dtype=BF16, device=DEV)
    for kw in (dict(), dict(err=err)):
        with pytest.raises(RuntimeError, match='4-byte aligned'):
            expert_ops.execute_experts_mxfp4(*args, out=buf[1:1 + 3 * H].view(3, H), **kw)
        assert not taken['execute_experts_mxfp4'] and bool((buf == 7).all())
    got = expert_ops.execute_experts_mxfp4(*args, out=buf[2:2 + 3 * H].view(3, H), err=err)
    assert taken['execute_experts_mxfp4'] and torch.equal(got, expert_ops.execute_experts_mxfp4(*args))
    assert bool((buf[:2] == 7).all()) and bool((buf[2 + 3 * H:] == 7).all()) and int(err) == 0


@pytest.mark.parametrize('scaling', [1e39, -1e39, 3.4028235677973366e38, 1.7e308])
def test_scaling_beyond_float32_is_refused_by_both_ways(taken, scaling):
    from ferry_b200 import expert_ops
    x = torch.randn(3, 16, device=DEV)
    with pytest.raises(RuntimeError, match='scaling'):
        expert_ops.route_experts(x, 2, scaling=scaling)
    assert not taken['route_experts']


@pytest.mark.parametrize('scaling', [3.4028234663852886e38, -3.4028235e38, float('inf'), float('nan'), 0.0, 1e-46])
def test_scaling_at_the_ends_of_float32(taken, monkeypatch, scaling):
    from ferry_b200 import expert_ops
    x = torch.randn(3, 16, device=DEV)
    (a, v), (b, w) = _both(monkeypatch, lambda: expert_ops.route_experts(x, 2, scaling=scaling,
                                                                         weights_dtype=torch.float32))
    assert torch.equal(a, b) and torch.equal(v.nan_to_num(7.0), w.nan_to_num(7.0))
