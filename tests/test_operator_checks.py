"""Refusals of route_experts, the MXFP4 operators and their C entry points, and
their ABI structs: no GPU."""
import ctypes

import numpy as np
import pytest
import torch

from ferry_b200 import _lib, expert_ops
from ferry_b200._lib import FerrybError
from ferry_b200.model import mxfp4_parts, mxfp4_row_bytes
from oracle import mxfp4 as ref

BF16 = torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(expert_ops, '_cuda_call', lambda dev, name, *args: seen.append((name, args)))
    monkeypatch.setattr(expert_ops, 'require_cuda', lambda *t: None)
    return seen


def test_cpu_tensors_are_refused():
    with pytest.raises(FerrybError, match='CUDA'):
        expert_ops.route_experts(torch.zeros(2, 8), 2)
    with pytest.raises(FerrybError, match='CUDA'):
        expert_ops.quantize_mxfp4(torch.zeros(2, 32))


def test_route_checks(calls):
    x = torch.zeros(3, 8)
    sel, w = expert_ops.route_experts(x, 2)
    assert sel.shape == w.shape == (3, 2) and w.dtype == BF16 and len(calls) == 1
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(topk=0), dict(topk=9), dict(score='tanh'),
                dict(group_score='sum'), dict(bias=torch.zeros(7)), dict(bias=torch.zeros(8, dtype=BF16)),
                dict(weights_dtype=torch.float64), dict(n_group=2**40)):
        args = dict(logits=x, topk=2)
        args.update(bad)
        with pytest.raises(FerrybError):
            expert_ops.route_experts(args.pop('logits'), args.pop('topk'), **args)
    assert len(calls) == 1


def _route_status(**change):
    a = _lib.RouteArgs(0x1000, 4, 64, 64, 4, 1, 1, 2, 0, 0, 0, 1, 1.0, 0, 0x1000, 0x1000)
    for k, v in change.items():
        setattr(a, k, v)
    return _lib.lib().ferryb_route_experts(ctypes.byref(a), None)


@pytest.mark.parametrize('change', [
    dict(tokens=-1), dict(experts=0), dict(experts=1025), dict(n_group=0), dict(n_group=33), dict(n_group=5),
    dict(topk_group=0), dict(topk_group=2), dict(topk=0), dict(topk=33), dict(n_group=32, topk=4, topk_group=1),
    dict(n_group=64), dict(score=2), dict(group_score=2), dict(n_group=32, experts=32, topk=1, group_score=1),
    dict(weights_type=3), dict(logits_type=3), dict(row_stride=63), dict(logits=0), dict(selected=0),
    dict(weights=0), dict(experts=1022, n_group=14, row_stride=1022),
], ids=str)
def test_route_refuses(change):
    assert _route_status(**change) == 1
    assert _lib.lib().ferryb_last_error()


def test_route_of_no_tokens_does_nothing():
    assert _route_status(tokens=0, logits=0) == 0


def test_quantize_checks(calls):
    x = torch.zeros(4, 64)
    codes, scales = expert_ops.quantize_mxfp4(x)
    assert codes.shape == (4, 32) and scales.shape == (4, 2)
    assert expert_ops.quantize_mxfp4(torch.zeros(2, 3, 64))[1].shape == (2, 3, 2)
    n = len(calls)
    for bad in (torch.zeros(4, 33), torch.zeros(4, 64, dtype=torch.float64), torch.zeros(())):
        with pytest.raises(FerrybError):
            expert_ops.quantize_mxfp4(bad)
    rows = torch.zeros(4, 34, dtype=torch.uint8)
    for out in ((codes[:3], scales), (codes, scales.float()), (codes[:, :31], scales), (codes.t().contiguous().t(), scales),
                (codes[:1].expand(4, 32), scales), (codes, scales.view(2, 4))):
        with pytest.raises(FerrybError):
            expert_ops.quantize_mxfp4(x, out=out)
    with pytest.raises(FerrybError, match='evenly'):
        expert_ops.quantize_mxfp4(torch.zeros(2, 2, 64), out=(
            torch.zeros(2, 3, 32, dtype=torch.uint8)[:, :2], torch.zeros(2, 2, 2, dtype=torch.uint8)))
    for c, s in ((codes, scales[:3]), (codes[:, :8], scales), (codes.int(), scales), (codes, scales.int())):
        with pytest.raises(FerrybError):
            expert_ops.dequantize_mxfp4(c, s)
    with pytest.raises(FerrybError):
        expert_ops.dequantize_mxfp4(codes, scales, torch.int32)
    with pytest.raises(FerrybError):
        expert_ops.dequantize_mxfp4(codes, scales, out=torch.zeros(4, 64))
    assert len(calls) == n
    expert_ops.quantize_mxfp4(x, out=mxfp4_parts(rows))
    assert len(calls) == n + 1


@pytest.mark.parametrize('change', [(0, 0), (1, 3), (1, -1), (2, -1), (3, 48), (3, -32), (4, 32), (5, 0), (6, 31), (7, 0),
                                    (8, 1), (0, 0x1001), (2, 1 << 41)], ids=str)
def test_quantize_entry_refuses(change):
    args = [0x1000, 1, 4, 64, 64, 0x1000, 32, 0x1000, 2]
    args[change[0]] = change[1]
    assert _lib.lib().ferryb_quantize_mxfp4(*args, None) == 1
    x, t, rows, width, stride, codes, cs, scales, ss = args
    assert _lib.lib().ferryb_dequantize_mxfp4(codes, cs, scales, ss, rows, width, x, t, stride, None) == 1


def _experts_args():
    H, I, K, T, G, R = 128, 256, 2, 6, 3, 9
    i64 = torch.int64
    return dict(cache=torch.zeros(2, mxfp4_row_bytes(H, I), dtype=torch.uint8), input=torch.zeros(T, H, dtype=BF16),
                routing_weights=torch.zeros(T, K), slots=torch.zeros(G, dtype=i64),
                starts=torch.zeros(G + 1, dtype=i64), rows=torch.zeros(R, dtype=i64), cols=torch.zeros(R, dtype=i64),
                hidden=H, intermediate=I, err=torch.zeros(1, dtype=torch.int32))


def test_experts_checks(calls):
    a = _experts_args()
    assert expert_ops.execute_experts_mxfp4(**a).shape == (9, 128) and len(calls) == 1
    bad = [dict(cache=a['cache'][:, :-1]), dict(cache=a['cache'].int()), dict(cache=a['cache'][:0]),
           dict(cache=a['cache'].view(-1)), dict(input=a['input'].float()), dict(input=a['input'][:, :64]),
           dict(routing_weights=a['routing_weights'][:5]), dict(routing_weights=a['routing_weights'].double()),
           dict(slots=a['slots'].int()), dict(slots=a['slots'][:2]), dict(starts=a['starts'][:3]),
           dict(starts=a['starts'].view(2, 2)), dict(rows=a['rows'].int()), dict(cols=a['cols'][:4]),
           dict(hidden=64), dict(hidden=0), dict(intermediate=200), dict(err=torch.zeros(2, dtype=torch.int32)),
           dict(err=torch.zeros(1)), dict(out=torch.zeros(9, 128)), dict(out=torch.zeros(8, 128, dtype=BF16)),
           dict(out=torch.zeros(128, 9, dtype=BF16).t())]
    for b in bad:
        with pytest.raises(FerrybError):
            expert_ops.execute_experts_mxfp4(**dict(a, **b))
    assert len(calls) == 1
    shifted = torch.zeros(2 * a['cache'].shape[1] + 16, dtype=torch.uint8)[1:-15].view(2, -1)
    with pytest.raises(FerrybError, match='aligned'):
        expert_ops.execute_experts_mxfp4(**dict(a, cache=shifted))
    assert expert_ops.execute_experts_mxfp4(**dict(a, rows=a['rows'][:0], cols=a['cols'][:0])).shape == (0, 128)


@pytest.mark.parametrize('change', [
    dict(hidden=100), dict(intermediate=0), dict(hidden=128 * 1024), dict(routes=-1), dict(n_groups=-1),
    dict(cache=0), dict(input=0), dict(out=0), dict(err=0), dict(workspace=0), dict(workspace=0x1010),
    dict(workspace_bytes=100), dict(cache_slots=0), dict(cache=0x1008), dict(input=0x1002), dict(input_stride=4),
    dict(input_stride=132), dict(weights_type=7), dict(routes=1 << 31),
    dict(routes=1 << 30, hidden=65536, intermediate=65536),
], ids=str)
def test_experts_entry_refuses(change):
    lib = _lib.lib()
    ws = lib.ferryb_execute_experts_mxfp4_workspace(9, 3, 128, 256)
    assert ws > 0
    a = _lib.Mxfp4ExpertsArgs(0x1000, 2, 0x1000, 6, 128, 0x1000, 2, 2, 0, 0x1000, 0x1000, 3, 0x1000, 0x1000, 9, 128,
                              256, 0x1000, 0x1000, ws, 0x1000)
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.ferryb_execute_experts_mxfp4(ctypes.byref(a), None) == 1
    assert lib.ferryb_last_error()
    assert lib.ferryb_execute_experts_mxfp4_workspace(1 << 31, 1, 128, 128) == -1


def test_struct_layouts(tmp_path):
    import subprocess
    from tests.test_abi import ROOT
    mirrors = {'ferryb_route_args': _lib.RouteArgs, 'ferryb_mxfp4_experts_args': _lib.Mxfp4ExpertsArgs}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "ferryb.h"', 'int main(void) {']
    for c, py in mirrors.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    (tmp_path / 'a.c').write_text('\n'.join(lines + ['return 0; }']))
    subprocess.run(['gcc', '-std=c99', '-Wall', '-Werror', f'-I{ROOT / "include"}', str(tmp_path / 'a.c'), '-o',
                    str(tmp_path / 'a')], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / 'a')], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for py in mirrors.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want


# ---- the oracle the GPU tests use ----

def test_oracle_quantize_by_search():
    """Nearest grid value by brute force, ties to the even code."""
    g = np.random.default_rng(0)
    x = np.concatenate([g.standard_normal((20, 32)) * 2.0 ** g.integers(-30, 30, (20, 1)),
                        np.tile([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5], (1, 4))])
    codes, scales = ref.quantize(x)
    v = ref.dequantize(codes, scales)
    for row, got, s in zip(x, v, scales[:, 0]):
        unit = 2.0 ** (int(s) - 127)
        assert 4 * unit <= np.abs(row).max() < 8 * unit
        d = np.abs(np.abs(row[:, None]) / unit - ref.GRID)
        best = d.min(1, keepdims=True)
        pick = [min(np.flatnonzero(r == b), key=lambda c: c % 2) for r, b in zip(d, best[:, 0])]
        np.testing.assert_array_equal(np.abs(got) / unit, ref.GRID[pick])
        assert (np.sign(got) * np.sign(row) >= 0).all()


def test_row_parts():
    rows = torch.arange(2 * mxfp4_row_bytes(128, 64)).view(2, -1)
    codes, scales = mxfp4_parts(rows)
    assert codes.shape == (2, 3 * 128 * 64 // 2) and scales.shape == (2, 3 * 128 * 64 // 32)
    assert codes.data_ptr() == rows.data_ptr() and int(scales[0, 0]) == codes.shape[1]


def test_the_extension_leaves_what_is_not_plain():
    """Built with the library; anything but plain CUDA tensors is left to the Python checks."""
    fast = _lib.fast()
    assert fast.__name__ == 'ferry_b200._fast'
    x, v = torch.zeros(2, 32), torch.zeros(3, dtype=torch.int64)
    assert fast.route_experts(x, 2, 'softmax', None, 1, 1, 'max', True, 1.0, BF16) is None
    assert fast.quantize_mxfp4(x) is None and fast.dequantize_mxfp4(x, x, BF16) is None
    assert fast.execute_experts_mxfp4(x, x, x, v, v, v, v, 128, 128, None, None) is None
    for bad in (None, 7, 'x', [x]):
        assert fast.quantize_mxfp4(bad) is None and fast.dequantize_mxfp4(bad, x, BF16) is None
        assert fast.route_experts(bad, 2, 'softmax', None, 1, 1, 'max', True, 1.0, BF16) is None
        assert fast.execute_experts_mxfp4(x, bad, x, v, v, v, v, 128, 128, None, None) is None
    assert fast.route_experts() is None and fast.route_experts(x) is None


def test_experts_output_at_an_odd_element_is_refused(calls):
    """The kernel stores bf16 pairs; contiguous views may start at any element."""
    a = _experts_args()
    buf = torch.zeros(9 * 128 + 2, dtype=BF16)
    with pytest.raises(FerrybError, match='4-byte aligned'):
        expert_ops.execute_experts_mxfp4(**dict(a, out=buf[1:-1].view(9, 128)))
    assert not calls
    expert_ops.execute_experts_mxfp4(**dict(a, out=buf[2:].view(9, 128)))
    assert len(calls) == 1


@pytest.mark.parametrize('change', [dict(out=0x1002), dict(out=0x1001), dict(err=0x1002), dict(slots=0x1004),
                                    dict(starts=0x1004), dict(rows=0x1004), dict(cols=0x1004),
                                    dict(routing_weights=0x1002)], ids=str)
def test_experts_entry_refuses_misaligned_pointers(change):
    lib = _lib.lib()
    ws = lib.ferryb_execute_experts_mxfp4_workspace(9, 3, 128, 256)
    a = _lib.Mxfp4ExpertsArgs(0x1000, 2, 0x1000, 6, 128, 0x1000, 2, 2, 0, 0x1000, 0x1000, 3, 0x1000, 0x1000, 9, 128,
                              256, 0x1000, 0x1000, ws, 0x1000)
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.ferryb_execute_experts_mxfp4(ctypes.byref(a), None) == 1
    assert b'aligned' in lib.ferryb_last_error()


@pytest.mark.parametrize('scaling', [1e39, -1e39, 3.4028235677973366e38, 1.7e308])
def test_route_refuses_a_scaling_beyond_float32(calls, scaling):
    with pytest.raises(FerrybError, match='scaling'):
        expert_ops.route_experts(torch.zeros(3, 8), 2, scaling=scaling)
    assert not calls
    expert_ops.route_experts(torch.zeros(3, 8), 2, scaling=float('inf'))
    expert_ops.route_experts(torch.zeros(3, 8), 2, scaling=-3.4028234663852886e38)
    assert len(calls) == 2


def test_packing_refuses_blocks_across_rows(calls):
    """Blocks of 32 run along H and I: other sizes would share scales between rows."""
    from ferry_b200.model import pack_expert_mxfp4
    w = torch.zeros
    for I, H in ((2, 16), (32, 48), (48, 32), (1, 32), (96, 80)):
        with pytest.raises(FerrybError, match='multiples of 32'):
            pack_expert_mxfp4(w(I, H), w(I, H), w(H, I))
        with pytest.raises(FerrybError, match='multiples of 32'):
            mxfp4_row_bytes(H, I)
    for gate, up, down in (((32, 64), (64, 32), (64, 32)), ((32, 64), (32, 64), (32, 64)), ((2048,), (2048,), (2048,))):
        with pytest.raises(FerrybError, match='gate'):
            pack_expert_mxfp4(w(gate), w(up), w(down))
    assert not calls
    assert pack_expert_mxfp4(w(32, 64), w(32, 64), w(64, 32)).shape == (mxfp4_row_bytes(64, 32),)
    assert len(calls) == 1


def test_parts_of_what_is_no_row():
    for n in (0, 16, 18, 16 * 17 + 1):
        with pytest.raises(FerrybError, match='17'):
            mxfp4_parts(torch.zeros(3, n, dtype=torch.uint8))


@pytest.mark.parametrize('change', [dict(logits=0x1002), dict(logits=0x1001, logits_type=0), dict(bias=0x1002),
                                    dict(selected=0x1004), dict(weights=0x1001), dict(weights=0x1002, weights_type=2)],
                         ids=str)
def test_route_entry_refuses_misaligned_pointers(change):
    assert _route_status(**change) == 1
    assert b'aligned' in _lib.lib().ferryb_last_error()
