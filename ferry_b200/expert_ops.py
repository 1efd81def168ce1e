"""Drop-in for the reference's native module ``ferry_expert_ops``
(ferry/csrc/expert_ops.cpp:144-157): same function names, argument meaning
and error behaviour (RuntimeError on bad input), backed by libferryb's sm_100a
kernels through the C ABI.  Outputs are allocated by the torch caching
allocator; inputs are borrowed.

Beside them, operators the reference has no counterpart of: route_experts
(softmax or sigmoid routers with a balance bias and groups),
quantize_mxfp4 / dequantize_mxfp4 (4-bit weight rows) and
execute_experts_mxfp4 (the routed experts over such rows).  They run on the
device and current stream of their tensors, allocate only their outputs and
workspace, and neither copy to the host nor wait for the GPU, so they can be
captured into a CUDA graph.
"""
import ctypes
import functools
import math
import struct

import torch

from . import _lib
from ._lib import call, ptr, require_cuda, stream_ptr

BF16 = torch.bfloat16


def _check(cond, msg):
    if not cond:
        raise _lib.FerrybError(msg)


def execute_experts(cache, input, routing_weights, slots, rows, cols, hidden, intermediate):
    """ferry/csrc/expert_ops.cpp:16-45.  Returns one [len(rows[i]), hidden] bf16
    tensor per group: (silu(x Wg^T) * (x Wu^T)) Wd^T * w[rows, cols]."""
    require_cuda(cache, input, routing_weights)
    _check(cache.dtype == BF16 and input.dtype == BF16 and routing_weights.dtype == BF16,
           'cache, input and routing_weights must be bf16')
    _check(cache.dim() == 2 and cache.is_contiguous() and cache.shape[1] == 3 * hidden * intermediate,
           'cache must be contiguous [slots, 3*hidden*intermediate]')
    _check(input.dim() == 2 and input.shape[1] == hidden, 'input must be [n, hidden]')
    _check(routing_weights.dim() == 2 and routing_weights.shape[0] == input.shape[0],
           'routing_weights must be [n, topk]')
    _check(len(slots) == len(rows) == len(cols), 'slots, rows and cols must have equal length')
    sizes = []
    for r, c in zip(rows, cols):
        _check(r.dtype == torch.long and c.shape == r.shape, 'rows/cols must be matching int64')
        sizes.append(int(r.numel()))
    total = sum(sizes)
    out = torch.empty((total, hidden), dtype=BF16, device=input.device)
    if total:
        input_c = input.contiguous()
        rw = routing_weights.contiguous()
        rows_c = torch.cat([r.reshape(-1) for r in rows]).to(input.device)
        cols_c = torch.cat([c.reshape(-1) for c in cols]).to(input.device)
        n_groups = len(slots)
        ws_bytes = _lib.lib().ferryb_execute_experts_workspace(total, n_groups, hidden, intermediate)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=input.device)
        call('ferryb_execute_experts', ptr(cache), cache.shape[0], ptr(input_c), input_c.shape[0],
             ptr(rw), rw.shape[1], _lib.host_i64(slots), _lib.host_i64(sizes), n_groups,
             ptr(rows_c), ptr(cols_c), hidden, intermediate, ptr(out), ptr(ws), ws_bytes,
             stream_ptr(input.device))
    return list(out.split(sizes)) if sizes else []


def pack_dispatch(hidden, selected, weights, send_idx, send_ids, experts):
    """ferry/csrc/expert_ops.cpp:50-66 -> uint8 [n, 2H + 3k] packets."""
    require_cuda(hidden, selected, weights, send_idx, send_ids)
    _check(hidden.dtype == BF16 and weights.dtype == BF16, 'hidden and weights must be bf16')
    _check(hidden.dim() == 2 and selected.dim() == 2 and send_idx.dim() == 1 and send_ids.dim() == 2,
           'hidden, selected and send_ids must be 2-D, send_idx 1-D')
    n, h, k = send_idx.shape[0], hidden.shape[1], send_ids.shape[1]
    _check(selected.shape == (hidden.shape[0], k) and weights.shape == selected.shape
           and send_ids.shape[0] == n, 'selected/weights must be [tokens, k], send_ids [n, k]')
    payload = torch.empty((n, 2 * h + 3 * k), dtype=torch.uint8, device=hidden.device)
    if n:
        hid = hidden.contiguous()
        sel = selected.contiguous().long()
        w = weights.contiguous()
        si, sids = send_idx.contiguous().long(), send_ids.contiguous().long()
        err = torch.zeros(1, dtype=torch.int32, device=hidden.device)
        call('ferryb_pack_dispatch', ptr(hid), hid.shape[0], h, ptr(sel), ptr(w), k, ptr(si),
             ptr(sids), n, experts, ptr(payload), ptr(err), stream_ptr(hidden.device))
        _lib.check_device_error(err, 'pack_dispatch')
    return payload


def unpack_dispatch(raw, hidden, topk):
    """ferry/csrc/expert_ops.cpp:68-73 -> (x [m, H] bf16, w [m, k] bf16)."""
    require_cuda(raw)
    _check(raw.dtype == torch.uint8 and raw.dim() == 2 and raw.shape[1] == 2 * hidden + 3 * topk,
           f'raw must be uint8 [m, 2*hidden + 3*topk = {2 * hidden + 3 * topk}]')
    m = raw.shape[0]
    x = torch.empty((m, hidden), dtype=BF16, device=raw.device)
    w = torch.empty((m, topk), dtype=BF16, device=raw.device)
    if m:
        r = raw.contiguous()
        call('ferryb_unpack_dispatch', ptr(r), m, hidden, topk, ptr(x), ptr(w), stream_ptr(raw.device))
    return x, w


def reduce_partials(parts, rows, received, hidden, like):
    """ferry/csrc/expert_ops.cpp:76-83: float32 sum of the groups' outputs per
    receive row (in group order), returned as bf16 [received, hidden]."""
    require_cuda(like, *parts)
    _check(len(parts) == len(rows), 'parts and rows must have equal length')
    for p, r in zip(parts, rows):
        _check(p.dim() == 2 and p.shape[1] == hidden and p.shape[0] == r.numel(),
               'each part must be [len(rows[i]), hidden]')
    if not parts:
        return torch.zeros((received, hidden), dtype=BF16, device=like.device)
    src = torch.cat([p.to(BF16) for p in parts])
    keys = torch.cat([r.reshape(-1) for r in rows]).to(like.device)
    if src.shape[0] == 0:
        return torch.zeros((received, hidden), dtype=BF16, device=like.device)
    out = torch.empty((received, hidden), dtype=BF16, device=like.device)
    ws_bytes = _lib.lib().ferryb_segment_sum_workspace(src.shape[0], received)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=like.device)
    call('ferryb_reduce_partials', ptr(src), ptr(keys.long()), src.shape[0], received, hidden,
         ptr(out), ptr(ws), ws_bytes, stream_ptr(like.device))
    return out


def scatter_returned(returned, send_idx, tokens):
    """ferry/csrc/expert_ops.cpp:86-92: float32 sum of returned partials per
    token (in packet order), bf16 [tokens, hidden]."""
    require_cuda(returned, send_idx)
    _check(returned.dim() == 2 and send_idx.numel() == returned.shape[0],
           'returned must be [n, hidden] with one send_idx per row')
    hidden = returned.shape[1]
    if returned.shape[0] == 0:
        return torch.zeros((tokens, hidden), dtype=returned.dtype, device=returned.device)
    out = torch.empty((tokens, hidden), dtype=BF16, device=returned.device)
    ret = returned.contiguous().to(BF16)
    idx = send_idx.contiguous().long()
    ws_bytes = _lib.lib().ferryb_segment_sum_workspace(ret.shape[0], tokens)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=returned.device)
    call('ferryb_scatter_returned', ptr(ret), ptr(idx), ret.shape[0], tokens, hidden, ptr(out),
         ptr(ws), ws_bytes, stream_ptr(returned.device))
    return out.to(returned.dtype)


def _cuda_call(device, name, *args):
    """call() on `device`'s current stream, whatever the current device is."""
    # the raw stream costs a tenth of a microsecond, a torch.cuda.Stream three
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        call(name, *args, stream)
    else:
        with torch.cuda.device(device):
            call(name, *args, stream)


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise _lib.FerrybError(f'{name} is on {t.device}, expected {device}')


def _dense_rows(t):
    """2-D t itself if the values of a row are adjacent and its rows do not
    overlap, else a contiguous copy."""
    if t.is_contiguous():
        return t
    rows, width = t.shape
    stride, step = t.stride()
    return t if (step == 1 or width <= 1) and (stride >= width or rows <= 1) else t.contiguous()


SCORES = {'softmax': 0, 'sigmoid': 1}
GROUP_SCORES = {'max': 0, 'top2': 1}


def route_experts(logits, topk, *, score='softmax', bias=None, n_group=1, topk_group=1,
                  group_score='max', norm_topk_prob=True, scaling=1.0, weights_dtype=BF16):
    """Top-k routing from router logits [tokens, experts] (bf16, fp16 or
    float32): (selected int64 [tokens, topk], weights [tokens, topk]), as
    OffloadRuntime.execute takes them.

    The scores are softmax(logits) or sigmoid(logits) (`score`); `bias`
    (float32 [experts]) is added for the selection only.  With n_group > 1,
    groups of consecutive experts, the topk_group groups of the largest
    biased score (group_score 'max') or sum of their two largest ('top2')
    stay.  The topk largest biased scores are selected, descending, ties to
    the lower id.  The weights are the unbiased scores, divided by their sum
    with norm_topk_prob, times `scaling` (a float32).  -inf logits mask experts with
    softmax (a row of nothing else has weights 0); NaN scores are taken last
    and give NaN weights.  Scores are compared in 64 bits.  At most 1024
    experts, topk <= 32, n_group <= 32, and in a group at most 32 * (the power of
    two <= 32 / n_group) experts: 1024 for one group, 512 for 2, 256 for 3 and 4,
    128 up to 8, 64 up to 16, 32 above."""
    done = _lib.fast().route_experts(logits, topk, score, bias, n_group, topk_group, group_score, norm_topk_prob,
                                     scaling, weights_dtype)
    if done is not None:
        return done
    require_cuda(logits, bias)
    logits_type, weights_type = _lib.ELEMENT_TYPES.get(logits.dtype), _lib.ELEMENT_TYPES.get(weights_dtype)
    if logits_type is None or logits.dim() != 2:
        raise _lib.FerrybError('logits must be bf16, fp16 or float32 [tokens, experts]')
    if weights_type is None:
        raise _lib.FerrybError('weights_dtype must be bf16, fp16 or float32')
    if score not in SCORES:
        raise _lib.FerrybError(f'score must be one of {sorted(SCORES)}')
    if group_score not in GROUP_SCORES:
        raise _lib.FerrybError(f'group_score must be one of {sorted(GROUP_SCORES)}')
    tokens, experts = logits.shape
    dev = logits.device
    if bias is not None:
        _check(bias.dtype == torch.float32 and bias.shape == (experts,), 'bias must be float32 [experts]')
        _same_device(dev, bias=bias)
        bias = bias.contiguous()
    logits = _dense_rows(logits)
    topk = int(topk)
    if not 0 < topk <= experts:
        raise _lib.FerrybError(f'topk must be in [1, {experts}]')
    scaling = float(scaling)
    if math.isinf(ctypes.c_float(scaling).value) and not math.isinf(scaling):
        raise _lib.FerrybError(f'scaling ({scaling}) is beyond float32')
    selected = logits.new_empty((tokens, topk), dtype=torch.int64)
    weights = logits.new_empty((tokens, topk), dtype=weights_dtype)
    try:
        args = _lib.pack_route_args(
            logits.data_ptr(), tokens, logits.stride(0), experts, topk, int(n_group), int(topk_group), logits_type,
            weights_type, SCORES[score], GROUP_SCORES[group_score], int(bool(norm_topk_prob)), scaling,
            _lib.addr(bias), selected.data_ptr(), weights.data_ptr())
    except (struct.error, OverflowError):
        raise _lib.FerrybError(f'n_group ({n_group}) or topk_group ({topk_group}) is too large') from None
    _cuda_call(dev, 'ferryb_route_experts', args)
    return selected, weights


def _rows_2d(t, name):
    """t as [rows, width] without a copy, the values of a row adjacent."""
    if t.dim() != 2:
        try:
            t = t.view(-1, t.shape[-1])
        except RuntimeError:
            raise _lib.FerrybError(f'{name}: the rows must be evenly spaced, their values adjacent') from None
    rows, width = t.shape
    stride, step = t.stride()
    if step != 1 and width > 1:
        raise _lib.FerrybError(f'{name}: the values of a row must be adjacent')
    if stride < width and rows > 1:
        raise _lib.FerrybError(f'{name}: rows overlap')
    return t


def _mxfp4_out(out, x):
    """(codes, scales) for the values of x: `out` checked, or new tensors."""
    *lead, width = x.shape
    if out is None:
        return (x.new_empty((*lead, width // 2), dtype=torch.uint8),
                x.new_empty((*lead, width // 32), dtype=torch.uint8))
    codes, scales = out
    for name, t, n in (('codes', codes, width // 2), ('scales', scales, width // 32)):
        if t.dtype != torch.uint8 or t.shape != (*lead, n):
            raise _lib.FerrybError(f'{name} must be uint8 {[*lead, n]}, got {t.dtype} {list(t.shape)}')
        _same_device(x.device, **{name: t})
    return codes, scales


def quantize_mxfp4(x, out=None):
    """MXFP4 of the last dimension of x (bf16, fp16 or float32, a multiple of
    32 values): (codes uint8 [..., width / 2], scales uint8 [..., width / 32]).

    Every 32 values share a power of two 2^(s - 127), s = the float32 exponent
    field of their largest magnitude minus 2 (at least 0); a code is the value
    over it, rounded half to even to {0, 0.5, 1, 1.5, 2, 3, 4, 6} and a sign,
    two codes a byte, the lower nibble first.  A block holding an infinity or
    a NaN has s = 255 and reads back as NaN.  `out`: (codes, scales) to write
    to, such as the two parts of expert rows (ferry_b200.model.mxfp4_parts)."""
    done = _lib.fast().quantize_mxfp4(x) if out is None else None
    if done is not None:
        return done
    require_cuda(x)
    kind = _lib.ELEMENT_TYPES.get(x.dtype)
    if kind is None or x.dim() < 1:
        raise _lib.FerrybError('x must be bf16, fp16 or float32')
    width = x.shape[-1]
    if width % 32:
        raise _lib.FerrybError(f'the last dimension ({width}) must be a multiple of 32')
    codes, scales = _mxfp4_out(out, x)
    if x.numel() == 0:
        return codes, scales
    x2 = _dense_rows(x if x.dim() == 2 else x.reshape(-1, width))
    code_stride, scale_stride = width // 2, width // 32
    if out is not None:
        code_stride = _rows_2d(codes, 'codes').stride(0)
        scale_stride = _rows_2d(scales, 'scales').stride(0)
    _cuda_call(x.device, 'ferryb_quantize_mxfp4', x2.data_ptr(), kind, x2.shape[0], width, x2.stride(0),
               codes.data_ptr(), code_stride, scales.data_ptr(), scale_stride)
    return codes, scales


def dequantize_mxfp4(codes, scales, dtype=BF16, out=None):
    """The values of quantize_mxfp4's codes and scales, rounded once to `dtype`
    (bf16 and float32 hold them exactly, but for 6 * 2^127 and its like)."""
    done = _lib.fast().dequantize_mxfp4(codes, scales, dtype) if out is None else None
    if done is not None:
        return done
    require_cuda(codes, scales, out)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() < 1:
        raise _lib.FerrybError('codes and scales must be uint8')
    *lead, half = codes.shape
    width = 2 * half
    if width % 32 or scales.shape != (*lead, width // 32):
        raise _lib.FerrybError(f'codes {list(codes.shape)} need scales {[*lead, width // 32]} '
                               f'(blocks of 32 values), got {list(scales.shape)}')
    kind = _lib.ELEMENT_TYPES.get(dtype)
    if kind is None:
        raise _lib.FerrybError('dtype must be bf16, fp16 or float32')
    _same_device(codes.device, scales=scales, out=out)
    out_stride = width
    if out is None:
        out = codes.new_empty((*lead, width), dtype=dtype)
    elif out.dtype != dtype or out.shape != (*lead, width):
        raise _lib.FerrybError(f'out must be {dtype} {[*lead, width]}')
    else:
        out_stride = _rows_2d(out, 'out').stride(0) if out.numel() else 0
    if out.numel() == 0:
        return out
    c2, s2 = (_dense_rows(t if t.dim() == 2 else t.reshape(-1, t.shape[-1])) for t in (codes, scales))
    _cuda_call(codes.device, 'ferryb_dequantize_mxfp4', c2.data_ptr(), c2.stride(0), s2.data_ptr(), s2.stride(0),
               c2.shape[0], width, out.data_ptr(), kind, out_stride)
    return out


@functools.lru_cache(maxsize=256)
def _mxfp4_workspace(routes, groups, hidden, intermediate):
    size = _lib.lib().ferryb_execute_experts_mxfp4_workspace(routes, groups, hidden, intermediate)
    if size < 0:
        raise _lib.FerrybError(_lib.lib().ferryb_last_error().decode())
    return size


def execute_experts_mxfp4(cache, input, routing_weights, slots, starts, rows, cols, hidden, intermediate,
                          *, out=None, err=None):
    """execute_experts over MXFP4 expert rows: bf16 [routes, hidden], row p of
    group g = (silu(x Wg^T) * (x Wu^T)) Wd^T * routing_weights[rows[p],
    cols[p]] with x = input[rows[p]] and the weights of cache row slots[g].

    cache: uint8 [slots, model.mxfp4_row_bytes(hidden, intermediate)], rows
    as model.pack_expert_mxfp4 makes them.  Group g is the routes [starts[g],
    starts[g + 1]): slots [G], starts [G + 1], rows and cols [routes] are
    int64 CUDA tensors (LayoutBuffers' starts, rows and cols, for instance);
    groups may be empty, and rows of `out` outside [starts[0], starts[G]) are
    left as they were.  input is bf16, routing_weights [tokens, topk] bf16,
    fp16 or float32.  hidden and intermediate are multiples of 128.

    Sums, gate and up are float32, the result is rounded to bf16 once.  Inputs
    and activations (times the route's weight) go into the products as two e4m3
    numbers each, which hold a bf16 input down to 2^-13 of the largest of its 32
    neighbours exactly and an activation to a bit more than bf16 does; a row that
    is not finite comes out as NaN.  cache is 32-byte aligned, `out` 4-byte aligned (a
    contiguous bf16 view that starts at an odd element is refused).  Index errors
    are found on the device: the routes' rows become NaN (starts out of order: no
    row is written).  Without `err` the call waits for the GPU and raises; with
    `err`, an int32 [1] CUDA tensor that starts at 0, it returns at once and
    leaves a non-zero code there for the caller to check, and can be captured
    into a CUDA graph."""
    done = _lib.fast().execute_experts_mxfp4(cache, input, routing_weights, slots, starts, rows, cols, hidden,
                                             intermediate, out, err)
    if done is not None:
        return done
    require_cuda(cache, input, routing_weights, slots, starts, rows, cols, out, err)
    dev, index = input.device, input.get_device()
    for t in (cache, routing_weights, slots, starts, rows, cols, out, err):
        if t is not None and t.get_device() != index:
            _same_device(dev, cache=cache, routing_weights=routing_weights, slots=slots, starts=starts,
                         rows=rows, cols=cols, out=out, err=err)
    hidden, intermediate = int(hidden), int(intermediate)
    if hidden <= 0 or intermediate <= 0 or hidden % 128 or intermediate % 128:
        raise _lib.FerrybError(f'hidden ({hidden}) and intermediate ({intermediate}) must be multiples of 128')
    row_bytes = 3 * hidden * intermediate // 32 * 17
    if (cache.dtype != torch.uint8 or cache.dim() != 2 or cache.shape[1] != row_bytes
            or not cache.is_contiguous() or cache.data_ptr() % 32):
        raise _lib.FerrybError(f'cache must be contiguous 32-byte aligned uint8 [slots, {row_bytes}]')
    if input.dtype != BF16 or input.dim() != 2 or input.shape[1] != hidden:
        raise _lib.FerrybError(f'input must be bf16 [n, {hidden}]')
    tokens = input.shape[0]
    weights_type = _lib.ELEMENT_TYPES.get(routing_weights.dtype)
    if weights_type is None or routing_weights.dim() != 2 or routing_weights.shape[0] != tokens:
        raise _lib.FerrybError('routing_weights must be bf16, fp16 or float32 [n, topk]')
    for t in (slots, starts, rows, cols):
        if t.dtype != torch.int64 or t.dim() != 1:
            raise _lib.FerrybError('slots, starts, rows and cols must be 1-D int64 tensors')
    groups, routes = slots.shape[0], rows.shape[0]
    if starts.shape[0] != groups + 1:
        raise _lib.FerrybError(f'starts must have {groups + 1} entries (one more than slots)')
    _check(cols.shape[0] == routes, 'rows and cols must have equal length')
    if out is None:
        out = input.new_empty((routes, hidden))
    elif out.dtype != BF16 or out.shape != (routes, hidden) or not out.is_contiguous():
        raise _lib.FerrybError(f'out must be contiguous bf16 [{routes}, {hidden}]')
    elif out.data_ptr() % 4:
        raise _lib.FerrybError('out must be 4-byte aligned')
    wait = err is None
    if not wait:
        _check(err.dtype == torch.int32 and err.numel() == 1, 'err must be an int32 tensor of one element')
    if routes == 0 or groups == 0:
        return out
    _check(cache.shape[0] > 0, 'cache has no slots')
    stride, step = input.stride()
    if step != 1 or input.data_ptr() % 16 or tokens > 1 and (stride % 8 or stride < hidden):
        input = input.clone(memory_format=torch.contiguous_format)
        stride = hidden
    routing_weights = routing_weights.contiguous()
    slots, starts, rows, cols = slots.contiguous(), starts.contiguous(), rows.contiguous(), cols.contiguous()
    ws_bytes = _mxfp4_workspace(routes, groups, hidden, intermediate)
    ws = cache.new_empty((ws_bytes,))
    if wait:
        err = torch.zeros(1, dtype=torch.int32, device=dev)
    args = _lib.pack_mxfp4_experts_args(
        cache.data_ptr(), cache.shape[0], input.data_ptr(), tokens, stride, routing_weights.data_ptr(),
        routing_weights.shape[1], weights_type, 0, slots.data_ptr(), starts.data_ptr(), groups, rows.data_ptr(),
        cols.data_ptr(), routes, hidden, intermediate, out.data_ptr(), ws.data_ptr(), ws_bytes, err.data_ptr())
    _cuda_call(dev, 'ferryb_execute_experts_mxfp4', args)
    if wait:
        _lib.check_device_error(err, 'execute_experts_mxfp4')
    return out


class H2DEngine:
    """ferry/csrc/expert_ops.cpp:97-142: pinned-pool -> cache-slot copies on
    copy-engine streams, per-slot events, last-use ordering."""

    def __init__(self, cache, pool, n_streams=1):
        require_cuda(cache)
        _check(pool.is_pinned() and pool.shape[1] == cache.shape[1],
               'pool must be pinned with the cache row size')
        self.cache, self.pool = cache, pool
        h = ctypes.c_void_p()
        call('ferryb_h2d_create', ptr(cache), cache.shape[0], cache.shape[1] * cache.element_size(),
             ptr(pool), pool.shape[0], int(n_streams), ctypes.byref(h))
        self._h = h

    def _arr(self, values):
        return _lib.host_i64(values), len(values)

    def fetch(self, slots, keys):
        s, n = self._arr(slots)
        k, _ = self._arr(keys)
        call('ferryb_h2d_fetch', self._h, s, k, n)

    def wait_host(self, slots):
        s, n = self._arr(slots)
        call('ferryb_h2d_wait_host', self._h, s, n)

    def wait_device(self, slots):
        s, n = self._arr(slots)
        call('ferryb_h2d_wait_device', self._h, s, n, stream_ptr(self.cache.device))

    def mark_used(self, slots):
        s, n = self._arr(slots)
        call('ferryb_h2d_mark_used', self._h, s, n, stream_ptr(self.cache.device))

    def synchronize(self):
        call('ferryb_h2d_synchronize', self._h)

    @property
    def copies(self):
        return int(_lib.lib().ferryb_h2d_copies(self._h))

    @property
    def handle(self):
        return self._h

    def close(self):
        if self._h:
            _lib.lib().ferryb_h2d_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
