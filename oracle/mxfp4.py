"""float64 restatement of the operators that the reference has no counterpart
of: routing with biases and groups, MXFP4 rows and the routed experts over
them (test infrastructure only; numpy, from the definitions)."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
CODES = np.concatenate([GRID, -GRID])


def route(logits, topk, score='softmax', bias=None, n_group=1, topk_group=1, group_score='max',
          norm=True, scaling=1.0):
    """(selected, weights) of float64 logits [T, E]; NaN keys rank last."""
    x = np.asarray(logits, np.float64)
    T, E = x.shape
    with np.errstate(all='ignore'):
        if score == 'softmax':
            m = x.max(1, keepdims=True)
            e = np.where(np.isneginf(m), 0.0, np.exp(x - m))
            z = e.sum(1, keepdims=True)
            s = np.where(z == 0, 0.0, e / z)
        else:
            s = 1.0 / (1.0 + np.exp(-x))
    key = s if bias is None else s + np.asarray(bias, np.float64)
    selected = np.empty((T, topk), np.int64)
    size = E // n_group
    for t in range(T):
        k = [(-np.inf if np.isnan(v) else v, not np.isnan(v)) for v in key[t]]
        worth = []
        for g in range(n_group):
            part = key[t, g * size:(g + 1) * size]
            best = np.sort(part)[::-1]
            w = np.nan if np.isnan(part).any() else best[0] if group_score == 'max' or n_group == 1 else best[0] + best[1]
            worth.append((-np.inf, False) if np.isnan(w) else (w, True))
        groups = sorted(range(n_group), key=lambda g: (not worth[g][1], -worth[g][0], g))[:topk_group]
        cand = [e for g in sorted(groups) for e in range(g * size, (g + 1) * size)]
        cand.sort(key=lambda e: (not k[e][1], -k[e][0], e))
        selected[t] = cand[:topk]
    w = np.take_along_axis(s, selected, 1)
    if norm:
        total = w.sum(1, keepdims=True)
        with np.errstate(all='ignore'):
            w = np.where(total == 0, 0.0, w / total)
    return selected, w * scaling


def quantize(x):
    """(codes uint8 [..., n / 2], scales uint8 [..., n / 32]) of x [..., n]."""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    top = np.abs(b).max(-1)
    finite = np.isfinite(b).all(-1)
    _, e = np.frexp(np.where(finite & (top > 0), top, 1.0))
    power = np.where(top > 0, np.maximum(e - 1 - 2, -127), -127)
    scale = np.where(finite, power + 127, 255).astype(np.uint8)
    y = np.where(finite[..., None], np.ldexp(np.abs(np.where(finite[..., None], b, 0.0)), -power[..., None]), 0.0)
    code = np.zeros(y.shape, np.uint8)
    for i in range(7):  # a value on the border between two codes goes to the even one
        border = (GRID[i] + GRID[i + 1]) / 2
        code = np.where((y > border) | ((y == border) & (i % 2 == 1)), i + 1, code)
    sign = np.signbit(np.where(finite[..., None], b, 0.0))
    code = (code + 8 * sign).astype(np.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def dequantize(codes, scales):
    codes, scales = np.asarray(codes), np.asarray(scales)
    c = np.empty(codes.shape[:-1] + (codes.shape[-1] * 2,), np.uint8)
    c[..., 0::2], c[..., 1::2] = codes & 15, codes >> 4
    v = CODES[c].reshape(c.shape[:-1] + (-1, 32))
    f = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * f[..., None]).reshape(c.shape)


def execute_experts(cache, x, weights, slots, starts, rows, cols, hidden, inter):
    """[routes, hidden] float64 of uint8 rows `cache` (codes, then scales)."""
    n = 3 * hidden * inter
    out = np.full((len(rows), hidden), np.nan)
    for g, slot in enumerate(slots):
        a, b = int(starts[g]), int(starts[g + 1])
        if a == b:
            continue
        w = dequantize(cache[slot][:n // 2], cache[slot][n // 2:])
        gate, up, down = np.split(w, 3)
        xs = np.asarray(x, np.float64)[rows[a:b]]
        u = xs @ gate.reshape(inter, hidden).T
        act = u / (1 + np.exp(-u)) * (xs @ up.reshape(inter, hidden).T)
        y = act @ down.reshape(hidden, inter).T
        out[a:b] = y * np.asarray(weights, np.float64)[rows[a:b], cols[a:b]][:, None]
    return out
