"""Plain 64 bit forms of the operators that serve a decoder token by token, and helpers to call them on the GPU."""
import ctypes
import math

import numpy as np

import kyanite_amd as kn

NP = {kn.DType.F16: np.float16, kn.DType.F32: np.float32, kn.DType.I8: np.int8}


def upload(device, array):
    return kn.DeviceBuffer.from_array(device, np.ascontiguousarray(array))


def quantise(x):
    """(whole numbers, scale) of the last axis, in the f32 steps of the definition"""
    x = np.clip(np.nan_to_num(x.astype(np.float32), nan=0.0, posinf=65504, neginf=-65504), -65504, 65504)
    scale = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint(x / scale[..., None])
    q = np.where(scale[..., None] > 0, np.clip(q, -127, 127), 0)
    return q.astype(np.int8), scale


def attend(q, k, v, at, places, visible, scale, cap, slope):
    """One head: q [rows, width], k, v [keys, width] in f64; visible [rows, keys]. (result, bound on its error).

    The bound: f32 sums of `width` products and the few operations behind them move a score by at most
    (width + 16) 2^-24 of what it is summed from (|q| |k|, the cap, the bias); a moved score changes weights by as much,
    twice (numerator and sum). Weights and result are rounded to f16 once each, half a step of 2^-11, and a result below
    the normal numbers by half of 2^-24."""
    score = (q @ k.T) * scale
    size = (np.abs(q) @ np.abs(k).T) * abs(scale)
    if cap:
        score = cap * np.tanh(score / cap)
        size = size + cap
    bias = slope * np.abs(at[:, None] - places[None, :])
    score, size = score - bias, size + np.abs(bias)
    score = np.where(visible, score, -np.inf)
    top = score.max(-1, keepdims=True, initial=-np.inf)
    e = np.exp(score - np.where(np.isfinite(top), top, 0.0))
    total = e.sum(-1, keepdims=True)
    w = np.divide(e, total, out=np.zeros_like(e), where=total > 0)
    out, spread = w @ v, w @ np.abs(v)
    moved = np.where(visible, size, 0).max(-1, keepdims=True, initial=0) * (q.shape[1] + 16) * 2.0 ** -24
    return out, spread * (2.0 ** -11 + 2 * moved) + np.abs(out) * 2.0 ** -11 + 2.0 ** -24


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    """(tokens, probabilities) from the definition"""
    tokens, chance = np.full(len(logits), -1, np.int32), np.zeros(len(logits))
    for r, row in enumerate(logits):
        x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
        if len(x) == 0 or x.max() == -np.inf:
            continue
        t = 1.0 if temperature is None else float(temperature[r])
        if not t > 0:
            tokens[r], chance[r] = np.argmax(x), 1.0
            continue
        top = x.max()
        with np.errstate(invalid="ignore"):
            w = np.where(x == top, 1.0, 0.0 if top == np.inf else np.exp((x - top) / t))
        real, step = w, 2.0 ** -min(51, 62 - math.ceil(math.log2(len(x))))
        w = np.round(w / step) * step  # the fixed point of the definition: smaller weights are never drawn
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        if top_k is not None and top_k[r] > 0:
            order = order[:top_k[r]]
        if top_p is not None and top_p[r] < 1:
            before = np.cumsum(w[order]) - w[order]
            order = order[(before < float(top_p[r]) * w[order].sum()) | (np.arange(len(order)) == 0)]
        if min_p is not None:
            order = order[(real[order] >= float(min_p[r])) | (x[order] == top)]
        order = np.sort(order)
        sums = np.cumsum(w[order])
        u = min(max(float(uniform[r]), 0.0), 1 - 2.0 ** -24)
        i = min(np.searchsorted(sums, u * sums[-1], side="right"), len(order) - 1)
        tokens[r], chance[r] = order[i], w[order[i]] / sums[-1]
    return tokens, chance


class Graph:
    """What is queued on `stream` inside the `with` block, as a HIP graph."""

    def __init__(self, stream):
        self.hip = ctypes.CDLL("libamdhip64.so.7")
        self.stream, self.graph, self.exec = ctypes.c_void_p(stream.handle), ctypes.c_void_p(), ctypes.c_void_p()

    def _ok(self, status):
        assert status == 0, f"hip status {status}"

    def __enter__(self):
        self._ok(self.hip.hipStreamBeginCapture(self.stream, 2))  # relaxed
        return self

    def __exit__(self, *error):
        self._ok(self.hip.hipStreamEndCapture(self.stream, ctypes.byref(self.graph)))
        self._ok(self.hip.hipGraphInstantiate(ctypes.byref(self.exec), self.graph, None, None, ctypes.c_size_t(0)))

    def launch(self):
        self._ok(self.hip.hipGraphLaunch(self.exec, self.stream))
