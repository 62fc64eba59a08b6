"""The serving operators where magnitudes are extreme. Bounds are those of the operators' own rounding steps, key by key."""
import numpy as np
import pytest

import kyanite_amd as kn
from kyanite_amd import DType
from serving_oracle import Graph, sample, upload

PAGE = 16


def attend(q, k, v, at, places, visible, scale, cap, slope, value_scales=None):
    """One head in 64 bits: q [rows, width], k, v [keys, width], visible [rows, keys]. (result, bound on its error).

    A score is a sum of `width` products and the few operations behind it, in f32: off by (width + 16) 2^-24 of the sum of
    its products' sizes. The cap does not enlarge that; its own formula is off by 16 x 2^-24 of its result (a quotient
    of 1 - 2 / (1 + e) is known to 2^-22, its result is at least a third of the cap), or by 2^-22 of a cap of up to 45. Factors and the bias in units of log2, the
    difference to the reference, the power of two and, for 8 bit values, the logarithm of their scale (below 2^5 in size) add
    roundings of 2^-24 each of what they round: 8 x 2^-24 of score and bias, 64 x 2^-24 of one. An error d of a score moves
    its term of the result by d times its share. Weights are rounded to f16: half a step of 2^-11, and half of 2^-24 where
    they are below the normal numbers while the largest of a row is at least 2^7 (8 bit: the largest product of weight and scale,
    for values of up to 127). Chains of sums over the keys: 2^-24 per matrix instruction. The result is rounded to f16."""
    rows, keys = visible.shape
    if keys == 0:
        return np.zeros((rows, v.shape[1])), np.full((rows, v.shape[1]), 2.0 ** -24)
    with np.errstate(invalid="ignore"):
        s = (q @ k.T) * scale
        off = (np.abs(q) @ np.abs(k).T) * abs(scale) * (q.shape[1] + 16) * 2.0 ** -24
    z = cap * np.tanh(s / cap) if cap else s
    bias = slope * np.abs(at[:, None] - places[None, :])
    off = off + (24 * np.abs(z) + 8 * np.abs(bias) + 64) * 2.0 ** -24 + (cap * 2.0 ** -22 if cap <= 45 else 0.0)
    z = np.where(visible, z - bias, -np.inf)
    top = z.max(-1, keepdims=True)
    e = np.exp(z - np.where(np.isfinite(top), top, 0.0))
    total = e.sum(-1, keepdims=True)
    safe = np.where(total > 0, total, 1.0)
    w, off = e / safe, np.where(visible, off, 0.0)
    v = np.where(visible.any(0)[:, None], v, 0.0)  # what nobody sees
    out = w @ v
    moved = ((w * off) @ np.abs(v) + np.abs(out) * (w * off).sum(-1, keepdims=True)) * 1.1
    if value_scales is None:
        below = 2.0 ** -32 * (visible.astype(float) @ np.abs(v)) / safe
    else:
        held = np.where(visible.any(0), value_scales, 0.0)  # (scales below 2^-40 count as that)
        below = 2.0 ** -32 * 127 * visible.sum(-1, keepdims=True) * (e * np.maximum(held, 2.0 ** -40)).max(-1, keepdims=True) / safe + 2.0 ** -33
    chain = (keys / 16 + 16) * 2.0 ** -24
    return out, (w @ np.abs(v)) * (2.0 ** -11 + chain) + below + moved + np.abs(out) * 2.0 ** -11 + 2.0 ** -24


class Case:
    """Sequences over a cache whose pages lie one behind the other: the prefix's first, then `table_pages` per sequence. Keys and
    values are given per place, [place, heads, width] in f64; 8 bit rows are quantised here."""

    def __init__(self, dtype, lengths, kv=1, group=2, width=64, queries=1, prefix=0, page=PAGE, seed=0, **scores):
        self.rng = np.random.default_rng(seed)
        self.dtype, self.lengths, self.kv, self.group, self.width, self.queries, self.prefix, self.page = dtype, lengths, kv, group, width, queries, prefix, page
        self.scores = dict(dict(scale=width ** -0.5, cap=0.0, window=0, slopes=None), **scores)
        self.table_pages, self.prefix_pages = max(1, -(-max(lengths) // page)), -(-prefix // page)
        self.pages = self.prefix_pages + len(lengths) * self.table_pages
        shape = (self.pages * page, kv, width)
        self.q = self.rng.standard_normal((len(lengths), queries, kv * group, width)).astype(np.float16)
        self.k, self.v = self.rng.standard_normal(shape), self.rng.standard_normal(shape)
        self.spoilt = []  # (place, whose scale, value)

    def place(self, b, j):
        """where key j of sequence b lies (j < prefix: in the prefix)"""
        return j if j < self.prefix else (self.prefix_pages + b * self.table_pages) * self.page + j - self.prefix

    def held(self):
        """what the cache holds: (k, v, scales of k, scales of v), [place, heads, ...]"""
        if self.dtype == DType.F16:
            return self.k.astype(np.float16), self.v.astype(np.float16), None, None
        out = []
        for x in (self.k, self.v):
            scale = (np.abs(x).max(-1) / 127).astype(np.float32)
            out.append((np.rint(x / np.where(scale > 0, scale, 1)[..., None]).clip(-127, 127).astype(np.int8), scale))
        return out[0][0], out[1][0], out[0][1], out[1][1]

    def run(self, device):
        held = list(self.held())
        for place, which, value in self.spoilt:
            held[2 + which][place] = value
        paged = [None if x is None else np.ascontiguousarray(np.moveaxis(x.reshape((self.pages, self.page) + x.shape[1:]), 1, 2)) for x in held]
        tables = (self.prefix_pages + np.arange(len(self.lengths) * self.table_pages)).astype(np.int32)
        mem = [upload(device, x if x is not None else np.zeros(1, np.float32)) for x in paged]
        B, T, H, W = self.q.shape
        dev = [upload(device, x) for x in (self.q, np.array(self.lengths, np.int32), tables, np.arange(max(self.prefix_pages, 1), dtype=np.int32),
                                           np.asarray(self.scores["slopes"] if self.scores["slopes"] is not None else [0], np.float32))]
        out = kn.DeviceBuffer(device, self.q.nbytes)
        scales = (mem[2].ptr, mem[3].ptr) if self.dtype == DType.I8 else (0, 0)
        cache = kn.kv_cache(self.dtype, self.pages, self.kv, self.page, W, mem[0].ptr, mem[1].ptr, *scales)
        strides = (T * H * W, H * W, W)
        args = kn.cached_attention_args(B, T, H, cache, dev[0].ptr, strides, out.ptr, strides, dev[1].ptr, dev[2].ptr, self.table_pages, self.table_pages,
                                        prefix_tokens=self.prefix, prefix_table=dev[3].ptr if self.prefix else 0, scale=self.scores["scale"],
                                        cap=self.scores["cap"], window=self.scores["window"], slopes=dev[4].ptr if self.scores["slopes"] is not None else 0)
        stream = kn.HipStream(device)
        kn.cached_attention(device, stream, args, kn.DeviceBuffer(device, max(kn.cached_attention_workspace_bytes(args), 1)))
        stream.synchronize()
        return out.to_array(np.float16, self.q.shape)

    def check(self, got, what=""):
        k, v, ks, vs = (None if x is None else x.astype(np.float64) for x in self.held())
        if self.dtype == DType.I8:
            k, v = k * ks[..., None], v * vs[..., None]
        T = self.queries
        for b, n in enumerate(self.lengths):
            places = np.arange(self.prefix + n)
            at = self.prefix + n - T + np.arange(T)
            where = np.array([self.place(b, j) for j in places], np.int64)
            visible = (places <= at[:, None]) & (at[:, None] >= self.prefix)
            if self.scores["window"]:
                visible &= places > at[:, None] - self.scores["window"]
            for h in range(self.kv * self.group):
                g = h // self.group
                slope = 0.0 if self.scores["slopes"] is None else float(self.scores["slopes"][h])
                out, bound = attend(self.q[b, :, h].astype(np.float64), k[where, g], v[where, g], at, places, visible, float(np.float32(self.scores["scale"])),
                                    float(np.float32(self.scores["cap"])), slope, None if vs is None else vs[where, g])
                off = np.abs(got[b, :, h].astype(np.float64) - out)
                assert (off <= bound).all(), f"{what}: sequence {b} head {h}: {np.max(off / bound):.2f} of the bound, {np.max(off):.3e} off"


# (which kernel: few rows, a prefix beside few rows in one launch or in its own, many rows, a prefix for many rows)
FORMS = {
    "rows": dict(lengths=[50, 33, 100, 7]),
    "rows_odd_pages": dict(lengths=[50, 33, 100, 7], page=5),
    "rows_wide": dict(lengths=[50, 333], width=128, group=4, queries=3),
    "rows_in_parts": dict(lengths=[2500, 40], width=128),
    "prefix_inside": dict(lengths=[50, 3], prefix=100, queries=2),
    "prefix_in_rows": dict(lengths=[50, 3], prefix=1000, width=128),
    "prefix_of_many": dict(lengths=[50 + i % 7 for i in range(24)], prefix=2100, group=4),
    "prefix_of_many_wide": dict(lengths=[50 + i % 7 for i in range(24)], prefix=2100, group=4, width=128),
    "tiles": dict(lengths=[200, 90], queries=40),
    "tiles_wide": dict(lengths=[300, 90], queries=40, width=128, group=3),
}


# ---- many sequences ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    dict(lengths=[(37 * i) % 50 for i in range(400)]),                                                  # every item a sequence
    dict(lengths=[(37 * i) % 50 for i in range(399)] + [2500], dtype=DType.I8, width=16),               # one of them in parts
    dict(lengths=[2500] + [1] * 400 + [0, 1500], group=1, width=32),
    dict(lengths=[(11 * i) % 90 for i in range(300)], kv=2, width=128, queries=3, window=20, page=5),
    dict(lengths=[(11 * i) % 90 for i in range(500)], prefix=30, dtype=DType.I8),                        # a prefix beside the own keys
    dict(lengths=[(11 * i) % 90 for i in range(400)], prefix=1900, group=1),                             # a prefix in tiles
], ids=["one_item_each", "one_in_parts", "long_and_empty", "window", "prefix_inside", "prefix_apart"])
def test_many_sequences(case, hip_device):
    """so many that their items are listed"""
    c = Case(**dict(dict(dtype=DType.F16), **case))
    for call in range(2):
        c.check(c.run(hip_device), f"call {call}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [DType.I8, DType.F16], ids=lambda d: d.name)
def test_many_sequences_captured_and_replayed(dtype, hip_device):
    """lengths that change from replay to replay move the items of the list: results are those of the call outside the graph"""
    rng = np.random.default_rng(4)
    B, W, table_pages = 400, 32, 100
    pages = 150  # (sequences share them)
    k, v = (rng.standard_normal((pages, 1, PAGE, W)) for _ in range(2))
    held = [np.rint(x * 30).clip(-127, 127).astype(np.int8) if dtype == DType.I8 else x.astype(np.float16) for x in (k, v)]
    mem = [upload(hip_device, x) for x in held]
    scales = upload(hip_device, np.full(pages * PAGE, 1 / 30, np.float32))
    q, tables = upload(hip_device, rng.standard_normal((B, 2, W)).astype(np.float16)), upload(hip_device, rng.integers(0, pages, (B, table_pages)).astype(np.int32))
    lengths, out = kn.DeviceBuffer(hip_device, B * 4), kn.DeviceBuffer(hip_device, B * 2 * W * 2)
    cache = kn.kv_cache(dtype, pages, 1, PAGE, W, mem[0].ptr, mem[1].ptr, *([scales.ptr] * 2 if dtype == DType.I8 else []))
    args = kn.cached_attention_args(B, 1, 2, cache, q.ptr, (2 * W, 2 * W, W), out.ptr, (2 * W, 2 * W, W), lengths.ptr, tables.ptr, table_pages, table_pages)
    workspace, other = (kn.DeviceBuffer(hip_device, kn.cached_attention_workspace_bytes(args)) for _ in range(2))
    stream, graph, seen = kn.HipStream(hip_device), None, []
    for replay in range(4):
        n = rng.integers(0, 40, B).astype(np.int32)
        n[rng.integers(0, B, replay)] = 1600  # some in parts
        kn._lib.check(kn._lib.lib.knhip_memcpy_h2d(hip_device.index, lengths.ptr, n.ctypes.data, n.nbytes))
        if graph is None:
            with Graph(stream) as graph:
                kn.cached_attention(hip_device, stream, args, workspace)
        graph.launch()
        stream.synchronize()
        replayed = out.to_array(np.uint16, B * 2 * W)
        kn.cached_attention(hip_device, stream, args, other)
        stream.synchronize()
        assert np.array_equal(replayed, out.to_array(np.uint16, B * 2 * W)), replay
        assert (replayed.reshape(B, -1)[n == 0] == 0).all() and (replayed.reshape(B, -1)[n > 0] != 0).any(-1).all()
        seen.append(replayed)
    assert not np.array_equal(seen[0], seen[1])


@pytest.mark.gpu
def test_time_grows_with_the_number_of_sequences(hip_device):
    """sixteen times the sequences take less than 64 times as long: their number, not its square"""
    W, times = 64, []
    stream = kn.HipStream(hip_device)
    for B in (4096, 65536):
        rows, out = upload(hip_device, np.zeros(B * W, np.float16)), kn.DeviceBuffer(hip_device, B * W * 2)
        lengths, tables = upload(hip_device, np.ones(B, np.int32)), upload(hip_device, np.arange(B, dtype=np.int32))
        cache = kn.kv_cache(DType.F16, B, 1, 1, W, rows.ptr, rows.ptr)
        args = kn.cached_attention_args(B, 1, 1, cache, rows.ptr, (W, W, W), out.ptr, (W, W, W), lengths.ptr, tables.ptr, 1, 1)
        workspace = kn.DeviceBuffer(hip_device, max(kn.cached_attention_workspace_bytes(args), 1))
        seconds = []
        for _ in range(4):
            start = stream.record_event()
            kn.cached_attention(hip_device, stream, args, workspace)
            end = stream.record_event()
            stream.synchronize()
            seconds.append(end.time_elapsed_since(start))
        times.append(min(seconds))
    assert times[1] < 64 * times[0], times


# ---- scales that nobody sees ---------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 3e38, 1e12], ids=str)
@pytest.mark.parametrize("form", FORMS)
def test_scales_of_unseen_slots_change_nothing(form, value, hip_device):
    """slots behind a sequence's last key, and keys in front of every query's window"""
    c = dict(FORMS[form])
    window = c["prefix"] // 2 + max(c["lengths"]) if "prefix" in c else 30 + c.get("queries", 1)
    case = Case(DType.I8, window=window, **c)
    clean = case.run(hip_device)
    case.check(clean, "clean")
    for b, n in enumerate(case.lengths):
        first = case.prefix + n - case.queries - window + 1  # the first key that any query sees
        end = case.place(b, case.prefix) + case.table_pages * case.page
        unseen = list(range(case.place(b, case.prefix + n - 1) + 1, end)) + [case.place(b, j) for j in range(case.prefix, max(first, case.prefix))]
        case.spoilt += [(p, which, value) for p in unseen for which in (0, 1)]
    seen_prefix = min(max(0, case.prefix + n - case.queries - window + 1) for n in case.lengths)
    case.spoilt += [(p, which, value) for p in range(min(seen_prefix, case.prefix)) for which in (0, 1)]
    case.spoilt += [(p, which, value) for p in range(case.prefix, case.prefix_pages * case.page) for which in (0, 1)]
    assert case.spoilt
    assert np.array_equal(case.run(hip_device).view(np.uint16), clean.view(np.uint16))


@pytest.mark.gpu
@pytest.mark.parametrize("value", [np.nan, np.inf, 3e38], ids=str)
@pytest.mark.parametrize("form", ["rows_wide", "tiles", "tiles_wide"])
def test_scales_that_one_query_sees_leave_the_others_alone(form, value, hip_device):
    """the newest key's scales: the last query sees them, the queries before do not"""
    case = Case(DType.I8, **FORMS[form])
    clean = case.run(hip_device)
    case.spoilt = [(case.place(b, n - 1), which, value) for b, n in enumerate(case.lengths) for which in (0, 1)]
    got = case.run(hip_device)
    assert np.array_equal(got[:, :-1].view(np.uint16), clean[:, :-1].view(np.uint16))
    if value != 3e38:
        assert np.isnan(got[:, -1]).all()


# ---- values of different magnitudes --------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [DType.I8, DType.F16], ids=lambda d: d.name)
@pytest.mark.parametrize("spread", ["from_1e-3_to_6e4", "later_outlier", "dominant_outlier", "rising", "zeros"])
@pytest.mark.parametrize("form", FORMS)
def test_values_of_different_magnitudes(form, spread, dtype, hip_device):
    case = Case(dtype, seed=3, **FORMS[form])
    rng, n = case.rng, len(case.v)
    if spread == "from_1e-3_to_6e4":
        case.v *= np.exp(rng.uniform(np.log(1e-3), np.log(1e4), n))[:, None, None]
    else:
        case.v *= 0.05
    if spread == "rising":
        case.v *= 4.0 ** (np.arange(n) // 64 % 9)[:, None, None]
    for b in range(len(case.lengths)):
        first, last = case.place(b, 0), case.place(b, case.prefix + case.lengths[b] - case.queries)
        if spread == "zeros":
            case.v[first] = 0
            case.k[first] = case.q[b, 0, 0] * 2.0  # most of the weight, for one head
        for place in (last - 3, (first + last) // 2 if case.prefix == 0 else case.prefix // 2 + 1):
            if spread == "later_outlier":  # a score far below all others
                case.v[place] = rng.standard_normal((case.kv, case.width)).clip(-2, 2) * 15000
                case.k[place] = 0
                case.q[..., 0] = 30
                case.k[place, :, 0] = -8
            if spread == "dominant_outlier":
                case.v[place] = rng.standard_normal((case.kv, case.width)).clip(-2, 2) * 15000
                case.k[place] = 0
                case.q[..., 0] = 20
                case.k[place, :, 0] = 4
    case.check(case.run(hip_device), f"{form} {spread}")


# ---- weights far below the largest ---------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [DType.I8, DType.F16], ids=lambda d: d.name)
@pytest.mark.parametrize("first", [True, False], ids=["sink_first", "sink_last"])
@pytest.mark.parametrize("form", FORMS)
def test_weights_far_below_the_largest(form, first, dtype, hip_device):
    """one key of no value takes most of the weight, all others get the same 2^-17 or so of it: a number in the middle between two
    multiples of 2^-24"""
    case = Case(dtype, scale=1.0, **FORMS[form])
    case.q[:], case.k[:], case.v[:] = 0, 0, 1.0
    case.q[..., 0] = 1
    scores = np.arange(-12, -11.5, 2.0 ** -7)  # numbers of f16
    case.k[..., 0] = scores[np.argmin(np.abs(np.exp(scores) * 2.0 ** 24 % 1 - 0.5))]
    for b in range(len(case.lengths)):
        sink = case.place(b, 0) if first else case.place(b, case.prefix + case.lengths[b] - case.queries)
        case.k[sink], case.v[sink] = 0, 0
    case.check(case.run(hip_device), form)


# ---- caps ----------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.5, 30.0, 1e4, 1e6, 1e30, 1e38])
@pytest.mark.parametrize("dtype", [DType.I8, DType.F16], ids=lambda d: d.name)
@pytest.mark.parametrize("form", FORMS)
def test_caps_of_any_size(form, dtype, cap, hip_device):
    """the cap's error goes by the score, not by the cap"""
    case = Case(dtype, cap=cap, seed=1, **FORMS[form])
    case.check(case.run(hip_device), form)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [DType.I8, DType.F16], ids=lambda d: d.name)
@pytest.mark.parametrize("form", FORMS)
def test_scores_on_both_sides_of_a_cap(form, dtype, hip_device):
    """one key of a few has a score beyond a large cap (negative: without weight), the others lie far below it"""
    case = Case(dtype, cap=2e5, seed=2, **FORMS[form])
    case.q[..., 0] = 300
    case.k[..., 0] = 0
    case.k[::5, :, 0] = -60000
    case.check(case.run(hip_device), form)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [30.0, 1e6, 1e30, 2e5])
@pytest.mark.parametrize("queries,keys,width", [(40, 40, 64), (150, 150, 128), (70, 1500, 64)])
def test_caps_of_prompts(queries, keys, width, cap, hip_device):
    rng = np.random.default_rng(queries)
    q, k, v = (rng.standard_normal((n, 2, width)).astype(np.float16) for n in (queries, keys, keys))
    if cap == 2e5:
        q[..., 0], k[..., 0], k[::5, :, 0] = 300, 0, -60000
    dev = [upload(hip_device, x) for x in (q, k, v)]
    out = kn.DeviceBuffer(hip_device, q.nbytes)
    s = (0, 2 * width, width)
    args = kn.attention_args(1, queries, keys, 2, 2, width, dev[0].ptr, s, dev[1].ptr, s, dev[2].ptr, s, out.ptr, s, causal=True, cap=cap)
    stream = kn.HipStream(hip_device)
    kn.attention(hip_device, stream, args, kn.DeviceBuffer(hip_device, max(kn.attention_workspace_bytes(args), 1)))
    stream.synchronize()
    got, at, places = out.to_array(np.float16, q.shape), np.arange(queries) + keys - queries, np.arange(keys)
    for h in range(2):
        e, bound = attend(*(x[:, h].astype(np.float64) for x in (q, k, v)), at, places, places <= at[:, None], float(np.float32(width ** -0.5)), float(np.float32(cap)), 0.0)
        off = np.abs(got[:, h].astype(np.float64) - e)
        assert (off <= bound).all(), f"{np.max(off / bound):.2f} of the bound, {np.max(off):.3e} off"


# ---- sampling ------------------------------------------------------------------------------------------------------

def _draw(device, logits, uniform, **filters):
    """(tokens, probabilities) of f32 rows"""
    types = dict(temperature=np.float32, top_k=np.int32, top_p=np.float32, min_p=np.float32)
    rows, vocab = logits.shape
    dev = {n: upload(device, np.full(rows, v, types[n])) for n, v in filters.items()}
    x, u = upload(device, logits.astype(np.float32)), upload(device, uniform.astype(np.float32))
    tokens, chance = upload(device, np.full(rows, -7, np.int32)), upload(device, np.full(rows, -7, np.float32))
    args = kn.sample_args(DType.F32, rows, vocab, x.ptr, vocab, u.ptr, tokens.ptr, probabilities=chance.ptr, **{n: d.ptr for n, d in dev.items()})
    stream = kn.HipStream(device)
    kn.sample(device, stream, args)
    stream.synchronize()
    return tokens.to_array(np.int32, rows), chance.to_array(np.float32, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("min_p", [1.0000001, 2.0, np.inf])
@pytest.mark.parametrize("filters", [{}, dict(top_k=7), dict(top_k=100), dict(top_k=3000), dict(top_p=0.9), dict(top_k=2000, top_p=0.9, temperature=0.5)], ids=str)
def test_min_p_beyond_one_keeps_the_first_of_equal_maxima(filters, min_p, hip_device):
    rng = np.random.default_rng(1)
    x = np.round(rng.standard_normal((40, 5000)) * 2).clip(-3, 3)  # tens of equal maxima per row
    x[1] = 0
    x[2, 4000:] = np.inf
    tokens, chance = _draw(hip_device, x, rng.random(40), min_p=min_p, **filters)
    assert np.array_equal(tokens, x.argmax(-1)) and (chance == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("min_p", [np.nan, -1.0, 0.0])
@pytest.mark.parametrize("filters", [{}, dict(top_k=40), dict(top_p=0.9)], ids=str)
def test_min_p_that_is_no_positive_number_is_off(filters, min_p, hip_device):
    rng = np.random.default_rng(2)
    x, u = rng.standard_normal((30, 3000)), rng.random(30)
    for a, b in zip(_draw(hip_device, x, u, min_p=min_p, **filters), _draw(hip_device, x, u, **filters)):
        assert np.array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-45, 1e-41, 1e-39, 1e-38, 3e-38, 1e-37, 3e-37, 1e-36, 1e-30, 1e30, 1e35, 3e35, 1e36])
@pytest.mark.parametrize("filters", [dict(top_p=0.9), dict(top_k=40), dict(top_k=3000, top_p=0.95), dict(min_p=0.05), {}], ids=str)
def test_temperatures_at_both_ends_of_the_range(filters, temperature, hip_device):
    """logits a few temperatures apart, so that several tokens have weight"""
    rng = np.random.default_rng(3)
    temperature = np.float32(temperature)
    x = (rng.standard_normal((12, 5000)) * 2.5 * float(temperature)).astype(np.float32)
    x[0, 7], x[1, 8] = np.inf, -np.inf
    x[2] = np.round(x[2] / temperature) * temperature  # few values
    u = rng.random(12).astype(np.float32)
    each = {n: np.full(12, v, np.int32 if n == "top_k" else np.float32) for n, v in dict(filters, temperature=temperature).items()}
    expected, probability = sample(x, u, **each)
    tokens, chance = _draw(hip_device, x, u, temperature=temperature, **filters)
    assert np.array_equal(tokens, expected)
    # (weights are off by half of 2^-49 each, f32 rounds by 2^-24 of the value)
    assert (np.abs(chance - probability) <= probability * 2.0 ** -23 + 5000 * 2.0 ** -49).all()


# ---- sizes ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("call", [kn.cache_write, kn.cache_read])
@pytest.mark.parametrize("tokens,heads", [((1 << 27) - 7, 1), (1 << 27, 1), ((1 << 24) - 1, 8 + 1), ((1 << 31) - 1, 1)])
def test_more_rows_than_a_launch_holds_are_refused(call, tokens, heads):
    """(made up addresses: refused by size before anything else is looked at)"""
    cache = kn.kv_cache(DType.F16, 1 << 20, heads, 128, 256, 256, 512)
    rows = kn.cache_rows(DType.F16, tokens, 256, (heads * 256, 256), 512, (heads * 256, 256), 256)
    with pytest.raises(kn.KnError, match="tokens \\* heads must stay below 2\\^27 - 7"):
        call(0, 0, cache, rows)


# ---- errors of others ----------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_an_error_that_an_earlier_call_left_is_not_reported_again(hip_device):
    stream, W = kn.HipStream(hip_device), 64
    mem = upload(hip_device, np.zeros(64 * W, np.float32))
    slots = upload(hip_device, np.arange(4, dtype=np.int32))
    zeros = upload(hip_device, np.zeros(64, np.int32))
    out = kn.DeviceBuffer(hip_device, 64 * W * 4)
    cache = kn.kv_cache(DType.F16, 4, 1, 16, W, mem.ptr, mem.ptr)
    rows = kn.cache_rows(DType.F32, 4, out.ptr, (2 * W, W), out.ptr + 4 * W, (2 * W, W), slots.ptr)
    cached = kn.cached_attention_args(1, 1, 1, cache, mem.ptr, (W, W, W), out.ptr, (W, W, W), zeros.ptr, zeros.ptr, 1, 1)
    prompt = kn.attention_args(1, 4, 4, 1, 1, W, mem.ptr, (0, W, W), mem.ptr, (0, W, W), mem.ptr, (0, W, W), out.ptr, (0, W, W))
    draw = kn.sample_args(DType.F32, 1, 64, mem.ptr, 64, mem.ptr, zeros.ptr)
    workspace = kn.DeviceBuffer(hip_device, max(kn.cached_attention_workspace_bytes(cached), kn.attention_workspace_bytes(prompt), 1))
    for call in (lambda: kn.cache_write(hip_device, stream, cache, rows), lambda: kn.cache_read(hip_device, stream, cache, rows),
                 lambda: kn.cached_attention(hip_device, stream, cached, workspace), lambda: kn.attention(hip_device, stream, prompt, workspace),
                 lambda: kn.sample(hip_device, stream, draw)):
        with pytest.raises(kn.KnError, match="hipMalloc"):
            kn.DeviceBuffer(hip_device, 1 << 50)
        call()
        stream.synchronize()

def test_strides_of_a_cache_are_named():
    with pytest.raises(kn.KnError, match=r"three strides \(page, head, token\)"):
        kn.kv_cache(DType.F16, 1, 1, 16, 64, 0, 0, strides=(64, 64))
