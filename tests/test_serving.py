"""The operators that serve a decoder token by token, against plain 64 bit forms of their definitions: sizes and masks
where they can go wrong, what they refuse, and a run of them together."""
import math

import numpy as np
import pytest

import kyanite_amd as kn
from kyanite_amd import DType
from serving_oracle import NP, Graph, attend, quantise, sample, upload

GUARD = 0x5A


class CacheCase:
    """A cache whose unused elements hold NaN (f16) or 127 with a NaN scale (i8): nothing of them may be seen."""

    def __init__(self, device, dtype, pages, heads, page_tokens, width, spread=0, order="dense"):
        self.device, self.dtype, self.shape = device, dtype, (pages, heads, page_tokens, width)
        pitch = width + spread
        if order == "dense":  # [pages, heads, tokens, width]
            self.axes, self.strides = (0, 1, 2), (heads * page_tokens * pitch, page_tokens * pitch, pitch)
        else:  # [pages, tokens, heads, width]
            self.axes, self.strides = (0, 2, 1), (heads * page_tokens * pitch, pitch, heads * pitch)
        mem = [(pages, heads, page_tokens)[a] for a in self.axes] + [pitch]
        fill = np.nan if dtype == DType.F16 else 127
        self.k, self.v = (np.full(mem, fill, NP[dtype]) for _ in range(2))
        self.ks, self.vs = (np.full((pages, heads, page_tokens), np.nan, np.float32) for _ in range(2))

    def view(self, mem):
        return np.moveaxis(mem, (0, 1, 2), self.axes)[..., :self.shape[3]]  # [pages, heads, tokens, width]

    def put(self, slots, k, v):
        for t, s in enumerate(slots):
            page, at = divmod(int(s), self.shape[2])
            for mem, scales, x in ((self.k, self.ks, k[t]), (self.v, self.vs, v[t])):
                if self.dtype == DType.I8:
                    self.view(mem)[page, :, at], scales[page, :, at] = quantise(x)
                else:
                    self.view(mem)[page, :, at] = x

    def held(self, slots):
        """what the slots stand for, f64 [tokens, heads, width], for k and v"""
        out = []
        for mem, scales in ((self.k, self.ks), (self.v, self.vs)):
            page, at = np.divmod(np.asarray(slots, np.int64), self.shape[2])
            x = self.view(mem)[page, :, at].astype(np.float64)
            out.append(x * scales[page, :, at].astype(np.float64)[..., None] if self.dtype == DType.I8 else x)
        return out

    def upload(self):
        self.buffers = [upload(self.device, a) for a in (self.k, self.v, self.ks, self.vs)]
        scales = [b.ptr for b in self.buffers[2:]] if self.dtype == DType.I8 else [0, 0]
        return kn.kv_cache(self.dtype, *self.shape, self.buffers[0].ptr, self.buffers[1].ptr, *scales, strides=self.strides)

    def download(self):
        self.k, self.v = (b.to_array(NP[self.dtype], a.shape) for b, a in zip(self.buffers, (self.k, self.v)))
        self.ks, self.vs = (b.to_array(np.float32, self.ks.shape) for b in self.buffers[2:])


def _same(got, expected, what):
    assert got.shape == expected.shape and got.dtype == expected.dtype
    assert np.array_equal(got.view(np.uint8), np.ascontiguousarray(expected).view(np.uint8)), what


# ---- the cache -----------------------------------------------------------------------------------------------------

CACHE_CASES = [
    # cache, rows, tokens, heads, width, page, layout, padding behind a row
    (DType.I8, DType.F16, 1, 8, 128, 16, "dense", 0),
    (DType.I8, DType.F32, 37, 3, 64, 16, "dense", 0),
    (DType.I8, DType.F16, 130, 5, 80, 48, "tokens first", 16),
    (DType.I8, DType.F16, 19, 2, 256, 7, "dense", 32),
    (DType.I8, DType.F32, 33, 1, 16, 1, "dense", 0),
    (DType.F16, DType.F16, 65, 2, 96, 16, "tokens first", 8),
    (DType.F16, DType.F32, 41, 4, 144, 5, "dense", 0),
    (DType.F16, DType.F16, 1, 1, 16, 1000, "dense", 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CACHE_CASES, ids=lambda c: f"{c[0].name}-{c[1].name}-{c[2]}x{c[3]}x{c[4]}-p{c[5]}-{c[6].split()[0]}{c[7]}")
def test_cache_write_and_read_back(case, hip_device):
    dtype, rows_dtype, tokens, heads, width, page, order, spread = case
    rng = np.random.default_rng(tokens + width)
    pages = tokens // page + 3
    cache = CacheCase(hip_device, dtype, pages, heads, page, width, spread, order)
    args = cache.upload()
    # rows of the caller lie apart, [heads, tokens, width + 3]: another order than the cache's, at odd addresses
    mem = rng.standard_normal((2, heads, tokens, width + 3)).astype(NP[rows_dtype])
    mem[0, 0, 0, :width] = 0  # a row of zeros
    if tokens > 4:
        mem[0, :, 1] *= np.float32(1e-6)       # f16: below the normal numbers
        mem[1, :, 2, 5] = np.inf
        mem[1, :, 3, 7] = -np.inf
        mem[0, :, 4, 3] = np.nan
    if rows_dtype == DType.F32:
        mem[1, :, -1, 0] = 1e30                # beyond what f16 holds
        mem[1, 0, -1, 1:width] = 1e-44
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    skipped = np.zeros(tokens, bool)
    if tokens > 6:
        slots[5], slots[6] = -1, pages * page
        skipped[5:7] = True
    rows_dev, slots_dev = upload(hip_device, mem), upload(hip_device, slots)
    elem = mem.itemsize
    strides = (width + 3, tokens * (width + 3))
    stream = kn.HipStream(hip_device)
    rows = kn.cache_rows(rows_dtype, tokens, rows_dev.ptr, strides, rows_dev.ptr + mem[0].size * elem, strides, slots_dev.ptr)
    kn.cache_write(hip_device, stream, args, rows)
    stream.synchronize()

    expected = CacheCase(hip_device, dtype, pages, heads, page, width, spread, order)
    x = np.moveaxis(mem[..., :width], 1, 2)  # [2, tokens, heads, width]
    if dtype == DType.F16:
        with np.errstate(over="ignore"):
            x = np.clip(x, -65504, 65504).astype(np.float16)  # (clip keeps a NaN)
    expected.put(slots[~skipped], x[0][~skipped], x[1][~skipped])
    cache.download()
    _same(cache.k, expected.k, "k")
    _same(cache.v, expected.v, "v")
    _same(cache.ks, expected.ks, "k_scales: " + ("division of a row's maximum by 127" if dtype == DType.I8 else "not touched"))
    _same(cache.vs, expected.vs, "v_scales")

    for out_dtype in (DType.F16, DType.F32):
        want = np.concatenate([slots, slots[:1]])  # a slot twice
        back = np.full((2, tokens + 1, heads, width + 5), 7, NP[out_dtype])
        back_dev, want_dev = upload(hip_device, back), upload(hip_device, want)
        o = (heads * (width + 5), width + 5)
        kn.cache_read(hip_device, stream, args, kn.cache_rows(out_dtype, tokens + 1, back_dev.ptr, o, back_dev.ptr + back[0].nbytes, o, want_dev.ptr))
        stream.synchronize()
        got = back_dev.to_array(back.dtype, back.shape)
        inside = (want >= 0) & (want < pages * page)
        for i, held in enumerate(expected.held(np.where(inside, want, 0))):
            with np.errstate(invalid="ignore"):
                # (a product of a whole number and an f32 scale has 31 bits: rounded to f32 first, then to the rows' type)
                held = np.where(inside[:, None, None], held, 0.0).astype(np.float32).astype(back.dtype)
            a, e = got[i, :, :, :width], held
            assert np.array_equal(a, e, equal_nan=True), f"{out_dtype.name} {'kv'[i]}"
        assert (got[..., width:] == 7).all(), "between the rows"


# ---- attention over the cache --------------------------------------------------------------------------------------

def _cached_case(device, c, seed=0):
    rng = np.random.default_rng(seed + 1000)
    N, G, W, T, page, P = c["kv"], c["group"], c["width"], c.get("queries", 1), c["page"], c.get("prefix", 0)
    lengths, B, H = list(c["lengths"]), len(c["lengths"]), c["kv"] * c["group"]
    table_pages = c.get("table_pages", max(1, max(-(-max(n, 0) // page) for n in lengths)))
    need = -(-P // page) + sum(-(-min(max(n, 0), table_pages * page) // page) for n in lengths)
    cache = CacheCase(device, c["dtype"], need + 2, N, page, W, c.get("spread", 0), c.get("order", "dense"))
    free = list(rng.permutation(need + 2))
    prefix_table = np.array([free.pop() for _ in range(-(-P // page))], np.int32)
    tables = np.full((B, table_pages + 2), 1 << 30, np.int32)  # what lies behind a table or a sequence is no page
    for b, n in enumerate(lengths):
        n = min(max(n, 0), table_pages * page)
        tables[b, :-(-n // page)] = [free.pop() for _ in range(-(-n // page))]

    def slots(table, n):
        j = np.arange(n)
        return table[j // page].astype(np.int64) * page + j % page

    def fill(s):
        k = rng.standard_normal((len(s), N, W)) * c.get("size", 1.0)
        cache.put(s, k.astype(np.float16), rng.standard_normal((len(s), N, W)).astype(np.float16))

    fill(slots(prefix_table, P))
    for b, n in enumerate(lengths):
        fill(slots(tables[b], min(max(n, 0), table_pages * page)))
    if "infinite" in c:  # (key, element) of the first sequence
        at, d = c["infinite"]
        k, v = cache.held(slots(tables[0], at + 1)[-1:])
        v[..., d] = -np.inf
        cache.put(slots(tables[0], at + 1)[-1:], k.astype(np.float16), v.astype(np.float16))
    poisoned = c.get("poison", False)  # the last token of every sequence: only its own query sees it
    if poisoned:
        for b, n in enumerate(lengths):
            if n > 0:
                cache.put(slots(tables[b], n)[-1:], np.full((1, N, W), np.nan, np.float16), np.full((1, N, W), -np.inf, np.float16))
    lost = c.get("lost", ())  # (sequence or -1 for the prefix, page of its table): not there
    gone = {}
    for b, i in lost:
        table = prefix_table if b < 0 else tables[b]
        gone[(b, i)] = table[i]
        table[i] = rng.choice([-1, need + 2, -(1 << 31), (1 << 31) - 1])
    # q and out are strided views, [heads, batch, tokens, width + 8] and [batch, heads, tokens, width + 3]
    q_mem = rng.standard_normal((H, B, T, W + 8)).astype(np.float16)
    out_mem = np.full((B, H, T, W + 3), GUARD, np.float16)
    slopes = np.array([2.0 ** -(1 + h % 8) for h in range(H)], np.float32) if c.get("slopes") else None
    scale, cap, window = c.get("scale", W ** -0.5), c.get("cap", 0.0), c.get("window", 0)

    args_cache = cache.upload()
    dev = [upload(device, a) for a in (q_mem, out_mem, np.array(lengths, np.int32), tables, prefix_table, slopes if slopes is not None else np.zeros(1, np.float32))]
    args = kn.cached_attention_args(B, T, H, args_cache, dev[0].ptr, (T * (W + 8), W + 8, B * T * (W + 8)), dev[1].ptr,
                                    (H * T * (W + 3), W + 3, T * (W + 3)), dev[2].ptr, dev[3].ptr, table_pages + 2, table_pages,
                                    prefix_tokens=P, prefix_table=dev[4].ptr if P else 0, scale=scale, cap=cap,
                                    slopes=dev[5].ptr if slopes is not None else 0, window=window)

    def expected():
        out, bound = np.zeros((B, H, T, W)), np.zeros((B, H, T, W))
        for b, n in enumerate(lengths):
            n = min(max(n, 0), table_pages * page)
            table, first = tables[b].copy(), prefix_table.copy()
            there = np.ones(P + n, bool)
            for (s, i), was in gone.items():
                if s < 0:
                    first[i] = was
                    there[i * page:min((i + 1) * page, P)] = False
                elif s == b:
                    table[i] = was
                    there[P + i * page:P + min((i + 1) * page, n)] = False
            kp, vp = cache.held(slots(first, P))
            ko, vo = cache.held(slots(table, n))
            k, v = np.concatenate([kp, ko]), np.concatenate([vp, vo])
            at = P + n - T + np.arange(T)
            places = np.arange(P + n)
            if poisoned and n > 0:
                k[-1], v[-1] = 0, 0
            visible = (places <= at[:, None]) & (at[:, None] >= P) & there
            if window:
                visible &= places > at[:, None] - window
            for h in range(H):
                q = q_mem[h, b, :, :W].astype(np.float64)
                out[b, h], e = attend(q, k[:, h // G], v[:, h // G], at, places, visible, scale, cap, slopes[h] if slopes is not None else 0.0)
                if c["dtype"] == DType.I8 and len(places):
                    # keys and values of 8 bits may be rounded to f16 on their way into the products: half a step each
                    move = 2.0 ** -11 * abs(scale) * np.where(visible, np.abs(q) @ np.abs(k[:, h // G]).T, 0).max(-1, keepdims=True, initial=0)
                    e = e + (e * 2.0 ** 11) * 2 * move + e
                bound[b, h] = e
        return out, bound

    return dict(args=args, dev=dev, cache=cache, out_mem=out_mem, expected=expected, W=W, compared=T - 1 if poisoned else T)


CACHED_CASES = {
    "one_token_one_key": dict(dtype=DType.F16, kv=1, group=1, width=64, page=16, lengths=[1]),
    "one_sequence": dict(dtype=DType.I8, kv=8, group=4, width=128, page=16, lengths=[517]),
    "ragged_with_empty": dict(dtype=DType.I8, kv=2, group=3, width=64, page=16, lengths=[0, 1, 15, 16, 17, 63, 64, 65, 300, -4]),
    "ragged_f16": dict(dtype=DType.F16, kv=2, group=8, width=128, page=16, lengths=[1, 1200, 31, 33, 0, 500]),
    "odd_pages": dict(dtype=DType.F16, kv=2, group=2, width=96, page=7, lengths=[50, 3, 129]),
    "single_token_pages": dict(dtype=DType.I8, kv=1, group=5, width=80, page=1, lengths=[40, 77]),
    "one_page_per_sequence": dict(dtype=DType.F16, kv=2, group=1, width=64, page=700, lengths=[700, 1, 333]),
    "several_queries": dict(dtype=DType.I8, kv=2, group=4, width=128, page=16, lengths=[3, 100, 5, 4, 513], queries=4),
    "more_queries_than_a_tile": dict(dtype=DType.F16, kv=2, group=4, width=128, page=16, lengths=[70, 300, 20], queries=37),
    "a_prompt_over_the_cache": dict(dtype=DType.I8, kv=1, group=2, width=64, page=16, lengths=[260, 129], queries=130),
    "prefix": dict(dtype=DType.I8, kv=2, group=4, width=128, page=16, lengths=[5, 40, 0, 100], prefix=333),
    "prefix_of_one": dict(dtype=DType.F16, kv=1, group=3, width=64, page=16, lengths=[1, 2, 30], prefix=1),
    "prefix_many_rows": dict(dtype=DType.I8, kv=2, group=4, width=128, page=48, lengths=[(7 * i) % 60 for i in range(45)], prefix=1000),
    "prefix_f16_many_rows": dict(dtype=DType.F16, kv=1, group=8, width=96, page=16, lengths=[(11 * i) % 90 for i in range(33)], prefix=515),
    "prefix_and_queries": dict(dtype=DType.I8, kv=2, group=2, width=64, page=16, lengths=[9, 2, 70], queries=3, prefix=100),
    "cap_bias_window": dict(dtype=DType.I8, kv=2, group=4, width=128, page=16, lengths=[300, 10, 64], cap=20.0, slopes=True, window=100, size=3.0),
    "cap_bias_window_prefix": dict(dtype=DType.F16, kv=2, group=4, width=64, page=16, lengths=[30, 100, 5], prefix=200, cap=5.0, slopes=True, window=120, size=3.0),
    "window_of_one": dict(dtype=DType.I8, kv=1, group=4, width=128, page=16, lengths=[40, 1, 33], window=1),
    "window_inside_own": dict(dtype=DType.F16, kv=1, group=2, width=128, page=16, lengths=[200, 90], prefix=64, window=50, queries=2),
    "bias_long_prefix": dict(dtype=DType.I8, kv=1, group=8, width=64, page=16, lengths=[12] * 20, prefix=2100, slopes=True),
    "lost_pages": dict(dtype=DType.I8, kv=2, group=4, width=128, page=16, lengths=[100, 40, 16], lost=[(0, 2), (1, 0), (2, 0)], prefix=50),
    "lost_prefix": dict(dtype=DType.F16, kv=1, group=4, width=128, page=16, lengths=[20] * 12, prefix=96, lost=[(-1, 1), (-1, 5), (3, 1)]),
    "table_too_short": dict(dtype=DType.I8, kv=1, group=2, width=64, page=16, lengths=[100, 20], table_pages=3),
    "tokens_first_layout": dict(dtype=DType.I8, kv=3, group=2, width=64, page=16, lengths=[77, 200], order="tokens first", spread=16),
    "scale_of_zero": dict(dtype=DType.F16, kv=1, group=1, width=64, page=16, lengths=[90], scale=0.0),
    "negative_scale": dict(dtype=DType.I8, kv=1, group=1, width=64, page=16, lengths=[90], scale=-0.2),
    "peaked": dict(dtype=DType.F16, kv=1, group=4, width=128, page=16, lengths=[600, 50], size=30.0),
    "narrow": dict(dtype=DType.I8, kv=2, group=2, width=16, page=16, lengths=[70, 5]),
    "newest_is_not_finite": dict(dtype=DType.F16, kv=2, group=4, width=128, page=16, lengths=[40, 7, 33, 0, 700], queries=3, poison=True),
    "newest_is_not_finite_odd_pages": dict(dtype=DType.F16, kv=1, group=3, width=64, page=5, lengths=[40, 300], queries=7, poison=True, prefix=20),
    "newest_is_not_finite_tiles": dict(dtype=DType.F16, kv=1, group=4, width=64, page=16, lengths=[100, 50, 290], queries=50, poison=True),
    "long_windows": dict(dtype=DType.I8, kv=1, group=2, width=64, page=16, lengths=[3, 100, 0], queries=5, window=(1 << 31) - 1, prefix=40),
    "many_sequences": dict(dtype=DType.I8, kv=1, group=2, width=64, page=16, lengths=[(13 * i) % 70 for i in range(150)]),
    "long_and_short": dict(dtype=DType.I8, kv=1, group=2, width=64, page=16, lengths=[9000, 5, 0, 2500]),
    "long_f16_wide_rows": dict(dtype=DType.F16, kv=1, group=4, width=128, page=16, lengths=[5000, 40], queries=8),
    "prefix_apart": dict(dtype=DType.I8, kv=2, group=4, width=128, page=16, lengths=[(7 * i) % 60 for i in range(40)], prefix=1801, lost=[(-1, 3), (2, 0)]),
    "prefix_apart_f16": dict(dtype=DType.F16, kv=1, group=4, width=64, page=48, lengths=[(7 * i) % 60 for i in range(20)], prefix=1999, cap=9.0, slopes=True, window=1900),
    "prefix_apart_few_rows": dict(dtype=DType.I8, kv=2, group=4, width=128, page=16, lengths=[50, 0, 1300], prefix=1000, queries=2),
    "prefix_inside_several_items": dict(dtype=DType.I8, kv=2, group=4, width=128, page=16, lengths=[3000, 0, 5, 1300], prefix=333, queries=3),
    "prefix_inside_window": dict(dtype=DType.F16, kv=1, group=8, width=96, page=16, lengths=[30, 400, 5], prefix=200, window=100, queries=2, slopes=True),
    "prefix_inside_lost": dict(dtype=DType.F16, kv=1, group=4, width=128, page=7, lengths=[20, 3, 0], queries=3, prefix=50, lost=[(-1, 0), (-1, 6), (0, 1)], poison=True),
    "many_prompts_over_the_cache": dict(dtype=DType.F16, kv=2, group=1, width=128, page=16, lengths=[40 + (9 * i) % 100 for i in range(200)], queries=40, poison=True),
    "many_long_prompts_over_the_cache": dict(dtype=DType.F16, kv=2, group=8, width=128, page=16, lengths=[120 + i for i in range(70)], queries=130, prefix=70),
    "many_prompts_over_the_cache_i8": dict(dtype=DType.I8, kv=2, group=1, width=64, page=16, lengths=[(9 * i) % 120 for i in range(200)], queries=40, prefix=100, cap=9.0),
    "many_heads_of_one": dict(dtype=DType.I8, kv=1, group=71, width=64, page=16, lengths=[300, 4]),
}


def _check(got, out, bound, width, what):
    assert not np.isnan(got[..., :width]).any(), f"{what}: NaN"
    off = np.abs(got[..., :width].astype(np.float64) - out)
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert (off <= bound).all(), f"{what}: {off[worst]:.3e} off at {worst}, at most {bound[worst]:.3e} ({(off > bound).mean():.2%} of the values)"
    assert (got[..., width:] == GUARD).all(), f"{what}: written between the rows"


@pytest.mark.gpu
@pytest.mark.parametrize("name", CACHED_CASES)
def test_cached_attention(name, hip_device):
    c = _cached_case(hip_device, CACHED_CASES[name])
    stream = kn.HipStream(hip_device)
    need = kn.cached_attention_workspace_bytes(c["args"])
    workspace = kn.DeviceBuffer(hip_device, need) if need else None
    out, bound = c["expected"]()
    for round_ in range(2):  # on the same workspace
        kn.cached_attention(hip_device, stream, c["args"], workspace)
        stream.synchronize()
        got, n = c["dev"][1].to_array(np.float16, c["out_mem"].shape), c["compared"]
        _check(got[:, :, :n], out[:, :, :n], bound[:, :, :n], c["W"], f"{name}, call {round_}")


# ---- attention of prompts ------------------------------------------------------------------------------------------

def _documents(tokens, cuts):
    s = np.zeros((tokens, 2), np.int32)
    cuts = [0] + list(cuts) + [tokens]
    for lo, hi in zip(cuts, cuts[1:]):
        s[lo:hi] = (lo, hi)
    return s


PROMPT_CASES = {
    "one_token": dict(queries=1, heads=1, kv=1, width=64, causal=True),
    "no_mask": dict(queries=70, heads=2, kv=2, width=64),
    "causal": dict(batch=2, queries=200, heads=4, kv=2, width=128, causal=True),
    "causal_long": dict(queries=1100, heads=2, kv=1, width=128, causal=True),
    "odd_width": dict(queries=129, heads=3, kv=3, width=72, causal=True),
    "narrow": dict(queries=65, heads=2, kv=1, width=8, causal=True),
    "last_queries": dict(queries=40, keys=333, heads=4, kv=4, width=64, causal=True),
    "more_queries_than_keys": dict(queries=100, keys=30, heads=2, kv=2, width=64, causal=True),
    "no_keys": dict(queries=5, keys=0, heads=2, kv=2, width=64),
    "cross": dict(batch=3, queries=50, keys=77, heads=4, kv=2, width=40),
    "cap": dict(queries=257, heads=2, kv=2, width=128, causal=True, cap=5.0, size=4.0),
    "tiny_cap": dict(queries=150, heads=2, kv=2, width=128, causal=True, cap=1e-6),
    "tiny_cap_equal_scores": dict(queries=150, heads=2, kv=2, width=128, causal=True, cap=1e-6, scale=0.0),
    "huge_cap": dict(queries=150, heads=2, kv=2, width=64, causal=True, cap=1e30),
    "bias": dict(queries=300, heads=4, kv=4, width=64, causal=True, slopes=True),
    "bias_both_sides": dict(queries=150, heads=2, kv=2, width=64, slopes=True),
    "window": dict(queries=400, heads=2, kv=1, width=128, causal=True, window=37),
    "window_of_one": dict(queries=130, heads=1, kv=1, width=64, causal=True, window=1),
    "longest_window": dict(queries=50, keys=20, heads=1, kv=1, width=64, window=(1 << 31) - 1),
    "window_not_causal": dict(queries=200, heads=1, kv=1, width=64, window=20),
    "documents": dict(batch=2, queries=500, heads=2, kv=2, width=128, causal=True, spans=[[3, 130, 131, 300], [64, 128, 448]]),
    "documents_not_causal": dict(queries=300, heads=2, kv=1, width=64, spans=[[100, 164]]),
    "prefix": dict(batch=3, queries=190, heads=2, kv=2, width=64, causal=True, prefix=[0, 77, 1000]),
    "everything": dict(batch=2, queries=333, heads=4, kv=2, width=80, causal=True, cap=10.0, slopes=True, window=90, prefix=[40, 0],
                       spans=[[50, 200], [111]], size=3.0),
    "padded_batch": dict(batch=3, queries=140, heads=2, kv=2, width=128, causal=True, lengths=[140, 1, 0]),
    "unseen_is_nan": dict(batch=2, queries=260, heads=2, kv=2, width=64, causal=True, lengths=[100, 259], poison=True),
    "future_is_nan": dict(queries=200, keys=200, heads=2, kv=2, width=64, causal=True, poison_from=150),
    "many_prompts": dict(batch=210, queries=70, heads=2, kv=2, width=128, causal=True, lengths=[(7 * i) % 71 for i in range(210)], poison=True),
    "many_long_prompts": dict(batch=70, queries=130, heads=16, kv=2, width=128, causal=True, lengths=[(7 * i) % 131 for i in range(70)], poison=True),
    "many_long_prompts_capped": dict(batch=70, queries=130, keys=150, heads=16, kv=2, width=104, causal=True, cap=8.0, slopes=True, window=90, size=2.0),
    "many_prompts_everything": dict(batch=200, queries=40, keys=150, heads=4, kv=2, width=64, causal=True, cap=8.0, slopes=True, window=90,
                                    prefix=[i % 60 for i in range(200)], size=2.0),
    "past_is_nan": dict(queries=200, heads=1, kv=1, width=128, causal=True, window=30, poison_to=71),
}


# (key, element, value): +inf or -inf among the values, which makes that element of all that see the key infinite
PROMPT_INFINITE = {
    "first_block": dict(queries=50, heads=2, kv=1, width=64, causal=True, infinite=[(0, 5, 1), (20, 9, -1), (49, 63, 1)]),
    "later_blocks": dict(queries=300, heads=2, kv=2, width=128, causal=True, window=150, infinite=[(63, 0, 1), (64, 127, -1), (200, 64, 1)]),
    "whole_blocks": dict(queries=64, keys=128, heads=1, kv=1, width=64, infinite=[(10, 3, 1), (100, 4, -1)]),
    "many": dict(batch=400, queries=35, keys=100, heads=1, kv=1, width=64, causal=True, infinite=[(0, 5, 1), (70, 9, -1), (99, 63, 1)]),
    "in_parts": dict(queries=100, keys=1500, heads=1, kv=1, width=64, causal=True, infinite=[(3, 1, 1), (700, 2, -1), (1450, 3, 1)]),
}


def _prompt_case(device, c, seed=0):
    rng = np.random.default_rng(seed + 7)
    B, S, H, N, W = c.get("batch", 1), c["queries"], c["heads"], c["kv"], c["width"]
    K = c.get("keys", S)
    # q [batch, heads, tokens, width + 1], k [batch, tokens, heads, width], v the same with 5 elements in front, out [heads, ...]
    q_mem = rng.standard_normal((B, H, S, W + 1)).astype(np.float16)
    k_mem = (rng.standard_normal((B, K, N, W)) * c.get("size", 1.0)).astype(np.float16)
    v_mem = rng.standard_normal((B, K, N, W + 5)).astype(np.float16)
    spans = None
    if "spans" in c:
        spans = np.stack([_documents(S, cuts) for cuts in c["spans"]])
    if "lengths" in c:
        spans = np.zeros((B, S, 2), np.int32)
        for b, n in enumerate(c["lengths"]):
            spans[b, :n] = (0, n)
            spans[b, n:] = (n, n) if n % 2 else (5, -3)  # empty either way
            if c.get("poison"):
                k_mem[b, n:], v_mem[b, n:] = np.nan, np.inf
    at = np.arange(S) + K - S
    places = np.arange(K)
    visible = np.ones((B, S, K), bool)
    if c.get("causal"):
        seen = np.broadcast_to(places <= at[:, None], (B, S, K)).copy()
        if "prefix" in c:
            seen |= places < np.array(c["prefix"])[:, None, None]
        visible &= seen
    if c.get("window"):
        visible &= places > at[:, None] - c["window"]
    if spans is not None:
        visible &= (places >= spans[..., :1]) & (places < spans[..., 1:])
    clean_k, clean_v = k_mem.copy(), v_mem.copy()
    if "poison_from" in c:
        k_mem[:, c["poison_from"]:], v_mem[:, c["poison_from"]:] = np.inf, np.nan
    if "poison_to" in c:
        k_mem[:, :c["poison_to"]], v_mem[:, :c["poison_to"]] = np.nan, -np.inf
    for key, d, sign in c.get("infinite", ()):
        v_mem[:, key, :, 5 + d] = sign * np.inf
        clean_v[:, key, :, 5 + d] = 0
    slopes = np.array([2.0 ** -(1 + h % 8) for h in range(H)], np.float32) if c.get("slopes") else None
    out_mem = np.full((H, B, S, W + 3), GUARD, np.float16)
    prefix = np.array(c.get("prefix", [0]), np.int32)
    dev = [upload(device, a) for a in (q_mem, k_mem, v_mem, out_mem, spans if spans is not None else np.zeros(1, np.int32), prefix,
                                       slopes if slopes is not None else np.zeros(1, np.float32))]
    scale, cap = c.get("scale", W ** -0.5), c.get("cap", 0.0)
    args = kn.attention_args(B, S, K, H, N, W, dev[0].ptr, (H * S * (W + 1), W + 1, S * (W + 1)), dev[1].ptr, (K * N * W, N * W, W),
                             dev[2].ptr + 10, (K * N * (W + 5), N * (W + 5), W + 5), dev[3].ptr, (S * (W + 3), W + 3, B * S * (W + 3)),
                             scale=scale, cap=cap, slopes=dev[6].ptr if slopes is not None else 0, causal=c.get("causal", False),
                             window=c.get("window", 0), spans=dev[4].ptr if spans is not None else 0, prefix=dev[5].ptr if "prefix" in c else 0)
    # rows that see something poisoned are left out of the comparison
    bad = np.zeros((B, K), bool)
    if "poison_from" in c:
        bad[:, c["poison_from"]:] = True
    if "poison_to" in c:
        bad[:, :c["poison_to"]] = True
    compared = ~(visible & bad[:, None]).any(-1)

    def expected():
        out, bound = np.zeros((H, B, S, W)), np.zeros((H, B, S, W))
        for b in range(B):
            for h in range(H):
                k, v = clean_k[b, :, h * N // H].astype(np.float64), clean_v[b, :, h * N // H, 5:].astype(np.float64)
                seen = visible[b] & compared[b][:, None]
                dead = ~seen.any(0)
                k[dead], v[dead] = 0, 0
                out[h, b], bound[h, b] = attend(q_mem[b, h, :, :W].astype(np.float64), k, v, at, places, seen, scale, cap, slopes[h] if slopes is not None else 0.0)
        return out, bound

    infinite = np.zeros((H, B, S, W))
    for key, d, sign in c.get("infinite", ()):
        infinite[..., d] = np.where(visible[None, :, :, key], sign, 0)
    return dict(args=args, dev=dev, out_mem=out_mem, expected=expected, W=W, compared=compared, infinite=infinite)


@pytest.mark.gpu
@pytest.mark.parametrize("name", PROMPT_CASES)
def test_attention_of_prompts(name, hip_device):
    c = _prompt_case(hip_device, PROMPT_CASES[name])
    stream = kn.HipStream(hip_device)
    need = kn.attention_workspace_bytes(c["args"])
    workspace = kn.DeviceBuffer(hip_device, need) if need else None
    out, bound = c["expected"]()
    for round_ in range(2):
        kn.attention(hip_device, stream, c["args"], workspace)
        stream.synchronize()
        got = c["dev"][3].to_array(np.float16, c["out_mem"].shape)
        got[..., :c["W"]][:, ~c["compared"]] = 0
        _check(got, out, bound, c["W"], f"{name}, call {round_}")


@pytest.mark.gpu
@pytest.mark.parametrize("name", PROMPT_INFINITE)
def test_attention_of_prompts_keeps_infinities(name, hip_device):
    c = _prompt_case(hip_device, PROMPT_INFINITE[name])
    stream = kn.HipStream(hip_device)
    need = kn.attention_workspace_bytes(c["args"])
    workspace = kn.DeviceBuffer(hip_device, need) if need else None
    out, bound = c["expected"]()
    kn.attention(hip_device, stream, c["args"], workspace)
    stream.synchronize()
    got = c["dev"][3].to_array(np.float16, c["out_mem"].shape)
    values, there = got[..., :c["W"]], c["infinite"] != 0
    assert (values[there] == np.copysign(np.inf, c["infinite"][there])).all(), name
    values[there] = out[there]
    _check(got, out, bound, c["W"], name)


@pytest.mark.gpu
@pytest.mark.parametrize("queries,length,key", [(40, 50, 12), (40, 50, 0), (40, 300, 270), (1, 40, 39), (3, 100, 98), (3, 2500, 1200)])
def test_cached_attention_keeps_infinities(queries, length, key, hip_device):
    """an infinity among the values of a key: the same element of every query that sees it"""
    c = dict(dtype=DType.F16, kv=1, group=2, width=64, page=16, lengths=[length], queries=queries)
    finite, with_one = _cached_case(hip_device, c), _cached_case(hip_device, dict(c, infinite=(key, 7)))
    stream = kn.HipStream(hip_device)
    got = []
    for case in (finite, with_one):
        need = kn.cached_attention_workspace_bytes(case["args"])
        kn.cached_attention(hip_device, stream, case["args"], kn.DeviceBuffer(hip_device, need) if need else None)
        stream.synchronize()
        got.append(case["dev"][1].to_array(np.float16, case["out_mem"].shape))
    sees = length - queries + np.arange(queries) >= key
    assert (got[1][:, :, sees, 7] == -np.inf).all()
    got[1][:, :, sees, 7] = got[0][:, :, sees, 7]
    assert np.array_equal(got[0], got[1])


# ---- sampling ------------------------------------------------------------------------------------------------------

def _logits(rng, kind, rows, vocab):
    x = rng.standard_normal((rows, vocab)) * 2.5
    if kind == "flat":
        x[:] = rng.standard_normal((rows, 1))
    elif kind == "few values":
        x = np.round(x)
    elif kind == "peaked":
        x[np.arange(rows), rng.integers(0, vocab, rows)] += 30
    elif kind == "wide":
        x *= 1000
    elif kind == "special":
        x[0] = -np.inf
        x[1, rng.integers(0, vocab, vocab // 2)] = -np.inf
        x[2, rng.integers(0, vocab, vocab // 2)] = np.nan
        x[3, rng.integers(0, vocab, 3)] = np.inf
        x[4] = np.nan
        x[5] = -np.inf
        x[5, vocab // 2] = -1e4
        x[6] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
        x[7] = -65504.0
        x[8] = np.inf
    return x


SAMPLE_CASES = [
    # rows, vocab, dtype, logits, temperature, top_k, top_p, min_p (a number, or None: off)
    (1, 1, DType.F32, "normal", None, None, None, None),
    (3, 2, DType.F16, "normal", 1.0, 1, 0.5, None),
    (5, 1000, DType.F32, "normal", None, None, None, None),
    (4, 1001, DType.F16, "normal", 0.0, 5, 0.5, 0.1),
    (1, 32000, DType.F16, "normal", 0.8, 40, 0.95, None),
    (7, 32003, DType.F32, "normal", 1.3, None, 0.9, None),
    (6, 50001, DType.F16, "normal", 1.0, None, 0.92, None),
    (3, 128001, DType.F32, "normal", 0.7, 1000, 0.9, 0.02),
    (3, 128001, DType.F32, "normal", 1.0, 100000, 0.999, None),
    (2, 9000, DType.F32, "flat", 0.5, None, None, None),
    (4, 9000, DType.F16, "flat", 0.5, 777, 0.3, 0.9),
    (4, 20000, DType.F32, "flat", 1.0, None, 0.7, 1.0),
    (6, 30000, DType.F16, "few values", 1.0, 4321, 0.8, None),
    (6, 30000, DType.F32, "few values", 0.9, None, 0.999999, 0.001),
    (5, 40000, DType.F32, "peaked", 1.0, 50, 0.95, 0.05),
    (5, 40000, DType.F32, "peaked", 25.0, None, 0.5, None),
    (3, 5000, DType.F32, "wide", 1.0, 3000, 1.0, None),
    (3, 5000, DType.F32, "wide", 700.0, 1, 0.9, None),
    (9, 3000, DType.F32, "special", 1.0, 40, 0.9, None),
    (9, 3000, DType.F16, "special", 1.0, None, None, None),
    (9, 3000, DType.F16, "special", 0.0, None, None, None),
    (300, 257, DType.F32, "normal", 1.0, 20, 0.9, 0.01),
    (2, 1 << 20, DType.F16, "normal", 1.0, None, 0.9, None),
    (3, 700, DType.F32, "normal", 1.0, 5000, 1.5, 2.0),
    (3, 700, DType.F32, "normal", 1.0, -3, 0.0, -1.0),
]


def _sample_call(device, logits, dtype, uniform, pad=0, **filters):
    rows, vocab = logits.shape
    mem = np.full((rows, vocab + pad), np.inf, NP[dtype])
    mem[:, :vocab] = logits
    types = dict(temperature=np.float32, top_k=np.int32, top_p=np.float32, min_p=np.float32)
    dev = {n: upload(device, np.asarray(v, types[n])) for n, v in filters.items() if v is not None}
    dev.update(logits=upload(device, mem), uniform=upload(device, uniform.astype(np.float32)),
               tokens=upload(device, np.full(rows + 1, GUARD, np.int32)), probabilities=upload(device, np.full(rows + 1, GUARD, np.float32)))
    args = kn.sample_args(dtype, rows, vocab, dev["logits"].ptr, vocab + pad, dev["uniform"].ptr, dev["tokens"].ptr,
                          probabilities=dev["probabilities"].ptr, **{n: dev[n].ptr for n in filters if filters[n] is not None})
    need = kn.sample_workspace_bytes(args)
    return args, dev, kn.DeviceBuffer(device, need) if need else None


@pytest.mark.gpu
@pytest.mark.parametrize("case", SAMPLE_CASES, ids=lambda c: "-".join(str(getattr(x, "name", x)).replace(" ", "_") for x in c))
def test_sample(case, hip_device):
    rows, vocab, dtype, kind, *given = case
    rng = np.random.default_rng(vocab + rows)
    with np.errstate(over="ignore"):
        logits = _logits(rng, kind, rows, vocab).astype(NP[dtype])
    uniform = rng.random(rows).astype(np.float32)
    uniform[0] = 0.0
    if rows > 2:
        uniform[1], uniform[2] = 1.0, -3.0  # count as the nearest number in [0, 1)
    filters = {}
    for name, value in zip(("temperature", "top_k", "top_p", "min_p"), given):
        if value is None:
            continue
        each = np.full(rows, value, np.int32 if name == "top_k" else np.float32)
        if rows > 4:  # rows of one call differ
            each[3] = {"temperature": 0.9, "top_k": 3, "top_p": 0.2, "min_p": 0.3}[name]
        filters[name] = each
    args, dev, workspace = _sample_call(hip_device, logits, dtype, uniform, pad=rows % 4, **filters)
    tokens, chance = sample(logits, uniform, **filters)
    stream = kn.HipStream(hip_device)
    for round_ in range(2):
        kn.sample(hip_device, stream, args, workspace)
        stream.synchronize()
        got, p = dev["tokens"].to_array(np.int32, rows + 1), dev["probabilities"].to_array(np.float32, rows + 1)
        assert np.array_equal(got[:rows], tokens) and got[rows] == GUARD and p[rows] == GUARD, (round_, got[:rows], tokens)
        # fixed point weights are off by half of 2^-(62 - 20) at most each, f32 rounds by 2^-24 of the value
        assert (np.abs(p[:rows] - chance) <= chance * 2.0 ** -23 + vocab * 2.0 ** -42).all()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(30))
def test_sample_random(seed, hip_device):
    """sizes and filters anywhere in their ranges, every row with its own"""
    rng = np.random.default_rng(100 + seed)
    rows, vocab = int(rng.integers(1, 9)), int(np.exp(rng.uniform(0, np.log(400000))))
    dtype, kind = [(DType.F16, DType.F32)[seed % 2], ("normal", "normal", "few values", "peaked", "wide", "flat")[seed % 6]]
    with np.errstate(over="ignore"):
        logits = _logits(rng, kind, rows, vocab).astype(NP[dtype])
    filters = dict(temperature=rng.choice([0.3, 0.7, 1.0, 1.0, 2.0, 20.0], rows).astype(np.float32),
                   top_k=rng.choice([0, 1, 2, 7, 40, 63, 64, 65, 300, 1024, 1025, 20000], rows).astype(np.int32),
                   top_p=rng.choice([1.0, 0.999, 0.95, 0.9, 0.5, 0.01], rows).astype(np.float32), min_p=rng.choice([0.0, 0.0, 1e-4, 0.05, 0.5], rows).astype(np.float32))
    filters = {n: a for n, a in filters.items() if rng.random() < 0.8}
    uniform = rng.random(rows).astype(np.float32)
    args, dev, workspace = _sample_call(hip_device, logits, dtype, uniform, pad=int(rng.integers(0, 4)), **filters)
    stream = kn.HipStream(hip_device)
    kn.sample(hip_device, stream, args, workspace)
    stream.synchronize()
    tokens, chance = sample(logits, uniform, **filters)
    got, p = dev["tokens"].to_array(np.int32, rows), dev["probabilities"].to_array(np.float32, rows)
    assert np.array_equal(got, tokens), (vocab, dtype, kind, filters)
    assert (np.abs(p - chance) <= chance * 2.0 ** -23 + vocab * 2.0 ** -42).all()


@pytest.mark.gpu
def test_sampling_follows_the_probabilities(hip_device):
    """evenly spaced random numbers draw every token as often as its probability says"""
    rng = np.random.default_rng(2)
    rows = 4096
    row = rng.standard_normal(50).astype(np.float32)
    uniform = (np.arange(rows) + 0.5) / rows
    args, dev, workspace = _sample_call(hip_device, np.tile(row, (rows, 1)), DType.F32, uniform)
    stream = kn.HipStream(hip_device)
    kn.sample(hip_device, stream, args, workspace)
    stream.synchronize()
    drawn = np.bincount(dev["tokens"].to_array(np.int32, rows), minlength=50) / rows
    w = np.exp(row.astype(np.float64))
    assert np.abs(drawn - w / w.sum()).max() <= 2 / rows


# ---- a step of them together, captured and replayed ----------------------------------------------------------------

@pytest.mark.gpu
def test_a_decoding_step_captured_and_replayed(hip_device):
    """write the new token's keys and values, attend, draw, as one HIP graph: every replay takes the new inputs, and its
    results are those of the calls made one by one"""
    rng = np.random.default_rng(5)
    B, N, G, W, page, P, V = 6, 2, 4, 128, 16, 100, 1024
    H = N * G
    cache = CacheCase(hip_device, DType.I8, 40, N, page, W)
    prefix_table = np.arange(7, dtype=np.int32)
    tables = (7 + np.arange(B * 5).reshape(B, 5)).astype(np.int32)
    cache.put(np.arange(P), *(rng.standard_normal((2, P, N, W)).astype(np.float16)))
    args_cache = cache.upload()
    stream = kn.HipStream(hip_device)
    dev = {n: kn.DeviceBuffer(hip_device, size) for n, size in dict(k=B * N * W * 2, v=B * N * W * 2, q=B * H * W * 2, out=B * H * W * 2, slots=B * 4,
                                                                    lengths=B * 4, uniform=B * 4, tokens=B * 4, logits=B * V * 2).items()}
    dev.update(tables=upload(hip_device, tables), prefix_table=upload(hip_device, prefix_table))
    rows = kn.cache_rows(DType.F16, B, dev["k"].ptr, (N * W, W), dev["v"].ptr, (N * W, W), dev["slots"].ptr)
    att = kn.cached_attention_args(B, 1, H, args_cache, dev["q"].ptr, (H * W, H * W, W), dev["out"].ptr, (H * W, H * W, W), dev["lengths"].ptr,
                                   dev["tables"].ptr, 5, 5, prefix_tokens=P, prefix_table=dev["prefix_table"].ptr)
    draw = kn.sample_args(DType.F16, B, V, dev["out"].ptr, H * W, dev["uniform"].ptr, dev["tokens"].ptr)  # (the result as logits)
    spaces = [kn.DeviceBuffer(hip_device, max(n, 1)) for n in (kn.cached_attention_workspace_bytes(att), kn.sample_workspace_bytes(draw))]

    def step():
        kn.cache_write(hip_device, stream, args_cache, rows)
        kn.cached_attention(hip_device, stream, att, spaces[0])
        kn.sample(hip_device, stream, draw, spaces[1])

    def put(name, array):
        from ctypes import c_void_p
        kn._lib.check(kn._lib.lib.knhip_memcpy_h2d(hip_device.index, c_void_p(dev[name].ptr), array.ctypes.data, array.nbytes))

    def results():
        stream.synchronize()
        return dev["out"].to_array(np.float16, (B, 1, H, W)), dev["tokens"].to_array(np.int32, B)

    graph = None
    lengths = np.array([0, 3, 15, 16, 31, 60], np.int32)
    own_slots = [[] for _ in range(B)]
    for b in range(B):  # what the sequences hold so far
        own_slots[b] = [int(tables[b, i // page]) * page + i % page for i in range(lengths[b])]
        if own_slots[b]:
            k, v = rng.standard_normal((2, lengths[b], N, W)).astype(np.float16)
            cache.put(own_slots[b], k, v)
    for mem, buf in zip((cache.k, cache.v, cache.ks, cache.vs), cache.buffers):
        from ctypes import c_void_p
        kn._lib.check(kn._lib.lib.knhip_memcpy_h2d(hip_device.index, c_void_p(buf.ptr), mem.ctypes.data, mem.nbytes))
    for step_no in range(5):
        k, v = rng.standard_normal((2, B, N, W)).astype(np.float16)
        q = rng.standard_normal((B, H, W)).astype(np.float16)
        slots = np.array([int(tables[b, lengths[b] // page]) * page + lengths[b] % page for b in range(B)], np.int32)
        lengths = lengths + 1
        u = rng.random(B).astype(np.float32)
        for name, array in dict(k=k, v=v, q=q, slots=slots, lengths=lengths.astype(np.int32), uniform=u).items():
            put(name, np.ascontiguousarray(array))
        if graph is None:
            with Graph(stream) as graph:
                step()
        graph.launch()
        out, tokens = results()
        step()  # the same once more, call by call
        out_again, tokens_again = results()
        assert np.array_equal(out, out_again) and np.array_equal(tokens, tokens_again), step_no
        cache.put(slots, k, v)
        for b in range(B):
            own_slots[b].append(int(slots[b]))
            n = len(own_slots[b])
            kk, vv = cache.held(list(range(P)) + own_slots[b])
            at, places = np.array([P + n - 1]), np.arange(P + n)
            for h in range(H):
                e, bound = attend(q[b, h][None].astype(np.float64), kk[:, h // G], vv[:, h // G], at, places, np.ones((1, P + n), bool), W ** -0.5, 0.0, 0.0)
                move = 2.0 ** -11 * W ** -0.5 * (np.abs(q[b, h].astype(np.float64)) @ np.abs(kk[:, h // G]).T).max()
                assert (np.abs(out[b, 0, h] - e[0]) <= (bound * 2 + bound * 2.0 ** 12 * move)[0]).all(), (step_no, b, h)
        expected, _ = sample(out.reshape(B, H * W), u)
        assert np.array_equal(tokens, expected)


# ---- shapes, masks and options anywhere in their ranges --------------------------------------------------------------

def _random_scores(rng):
    return dict(cap=float(rng.choice([0.0, 0.0, 3.0, 30.0])), slopes=bool(rng.random() < 0.3), size=float(rng.choice([1.0, 1.0, 4.0])))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_cached_attention_random(seed, hip_device):
    rng = np.random.default_rng(500 + seed)
    page, batch = int(rng.choice([1, 5, 16, 16, 32, 100])), int(rng.integers(1, 12))
    longest = int(np.exp(rng.uniform(0, np.log(1800))))
    c = dict(dtype=[DType.I8, DType.F16][seed % 2], kv=int(rng.integers(1, 4)), group=int(rng.choice([1, 2, 3, 4, 8, 13])), width=16 * int(rng.integers(1, 9)),
             page=page, lengths=[int(n) for n in rng.integers(-2, longest + 1, batch)], queries=int(rng.choice([1, 1, 1, 2, 5, 33])),
             prefix=int(rng.choice([0, 0, 1, 70, 700])), window=int(rng.choice([0, 0, 1, 40, 500])), order=str(rng.choice(["dense", "tokens first"])), **_random_scores(rng))
    case = _cached_case(hip_device, c, seed)
    stream = kn.HipStream(hip_device)
    workspace = kn.DeviceBuffer(hip_device, max(kn.cached_attention_workspace_bytes(case["args"]), 1))
    kn.cached_attention(hip_device, stream, case["args"], workspace)
    stream.synchronize()
    out, bound = case["expected"]()
    _check(case["dev"][1].to_array(np.float16, case["out_mem"].shape), out, bound, case["W"], str(c))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_attention_of_prompts_random(seed, hip_device):
    rng = np.random.default_rng(700 + seed)
    queries, kv, batch = int(np.exp(rng.uniform(0, np.log(700)))), int(rng.integers(1, 4)), int(rng.integers(1, 4))
    c = dict(batch=batch, queries=queries, heads=kv * int(rng.choice([1, 2, 3, 8])), kv=kv, width=8 * int(rng.integers(1, 17)), causal=bool(rng.random() < 0.7),
             window=int(rng.choice([0, 0, 1, 33, 200])), **_random_scores(rng))
    if rng.random() < 0.5:
        c["keys"] = int(np.exp(rng.uniform(0, np.log(1500))))
    else:
        cuts = [sorted({int(x) for x in rng.integers(0, queries, 3)}) for _ in range(batch)]
        if rng.random() < 0.5:
            c["spans"] = cuts
    if c["causal"] and rng.random() < 0.4:
        c["prefix"] = [int(x) for x in rng.integers(-5, 2 * queries, batch)]
    case = _prompt_case(hip_device, c, seed)
    stream = kn.HipStream(hip_device)
    workspace = kn.DeviceBuffer(hip_device, max(kn.attention_workspace_bytes(case["args"]), 1))
    kn.attention(hip_device, stream, case["args"], workspace)
    stream.synchronize()
    out, bound = case["expected"]()
    _check(case["dev"][3].to_array(np.float16, case["out_mem"].shape), out, bound, case["W"], str(c))


# ---- large offsets, many rows, other streams, graphs ---------------------------------------------------------------

def _h2d(device, ptr, array):
    from ctypes import c_void_p
    array = np.ascontiguousarray(array)
    kn._lib.check(kn._lib.lib.knhip_memcpy_h2d(device.index, c_void_p(ptr), array.ctypes.data, array.nbytes))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,queries", [(DType.I8, 1), (DType.I8, 40), (DType.F16, 1), (DType.F16, 40)], ids=lambda x: str(getattr(x, "name", x)))
def test_cache_offsets_beyond_32_bits(dtype, queries, hip_device):
    """a cache whose pages lie 2^27 bytes apart gives the results of a dense one, bit for bit"""
    rng = np.random.default_rng(3)
    pages, N, page, W, G, n = 40, 2, 16, 64, 3, 300
    size = NP[dtype]().nbytes
    apart = (1 << 27) // size
    stream = kn.HipStream(hip_device)
    # the tokens fill the last pages, in any order; a prefix of 40 in the first ones
    prefix_table, table = np.array([0, 39, 1], np.int32), (20 + rng.permutation(19)).astype(np.int32)
    slots = np.concatenate([prefix_table[np.arange(40) // page] * page + np.arange(40) % page, table[np.arange(n) // page] * page + np.arange(n) % page])
    rows_k, rows_v = (upload(hip_device, rng.standard_normal((len(slots), N, W)).astype(np.float16)) for _ in range(2))
    dev = [upload(hip_device, a) for a in (slots.astype(np.int32), np.array([n], np.int32), table, prefix_table, rng.standard_normal((1, queries, N * G, W)).astype(np.float16))]
    outs, backs = [], []
    for page_stride in (N * page * W, apart):
        mem = [kn.DeviceBuffer(hip_device, ((pages - 1) * page_stride + N * page * W) * size) for _ in range(2)]
        scales = [kn.DeviceBuffer(hip_device, pages * N * page * 4) for _ in range(2)]
        cache = kn.kv_cache(dtype, pages, N, page, W, mem[0].ptr, mem[1].ptr, *([s.ptr for s in scales] if dtype == DType.I8 else [0, 0]),
                            strides=(page_stride, page * W, W))
        kn.cache_write(hip_device, stream, cache, kn.cache_rows(DType.F16, len(slots), rows_k.ptr, (N * W, W), rows_v.ptr, (N * W, W), dev[0].ptr))
        back = [kn.DeviceBuffer(hip_device, len(slots) * N * W * 4) for _ in range(2)]
        kn.cache_read(hip_device, stream, cache, kn.cache_rows(DType.F32, len(slots), back[0].ptr, (N * W, W), back[1].ptr, (N * W, W), dev[0].ptr))
        out = kn.DeviceBuffer(hip_device, queries * N * G * W * 2)
        args = kn.cached_attention_args(1, queries, N * G, cache, dev[4].ptr, (0, N * G * W, W), out.ptr, (0, N * G * W, W), dev[1].ptr, dev[2].ptr, len(table),
                                        len(table), prefix_tokens=40, prefix_table=dev[3].ptr)
        need = kn.cached_attention_workspace_bytes(args)
        workspace = kn.DeviceBuffer(hip_device, max(need, 1))
        kn.cached_attention(hip_device, stream, args, workspace)
        stream.synchronize()
        outs.append(out.to_array(np.uint16, queries * N * G * W))
        backs.append([b.to_array(np.uint32, len(slots) * N * W) for b in back])
    assert np.array_equal(outs[0], outs[1]) and outs[0].any()
    assert np.array_equal(backs[0][0], backs[1][0]) and np.array_equal(backs[0][1], backs[1][1])


@pytest.mark.gpu
def test_prompt_and_logit_offsets_beyond_32_bits(hip_device):
    rng = np.random.default_rng(4)
    S, N, W, apart = 100, 2, 64, 1 << 25
    stream = kn.HipStream(hip_device)
    k, v, q = (rng.standard_normal((S, N, W)).astype(np.float16) for _ in range(3))
    dense = [upload(hip_device, a) for a in (k, v, q)]
    far = [kn.DeviceBuffer(hip_device, ((S - 1) * apart + N * W) * 2) for _ in range(2)]
    for t in range(S):
        for buf, a in zip(far, (k, v)):
            _h2d(hip_device, buf.ptr + t * apart * 2, a[t])
    outs = []
    for ks, stride in ((dense, N * W), (far, apart)):
        out = kn.DeviceBuffer(hip_device, S * N * W * 2)
        args = kn.attention_args(1, S, S, N, N, W, dense[2].ptr, (0, N * W, W), ks[0].ptr, (0, stride, W), ks[1].ptr, (0, stride, W), out.ptr, (0, N * W, W), causal=True)
        workspace = kn.DeviceBuffer(hip_device, max(kn.attention_workspace_bytes(args), 1))
        kn.attention(hip_device, stream, args, workspace)
        stream.synchronize()
        outs.append(out.to_array(np.uint16, S * N * W))
    assert np.array_equal(*outs) and outs[0].any()
    # rows of logits as far apart
    rows, vocab = S, 50
    logits, uniform = rng.standard_normal((rows, vocab)).astype(np.float16), rng.random(rows).astype(np.float32)
    for t in range(rows):
        _h2d(hip_device, far[0].ptr + t * apart * 2, logits[t])
    dev_uniform, tokens = upload(hip_device, uniform), kn.DeviceBuffer(hip_device, rows * 4)
    kn.sample(hip_device, stream, kn.sample_args(DType.F16, rows, vocab, far[0].ptr, apart, dev_uniform.ptr, tokens.ptr))
    stream.synchronize()
    assert np.array_equal(tokens.to_array(np.int32, rows), sample(logits, uniform)[0])


@pytest.mark.gpu
def test_very_many_sequences_and_rows(hip_device):
    """70000 sequences of no or one token: zeros or that token's values; as many prompts of one token, rows of logits"""
    rng = np.random.default_rng(6)
    B, N, G, W = 70000, 1, 2, 16
    stream = kn.HipStream(hip_device)
    k, v, q = rng.standard_normal((B, N, W)).astype(np.float16), rng.standard_normal((B, N, W)).astype(np.float16), rng.standard_normal((B, N * G, W)).astype(np.float16)
    lengths = (np.arange(B) % 3 > 0).astype(np.int32)
    dev = [upload(hip_device, a) for a in (k, v, q, lengths, np.arange(B, dtype=np.int32))]
    out = kn.DeviceBuffer(hip_device, B * N * G * W * 2)
    cache = kn.kv_cache(DType.F16, B, N, 1, W, dev[0].ptr, dev[1].ptr)
    args = kn.cached_attention_args(B, 1, N * G, cache, dev[2].ptr, (N * G * W, W, W), out.ptr, (N * G * W, N * G * W, W), dev[3].ptr, dev[4].ptr, 1, 1)
    workspace = kn.DeviceBuffer(hip_device, max(kn.cached_attention_workspace_bytes(args), 1))
    kn.cached_attention(hip_device, stream, args, workspace)
    stream.synchronize()
    expected = np.repeat(v, G, 1) * (lengths[:, None, None] > 0)
    assert np.array_equal(out.to_array(np.float16, (B, N * G, W)), expected)
    args = kn.attention_args(B, 1, 1, N * G, N, W, dev[2].ptr, (N * G * W, W, W), dev[0].ptr, (N * W, W, W), dev[1].ptr, (N * W, W, W), out.ptr,
                             (N * G * W, N * G * W, W), causal=True)
    workspace = kn.DeviceBuffer(hip_device, max(kn.attention_workspace_bytes(args), 1))
    kn.attention(hip_device, stream, args, workspace)
    stream.synchronize()
    assert np.array_equal(out.to_array(np.float16, (B, N * G, W)), np.repeat(v, G, 1))
    uniform = rng.random(B).astype(np.float32)
    dev_uniform, tokens = upload(hip_device, uniform), kn.DeviceBuffer(hip_device, B * 4)
    kn.sample(hip_device, stream, kn.sample_args(DType.F16, B, W, dev[0].ptr, W, dev_uniform.ptr, tokens.ptr))
    stream.synchronize()
    assert np.array_equal(tokens.to_array(np.int32, B), sample(k[:, 0], uniform)[0])


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(hip_device):
    """prompts in parts, a shared prefix and draws on two streams, each with its own workspace: the results of calls made alone"""
    streams = [kn.HipStream(hip_device) for _ in range(2)]
    prompts = [_prompt_case(hip_device, dict(queries=90, keys=1500, heads=2, kv=1, width=64, causal=True), seed=s) for s in range(2)]
    cached = [_cached_case(hip_device, dict(dtype=DType.I8, kv=2, group=4, width=128, page=16, lengths=[700 + i for i in range(9)], prefix=900), seed=s) for s in range(2)]
    rng = np.random.default_rng(8)
    draws = [_sample_call(hip_device, rng.standard_normal((5, 40000)).astype(np.float32), DType.F32, rng.random(5), top_p=np.full(5, 0.9)) for _ in range(2)]
    spaces = [[kn.DeviceBuffer(hip_device, max(n, 1)) for n in (kn.attention_workspace_bytes(prompts[i]["args"]), kn.cached_attention_workspace_bytes(cached[i]["args"]))]
              for i in range(2)]

    def call(i):
        kn.attention(hip_device, streams[i], prompts[i]["args"], spaces[i][0])
        kn.cached_attention(hip_device, streams[i], cached[i]["args"], spaces[i][1])
        kn.sample(hip_device, streams[i], draws[i][0], draws[i][2])

    def results(i):
        streams[i].synchronize()
        return (prompts[i]["dev"][3].to_array(np.uint16, prompts[i]["out_mem"].shape), cached[i]["dev"][1].to_array(np.uint16, cached[i]["out_mem"].shape),
                draws[i][1]["tokens"].to_array(np.int32, 5))

    alone = []
    for i in range(2):
        call(i)
        alone.append(results(i))
    for _ in range(20):
        for i in range(2):
            call(i)
    for i in range(2):
        for a, b in zip(alone[i], results(i)):
            assert np.array_equal(a, b)


@pytest.mark.gpu
def test_prompts_and_reads_captured_and_replayed(hip_device):
    """a prompt in parts over keys that are read out of a cache, and a draw with every filter, as one graph"""
    rng = np.random.default_rng(9)
    S, K, N, W, rows, vocab = 70, 1100, 1, 64, 3, 33000
    stream = kn.HipStream(hip_device)
    cache = CacheCase(hip_device, DType.I8, 70, N, 16, W)
    cache.put(np.arange(70 * 16), *rng.standard_normal((2, 70 * 16, N, W)).astype(np.float16))
    args_cache = cache.upload()
    dev = dict(k=kn.DeviceBuffer(hip_device, K * N * W * 2), v=kn.DeviceBuffer(hip_device, K * N * W * 2), q=kn.DeviceBuffer(hip_device, S * N * W * 2),
               out=kn.DeviceBuffer(hip_device, S * N * W * 2), slots=kn.DeviceBuffer(hip_device, K * 4))
    read = kn.cache_rows(DType.F16, K, dev["k"].ptr, (N * W, W), dev["v"].ptr, (N * W, W), dev["slots"].ptr)
    prompt = kn.attention_args(1, S, K, N, N, W, dev["q"].ptr, (0, N * W, W), dev["k"].ptr, (0, N * W, W), dev["v"].ptr, (0, N * W, W), dev["out"].ptr,
                               (0, N * W, W), causal=True)
    logits = rng.standard_normal((rows, vocab)).astype(np.float32) * 3
    draw, parts, _ = _sample_call(hip_device, logits, DType.F32, rng.random(rows), temperature=np.full(rows, 0.8), top_k=np.array([900, 0, 40]),
                                  top_p=np.full(rows, 0.9), min_p=np.full(rows, 0.001))
    need = kn.attention_workspace_bytes(prompt)
    assert need > 0
    workspace = kn.DeviceBuffer(hip_device, need)

    def step():
        kn.cache_read(hip_device, stream, args_cache, read)
        kn.attention(hip_device, stream, prompt, workspace)
        kn.sample(hip_device, stream, draw)

    def results():
        stream.synchronize()
        return dev["out"].to_array(np.uint16, S * N * W), parts["tokens"].to_array(np.int32, rows)

    graph, seen = None, []
    for _ in range(4):
        _h2d(hip_device, dev["slots"].ptr, rng.permutation(70 * 16)[:K].astype(np.int32))
        _h2d(hip_device, dev["q"].ptr, rng.standard_normal((S, N, W)).astype(np.float16))
        _h2d(hip_device, parts["uniform"].ptr, rng.random(rows).astype(np.float32))
        if graph is None:
            with Graph(stream) as graph:
                step()
        graph.launch()
        replayed = results()
        step()
        for a, b in zip(replayed, results()):
            assert np.array_equal(a, b)
        seen.append(replayed[0])
    assert not any(np.array_equal(seen[0], other) for other in seen[1:])


# ---- what is refused (on the host, before anything is launched) ----------------------------------------------------

def _valid():
    cache = kn.kv_cache(DType.I8, 4, 2, 16, 64, 256, 512, 256, 512)
    rows = kn.cache_rows(DType.F16, 3, 256, (128, 64), 512, (128, 64), 256)
    cached = kn.cached_attention_args(2, 1, 4, cache, 256, (256, 256, 64), 512, (256, 256, 64), 256, 256, 4, 4, prefix_tokens=5, prefix_table=256)
    prompt = kn.attention_args(2, 8, 8, 4, 2, 64, 256, (2048, 256, 64), 256, (1024, 128, 64), 256, (1024, 128, 64), 512, (2048, 256, 64))
    draw = kn.sample_args(DType.F32, 2, 100, 256, 100, 256, 256)
    return dict(cache=cache, rows=rows, cached=cached, prompt=prompt, draw=draw)


REFUSED = [
    # what is asked, the field, its value, and the message
    ("cache", "cache.dtype", int(DType.F32), "a cache holds f16 or i8"),
    ("cache", "cache.width", 40, "multiple of 16"),
    ("cache", "cache.width", 272, "multiple of 16"),
    ("cache", "cache.page_tokens", 0, "tokens"),
    ("cache", "cache.pages", -1, "pages"),
    ("cache", "cache.pages", 1 << 28, "below 2\\^31"),
    ("cache", "cache.k", 0, "k is null"),
    ("cache", "cache.v", 8, "16 byte aligned"),
    ("cache", "cache.v_scales", 0, "v_scales is null"),
    ("cache", "cache.k_scales", 2, "k_scales must be 4 byte aligned"),
    ("cache", "cache.token_stride", 32, "less than a row"),
    ("cache", "cache.token_stride", 72, "multiple of 16 bytes"),
    ("cache", "cache.page_stride", -2048, "less than a row"),
    ("cache", "rows.dtype", int(DType.I8), "rows are f16 or f32"),
    ("cache", "rows.tokens", -1, "negative size"),
    ("cache", "rows.tokens", 1 << 26, "below 2\\^27"),
    ("cache", "rows.k", 0, "rows' k is null"),
    ("cache", "rows.v", 3, "2 byte aligned"),
    ("cache", "rows.slots", 0, "slots is null"),
    ("cache", "cache.head_stride", 512, "may not overlap"),
    ("cache", "cache.page_stride", 1024, "may not overlap"),
    ("read", "rows.k_token_stride", 0, "may not overlap"),
    ("read", "rows.k_token_stride", 64, "may not overlap"),
    ("read", "rows.v_token_stride", -127, "may not overlap"),
    ("read", "rows.v_head_stride", 8, "may not overlap"),
    ("cached", "cache.width", 144, "at most 128"),
    ("cached", "cache.heads", 3, "evenly"),
    ("cached", "heads", 5, "evenly"),
    ("cached", "batch", -1, "negative size"),
    ("cached", "queries", 1 << 24, "below 2\\^24"),
    ("cached", "batch", 1 << 21, "below 2\\^22"),
    ("prompt", "batch", 1 << 21, "below 2\\^22"),
    ("prompt", "cap", 1e-44, "too small"),
    ("cached", "cap", 3.2e38, "cap must be finite"),
    ("cached", "table_pages", 1 << 27, "below 2\\^30"),
    ("cached", "prefix_tokens", 1 << 30, "below 2\\^30"),
    ("cached", "prefix_table", 0, "prefix_table is null"),
    ("cached", "lengths", 0, "lengths is null"),
    ("cached", "tables", 2, "tables must be 4 byte aligned"),
    ("cached", "q", 1, "q must be 2 byte aligned"),
    ("cached", "out", 0, "out is null"),
    ("cached", "out_head_stride", 0, "out may not overlap"),
    ("cached", "out_batch_stride", 128, "out may not overlap"),
    ("cached", "scale", math.inf, "scale must be finite"),
    ("cached", "cap", -1.0, "cap must be finite"),
    ("cached", "cap", math.nan, "cap must be finite"),
    ("cached", "window", -1, "window"),
    ("cached", "slopes", 6, "slopes must be 4 byte aligned"),
    ("prompt", "width", 12, "multiple of 8"),
    ("prompt", "width", 136, "multiple of 8"),
    ("prompt", "kv_heads", 3, "evenly"),
    ("prompt", "kv_heads", 0, "evenly"),
    ("prompt", "keys", -1, "negative size"),
    ("prompt", "keys", 1 << 30, "below 2\\^30"),
    ("prompt", "queries", 1 << 26, "below 2\\^27"),
    ("prompt", "k", 0, "k is null"),
    ("prompt", "v", 1, "v must be 2 byte aligned"),
    ("prompt", "out_token_stride", 63, "out may not overlap"),
    ("prompt", "scale", math.nan, "scale must be finite"),
    ("prompt", "spans", 2, "spans must be 4 byte aligned"),
    ("prompt", "prefix", 1, "prefix must be 4 byte aligned"),
    ("draw", "dtype", int(DType.I32), "logits are f16 or f32"),
    ("draw", "rows", -1, "negative size"),
    ("draw", "rows", (1 << 20) + 1, "at most 2\\^20 rows"),
    ("draw", "vocab", (1 << 20) + 1, "at most 1048576 logits"),
    ("draw", "logits", 0, "logits is null"),
    ("draw", "uniform", 0, "uniform is null"),
    ("draw", "tokens", 2, "tokens must be 4 byte aligned"),
    ("draw", "top_k", 2, "4 byte aligned"),
]


def _ask(which, v):
    if which == "cache":
        kn.cache_write(0, 0, v["cache"], v["rows"])
    elif which == "read":
        kn.cache_read(0, 0, v["cache"], v["rows"])
    elif which == "cached":
        kn.cached_attention_workspace_bytes(v["cached"])
    elif which == "prompt":
        kn.attention_workspace_bytes(v["prompt"])
    else:
        kn.sample_workspace_bytes(v["draw"])


@pytest.mark.parametrize("which,field,value,message", REFUSED, ids=lambda x: str(x)[:24])
def test_refusals(which, field, value, message):
    """(addresses here are made up: a call that is not refused would fail for want of a device instead)"""
    v = _valid()
    owner, _, name = field.rpartition(".")
    target = v["cached"].cache if which == "cached" and owner == "cache" else v[owner] if owner else v[which]
    setattr(target, name, value)
    with pytest.raises(kn.KnError, match=message):
        _ask(which, v)


def test_valid_arguments_are_planned_without_a_device():
    v = _valid()
    assert kn.cached_attention_workspace_bytes(v["cached"]) >= 0
    assert kn.attention_workspace_bytes(v["prompt"]) >= 0
    assert kn.sample_workspace_bytes(v["draw"]) >= 0
    # nothing to do: no addresses are asked for
    kn.cache_write(0, 0, kn.kv_cache(DType.I8, 0, 0, 16, 64, 0, 0), kn.cache_rows(DType.F16, 0, 0, (0, 0), 0, (0, 0), 0))
    empty = kn.attention_args(0, 8, 8, 4, 2, 64, 0, (0, 0, 0), 0, (0, 0, 0), 0, (0, 0, 0), 0, (0, 0, 0))
    assert kn.attention_workspace_bytes(empty) == 0
    kn.attention(0, 0, empty)
    kn.sample(0, 0, kn.sample_args(DType.F32, 0, 10, 0, 10, 0, 0))


def test_builders_refuse_wrong_strides():
    with pytest.raises(kn.KnError, match="three strides"):
        kn.attention_args(1, 1, 1, 1, 1, 64, 0, (0, 0), 0, (0, 0, 0), 0, (0, 0, 0), 0, (0, 0, 0))
    with pytest.raises(kn.KnError, match="two strides"):
        kn.cache_rows(DType.F16, 1, 0, (0,), 0, (0, 0), 0)


@pytest.mark.gpu
def test_short_or_misaligned_workspaces_are_refused(hip_device):
    stream = kn.HipStream(hip_device)
    c = _cached_case(hip_device, CACHED_CASES["prefix_many_rows"])
    p = _prompt_case(hip_device, PROMPT_CASES["last_queries"])
    s, _, _ = _sample_call(hip_device, np.zeros((2, 100000), np.float32), DType.F32, np.zeros(2))
    for call, need, args in ((kn.cached_attention, kn.cached_attention_workspace_bytes, c["args"]),
                             (kn.attention, kn.attention_workspace_bytes, p["args"]), (kn.sample, kn.sample_workspace_bytes, s)):
        n = need(args)
        if n == 0:
            call(hip_device, stream, args)
            continue
        with pytest.raises(kn.KnError, match="bytes of workspace"):
            call(hip_device, stream, args)
        with pytest.raises(kn.KnError, match="bytes of workspace"):
            call(hip_device, stream, args, kn.DeviceBuffer(hip_device, n - 1))
        whole = kn.DeviceBuffer(hip_device, n + 256)

        class Shifted:
            ptr, nbytes = whole.ptr + 4, n + 4
        with pytest.raises(kn.KnError, match="256 byte aligned"):
            call(hip_device, stream, args, Shifted)
    stream.synchronize()


def test_struct_fields_are_those_of_the_header():
    from kyanite_amd._lib import AttentionArgsT, CachedAttentionArgsT, CacheRowsT, KvCacheT, SampleArgsT
    from test_rust_shim import _c_struct_fields, _rust_struct_fields
    for name, struct in (("knhip_kv_cache", KvCacheT), ("knhip_cache_rows", CacheRowsT), ("knhip_cached_attention_args", CachedAttentionArgsT),
                         ("knhip_attention_args", AttentionArgsT), ("knhip_sample_args", SampleArgsT)):
        assert [f for f, _ in struct._fields_] == _c_struct_fields(name) == _rust_struct_fields(name), name
