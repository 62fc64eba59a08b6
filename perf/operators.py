"""The operators that serve a decoder token by token, as cases to be measured: writing keys and values into a quantised
cache and reading them back, attention over that cache for a batch that shares a long prefix, attention of whole prompts
with capped scores, distance bias, document and prefix masks, and sampling from logits with given random numbers.

`own` selects what `run` computes: the plain form in elementary torch operations, or the calls of `kyanite_amd`. Sizes of
the decoder (32 heads of width 128, 4096 wide, 512 tokens) are those of the decoder layer this repository benchmarks; the
others are generic."""
import math
import random

import numpy as np
import torch

own = False

PAGE = 16      # tokens per page of the cache
PAGE_LONG = 48  # a page size that is no power of two


# ---- the cases -----------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new token of 16 sequences goes into the cache: the write of every decoding step, where latency counts
        dict(name="cache_step", op="cache", tokens=16, kv_heads=8, width=128, cache="i8", rows="f16", page=PAGE),
        # a prompt of odd length, kept in f16, from f32 activations
        dict(name="cache_prompt_f16", op="cache", tokens=2049, kv_heads=8, width=64, cache="f16", rows="f32", page=PAGE_LONG),
        # the prompts of a whole batch
        dict(name="cache_prompts", op="cache", tokens=32768, kv_heads=8, width=128, cache="i8", rows="f16", page=PAGE),
        # one token of one sequence: the smallest decoding step
        dict(name="decode_one", op="cached", batch=1, queries=1, heads=32, kv_heads=8, width=128, longest=517, shortest=517, prefix=0,
             cache="i8", page=PAGE, cap=0.0, slopes=False, window=0),
        # a batch of ragged sequences with nothing in common, f16 cache, capped scores and a window
        dict(name="decode_ragged", op="cached", batch=48, queries=1, heads=32, kv_heads=8, width=128, longest=6000, shortest=1, prefix=0,
             cache="f16", page=PAGE, cap=30.0, slopes=False, window=4096),
        # a batch that answers questions about one long document: 16384 tokens in common, up to 700 each of their own
        dict(name="decode_shared", op="cached", batch=64, queries=1, heads=32, kv_heads=8, width=128, longest=700, shortest=5, prefix=16384,
             cache="i8", page=PAGE, cap=0.0, slopes=False, window=0),
        # a short prompt seen from both sides (prefix mask), narrow heads, distance bias
        dict(name="prompt_short", op="attention", batch=2, tokens=77, heads=8, kv_heads=8, width=64, documents=1, prefix=40, cap=0.0,
             slopes=True, window=0),
        # packed documents in one row of 4096 tokens
        dict(name="prompt_documents", op="attention", batch=1, tokens=4096, heads=32, kv_heads=8, width=128, documents=9, prefix=0, cap=0.0,
             slopes=False, window=0),
        # one long prompt with capped scores: the largest
        dict(name="prompt_capped", op="attention", batch=1, tokens=8192, heads=32, kv_heads=8, width=128, documents=1, prefix=0, cap=50.0,
             slopes=False, window=0),
        # the next token of one sequence
        dict(name="sample_one", op="sample", rows=1, vocab=32000, dtype="f16", temperature=0.8, top_k=40, top_p=0.95, min_p=0.0),
        # a serving batch with every filter
        dict(name="sample_batch", op="sample", rows=64, vocab=128001, dtype="f32", temperature=0.7, top_k=1000, top_p=0.9, min_p=0.02),
        # many rows, only the nucleus
        dict(name="sample_nucleus", op="sample", rows=256, vocab=50001, dtype="f16", temperature=1.0, top_k=0, top_p=0.92, min_p=0.0),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("cache", "cached", "attention", "sample"))
    if op == "cache":
        return dict(op=op, tokens=_spread(rng, 1, 32768), kv_heads=rng.choice((1, 2, 5, 8)), width=rng.choice((64, 80, 128)),
                    cache=rng.choice(("i8", "f16")), rows=rng.choice(("f16", "f32")), page=rng.choice((PAGE, PAGE_LONG)))
    if op == "cached":
        kv_heads = rng.choice((1, 4, 8))
        return dict(op=op, batch=_spread(rng, 1, 64), queries=rng.choice((1, 1, 1, 2, 5)), heads=kv_heads * rng.choice((1, 3, 4, 8)),
                    kv_heads=kv_heads, width=rng.choice((64, 96, 128)), longest=_spread(rng, 8, 3000), shortest=rng.choice((0, 1, 6)),
                    prefix=rng.choice((0, _spread(rng, 1, 16384))), cache=rng.choice(("i8", "f16")), page=rng.choice((PAGE, PAGE_LONG)),
                    cap=rng.choice((0.0, 0.0, 30.0)), slopes=rng.choice((False, True)), window=rng.choice((0, 0, _spread(rng, 16, 8192))))
    if op == "attention":
        kv_heads = rng.choice((1, 4, 8))
        tokens = _spread(rng, 1, 5000)
        return dict(op=op, batch=rng.choice((1, 2, 3)) if tokens < 2000 else 1, tokens=tokens, heads=kv_heads * rng.choice((1, 2, 4)),
                    kv_heads=kv_heads, width=rng.choice((64, 72, 128)), documents=rng.choice((1, 1, 2, 7)),
                    prefix=rng.choice((0, 0, tokens // 3)), cap=rng.choice((0.0, 0.0, 20.0)), slopes=rng.choice((False, True)),
                    window=rng.choice((0, 0, _spread(rng, 8, 4096))))
    return dict(op=op, rows=_spread(rng, 1, 128), vocab=_spread(rng, 1000, 128001), dtype=rng.choice(("f16", "f32")),
                temperature=rng.choice((0.0, 0.6, 1.0, 1.3)), top_k=rng.choice((0, 1, 50, 700)), top_p=rng.choice((1.0, 0.95, 0.6)),
                min_p=rng.choice((0.0, 0.0, 0.05)))


# ---- what a case is made of (the sizes go by the case alone, the values by the seed) ---------------------------------

def _lengths(c):
    """own tokens of every sequence, the new ones among them"""
    r = random.Random("%d %d %d" % (c["batch"], c["longest"], c["shortest"]))
    got = [r.randint(min(c["shortest"], c["longest"]), c["longest"]) for _ in range(c["batch"])]
    got[r.randrange(len(got))] = c["longest"]
    return got


def _document_bounds(c):
    """cuts of a row of tokens into documents"""
    r = random.Random("%d %d" % (c["tokens"], c["documents"]))
    return [0] + sorted(r.randint(0, c["tokens"]) for _ in range(c["documents"] - 1)) + [c["tokens"]]


def _spans(c):
    """[tokens, 2]: first and one past the last token of the document of each token"""
    b = _document_bounds(c)
    first = np.zeros((c["tokens"], 2), np.int32)
    for lo, hi in zip(b, b[1:]):
        first[lo:hi] = (lo, hi)
    return first


def _dtype(name):
    return {"f16": torch.float16, "f32": torch.float32, "i8": torch.int8}[name]


def _quantised(x):
    """symmetric 8 bit rows: the values and one scale per row"""
    scale = x.float().abs().amax(-1) / 127.0
    return torch.where(scale[..., None] > 0, x.float() / scale[..., None], torch.zeros_like(x, dtype=torch.float32)).round().to(torch.int8), scale


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32)


def prepare(case, seed):
    c = dict(case)
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    s = {"case": c}
    if c["op"] == "cache":
        # rows of keys have a few large channels, as projected keys do; the slots are scattered over a cache half as large again
        channel = torch.exp(normal(c["kv_heads"], c["width"]) * 0.7)
        s["k"] = (normal(c["tokens"], c["kv_heads"], c["width"]) * channel).to(_dtype(c["rows"]))
        s["v"] = normal(c["tokens"], c["kv_heads"], c["width"]).to(_dtype(c["rows"]))
        pages = -(-c["tokens"] * 3 // (2 * c["page"])) + 1
        order = torch.randperm(pages, generator=g, device=dev)
        at = torch.arange(c["tokens"], device=dev)
        s["slots"] = (order[at // c["page"]] * c["page"] + at % c["page"]).to(torch.int32)
        shape = (pages, c["kv_heads"], c["page"], c["width"])
        s["cache_k"], s["cache_v"] = (torch.zeros(shape, dtype=_dtype(c["cache"]), device=dev) for _ in range(2))
        s["scale_k"], s["scale_v"] = (torch.zeros(shape[:3], dtype=torch.float32, device=dev) for _ in range(2))
    elif c["op"] == "cached":
        lengths = _lengths(c)
        table_pages = max(1, -(-max(lengths) // c["page"]))
        prefix_pages = -(-c["prefix"] // c["page"])
        used = [-(-n // c["page"]) for n in lengths]
        pages = prefix_pages + sum(used) + 3
        order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        s["prefix_table"] = order[:prefix_pages].contiguous()
        s["tables"] = torch.zeros((c["batch"], table_pages), dtype=torch.int32, device=dev)
        at = prefix_pages
        for b, n in enumerate(used):
            s["tables"][b, :n] = order[at:at + n]
            at += n
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        shape = (pages, c["kv_heads"], c["page"], c["width"])
        k, v = normal(*shape), normal(*shape)
        if c["cache"] == "i8":
            (s["cache_k"], s["scale_k"]), (s["cache_v"], s["scale_v"]) = _quantised(k), _quantised(v)
        else:
            s["cache_k"], s["cache_v"] = k.half(), v.half()
            s["scale_k"] = s["scale_v"] = None
        s["q"] = normal(c["batch"], c["queries"], c["heads"], c["width"]).half()
        s["slopes"] = _slopes(c["heads"]).to(dev) if c["slopes"] else None
    elif c["op"] == "attention":
        s["q"] = normal(c["batch"], c["tokens"], c["heads"], c["width"]).half()
        s["k"], s["v"] = (normal(c["batch"], c["tokens"], c["kv_heads"], c["width"]).half() for _ in range(2))
        s["slopes"] = _slopes(c["heads"]).to(dev) if c["slopes"] else None
        s["spans"] = torch.from_numpy(_spans(c)).to(dev).expand(c["batch"], -1, -1).contiguous() if c["documents"] > 1 else None
        s["prefix"] = torch.full((c["batch"],), c["prefix"], dtype=torch.int32, device=dev) if c["prefix"] else None
    else:
        s["logits"] = (normal(c["rows"], c["vocab"]) * 2.5).to(_dtype(c["dtype"]))
        s["uniform"] = torch.rand(c["rows"], generator=g, device=dev)

        def each(v, dtype):
            return torch.full((c["rows"],), v, dtype=dtype, device=dev)

        s["temperature"] = each(c["temperature"], torch.float32)
        s["top_k"] = each(c["top_k"], torch.int32) if c["top_k"] else None
        s["top_p"] = each(c["top_p"], torch.float32) if c["top_p"] < 1 else None
        s["min_p"] = each(c["min_p"], torch.float32) if c["min_p"] else None
    if own:
        s["plan"] = _plan(s)  # the argument blocks, results and workspaces that a serving loop keeps from step to step
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"cache": _plain_cache, "cached": _plain_cached, "attention": _plain_attention, "sample": _plain_sample}[s["case"]["op"]](s)


def _plain_cache(s):
    c = s["case"]
    slot = s["slots"].long()
    page, at = slot // c["page"], slot % c["page"]
    out = {}
    for name in ("k", "v"):
        x = s[name].float()
        if c["cache"] == "i8":
            scale = x.abs().amax(-1) / 127.0
            q = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x)).round()
            s["cache_" + name][page, :, at] = q.to(torch.int8)
            s["scale_" + name][page, :, at] = scale
            back = s["cache_" + name][page, :, at].float() * s["scale_" + name][page, :, at][..., None]
            out["scale_" + name] = s["scale_" + name]
        else:
            s["cache_" + name][page, :, at] = x.half()
            back = s["cache_" + name][page, :, at].float()
        out[name] = back.half()
    return out


def _plain_weights(score, visible):
    """softmax over the last axis among what is visible; rows without anything visible get zeros"""
    score = torch.where(visible, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _plain_cached(s):
    c = s["case"]
    B, T, H, N, W, P = c["batch"], c["queries"], c["heads"], c["kv_heads"], c["width"], c["prefix"]
    G = H // N

    def values(name, table):  # [..., pages] -> [..., heads, tokens, width]
        x = s["cache_" + name][table.long()].float()
        if c["cache"] == "i8":
            x = x * s["scale_" + name][table.long()][..., None]
        x = x.transpose(-4, -3)
        return x.reshape(x.shape[:-3] + (x.shape[-3] * x.shape[-2], W))

    q = s["q"].float().reshape(B, T, N, G, W).permute(0, 2, 1, 3, 4).reshape(B, N, T * G, W)
    k, v = values("k", s["tables"]), values("v", s["tables"])
    L = k.shape[2]
    score = torch.matmul(q, k.transpose(-1, -2))
    key = torch.arange(P, P + L, device=q.device)
    if P:
        pk, pv = values("k", s["prefix_table"])[:, :P], values("v", s["prefix_table"])[:, :P]
        stacked = q.permute(1, 0, 2, 3).reshape(N, B * T * G, W)
        first = torch.matmul(stacked, pk.transpose(-1, -2)).reshape(N, B, T * G, P).permute(1, 0, 2, 3)
        score = torch.cat([first, score], -1)
        key = torch.arange(P + L, device=q.device)
    score = score * W ** -0.5
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    own_at = s["lengths"].long()[:, None] - T + torch.arange(T, device=q.device)  # [B, T], below 0: a row of padding
    at = (own_at + P).repeat_interleave(G, 1)[:, None, :, None]                   # [B, 1, T G, 1]
    if c["slopes"]:
        slope = s["slopes"].reshape(N, 1, G).expand(N, T, G).reshape(1, N, T * G, 1)
        score = score - slope * (at - key).abs().float()
    visible = (key <= at) & (at >= P)
    if c["window"]:
        visible = visible & (key > at - c["window"])
    w = _plain_weights(score, visible)
    out = torch.matmul(w[..., -L:], v)
    if P:
        wp = w[..., :P].permute(1, 0, 2, 3).reshape(N, B * T * G, P)
        out = out + torch.matmul(wp, pv).reshape(N, B, T * G, W).permute(1, 0, 2, 3)
    return out.reshape(B, N, T, G, W).permute(0, 2, 1, 3, 4).reshape(B, T, H, W).half()


def _plain_attention(s):
    c = s["case"]
    G, S = c["heads"] // c["kv_heads"], c["tokens"]
    q = s["q"].float().transpose(1, 2)
    k, v = (s[n].float().transpose(1, 2).repeat_interleave(G, 1) for n in ("k", "v"))
    score = torch.matmul(q, k.transpose(-1, -2)) * c["width"] ** -0.5
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    at = torch.arange(S, device=q.device)
    away = at[:, None] - at
    if c["slopes"]:
        score = score - s["slopes"][:, None, None] * away.abs().float()
    visible = (away >= 0)[None, None]
    if s["prefix"] is not None:
        visible = visible | (at < s["prefix"][:, None])[:, None, None]
    if c["window"]:
        visible = visible & (away < c["window"])
    if s["spans"] is not None:
        visible = visible & ((at >= s["spans"][..., :1]) & (at < s["spans"][..., 1:]))[:, None]
    return torch.matmul(_plain_weights(score, visible), v).transpose(1, 2).half()


def _plain_sample(s):
    c = s["case"]
    # 64 bits: the draw falls next to the border of two tokens now and then
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0  # the most probable token, the first of several
    first = (x == top) & (torch.cumsum(x == top, -1) == 1)
    w = torch.where(greedy, first.double(), torch.exp((x - top) / torch.where(greedy, torch.ones_like(t), t)))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    sorted_w = w.gather(-1, order)
    keep = torch.ones_like(sorted_w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = (torch.arange(c["vocab"], device=x.device) < k) | (k <= 0)
    if s["top_p"] is not None:
        mass = torch.where(keep, sorted_w, torch.zeros_like(sorted_w))
        before = torch.cumsum(mass, -1) - mass
        keep = keep & (before < s["top_p"].double()[:, None] * mass.sum(-1, keepdim=True))
    if s["min_p"] is not None:
        keep = keep & (sorted_w >= s["min_p"].double()[:, None])
    keep = keep | (torch.arange(c["vocab"], device=x.device) == 0)  # the most probable token stays whatever the filters say
    kept = torch.zeros_like(w).scatter(-1, order, torch.where(keep, sorted_w, torch.zeros_like(sorted_w)))
    u = torch.where(greedy, torch.zeros_like(t), s["uniform"].double()[:, None])
    sums = torch.cumsum(kept, -1)
    passed = sums > u * sums[:, -1:]
    token = passed.to(torch.uint8).argmax(-1, keepdim=True)
    return {"tokens": token[:, 0].int(), "probabilities": (kept.gather(-1, token)[:, 0] / sums[:, -1]).float()}


# ---- the framework's calls -----------------------------------------------------------------------------------------

def _plan(s):
    import kyanite_amd as kn

    c, p = s["case"], {}
    dt = {torch.float16: kn.DType.F16, torch.float32: kn.DType.F32, torch.int8: kn.DType.I8}

    def at(t):
        return 0 if t is None else t.data_ptr()

    def cache():
        return kn.kv_cache(dt[s["cache_k"].dtype], *s["cache_k"].shape, at(s["cache_k"]), at(s["cache_v"]), at(s["scale_k"]), at(s["scale_v"]))

    if c["op"] == "cache":
        back = {n: torch.empty_like(s[n], dtype=torch.float16) for n in ("k", "v")}
        strides = (s["k"].stride(0), s["k"].stride(1))
        p["cache"] = cache() if c["cache"] == "i8" else kn.kv_cache(kn.DType.F16, *s["cache_k"].shape, at(s["cache_k"]), at(s["cache_v"]))
        p["rows"] = kn.cache_rows(dt[s["k"].dtype], c["tokens"], at(s["k"]), strides, at(s["v"]), strides, at(s["slots"]))
        p["back"] = kn.cache_rows(kn.DType.F16, c["tokens"], at(back["k"]), strides, at(back["v"]), strides, at(s["slots"]))
        p["out"] = dict(back, scale_k=s["scale_k"], scale_v=s["scale_v"]) if c["cache"] == "i8" else back
        return p
    if c["op"] == "cached":
        p["out"] = torch.empty_like(s["q"])
        strides = s["q"].stride()[:3]
        p["args"] = kn.cached_attention_args(c["batch"], c["queries"], c["heads"], cache(), at(s["q"]), strides, at(p["out"]), strides, at(s["lengths"]),
                                             at(s["tables"]), s["tables"].stride(0), s["tables"].shape[1], prefix_tokens=c["prefix"],
                                             prefix_table=at(s["prefix_table"]), cap=c["cap"], slopes=at(s["slopes"]), window=c["window"])
        need = kn.cached_attention_workspace_bytes(p["args"])
    elif c["op"] == "attention":
        p["out"] = torch.empty_like(s["q"])
        p["args"] = kn.attention_args(c["batch"], c["tokens"], c["tokens"], c["heads"], c["kv_heads"], c["width"], at(s["q"]), s["q"].stride()[:3],
                                      at(s["k"]), s["k"].stride()[:3], at(s["v"]), s["v"].stride()[:3], at(p["out"]), s["q"].stride()[:3],
                                      causal=True, cap=c["cap"], slopes=at(s["slopes"]), window=c["window"], spans=at(s["spans"]),
                                      prefix=at(s["prefix"]))
        need = kn.attention_workspace_bytes(p["args"])
    else:
        tokens = torch.empty(c["rows"], dtype=torch.int32, device=s["logits"].device)
        p["out"] = {"tokens": tokens, "probabilities": torch.empty(c["rows"], dtype=torch.float32, device=tokens.device)}
        p["args"] = kn.sample_args(dt[s["logits"].dtype], c["rows"], c["vocab"], at(s["logits"]), s["logits"].stride(0), at(s["uniform"]),
                                   at(tokens), temperature=at(s["temperature"]), top_k=at(s["top_k"]), top_p=at(s["top_p"]),
                                   min_p=at(s["min_p"]), probabilities=at(p["out"]["probabilities"]))
        need = kn.sample_workspace_bytes(p["args"])
    p["workspace"] = kn.DeviceBuffer(0, need) if need else None
    return p


def _run_own(s):
    import kyanite_amd as kn

    p, stream = s["plan"], torch.cuda.current_stream().cuda_stream
    op = s["case"]["op"]
    if op == "cache":
        kn.cache_write(0, stream, p["cache"], p["rows"])
        kn.cache_read(0, stream, p["cache"], p["back"])
    elif op == "cached":
        kn.cached_attention(0, stream, p["args"], p["workspace"])
    elif op == "attention":
        kn.attention(0, stream, p["args"], p["workspace"])
    else:
        kn.sample(0, stream, p["args"], p["workspace"])
    return p["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def _visible_pairs(c):
    """how many (query, key) pairs of one row of tokens are visible, and how many tokens are"""
    i = np.arange(c["tokens"], dtype=np.int64)
    lo, hi = np.zeros_like(i), i + 1
    if c["prefix"]:
        hi = np.maximum(hi, c["prefix"])
    if c["window"]:
        lo = np.maximum(lo, i - c["window"] + 1)
    span = _spans(c).astype(np.int64)
    lo, hi = np.maximum(lo, span[:, 0]), np.minimum(hi, span[:, 1])
    return int(np.maximum(hi - lo, 0).sum())


def work(c):
    size = {"f16": 2, "f32": 4, "i8": 1}
    if c["op"] == "cache":
        n = 2 * c["tokens"] * c["kv_heads"]
        held = size[c["cache"]] * c["width"] + (4 if c["cache"] == "i8" else 0)
        return {"bytes": n * (size[c["rows"]] * c["width"] + 2 * held + 2 * c["width"]) + 8 * c["tokens"], "flops": 0}
    if c["op"] == "cached":
        held = size[c["cache"]] * c["width"] + (4 if c["cache"] == "i8" else 0)
        pairs, read, in_prefix = 0, 0, 0
        for n in _lengths(c):
            low = n
            for t in range(c["queries"]):
                at = n - c["queries"] + t
                if at < 0:
                    continue
                first = max(0, c["prefix"] + at + 1 - c["window"]) if c["window"] else 0
                pairs += c["prefix"] + at + 1 - first
                low = min(low, max(0, first - c["prefix"]))
                in_prefix = max(in_prefix, c["prefix"] - first)
            read += n - low
        bytes_ = 2 * c["kv_heads"] * held * (read + in_prefix) + 4 * c["batch"] * c["queries"] * c["heads"] * c["width"]
        return {"bytes": bytes_, "flops": 4 * c["width"] * c["heads"] * pairs}
    if c["op"] == "attention":
        return {"bytes": 4 * c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["width"],
                "flops": 4 * c["width"] * c["heads"] * c["batch"] * _visible_pairs(c)}
    return {"bytes": c["rows"] * (c["vocab"] * size[c["dtype"]] + 28), "flops": 0}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"cache": _exact_cache, "cached": _exact_cached, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](s)


def _exact_cache(s):
    c = s["case"]
    if c["cache"] == "f16":
        return {n: s[n].double().half().double() for n in ("k", "v")}
    out = {}
    for n in ("k", "v"):
        x = s[n].double()
        step = x.abs().max(-1, keepdim=True).values / 127
        whole = torch.round(torch.nan_to_num(x / step))
        out[n] = whole * step
        held = torch.zeros_like(s["scale_" + n], dtype=torch.float64).transpose(1, 2).reshape(-1, c["kv_heads"])
        held[s["slots"].long()] = step[..., 0]
        out["scale_" + n] = held.reshape(-1, c["page"], c["kv_heads"]).transpose(1, 2)
    return out


def _exact_rows(q, k, v, at, key_at, lo, hi, scale, cap, slopes):
    """q [heads, rows, width], k and v [heads, keys, width]; row r sees the keys whose place is in [lo_r, hi_r)"""
    z = (q.double() @ k.double().transpose(1, 2)) * scale
    if cap:
        z = torch.tanh(z / cap) * cap
    if slopes is not None:
        z = z - slopes.double()[:, :, None] * (at[:, None] - key_at[None]).abs().double()
    hidden = (key_at[None] < lo[:, None]) | (key_at[None] >= hi[:, None])
    z = z.masked_fill(hidden, -math.inf)
    empty = hidden.all(1)
    z[:, empty] = 0.0
    p = torch.softmax(z, 2)
    p[:, empty] = 0.0
    return p @ v.double()


def _exact_cached(s):
    c = s["case"]
    N, G, T, P, W = c["kv_heads"], c["heads"] // c["kv_heads"], c["queries"], c["prefix"], c["width"]
    if c["batch"] * c["heads"] * T * (P + c["longest"]) * W > 4e11:
        return None
    dev = s["q"].device
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)

    def rows(name, table, n):
        x = s["cache_" + name][table.long()].double()
        if s["scale_" + name] is not None:
            x = x * s["scale_" + name][table.long()].double().unsqueeze(-1)
        return x.permute(1, 0, 2, 3).reshape(N, -1, W)[:, :n]

    pk, pv = rows("k", s["prefix_table"], P), rows("v", s["prefix_table"], P)
    for b, n in enumerate(_lengths(c)):
        k, v = torch.cat([pk, rows("k", s["tables"][b], n)], 1), torch.cat([pv, rows("v", s["tables"][b], n)], 1)
        places = torch.arange(P + n, device=dev)
        t = torch.arange(max(0, T - n), T, device=dev)
        if len(t) == 0:
            continue
        at = (P + n - T + t).repeat_interleave(G)
        q = s["q"][b, t].reshape(len(t), N, G, W).permute(1, 0, 2, 3).reshape(N, len(t) * G, W)
        lo = at - c["window"] + 1 if c["window"] else torch.zeros_like(at)
        slopes = s["slopes"].reshape(N, G).repeat(1, len(t)) if s["slopes"] is not None else None
        o = _exact_rows(q, k, v, at, places, lo, at + 1, 1 / math.sqrt(W), c["cap"], slopes)
        out[b, t] = o.reshape(N, len(t), G, W).permute(1, 0, 2, 3).reshape(len(t), c["heads"], W)
    return out


def _exact_attention(s):
    c = s["case"]
    dev, G, S = s["q"].device, c["heads"] // c["kv_heads"], c["tokens"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
    place = torch.arange(S, device=dev)
    for b in range(c["batch"]):
        lo, hi = torch.zeros_like(place), place + 1
        if s["prefix"] is not None:
            hi = torch.clamp(hi, min=int(s["prefix"][b]))
        if c["window"]:
            lo = torch.clamp(place - c["window"] + 1, min=0)
        if s["spans"] is not None:
            lo, hi = torch.maximum(lo, s["spans"][b, :, 0].long()), torch.minimum(hi, s["spans"][b, :, 1].long())
        for h in range(c["heads"]):
            slopes = s["slopes"][h].reshape(1, 1).expand(1, S) if s["slopes"] is not None else None
            out[b, :, h] = _exact_rows(s["q"][b, :, h][None], s["k"][b, :, h // G][None], s["v"][b, :, h // G][None], place, place, lo, hi,
                                       1 / math.sqrt(c["width"]), c["cap"], slopes)[0]
    return out


def _exact_sample(s):
    c = s["case"]
    logits, uniform = s["logits"].cpu().numpy().astype(np.float64), s["uniform"].cpu().numpy().astype(np.float64)
    f32 = {n: float(np.float32(c[n])) for n in ("temperature", "top_p", "min_p")}
    tokens, chance = np.zeros(c["rows"], np.int32), np.zeros(c["rows"])
    for r in range(c["rows"]):
        x = logits[r]
        if f32["temperature"] <= 0:
            tokens[r], chance[r] = int(np.argmax(x)), 1.0
            continue
        weight = np.exp((x - x.max()) / f32["temperature"])
        best = np.argsort(-x, kind="stable")
        if c["top_k"] > 0:
            best = best[:c["top_k"]]
        if c["top_p"] < 1:
            mass = weight[best]
            best = best[np.cumsum(mass) - mass < f32["top_p"] * mass.sum()]
        best = np.sort(best[weight[best] >= f32["min_p"]])
        sums = np.cumsum(weight[best])
        i = min(int(np.searchsorted(sums, uniform[r] * sums[-1], side="right")), len(best) - 1)
        tokens[r], chance[r] = best[i], weight[best[i]] / sums[-1]
    return {"tokens": torch.from_numpy(tokens), "probabilities": torch.from_numpy(chance)}
