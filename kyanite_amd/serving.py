"""The operators that serve a decoder token by token (include/knhip.h): keys and values into a cache and back, attention
over the cache and of whole prompts, and the draw of a token. Like `matmul_args` / `batched_mat_mul` each operator has a
builder for its argument block, which holds device addresses and can be kept from step to step, and a call that queues
the work on a stream. `stream`: a HipStream, or the address of a stream (0: the device's default stream)."""
from ctypes import byref, c_size_t, c_void_p

from ._lib import (AttentionArgsT, CachedAttentionArgsT, CacheRowsT, KnError, KvCacheT, SampleArgsT, check, lib)
from .graph import DType
from .runtime import HipStream, _index


def _three(name, strides, axes="batch, token, head"):
    strides = tuple(int(s) for s in strides)
    if len(strides) != 3:
        raise KnError(f"{name} takes three strides ({axes}), got {strides}")
    return strides


def _two(name, strides):
    strides = tuple(int(s) for s in strides)
    if len(strides) != 2:
        raise KnError(f"{name} takes two strides (token, head), got {strides}")
    return strides


def kv_cache(dtype, pages, heads, page_tokens, width, k, v, k_scales=0, v_scales=0, strides=None):
    """`k`, `v`: addresses of [pages, heads, page_tokens, width]; `strides` (page, head, token) in elements, dense when
    not given; the scales of a DType.I8 cache are dense f32 [pages, heads, page_tokens]."""
    c = KvCacheT()
    c.dtype, c.pages, c.heads, c.page_tokens, c.width = int(DType(dtype)), pages, heads, page_tokens, width
    c.k, c.v, c.k_scales, c.v_scales = k, v, k_scales or None, v_scales or None
    if strides is None:
        strides = (heads * page_tokens * width, page_tokens * width, width)
    c.page_stride, c.head_stride, c.token_stride = _three("a cache", strides, "page, head, token")
    return c


def cache_rows(dtype, tokens, k, k_strides, v, v_strides, slots):
    """`k`, `v`: addresses of [tokens, heads, width] with (token, head) strides; `slots`: address of i32 [tokens]."""
    r = CacheRowsT()
    r.dtype, r.tokens, r.k, r.v, r.slots = int(DType(dtype)), tokens, k, v, slots
    r.k_token_stride, r.k_head_stride = _two("k", k_strides)
    r.v_token_stride, r.v_head_stride = _two("v", v_strides)
    return r


def _stream(stream):
    return stream._h if isinstance(stream, HipStream) else c_void_p(stream)


def _workspace(workspace):
    return (c_void_p(workspace.ptr), workspace.nbytes) if workspace is not None else (None, 0)


def cache_write(device, stream, cache, rows):
    """Queue the write of `rows` into their slots of `cache`."""
    check(lib.knhip_cache_write(_index(device), _stream(stream), byref(cache), byref(rows)))


def cache_read(device, stream, cache, rows):
    """Queue the read of the slots of `rows` out of `cache` into the rows."""
    check(lib.knhip_cache_read(_index(device), _stream(stream), byref(cache), byref(rows)))


def cached_attention_args(batch, queries, heads, cache, q, q_strides, out, out_strides, lengths, tables, table_stride, table_pages,
                          prefix_tokens=0, prefix_table=0, scale=None, cap=0.0, slopes=0, window=0):
    """Strides are (batch, token, head) in elements; `scale` is 1 / sqrt(width) when not given."""
    a = CachedAttentionArgsT()
    a.batch, a.queries, a.heads, a.cache = batch, queries, heads, cache
    a.q, (a.q_batch_stride, a.q_token_stride, a.q_head_stride) = q, _three("q", q_strides)
    a.out, (a.out_batch_stride, a.out_token_stride, a.out_head_stride) = out, _three("out", out_strides)
    a.lengths, a.tables, a.table_stride, a.table_pages = lengths, tables, table_stride, table_pages
    a.prefix_tokens, a.prefix_table = prefix_tokens, prefix_table or None
    a.scale = max(cache.width, 1) ** -0.5 if scale is None else scale
    a.cap, a.slopes, a.window = cap, slopes or None, window
    return a


def cached_attention_workspace_bytes(args):
    n = c_size_t()
    check(lib.knhip_cached_attention_workspace_bytes(byref(args), byref(n)))
    return n.value


def cached_attention(device, stream, args, workspace=None):
    """`workspace`: a DeviceBuffer of at least `cached_attention_workspace_bytes(args)` when that is not 0."""
    ptr, size = _workspace(workspace)
    check(lib.knhip_cached_attention(_index(device), _stream(stream), byref(args), ptr, size))


def attention_args(batch, queries, keys, heads, kv_heads, width, q, q_strides, k, k_strides, v, v_strides, out, out_strides, scale=None,
                   cap=0.0, slopes=0, causal=False, window=0, spans=0, prefix=0):
    """Strides are (batch, token, head) in elements; `scale` is 1 / sqrt(width) when not given."""
    a = AttentionArgsT()
    a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.width = batch, queries, keys, heads, kv_heads, width
    a.q, (a.q_batch_stride, a.q_token_stride, a.q_head_stride) = q, _three("q", q_strides)
    a.k, (a.k_batch_stride, a.k_token_stride, a.k_head_stride) = k, _three("k", k_strides)
    a.v, (a.v_batch_stride, a.v_token_stride, a.v_head_stride) = v, _three("v", v_strides)
    a.out, (a.out_batch_stride, a.out_token_stride, a.out_head_stride) = out, _three("out", out_strides)
    a.scale = max(width, 1) ** -0.5 if scale is None else scale
    a.cap, a.slopes, a.causal, a.window, a.spans, a.prefix = cap, slopes or None, int(causal), window, spans or None, prefix or None
    return a


def attention_workspace_bytes(args):
    n = c_size_t()
    check(lib.knhip_attention_workspace_bytes(byref(args), byref(n)))
    return n.value


def attention(device, stream, args, workspace=None):
    """`workspace`: a DeviceBuffer of at least `attention_workspace_bytes(args)` when that is not 0."""
    ptr, size = _workspace(workspace)
    check(lib.knhip_attention(_index(device), _stream(stream), byref(args), ptr, size))


def sample_args(dtype, rows, vocab, logits, row_stride, uniform, tokens, temperature=0, top_k=0, top_p=0, min_p=0, probabilities=0):
    """Everything behind `row_stride` is the address of an array with an entry per row; 0 switches that filter off."""
    a = SampleArgsT()
    a.dtype, a.rows, a.vocab, a.logits, a.row_stride = int(DType(dtype)), rows, vocab, logits, row_stride
    a.uniform, a.tokens, a.probabilities = uniform, tokens, probabilities or None
    a.temperature, a.top_k, a.top_p, a.min_p = temperature or None, top_k or None, top_p or None, min_p or None
    return a


def sample_workspace_bytes(args):
    n = c_size_t()
    check(lib.knhip_sample_workspace_bytes(byref(args), byref(n)))
    return n.value


def sample(device, stream, args, workspace=None):
    """`workspace`: a DeviceBuffer of at least `sample_workspace_bytes(args)` when that is not 0."""
    ptr, size = _workspace(workspace)
    check(lib.knhip_sample(_index(device), _stream(stream), byref(args), ptr, size))
