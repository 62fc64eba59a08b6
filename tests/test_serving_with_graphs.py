"""A decoder whose dense parts are executor graphs and whose attention runs over a cache: tokens one by one, every step queued from
device memory to device memory, the host waits for the drawn tokens alone."""
import numpy as np
import pytest

import kyanite_amd as kn
from kyanite_amd import BATCH, DType, Graph, HipExecutor
from serving_oracle import attend, sample, upload


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [DType.F16, DType.I8], ids=lambda d: d.name)
def test_a_decoder_of_graphs_around_a_cache(cache_dtype, hip_device):
    B, D, H, N, W, V, page, steps = 3, 128, 4, 2, 32, 300, 16, 20
    rng = np.random.default_rng(11)
    weights = {n: (rng.standard_normal(shape) * shape[1] ** -0.5).astype(np.float16)
               for n, shape in dict(q=(H * W, D), k=(N * W, D), v=(N * W, D), o=(D, H * W), e=(V, D)).items()}

    before = Graph()  # x -> q, k, v
    x_in = before.input([BATCH, D], DType.F16)
    before.output_all([before.linear(x_in, before.constant(list(weights[n].shape), weights[n])) for n in "qkv"])
    after = Graph()  # what attention gives, x -> logits
    a_in, r_in = after.input([BATCH, H * W], DType.F16), after.input([BATCH, D], DType.F16)
    hidden = after.add(r_in, after.linear(a_in, after.constant([D, H * W], weights["o"])))
    after.output(after.linear(hidden, after.constant([V, D], weights["e"])))
    first, second = HipExecutor(hip_device, before, B), HipExecutor(hip_device, after, B, preserve_inputs=True)
    streams = [kn.HipStream.borrowed(hip_device, ex.stream()) for ex in (first, second)]

    table_pages = -(-steps // page)
    elem = 2 if cache_dtype == DType.F16 else 1
    mem = [kn.DeviceBuffer(hip_device, B * table_pages * N * page * W * elem) for _ in range(2)]
    scales = [kn.DeviceBuffer(hip_device, B * table_pages * N * page * 4) for _ in range(2)]
    cache = kn.kv_cache(cache_dtype, B * table_pages, N, page, W, mem[0].ptr, mem[1].ptr, *([s.ptr for s in scales] if cache_dtype == DType.I8 else [0, 0]))
    tables = upload(hip_device, np.arange(B * table_pages, dtype=np.int32))
    # what changes from step to step, for all steps at once: the calls of a step read their part
    slots = upload(hip_device, np.stack([np.arange(B) * table_pages * page + t for t in range(steps)]).astype(np.int32))
    lengths = upload(hip_device, np.repeat(np.arange(1, steps + 1)[:, None], B, 1).astype(np.int32))
    u = rng.random((steps, B)).astype(np.float32)
    uniform, temperature, tokens = upload(hip_device, u), upload(hip_device, np.full(B, 0.7, np.float32)), kn.DeviceBuffer(hip_device, B * 4)
    q, k, v = (first.output_ptr(i) for i in range(3))
    draw_args = [kn.sample_args(DType.F16, B, V, second.output_ptr(0), V, uniform.ptr + t * B * 4, tokens.ptr, temperature=temperature.ptr) for t in range(steps)]
    keys, values = np.zeros((B, steps, N, W)), np.zeros((B, steps, N, W))
    x = weights["e"][:B]
    for t in range(steps):
        first.upload_input(0, x)
        second.upload_input(1, x)
        first.run_async()
        kn.cache_write(hip_device, streams[0], cache, kn.cache_rows(DType.F16, B, k, (N * W, W), v, (N * W, W), slots.ptr + t * B * 4))
        args = kn.cached_attention_args(B, 1, H, cache, q, (H * W, H * W, W), second.input_ptr(0), (H * W, H * W, W), lengths.ptr + t * B * 4, tables.ptr,
                                        table_pages, table_pages)
        workspace = kn.DeviceBuffer(hip_device, max(kn.cached_attention_workspace_bytes(args), 1))
        kn.cached_attention(hip_device, streams[0], args, workspace)
        streams[1].wait_for_event(streams[0].record_event())
        second.run_async()
        kn.sample(hip_device, streams[1], draw_args[t])
        streams[1].synchronize()
        drawn = tokens.to_array(np.int32, B)

        got = {n: first.download_output(i).astype(np.float64) for i, n in enumerate("qkv")}
        for n in "qkv":
            e = x.astype(np.float64) @ weights[n].astype(np.float64).T
            # (sums of D products in f32, rounded to f16)
            assert (np.abs(got[n] - e) <= np.abs(e) * 2.0 ** -11 + np.abs(x.astype(np.float64)) @ np.abs(weights[n].astype(np.float64)).T * (D + 1) * 2.0 ** -24 + 2.0 ** -24).all()
        keys[:, t], values[:, t] = got["k"].reshape(B, N, W), got["v"].reshape(B, N, W)
        att = np.zeros((B, H, W))
        bound = np.zeros((B, H, W))
        for b in range(B):
            for h in range(H):
                kk, vv = keys[b, :t + 1, h * N // H], values[b, :t + 1, h * N // H]
                qq = got["q"][b].reshape(H, W)[h][None]
                o, e = attend(qq, kk, vv, np.array([t]), np.arange(t + 1), np.ones((1, t + 1), bool), W ** -0.5, 0.0, 0.0)
                if cache_dtype == DType.I8:  # rows are off by half a step of their largest element over 127
                    step_k, step_v = np.abs(kk).max(-1) / 127 / 2, np.abs(vv).max() / 127 / 2
                    moved = W ** -0.5 * np.abs(qq).sum() * step_k.max()
                    e = e + step_v + 2 * np.expm1(moved) * np.abs(vv).max()
                att[b, h], bound[b, h] = o[0], e[0]
        # the logits from what the attention ought to give, its error going through both products
        x64, wo, we = x.astype(np.float64), weights["o"].astype(np.float64), weights["e"].astype(np.float64)
        hidden64, logits = x64 + att.reshape(B, -1) @ wo.T, second.download_output(0)
        off = bound.reshape(B, -1) @ np.abs(wo).T
        size = np.abs(x64) + np.abs(att.reshape(B, -1)) @ np.abs(wo).T
        off = off + size * (2.0 ** -10 + (H * W) * 2.0 ** -24)  # (rounded to f16 behind the product and behind the sum)
        e = hidden64 @ we.T
        off = off @ np.abs(we).T + np.abs(hidden64) @ np.abs(we).T * (D + 1) * 2.0 ** -24 + np.abs(e) * 2.0 ** -11 + 2.0 ** -24
        assert (np.abs(logits.astype(np.float64) - e) <= off).all(), f"step {t}: {np.max(np.abs(logits - e) / off):.2f} of the bound"
        assert np.array_equal(drawn, sample(logits, u[t], temperature=np.full(B, 0.7, np.float32))[0])
        x = weights["e"][drawn]
