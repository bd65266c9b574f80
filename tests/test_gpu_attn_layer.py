"""GPU tests of the attention layer's train (saber_engine_amd/attn.py) on caches of both kinds, with drafted rows, and without norms and rotation:
every step of a call from the one before it."""
import numpy as np
import pytest
import torch

from oracle import ref
from saber_engine_amd import iu8, synth
from saber_engine_amd.attn import PagedKvCache
from tests.attn_util import BF16, E4M3, Paged, attention, check, e4m3_of, f64
from tests.gpu_util import dev_bf16_bits, host_u16, say
from tests.test_gpu_attn import ends, layer, layer_weights, normed, rotated

pytestmark = pytest.mark.gpu


def rows_of(c):
    """PagedKvCache's rows as attn_util's Paged gives them."""
    p, e4m3 = Paged.__new__(Paged), c.kind == iu8.KV_E4M3
    p.h, p.dim, p.page, p.pages, p.table, p.e4m3, p.e = c.kv_heads, c.head_dim, c.page_tokens, c.pages, c.table, e4m3, 16 if e4m3 else 8
    p.kind, p.scales = torch.float8_e4m3fn if e4m3 else torch.bfloat16, [c.k_scale, c.v_scale]
    p.k = c.k.view(p.kind).view(c.pages, p.h, p.page // 16, p.dim // p.e, 16, p.e)
    p.v = c.v.view(p.kind).view(c.pages, p.h, p.page, p.dim)
    return p


def check_step(n, host, x, news, before):
    cache, T, D, kv = n.cache, n.T, n.cache.head_dim, rows_of(n.cache)
    live, qkv = sum(news), host_u16(n.qkv)
    np.testing.assert_array_equal(qkv, ref.linear(x, host["qkv"]["W"], host["qkv"]["ws"], False, threads=8)["C"])
    rows, rot = f64(n.qkv.view(torch.bfloat16).float()), 0 if n.inv_freq is None else 2 * len(n.inv_freq)
    fr = None if n.inv_freq is None else f64(n.inv_freq)
    q, core = (f64(t.view(torch.bfloat16).float()).reshape(T, n.heads, D) for t in (n.q, n.core))
    slack = lambda y: 1.5e-5 * (np.abs(y).max(-1, keepdims=True) + 1e-30)  # noqa: E731
    t = 0
    for s, new in enumerate(news):
        total = before[s] + new
        k, v, there = kv.rows(s, total)
        if new:
            pos, x0 = np.arange(before[s], total), rows[t:t + new]
            wq = normed(np.stack([x0[:, h * n.q_head:h * n.q_head + D] for h in range(n.heads)], 1), host["norms"][0], n.eps)
            wk = normed(x0[:, n.heads * n.q_head:][:, :kv.h * D].reshape(new, kv.h, D), host["norms"][1], n.eps)
            wv = x0[:, n.heads * n.q_head + kv.h * D:].reshape(new, kv.h, D)
            turned = rotated(wq, pos, fr, rot, n.interleaved)
            check(q[t:t + new], turned, np.abs(turned) * BF16 * 1.01 + slack(wq), f"q of sequence {s}")
            turned = rotated(wk, pos, fr, rot, n.interleaved)
            if kv.e4m3:
                ks, vs = (f64(x)[:, None] for x in kv.scales)
                want = np.clip(turned / ks, -448, 448)
                check(k[before[s]:] / ks, want, np.abs(want) * E4M3 * 1.01 + 2.0 ** -10 + slack(wk / ks), f"k of sequence {s}")
                for h in range(kv.h):
                    assert np.array_equal(v[before[s]:, h] / vs[h], e4m3_of(wv[:, h], vs[h, 0])), f"v of sequence {s}"
            else:
                check(k[before[s]:], turned, np.abs(turned) * BF16 * 1.01 + slack(wk), f"k of sequence {s}")
                assert np.array_equal(v[before[s]:], wv), f"v of sequence {s}"
            want, tol = attention(q[t:t + new], k, v, there, n.scale)
            check(core[t:t + new], want, tol, f"attention of sequence {s}")
        t += new
    bits = host_u16(n.core).reshape(T, -1)[:live]
    if n.gated:
        codes, scales = ref.attn_gate_quant_had(bits, qkv[:live], host["t"], D)
        S, _ = ref.gemm_fast(codes, host["o"]["W"], False, threads=8)
        want = ref.epilogue(S, scales, host["o"]["ws"], False)
    else:
        want = ref.linear(bits, host["o"]["W"], host["o"]["ws"], False, threads=8)["C"]
    np.testing.assert_array_equal(host_u16(n.out)[:live], want)


@pytest.mark.parametrize("e4m3,gated,heads,kvh,dim,hidden,plain", [
    (True, True, 4, 1, 256, 512, False), (True, False, 8, 2, 128, 256, False), (True, False, 4, 2, 64, 256, True), (False, True, 4, 2, 64, 256, False),
    (False, False, 8, 2, 128, 256, True)])
def test_layer_prompts_drafted_rows_single_tokens(ctx, e4m3, gated, heads, kvh, dim, hidden, plain):
    """Packed prompts, then steps of up to four drafted rows a sequence and of single tokens, each captured once and replayed while the counts, the rows'
    ends and the page table change. `plain`: no norms, no rotation."""
    say(f"attention layer, e4m3 {e4m3}, gated {gated}, {heads} heads of {dim}, plain {plain}")
    rng = np.random.default_rng(dim + e4m3)
    host, weights = layer_weights(heads, kvh, dim, hidden, gated, 70 + dim)
    freq = None if plain else torch.tensor([1e6 ** (-i / 16) for i in range(16)], dtype=torch.float64).cuda()
    if plain:
        host["norms"], weights = (None, None), (*weights[:-2], None, None)
    scales = [torch.rand(kvh, generator=torch.Generator().manual_seed(7)).add_(0.5).div_(64).cuda() for _ in range(2)] if e4m3 else (None, None)
    cache = PagedKvCache(3, kvh, dim, 700, page_tokens=32, kind=iu8.KV_E4M3 if e4m3 else iu8.KV_BF16, k_scale=scales[0], v_scale=scales[1])
    lens = [0, 0, 0]

    def reserve(news):
        before = list(lens)
        for s, new in enumerate(news):
            lens[s] += new
            cache.reserve(s, lens[s])
        cache.kv_len.copy_(torch.tensor(lens))
        return before

    for news, T in (([70, 0, 200], 272), ([30, 129, 5], 164)):
        n = layer(ctx, cache, T, max(news), gated, heads, hidden, weights, freq)
        x = synth.activations(rng, T, hidden)
        n.cu_q.copy_(ends(news))
        before = reserve(news)
        n.forward(dev_bf16_bits(x), max_kv=max(lens))
        torch.cuda.synchronize()
        check_step(n, host, x, news, before)

    for T, max_q, steps in ((12, 4, ([4, 1, 3], [2, 4, 0], [4, 4, 4], [1, 0, 1])), (3, 1, ([1, 1, 1],) * 3)):
        n = layer(ctx, cache, T, max_q, gated, heads, hidden, weights, freq)
        x_dev = torch.zeros((T, hidden), dtype=torch.int16, device="cuda")
        stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            n.forward(x_dev, stream.cuda_stream)
        for i, news in enumerate(steps):
            if i == 2:                     # a sequence leaves, another takes its pages and its place; drafted rows of another are refused
                cache.release(0)
                lens[0], lens[1] = 0, lens[1] - 1
            before = reserve(news)
            if n.cu_q is not None:
                n.cu_q.copy_(ends(news))
            x = synth.activations(rng, T, hidden)
            x_dev.copy_(dev_bf16_bits(x))
            n.core.fill_(0x7FC0)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
            torch.cuda.synchronize()
            check_step(n, host, x, news, before)
            assert (n.core[sum(news):] == 0x7FC0).all(), "rows behind the last sequence"
            assert n._attn_ws[1] is None or not n._attn_ws[1].any()
