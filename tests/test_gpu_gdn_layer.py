"""GPU tests of the delta-net layer's train and of sequences forked in a hybrid graph's memory (saber_engine_amd/gdn.py, attn.py): every step of a call from the one
before it."""
import numpy as np
import pytest
import torch

from oracle import ref
from saber_engine_amd import iu8, synth
from saber_engine_amd.attn import PagedKvCache
from saber_engine_amd.gdn import GdnLayerIU8, GdnState
from tests.attn_util import check, f64
from tests.gdn_util import D, convolved, ends, rule
from tests.gpu_util import dev_bf16_bits, dev_f32, dev_u8, host_u16, say
from tests.test_gpu_had import device_silu_f32_table

pytestmark = pytest.mark.gpu


def layer_weights(kh, heads, hidden, width, bias, seed):
    rng = np.random.default_rng(seed)
    channels, core = (2 * kh + heads) * D, heads * D
    lin = [synth.dense_case(1, n, k, seed=seed + i) for i, (n, k) in enumerate(((channels + core, hidden), (2 * heads, hidden), (hidden, core)))]
    bf = lambda *n: torch.from_numpy(rng.standard_normal(n).astype(np.float32) * 0.4).bfloat16().cuda()  # noqa: E731
    t = rng.choice([-1.0, 1.0], size=core).astype(np.float32)
    host = dict(lin=lin, t=t, conv=bf(channels, width), conv_bias=bf(channels) if bias else None, norm=bf(128), a_log=np.log(rng.uniform(0.01, 8, heads)), dt=rng.standard_normal(heads) - 2)
    dev = [x for w in lin for x in (dev_u8(iu8.repack_w4(w["W"])), dev_f32(w["ws"]))]
    return host, dict(zip("wqkvz_frag wsqkvz wba_frag wsba wo_frag wso".split(), dev), conv=host["conv"], conv_bias=host["conv_bias"], a_log=dev_f32(host["a_log"]),
                      dt_bias=dev_f32(host["dt"]), norm=host["norm"], had_t=dev_f32(t))


def check_step(n, host, x, news, state, tail, silu, kept=None, chunked=False):
    """The linears' and producer's bytes are the oracle's, what lies between them within the rounding; state, tail: as they were."""
    st, T, live = n.state, n.T, sum(news)
    lin = [ref.linear(x, w["W"], w["ws"], False, threads=8)["C"] for w in host["lin"][:2]]
    qkvz, ba = host_u16(n.qkvz), host_u16(n.ba)
    np.testing.assert_array_equal(qkvz, lin[0])
    np.testing.assert_array_equal(ba, lin[1])
    val = lambda t: f64(t.view(torch.bfloat16).float())  # noqa: E731
    rows, mixed, gates, core = val(n.qkvz)[:, :st.channels], val(n.qkv), val(n.ba), val(n.core).reshape(T, st.heads, D)
    t, keys = 0, st.key_heads * D
    for s, new in enumerate(news):
        p = st._held[s]
        if new and p is not None:
            want, tol = convolved(rows[t:t + new], tail[p], f64(n.conv.float()), None if n.conv_bias is None else f64(n.conv_bias.float()))
            check(mixed[t:t + new], want, tol, f"convolution of sequence {s}")
            m, take = mixed[t:t + new], new if kept is None else kept[s]
            want, tol, states, tols = rule(m[:, :keys].reshape(new, -1, D), m[:, keys:2 * keys].reshape(new, -1, D), m[:, 2 * keys:].reshape(new, st.heads, D),
                                           gates[t:t + new, st.heads:], gates[t:t + new, :st.heads], f64(n.a_log), f64(n.dt_bias), state[p], n.eps, n.scale, chunked)
            check(core[t:t + new], want, tol, f"rule of sequence {s}")
            check(f64(st.state[p]), states[take], np.broadcast_to(tols[take], state[p].shape), f"state of sequence {s}")
            assert np.array_equal(val(st.tail[p]), np.concatenate((tail[p], rows[t:t + take]))[take:]), f"tail of sequence {s}"
        t += new
    bits, z = host_u16(n.core)[:live], qkvz[:live, st.channels:]
    q, sc = ref.gdn_norm_quant_had(bits, z, n.norm.view(torch.int16).cpu().numpy().view(np.uint16), host["t"], n.eps, silu_tab=silu)
    S, _ = ref.gemm_fast(q, host["lin"][2]["W"], False, threads=8)
    np.testing.assert_array_equal(host_u16(n.out)[:live], ref.epilogue(S, sc, host["lin"][2]["ws"], False))


@pytest.mark.parametrize("kh,heads,hidden,width,bias", [(2, 8, 256, 4, False), (8, 16, 512, 3, True), (16, 48, 256, 4, False)])
def test_layer_prompts_drafted_rows_single_tokens(ctx, kh, heads, hidden, width, bias):
    """Packed prompts, drafted rows of which some are accepted, single tokens in a captured step while the slots change; a fork between."""
    say(f"delta-net layer, {heads} heads on {kh}, width {width}")
    silu = device_silu_f32_table(ctx)
    rng = np.random.default_rng(heads)
    host, weights = layer_weights(kh, heads, hidden, width, bias, 40 + kh)
    st = GdnState(4, kh, heads, slots=5, width=width)
    val = lambda t: f64(t.view(torch.bfloat16).float())  # noqa: E731
    for s in (2, 0, 3):
        st.begin(s)

    def step(n, news, graph=None, stream=0, **more):
        x = synth.activations(rng, n.T, hidden)
        xd = dev_bf16_bits(x)
        was = f64(st.state), val(st.tail)
        if graph is None:
            n.forward(xd, stream=stream, **more)
        else:
            graph[1].copy_(xd)
            graph[0].replay()
        torch.cuda.synchronize()
        return x, was

    def train(tokens, max_q):
        n = GdnLayerIU8(ctx, st, tokens, hidden, max_q=max_q)
        n.set_weights(**weights)
        return n

    prompt = train(150, 100)
    news = [70, 0, 45, 35]
    prompt.cu_q.copy_(ends(news))
    x, was = step(prompt, news)
    check_step(prompt, host, x, news, *was, silu, chunked=True)
    st.fork(ctx, 2, [1])
    torch.cuda.synchronize()
    assert torch.equal(st.state[st._held[1]], st.state[st._held[2]]) and torch.equal(st.tail[st._held[1]], st.tail[st._held[2]])
    # drafted rows: nothing moves, then the accepted ones do
    draft, news, take = train(14, 5), [4, 1, 5, 3], [2, 0, 5, 1]
    draft.cu_q.copy_(ends(news))
    zeros, kept = (torch.tensor(k, dtype=torch.int32, device="cuda") for k in ([0] * 4, take))
    x, was = step(draft, news, kept=zeros)
    check_step(draft, host, x, news, *was, silu, kept=[0] * 4)
    assert np.array_equal(f64(st.state), was[0]) and np.array_equal(val(st.tail), was[1])
    draft.accept(kept)
    torch.cuda.synchronize()
    check_step(draft, host, x, news, *was, silu, kept=take)
    # single tokens, captured once
    one, side = train(4, 1), torch.cuda.Stream()
    xd = torch.zeros((4, hidden), dtype=torch.int16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        one.forward(xd, stream=side.cuda_stream)
    for i in range(4):
        if i == 1:
            st.release(3)
        if i == 2:
            st.begin(3)
        if i == 3:
            st.release(0), st.release(1)
            st.fork(ctx, 3, [0, 1])
        torch.cuda.synchronize()
        live = [st._held[s] is not None for s in range(4)]
        one.core.zero_()
        x, was = step(one, [1] * 4, graph=(graph, xd))
        check_step(one, host, x, [1] * 4, *was, silu)
        assert (host_u16(one.core)[[s for s in range(4) if not live[s]]] == 0).all()


def test_a_hybrid_sequence_forked(ctx):
    """Pages and states of one sequence to two others, each of which goes on by itself as the first would have."""
    say("a sequence forked: pages and states")
    kvh, dim, page = 2, 128, 32
    c, st = PagedKvCache(3, kvh, dim, 300, page_tokens=page), GdnState(3, 2, 4)
    g = torch.Generator().manual_seed(5)
    n = 75
    c.reserve(0, n), st.begin(0)
    rows = torch.randn(n + 9, 2 * kvh * dim + 4 * dim, generator=g).bfloat16().cuda()
    q = torch.zeros(n, 4, dim, dtype=torch.bfloat16, device="cuda")
    c.kv_len[0] = n
    cu = torch.tensor([0, n, n, n], dtype=torch.int32, device="cuda")
    p = rows.data_ptr()
    ctx.kv_append(p + 4 * kvh * dim, p, p + 2 * kvh * dim, q.data_ptr(), c.desc, cu.data_ptr(), n, 3, 4, rows.shape[1], dim, rows.shape[1])
    st.state[st._held[0]] = torch.randn(4, D, D, generator=g).cuda()
    for d in (1, 2):
        c.fork(ctx, 0, d, n)
    st.fork(ctx, 0, [1, 2])
    # each sequence's next three tokens, which are not the others'
    c.kv_len += 3
    for s in range(3):
        c.reserve(s, n + 3)
    cu = torch.tensor([0, 3, 6, 9], dtype=torch.int32, device="cuda")
    p = rows[n:].data_ptr()
    ctx.kv_append(p + 4 * kvh * dim, p, p + 2 * kvh * dim, q.data_ptr(), c.desc, cu.data_ptr(), 9, 3, 4, rows.shape[1], dim, rows.shape[1])
    torch.cuda.synchronize()
    v = c.v.view(torch.bfloat16).view(c.pages, kvh, page, dim)
    for s in range(3):
        want = torch.cat((rows[:n], rows[n + 3 * s:n + 3 * s + 3]))[:, kvh * dim:2 * kvh * dim].view(-1, kvh, dim)
        at = torch.arange(n + 3)
        pages = torch.tensor(c._held[s])[at // page]
        assert torch.equal(v[pages.cuda(), :, (at % page).cuda()], want), s
        assert torch.equal(st.state[st._held[s]], st.state[st._held[0]])
    assert c._held[1][:2] == c._held[0][:2] == c._held[2][:2] and len({h[2] for h in c._held}) == 3
    for s in (0, 1):
        c.release(s)
    before = {t: v[c._held[2][t // page], :, t % page].clone() for t in (0, 40, 77)}
    assert c.compact(ctx) == 3 and max(c._held[2]) < 3
    torch.cuda.synchronize()
    for t, x in before.items():
        assert torch.equal(v[c._held[2][t // page], :, t % page], x)
