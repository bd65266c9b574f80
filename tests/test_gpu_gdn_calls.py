"""GPU tests of calls that a serving step makes of a delta-net layer's core: long runs of the convolution, prompts and single or drafted rows in one batch, keys and
queries of any size, a hybrid graph's sequence that goes on in two ways after a fork."""
import numpy as np
import pytest
import torch

from saber_engine_amd import iu8
from saber_engine_amd.attn import PagedKvCache
from saber_engine_amd.gdn import GdnState
from tests.attn_util import f64
from tests.gdn_util import D, Rows, ends
from tests.gpu_util import say
from tests.test_gpu_gdn import conv_case, rule_case, workspace
from tests.test_gpu_gdn_sizes import compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels,tokens", [(264, 2100), (10240, 440)])
def test_conv_runs_of_eight_rows(ctx, channels, tokens, width):
    """As many rows a thread as the kernel takes: sequences that begin at every place of a run, and shorter than the width across a run's end."""
    say(f"conv, {tokens} rows of {channels} channels, width {width}")
    rng = np.random.default_rng(width)
    lens = [n for first in range(1, 9) for n in (first, 1, 2, 1, 3, 8 + first)]
    while sum(lens) < tokens:
        lens.append(int(rng.choice([0, 1, 1, 2, 3, 4, 5, 7, 8, 9, 16, 33])))
    conv_case(ctx, channels, width, lens, bias=width == 3, front=width, behind=3, more=8)
    conv_case(ctx, channels, width, lens, kept=[int(rng.integers(-1, n + 2)) for n in lens], lost=[(5, -1), (20, len(lens) + 2)])


@pytest.mark.parametrize("lens", [[1] * 20 + [150] + [1] * 11, [130, 5, 5, 0, 1, 67]])
def test_prompts_and_single_rows_in_one_batch(ctx, lens):
    say(f"delta rule, a batch of {len(lens)} sequences of up to {max(lens)} rows")
    rule_case(ctx, Rows(2, 4, lens, front=1, behind=2, seed=60), chunked=True)
    rule_case(ctx, Rows(2, 4, lens, front=1, behind=2, seed=60))


def test_prompts_and_drafted_rows_in_one_batch(ctx):
    """kept for the drafted rows, a prompt whole beside them, and the call that makes the accepted ones count; a workspace is there."""
    say("delta rule, a prompt beside drafted rows")
    lens, take = [100, 5, 3, 0, 70, 5], [100, 0, 0, 0, 70, 0]
    r = Rows(2, 4, lens, seed=61)
    was, ws = f64(r.state), workspace(r)
    r.call(ctx, kept=torch.tensor(take, dtype=torch.int32, device="cuda"), workspace=ws)
    r.call(ctx, kept=torch.tensor([0, 2, 3, 0, 0, 1], dtype=torch.int32, device="cuda"), workspace=ws, out=False)
    torch.cuda.synchronize()
    counted = [100, 2, 3, 0, 70, 1]
    for s, t, p, (want, tol, states, tols) in r.want(was):
        assert (np.abs(f64(r.out[t:t + lens[s]].float()) - want) <= tol).all(), s
        assert (np.abs(f64(r.state[p]) - states[counted[s]]) <= tols[counted[s]]).all(), s


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("k,q", [(2.0 ** 58, 2.0 ** -20), (2.0 ** -12, 2.0 ** 58), (2.0 ** 30, 2.0 ** 30)])
def test_keys_and_queries_of_any_size(ctx, k, q, chunked):
    say(f"delta rule, keys of {k}, queries of {q}, chunked {chunked}")
    r = Rows(2, 4, [100, 30], seed=62)
    keys = r.kh * D
    r.rows[:, :keys] *= q
    r.rows[:, keys:2 * keys] *= k
    was = f64(r.state)
    r.call(ctx, workspace=workspace(r) if chunked else None)
    torch.cuda.synchronize()
    compare(r, was, chunked, 1.0)


def test_a_hybrid_sequence_goes_on_in_two_ways_after_a_fork(ctx):
    """Pages (K and V) and states of a fork, and of the sequence that it was forked from, moved on by the same rows and by others: the first two alike byte for byte, and as
    without a fork."""
    say("a hybrid sequence forked and moved on")
    kvh, dim, page, n, more, heads = 2, 128, 32, 75, 40, 4
    g = torch.Generator().manual_seed(63)
    kv = torch.randn(n + 3 * more, 2 * kvh * dim + 4 * dim, generator=g).bfloat16().cuda()
    kv[n + more:n + 2 * more] = kv[n:n + more]                      # sequence 1 goes on as sequence 0 does, sequence 2 by itself
    r = Rows(2, heads, [n] + [more] * 3, seed=64)
    r.rows[n + more:n + 2 * more], r.ab[n + more:n + 2 * more] = r.rows[n:n + more], r.ab[n:n + more]
    q = torch.zeros(3 * more, 4, dim, dtype=torch.bfloat16, device="cuda")

    def append(c, at, lens):
        p, cu = kv[at:].data_ptr(), ends(lens)
        ctx.kv_append(p + 4 * kvh * dim, p, p + 2 * kvh * dim, q.data_ptr(), c.desc, cu.data_ptr(), sum(lens), 3, 4, kv.shape[1], dim, kv.shape[1])
        torch.cuda.synchronize()

    def advance(st, at, lens):
        out, cu, tokens, rows = torch.zeros(sum(lens), heads, D, dtype=torch.bfloat16, device="cuda"), ends(lens), sum(lens), r.rows[at:].data_ptr()
        ws = torch.empty(iu8.gdn_workspace(tokens, 3, max(lens), 2, heads), dtype=torch.uint8, device="cuda")
        ctx.gdn(rows, rows + 4 * D, rows + 8 * D, r.row, r.ab[at:].data_ptr(), r.ab[at:].data_ptr() + 2 * heads, r.ab.shape[1], r.a_log.data_ptr(), r.dt_bias.data_ptr(),
                st.state.data_ptr(), st.slots, out.data_ptr(), tokens, 3, max(lens), 2, heads, r.scale, slot=st.slot.data_ptr(), cu_q=cu.data_ptr(), workspace=ws.data_ptr())
        torch.cuda.synchronize()
        return out

    def begin():
        c, st = PagedKvCache(3, kvh, dim, 300, page_tokens=page), GdnState(3, 2, heads)
        c.reserve(0, n), st.begin(0)
        c.kv_len[0] = n
        append(c, 0, [n, 0, 0]), advance(st, 0, [n, 0, 0])
        return c, st

    def pages(c, s, count):
        """K and V of a sequence's positions, as bytes: of K the 16 tokens that lie together."""
        at = torch.arange(count, device="cuda")
        held = torch.tensor(c._held[s], device="cuda")[at // page]
        k = c.k.view(c.pages, kvh, page // 16, dim // 8, 16, 16)[held, :, at % page // 16, :, at % 16]
        return k, c.v.view(c.pages, kvh, page, dim * 2)[held, :, at % page]

    c, st = begin()
    for d in (1, 2):
        c.fork(ctx, 0, d, n)
    st.fork(ctx, 0, [1, 2])
    for s in range(3):
        c.reserve(s, n + more)
    c.kv_len += more
    append(c, n, [more] * 3)
    out = advance(st, n, [more] * 3)
    alone, alone_st = begin()
    alone.reserve(0, n + more)
    alone.kv_len[0] = n + more
    append(alone, n, [more, 0, 0])
    want = advance(alone_st, n, [more, 0, 0])
    of = [pages(c, s, n + more) for s in range(3)]
    for i, what in enumerate(("K", "V")):
        assert torch.equal(of[0][i], of[1][i]) and torch.equal(of[0][i], pages(alone, 0, n + more)[i]), what
        assert torch.equal(of[2][i][:n], of[0][i][:n]) and not torch.equal(of[2][i][n:], of[0][i][n:]), what
    v = kv[:n + more, kvh * dim:2 * kvh * dim].reshape(-1, kvh, dim)
    assert torch.equal(of[0][1].contiguous().view(torch.bfloat16), v)
    assert torch.equal(of[0][0].contiguous().view(torch.bfloat16).reshape(-1, kvh, dim), kv[:n + more, :kvh * dim].reshape(-1, kvh, dim))
    assert torch.equal(out[:more], out[more:2 * more]) and torch.equal(out[:more], want) and not torch.equal(out[2 * more:], want)
    state = [st.state[p] for p in st._held]
    assert torch.equal(state[0], state[1]) and torch.equal(state[0], alone_st.state[alone_st._held[0]]) and not torch.equal(state[0], state[2])
