"""GPU tests of a delta-net layer's core (code object `delta_net`), through the C ABI, against its definition in 64 bits (gdn_util.py, which derives the
tolerances)."""
import numpy as np
import pytest
import torch

from saber_engine_amd import iu8
from tests.attn_util import check, f64
from tests.gdn_util import D, Rows, convolved, ends
from tests.gpu_util import say

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ convolution

def conv_case(ctx, channels, width, lens, packed=True, bias=False, front=0, behind=0, more=0, kept=None, lost=(), slots=None, seed=3):
    g = torch.Generator().manual_seed(seed)
    seqs, live = len(lens), sum(lens)
    tokens, slots = front + live + behind, slots or seqs + 2
    x = torch.full((tokens, channels + more), float("nan"), dtype=torch.bfloat16)
    x[front:front + live] = torch.randn(live, channels + more, generator=g).bfloat16()
    weight, b = (torch.randn(channels, width, generator=g) * 0.5).bfloat16().cuda(), torch.randn(channels, generator=g).bfloat16().cuda() if bias else None
    tail = torch.randn(slots, width - 1, channels, generator=g).bfloat16().cuda()
    slot = torch.randperm(slots, generator=g)[:seqs].int()
    for s, value in lost:
        slot[s] = value
    x, slot_d, was = x.cuda(), slot.cuda(), f64(tail.float())
    out = torch.full((tokens, channels + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    cu = ends(lens, front)
    k = torch.tensor(kept, dtype=torch.int32, device="cuda") if kept else None
    ctx.gdn_conv(x.data_ptr(), channels + more, weight.data_ptr(), tail.data_ptr(), slots, out.data_ptr(), channels + 8, tokens, seqs, channels, width,
                 bias=b.data_ptr() if bias else None, slot=slot_d.data_ptr(), cu_q=cu.data_ptr() if packed else None, kept=k.data_ptr() if kept else None)
    torch.cuda.synchronize()
    got, now, xs = f64(out.float()), f64(tail.float()), f64(x.float())
    assert (got[:, channels:] == 7).all(), "between the rows"
    t, want_tail, written = front, was.copy(), np.zeros(tokens, bool)
    for s, n in enumerate(lens):
        p = int(slot[s])
        if 0 <= p < slots and n:
            r = xs[t:t + n, :channels]
            want, tol = convolved(r, was[p], f64(weight.float()), f64(b.float()) if bias else None)
            check(got[t:t + n, :channels], want, tol, f"rows of sequence {s}")
            take = n if not kept else min(max(kept[s], 0), n)
            want_tail[p] = np.concatenate((was[p], r[:take]))[take:]
            written[t:t + n] = True
        t += n
    assert np.array_equal(now, want_tail), "tails"
    assert (got[~written, :channels] == 7).all(), "rows of no sequence"


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels", [8, 520, 2048, 4104])
def test_conv_single_tokens(ctx, channels, width):
    say(f"conv of single tokens, {channels} channels, width {width}")
    conv_case(ctx, channels, width, [1] * 5, packed=False, bias=width == 3)
    conv_case(ctx, channels, width, [1] * 70, packed=False, lost=[(3, -1), (9, 72)], more=16)
    conv_case(ctx, channels, width, [1] * 3, packed=False, kept=[1, 0, 5])


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("lens", [[1], [2], [3], [4], [5], [64], [1, 2, 3, 4, 5, 0, 6], [0, 0, 7], [33, 1, 90], [300]])
def test_conv_packed_rows(ctx, lens, width):
    say(f"conv of rows {lens}, width {width}")
    conv_case(ctx, 264, width, lens, bias=True, front=2, behind=3, more=8)


@pytest.mark.parametrize("width", [2, 3, 4])
def test_conv_sequences_that_begin_at_any_place_of_a_run(ctx, width):
    say(f"conv across runs of rows, width {width}")
    for first in range(1, 19):
        conv_case(ctx, 2048, width, [first, 1, 2, 3, 500, 16, 15, 17, 1, 1, 600], seed=first)


def test_conv_many_sequences_drafted_rows_and_slots_outside(ctx):
    say("conv of 300 sequences")
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 9, 300).tolist()
    conv_case(ctx, 1032, 4, lens, behind=1)
    conv_case(ctx, 1032, 4, lens, kept=rng.integers(-1, 9, 300).tolist())
    conv_case(ctx, 1032, 3, lens, lost=[(7, -5), (100, 302), (299, 1 << 30)])


def test_conv_ends_past_the_rows(ctx):
    say("conv, an end past the call's rows")
    x = torch.randn(10, 64, device="cuda").bfloat16()
    w, tail, out = torch.randn(64, 4, device="cuda").bfloat16(), torch.zeros(2, 3, 64, dtype=torch.bfloat16, device="cuda"), torch.full((10, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 3, 99], dtype=torch.int32, device="cuda")
    ctx.gdn_conv(x.data_ptr(), 64, w.data_ptr(), tail.data_ptr(), 2, out.data_ptr(), 64, 8, 2, 64, 4, cu_q=cu.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(tail[1], x[5:8]) and torch.equal(tail[0], x[:3]) and (out[8:] == 7).all() and not (out[:8] == 7).any()


# ------------------------------------------------------------------ the rule

def workspace(r, max_q=None):
    n = iu8.gdn_workspace(r.tokens, r.seqs, max_q or max(r.lens), r.kh, r.heads)
    return torch.full((n,), 255, dtype=torch.uint8, device="cuda") if n else None      # (all ones: NaN in any type)


def rule_case(ctx, r, packed=True, kept=None, chunked=False, out=True, max_q=None):
    was = f64(r.state)
    k = torch.tensor(kept, dtype=torch.int32, device="cuda") if kept else None
    ws = workspace(r, max_q) if chunked else None
    assert (ws is not None) == chunked
    r.call(ctx, packed, max_q, k, ws, out)
    torch.cuda.synchronize()
    got, now = f64(r.out.float()), f64(r.state)
    left, rows = np.ones(r.slots, bool), np.ones(r.tokens, bool)
    for s, t, p, (want, tol, states, tols) in r.want(was, chunked):
        n = r.lens[s]
        take = n if not kept else min(max(kept[s], 0), n)
        if out:
            check(got[t:t + n], want, tol, f"rows of sequence {s}")
            rows[t:t + n] = False
        check(now[p], states[take], np.broadcast_to(tols[take], now[p].shape), f"state of sequence {s}")
        left[p] = False
        if not take:
            assert np.array_equal(now[p], was[p]), "a state that no row enters"
    assert np.array_equal(now[left], was[left]), "states of no sequence"
    assert (got[rows] == 7).all(), "rows of no sequence"


@pytest.mark.parametrize("kh,heads", [(1, 1), (2, 6), (4, 4), (3, 12)])
def test_rule_single_tokens(ctx, kh, heads):
    say(f"delta rule of single tokens, {heads} heads on {kh}")
    rule_case(ctx, Rows(kh, heads, [1] * 5, more=24), packed=False)
    r = Rows(kh, heads, [1] * 4)
    r.slot[1], r.slot[2] = -1, r.slots
    rule_case(ctx, r, packed=False)
    rule_case(ctx, Rows(kh, heads, [1] * 3), packed=False, kept=[1, 0, 2])


@pytest.mark.parametrize("lens", [[2], [8], [9], [17], [5, 0, 3, 1, 31], [0, 0, 4], [32, 32]])
def test_rule_few_rows(ctx, lens):
    say(f"delta rule a row at a time, {lens}")
    rule_case(ctx, Rows(2, 4, lens, front=1, behind=2, seed=sum(lens)))
    rule_case(ctx, Rows(2, 4, lens, behind=2, seed=sum(lens)), kept=[(3 * i + 2) % (n + 2) for i, n in enumerate(lens)])
    rule_case(ctx, Rows(2, 4, lens, behind=2, seed=sum(lens)), kept=[n - 1 for n in lens], out=False)
    rule_case(ctx, Rows(2, 4, lens, front=3, seed=sum(lens)), out=False)


@pytest.mark.parametrize("kh,heads,lens", [(16, 48, [5, 0, 3, 1, 17]), (2, 4, [(3 * i) % 11 for i in range(60)]), (1, 3, [9] * 50)])
def test_rule_few_rows_of_many_heads(ctx, kh, heads, lens):
    """More sequences and heads than waves of 16 columns are taken for."""
    say(f"delta rule a row at a time, {len(lens)} sequences of {heads} heads")
    rule_case(ctx, Rows(kh, heads, lens, front=1, behind=2, seed=1))
    rule_case(ctx, Rows(kh, heads, lens, more=8, seed=2), kept=[(3 * i + 2) % (n + 2) for i, n in enumerate(lens)])
    rule_case(ctx, Rows(kh, heads, lens, seed=3), out=False)
    rule_case(ctx, Rows(kh, heads, [1] * len(lens), seed=4), packed=False)


@pytest.mark.parametrize("lens", [[33], [63], [64], [65], [128], [129], [200, 1, 0, 64, 70], [0, 90, 0], [300], [40, 40, 40, 40]])
def test_rule_in_chunks(ctx, lens):
    say(f"delta rule in chunks, {lens}")
    rule_case(ctx, Rows(2, 4, lens, front=1, behind=2, more=8, seed=sum(lens)), chunked=True)
    rule_case(ctx, Rows(1, 3, lens, seed=sum(lens)), chunked=True)


@pytest.mark.parametrize("kh,heads,seqs", [(1, 1, 1), (16, 48, 1), (8, 24, 4), (16, 16, 12), (20, 60, 5)])
def test_rule_in_chunks_by_the_waves_of_a_workgroup(ctx, kh, heads, seqs):
    """Few heads and sequences, and more than the card holds at once."""
    say(f"delta rule in chunks, {seqs} sequences of {heads} heads")
    rule_case(ctx, Rows(kh, heads, [70 + 13 * i % 60 for i in range(seqs)], seed=seqs), chunked=True)


@pytest.mark.parametrize("seqs", [64, 65, 90])
def test_rule_in_chunks_of_many_sequences(ctx, seqs):
    """The longest are taken first where they are few; places of a batch that are idle, states that are nobody's."""
    say(f"delta rule in chunks, {seqs} sequences")
    r = Rows(1, 3, [(37 * i) % 71 for i in range(seqs - 1)] + [330], front=2, behind=3, seed=seqs)
    r.slot[5], r.slot[7] = -1, r.slots
    rule_case(ctx, r, chunked=True)


@pytest.mark.parametrize("kh,heads,seqs", [(8, 24, 45), (6, 30, 60), (7, 14, 50)])
def test_rule_in_chunks_whose_preparation_shares_a_key_head(ctx, kh, heads, seqs):
    """Two, three and five value heads on a key head, in workgroups of up to four of them."""
    say(f"delta rule in chunks, {seqs} sequences of {heads} heads on {kh}")
    rule_case(ctx, Rows(kh, heads, [33] + [3 + (5 * i) % 17 for i in range(seqs - 2)] + [66], seed=seqs), chunked=True)


@pytest.mark.parametrize("lens,heads", [([10], 4), ([11, 3], 4), ([14, 9], 96), ([15, 2], 96)])
def test_rule_by_its_longest_rows(ctx, lens, heads):
    """The recurrent kernel up to a length, the chunks past it, whatever a workspace was made for."""
    say(f"delta rule of {lens} rows, {heads} heads")
    r = Rows(1, heads, lens, seed=heads)
    ws = workspace(r, 64)
    was = f64(r.state)
    r.call(ctx, workspace=ws)
    torch.cuda.synchronize()
    for s, t, p, (want, tol, states, tols) in r.want(was, True):
        check(f64(r.out[t:t + r.lens[s]].float()), want, tol, f"rows of sequence {s}")
        check(f64(r.state[p]), states[-1], np.broadcast_to(tols[-1], states[-1].shape), f"state of sequence {s}")


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("like,a_at", [(0.0, 0.0), (1.0, -30.0), (0.9, -8.0), (0.0, 30.0), (0.5, 3000.0), (0.0, -3000.0)])
def test_rule_of_like_keys_and_any_decay(ctx, like, a_at, chunked):
    """Keys that are all the same on a state that keeps everything, where a chunk's system is furthest from the identity; decays that leave nothing."""
    say(f"delta rule, keys alike {like}, decays at {a_at}, chunked {chunked}")
    rule_case(ctx, Rows(1, 4, [150, 40], like=like, a_at=a_at, seed=11), chunked=chunked)


@pytest.mark.parametrize("chunked", [False, True])
def test_rule_after_a_row_that_clears_the_state(ctx, chunked):
    """One row of a decay of nothing among rows of weak ones: the later rows' decays keep their digits."""
    say(f"delta rule, a cleared state, chunked {chunked}")
    r = Rows(1, 2, [100], a_at=-2.0, seed=12)
    r.ab[[5, 6, 70], :r.heads] = 20000.0
    rule_case(ctx, r, chunked=chunked)


@pytest.mark.parametrize("chunked", [False, True])
def test_rule_of_zero_rows(ctx, chunked):
    say(f"delta rule, rows of zeros, chunked {chunked}")
    r = Rows(2, 4, [70], seed=13)
    r.rows[3:9] = 0
    r.rows[20] = -0.0
    rule_case(ctx, r, chunked=chunked)
    r = Rows(2, 4, [66], seed=14)
    r.rows.zero_(), r.state.zero_()
    rule_case(ctx, r, chunked=chunked)
    assert (r.out == 0).all() and (r.state == 0).all()


@pytest.mark.parametrize("chunked", [False, True])
def test_rule_ends_past_the_rows(ctx, chunked):
    """An end past the call's rows: those that are there, and none behind them."""
    say(f"delta rule, an end past the rows, chunked {chunked}")
    r = Rows(2, 2, [40, 50], seed=15)
    was = f64(r.state)
    r.call(ctx, workspace=workspace(r) if chunked else None, tokens=75)
    torch.cuda.synchronize()
    r.lens = [40, 35]
    for s, t, p, (want, tol, states, tols) in r.want(was, chunked):
        check(f64(r.out[t:t + r.lens[s]].float()), want, tol, f"rows of sequence {s}")
        check(f64(r.state[p]), states[-1], np.broadcast_to(tols[-1], states[-1].shape), f"state of sequence {s}")
    assert (r.out[75:] == 7).all()


def test_rule_answers_do_not_depend_on_the_run(ctx):
    say("delta rule twice")
    got = []
    for _ in range(2):
        r = Rows(16, 48, [500, 77], seed=16)
        r.call(ctx, workspace=workspace(r))
        torch.cuda.synchronize()
        got.append((r.out, r.state))
    assert torch.equal(got[0][0].view(torch.int16), got[1][0].view(torch.int16)) and torch.equal(got[0][1], got[1][1])


def test_rule_workspace_of_the_largest_call_serves_smaller_ones(ctx):
    say("delta rule, one workspace")
    big = iu8.gdn_workspace(1000, 20, 1000, 2, 4)
    ws = torch.full((big,), 255, dtype=torch.uint8, device="cuda")
    for lens in ([1000], [50] * 20, [3, 0, 70], [981] + [1] * 19):
        assert iu8.gdn_workspace(sum(lens), len(lens), max(lens), 2, 4) <= big
        r = Rows(2, 4, lens, seed=17)
        was = f64(r.state)
        r.call(ctx, workspace=ws)
        torch.cuda.synchronize()
        for s, t, p, (want, tol, states, tols) in r.want(was, True):
            check(f64(r.out[t:t + lens[s]].float()), want, tol, f"rows of sequence {s}")
            check(f64(r.state[p]), states[-1], np.broadcast_to(tols[-1], states[-1].shape), f"state of sequence {s}")


def test_drafted_rows_and_the_accepted_ones(ctx):
    """A verify step answers all rows and moves no state; the accepted rows then count: as if they alone had come."""
    say("delta rule, drafted rows")
    lens, take = [5, 3, 0, 5], [2, 3, 0, 0]
    r, none = Rows(2, 4, lens, seed=18), torch.zeros(4, dtype=torch.int32, device="cuda")
    was = r.state.clone()
    r.call(ctx, kept=none)
    torch.cuda.synchronize()
    first = r.out.clone()
    assert torch.equal(r.state, was)
    r.call(ctx, kept=torch.tensor(take, dtype=torch.int32, device="cuda"), out=False)
    torch.cuda.synchronize()
    alone = Rows(2, 4, lens, seed=18)
    r2, t = [], 0
    for n, k in zip(lens, take):
        r2 += list(range(t, t + k))
        t += n
    alone.rows, alone.ab, alone.lens, alone.cu, alone.tokens = alone.rows[r2].contiguous(), alone.ab[r2].contiguous(), take, ends(take), len(r2)
    alone.call(ctx)
    torch.cuda.synchronize()
    assert torch.equal(r.state, alone.state)
    assert torch.equal(first[r2].view(torch.int16), alone.out[:len(r2)].view(torch.int16))


# ------------------------------------------------------------------ captured, on another stream

def test_captured_calls_follow_rows_slots_and_kept(ctx):
    say("delta-net core, captured")
    kh, heads, seqs, tokens = 2, 4, 3, 140
    channels = (2 * kh + heads) * D
    g = torch.Generator().manual_seed(19)
    proj = torch.randn(tokens, channels + 64, generator=g).bfloat16().cuda()
    r = Rows(kh, heads, [100, 0, 40], slots=6, seed=19)
    r.row, r.rows = channels, torch.zeros(tokens, channels, dtype=torch.bfloat16, device="cuda")
    w = (torch.randn(channels, 4, generator=g) * 0.5).bfloat16().cuda()
    tail, ws = torch.zeros(6, 3, channels, dtype=torch.bfloat16, device="cuda"), workspace(r, 140)
    src, dst = (torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()

    def step(stream):
        ctx.gdn_conv(proj.data_ptr(), channels + 64, w.data_ptr(), tail.data_ptr(), 6, r.rows.data_ptr(), channels, tokens, seqs, channels, 4, slot=r.slot.data_ptr(),
                     cu_q=r.cu.data_ptr(), stream=stream)
        r.call(ctx, max_q=140, workspace=ws, stream=stream)
        ctx.gdn_copy(r.state.data_ptr(), tail.data_ptr(), 6, heads, channels, 4, src.data_ptr(), dst.data_ptr(), 2, stream=stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for i, (lens, slot, pairs) in enumerate([([100, 0, 40], [5, 1, 0], [(5, 3), (0, 2)]), ([1, 64, 65], [3, 1, 2], [(1, 0), (9, 4)]), ([0, 0, 140], [0, 1, 4], [(4, 4), (-1, 0)]),
                                             ([139, 1, 0], [5, 4, 3], [(3, 1), (2, 6)])]):
        proj.copy_(torch.randn(proj.shape, generator=g).bfloat16())
        r.cu.copy_(ends(lens)), r.slot.copy_(torch.tensor(slot)), src.copy_(torch.tensor([p[0] for p in pairs])), dst.copy_(torch.tensor([p[1] for p in pairs]))
        before, tails = r.state.clone(), tail.clone()
        r.out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (r.out, r.state, tail)]
        r.state.copy_(before), tail.copy_(tails), r.out.fill_(7)
        step(0)
        torch.cuda.synchronize()
        for x, y, what in zip(got, (r.out, r.state, tail), ("rows", "states", "tails")):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16)), (i, what)


def test_calls_at_once_with_workspaces_of_their_own(ctx):
    """Two batches on two streams, their launches alternating: the bytes of one after the other."""
    say("delta rule, two calls at once")
    def batch(i):
        return Rows(2, 6, [150 + 40 * i, 3, 70], seed=30 + i)
    want = []
    for i in range(2):
        r = batch(i)
        for _ in range(4):
            r.call(ctx, workspace=workspace(r))
        torch.cuda.synchronize()
        want.append((r.out, r.state))
    both, streams = [batch(i) for i in range(2)], [torch.cuda.Stream() for _ in range(2)]
    spaces = [workspace(r) for r in both]
    torch.cuda.synchronize()
    for _ in range(4):
        for r, ws, stream in zip(both, spaces, streams):
            r.call(ctx, workspace=ws, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for r, (out, state) in zip(both, want):
        assert torch.equal(r.out, out) and torch.equal(r.state, state)


def test_calls_on_another_stream_follow_its_order(ctx):
    say("delta-net core on a side stream")
    r, side = Rows(2, 4, [200, 30], seed=20), torch.cuda.Stream()
    want = Rows(2, 4, [200, 30], seed=20)
    want.call(ctx, workspace=workspace(want))
    torch.cuda.synchronize()
    rows = r.rows.clone()
    r.rows.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        busy = torch.randn(4096, 4096, device="cuda") @ torch.randn(4096, 4096, device="cuda")
        r.rows.copy_(rows)
        r.call(ctx, workspace=workspace(r), stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert busy.isfinite().all() and torch.equal(r.out.view(torch.int16), want.out.view(torch.int16)) and torch.equal(r.state, want.state)


# ------------------------------------------------------------------ copies

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("page,kvh,dim", [(16, 1, 64), (64, 4, 256), (256, 3, 128), (32, 5, 64)])
def test_pages_copied(ctx, page, kvh, dim, e4m3):
    say(f"pages of {page} tokens, {kvh} heads of {dim}, e4m3 {e4m3}")
    pages, g = 40, torch.Generator().manual_seed(page)
    size = iu8.kv_bytes(pages, kvh, dim, page, iu8.KV_E4M3 if e4m3 else iu8.KV_BF16)
    k, v = (torch.randint(0, 256, (pages, size // pages), generator=g, dtype=torch.uint8).cuda() for _ in range(2))
    some = torch.zeros(8, dtype=torch.int32, device="cuda")
    one = torch.ones(kvh, device="cuda")
    c = iu8.KvCache.of(k.data_ptr(), v.data_ptr(), some.data_ptr(), some.data_ptr(), kv_heads=kvh, head_dim=dim, page_tokens=page, pages=pages, table_stride=4,
                       kind=iu8.KV_E4M3 if e4m3 else iu8.KV_BF16, k_scale=one.data_ptr(), v_scale=one.data_ptr())
    src = torch.tensor([3, 3, 39, -1, 4, 40, 5, 7, 0], dtype=torch.int32, device="cuda")
    dst = torch.tensor([10, 11, 0, 12, 40, 13, -3, 7, 20], dtype=torch.int32, device="cuda")
    want = [x.clone() for x in (k, v)]
    for x in want:
        x[[10, 11, 0]] = x[[3, 3, 39]]
    ctx.kv_copy(c, src.data_ptr(), dst.data_ptr(), 8)
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    ctx.kv_copy(c, src.data_ptr(), dst.data_ptr(), 0)
    torch.cuda.synchronize()
    assert torch.equal(k, want[0])


def test_states_copied_and_offsets_past_32_bits(ctx):
    say("states copied, a pool of more than 4 GiB")
    heads, channels, slots = 48, 10240, 1500                       # 3 MiB a state
    state, tail = torch.empty(slots, heads, D, D, device="cuda"), torch.empty(slots, 3, channels, dtype=torch.bfloat16, device="cuda")
    assert state.numel() * 4 > 1 << 32
    for s in (0, 1, 700, 1498, 1499):
        state[s], tail[s] = torch.randn(heads, D, D, device="cuda"), torch.randn(3, channels, device="cuda")
    src, dst = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1499, 1499], [1490, 3, 1400]))
    ctx.gdn_copy(state.data_ptr(), tail.data_ptr(), slots, heads, channels, 4, src.data_ptr(), dst.data_ptr(), 3)
    torch.cuda.synchronize()
    for a, b in ((0, 1490), (1499, 3), (1499, 1400)):
        assert torch.equal(state[a], state[b]) and torch.equal(tail[a], tail[b])
    # the rule and the convolution on its last slot
    r = Rows(16, 48, [70], slots=1, seed=21)
    was = f64(state[1499][None])
    r.state, r.slots, r.slot = state, slots, torch.tensor([1499], dtype=torch.int32, device="cuda")
    r.call(ctx, workspace=workspace(r))
    torch.cuda.synchronize()
    for _, t, p, (want, tol, states, tols) in r.want({1499: was[0]}, True):
        check(f64(r.out.float()), want, tol, "rows")
        check(f64(state[p]), states[-1], np.broadcast_to(tols[-1], states[-1].shape), "state")


@pytest.mark.parametrize("chunked", [False, True])
def test_states_past_32_bits_are_the_same_states(ctx, chunked):
    """The last slots of a pool past 4 GiB answer and are left as the same ones of a small pool, byte for byte."""
    say(f"delta rule on states past 4 GiB, chunked {chunked}")
    small, large = (Rows(1, 1, [70, 3], slots=2, seed=21) for _ in range(2))
    small.slot.copy_(torch.arange(2))
    first = 70000 - 2
    pool = torch.zeros((first + 2, 1, 128, 128), dtype=torch.float32, device="cuda")
    pool[first:] = large.state
    large.state, large.slots = pool, first + 2
    large.slot.copy_(torch.arange(first, first + 2))
    for r in (small, large):
        r.call(ctx, workspace=workspace(r) if chunked else None)
    torch.cuda.synchronize()
    assert torch.equal(small.out, large.out) and torch.equal(small.state, pool[first:]) and not pool[:first].any()


def test_tails_past_32_bits_are_the_same_tails(ctx):
    say("convolution on tails past 4 GiB")
    channels, width, first = 384, 4, 2_000_000
    g = torch.Generator().manual_seed(22)
    x, weight = torch.randn(9, channels, generator=g).bfloat16().cuda(), torch.randn(channels, width, generator=g).bfloat16().cuda()
    small = torch.randn(2, width - 1, channels, generator=g).bfloat16().cuda()
    large = torch.zeros((first + 2, width - 1, channels), dtype=torch.bfloat16, device="cuda")
    large[first:] = small
    outs, cu = [], ends([7, 2])
    for tail, at in ((small, 0), (large, first)):
        slot = torch.arange(at, at + 2, dtype=torch.int32, device="cuda")
        outs.append(torch.zeros(9, channels, dtype=torch.bfloat16, device="cuda"))
        ctx.gdn_conv(x.data_ptr(), channels, weight.data_ptr(), tail.data_ptr(), len(tail), outs[-1].data_ptr(), channels, 9, 2, channels, width,
                     slot=slot.data_ptr(), cu_q=cu.data_ptr())
        torch.cuda.synchronize()
    assert torch.equal(*outs) and torch.equal(small, large[first:]) and not large[:first].any()
