"""GPU tests of the paged key/value cache and the attention that reads it (code object `attn_paged`), through the C ABI, against
their definitions in 64 bits (attn_util.py, which derives the tolerances)."""
import math

import numpy as np
import pytest
import torch

from oracle import ref
from saber_engine_amd import iu8, synth
from saber_engine_amd.attn import AttnLayerIU8, PagedKvCache
from tests.attn_util import BF16, E4M3, Paged, Workspace, attention, check, f64, random_rows
from tests.gpu_util import dev_bf16_bits, dev_f32, dev_u8, host_u16, say

pytestmark = pytest.mark.gpu


def ends(lens):
    return torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ append

def normed(x, w, eps):
    return x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 + f64(w))


def rotated(x, pos, freq, rot, interleaved):
    y = x.copy()
    if rot:
        ang = pos[:, None, None] * freq
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        y[..., a] = x[..., a] * np.cos(ang) - x[..., b] * np.sin(ang)
        y[..., b] = x[..., b] * np.cos(ang) + x[..., a] * np.sin(ang)
    return y


def append_case(ctx, dim, heads, kvh, lens, news, page=32, rot=0, interleaved=False, gated=False, norm=False, e4m3=False, packed=True, behind=0,
                hole=False, apart=False, seed=1):
    seqs = len(lens)
    g = torch.Generator().manual_seed(seed)
    c = Paged(seqs, kvh, dim, page, max(max(lens), 1), e4m3, seed, pages=None if max(lens) < 5000 else 4096 if seqs == 1 else None)
    c.kv_len.copy_(torch.tensor(lens))
    if hole:
        c.table[0, -1] = -1
        c.table[1, 0] = c.pages
    tokens = sum(news) + behind
    step = 2 * dim if gated else dim
    wide = heads * step + 2 * kvh * dim + (64 if apart else 0)
    rows = random_rows(g, tokens, wide)
    kv = random_rows(g, tokens, 2 * kvh * dim + 8) if apart else None
    qn, kn = ((torch.randn(dim, generator=g) * 0.2).bfloat16().cuda() if norm else None for _ in range(2))
    freq = torch.tensor([1e6 ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64).cuda() if rot else None
    q_out = torch.full((tokens, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    k0, v0 = c.k.clone(), c.v.clone()
    cu = ends(news) if packed else None
    kp = kv.data_ptr() if apart else rows.data_ptr() + 2 * heads * step
    ctx.kv_append(rows.data_ptr(), kp, kp + 2 * kvh * dim, q_out.data_ptr(), c.desc(), cu.data_ptr() if packed else None, tokens, seqs, heads, wide, step,
                  kv.shape[1] if apart else wide, freq.data_ptr() if rot else None, rot, interleaved, qn.data_ptr() if norm else None,
                  kn.data_ptr() if norm else None, 1e-6)
    torch.cuda.synchronize()
    x = f64(rows.float())
    src = f64(kv.float()) if apart else x[:, heads * step:]
    fr = f64(freq) if rot else None
    written = torch.zeros(c.pages, kvh, page, dtype=torch.bool)
    t = 0
    for s, n in enumerate(news):
        for i in range(n):
            pos = lens[s] - n + i
            if pos < 0:
                assert (q_out[t] == 7).all(), "a row of no position"
                t += 1
                continue
            at = np.array([pos])
            part = x[t:t + 1]
            q = np.stack([part[:, h * step:h * step + dim] for h in range(heads)], 1)
            k = src[t:t + 1, :kvh * dim].reshape(1, kvh, dim)
            q0, k0_ = normed(q, qn, 1e-6), normed(k, kn, 1e-6)
            q, k = rotated(q0, at, fr, rot, interleaved), rotated(k0_, at, fr, rot, interleaved)
            # f32: 1e-6 of the pair's magnitude for sine, cosine and their angle's fraction, 1e-5 relative for the norm
            slack = lambda y: 1.5e-5 * (np.abs(y).max(-1, keepdims=True) + 1e-30)  # noqa: E731
            check(f64(q_out[t:t + 1].float()), q, np.abs(q) * BF16 * 1.01 + slack(q0), f"q of row {t}")
            p = int(c.table[s, pos // page])
            if 0 <= p < c.pages:
                o = pos % page
                written[p, :, o] = True
                gk = f64(c.raw(c.k)[p, :, o // 16, :, o % 16].reshape(kvh, dim).view(c.kind).float())
                gv = c.raw(c.v)[p, :, o].view(c.kind)
                v = src[t, kvh * dim:2 * kvh * dim].reshape(kvh, dim)
                if e4m3:
                    ks, vs = f64(c.scales[0])[:, None], f64(c.scales[1])[:, None]
                    for got, want, more in ((gk, k[0] / ks, slack(k0_[0] / ks)), (f64(gv.float()), v / vs, 1e-6 * np.abs(v / vs))):
                        want = np.clip(want, -448, 448)
                        check(got, want, np.abs(want) * E4M3 * 1.01 + 2.0 ** -10 + more, f"cache of row {t}")
                else:
                    check(gk, k[0], np.abs(k[0]) * BF16 * 1.01 + slack(k0_[0]), f"k of row {t}")
                    assert np.array_equal(f64(gv.float()), v), f"v of row {t}"
            t += 1
    assert (q_out[t:] == 7).all(), "rows behind the last sequence"
    left = ~written.cuda()
    kk = c.raw(c.k).permute(0, 1, 2, 4, 3, 5).reshape(c.pages, kvh, page, dim)
    k_was = c.raw(k0).permute(0, 1, 2, 4, 3, 5).reshape(c.pages, kvh, page, dim)
    assert torch.equal(kk[left], k_was[left]) and torch.equal(c.raw(c.v)[left], c.raw(v0)[left]), "tokens that no row belongs to"


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh", [(64, 7, 1), (128, 40, 8), (256, 24, 4), (256, 3, 3), (64, 1, 1)])
def test_append_single_tokens(ctx, dim, heads, kvh, e4m3):
    say(f"append one token a sequence {dim} {heads} {kvh} {e4m3}")
    lens = [1, 37, 0, 64, 65, 200]
    append_case(ctx, dim, heads, kvh, lens, [1] * 6, rot=dim // 4, gated=dim == 256, norm=dim == 256, e4m3=e4m3, packed=False)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot,page,norm,e4m3", [(64, 64, 16, True, False), (64, 16, 256, False, True), (128, 0, 64, True, True), (128, 128, 128, False, False),
                                                    (128, 96, 16, True, False), (256, 64, 32, True, True), (256, 256, 64, False, False)])
def test_append_packed_rows(ctx, dim, rot, page, norm, e4m3, interleaved):
    say(f"append packed {dim} rot {rot} page {page} {norm} {e4m3} {interleaved}")
    append_case(ctx, dim, 6, 2, [5, 70, 3, 0, 19], [5, 33, 0, 0, 17], page=page, rot=rot, interleaved=interleaved, norm=norm, e4m3=e4m3, behind=3, apart=norm)


def test_append_more_rows_than_positions_and_holes(ctx):
    say("append: rows of no position, holes in the table")
    append_case(ctx, 128, 4, 2, [3, 20, 40], [5, 20, 2], page=16, rot=32, behind=1)
    append_case(ctx, 128, 4, 2, [40, 40, 40], [12, 40, 2], page=16, rot=32, hole=True)


def test_append_at_far_positions(ctx):
    say("append: positions of a million")
    append_case(ctx, 128, 2, 1, [1048569], [9], page=256, rot=128)
    append_case(ctx, 128, 2, 1, [1048576], [3], page=256, rot=128, interleaved=True, e4m3=True)


def test_append_among_many_sequences(ctx):
    say("append: 200 packed sequences")
    rng = np.random.default_rng(4)
    news = rng.integers(0, 4, 200).tolist()
    append_case(ctx, 64, 2, 1, [n + int(rng.integers(0, 30)) for n in news], news, page=16, rot=32, behind=2)


def test_append_saturates_and_keeps_nan(ctx):
    say("append: values past e4m3's range, NaN")
    c = Paged(1, 1, 64, 16, 16, True, fill=0.0)
    c.scales = [torch.tensor([0.001], device="cuda"), torch.tensor([0.001], device="cuda")]
    c.kv_len[0] = 1
    rows = torch.zeros(1, 3 * 64, dtype=torch.bfloat16, device="cuda")
    rows[0, 64:68] = torch.tensor([1e3, -1e3, float("nan"), float("inf")])
    rows[0, 128:132] = torch.tensor([float("-inf"), 0.448, -0.4, float("nan")])
    q_out = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    p = rows.data_ptr()
    ctx.kv_append(p, p + 128, p + 256, q_out.data_ptr(), c.desc(), None, 1, 1, 1, 192, 64, 192)
    torch.cuda.synchronize()
    page = int(c.table[0, 0])
    k = c.k[page, 0, 0, 0, 0, :4].float().cpu().numpy()
    v = c.v[page, 0, 0, :4].float().cpu().numpy()
    assert k[0] == 448 and k[1] == -448 and np.isnan(k[2]) and k[3] == 448
    assert v[0] == -448 and v[1] == 448 and v[2] == -416 and np.isnan(v[3])    # -400: a tie's even side is -384, bf16(-0.4) lies past it


# ------------------------------------------------------------------ attention

def attn_case(ctx, dim, heads, kvh, lens, news, page=64, e4m3=False, packed=True, behind=0, max_kv=None, split=True, seed=2, holes=(), scale=None,
              stretch=1.0, wide=0, spoil=None, stream=None):
    seqs, most = len(lens), max(max(lens), 1)
    g = torch.Generator().manual_seed(seed)
    c = Paged(seqs, kvh, dim, page, most, e4m3, seed)
    c.kv_len.copy_(torch.tensor(lens))
    for s, n in enumerate(lens):
        if n:
            c.put(s, 0, random_rows(g, n, kvh, dim, e4m3=e4m3), random_rows(g, n, kvh, dim, e4m3=e4m3))
    for s, p, to in holes:
        c.table[s, p] = to
    if spoil:
        spoil(c)
    tokens = sum(news) + behind
    row = heads * dim + wide
    q = (random_rows(g, tokens, row).float() * stretch).bfloat16()
    out = torch.full((tokens, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    cu = ends(news) if packed else None
    max_q = max(max(news), 1)
    ws = Workspace(seqs, max_q, most if max_kv is None else max_kv, heads, kvh, dim)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    again = []
    for _ in range(2):
        torch.cuda.synchronize()
        ctx.attn(q.data_ptr(), row, c.desc(), cu.data_ptr() if packed else None, out.data_ptr(), tokens, seqs, max_q, most if max_kv is None else max_kv,
                 heads, scale, *(ws.args() if split else (None, None)), stream=stream.cuda_stream if stream else 0)
        torch.cuda.synchronize()
        again.append(out.clone())
        assert ws.counter is None or not ws.counter.any(), "the counters are left zero"
    assert torch.equal(again[0].view(torch.int16), again[1].view(torch.int16)), "the same bytes on every run"
    t = 0
    x = f64(q[:, :heads * dim].float()).reshape(tokens, heads, dim)
    for s, n in enumerate(news):
        k, v, there = c.rows(s, lens[s])
        want, tol = attention(x[t:t + n], k, v, there, scale)
        check(f64(out[t:t + n].float()), want, tol, f"sequence {s} ({n} of {lens[s]})")
        t += n
    assert (out[t:] == 7).all(), "rows behind the last sequence"
    return c, q, out


KINDS = [(64, 8, 8), (64, 14, 2), (128, 5, 1), (128, 16, 1), (256, 10, 2), (256, 4, 4)]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh", KINDS + [(128, 32, 1)])
def test_attn_single_tokens(ctx, dim, heads, kvh, e4m3):
    say(f"attn, one token a sequence {dim} {heads} {kvh} {e4m3}")
    attn_case(ctx, dim, heads, kvh, [1, 0, 31, 32, 33, 500, 129, 16], [1] * 8, page=16 if dim == 64 else 64, e4m3=e4m3, packed=False)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh,new", [(64, 2, 2, 16), (64, 2, 2, 29), (128, 5, 1, 3), (128, 10, 2, 6), (256, 6, 1, 5), (256, 8, 2, 4)])
def test_attn_few_rows(ctx, dim, heads, kvh, new, e4m3):
    say(f"attn, few rows {dim} {heads} {kvh} {new} {e4m3}")
    attn_case(ctx, dim, heads, kvh, [new, 300, 64 + new, 2, 0, 77], [new, new, max(1, new - 2), 2, 0, 1], page=32, e4m3=e4m3, behind=2)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh", KINDS)
def test_attn_many_rows(ctx, dim, heads, kvh, e4m3):
    say(f"attn, many rows {dim} {heads} {kvh} {e4m3}")
    news = [70, 1, 0, 33, 129]
    attn_case(ctx, dim, heads, kvh, [70, 40, 0, 133, 129], news, page=16 if dim == 128 else 128, e4m3=e4m3, behind=3)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("dim,heads,kvh,lens,news", [
    (128, 5, 1, [3001, 129, 5], [1, 1, 1]), (256, 6, 1, [4099], [5]), (64, 4, 1, [2600, 700], [40, 50]), (256, 10, 2, [1900], [90]), (128, 16, 2, [1500], [64])])
def test_attn_split_over_the_cache(ctx, dim, heads, kvh, lens, news, split):
    say(f"attn, split {dim} {heads} {kvh} {lens} {news} {split}")
    assert iu8.attn_workspace(len(lens), max(news), max(lens), heads, kvh, dim)[0] > 0
    attn_case(ctx, dim, heads, kvh, lens, news, split=split)


@pytest.mark.parametrize("news", [[1, 1], [50, 3]])
def test_attn_longer_than_told(ctx, news):
    say(f"attn, kv_len past max_kv {news}")
    attn_case(ctx, 128, 4, 2, [2000, 700], news, max_kv=600, page=32)
    attn_case(ctx, 128, 4, 2, [2000, 700], news, max_kv=0, page=32)


@pytest.mark.parametrize("news", [[1, 1, 1], [4, 1, 2], [40, 60, 3]])
def test_attn_holes_rows_of_no_key_and_strided_rows(ctx, news):
    say(f"attn, holes and more rows than keys {news}")
    attn_case(ctx, 64, 4, 2, [90, 60, 1], news, page=16, holes=[(0, 1, -1), (0, 5, 1 << 30), (1, 0, -5), (1, 1, -1), (1, 2, -1), (1, 3, -1), (2, 0, -1)], wide=24)
    if news[0] > 1:
        attn_case(ctx, 128, 4, 2, [2, 20, 1], [news[0] + 2, news[1], 3], page=16, wide=8)


@pytest.mark.parametrize("news", [[1], [40]])
def test_attn_sharp_flat_and_turned_scores(ctx, news):
    say(f"attn, scores of hundreds, equal scores, negative scale {news}")
    attn_case(ctx, 128, 4, 2, [333], news, stretch=8.0)
    attn_case(ctx, 128, 4, 2, [333], news, stretch=0.0)
    attn_case(ctx, 128, 4, 2, [333], news, scale=-0.2)
    attn_case(ctx, 128, 4, 2, [333], news, scale=0.0)


def test_attn_on_a_side_stream(ctx):
    say("attn on another stream")
    attn_case(ctx, 128, 8, 2, [900, 40], [1, 1], stream=torch.cuda.Stream())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh,news", [(64, 4, 2, [8]), (128, 3, 1, [5]), (256, 6, 2, [10]), (128, 1, 1, [2])])
def test_attn_values_that_are_not_finite_where_a_row_does_not_look(ctx, dim, heads, kvh, news, e4m3):
    """The last new tokens' keys and values are NaN (and infinite): the rows before them give what they give without, the last
    ones, which see them, NaN."""
    say(f"attn, NaN ahead {dim} {heads} {kvh} {news} {e4m3}")
    n, total = news[0], 75
    last = n - 1

    def spoil(c):
        bad = torch.full((1, kvh, dim), float("nan")).cuda()
        if not e4m3:
            bad[:, :, ::2] = float("inf")
        c.put(0, total - 1, bad.to(c.kind), bad.to(c.kind))

    clean = attn_case(ctx, dim, heads, kvh, [total], news, page=16, e4m3=e4m3)[2]
    c = Paged(1, kvh, dim, 16, total, e4m3, 2)
    g = torch.Generator().manual_seed(2)
    c.kv_len[0] = total
    c.put(0, 0, random_rows(g, total, kvh, dim, e4m3=e4m3), random_rows(g, total, kvh, dim, e4m3=e4m3))
    spoil(c)
    q = random_rows(g, n, heads * dim)
    out = torch.zeros_like(clean)
    ctx.attn(q.data_ptr(), heads * dim, c.desc(), ends(news).data_ptr(), out.data_ptr(), n, 1, n, total, heads, 1 / math.sqrt(dim))
    torch.cuda.synchronize()
    k, v, there = c.rows(0, total - 1)
    want, tol = attention(f64(q[:last].float()).reshape(last, heads, dim), k, v, there, 1 / math.sqrt(dim))
    check(f64(out[:last].float()), want, tol, "rows before the NaN")
    assert torch.isnan(out[last]).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("most_new", [1, 3])
def test_attn_among_many_sequences(ctx, most_new, e4m3):
    """More sequences than a wave has lanes, ragged, idle ones and empty ones among them: the deal of the units."""
    say(f"attn, 150 sequences of up to {most_new} rows {e4m3}")
    rng = np.random.default_rng(most_new)
    lens = [int(x) for x in rng.integers(0, 500, 150)]
    news = [int(x) for x in rng.integers(0, most_new + 1, 150)]
    lens[7], news[7], lens[149], news[149], news[0] = 0, most_new, 3, 2, 0
    attn_case(ctx, 64, 4, 2, lens, news, page=32, e4m3=e4m3, behind=1)


@pytest.mark.parametrize("dim,heads,kvh,total,new", [(64, 4, 1, 40000, 1), (64, 20, 1, 30000, 1), (64, 8, 2, 20000, 40), (128, 2, 1, 16500, 1)])
def test_attn_as_many_parts_as_a_join_holds(ctx, dim, heads, kvh, total, new):
    say(f"attn, one long sequence {dim} {heads} {kvh} {total} {new}")
    attn_case(ctx, dim, heads, kvh, [total], [new], page=256)


@pytest.mark.parametrize("dim,heads,kvh,total,new", [(64, 5, 1, 1500, 9), (128, 4, 2, 2100, 33), (256, 6, 1, 1100, 15)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_attn_row_tiles_of_the_few_row_kernels(ctx, dim, heads, kvh, total, new, e4m3):
    say(f"attn, {new} rows of group {heads // kvh} behind {total} keys {e4m3}")
    attn_case(ctx, dim, heads, kvh, [total, 40, 1300], [new, new - 1, 1], e4m3=e4m3)


@pytest.mark.parametrize("dim,heads,kvh,lens,news", [
    (64, 200, 1, [300, 41], [1, 2]), (64, 300, 300, [70, 1, 150], [1, 1, 1]), (64, 2, 2, [20 + i % 50 for i in range(300)], [20 + i % 17 for i in range(300)])])
def test_attn_wide_groups_many_heads_many_prompts(ctx, dim, heads, kvh, lens, news):
    say(f"attn, {heads} heads on {kvh}, {len(lens)} sequences")
    attn_case(ctx, dim, heads, kvh, lens, news, page=16, e4m3=kvh == 300)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 40])
def test_attn_over_pages_that_sequences_share(ctx, new, e4m3):
    """A prefix that lies in the same pages for every sequence, the rest in pages of its own."""
    say(f"attn, a shared prefix, {new} new rows {e4m3}")
    def share(c):
        c.table[1, :3] = c.table[0, :3]
        c.table[2, :2] = c.table[0, :2]
    attn_case(ctx, 128, 4, 2, [150, 170, 100], [new] * 3, page=32, e4m3=e4m3, spoil=share)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attn_lengths_around_a_tile(ctx, dim, e4m3):
    """Prompts that end one before, at and behind a tile (32 and 64 tokens), a row tile (128 rows) and a page."""
    say(f"attn, lengths around a tile {dim} {e4m3}")
    lens = [31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 193]
    attn_case(ctx, dim, 2, 1, lens, lens, page=16, e4m3=e4m3)
    attn_case(ctx, dim, 2, 1, [x + 100 for x in lens], lens, page=128, e4m3=e4m3)


def test_attn_one_workspace_for_every_smaller_call(ctx):
    """Workspaces of the largest call, smaller ones in them, with what lies behind them looked at."""
    say("attn, shared workspaces")
    heads, kvh, dim, seqs, most = 4, 2, 64, 6, 4000
    pb, cb = iu8.attn_workspace(seqs, 70, most, heads, kvh, dim)
    partial, counter = torch.full((pb // 4 + 64,), 3.0, device="cuda"), torch.zeros(cb // 4 + 64, dtype=torch.int32, device="cuda")
    counter[cb // 4:] = 5
    g = torch.Generator().manual_seed(8)
    c = Paged(seqs, kvh, dim, 64, most, fill=0.0)
    for s in range(seqs):
        c.put(s, 0, random_rows(g, most, kvh, dim), random_rows(g, most, kvh, dim))
    for n_seqs, new, total in ((6, 70, 4000), (1, 1, 4000), (6, 1, 4000), (2, 9, 3000), (1, 70, 4000), (3, 40, 700), (6, 5, 129), (1, 33, 2000)):
        c.kv_len[:n_seqs] = total
        tokens = n_seqs * new
        q, out = random_rows(g, tokens, heads * dim), torch.zeros(tokens, heads, dim, dtype=torch.bfloat16, device="cuda")
        ctx.attn(q.data_ptr(), heads * dim, c.desc(), ends([new] * n_seqs).data_ptr(), out.data_ptr(), tokens, n_seqs, new, total, heads, 0.125,
                 partial.data_ptr(), counter.data_ptr())
        torch.cuda.synchronize()
        assert (partial[pb // 4:] == 3).all() and (counter[cb // 4:] == 5).all() and not counter[:cb // 4].any(), (n_seqs, new, total)
        s = n_seqs - 1
        k, v, there = c.rows(s, total)
        want, tol = attention(f64(q[-new:].float()).reshape(new, heads, dim), k, v, there, 0.125)
        check(f64(out[-new:].float()), want, tol, f"{n_seqs} sequences of {new} rows on {total}")


@pytest.mark.parametrize("new", [1, 40])
def test_cache_past_four_gibibytes(ctx, new):
    """A pool of pages whose byte offsets pass 32 bits: append into its far end, attention over it."""
    say(f"cache of 5 GiB, {new} new rows")
    heads, kvh, dim, page, total, pages = 4, 1, 256, 256, 900, 40000
    g = torch.Generator().manual_seed(9)
    c = Paged(1, kvh, dim, page, total, pages=pages, fill=0.0)
    c.table[0] = torch.tensor([pages - 1, 3, 33000, pages - 2])
    assert iu8.kv_bytes(pages, kvh, dim, page) > 1 << 32
    c.put(0, 0, random_rows(g, total - new, kvh, dim), random_rows(g, total - new, kvh, dim))
    c.kv_len[0] = total
    row = heads * dim + 2 * dim
    x, q = random_rows(g, new, row), torch.zeros(new, heads, dim, dtype=torch.bfloat16, device="cuda")
    out, cu, p, ws = torch.zeros_like(q), ends([new]), x.data_ptr(), Workspace(1, new, total, heads, kvh, dim)
    ctx.kv_append(p, p + 2 * heads * dim, p + 2 * (heads + 1) * dim, q.data_ptr(), c.desc(), cu.data_ptr(), new, 1, heads, row, dim, row)
    ctx.attn(q.data_ptr(), heads * dim, c.desc(), cu.data_ptr(), out.data_ptr(), new, 1, new, total, heads, 1 / 16,
             *ws.args())
    torch.cuda.synchronize()
    assert torch.equal(q.view(new, -1), x[:, :heads * dim])
    k, v, there = c.rows(0, total)
    src = f64(x.float())
    assert np.array_equal(k[-new:, 0], src[:, heads * dim:-dim]) and np.array_equal(v[-new:, 0], src[:, -dim:])
    want, tol = attention(f64(q.float()), k, v, there, 1 / 16)
    check(f64(out.float()), want, tol, "rows on far pages")


def test_rows_in_front_of_the_first_sequence(ctx):
    """cu_q that does not begin at 0: the rows in front belong to nobody, in the cache as in the outputs."""
    say("rows in front of the first sequence")
    heads, kvh, dim, lens, news, front = 4, 2, 64, [30, 9], [4, 9], 3
    c = Paged(2, kvh, dim, 16, 32, fill=0.0)
    c.kv_len.copy_(torch.tensor(lens))
    g = torch.Generator().manual_seed(3)
    tokens, row = front + sum(news), (heads + 2 * kvh) * dim
    x = random_rows(g, tokens, row)
    q, out = (torch.full((tokens, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cu, p = ends(news) + front, x.data_ptr()
    ctx.kv_append(p, p + 2 * heads * dim, p + 2 * (heads + kvh) * dim, q.data_ptr(), c.desc(), cu.data_ptr(), tokens, 2, heads, row, dim, row)
    ctx.attn(q.data_ptr(), heads * dim, c.desc(), cu.data_ptr(), out.data_ptr(), tokens, 2, 9, 30, heads, 0.125)
    torch.cuda.synchronize()
    assert (q[:front] == 7).all() and (out[:front] == 7).all()
    t = front
    for s, n in enumerate(news):
        k, v, there = c.rows(s, lens[s])
        assert not k[:-n].any() and not v[:-n].any()
        assert np.array_equal(k[-n:].reshape(n, -1), f64(x[t:t + n, heads * dim:(heads + kvh) * dim].float()))
        want, tol = attention(f64(x[t:t + n, :heads * dim].float()).reshape(n, heads, dim), k, v, there, 0.125)
        check(f64(out[t:t + n].float()), want, tol, f"sequence {s}")
        t += n


def test_append_in_place(ctx):
    say("append: q_out is q")
    heads, kvh, dim, n = 6, 2, 128, 9
    freq = torch.tensor([1e4 ** (-i / 32) for i in range(32)], dtype=torch.float64).cuda()
    got = []
    for in_place in (False, True):
        c = Paged(1, kvh, dim, 32, n, fill=0.0)
        c.kv_len[0] = n
        q, kv = random_rows(torch.Generator().manual_seed(5), n, heads * dim), random_rows(torch.Generator().manual_seed(6), n, 2 * kvh * dim)
        to = q if in_place else torch.zeros_like(q)
        ctx.kv_append(q.data_ptr(), kv.data_ptr(), kv.data_ptr() + 2 * kvh * dim, to.data_ptr(), c.desc(), ends([n]).data_ptr(), n, 1, heads, heads * dim, dim,
                      2 * kvh * dim, freq.data_ptr(), 64)
        torch.cuda.synchronize()
        got.append((to, c.k, c.v))
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(*got))


# ------------------------------------------------------------------ the run of them

def layer(ctx, cache, tokens, max_q, gated, heads, hidden, weights, freq, **more):
    n = AttnLayerIU8(ctx, cache, tokens, heads, hidden, max_q=max_q, gated=gated, inv_freq=freq, **more)
    n.set_weights(*weights)
    return n


def layer_weights(heads, kvh, dim, hidden, gated, seed):
    n_core, n_qkv = heads * dim, heads * dim * (2 if gated else 1) + 2 * kvh * dim
    a, b = synth.dense_case(1, n_qkv, hidden, seed=seed), synth.dense_case(1, hidden, n_core, seed=seed + 1)
    rng = np.random.default_rng(seed + 2)
    t = rng.choice([-1.0, 1.0], size=n_core).astype(np.float32)
    norms = [torch.from_numpy(rng.standard_normal(dim).astype(np.float32) * 0.2).bfloat16().cuda() for _ in range(2)]
    host = dict(qkv=a, o=b, t=t, norms=norms)
    return host, (dev_u8(iu8.repack_w4(a["W"])), dev_f32(a["ws"]), dev_u8(iu8.repack_w4(b["W"])), dev_f32(b["ws"]), dev_f32(t) if gated else None, *norms)


def check_layer(n, host, x, news, before, kv):
    """Every step of a call from the one before it: the linears' bytes are the oracle's, what lies between them within the rounding."""
    cache, T, D = n.cache, n.T, n.cache.head_dim
    live = sum(news)
    qkv = host_u16(n.qkv)
    np.testing.assert_array_equal(qkv, ref.linear(x, host["qkv"]["W"], host["qkv"]["ws"], False, threads=8)["C"])
    rows = f64(n.qkv.view(torch.bfloat16).float())
    fr = f64(n.inv_freq)
    q = f64(n.q.view(torch.bfloat16).float()).reshape(T, n.heads, D)
    core = f64(n.core.view(torch.bfloat16).float()).reshape(T, n.heads, D)
    t = 0
    for s, new in enumerate(news):
        total = before[s] + new
        k, v, there = kv.rows(s, total)
        if new:
            pos = np.arange(before[s], total)
            x0 = rows[t:t + new]
            wq = normed(np.stack([x0[:, h * n.q_head:h * n.q_head + D] for h in range(n.heads)], 1), host["norms"][0], n.eps)
            wk = normed(x0[:, n.heads * n.q_head:][:, :kv.h * D].reshape(new, kv.h, D), host["norms"][1], n.eps)
            slack = lambda y: 1.5e-5 * (np.abs(y).max(-1, keepdims=True) + 1e-30)  # noqa: E731
            for got, want in ((q[t:t + new], wq), (k[before[s]:], wk)):
                turned = rotated(want, pos, fr, 2 * len(fr), n.interleaved)
                check(got, turned, np.abs(turned) * BF16 * 1.01 + slack(want), f"sequence {s}")
            assert np.array_equal(v[before[s]:], x0[:, n.heads * n.q_head + kv.h * D:].reshape(new, kv.h, D))
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


class Rows:
    """PagedKvCache's rows as attn_util's Paged gives them."""

    def __init__(self, c):
        self.h, d, page = c.kv_heads, c.head_dim, c.page_tokens
        self.p = Paged.__new__(Paged)
        self.p.h, self.p.dim, self.p.page, self.p.e4m3, self.p.e, self.p.pages, self.p.kind, self.p.table = self.h, d, page, False, 8, c.pages, torch.bfloat16, c.table
        self.p.k = c.k.view(torch.bfloat16).view(c.pages, self.h, page // 16, d // 8, 16, 8)
        self.p.v = c.v.view(torch.bfloat16).view(c.pages, self.h, page, d)

    def rows(self, s, n):
        return self.p.rows(s, n)


@pytest.mark.parametrize("gated,heads,kvh,dim,hidden,interleaved", [(True, 4, 1, 256, 512, False), (False, 8, 2, 128, 256, True)])
def test_layer_prompts_then_single_tokens(ctx, gated, heads, kvh, dim, hidden, interleaved):
    """Packed prompts of ragged lengths, a chunk behind them, then decode steps captured once and replayed while the counts and the page
    table change and eager work runs between; a prompt train of another graph beside it."""
    say(f"attention layer, gated {gated}, {heads} heads of {dim}")
    rng = np.random.default_rng(dim)
    host, weights = layer_weights(heads, kvh, dim, hidden, gated, 40 + dim)
    freq = torch.tensor([1e6 ** (-i / 32) for i in range(32)], dtype=torch.float64).cuda()
    cache = PagedKvCache(3, kvh, dim, 600, page_tokens=32)
    kv = Rows(cache)
    lens = [0, 0, 0]

    def prompt(news, T):
        n = layer(ctx, cache, T, max(news), gated, heads, hidden, weights, freq, interleaved=interleaved)
        x = synth.activations(rng, T, hidden)
        n.cu_q.copy_(ends(news))
        before = list(lens)
        for s, new in enumerate(news):
            lens[s] += new
            cache.reserve(s, lens[s])
        cache.kv_len.copy_(torch.tensor(lens))
        n.forward(dev_bf16_bits(x), max_kv=max(lens))
        torch.cuda.synchronize()
        check_layer(n, host, x, news, before, kv)

    prompt([70, 0, 200], 272)
    prompt([30, 129, 5], 164)
    n = layer(ctx, cache, 3, 1, gated, heads, hidden, weights, freq, interleaved=interleaved)
    x_dev = torch.zeros((3, hidden), dtype=torch.int16, device="cuda")
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        n.forward(x_dev, stream.cuda_stream)
    for step in range(4):
        if step == 2:                     # a sequence leaves, another takes its pages and its place
            cache.release(0)
            lens[0] = 0
        before = list(lens)
        for s in range(3):
            lens[s] += 1
            cache.reserve(s, lens[s])
        cache.kv_len.copy_(torch.tensor(lens))
        x = synth.activations(rng, 3, hidden)
        x_dev.copy_(dev_bf16_bits(x))
        n.core.fill_(0x7FC0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        torch.cuda.synchronize()
        check_layer(n, host, x, [1, 1, 1], before, kv)
        assert n._attn_ws[1] is None or not n._attn_ws[1].any()


def test_two_captured_trains_at_once(ctx):
    """Two graphs, each with its own cache and workspaces, replayed on two streams at once: the bytes of each by itself."""
    say("two captured attention layers at once")
    heads, kvh, dim, hidden = 8, 2, 64, 256
    host, weights = layer_weights(heads, kvh, dim, hidden, False, 90)
    freq = torch.tensor([1e4 ** (-i / 16) for i in range(16)], dtype=torch.float64).cuda()
    trains = []
    for i in range(2):
        cache = PagedKvCache(2, kvh, dim, 3000, page_tokens=64)
        for s in range(2):
            cache.reserve(s, 3000)
        gen = torch.Generator().manual_seed(i)
        for t in (cache.k, cache.v):
            t.view(torch.bfloat16).copy_(torch.randn(t.numel() // 2, generator=gen))
        cache.kv_len.copy_(torch.tensor([2900 + i, 1700]))
        n = layer(ctx, cache, 2, 1, False, heads, hidden, weights, freq)
        x = dev_bf16_bits(synth.activations(np.random.default_rng(i), 2, hidden))
        n.forward(x)
        torch.cuda.synchronize()
        want, core = n.out.clone(), n.core.clone()
        stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            n.forward(x, stream.cuda_stream)
        trains.append((n, x, want, core, stream, g))
    for rep in range(4):
        for n, *_ in trains:
            n.out.zero_(), n.core.zero_()
        torch.cuda.synchronize()
        for *_, stream, g in trains:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for n, _, want, core, *_ in trains:
            assert torch.equal(n.out, want) and torch.equal(n.core, core) and want.any(), rep
