"""GPU tests of the paged key/value cache and the attention that reads it (code object `attn_paged`), through the C ABI, against
their definitions in 64 bits (attn_util.py, which derives the tolerances)."""
import math

import numpy as np
import pytest
import torch

from saber_engine_amd import iu8
from tests.attn_util import BF16, E4M3, Paged, Workspace, attention, check, f64, random_rows
from tests.gpu_util import say

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


KINDS = [(64, 8, 8), (64, 14, 2), (128, 5, 1), (128, 16, 1), (256, 12, 2), (256, 4, 4)]


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
    (128, 5, 1, [3001, 129, 5], [1, 1, 1]), (256, 6, 1, [4099], [5]), (64, 4, 1, [2600, 700], [40, 50]), (256, 12, 2, [1900], [90]), (128, 16, 2, [1500], [64])])
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
