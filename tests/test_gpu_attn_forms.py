"""GPU tests of the paged cache's attention by the kernel that a call takes: each case says which kernel, and how many parts, it is made for,
so that no change of the launch law empties it. Definitions in 64 bits and tolerances: attn_util.py."""
import math

import numpy as np
import pytest
import torch

from saber_engine_amd import iu8
from tests.attn_util import Paged, Workspace, attention, check, e4m3_of, f64, random_rows
from tests.gpu_util import say
from tests.test_gpu_attn import ends

pytestmark = pytest.mark.gpu


def splits_of(d):
    return next((s.ival for s in d.args[:d.n_args] if s.name == b"splits"), None)


class Call:
    """A cache of `lens` keys filled with seeded values, rows `news` and the launch that attn makes of them."""

    def __init__(self, dim, heads, kvh, lens, news, e4m3=False, page=64, max_kv=None, split=True, seed=1):
        self.dim, self.heads, self.kvh, self.lens, self.news = dim, heads, kvh, lens, news
        g = torch.Generator().manual_seed(seed)
        self.c = Paged(len(lens), kvh, dim, page, max(lens), e4m3, seed)
        self.c.kv_len.copy_(torch.tensor(lens))
        for s, n in enumerate(lens):
            self.c.put(s, 0, random_rows(g, n, kvh, dim, e4m3=e4m3), random_rows(g, n, kvh, dim, e4m3=e4m3))
        self.tokens, self.max_q, self.max_kv = sum(news), max(news), max(lens) if max_kv is None else max_kv
        self.q = random_rows(g, self.tokens, heads * dim)
        self.out = torch.full((self.tokens, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
        self.cu, self.scale = ends(news), 1 / math.sqrt(dim)
        self.ws = Workspace(len(lens), self.max_q, self.max_kv, heads, kvh, dim) if split else None
        self.plan = iu8.resolve_attn(self.c.desc(), heads * dim, self.tokens, len(lens), self.max_q, self.max_kv, heads, self.scale, True, split)

    def takes(self, form, parts):
        """`form`: the kernel's name without type and width, `parts`: its launch is split."""
        name = self.plan.kernel.decode()
        assert name.startswith(form.split("_r")[0]) and (form[-4:-2] != "_r" or name.endswith(form[-4:])), name
        assert name.split("_")[2:4] == ["e4m3" if self.c.e4m3 else "bf16", f"d{self.dim}"], name
        assert (splits_of(self.plan) > 1 if "many" in form else self.plan.n_workspaces > 0) == parts, (name, splits_of(self.plan))
        return self

    def run(self, ctx):
        args = self.ws.args() if self.ws else (None, None)
        ctx.attn(self.q.data_ptr(), self.heads * self.dim, self.c.desc(), self.cu.data_ptr(), self.out.data_ptr(), self.tokens, len(self.lens), self.max_q, self.max_kv,
                 self.heads, self.scale, *args)
        torch.cuda.synchronize()
        assert self.ws is None or self.ws.counter is None or not self.ws.counter.any(), "the counters are left zero"
        return self.out

    def launch(self, ctx, out):
        """The same by the descriptor."""
        b = dict(q=self.q, kc=self.c.k, vc=self.c.v, k_scale=self.c.scales[0], v_scale=self.c.scales[1], table=self.c.table, kv_len=self.c.kv_len, cu_q=self.cu, out=out,
                 partial=self.ws.partial if self.ws else None, counter=self.ws.counter if self.ws else None)
        ctx.launch(self.plan, {n: t.data_ptr() for n, t in b.items() if t is not None})
        torch.cuda.synchronize()

    def check(self, rows):
        """Rows [(sequence, row of it)] against the definition; where that is not finite, the same infinity or a NaN."""
        got, x = f64(self.out.float()), f64(self.q.float()).reshape(self.tokens, self.heads, self.dim)
        at = np.concatenate(([0], np.cumsum(self.news)))
        for s in sorted({s for s, _ in rows}):
            k, v, there = self.c.rows(s, self.lens[s])
            for i in (i for r, i in rows if r == s):
                sees, t = self.lens[s] - self.news[s] + i + 1, at[s] + i
                with np.errstate(invalid="ignore"):
                    want, tol = attention(x[t:t + 1], k[:sees], v[:sees], there[:sees], self.scale)
                fine = np.isfinite(want)
                same = (got[t:t + 1] == want) | (np.isnan(got[t:t + 1]) & np.isnan(want))
                assert (fine | same).all(), f"row {i} of sequence {s}: not finite where the definition is not"
                check(np.where(fine, got[t:t + 1], 0), np.where(fine, want, 0), np.where(fine, tol, 0), f"row {i} of sequence {s}")

    def sample(self, n=5):
        """Rows of every sequence: the first, the last, some between."""
        rng = np.random.default_rng(self.tokens)
        return [(s, int(i)) for s, m in enumerate(self.news) if m for i in sorted({0, m - 1, *rng.integers(0, m, n)})]


WIDTHS = [(64, 12, 2), (128, 12, 2), (256, 12, 2)]


# ------------------------------------------------------------------ many rows, in parts

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh", WIDTHS)
def test_many_rows_in_parts(ctx, dim, heads, kvh, e4m3):
    say(f"attn many, in parts {dim} {e4m3}")
    c = Call(dim, heads, kvh, [6001], [300], e4m3).takes("attn_many", True)
    c.run(ctx)
    c.check(c.sample())
    again = torch.zeros_like(c.out)
    c.launch(ctx, again)
    assert torch.equal(again.view(torch.int16), c.out.view(torch.int16)), "the call and its descriptor"


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh", WIDTHS)
def test_many_rows_in_parts_of_ragged_sequences_and_holes(ctx, dim, heads, kvh, e4m3):
    """Sequences with fewer parts than the launch has, one row tile's last rows alone; a part that has no key at all."""
    say(f"attn many, in parts, ragged {dim} {e4m3}")
    c = Call(dim, heads, kvh, [6001, 150, 3100, 1], [300, 150, 257, 1], e4m3, page=128).takes("attn_many", True)
    c.c.table[0, 10:30] = -1
    c.c.table[2, 3] = c.c.pages
    c.run(ctx)
    c.check(c.sample())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh", WIDTHS)
def test_many_rows_in_parts_longer_than_told(ctx, dim, heads, kvh, e4m3):
    """Lengths past max_kv where that is already cut: the parts grow."""
    say(f"attn many, parts of a longer cache than told {dim} {e4m3}")
    c = Call(dim, heads, kvh, [6001, 2600], [600, 600], e4m3, max_kv=2500).takes("attn_many", True)
    assert splits_of(c.plan) * next(s.ival for s in c.plan.args[:c.plan.n_args] if s.name == b"chunk") < 6001
    c.run(ctx)
    c.check(c.sample(3))


# ------------------------------------------------------------------ values that are not finite

def spoil(c, s, at, what, channels, head=0):
    """Channels of the value at position `at` of sequence s's kv head `head`."""
    p, o = int(c.table[s, at // c.page]), at % c.page
    c.v[p, head, o, channels] = torch.tensor(what, device="cuda").to(c.kind)


BAD = [70, 71, 95, 96, 127, 128, 133, 160, 198, 199]


@pytest.mark.parametrize("at", BAD)
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_beside_values_that_are_not_finite(ctx, dim, e4m3, at):
    """A new token's value has infinities and NaNs (a tile's first, middle and last token, both of its halves): in the rows from its own on they
    are what the definition gives, in those channels alone; the rows before it are what they are without."""
    say(f"attn many, NaN at {at} of 200, {dim} {e4m3}")
    c = Call(dim, 4, 2, [200, 90], [130, 90], e4m3, page=32).takes("attn_many", False)
    nan = float("nan")
    spoil(c.c, 0, at, nan, [5, dim - 1])
    spoil(c.c, 0, min(at + 3, 199), nan, [6], head=1)
    if not e4m3:
        spoil(c.c, 0, at, float("inf"), [0, 17, dim // 2 + 1])
        spoil(c.c, 0, at, float("-inf"), [30])
        spoil(c.c, 1, 64, float("-inf"), [33], head=1)
    c.run(ctx)
    assert torch.isnan(c.out[at - 70:130, :2, 5]).all() and torch.isfinite(c.out[:max(at - 70, 0)]).all() and torch.isfinite(c.out[:130, :2, 7]).all()
    c.check([(0, i) for i in sorted({0, 1, at - 71, at - 70, at - 69, 58, 100, 129}) if 0 <= i < 130] + [(1, 0), (1, 63), (1, 64), (1, 89)])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_beside_bad_values_holes_and_ends(ctx, dim, e4m3):
    """Bad values in one tile with a hole and with the end of the sequence, and in both of a tile's halves."""
    say(f"attn many, NaN, holes, ends {dim} {e4m3}")
    c = Call(dim, 4, 2, [150], [140], e4m3, page=16).takes("attn_many", False)
    for at in (33, 62, 97, 126, 145, 149):
        spoil(c.c, 0, at, float("nan"), [at % dim])
    c.c.table[0, 3] = -1        # positions 48 .. 63: the bad value at 62 is nobody's
    c.c.table[0, 7] = c.c.pages
    c.run(ctx)
    c.check([(0, i) for i in range(0, 140, 7)] + [(0, 23), (0, 52), (0, 87), (0, 139)])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,heads,kvh", WIDTHS)
def test_many_rows_in_parts_beside_values_that_are_not_finite(ctx, dim, heads, kvh, e4m3):
    say(f"attn many, in parts, NaN {dim} {e4m3}")
    c = Call(dim, heads, kvh, [6000], [300], e4m3).takes("attn_many", True)
    spoil(c.c, 0, 5800, float("nan"), [9])
    spoil(c.c, 0, 5999, float("nan"), [10], head=1)
    c.run(ctx)
    c.check([(0, i) for i in (0, 99, 100, 101, 200, 298, 299)])


@pytest.mark.parametrize("at", [1940, 1951, 1983, 1984, 1999])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_row_tiles_of_few_beside_values_that_are_not_finite(ctx, dim, e4m3, at):
    """The few-row kernels' tiles of 32 rows, several a sequence."""
    say(f"attn few, row tiles, NaN at {at} of 2000, {dim} {e4m3}")
    c = Call(dim, 4, 2, [2000], [60], e4m3).takes("attn_few_r32", True)
    spoil(c.c, 0, at, float("nan"), [3])
    if not e4m3:
        spoil(c.c, 0, at, float("inf"), [40])
    c.run(ctx)
    c.check([(0, i) for i in sorted({0, 15, 16, at - 1941, at - 1940, 59}) if i >= 0])


@pytest.mark.parametrize("e4m3", [False, True])
def test_few_rows_by_their_descriptor(ctx, e4m3):
    say(f"attn few, by descriptor {e4m3}")
    for form, lens, news in (("attn_few_r16", [1500, 70], [2, 1]), ("attn_few_r32", [900, 1300], [4, 5])):
        c = Call(128, 12, 2, lens, news, e4m3).takes(form, True)
        c.run(ctx)
        c.check(c.sample(2))
        again = torch.zeros_like(c.out)
        c.launch(ctx, again)
        assert torch.equal(again.view(torch.int16), c.out.view(torch.int16)) and not c.ws.counter.any()


# ------------------------------------------------------------------ rounding

@pytest.mark.parametrize("scale", [0.3, 0.7, 1.0, 0.0123, 3.1415927, 1 / 448])
def test_e4m3_values_are_the_rounded_quotients(ctx, scale):
    """Every bf16 value as k and as v: the byte of value / scale, an f32 quotient rounded to nearest even, saturated, a NaN kept."""
    say(f"append e4m3, every bf16 value at a scale of {scale}")
    n, dim = 256, 256
    c = Paged(1, 1, dim, 64, n, True)
    c.scales = [torch.full((1,), scale, device="cuda") for _ in range(2)]
    c.kv_len[0] = n
    values = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(n, dim)
    rows = torch.cat((torch.zeros(n, dim, dtype=torch.bfloat16), values, values.flip(0)), 1).cuda()
    q_out, p = torch.zeros(n, dim, dtype=torch.bfloat16, device="cuda"), rows.data_ptr()
    ctx.kv_append(p, p + 2 * dim, p + 4 * dim, q_out.data_ptr(), c.desc(), ends([n]).data_ptr(), n, 1, 1, 3 * dim, dim, 3 * dim)
    torch.cuda.synchronize()
    c.scales = [torch.ones(1, device="cuda")] * 2
    k, v, _ = c.rows(0, n)
    want = e4m3_of(f64(values.float()), scale)
    assert np.array_equal(k[:, 0], want, equal_nan=True) and np.array_equal(v[::-1, 0], want, equal_nan=True)
    number = ~np.isnan(want)       # a zero keeps its value's sign
    negative = np.signbit(f64(values.float()))[number]
    assert np.array_equal(np.signbit(k[:, 0])[number], negative) and np.array_equal(np.signbit(v[::-1, 0])[number], negative)


# ------------------------------------------------------------------ rows and positions

@pytest.mark.parametrize("dim,heads,kvh,lens,news,form", [
    (64, 4, 2, [50, 300], [3, 6], "attn_few_r16"), (128, 8, 2, [50, 300], [3, 8], "attn_few_r32"), (256, 4, 2, [50, 200], [30, 130], "attn_many"),
    (128, 4, 2, [50, 200], [30, 130], "attn_many")])
def test_an_end_past_the_call_s_rows_counts_for_the_positions(ctx, dim, heads, kvh, lens, news, form):
    """The last sequence's end lies behind `tokens`: both operators give the rows that are there what they are given in the whole call, and
    touch no others."""
    say(f"end past tokens {form} {dim}")
    c = Call(dim, heads, kvh, lens, news, split=False).takes(form, False)
    whole, less = c.run(ctx).clone(), c.tokens - 2
    c.check([(1, news[1] - 3)])
    c.out.fill_(7.0)
    c.tokens = less
    c.run(ctx)
    assert torch.equal(c.out[:less].view(torch.int16), whole[:less].view(torch.int16)) and (c.out[less:] == 7).all()
    rows = random_rows(torch.Generator().manual_seed(3), sum(news), (heads + 2 * kvh) * dim)
    p, row, got = rows.data_ptr(), rows.shape[1], []
    for tokens in (sum(news), less):
        c.c.k.view(torch.uint8).zero_(), c.c.v.view(torch.uint8).zero_()
        q_out = torch.full((sum(news), heads * dim), 7.0, dtype=torch.bfloat16, device="cuda")
        ctx.kv_append(p, p + 2 * heads * dim, p + 2 * (heads + kvh) * dim, q_out.data_ptr(), c.c.desc(), c.cu.data_ptr(), tokens, 2, heads, row, dim, row)
        torch.cuda.synchronize()
        got.append((q_out, *c.c.rows(1, lens[1])[:2]))
    (q0, k0, v0), (q1, k1, v1) = got
    assert torch.equal(q0[:less], q1[:less]) and (q1[less:] == 7).all()
    assert k0[-1].any() and np.array_equal(k0[:-2], k1[:-2]) and np.array_equal(v0[:-2], v1[:-2]) and not k1[-2:].any() and not v1[-2:].any()
