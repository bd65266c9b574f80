"""CPU tests of what the host deals and refuses: pages that are forked, trimmed and compacted (saber_engine_amd/attn.py), a delta-net layer's slots and
train (saber_engine_amd/gdn.py)."""
import ctypes
import random

import numpy as np
import pytest
import torch

from saber_engine_amd import attn, gdn, iu8


def numbers(address, n):
    return list((ctypes.c_int32 * n).from_address(address))


class Copies:
    """A context that copies on the host, and keeps what it was asked for."""

    def __init__(self):
        self.calls = []

    def kv_copy(self, cache, src, dst, n, stream=0):
        pairs = list(zip(numbers(src, n), numbers(dst, n)))
        self.calls.append(pairs)
        assert len({d for _, d in pairs}) == n and not {s for s, _ in pairs} & {d for _, d in pairs}
        assert all(0 <= p < cache.pages for pair in pairs for p in pair)
        size = iu8.kv_bytes(1, cache.kv_heads, cache.head_dim, cache.page_tokens, cache.kind)
        for base in (cache.k, cache.v):
            for s, d in pairs:
                ctypes.memmove(base + d * size, base + s * size, size)

    def gdn_copy(self, state, tail, slots, heads, channels, width, src, dst, n, stream=0):
        self.calls.append(list(zip(numbers(src, n), numbers(dst, n))))
        for base, size in ((state, heads * 65536), (tail, (width - 1) * channels * 2)):
            for s, d in self.calls[-1]:
                ctypes.memmove(base + d * size, base + s * size, size)


def held_pages(c):
    """What each sequence's table says, and that the host says the same."""
    got = [t[t >= 0].tolist() for t in c.table]
    assert got == c._held
    count = [0] * c.pages
    for pages in got:
        assert len(set(pages)) == len(pages)
        for p in pages:
            count[p] += 1
    assert count == c._holders and sorted(c._free) == [p for p in range(c.pages) if not count[p]]
    return got


def test_random_forks_trims_compactions_keep_every_sequence():
    """Against sequences that have pages of their own: every position's bytes, whatever shares them."""
    rng, page = random.Random(3), 16
    c, ctx = attn.PagedKvCache(6, 1, 64, 400, pages=60, page_tokens=page, device="cpu"), Copies()
    size = 64 * 2
    k = c.k.view(c.pages, page, size)     # (of one head a token's bytes lie in its page: which place is the test's to say)
    want, stamp = [[] for _ in range(6)], 0
    for step in range(600):
        s, d = rng.sample(range(6), 2)
        what = rng.choice(("append", "append", "append", "fork", "trim", "release", "compact"))
        try:
            if what == "append":
                n = rng.randint(1, 40)
                c.reserve(s, len(want[s]) + n)
                for _ in range(n):
                    stamp += 1
                    t = len(want[s])
                    place = c._held[s][t // page]
                    assert c._holders[place] == 1, "a page that is written belongs to one sequence"
                    k[place, t % page] = torch.tensor([stamp >> 16 & 255, stamp >> 8 & 255, stamp & 255] + [0] * (size - 3), dtype=torch.uint8)
                    want[s].append(stamp)
                c.kv_len[s] = len(want[s])
            elif what == "fork":
                if want[d]:
                    c.release(d)
                    want[d] = []
                n = rng.randint(0, len(want[s]))
                if not c._held[d]:
                    c.fork(ctx, s, d, n)
                    want[d] = want[s][:n]
            elif what == "trim":
                n = rng.randint(0, len(want[s]))
                c.trim(ctx, s, n)
                want[s] = want[s][:n]
            elif what == "release":
                c.release(s)
                want[s] = []
            else:
                n = c.compact(ctx)
                assert n == len({p for held in c._held for p in held}) and all(p < n for held in c._held for p in held)
        except iu8.IU8Error as e:
            assert "free" in str(e) or "hold" in str(e)
        held = held_pages(c)
        for x in range(6):
            got = [k[held[x][t // page], t % page, :3].tolist() for t in range(len(want[x]))]
            assert [a << 16 | b << 8 | e for a, b, e in got] == want[x], (step, what, x)
            assert c.kv_len[x] == len(want[x])
    assert len(ctx.calls) > 50


def test_forks_share_whole_pages_and_copy_the_last():
    c, ctx = attn.PagedKvCache(4, 2, 64, 200, pages=8, page_tokens=32, device="cpu"), Copies()
    c.reserve(0, 96)
    c.fork(ctx, 0, 1, 64)
    assert not ctx.calls and c._held[1] == c._held[0][:2] and c.kv_len[1] == 64
    c.fork(ctx, 0, 2, 70)
    assert ctx.calls == [[(c._held[0][2], c._held[2][2])]] and c._held[2][:2] == c._held[0][:2] and len(c._free) == 4
    c.release(0)
    assert len(c._free) == 5
    c.trim(ctx, 2, 40)                    # the second page is sequence 1's too
    assert ctx.calls[1] == [(c._held[1][1], c._held[2][1])] and c.kv_len[2] == 40
    c.trim(ctx, 2, 500)
    c.trim(ctx, 2, 32)
    assert len(ctx.calls) == 2 and held_pages(c)[2] == c._held[1][:1]
    c.fork(ctx, 1, 3, 0)
    assert c._held[3] == [] and c.kv_len[3] == 0
    c.trim(ctx, 1, 0)
    assert c._held[1] == [] and len(c._free) == 7


def test_forks_that_are_refused():
    c, ctx = attn.PagedKvCache(3, 1, 64, 200, pages=3, page_tokens=32, device="cpu"), Copies()
    c.reserve(0, 80)
    for a in ((0, 0, 10), (0, 1, 97), (0, 1, -1), (1, 2, 1)):
        with pytest.raises(iu8.IU8Error, match="tokens of sequence"):
            c.fork(ctx, *a)
    with pytest.raises(iu8.IU8Error, match="none free"):
        c.fork(ctx, 0, 1, 80)
    c.fork(ctx, 0, 1, 64)
    with pytest.raises(iu8.IU8Error, match="tokens of sequence"):
        c.fork(ctx, 0, 1, 64)
    with pytest.raises(iu8.IU8Error, match="none free"):
        c.trim(ctx, 1, 40)
    held_pages(c)
    c.trim(ctx, 0, 40)                    # its third page comes free, and takes the copy
    assert held_pages(c)[0][1] != c._held[1][1] and not ctx.calls[1:]


def test_states_are_dealt_forked_and_come_back():
    s, ctx = gdn.GdnState(5, 1, 2, slots=3, device="cpu"), Copies()
    assert s.channels == 512 and (s.slot == -1).all()
    s.state.fill_(5), s.tail.fill_(5)
    s.begin(3), s.begin(0)
    assert (s.state[s.slot[3]] == 0).all() and (s.tail[s.slot[0]] == 0).all() and s.slot[1] == -1
    s.state[s.slot[3]] = torch.randn(2, 128, 128)
    s.tail[s.slot[3]] = torch.randint(0, 999, (3, 512), dtype=torch.int16)
    s.fork(ctx, 3, [4])
    assert torch.equal(s.state[s.slot[4]], s.state[s.slot[3]]) and torch.equal(s.tail[s.slot[4]], s.tail[s.slot[3]]) and len(ctx.calls) == 1
    for bad in (lambda: s.begin(1), lambda: s.begin(3), lambda: s.fork(ctx, 1, [2]), lambda: s.fork(ctx, 3, [2]), lambda: s.fork(ctx, 3, [0])):
        with pytest.raises(iu8.IU8Error):
            bad()
    s.release(0), s.release(3), s.release(3)
    assert sorted(s._free + [s._held[4]]) == [0, 1, 2] and s.slot.tolist() == [-1, -1, -1, -1, s._held[4]]
    s.fork(ctx, 4, [1, 2])
    assert sorted(s.slot[[1, 2, 4]].tolist()) == [0, 1, 2] and torch.equal(s.state[s.slot[2]], s.state[s.slot[4]])
    with pytest.raises(iu8.IU8Error):
        s.fork(ctx, 4, [0, 0])
    s.fork(ctx, 4, [])
    for bad in (dict(heads=3), dict(width=5), dict(slots=0), dict(seqs=0)):
        with pytest.raises(iu8.IU8Error):
            gdn.GdnState(**dict(dict(seqs=2, key_heads=2, heads=4, device="cpu"), **bad))


def test_layers_of_tensors_that_do_not_fit():
    s = gdn.GdnState(3, 2, 8, device="cpu")
    with pytest.raises(iu8.IU8Error, match="one a sequence"):
        gdn.GdnLayerIU8(None, s, 4, 256)
    n = gdn.GdnLayerIU8(None, s, 3, 256)
    f, bf = lambda *k: torch.ones(*k), lambda *k: torch.ones(*k, dtype=torch.bfloat16)  # noqa: E731
    good = dict(conv=bf(s.channels, 4), a_log=f(8), dt_bias=f(8), norm=bf(128), had_t=f(1024))
    w = (None,) * 6
    n.set_weights(*w, **good)
    n.set_weights(*w, **good, conv_bias=bf(s.channels))
    for bad, words in ((dict(conv=bf(s.channels, 3)), "conv"), (dict(conv=f(s.channels, 4)), "conv"), (dict(a_log=f(7)), "a_log"), (dict(dt_bias=f(8).double()), "dt_bias"),
                       (dict(norm=bf(64)), "norm"), (dict(had_t=f(2048)[::2]), "had_t"), (dict(had_t=None), "had_t"), (dict(conv_bias=bf(8)), "conv_bias")):
        with pytest.raises(iu8.IU8Error, match=words):
            n.set_weights(*w, **dict(good, **bad))
    with pytest.raises(iu8.IU8Error, match="made for"):
        n.forward(torch.zeros((2, 256), dtype=torch.int16))
    for bad in (torch.zeros((3, 256)), torch.zeros((256, 3), dtype=torch.int16).t()):
        with pytest.raises(iu8.IU8Error, match="in one piece"):
            n.forward(bad)
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(3), np.zeros(3, np.int32)):
        with pytest.raises((iu8.IU8Error, AttributeError)):
            n.accept(bad)
