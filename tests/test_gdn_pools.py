"""CPU tests of the pools' books (saber_engine_amd/attn.py, saber_engine_amd/gdn.py): what a call that fails on the device leaves of them."""
import pytest
import torch

from saber_engine_amd import attn, gdn, iu8
from tests.test_gdn_layer import Copies, held_pages


class Fails(Copies):
    """A context whose copies raise."""

    def kv_copy(self, *a, **k):
        raise iu8.IU8Error(iu8.E_HIP, "no copy")

    gdn_copy = kv_copy


def books(c):
    return [list(h) for h in c._held], list(c._holders), list(c._free), c.table.clone(), c.kv_len.clone()


def same(a, b):
    return all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b))


def test_a_copy_that_fails_leaves_the_pages_as_they_were():
    c, ctx = attn.PagedKvCache(4, 1, 64, 200, pages=9, page_tokens=32, device="cpu"), Copies()
    c.reserve(0, 160)
    c.kv_len[0] = 150
    c.fork(ctx, 0, 1, 96)
    c.reserve(1, 150)
    was = books(c)
    for call in (lambda: c.fork(Fails(), 0, 2, 80), lambda: c.trim(Fails(), 0, 40), lambda: c.trim(Fails(), 1, 70)):
        with pytest.raises(iu8.IU8Error, match="no copy"):
            call()
        assert same(books(c), was)
        held_pages(c)
    c.release(0)
    was = books(c)
    with pytest.raises(iu8.IU8Error, match="no copy"):
        c.compact(Fails())
    assert same(books(c), was)
    c.fork(ctx, 1, 2, 80), c.trim(ctx, 1, 40), c.compact(ctx)
    assert len(held_pages(c)[2]) == 3 and len(c._free) == 9 - 4
    for s in range(4):
        c.release(s)
    held_pages(c)
    assert sorted(c._free) == list(range(9))


def test_a_copy_that_fails_leaves_the_slots_as_they_were():
    s = gdn.GdnState(4, 1, 2, device="cpu")
    s.begin(1)
    was = list(s._held), list(s._free), s.slot.clone()
    with pytest.raises(iu8.IU8Error, match="no copy"):
        s.fork(Fails(), 1, [0, 3])
    assert same((s._held, s._free, s.slot), was)
    s.fork(Copies(), 1, [0, 3])
    s.begin(2)
    assert sorted(s.slot.tolist()) == [0, 1, 2, 3] and s.slot.tolist() == s._held


def test_positions_that_are_not_written_yet_are_not_shared():
    """Pages reserved ahead of the count: shared, the source's next rows would be another sequence's too."""
    c, ctx = attn.PagedKvCache(3, 1, 64, 200, pages=9, page_tokens=32, device="cpu"), Copies()
    c.reserve(0, 96)
    c.kv_len[0] = 70
    was = books(c)
    for tokens in (71, 96):
        with pytest.raises(iu8.IU8Error, match="which counts 70"):
            c.fork(ctx, 0, 1, tokens)
        assert same(books(c), was) and not ctx.calls
    c.fork(ctx, 0, 1, 70)
    assert c._held[1][:2] == c._held[0][:2] and c._held[1][2] != c._held[0][2] and c._holders[c._held[0][2]] == 1
    c.kv_len[0] = 96
    c.fork(ctx, 0, 2, 96)
    assert c._held[2] == c._held[0] and len(ctx.calls) == 1
