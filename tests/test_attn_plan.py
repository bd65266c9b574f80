"""CPU tests of the launch that `attn` makes (csrc/host/attn.cpp), as resolve_attn describes it."""
import ctypes
import random

import pytest

from saber_engine_amd import iu8

P = 1 << 40        # an address: nothing here is launched


def cache(kvh, dim, e4m3=False, page=64, stride=4096):
    return iu8.KvCache.of(P, P, P, P, kv_heads=kvh, head_dim=dim, page_tokens=page, pages=1000, table_stride=stride, kind=iu8.KV_E4M3 if e4m3 else iu8.KV_BF16,
                          k_scale=P if e4m3 else None, v_scale=P if e4m3 else None)


def plan(dim, kvh, group, e4m3, seqs, max_q, max_kv, tokens=None, packed=True, split=True, **more):
    heads = kvh * group
    tokens = (seqs * max_q if packed else seqs) if tokens is None else tokens
    return iu8.resolve_attn(cache(kvh, dim, e4m3, **more), heads * dim, tokens, seqs, max_q, max_kv, heads, 0.125, packed, split)


def scalar(d, name):
    return next(s.ival for s in d.args[:d.n_args] if s.name == name.encode())


def kinds(d):
    return {s.name.decode(): s.kind for s in d.args[:d.n_args]}


def test_the_descriptor_says_what_the_call_takes():
    d = plan(256, 4, 6, False, 1, 1, 1800, packed=False)
    assert (d.op, d.plugin, d.kernel, d.grid[0], d.block[0]) == (b"attn", b"attn_paged", b"attn_few_bf16_d256_r16", 60, 256)
    k = kinds(d)
    assert k["cu_q"] == k["k_scale"] == k["v_scale"] == iu8.ARG_NULL_BUFFER and k["partial"] == k["counter"] == k["q"] == iu8.ARG_BUFFER
    assert [(w.name, w.bytes, w.zero_once) for w in d.workspaces[:d.n_workspaces]] == [(b"partial", 60 * 2 * 16 * 260 * 4, 0), (b"counter", 16, 1)]
    assert scalar(d, "shape") == 24 | 4 << 16 and scalar(d, "unit_shift") == 7 and scalar(d, "page_shift") == 6 and scalar(d, "q_row") == 24 * 256
    d = plan(128, 2, 6, True, 1, 300, 6000)
    assert d.kernel == b"attn_many_e4m3_d128" and scalar(d, "splits") > 1 and d.grid[0] == 2 * 15 * scalar(d, "splits")
    assert kinds(d)["k_scale"] == kinds(d)["cu_q"] == iu8.ARG_BUFFER
    d = plan(128, 2, 6, True, 1, 300, 6000, split=False)
    assert d.kernel == b"attn_many_e4m3_d128" and scalar(d, "splits") == 1 and d.n_workspaces == 0 and kinds(d)["partial"] == iu8.ARG_NULL_BUFFER


def test_the_descriptor_is_refused_as_the_call_is():
    for bad, words in ((dict(max_q=0, tokens=5), "from 1"), (dict(max_kv=1 << 31), "below 2"), (dict(tokens=0), "nothing to do"), (dict(tokens=2, packed=False), "one row a sequence"),
                       (dict(stride=1 << 26), "positions below")):
        a = dict(dim=64, kvh=2, group=2, e4m3=False, seqs=1, max_q=5, max_kv=100)
        a.update(bad)
        with pytest.raises(iu8.IU8Error, match=words) as e:
            plan(**a)
        assert e.value.code == iu8.E_RULE
    with pytest.raises(iu8.IU8Error, match="cover"):
        iu8.resolve_attn(cache(2, 64), 252, 1, 1, 1, 100, 4, 0.125)
    with pytest.raises(iu8.IU8Error, match="number"):
        iu8.resolve_attn(cache(2, 64), 256, 1, 1, 1, 100, 4, float("nan"))


def test_a_call_takes_no_more_than_its_workspaces():
    rng = random.Random(5)
    for _ in range(4000):
        kvh, group, dim, e4m3 = rng.choice([1, 2, 4, 8]), rng.choice([1, 3, 5, 6, 8, 16, 17, 40]), rng.choice([64, 128, 256]), rng.random() < 0.5
        most = [rng.choice([1, 2, 9, 64, 300]), rng.choice([1, 2, 5, 40, 200, 1000, 9000]), rng.choice([1, 129, 600, 1500, 5000, 140000])]
        less = [rng.randint(1, x) for x in most]
        sizes = iu8.attn_workspace(*most, kvh * group, kvh, dim)
        d = plan(dim, kvh, group, e4m3, *less)
        took = [w.bytes for w in d.workspaces[:d.n_workspaces]] or [0, 0]
        assert took[0] <= sizes[0] and took[1] <= sizes[1], (most, less, kvh, group, dim, e4m3)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_whole_prompts_take_the_kernels_that_skip_what_causality_hides(dim):
    """The few-row kernels walk a prompt's hidden half, the many-row kernels do not: from three (bf16) and eight (e4m3) units of 128 keys a CU on
    a whole prompt is the many-row kernels'; the same rows behind a prefix, and prompts below, stay."""
    def many(e4m3, kvh, group, new, kv, seqs=1):
        return b"many" in plan(dim, kvh, group, e4m3, seqs, new, kv).kernel
    for e4m3, kvh, group, new in ((True, 2, 8, 1024), (True, 1, 8, 1400), (True, 1, 5, 1700), (True, 2, 4, 1150), (True, 2, 8, 900), (False, 1, 4, 900), (False, 1, 4, 1000),
                                  (False, 1, 2, 300), (False, 1, 8, 300), (False, 1, 6, 200), (True, 4, 6, 200)):
        assert many(e4m3, kvh, group, new, new), (e4m3, kvh, group, new)
    for e4m3, kvh, group, new, kv in ((True, 2, 4, 900, 900), (True, 1, 8, 300, 300), (True, 1, 5, 1000, 1000), (False, 1, 3, 900, 900), (False, 1, 1, 1400, 1400), (False, 1, 4, 400, 400),
                                      (True, 2, 8, 500, 1000), (True, 1, 8, 1000, 1333), (False, 1, 4, 900, 1200), (False, 1, 8, 220, 293), (True, 1, 8, 300, 4800)):
        assert not many(e4m3, kvh, group, new, kv), (e4m3, kvh, group, new, kv)


@pytest.mark.parametrize("dim,kvh,group,max_q,seqs,kv,grid", [
    (64, 8, 1, 1, 64, 8192, 512), (64, 8, 5, 1, 256, 8192, 512), (64, 8, 5, 1, 32, 20000, 256), (64, 8, 4, 8, 64, 8192, 256), (128, 8, 5, 1, 64, 8192, 512),
    (128, 8, 4, 8, 32, 20000, 256), (256, 4, 6, 1, 128, 8192, 256), (256, 4, 6, 5, 128, 8192, 256)])
def test_long_streams_take_every_compute_unit(dim, kvh, group, max_q, seqs, kv, grid):
    """As many as fit: a workgroup's tiles are what is in flight, 32 KiB of them at width 64."""
    d = plan(dim, kvh, group, False, seqs, max_q, kv)
    assert b"few" in d.kernel and d.grid[0] == grid == plan(dim, kvh, group, False, seqs, max_q, 6000).grid[0]


def test_descriptors_without_what_the_kernel_reads_are_refused():
    """A buffer that a kernel reads, set to none by hand; rows of sequences that are not there; page sizes with more bits than a page has."""
    guard = ctypes.CDLL(iu8.LIB_PATH)["_ZN3iu810attn_guardEPK14saber_iu8_desc"]
    append = dict(shape=8 | 2 << 16, form=6 | 64 << 16, pages=10, table_stride=4, tokens=3, seqs=3)
    few = dict(shape=8 | 2 << 16, page_shift=6, pages=10, table_stride=4, tokens=3, seqs=3, unit_shift=7, qtiles=1)
    many = dict(shape=8 | 2 << 16, page_shift=6, pages=10, table_stride=4, tokens=300, chunk=128, splits=2, qtiles=3)

    def check(kernel, scalars, none=(), **more):
        d = iu8.describe_raw(kernel, (12, 1, 1), 256, "attn_paged", **dict(scalars, **more))
        for s in d.args[:d.n_args]:
            if s.name.decode() in none:
                s.kind = iu8.ARG_NULL_BUFFER
        return guard(ctypes.byref(d))

    for kernel, scalars, needs in (("kv_append_bf16_d128", append, "q k v q_out kc vc table kv_len inv_freq"), ("kv_append_e4m3_d64", append, "q k_scale v_scale inv_freq"),
                                   ("attn_few_bf16_d64_r16", few, "q kc vc table kv_len out partial counter"), ("attn_few_e4m3_d256_r32", few, "k_scale v_scale"),
                                   ("attn_many_bf16_d256", many, "q kc vc table kv_len out partial counter"), ("attn_many_e4m3_d128", many, "k_scale v_scale")):
        assert check(kernel, scalars) == 0
        for name in needs.split():
            assert check(kernel, scalars, (name,)) == iu8.E_RULE, (kernel, name)
    assert check("kv_append_bf16_d64", append, ("k_scale", "v_scale", "cu_q", "q_norm", "k_norm")) == 0
    assert check("kv_append_bf16_d64", append, ("inv_freq",), form=6) == 0
    assert check("kv_append_bf16_d64", append, ("cu_q",), tokens=4) == iu8.E_RULE and check("kv_append_bf16_d64", append, (), tokens=4) == 0
    assert check("attn_few_bf16_d64_r16", few, page_shift=6 | 1 << 8) == iu8.E_RULE and check("attn_many_bf16_d64", many, page_shift=5 | 1 << 16) == iu8.E_RULE
