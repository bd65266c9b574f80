"""CPU tests of the paged key/value cache and its attention (csrc/host/attn.cpp, saber_engine_amd/attn.py): refusals, the forms that
arguments take, the cache's order, the workspaces' law, and what the built kernels are like."""
import ctypes
import math
import os
import random
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

from saber_engine_amd import attn, iu8, kbuild

P = 1 << 40        # an address: nothing here is launched


@pytest.fixture(scope="module", autouse=True)
def built():
    if not os.path.exists(iu8.LIB_PATH) or not os.path.exists(os.path.join(iu8.PREBUILT, "attn_paged.manifest.toml")):
        kbuild.build_all()


@pytest.fixture(params=["fastcall", "ctypes"])
def ctx(request):
    """A context that is not open: what the library does not refuse by itself it refuses for that."""
    c = iu8.Context.__new__(iu8.Context)
    c._h, c._addr, c._op = ctypes.c_void_p(), None, iu8._CtypesOperators() if request.param == "ctypes" else iu8.operators()
    return c


def cache(**more):
    a = dict(k=P, v=P, page_table=P, kv_len=P, kv_heads=4, head_dim=256, page_tokens=64, pages=100, table_stride=20, kind=iu8.KV_BF16)
    a.update(more)
    return iu8.KvCache.of(**a)


def append(c, desc=None, **more):
    a = dict(q=P, k=P, v=P, q_out=P, cu_q=P, tokens=9, seqs=3, heads=24, q_row=24 * 512 + 2048, q_head=512, kv_row=24 * 512 + 2048, inv_freq=P,
             rot_dim=64, interleaved=False, q_norm=P, k_norm=P, eps=1e-6)
    a.update(more)
    c.kv_append(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("q_out"), desc or cache(), **a)


def attend(c, desc=None, **more):
    a = dict(q=P, q_row=24 * 256, cu_q=P, out=P, tokens=9, seqs=3, max_q=5, max_kv=900, heads=24, scale=0.0625, partial=P, counter=P)
    a.update(more)
    c.attn(a.pop("q"), a.pop("q_row"), desc or cache(), **a)


def refused(call, code, words):
    with pytest.raises(iu8.IU8Error, match=words) as e:
        call()
    assert e.value.code == code, str(e.value)


CACHES = [(dict(k=None), iu8.E_ARG, "must be given"), (dict(v=None), iu8.E_ARG, "must be given"), (dict(page_table=None), iu8.E_ARG, "must be given"),
          (dict(kv_len=None), iu8.E_ARG, "must be given"), (dict(kind=2), iu8.E_ARG, "kind"), (dict(kind=iu8.KV_E4M3), iu8.E_ARG, "k_scale"),
          (dict(kind=iu8.KV_E4M3, k_scale=P), iu8.E_ARG, "k_scale"), (dict(k=P + 8), iu8.E_ARG, "16 bytes"), (dict(v=P + 2), iu8.E_ARG, "16 bytes"),
          (dict(head_dim=96), iu8.E_RULE, "head width"), (dict(head_dim=512), iu8.E_RULE, "head width"), (dict(page_tokens=8), iu8.E_RULE, "pages of"),
          (dict(page_tokens=48), iu8.E_RULE, "pages of"), (dict(page_tokens=512), iu8.E_RULE, "pages of"), (dict(kv_heads=5), iu8.E_RULE, "whole groups"),
          (dict(kv_heads=0), iu8.E_RULE, "whole groups"), (dict(pages=0), iu8.E_RULE, "at least one"), (dict(pages=1 << 31), iu8.E_RULE, "at least one"),
          (dict(table_stride=0), iu8.E_RULE, "at least one"), (dict(table_stride=1 << 25), iu8.E_RULE, "2\\^31")]


@pytest.mark.parametrize("bad,code,words", CACHES)
def test_caches_that_are_refused(ctx, bad, code, words):
    for call in (append, attend):
        refused(lambda: call(ctx, cache(**bad)), code, words)


@pytest.mark.parametrize("bad,code,words", [
    (dict(q=None), iu8.E_ARG, "null rows"), (dict(v=None), iu8.E_ARG, "null rows"), (dict(q_out=None), iu8.E_ARG, "null rows"),
    (dict(q=P + 2), iu8.E_ARG, "16 bytes"), (dict(k=P + 8), iu8.E_ARG, "16 bytes"), (dict(q_norm=P + 4), iu8.E_ARG, "16 bytes"),
    (dict(tokens=0), iu8.E_RULE, "nothing to do"), (dict(seqs=0), iu8.E_RULE, "nothing to do"), (dict(cu_q=None), iu8.E_RULE, "one row a sequence"),
    (dict(q_row=24 * 512 - 264), iu8.E_RULE, "cover"), (dict(q_row=24 * 512 + 4), iu8.E_RULE, "cover"), (dict(q_head=248), iu8.E_RULE, "cover"),
    (dict(q_head=260), iu8.E_RULE, "cover"), (dict(kv_row=1016), iu8.E_RULE, "cover"), (dict(kv_row=1028), iu8.E_RULE, "cover"),
    (dict(rot_dim=8), iu8.E_RULE, "rotated"), (dict(rot_dim=272), iu8.E_RULE, "rotated"), (dict(inv_freq=None), iu8.E_ARG, "inv_freq"),
    (dict(eps=-1.0), iu8.E_RULE, "eps"), (dict(eps=math.nan), iu8.E_RULE, "eps"), (dict(eps=math.inf), iu8.E_RULE, "eps"),
    (dict(heads=0), iu8.E_RULE, "whole groups"), (dict(heads=65536), iu8.E_RULE, "whole groups"), (dict(tokens=0x7FFFFFFF), iu8.E_RULE, "32-bit sizes"),
    (dict(tokens=8388608), iu8.E_RULE, "32-bit sizes"), (dict(tokens=8388607), iu8.E_ARG, "null argument"),
    (dict(), iu8.E_ARG, "null argument"), (dict(rot_dim=0, inv_freq=None), iu8.E_ARG, "null argument"),
    (dict(q_norm=None, k_norm=None, eps=-1.0), iu8.E_ARG, "null argument"), (dict(cu_q=None, tokens=3), iu8.E_ARG, "null argument"),
    (dict(q_row=23 * 512 + 256), iu8.E_ARG, "null argument")])       # a last head without its gate behind it
def test_append_refusals(ctx, bad, code, words):
    refused(lambda: append(ctx, **bad), code, words)


@pytest.mark.parametrize("bad,code,words", [
    (dict(q=None), iu8.E_ARG, "null rows"), (dict(out=None), iu8.E_ARG, "null rows"), (dict(out=P + 8), iu8.E_ARG, "16 bytes"),
    (dict(partial=P + 4), iu8.E_ARG, "16 bytes"), (dict(counter=P + 2), iu8.E_ARG, "16 bytes"), (dict(q_row=24 * 256 - 8), iu8.E_RULE, "cover"),
    (dict(q_row=24 * 256 + 4), iu8.E_RULE, "cover"), (dict(scale=math.nan), iu8.E_RULE, "scale"), (dict(scale=math.inf), iu8.E_RULE, "scale"),
    (dict(max_q=0), iu8.E_RULE, "from 1"), (dict(max_kv=1 << 31), iu8.E_RULE, "below 2\\^31"), (dict(max_q=0xFFFFFFFF), iu8.E_RULE, "32-bit sizes"),
    (dict(seqs=0x7FFFFFFE, max_q=1000), iu8.E_RULE, "32-bit sizes"),
    (dict(seqs=1 << 22, max_q=40, partial=None), iu8.E_RULE, "32-bit sizes"), (dict(seqs=(1 << 21) - 1, max_q=40), iu8.E_ARG, "null argument"), (dict(cu_q=None), iu8.E_RULE, "one row a sequence"),
    (dict(), iu8.E_ARG, "null argument"), (dict(partial=None, counter=None), iu8.E_ARG, "null argument"),
    (dict(cu_q=None, seqs=9, max_q=0), iu8.E_ARG, "null argument"), (dict(max_kv=0), iu8.E_ARG, "null argument")])
def test_attn_refusals(ctx, bad, code, words):
    refused(lambda: attend(ctx, **bad), code, words)


def test_workspace_refusals():
    for bad in ((0, 1, 100, 8, 8, 64), (1, 0, 100, 8, 8, 64), (1, 1, 1 << 31, 8, 8, 64), (1, 1, 100, 9, 8, 64), (1, 1, 100, 8, 0, 64), (1, 1, 100, 0, 8, 64),
                (1, 1, 100, 8, 8, 80), (1, 1, 100, 65536, 8, 64), (0xFFFFFFFF, 0xFFFFFFFF, 100, 8, 8, 64), (0xFFFFFFFF, 0x7FFFFFFF, 100, 65535, 1, 64)):
        with pytest.raises(iu8.IU8Error) as e:
            iu8.attn_workspace(*bad)
        assert e.value.code == iu8.E_RULE


def test_workspaces_hold_every_smaller_call():
    """A server allocates once: with fewer sequences, rows or keys the workspaces' sizes never grow, and they are bounded by what
    the card runs at once, whatever the call."""
    rng = random.Random(3)
    assert iu8.attn_workspace(64, 1, 128, 32, 8, 128) == (0, 0) and iu8.attn_workspace(64, 1, 0, 32, 8, 128) == (0, 0)
    for _ in range(4000):
        kvh, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 3, 5, 6, 8, 16, 17, 32, 40]), rng.choice([64, 128, 256])
        most = [rng.choice([1, 2, 9, 64, 300]), rng.choice([1, 2, 5, 40, 200, 9000]), rng.choice([1, 128, 129, 600, 5000, 140000])]
        less = [rng.randint(1, x) for x in most]
        big, small = (iu8.attn_workspace(*s, kvh * group, kvh, dim) for s in (most, less))
        assert small[0] <= big[0] and small[1] <= big[1], (most, less, kvh, group, dim)
        assert big[0] <= 1024 * 128 * (dim + 4) * 4 and big[1] <= 4 * max(most[0] * kvh, 512)


class Other(iu8.KvCache):
    pass


@pytest.mark.parametrize("name", ["kv_append", "attn"])
def test_the_cache_operators_take_the_forms_ctypes_takes(name):
    """Every argument in turn in every form that a caller may have it in, the cache's description among them: the ctypes function's
    result, message or exception. Without a context: the library refuses each call before a launch."""
    op = iu8.operators()
    if isinstance(op, iu8._CtypesOperators):
        pytest.skip("_fastcall is not built for this interpreter")
    f, g = getattr(op, name), getattr(iu8.lib(), "saber_iu8_" + name)
    T = cache()
    good = dict(kv_append=[None, P, P, P, P, T, P, 9, 3, 24, 14336, 512, 14336, P, 64, 0, P, P, 1e-6, None],
                attn=[None, P, 6144, T, P, P, 9, 3, 5, 900, 24, 0.0625, P, P, None])[name]
    assert len(good) == len(g.argtypes)
    forms = []
    for t in g.argtypes:
        if t is ctypes.c_void_p:
            forms.append([None, 0, -1, 1 << 63, ctypes.c_void_p(0), ctypes.c_void_p(64), ctypes.byref(T), b"x", True, np.int64(64), 1.5] if forms else [None])
        elif t is ctypes.c_float:
            forms.append([1, ctypes.c_float(2.0), np.float32(3.0), np.float64(3.0), True, None, "1", math.nan])
        elif t is ctypes.POINTER(iu8.KvCache):
            forms.append([ctypes.byref(T), ctypes.pointer(T), (iu8.KvCache * 1)(), Other(), None, ctypes.addressof(T), iu8.MoeTables(),
                          ctypes.byref(iu8.MoeTables()), ctypes.c_void_p(0), bytearray(ctypes.sizeof(T))])
        else:
            forms.append([8, 1, 0, -1, 9 - (1 << 32), (1 << 32) + 9, 1 << 70, np.int64(9), np.uint32(8), True, t(128), 1.5, None, "128"])

    def outcome(fn, a):
        try:
            return fn(*a), iu8.lib().saber_iu8_last_error()
        except Exception as e:
            return type(e), str(e)

    calls = [good, good[:-1], good + [0], []] + [good[:i] + [v] + good[i + 1:] for i, vs in enumerate(forms) for v in vs]
    assert sum(isinstance(outcome(g, a)[0], int) for a in calls) > len(good)
    for a in calls:
        want = outcome(g, a)
        assert want[0] != 0 and outcome(f, a) == want, (name, a)


# ------------------------------------------------------------------ the cache's order

@pytest.mark.parametrize("kind", [iu8.KV_BF16, iu8.KV_E4M3])
def test_cache_order_is_a_bijection(kind):
    L, pages, h, d, page = iu8.lib(), 3, 2, 64, 32
    size, e = (1, 16) if kind == iu8.KV_E4M3 else (2, 8)
    n = iu8.kv_bytes(pages, h, d, page, kind)
    assert n == pages * h * d * page * size
    at = np.arange(n // size).reshape(pages, h, page // 16, d // e, 16, e) * size
    k_seen, v_seen = set(), set()
    for p in range(pages):
        for b in range(h):
            for t in range(page):
                for c in range(d):
                    k, v = (f(p, b, t, c, h, d, page, kind) for f in (L.saber_iu8_kv_k_offset, L.saber_iu8_kv_v_offset))
                    assert k == at[p, b, t // 16, c // e, t % 16, c % e] and v == (((p * h + b) * page + t) * d + c) * size
                    k_seen.add(k), v_seen.add(v)
    assert k_seen == v_seen == set(range(0, n, size))


def test_cache_offsets_pass_32_bits():
    a = (70000, 1, 3, 5, 8, 256, 64, iu8.KV_BF16)
    block = (70000 * 8 + 1) * 64 * 256 * 2
    assert iu8.lib().saber_iu8_kv_v_offset(*a) == block + (3 * 256 + 5) * 2 > 1 << 33
    assert iu8.lib().saber_iu8_kv_k_offset(*a) == block + 3 * 16 + 5 * 2
    assert iu8.kv_bytes(70001, 8, 256, 64) == 70001 * 8 * 256 * 64 * 2


# ------------------------------------------------------------------ pages

def test_pages_are_dealt_once_and_come_back():
    c = attn.PagedKvCache(3, 2, 64, 200, pages=7, page_tokens=32, device="cpu")
    assert c.table.shape == (3, 7) and (c.table == -1).all() and c.desc.pages == 7 and c.desc.table_stride == 7
    c.reserve(0, 33), c.reserve(2, 1), c.reserve(0, 64), c.reserve(0, 65), c.reserve(1, 0)
    held = [c.table[s][c.table[s] >= 0].tolist() for s in range(3)]
    assert [len(x) for x in held] == [3, 0, 1] and len(set(sum(held, []))) == 4 and (c.table[0, :3] >= 0).all()
    c.reserve(1, 96)
    with pytest.raises(iu8.IU8Error, match="free"):
        c.reserve(2, 33)
    with pytest.raises(iu8.IU8Error, match="hold 200"):
        c.reserve(0, 201)
    c.kv_len[0] = 65
    c.release(0)
    assert (c.table[0] == -1).all() and c.kv_len[0] == 0
    c.reserve(2, 128)
    live = c.table[c.table >= 0].tolist()
    assert len(live) == len(set(live)) == 7 and set(live) == set(range(7))


def test_layer_refusals():
    c = attn.PagedKvCache(3, 2, 64, 200, device="cpu")
    with pytest.raises(iu8.IU8Error, match="one a sequence"):
        attn.AttnLayerIU8(None, c, 4, 4, 256)
    layer = attn.AttnLayerIU8(None, c, 3, 4, 256)
    with pytest.raises(iu8.IU8Error, match="had_t"):
        layer.set_weights(None, None, None, None)
    with pytest.raises(iu8.IU8Error, match="made for"):
        layer.forward(torch.zeros((2, 256), dtype=torch.int16))


# ------------------------------------------------------------------ the built kernels

def test_every_kernel_is_there_with_its_signature():
    text = open(os.path.join(iu8.PREBUILT, "attn_paged.manifest.toml")).read()
    want = {f"{stem}_{kind}_d{d}{tail}" for kind in ("bf16", "e4m3") for d in (64, 128, 256)
            for stem, tail in (("kv_append", ""), ("attn_few", "_r16"), ("attn_few", "_r32"), ("attn_many", ""))}
    assert set(re.findall(r'name = "((?:kv_append|attn)_\w+)"', text)) >= want
    scratch = {n: int(b) for n, b in re.findall(r'name = "(\w+)"(?:(?!\[\[kernel\]\]).)*?private_segment_fixed_size = (\d+)', text, flags=re.S) if int(b)}
    assert not scratch, scratch
    lds = [int(x) for x in re.findall(r"group_segment_fixed_size = (\d+)", text)]
    assert max(lds) <= 160 * 1024


def registers(operand):
    """The vector registers that an operand names."""
    m = re.fullmatch(r"\s*([va])(?:(\d+)|\[(\d+):(\d+)\])\s*", operand)
    if not m:
        return set()
    first, last = (m.group(2), m.group(2)) if m.group(2) else (m.group(3), m.group(4))
    return {(m.group(1), i) for i in range(int(first), int(last) + 1)}


def test_matrix_results_are_read_no_earlier_than_they_are_there(tmp_path):
    """The hardware does not wait where lane arithmetic reads a matrix instruction's result: the compiler owes wait states, over every
    path from it (8 of the 16 x 16 form, 12 of the 32 x 32 one, counted in instructions and the idle cycles that s_nop adds). Behind a
    branch it did not always give them, seen as wrong scores; the kernels read each result in the block that makes it."""
    tool = "/opt/rocm/llvm/bin/llvm-objdump"
    if not os.path.exists(tool):
        tool = shutil.which("llvm-objdump")
    if not tool:
        pytest.skip("no llvm-objdump")
    bundle = open(os.path.join(iu8.PREBUILT, "attn_paged.hsaco"), "rb").read()
    (tmp_path / "object").write_bytes(bundle[bundle.index(b"\x7fELF"):])
    text = subprocess.run([tool, "-d", "--no-show-raw-insn", str(tmp_path / "object")], capture_output=True, text=True, check=True).stdout
    checked = 0
    for name, body in re.findall(r"^[0-9a-f]+ <(attn_\w+)>:\n(.*?)(?=^[0-9a-f]+ <|\Z)", text, flags=re.S | re.M):
        code, place = [], {}
        for line in body.split("\n"):
            m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):?(.*)$", line)
            if m:
                place[int(m.group(2), 16)] = len(code)
                code.append((m.group(1), int(m.group(2), 16)))
        assert code, name

        def after(i):
            op, arg = (code[i][0].split(None, 1) + [""])[:2]
            if op == "s_endpgm":
                return []
            if op.startswith(("s_branch", "s_cbranch")):
                offset = int(arg)
                to = place[code[i][1] + 4 + 4 * (offset - 65536 if offset > 32767 else offset)]
                return [to] if op == "s_branch" else [i + 1, to]
            return [i + 1] if i + 1 < len(code) else []

        for i, (ins, _) in enumerate(code):
            if not ins.startswith("v_mfma"):
                continue
            dst, need, best = registers(ins.split(None, 1)[1].split(",")[0]), 12 if "32x32" in ins else 8, {}
            checked += 1
            assert dst, ins
            ways = [(k, 0) for k in after(i)]
            while ways:
                k, waited = ways.pop()
                if waited >= need or best.get(k, need) <= waited:
                    continue
                best[k] = waited
                op, arg = (code[k][0].split(None, 1) + [""])[:2]
                if op.startswith(("v_", "ds_", "global", "buffer", "flat", "scratch")):
                    operands = arg.split(",")
                    if op.startswith("v_mfma"):
                        assert not (registers(operands[1]) | registers(operands[2])) & dst, (name, ins, code[k][0], waited)
                        if registers(operands[0]) == dst:      # the next of a chain, followed by itself
                            continue
                    else:
                        touched = set().union(*(registers(re.sub(r"\s+(op_sel|clamp|quad_perm|row_|offset|off|sc|nt).*", "", o)) for o in operands))
                        assert not touched & dst, (name, ins, code[k][0], waited)
                idle = int(arg) + 1 if op == "s_nop" else 1
                ways += [(n, waited + idle) for n in after(k)]
    assert checked > 400


GUARDED = [
    ("kv_append_bf16_d128", dict(shape=8 | 2 << 16, form=6 | 64 << 16, pages=10, table_stride=4, tokens=3, seqs=3),
     [dict(shape=8), dict(shape=0), dict(shape=7 | 2 << 16), dict(form=3), dict(form=9), dict(form=6 | 24 << 16), dict(form=6 | 144 << 16), dict(pages=0),
      dict(table_stride=0), dict(table_stride=1 << 25), dict(tokens=0), dict(seqs=0)]),
    ("attn_few_e4m3_d64_r16", dict(shape=8 | 2 << 16, page_shift=6, pages=10, table_stride=4, tokens=3, seqs=3, unit_shift=7, qtiles=1),
     [dict(shape=8), dict(page_shift=3), dict(page_shift=9), dict(pages=-1), dict(table_stride=0), dict(tokens=0), dict(seqs=0), dict(qtiles=0),
      dict(unit_shift=6), dict(unit_shift=32), dict(seqs=1 << 30)]),
    ("attn_many_bf16_d256", dict(shape=8 | 2 << 16, page_shift=6, pages=10, table_stride=4, tokens=300, chunk=128, splits=2, qtiles=3),
     [dict(shape=8), dict(page_shift=3), dict(pages=0), dict(tokens=0), dict(qtiles=0), dict(splits=0), dict(splits=33), dict(chunk=0), dict(chunk=100),
      dict(qtiles=5)])]


@pytest.mark.parametrize("kernel,good,bad", GUARDED)
def test_descriptors_that_the_kernels_do_not_hold(kernel, good, bad):
    """The guard in front of a launch of a descriptor that a caller has set up: refuses by name."""
    guard = ctypes.CDLL(iu8.LIB_PATH)["_ZN3iu810attn_guardEPK14saber_iu8_desc"]

    def check(more, grid=(12, 1, 1), bound=True):
        d = iu8.describe_raw(kernel, grid, 256, "attn_paged", **dict(good, **more))
        for i in range(d.n_args):
            if not bound and d.args[i].name in (b"partial", b"counter"):
                d.args[i].kind = iu8.ARG_NULL_BUFFER
        return guard(ctypes.byref(d))

    assert check({}) == 0
    for more in bad:
        assert check(more) == iu8.E_RULE, more
        assert kernel.encode() in iu8.lib().saber_iu8_last_error()
    assert check({}, grid=(12, 2, 1)) == iu8.E_RULE
    if "attn" in kernel:
        assert check({}, bound=False) == iu8.E_RULE
        assert check(dict(unit_shift=31) if "few" in kernel else dict(splits=1), bound=False) == 0
    if "many" in kernel:
        assert check({}, grid=(13, 1, 1)) == iu8.E_RULE
