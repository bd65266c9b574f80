"""CPU tests of a delta-net layer's core and the copies of a sequence (csrc/host/gdn.cpp): refusals, the forms that arguments take, the workspace's law, and what
the built kernels are like."""
import ctypes
import math
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

from saber_engine_amd import iu8, kbuild
from tests.test_attn_host import CACHES, cache, refused, registers

P = 1 << 40        # an address: nothing here is launched


@pytest.fixture(scope="module", autouse=True)
def built():
    if not os.path.exists(iu8.LIB_PATH) or not os.path.exists(os.path.join(iu8.PREBUILT, "delta_net.manifest.toml")):
        kbuild.build_all()


@pytest.fixture(params=["fastcall", "ctypes"])
def ctx(request):
    """A context that is not open: what the library does not refuse by itself it refuses for that."""
    c = iu8.Context.__new__(iu8.Context)
    c._h, c._addr, c._op = ctypes.c_void_p(), None, iu8._CtypesOperators() if request.param == "ctypes" else iu8.operators()
    return c


def conv(c, **more):
    a = dict(x=P, x_row=16384, weight=P, tail=P, slots=5, out=P, out_row=10240, tokens=9, seqs=3, channels=10240, width=4, bias=P, slot=P, cu_q=P, kept=P)
    a.update(more)
    c.gdn_conv(**a)


def rule(c, **more):
    a = dict(q=P, k=P, v=P, row=10240, a=P, b=P, ab_row=96, a_log=P, dt_bias=P, state=P, slots=5, out=P, tokens=9, seqs=3, max_q=100, key_heads=16, heads=48, scale=0.09,
             eps=1e-6, slot=P, cu_q=P, kept=None, workspace=P)
    a.update(more)
    c.gdn(**a)


def copy(c, **more):
    a = dict(state=P, tail=P, slots=5, heads=48, channels=10240, width=4, src=P, dst=P, n=2)
    a.update(more)
    c.gdn_copy(**a)


@pytest.mark.parametrize("bad,code,words", [
    (dict(x=None), iu8.E_ARG, "must be given"), (dict(weight=None), iu8.E_ARG, "must be given"), (dict(tail=None), iu8.E_ARG, "must be given"),
    (dict(out=None), iu8.E_ARG, "must be given"), (dict(x=P + 2), iu8.E_ARG, "16 bytes"), (dict(tail=P + 8), iu8.E_ARG, "16 bytes"), (dict(bias=P + 2), iu8.E_ARG, "16 bytes"),
    (dict(out=P + 4), iu8.E_ARG, "16 bytes"), (dict(tokens=0), iu8.E_RULE, "nothing to do"), (dict(seqs=0), iu8.E_RULE, "nothing to do"),
    (dict(seqs=(1 << 31) - 1), iu8.E_RULE, "nothing to do"), (dict(cu_q=None), iu8.E_RULE, "one row a sequence"), (dict(slots=0), iu8.E_RULE, "slots"),
    (dict(slots=1 << 31), iu8.E_RULE, "slots"), (dict(slot=None, slots=2), iu8.E_RULE, "no table"), (dict(width=1), iu8.E_RULE, "hold 2, 3 and 4"),
    (dict(width=5), iu8.E_RULE, "hold 2, 3 and 4"), (dict(channels=0), iu8.E_RULE, "multiple of 8"), (dict(channels=1004), iu8.E_RULE, "multiple of 8"),
    (dict(x_row=10232), iu8.E_RULE, "cover"), (dict(x_row=16388), iu8.E_RULE, "cover"), (dict(out_row=10232), iu8.E_RULE, "cover"), (dict(out_row=10244), iu8.E_RULE, "cover"),
    (dict(x_row=1 << 31), iu8.E_RULE, "cover"), (dict(tokens=(1 << 31) - 1, channels=1 << 20, x_row=1 << 20, out_row=1 << 20), iu8.E_RULE, "32-bit sizes")])
def test_convolutions_that_are_refused(ctx, bad, code, words):
    refused(lambda: conv(ctx, **bad), code, words)


@pytest.mark.parametrize("bad,code,words", [
    (dict(q=None), iu8.E_ARG, "must be given"), (dict(k=None), iu8.E_ARG, "must be given"), (dict(v=None), iu8.E_ARG, "must be given"), (dict(a=None), iu8.E_ARG, "must be given"),
    (dict(b=None), iu8.E_ARG, "must be given"), (dict(a_log=None), iu8.E_ARG, "must be given"), (dict(dt_bias=None), iu8.E_ARG, "must be given"),
    (dict(state=None), iu8.E_ARG, "must be given"), (dict(q=P + 8), iu8.E_ARG, "16 bytes"), (dict(state=P + 4), iu8.E_ARG, "16 bytes"), (dict(workspace=P + 8), iu8.E_ARG, "16 bytes"),
    (dict(out=P + 2), iu8.E_ARG, "16 bytes"), (dict(a=P + 1), iu8.E_ARG, "elements"), (dict(dt_bias=P + 2), iu8.E_ARG, "elements"),
    (dict(tokens=0), iu8.E_RULE, "nothing to do"), (dict(seqs=0), iu8.E_RULE, "nothing to do"), (dict(cu_q=None), iu8.E_RULE, "one row a sequence"),
    (dict(slots=0), iu8.E_RULE, "slots"), (dict(slot=None, slots=2), iu8.E_RULE, "no table"), (dict(heads=40), iu8.E_RULE, "whole groups"), (dict(key_heads=0), iu8.E_RULE, "whole groups"),
    (dict(heads=1 << 16, row=1 << 24, ab_row=1 << 16), iu8.E_RULE, "whole groups"), (dict(max_q=0), iu8.E_RULE, "at most 0"), (dict(row=48 * 128 - 8), iu8.E_RULE, "cover"),
    (dict(row=10244), iu8.E_RULE, "cover"), (dict(ab_row=40), iu8.E_RULE, "cover"), (dict(eps=-1.0), iu8.E_RULE, "eps"), (dict(eps=math.nan), iu8.E_RULE, "eps"),
    (dict(scale=math.inf), iu8.E_RULE, "scale"), (dict(seqs=1 << 20, tokens=1 << 20, slots=1 << 20, max_q=1), iu8.E_RULE, "32-bit sizes"),
    (dict(seqs=1 << 20, tokens=1 << 22, slots=1 << 20), iu8.E_RULE, "32-bit sizes"), (dict(seqs=1 << 17, tokens=1 << 22, slots=1 << 17), iu8.E_RULE, "32-bit sizes"),
    (dict(row=(1 << 24) + 8), iu8.E_RULE, "16777224 elements")])
def test_rules_that_are_refused(ctx, bad, code, words):
    refused(lambda: rule(ctx, **bad), code, words)


@pytest.mark.parametrize("bad,code,words", [
    (dict(state=None), iu8.E_ARG, "must be given"), (dict(tail=None), iu8.E_ARG, "must be given"), (dict(state=P + 4), iu8.E_ARG, "16 bytes"), (dict(src=None), iu8.E_ARG, "src and dst"),
    (dict(dst=None), iu8.E_ARG, "src and dst"), (dict(heads=0), iu8.E_RULE, "whole groups"), (dict(channels=12), iu8.E_RULE, "multiple of 8"), (dict(width=1), iu8.E_RULE, "hold 2, 3"),
    (dict(slots=0), iu8.E_RULE, "slots")])
def test_copies_that_are_refused(ctx, bad, code, words):
    refused(lambda: copy(ctx, **bad), code, words)


@pytest.mark.parametrize("bad,code,words", CACHES[:-4] + CACHES[-4:])
def test_caches_whose_pages_are_not_copied(ctx, bad, code, words):
    if "kv_heads" in bad and bad["kv_heads"]:
        return                                                     # (any count of kv heads: no query heads stand beside them)
    refused(lambda: ctx.kv_copy(cache(**bad), P, P, 3), code, words)
    for a in ((None, P), (P, None)):
        refused(lambda: ctx.kv_copy(cache(), *a, 3), iu8.E_ARG, "src and dst")
    refused(lambda: ctx.kv_copy(cache(), P, P, 3), iu8.E_ARG, "null argument")


def test_no_context_is_refused(ctx):
    for call in (conv, rule, copy, lambda c: rule(c, workspace=None), lambda c: rule(c, kept=P, out=None, q=None), lambda c: conv(c, cu_q=None, tokens=3, slot=None, kept=None, bias=None),
                 lambda c: rule(c, cu_q=None, tokens=3, slot=None), lambda c: c.kv_copy(cache(), P, P, 3)):
        refused(lambda: call(ctx), iu8.E_ARG, "null argument")
    refused(lambda: copy(ctx, n=0), iu8.E_ARG, "null argument")


class Other(iu8.KvCache):
    pass


@pytest.mark.parametrize("name", ["gdn_conv", "gdn", "gdn_copy", "kv_copy"])
def test_the_operators_take_the_forms_ctypes_takes(name):
    """Every argument in turn in every form that a caller may have it in: the ctypes function's result, message or exception. Without a context: the library
    refuses each call before a launch."""
    op = iu8.operators()
    if isinstance(op, iu8._CtypesOperators):
        pytest.skip("_fastcall is not built for this interpreter")
    f, g = getattr(op, name), getattr(iu8.lib(), "saber_iu8_" + name)
    T = cache()
    good = dict(gdn_conv=[None, P, 16384, P, P, P, 5, P, P, P, P, 10240, 9, 3, 10240, 4, None],
                gdn=[None, P, P, P, 10240, P, P, 96, P, P, P, 5, P, P, None, P, 9, 3, 100, 16, 48, 1e-6, 0.09, P, None],
                gdn_copy=[None, P, P, 5, 48, 10240, 4, P, P, 2, None], kv_copy=[None, T, P, P, 2, None])[name]
    assert len(good) == len(g.argtypes)
    forms = []
    for t in g.argtypes:
        if t is ctypes.c_void_p:
            forms.append([None, 0, -1, 1 << 63, ctypes.c_void_p(0), ctypes.c_void_p(64), ctypes.byref(T), b"x", True, np.int64(64), 1.5] if forms else [None])
        elif t is ctypes.c_float:
            forms.append([1, ctypes.c_float(2.0), np.float32(3.0), np.float64(3.0), True, None, "1", math.nan])
        elif t is ctypes.POINTER(iu8.KvCache):
            forms.append([ctypes.byref(T), ctypes.pointer(T), (iu8.KvCache * 1)(), Other(), None, ctypes.addressof(T), iu8.MoeTables(), ctypes.c_void_p(0),
                          bytearray(ctypes.sizeof(T))])
        else:
            forms.append([8, 1, -1, 9 - (1 << 32), (1 << 32) + 9, 1 << 70, np.int64(9), np.uint32(8), True, t(128), 1.5, None, "128"])

    def outcome(fn, a):
        try:
            return fn(*a), iu8.lib().saber_iu8_last_error()
        except Exception as e:
            return type(e), str(e)

    calls = [good, good[:-1], good + [0], []] + [good[:i] + [v] + good[i + 1:] for i, vs in enumerate(forms) for v in vs]
    for a in calls:
        want = outcome(g, a)
        assert want[0] != 0 and outcome(f, a) == want, (name, a)


def test_workspaces_hold_every_smaller_call():
    bytes_of = iu8.gdn_workspace
    assert bytes_of(64, 64, 1, 16, 48) == bytes_of(300, 60, 5, 16, 48) == 0
    rng = np.random.default_rng(0)
    for _ in range(300):
        tokens, seqs = (int(2 ** rng.uniform(0, 16)) for _ in range(2))
        most = bytes_of(tokens, seqs, 4096, 2, 6)
        assert most % 16 == 0 and most >= bytes_of(int(rng.integers(1, tokens + 1)), int(rng.integers(1, seqs + 1)), int(rng.integers(1, 4097)), 2, 6)
        # a chunk's place: (first row / 64) + sequence + its number among the sequence's, no two the same, all in the workspace
        lens = rng.multinomial(tokens, np.ones(seqs) / seqs) if seqs < 3000 else []
        at, seen = 0, set()
        for s, n in enumerate(lens):
            for c in range(-(-int(n) // 64)):
                place = at // 64 + s + c
                assert place not in seen and (place + 1) * (2 * 32768 + 6 * 19456) <= most
                seen.add(place)
            at += int(n)
    for bad in ((0, 1, 9, 2, 6), (9, 0, 9, 2, 6), (9, 1, 9, 4, 6), (9, 1, 9, 0, 6)):
        with pytest.raises(iu8.IU8Error):
            bytes_of(*bad)


# ------------------------------------------------------------------ the built kernels

def test_every_kernel_is_there_without_scratch():
    text = open(os.path.join(iu8.PREBUILT, "delta_net.manifest.toml")).read()
    want = {"block_copy", "delta_step_c16", "delta_step_c32", "delta_prep"} | {f"delta_conv_w{w}" for w in (2, 3, 4)} | {f"delta_scan_w{w}" for w in (2, 4)}
    assert set(re.findall(r'name = "((?:delta_|block_)\w+)"', text)) >= want
    assert set(re.findall(r"private_segment_fixed_size = (\d+)", text)) == {"0"}
    assert max(int(x) for x in re.findall(r"group_segment_fixed_size = (\d+)", text)) <= 160 * 1024


@pytest.mark.parametrize("kernel", ["delta_step_c16", "delta_prep", "delta_scan_w4", "delta_conv_w3", "block_copy"])
def test_descriptors_of_the_kernels_are_refused(kernel):
    """Their walks follow sizes that the operators check: no launch by a descriptor that a caller has set up."""
    d = iu8.describe_raw(kernel, (1, 1, 1), 256, "delta_net")
    assert d.kernel.decode() == kernel and d.n_args
    with pytest.raises(iu8.IU8Error):
        iu8.Context.launch(type("C", (), {"_h": ctypes.c_void_p()})(), d, {})


def listing(tmp_path):
    """The delta kernels' instructions, as llvm-objdump prints them: (name, text) each."""
    tool = "/opt/rocm/llvm/bin/llvm-objdump"
    if not os.path.exists(tool):
        tool = shutil.which("llvm-objdump")
    if not tool:
        pytest.skip("no llvm-objdump")
    bundle = open(os.path.join(iu8.PREBUILT, "delta_net.hsaco"), "rb").read()
    (tmp_path / "object").write_bytes(bundle[bundle.index(b"\x7fELF"):])
    text = subprocess.run([tool, "-d", "--no-show-raw-insn", str(tmp_path / "object")], capture_output=True, text=True, check=True).stdout
    return re.findall(r"^[0-9a-f]+ <(delta_\w+)>:\n(.*?)(?=^[0-9a-f]+ <|\Z)", text, flags=re.S | re.M)


def test_matrix_results_are_read_no_earlier_than_they_are_there(tmp_path):
    """The wait states that the compiler owes between a matrix instruction and the first lane instruction that reads its result, over every path from it (8 of the bf16 form,
    10 of the f32 one, counted in instructions and the idle cycles of s_nop): tests/test_attn_host.py has why."""
    checked = 0
    for name, body in listing(tmp_path):
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
            dst, need, best = registers(ins.split(None, 1)[1].split(",")[0]), 10 if "x4_f32" in ins else 8, {}
            checked += 1
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
    assert checked > 250


def test_lanes_are_read_no_earlier_than_they_are_there(tmp_path):
    """A lane operation that reads other lanes' registers (DPP) comes two wait states behind the one that wrote them; in asm the compiler does not see to it."""
    checked = 0
    for name, body in listing(tmp_path):
        code = [m.group(1) for m in re.finditer(r"^\s+(\S.*?)\s*// [0-9A-F]+", body, flags=re.M)]
        for i, ins in enumerate(code):
            if not ins.startswith("v_fmac_f32_dpp"):
                continue
            source, waited, k = registers(ins.split(",")[1].strip().lstrip("-").split()[0]), 0, i
            checked += 1
            while waited < 2 and k:
                k -= 1
                op, arg = (code[k].split(None, 1) + [""])[:2]
                assert not (op.startswith("v_") and registers(arg.split(",")[0].strip()) & source), (name, code[k], ins)
                waited += int(arg) + 1 if op == "s_nop" else 1
    assert checked >= 100
