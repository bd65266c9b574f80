"""Performance cases of a delta-net layer's core and of the copies that fork a sequence, through the public binding.

Four kinds of call:
  conv    the projection's rows of new tokens through the short causal convolution and SiLU, the last inputs kept for the next call
  delta   the gated delta rule over those rows: single tokens (decode), a few drafted ones of which only some enter the state
          (verify), whole prompts or chunks on a state that is there
  pages   pages of a paged key/value cache to other pages: a sequence forked, a pool compacted
  states  the delta-net states and convolution tails of sequences to other slots, where sequences are forked

Sequences of different lengths are packed; sequence s's state and tail lie in slot[s]. A head's state is f32 [128 of the key][128 of the
value]; value head h reads key head h / (heads / key_heads).
"""
import functools
import math
import random

import torch

own = False

EPS = 1e-6
DIM = 128                     # of a head's keys and values

# The served 27B graph's delta-net layers: 16 key heads, 48 value heads, rows [q | k | v | z] of 16,384 and [b | a] of 96.
SERVED = dict(key_heads=16, heads=48)
# Its attention layers' cache, and the generic 27B-class one's
GATED = dict(kv_heads=4, dim=256)
DENSE = dict(kv_heads=8, dim=128)


def listed():
    return [
        # one token of one sequence
        dict(name="conv_1", kind="conv", seqs=1, new=1, width=4, ragged=False, bias=False, **SERVED),
        # prompts of different lengths in one call
        dict(name="conv_prompts", kind="conv", seqs=5, new=2100, width=4, ragged=True, bias=False, **SERVED),
        # a decode step of one sequence
        dict(name="delta_1", kind="delta", seqs=1, new=1, kept=False, ragged=False, **SERVED),
        # a large decode batch: bound by the states
        dict(name="delta_64", kind="delta", seqs=64, new=1, kept=False, ragged=False, **SERVED),
        # a speculative verify step: five drafted tokens of nine sequences, the state behind the accepted ones
        dict(name="verify_9x5", kind="delta", seqs=9, new=5, kept=True, ragged=True, **SERVED),
        # a short prompt
        dict(name="prompt_200", kind="delta", seqs=1, new=200, kept=False, ragged=False, **SERVED),
        # prompts of different lengths in one call
        dict(name="prompts_5", kind="delta", seqs=5, new=2100, kept=False, ragged=True, **SERVED),
        # a long prompt in one piece
        dict(name="prompt_8192", kind="delta", seqs=1, new=8192, kept=False, ragged=False, **SERVED),
        # a sequence forked in the middle of a page
        dict(name="fork_page", kind="pages", pages=1, page=64, e4m3=False, **GATED),
        # a pool compacted
        dict(name="compact_700", kind="pages", pages=700, page=128, e4m3=False, **DENSE),
        # a prompt's state to seven samples
        dict(name="fork_7_states", kind="states", copies=7, width=4, spread=True, **SERVED),
        # a batch of sequences, each into another slot
        dict(name="copy_33_states", kind="states", copies=33, width=4, spread=False, **SERVED),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(("conv", "delta", "delta", "delta", "delta", "pages", "states"))
        key_heads = rng.choice((1, 2, 4, 8, 16))
        heads = dict(SERVED) if rng.random() < 0.5 else dict(key_heads=key_heads, heads=key_heads * rng.choice((1, 2, 3, 4)))
        if kind in ("conv", "delta"):
            few = rng.random() < 0.5                  # decode and verify, or prompts
            seqs = _log_int(rng, 1, 128 if few else 16)
            new = rng.choice((1, 1, 1, 2, 3, 4, 5, 8)) if few else _log_int(rng, 9, 8192)
            case = dict(kind=kind, seqs=seqs, new=new, ragged=seqs > 1 and new > 1 and rng.random() < 0.7, **heads)
            if kind == "conv":
                case.update(width=rng.choice((2, 3, 4, 4)), bias=rng.random() < 0.3)
            else:
                case.update(kept=1 < new <= 8 and rng.random() < 0.5)
        elif kind == "pages":
            case = dict(kind=kind, pages=_log_int(rng, 1, 4000), page=rng.choice((16, 32, 64, 128, 256)), e4m3=rng.random() < 0.4,
                        kv_heads=rng.choice((1, 2, 4, 8)), dim=rng.choice((64, 128, 256)))
        else:
            case = dict(kind=kind, copies=_log_int(rng, 1, 64), width=rng.choice((2, 3, 4, 4)), spread=rng.random() < 0.4, **heads)
        cost = work(case)
        if cost["bytes"] <= 7e8 and cost["flops"] <= 3.8e10:
            return case


def _lengths(case):
    """New rows of each sequence. Ragged: the first as the case says, the others shorter; in a larger batch one place is idle."""
    if not case["ragged"]:
        return [case["new"]] * case["seqs"]
    rng = random.Random("%d %d" % (case["seqs"], case["new"]))
    got = [case["new"]] + [rng.randint(max(1, case["new"] // 8), case["new"]) for _ in range(case["seqs"] - 1)]
    if case["seqs"] >= 9:
        got[3] = 0
    return got


def _channels(case):
    return (2 * case["key_heads"] + case["heads"]) * DIM


class _Made:
    """Seeded values made on the device."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=dtype)

    def uniform(self, lo, hi, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda").mul_(hi - lo).add_(lo)

    def whole(self, least, past, n):
        return torch.randint(least, past, (n,), generator=self.g, device="cuda", dtype=torch.int32)

    def shuffled(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").int()


def prepare(case, seed):
    r, c = _Made(seed), case
    st = dict(c)
    if c["kind"] == "pages":
        n = 2 * c["pages"]
        e = 16 if c["e4m3"] else 8
        values = [r.normal(n, c["kv_heads"], c["page"] * c["dim"], dtype=torch.bfloat16) for _ in range(2)]
        if c["e4m3"]:
            values = [v.mul_(80).clamp_(-448, 448).to(torch.float8_e4m3fn) for v in values]
        st["k"] = values[0].view(n, c["kv_heads"], c["page"] // 16, c["dim"] // e, 16, e)
        st["v"] = values[1].view(n, c["kv_heads"], c["page"], c["dim"])
        order = r.shuffled(n)                                     # pages as they lie after long serving: in no order
        st["src"], st["dst"] = order[:c["pages"]].contiguous(), order[c["pages"]:].contiguous()
        st["scale"] = torch.ones(c["kv_heads"], device="cuda") if c["e4m3"] else None
        st["table"], st["kv_len"] = order.view(1, n), torch.zeros(1, dtype=torch.int32, device="cuda")
        return st
    channels = st["channels"] = _channels(c)
    if c["kind"] == "states":
        st["slots"] = 2 * c["copies"]
        st["state"] = r.normal(st["slots"], c["heads"], DIM, DIM).mul_(0.1)
        st["tail"] = r.normal(st["slots"], c["width"] - 1, channels, dtype=torch.bfloat16)
        order = r.shuffled(st["slots"])
        st["src"], st["dst"] = order[:c["copies"]].contiguous(), order[c["copies"]:].contiguous()
        if c["spread"]:
            st["src"].fill_(st["src"][0])
        return st
    lens = _lengths(c)
    tokens = st["tokens"] = sum(lens)
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    st["cu"] = torch.tensor(at, dtype=torch.int32, device="cuda") if c["new"] > 1 else None     # single tokens: row t is sequence t's
    st["slots"] = c["seqs"] + 3
    st["slot"] = r.shuffled(st["slots"])[:c["seqs"]].contiguous()
    if c["kind"] == "conv":
        st["rows"] = r.normal(tokens, channels + c["heads"] * DIM, dtype=torch.bfloat16)         # [q | k | v | z]
        st["weight"] = r.uniform(-0.5, 0.5, channels, c["width"]).bfloat16()
        st["bias"] = r.uniform(-0.1, 0.1, channels).bfloat16() if c["bias"] else None
        st["tail"] = r.normal(st["slots"], c["width"] - 1, channels, dtype=torch.bfloat16)
        st["out"] = torch.zeros(tokens, channels, dtype=torch.bfloat16, device="cuda")
        return st
    x = r.normal(tokens, channels, dtype=torch.bfloat16)
    st["rows"] = x.mul_(torch.sigmoid(x))                          # behind the convolution's SiLU: [q | k | v]
    st["ba"] = r.normal(tokens, 2 * c["heads"], dtype=torch.bfloat16)
    # decays as such layers are made: a rate of up to 16 a head, steps of 0.001 to 0.1
    step = torch.exp(r.uniform(math.log(0.001), math.log(0.1), c["heads"]))
    st["a_log"], st["dt_bias"] = torch.log(r.uniform(0.01, 16.0, c["heads"])), step + torch.log(-torch.expm1(-step))
    st["state"] = r.normal(st["slots"], c["heads"], DIM, DIM).mul_(0.1)
    st["kept"] = torch.minimum(r.whole(0, c["new"] + 1, c["seqs"]), torch.tensor(lens, dtype=torch.int32, device="cuda")) if c["kept"] else None
    st["out"] = torch.zeros(tokens, c["heads"], DIM, dtype=torch.bfloat16, device="cuda")
    st["scale"] = DIM ** -0.5
    return st


# ------------------------------------------------------------------ the framework's calls

@functools.lru_cache(maxsize=None)
def _ctx():
    from saber_engine_amd import iu8
    return iu8.Context()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_conv(st):
    _ctx().gdn_conv(st["rows"].data_ptr(), st["rows"].shape[1], st["weight"].data_ptr(), st["tail"].data_ptr(), st["slots"], st["out"].data_ptr(), st["channels"],
                    st["tokens"], st["seqs"], st["channels"], st["width"], bias=_ptr(st["bias"]), slot=st["slot"].data_ptr(), cu_q=_ptr(st["cu"]), stream=_stream())
    return dict(out=st["out"], tail=st["tail"])


def _workspace(st):
    """What a serving program keeps beside the buffers."""
    from saber_engine_amd import iu8
    n = iu8.gdn_workspace(st["tokens"], st["seqs"], st["new"], st["key_heads"], st["heads"])
    return dict(memory=torch.empty(n, dtype=torch.uint8, device="cuda") if n else None)


def _own_delta(st):
    plan = st.get("plan") or st.setdefault("plan", _workspace(st))
    q, ba = st["rows"].data_ptr(), st["ba"].data_ptr()
    keys = 2 * st["key_heads"] * DIM
    _ctx().gdn(q, q + keys, q + 2 * keys, st["channels"], ba + 2 * st["heads"], ba, 2 * st["heads"], st["a_log"].data_ptr(), st["dt_bias"].data_ptr(),
               st["state"].data_ptr(), st["slots"], st["out"].data_ptr(), st["tokens"], st["seqs"], st["new"], st["key_heads"], st["heads"], st["scale"], EPS,
               slot=st["slot"].data_ptr(), cu_q=_ptr(st["cu"]), kept=_ptr(st["kept"]), workspace=_ptr(plan["memory"]), stream=_stream())
    return dict(out=st["out"], state=st["state"])


def _cache(st):
    from saber_engine_amd import iu8
    return iu8.KvCache.of(st["k"].data_ptr(), st["v"].data_ptr(), st["table"].data_ptr(), st["kv_len"].data_ptr(), kv_heads=st["kv_heads"], head_dim=st["dim"],
                          page_tokens=st["page"], pages=st["k"].shape[0], table_stride=st["table"].shape[1], kind=iu8.KV_E4M3 if st["e4m3"] else iu8.KV_BF16,
                          k_scale=_ptr(st["scale"]), v_scale=_ptr(st["scale"]))


def _own_pages(st):
    cache = st.get("cache") or st.setdefault("cache", _cache(st))
    _ctx().kv_copy(cache, st["src"].data_ptr(), st["dst"].data_ptr(), st["pages"], stream=_stream())
    return dict(k=st["k"], v=st["v"])


def _own_states(st):
    _ctx().gdn_copy(st["state"].data_ptr(), st["tail"].data_ptr(), st["slots"], st["heads"], st["channels"], st["width"], st["src"].data_ptr(), st["dst"].data_ptr(),
                    st["copies"], stream=_stream())
    return dict(state=st["state"], tail=st["tail"])


# ------------------------------------------------------------------ the plain forms

def _places(st):
    """Sequence and row within it of every new row, and each sequence's rows."""
    t = torch.arange(st["tokens"], device="cuda")
    if st["cu"] is None:
        return t, torch.zeros_like(t), torch.ones_like(t)
    cu = st["cu"].long()
    s = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return s, t - cu[s], cu[1:] - cu[:-1]


def _plain_conv(st):
    behind, seqs, slot = st["width"] - 1, st["seqs"], st["slot"].long()
    s, i, n = _places(st)
    tails = st["tail"][slot]
    inputs = torch.cat((tails.view(seqs * behind, -1), st["rows"][:, :st["channels"]]))            # the tails in front of all rows

    def back(s, i, t, by):
        """Where the input `by` rows in front of row i of sequence s lies; t: where the sequence's row i does."""
        return torch.where(i >= by, seqs * behind + t - by, s * behind + behind + i - by)

    w, t = st["weight"].float(), torch.arange(st["tokens"], device="cuda")
    y = sum(inputs[back(s, i, t, behind - j)].float() * w[:, j] for j in range(st["width"]))
    if st["bias"] is not None:
        y = y + st["bias"].float()
    st["out"].copy_(y * torch.sigmoid(y))
    every = torch.arange(seqs, device="cuda").repeat_interleave(behind)
    by = torch.arange(behind, 0, -1, device="cuda").repeat(seqs)
    first = torch.cumsum(n, 0) - n
    st["tail"][slot] = inputs[back(every, n[every], (first + n)[every], by)].view_as(tails)
    return dict(out=st["out"], tail=st["tail"])


def _unit(x):
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPS)


def _plain_delta(st):
    """In chunks of up to 64 rows; within one by the inverse of a unit triangular matrix, from chunk to chunk by the state."""
    kh, heads, seqs, slot = st["key_heads"], st["heads"], st["seqs"], st["slot"].long()
    s, i, n = _places(st)
    size = min(64, st["new"])
    chunks = -(-st["new"] // size)

    def dealt(x):                                                  # [tokens, heads, ...] to [chunk, sequence, head, row, ...]; no row: zeros
        y = torch.zeros(seqs, chunks * size, *x.shape[1:], device="cuda", dtype=x.dtype)
        y[s, i] = x
        y = y.view(seqs, chunks, size, *x.shape[1:]).movedim(1, 0)
        return y.movedim(3, 2).contiguous()

    rows = st["rows"].float().view(st["tokens"], -1, DIM)
    q, k, v = dealt(_unit(rows[:, :kh]) * st["scale"]), dealt(_unit(rows[:, kh:2 * kh])), dealt(rows[:, 2 * kh:])
    q, k = (x.repeat_interleave(heads // kh, 2) for x in (q, k))
    beta = dealt(torch.sigmoid(st["ba"][:, :heads].float()))
    g = -torch.exp(st["a_log"]) * torch.nn.functional.softplus(st["ba"][:, heads:].float() + st["dt_bias"])
    total = dealt(g).double().cumsum(-1)
    row = torch.arange(size, device="cuda")
    lower = row[:, None] >= row
    decay = torch.where(lower, total[..., :, None] - total[..., None, :], -math.inf).exp().float()
    kt = k.transpose(-1, -2).contiguous()
    a = (k @ kt) * decay * beta[..., None] * (row[:, None] > row)
    inverse = torch.eye(size, device="cuda").expand_as(a).clone()
    for j in range(1, size):                                       # row j of (1 + a)^-1 from those above
        inverse[..., j, :] -= (a[..., j, None, :] @ inverse).squeeze(-2)
    inverse = inverse * beta[..., None, :]
    inner = (q @ kt) * decay
    from_start = total.exp().float()[..., None]
    state = st["state"][slot]
    out = torch.empty(chunks, seqs, heads, size, DIM, device="cuda")
    if st["kept"] is None:
        last, keeps = total[..., -1:], torch.ones_like(total, dtype=torch.bool)
    else:                                                          # (drafted rows: one chunk)
        kept = st["kept"].long()[None, :, None, None].expand(1, seqs, heads, 1)
        last = torch.where(kept > 0, total.gather(-1, (kept - 1).clamp(min=0)), 0.0)
        keeps = row < kept
    to_end = torch.where(keeps, last - total, -math.inf).exp().float()[..., None]
    for c in range(chunks):
        u = inverse[c] @ (v[c] - from_start[c] * (k[c] @ state))
        out[c] = from_start[c] * (q[c] @ state) + inner[c] @ u
        state = last[c].exp().float()[..., None] * state + kt[c] @ (to_end[c] * u)
    st["state"][slot] = state
    st["out"].copy_(out.movedim(0, 1).movedim(3, 2).reshape(seqs, chunks * size, heads, DIM)[s, i])
    return dict(out=st["out"], state=st["state"])


def _plain_pages(st):
    src, dst, raw = st["src"].long(), st["dst"].long(), torch.uint8 if st["e4m3"] else torch.bfloat16
    k, v = st["k"].view(raw), st["v"].view(raw)
    k[dst], v[dst] = k[src], v[src]
    return dict(k=st["k"], v=st["v"])


def _plain_states(st):
    src, dst = st["src"].long(), st["dst"].long()
    st["state"][dst], st["tail"][dst] = st["state"][src], st["tail"][src]
    return dict(state=st["state"], tail=st["tail"])


def run(state):
    kind = state["kind"]
    if own:
        return dict(conv=_own_conv, delta=_own_delta, pages=_own_pages, states=_own_states)[kind](state)
    return dict(conv=_plain_conv, delta=_plain_delta, pages=_plain_pages, states=_plain_states)[kind](state)


def work(case):
    c = case
    if c["kind"] == "pages":
        return dict(bytes=2 * 2 * c["pages"] * c["kv_heads"] * c["page"] * c["dim"] * (1 if c["e4m3"] else 2), flops=0)
    channels = _channels(c)
    if c["kind"] == "states":
        a_slot = 4 * c["heads"] * DIM * DIM + 2 * (c["width"] - 1) * channels
        return dict(bytes=a_slot * (c["copies"] + (1 if c["spread"] else c["copies"])), flops=0)
    lens = _lengths(c)
    tokens, live = sum(lens), sum(n > 0 for n in lens)
    if c["kind"] == "conv":
        return dict(bytes=4 * channels * (tokens + live * (c["width"] - 1)) + 2 * channels * (c["width"] + c["bias"]), flops=tokens * channels * (2 * c["width"] + 4))
    return dict(bytes=tokens * (2 * channels + 2 * c["heads"] * DIM + 4 * c["heads"]) + 8 * live * c["heads"] * DIM * DIM,
                flops=6 * tokens * c["heads"] * DIM * DIM)


# ------------------------------------------------------------------ in 64 bits, one row after the other

def _exact_conv(st, lens):
    out, tail = torch.empty(st["tokens"], st["channels"], dtype=torch.float64, device="cuda"), st["tail"].double()
    w, t = st["weight"].double().t().contiguous(), 0
    for s, n in enumerate(lens):
        x = torch.cat((tail[st["slot"][s]], st["rows"][t:t + n, :st["channels"]].double()))
        y = torch.zeros(n, st["channels"], dtype=torch.float64, device="cuda")
        for j in range(st["width"]):
            y += x[j:j + n] * w[j]
        if st["bias"] is not None:
            y += st["bias"].double()
        out[t:t + n] = y / (1 + torch.exp(-y))
        tail[st["slot"][s]] = x[n:]
        t += n
    return dict(out=out, tail=tail)


def _exact_delta(st, lens):
    kh, heads, longest = st["key_heads"], st["heads"], max(lens)
    out, state = torch.zeros(st["tokens"], heads, DIM, dtype=torch.float64, device="cuda"), st["state"].double()
    begin, n = torch.zeros(len(lens), dtype=torch.long, device="cuda"), torch.tensor(lens, device="cuda")
    begin[1:] = n.cumsum(0)[:-1]
    kept = n if st["kept"] is None else st["kept"].long()
    of = torch.arange(heads, device="cuda") // (heads // kh)
    b, a = st["ba"].double().split(heads, 1)
    rate = -torch.exp(st["a_log"].double())
    now = state[st["slot"].long()]                                 # [sequence, head, key, value]
    held = now.clone()
    for i in range(longest):
        on = (n > i).nonzero()[:, 0]
        t = begin[on] + i
        x = st["rows"][t].double().view(len(on), -1, DIM)
        q, k, v = x[:, :kh][:, of], x[:, kh:2 * kh][:, of], x[:, 2 * kh:]
        q, k = (y / torch.sqrt((y * y).sum(2, keepdim=True) + EPS) for y in (q, k))
        step = a[t] + st["dt_bias"].double()
        past = now[on] * torch.exp(rate * torch.logaddexp(step, torch.zeros_like(step)))[:, :, None, None]
        told = (past * k[..., None]).sum(2)
        past += k[..., None] * ((v - told) / (1 + torch.exp(-b[t]))[..., None])[:, :, None, :]
        now[on] = past
        out[t] = st["scale"] * (past * q[..., None]).sum(2)
        enters = on[kept[on] > i]
        held[enters] = now[enters]
    state[st["slot"].long()] = held
    return dict(out=out, state=state)


def exact(case, seed):
    if case["kind"] in ("pages", "states"):                        # copies: nothing is computed
        return None
    if case["kind"] == "delta" and case["new"] * max(8, case["seqs"] * case["heads"] / 48) > 70000:
        return None
    st = prepare(case, seed)
    return (_exact_conv if case["kind"] == "conv" else _exact_delta)(st, _lengths(case))
