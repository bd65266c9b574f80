"""Performance cases of the paged key/value cache and the attention that reads it: what stands between a decoder layer's qkv linear
and its output gate, through the public binding.

Two kinds of call:
  append  the projection's rows of new tokens: norm and position rotation of q and k, k and v into the cache's pages
  attn    the new tokens' attention over the cached keys and values: single tokens (decode), a few drafted ones (verify),
          whole prompts or chunks behind a cached prefix; causal, grouped heads, sequences of different lengths packed

The cache is in the library's order: K of one page and head [page / 16][D / E][16 tokens][E] with E the elements of 16 bytes
(8 bf16, 16 e4m3), V [page][D]; values of an e4m3 cache stand for value * scale of their head. `new` rows of a sequence are its
last: row i of n new ones is at position kv_len - n + i.
"""
import functools
import math
import random

import torch

own = False

EPS = 1e-6
BASE = 1e7                    # of the rotation's frequencies: long contexts

# The two attention layers of the benchmark's configurations: the served 27B graph's gated one (24 / 4 heads of 256, 64 of them
# rotated, [q | gate] heads in a row of 14,336) and the generic 27B-class one (40 / 8 heads of 128, a row of 7,168).
GATED = dict(heads=24, kv_heads=4, dim=256, rot=64, gated=True)
DENSE = dict(heads=40, kv_heads=8, dim=128, rot=128, gated=False)


def listed():
    return [
        # one token of one sequence: the smallest call, its launch counts
        dict(name="append_1", kind="append", seqs=1, new=1, kv=5000, page=64, e4m3=False, ragged=False, **GATED),
        # a full decode batch into an 8-bit cache
        dict(name="append_64_e4m3", kind="append", seqs=64, new=1, kv=40000, page=64, e4m3=True, ragged=True, **GATED),
        # prompts of different lengths in one chunk
        dict(name="append_prompts", kind="append", seqs=7, new=1500, kv=1500, page=128, e4m3=False, ragged=True, **DENSE),
        # a decode step of one sequence, a short conversation
        dict(name="decode_1", kind="attn", seqs=1, new=1, kv=1800, page=64, e4m3=False, ragged=False, **GATED),
        # one sequence, a long document in the cache
        dict(name="decode_1_long", kind="attn", seqs=1, new=1, kv=131072, page=128, e4m3=False, ragged=False, **GATED),
        # a large decode batch, lengths as they come
        dict(name="decode_64", kind="attn", seqs=64, new=1, kv=8192, page=64, e4m3=False, ragged=True, **DENSE),
        # the served layer's decode batch on its 8-bit cache
        dict(name="decode_33_e4m3", kind="attn", seqs=33, new=1, kv=16001, page=64, e4m3=True, ragged=True, **GATED),
        # a speculative verify step: five drafted tokens for nine sequences
        dict(name="verify_9x5", kind="attn", seqs=9, new=5, kv=6007, page=32, e4m3=False, ragged=True, **GATED),
        # a short prompt
        dict(name="prompt_200", kind="attn", seqs=1, new=200, kv=200, page=64, e4m3=False, ragged=False, **GATED),
        # prompts of different lengths in one chunk
        dict(name="prompts_5", kind="attn", seqs=5, new=2100, kv=2100, page=128, e4m3=False, ragged=True, **DENSE),
        # a chunk of a long prompt behind what is cached, 8-bit cache
        dict(name="chunk_512_behind_16k", kind="attn", seqs=1, new=512, kv=16896, page=64, e4m3=True, ragged=False, **GATED),
        # a long prompt in one piece
        dict(name="prompt_8192", kind="attn", seqs=1, new=8192, kv=8192, page=128, e4m3=False, ragged=False, **GATED),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(("append", "attn", "attn", "attn"))
        few = rng.random() < 0.5                 # decode and verify, or prompts and chunks
        seqs = _log_int(rng, 1, 128 if few else 16)
        new = rng.choice((1, 1, 1, 2, 3, 4, 5, 8)) if few else _log_int(rng, 9, 8192)
        kv = new + (_log_int(rng, 1, 131072) if few or rng.random() < 0.4 else 0)
        if rng.random() < 0.5:
            shape = dict(rng.choice((GATED, DENSE)))
        else:
            kv_heads, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 256))
            shape = dict(heads=kv_heads * rng.choice((1, 2, 4, 5, 7, 8, 16)), kv_heads=kv_heads, dim=dim,
                         rot=rng.choice((0, dim // 4, dim // 2, dim)), gated=rng.random() < 0.3)
        case = dict(kind=kind, seqs=seqs, new=new, kv=kv, page=rng.choice((16, 32, 64, 128, 256)), e4m3=rng.random() < 0.4,
                    ragged=seqs > 1 and rng.random() < 0.7, **shape)
        scores = seqs * case["heads"] * new * kv          # the plain form holds them all
        cost = work(case)
        if scores <= 1.7e9 and seqs * kv * case["kv_heads"] * case["dim"] <= 6e8 and cost["flops"] <= 8e11 and cost["bytes"] <= 1.2e9:
            return case


def _lengths(case):
    """(new rows, cached keys with the new ones) of each sequence. Ragged: the first as the case says, the others shorter; in a large
    batch of single tokens one place is idle (no keys) where the call allows it."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["new"], case["kv"]))
    got, before = [], case["kv"] - case["new"]
    for i in range(case["seqs"]):
        n, b = case["new"], before
        if case["ragged"] and i:
            n = n if n <= 8 else rng.randint(max(1, n // 8), n)
            b = rng.randint(b // 8, b)
        got.append((n, n + b))
    if case["kind"] == "attn" and case["ragged"] and case["seqs"] >= 16 and case["new"] == 1:
        got[3] = (1, 0)
    return got


class _Made:
    """Seeded values made on the device."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=dtype)

    def cache(self, e4m3, *shape):
        x = self.normal(*shape, dtype=torch.bfloat16)
        return x.mul_(80).clamp_(-448, 448).to(torch.float8_e4m3fn) if e4m3 else x

    def scales(self, n):
        return torch.rand(n, generator=self.g, device="cuda").add_(0.5).div_(80)

    def shuffled(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").int()


def prepare(case, seed):
    r, c = _Made(seed), case
    lens = _lengths(c)
    heads, kvh, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    tokens = sum(n for n, _ in lens)
    st = dict(c, tokens=tokens, max_new=max(n for n, _ in lens), max_kv=max(k for _, k in lens))
    ints = dict(dtype=torch.int32, device="cuda")
    st["kv_len"] = torch.tensor([k for _, k in lens], **ints)
    at = [0]
    for n, _ in lens:
        at.append(at[-1] + n)
    st["cu"] = torch.tensor(at, **ints) if c["new"] > 1 else None      # single tokens: row t is sequence t's
    # pages as they lie after long serving: in no order. The append's pool holds the pages that it writes, the rest are not looked at.
    per = -(-c["kv"] // page)
    if c["kind"] == "attn":
        pages = c["seqs"] * per
        st["table"] = r.shuffled(pages).view(c["seqs"], per)
    else:
        held = c["new"] // page + 2
        pages = c["seqs"] * held
        ring = torch.arange(per, device="cuda") % held
        st["table"] = r.shuffled(pages).view(c["seqs"], held)[:, ring].contiguous()
    e = 16 if c["e4m3"] else 8
    st["k"] = r.cache(c["e4m3"], pages, kvh, page // 16, dim // e, 16, e)
    st["v"] = r.cache(c["e4m3"], pages, kvh, page, dim)
    st["k_scale"], st["v_scale"] = (r.scales(kvh), r.scales(kvh)) if c["e4m3"] else (None, None)
    if c["kind"] == "attn":
        st["q"] = r.normal(tokens, heads, dim, dtype=torch.bfloat16).mul_(1.5)
        st["out"] = torch.zeros(tokens, heads, dim, dtype=torch.bfloat16, device="cuda")
        st["scale"] = 1.0 / math.sqrt(dim)
    else:
        wide = heads * (2 if c["gated"] else 1) + 2 * kvh
        st["rows"] = r.normal(tokens, wide * dim, dtype=torch.bfloat16)
        st["q_norm"], st["k_norm"] = (r.normal(dim).mul_(0.1).bfloat16() if c["gated"] else None for _ in range(2))
        rot = c["rot"]
        st["inv_freq"] = BASE ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / rot) if rot else None
        st["q_out"] = torch.zeros(tokens, heads, dim, dtype=torch.bfloat16, device="cuda")
    return st


# ------------------------------------------------------------------ the framework's calls

@functools.lru_cache(maxsize=None)
def _ctx():
    from saber_engine_amd import iu8
    return iu8.Context()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _plan(st):
    """What a serving program keeps beside the buffers: the cache's descriptor and the attention's workspaces."""
    from saber_engine_amd import iu8
    p = dict(cache=iu8.KvCache.of(st["k"].data_ptr(), st["v"].data_ptr(), st["table"].data_ptr(), st["kv_len"].data_ptr(), kv_heads=st["kv_heads"],
                                  head_dim=st["dim"], page_tokens=st["page"], pages=st["k"].shape[0], table_stride=st["table"].shape[1],
                                  kind=iu8.KV_E4M3 if st["e4m3"] else iu8.KV_BF16, k_scale=_ptr(st["k_scale"]), v_scale=_ptr(st["v_scale"])))
    if st["kind"] == "attn":
        pb, cb = iu8.attn_workspace(st["seqs"], st["max_new"], st["max_kv"], st["heads"], st["kv_heads"], st["dim"])
        p["partial"] = torch.empty(pb, dtype=torch.uint8, device="cuda") if pb else None
        p["counter"] = torch.zeros(cb // 4, dtype=torch.int32, device="cuda") if cb else None
    return p


def _own_append(st):
    plan = st.get("plan") or st.setdefault("plan", _plan(st))
    dim, heads, row = st["dim"], st["heads"], st["rows"].shape[1]
    q_head = dim * (2 if st["gated"] else 1)
    q = st["rows"].data_ptr()
    k = q + 2 * heads * q_head
    _ctx().kv_append(q, k, k + 2 * st["kv_heads"] * dim, st["q_out"].data_ptr(), plan["cache"], _ptr(st["cu"]), st["tokens"], st["seqs"], heads, row, q_head,
                     row, _ptr(st["inv_freq"]), st["rot"], q_norm=_ptr(st["q_norm"]), k_norm=_ptr(st["k_norm"]), eps=EPS,
                     stream=torch.cuda.current_stream().cuda_stream)
    return dict(q=st["q_out"], k=st["k"], v=st["v"])


def _own_attn(st):
    plan = st.get("plan") or st.setdefault("plan", _plan(st))
    _ctx().attn(st["q"].data_ptr(), st["heads"] * st["dim"], plan["cache"], _ptr(st["cu"]), st["out"].data_ptr(), st["tokens"], st["seqs"], st["max_new"],
                st["max_kv"], st["heads"], st["scale"], _ptr(plan["partial"]), _ptr(plan["counter"]), torch.cuda.current_stream().cuda_stream)
    return st["out"]


# ------------------------------------------------------------------ the plain forms

def _places(st):
    """Sequence, row within it and position of every new row."""
    t, kv_len = torch.arange(st["tokens"], device="cuda"), st["kv_len"].long()
    if st["cu"] is None:
        return t, torch.zeros_like(t), kv_len - 1
    cu = st["cu"].long()
    s = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    i = t - cu[s]
    return s, i, kv_len[s] - (cu[s + 1] - cu[s]) + i


def _normed(x, w):
    if w is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (w.float() + 1)


def _rotated(x, pos, inv_freq, rot):
    if not rot:
        return x
    angle = pos.double()[:, None, None] * inv_freq
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)


def _stored(x, scale):
    if scale is None:
        return x.bfloat16().view(torch.int16)
    return (x / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_append(st):
    heads, kvh, dim, page, tokens = st["heads"], st["kv_heads"], st["dim"], st["page"], st["tokens"]
    rows = st["rows"].view(tokens, -1, dim)
    nq = heads * (2 if st["gated"] else 1)
    q = rows[:, 0:nq:2 if st["gated"] else 1].float()
    k, v = rows[:, nq:nq + kvh].float(), rows[:, nq + kvh:].float()
    s, _, pos = _places(st)
    q = _rotated(_normed(q, st["q_norm"]), pos, st["inv_freq"], st["rot"])
    k = _rotated(_normed(k, st["k_norm"]), pos, st["inv_freq"], st["rot"])
    st["q_out"].copy_(q)
    p, o = st["table"][s, pos // page].long(), pos % page
    raw = torch.uint8 if st["e4m3"] else torch.int16
    e = st["k"].shape[-1]
    st["k"].view(raw)[p, :, o // 16, :, o % 16] = _stored(k, st["k_scale"]).view(tokens, kvh, dim // e, e)
    st["v"].view(raw)[p, :, o] = _stored(v, st["v_scale"])
    return dict(q=st["q_out"], k=st["k"], v=st["v"])


def _plain_attn(st):
    heads, kvh, dim, page, seqs = st["heads"], st["kv_heads"], st["dim"], st["page"], st["seqs"]
    table, g, most = st["table"].long(), heads // kvh, st["max_new"]
    raw = torch.uint8 if st["e4m3"] else torch.int16
    kind = st["k"].dtype
    keys = table.shape[1] * page
    k = st["k"].view(raw)[table].view(kind).permute(0, 2, 1, 3, 5, 4, 6).float().reshape(seqs, kvh, keys, dim)
    v = st["v"].view(raw)[table].view(kind).permute(0, 2, 1, 3, 4).float().reshape(seqs, kvh, keys, dim)
    if st["e4m3"]:
        k, v = k * st["k_scale"][:, None, None], v * st["v_scale"][:, None, None]
    s, i, pos = _places(st)
    q = torch.zeros(seqs, most, heads, dim, device="cuda")
    q[s, i] = st["q"].float()
    at = torch.full((seqs, most), -1, dtype=torch.long, device="cuda")
    at[s, i] = pos
    q = q.view(seqs, most, kvh, g, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, g * most, dim)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(seqs, kvh, g, most, keys).mul_(st["scale"])
    seen = torch.arange(keys, device="cuda") <= at[:, :, None]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=-3e38)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(seqs, kvh, g * most, keys), v).view(seqs, kvh, g, most, dim) / total.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)
    return out[s, i].bfloat16()


def run(state):
    if own:
        return _own_append(state) if state["kind"] == "append" else _own_attn(state)
    return _plain_append(state) if state["kind"] == "append" else _plain_attn(state)


def work(case):
    lens = _lengths(case)
    tokens, dim, heads, kvh = sum(n for n, _ in lens), case["dim"], case["heads"], case["kv_heads"]
    size = 1 if case["e4m3"] else 2
    if case["kind"] == "append":
        return dict(bytes=tokens * dim * (4 * heads + 2 * kvh * (2 + size)), flops=tokens * dim * (heads + kvh) * 6)
    pairs = sum(n * k - n * (n - 1) // 2 for n, k in lens if k)
    return dict(bytes=2 * size * dim * kvh * sum(k for _, k in lens) + 4 * tokens * heads * dim, flops=4 * dim * heads * pairs)


# ------------------------------------------------------------------ in 64 bits, one sequence (and head) after the other

def _exact_append(st, lens):
    heads, kvh, dim, page = st["heads"], st["kv_heads"], st["dim"], st["page"]
    x = st["rows"].double()
    step = 2 * dim if st["gated"] else dim
    e = st["k"].shape[-1]
    out_q = torch.empty(st["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    out_k, out_v = st["k"].double(), st["v"].double()
    flat_k, flat_v = out_k.view(-1), out_v.view(-1)
    ch = torch.arange(dim, device="cuda")
    t = 0
    for s, (n, total) in enumerate(lens):
        pos = torch.arange(total - n, total, device="cuda")
        pages = st["table"][s].long()[pos // page]
        part = x[t:t + n]

        def head(at, w):
            y = part[:, at:at + dim]
            if w is not None:
                y = y / torch.sqrt((y * y).sum(1, keepdim=True) / dim + EPS) * (1 + w.double())
            if st["rot"]:
                h = st["rot"] // 2
                z = torch.complex(y[:, :h], y[:, h:2 * h]) * torch.exp(1j * pos.double()[:, None] * st["inv_freq"])
                y = torch.cat((z.real, z.imag, y[:, 2 * h:]), 1)
            return y

        for h in range(heads):
            out_q[t:t + n, h] = head(h * step, st["q_norm"])
        for h in range(kvh):
            k = head(heads * step + h * dim, st["k_norm"])
            v = part[:, heads * step + (kvh + h) * dim:][:, :dim]
            if st["e4m3"]:
                k, v = (k / st["k_scale"][h].double()).clamp(-448, 448), (v / st["v_scale"][h].double()).clamp(-448, 448)
            block = (pages * kvh + h) * page * dim
            o = pos % page
            flat_v[(block + o * dim)[:, None] + ch] = v
            flat_k[(block + (o // 16) * 16 * dim + (o % 16) * e)[:, None] + (ch // e) * 16 * e + ch % e] = k
        t += n
    return dict(q=out_q, k=out_k, v=out_v)


def _exact_attn(st, lens):
    heads, kvh, dim, page = st["heads"], st["kv_heads"], st["dim"], st["page"]
    g, e = heads // kvh, st["k"].shape[-1]
    out = torch.zeros(st["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    ch = torch.arange(dim, device="cuda")
    raw = torch.uint8 if st["e4m3"] else torch.int16
    flat_k, flat_v = st["k"].view(raw).view(-1), st["v"].view(raw).view(-1)
    t = 0
    for s, (n, total) in enumerate(lens):
        if total:
            pos = torch.arange(total, device="cuda")
            pages, o = st["table"][s].long()[pos // page], pos % page
            for h in range(kvh):
                block = (pages * kvh + h) * page * dim
                v = flat_v[(block + o * dim)[:, None] + ch].view(st["v"].dtype).double()
                k = flat_k[(block + (o // 16) * 16 * dim + (o % 16) * e)[:, None] + (ch // e) * 16 * e + ch % e].view(st["k"].dtype).double()
                if st["e4m3"]:
                    k, v = k * st["k_scale"][h].double(), v * st["v_scale"][h].double()
                hidden = pos[None, :] > (total - n + torch.arange(n, device="cuda"))[:, None]
                for j in range(h * g, (h + 1) * g):
                    score = (st["q"][t:t + n, j].double() @ k.t()) * st["scale"]
                    out[t:t + n, j] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
        t += n
    return out


def exact(case, seed):
    st = prepare(case, seed)
    lens = _lengths(case)
    return _exact_append(st, lens) if case["kind"] == "append" else _exact_attn(st, lens)
