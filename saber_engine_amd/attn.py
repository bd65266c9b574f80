"""The attention block of a decoder layer as a launch train over the C ABI: per-token quant -> q, k, v linear -> new tokens into the
paged cache (head norms and rotation on the way) -> causal attention over it -> output gate and requant in the Hadamard basis (or the
plain requant) -> o linear.  Every GEMM keeps the iu8 contract; the train's two linears are W4, as the served layers' are (with W8 ones
the same operators are called one by one).  torch is used for device memory only.
"""
import torch

from . import iu8


def _is(t, dtype, n, device):
    """n values of the type (int16: of its width) or more, in one piece on the device: what a kernel may read from the tensor's address."""
    return (t is not None and (t.dtype == dtype or dtype is torch.int16 and t.dtype.itemsize == 2) and t.numel() >= n and t.is_contiguous() and
            t.device.type == device.type and device.index in (None, t.device.index))


def device_numbers(numbers, device):
    return torch.tensor(numbers, dtype=torch.int32, device=device)


def current_stream(device):
    return torch.cuda.current_stream(device).cuda_stream if device.type == "cuda" else 0


class PagedKvCache:
    """The pages of one layer's sequences. The host deals pages (reserve, release); the table and the counts lie on the device, where
    the kernels read them, so that a captured step follows them; reserve, release, fork, trim and compact write there on torch's current stream. While a step
    runs they must stand still: where steps take another stream than torch's current one, order the two (make it current around reserve, release
    and writes of kv_len, or wait for the step). A page that several sequences share (fork) is whole, and written by none of them: the count of a sequence that has
    been forked, or is a fork, goes back by trim alone, which gives it pages of its own to write in.
    """

    def __init__(self, seqs, kv_heads, head_dim, max_kv, pages=None, page_tokens=64, kind=iu8.KV_BF16, k_scale=None, v_scale=None, device="cuda"):
        """max_kv: the most tokens a sequence may hold; pages: of all sequences together (None: enough for all at that length);
        k_scale, v_scale: an e4m3 cache's scales, f32 [kv_heads]."""
        self.seqs, self.kv_heads, self.head_dim, self.page_tokens, self.kind = seqs, kv_heads, head_dim, page_tokens, kind
        self.max_kv, self.table_stride = max_kv, -(-max_kv // page_tokens)
        self.pages = pages or seqs * self.table_stride
        for s in (k_scale, v_scale):
            if kind == iu8.KV_E4M3 and not _is(s, torch.float32, kv_heads, torch.device(device)):
                raise iu8.IU8Error(iu8.E_ARG, f"an e4m3 cache has a k_scale and a v_scale, f32 [{kv_heads}] on {device}")
        size = iu8.kv_bytes(self.pages, kv_heads, head_dim, page_tokens, kind)
        self.k, self.v = (torch.zeros(size, dtype=torch.uint8, device=device) for _ in range(2))
        self.k_scale, self.v_scale = k_scale, v_scale
        self.table = torch.full((seqs, self.table_stride), -1, dtype=torch.int32, device=device)
        self.kv_len = torch.zeros(seqs, dtype=torch.int32, device=device)
        self._free, self._held = list(range(self.pages - 1, -1, -1)), [[] for _ in range(seqs)]
        self._holders = [0] * self.pages        # sequences that a page belongs to
        scale = [s.data_ptr() if s is not None else None for s in (k_scale, v_scale)]
        self.desc = iu8.KvCache.of(self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(), self.kv_len.data_ptr(), kv_heads=kv_heads,
                                   head_dim=head_dim, page_tokens=page_tokens, pages=self.pages, table_stride=self.table_stride, kind=kind,
                                   k_scale=scale[0], v_scale=scale[1])

    def reserve(self, seq, tokens):
        """Pages for the sequence's first `tokens` positions; those that it has stay."""
        held, want = self._held[seq], -(-tokens // self.page_tokens)
        if tokens > self.max_kv:
            raise iu8.IU8Error(iu8.E_RULE, f"{tokens} tokens; the cache's sequences hold {self.max_kv}")
        if want - len(held) > len(self._free):
            raise iu8.IU8Error(iu8.E_RULE, f"{want - len(held)} more pages wanted, {len(self._free)} free")
        if want > len(held):
            new = self._next(want - len(held))
            self.table[seq, len(held):want] = device_numbers(new, self.table.device)
            self._deal(new)
            held += new

    def release(self, seq):
        """The sequence's pages back (those that another sequence shares stay its), its count to zero."""
        self.table[seq] = -1
        self.kv_len[seq] = 0
        self._back(self._held[seq])
        self._held[seq] = []

    # (What can fail, on the device, comes in front of the books: a call that raises has dealt nothing.)
    def _next(self, n):  # the pages that _deal takes
        return self._free[:-n - 1:-1]

    def _deal(self, pages):
        for p in pages:
            self._free.pop()
            self._holders[p] = 1

    def _back(self, pages):
        for p in reversed(pages):
            self._holders[p] -= 1
            if not self._holders[p]:
                self._free.append(p)

    def _copy(self, ctx, pairs):  # [(page, the page it is copied to)]
        if pairs:
            src, dst = (device_numbers([p[i] for p in pairs], self.table.device) for i in range(2))
            ctx.kv_copy(self.desc, src.data_ptr(), dst.data_ptr(), len(pairs), current_stream(self.table.device))

    def fork(self, ctx, src, dst, tokens):
        """Sequence dst, which has none, gets sequence src's first `tokens` positions: the pages that they fill are shared, the last one, where
        they end inside it, is copied. dst's count becomes `tokens`. More than src counts is refused (its next rows would be written in pages that are shared); a
        count of 0 says nothing, as of pages that are filled before they are counted. The count is read here, which waits for torch's current stream."""
        held, whole, more = self._held[src], tokens // self.page_tokens, tokens % self.page_tokens > 0
        if self._held[dst] or src == dst or tokens < 0 or whole + more > len(held):
            raise iu8.IU8Error(iu8.E_RULE, f"{tokens} tokens of sequence {src}'s {len(held)} pages to sequence {dst}, which has {len(self._held[dst])}")
        if 0 < int(self.kv_len[src]) < tokens:
            raise iu8.IU8Error(iu8.E_RULE, f"{tokens} tokens of sequence {src}, which counts {int(self.kv_len[src])}")
        if more and not self._free:
            raise iu8.IU8Error(iu8.E_RULE, "a page more wanted, none free")
        own = self._next(more)
        new = held[:whole] + own
        self._copy(ctx, [(held[whole], p) for p in own])
        if new:
            self.table[dst, :len(new)] = device_numbers(new, self.table.device)
        self.kv_len[dst] = tokens
        self._deal(own)
        for p in held[:whole]:
            self._holders[p] += 1
        self._held[dst] = new

    def trim(self, ctx, seq, tokens):
        """The sequence's positions from `tokens` on back, as for drafted tokens that were not taken: pages behind them free, its count at most
        `tokens`. A shared page that the sequence would write in next becomes a copy of its own."""
        held, whole, more = self._held[seq], max(tokens, 0) // self.page_tokens, max(tokens, 0) % self.page_tokens > 0
        if whole + more > len(held):
            return
        own = more and self._holders[held[whole]] > 1
        if own and not self._free and all(self._holders[p] > 1 for p in held[whole + 1:]):
            raise iu8.IU8Error(iu8.E_RULE, "a page more wanted, none free")
        last, gone = held[whole:whole + more], held[whole + more:]
        if own:  # (where one of the pages behind comes free, into that)
            page = next((p for p in gone if self._holders[p] == 1), self._free[-1] if self._free else None)
            self._copy(ctx, [(last[0], page)])
            self.table[seq, whole] = page
        self.table[seq, whole + more:] = -1
        self.kv_len[seq].clamp_(max=max(tokens, 0))
        self._back(gone)
        if own:
            self._deal([page])
            self._back(last)
            last = [page]
        self._held[seq] = held[:whole] + last

    def compact(self, ctx):
        """The pages in use to the front of the pool; returns how many they are. Those behind them can then be given up, or another pool's."""
        used = [p for p in range(self.pages) if self._holders[p]]
        n = len(used)
        to = dict(zip([p for p in used if p >= n], [p for p in range(n) if not self._holders[p]]))
        self._copy(ctx, list(to.items()))
        if to:
            moved = {seq: [to.get(p, p) for p in held] for seq, held in enumerate(self._held) if any(p in to for p in held)}
            self.table[device_numbers(list(moved), self.table.device).long()] = device_numbers([h + [-1] * (self.table_stride - len(h)) for h in moved.values()],
                                                                                              self.table.device)
            for old, new in to.items():
                self._holders[new], self._holders[old] = self._holders[old], 0
            for seq, held in moved.items():
                self._held[seq] = held
            self._free = list(range(self.pages - 1, n - 1, -1))
        return n


class AttnLayerIU8:
    def __init__(self, ctx, cache, tokens, heads, hidden, max_q=1, gated=True, inv_freq=None, interleaved=False, eps=1e-6, scale=None):
        """A train for `tokens` rows a call on `cache`'s sequences, up to max_q of them a sequence's (1: one row a sequence in order).
        Trains of other sizes (prompts, decode) may share the cache; calls on it must not overlap in time.
        gated: the projection's rows are [q | gate] a head, then k, then v, and the o linear's weights lie in the Hadamard basis;
        else q, k, v, and o's weights as they are.  inv_freq: f64 [rot_dim / 2] on the device, or None."""
        self.ctx, self.cache, self.T, self.heads, self.H, self.max_q = ctx, cache, tokens, heads, hidden, max_q
        D, kvh, device = cache.head_dim, cache.kv_heads, cache.k.device
        if max_q == 1 and tokens != cache.seqs:
            raise iu8.IU8Error(iu8.E_RULE, f"{tokens} rows of {cache.seqs} sequences, one a sequence")
        if inv_freq is not None and not (2 * len(inv_freq) <= D and _is(inv_freq, torch.float64, len(inv_freq), device)):
            raise iu8.IU8Error(iu8.E_ARG, f"inv_freq: f64, at most {D // 2} of them, on {device}")
        self.gated, self.inv_freq, self.interleaved, self.eps = bool(gated), inv_freq, interleaved, eps
        self.scale = D ** -0.5 if scale is None else scale
        self.n_core, self.q_head = heads * D, 2 * D if gated else D
        self.n_qkv = heads * self.q_head + 2 * kvh * D
        bf = dict(dtype=torch.int16, device=device)
        self.qkv = torch.zeros((tokens, self.n_qkv), **bf)
        self.q, self.core = (torch.zeros((tokens, self.n_core), **bf) for _ in range(2))
        self.out = torch.zeros((tokens, hidden), **bf)
        self.a1, self.a2 = (torch.zeros(iu8.a_bytes(tokens, n), dtype=torch.uint8, device=device) for n in (hidden, self.n_core))
        self.s1, self.s2 = (torch.zeros(tokens, dtype=torch.float32, device=device) for _ in range(2))
        # a sequence's rows: cu_q[s] .. cu_q[s + 1] - 1, the caller's to fill; with one a sequence there is nothing to say
        self.cu_q = torch.zeros(cache.seqs + 1, dtype=torch.int32, device=device) if max_q > 1 else None
        self._ws = [self._workspace(iu8.gemm_workspace(iu8.W4, tokens, n, k)) for n, k in ((self.n_qkv, hidden), (hidden, self.n_core))]
        self._attn_ws = self._workspace(iu8.attn_workspace(cache.seqs, max_q, cache.max_kv, heads, kvh, D))
        # few rows: quantisation and GEMM of a linear in one launch, where the launch law holds it
        self.fused_qkv, self.fused_o = (iu8.fused_holds(tokens, k) for k in (hidden, self.n_core))
        self.had_t = self.q_norm = self.k_norm = None

    def _workspace(self, sizes):  # (scratch, counters: zeroed once, left zero by the kernels)
        device = self.cache.k.device
        return tuple(torch.zeros(n // 4, dtype=torch.int32, device=device) if n else None for n in sizes)

    def set_weights(self, wqkv_frag, wsqkv, wo_frag, wso, had_t=None, q_norm=None, k_norm=None):
        """gfx950 W4 fragments (uint8) and scales (f32) of the two linears; had_t f32 [heads * head_dim] (gated); q_norm, k_norm bf16
        bits [head_dim] or None."""
        if self.gated and had_t is None:
            raise iu8.IU8Error(iu8.E_ARG, "a gated layer's o linear lies in the Hadamard basis: had_t must be given")
        device = self.cache.k.device
        if self.gated and not _is(had_t, torch.float32, self.n_core, device):
            raise iu8.IU8Error(iu8.E_ARG, f"had_t: f32 [{self.n_core}] on {device}")
        for w in (q_norm, k_norm):
            if w is not None and not _is(w, torch.int16, self.cache.head_dim, device):
                raise iu8.IU8Error(iu8.E_ARG, f"head norms: bf16 bits [{self.cache.head_dim}] on {device}")
        self._w = (wqkv_frag, wsqkv, wo_frag, wso)
        self.had_t, self.q_norm, self.k_norm = had_t, q_norm, k_norm

    def forward(self, x, stream=0, max_kv=None):
        """x bf16 bits [T, H] (int16 tensor), the newest tokens of the cache's sequences, whose kv_len already counts them and whose
        pages are reserved; every launch on `stream`. max_kv: what kv_len reaches in this call, where the caller knows it (a
        captured call: in any replay); the cache's length is shared among workgroups accordingly."""
        if tuple(x.shape) != (self.T, self.H):
            raise iu8.IU8Error(iu8.E_RULE, f"rows of shape {tuple(x.shape)}; the train is made for {(self.T, self.H)}")
        if not _is(x, torch.int16, self.T * self.H, self.cache.k.device):
            raise iu8.IU8Error(iu8.E_ARG, f"rows: bf16 bits in one piece on {self.cache.k.device}")
        c, T, D, P = self.ctx, self.T, self.cache.head_dim, lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        wqkv, wsqkv, wo, wso = self._w
        cache, qkv, cu = self.cache.desc, self.qkv.data_ptr(), P(self.cu_q)
        k = qkv + 2 * self.heads * self.q_head
        if self.fused_qkv:
            c.linear_fused(iu8.W4, x.data_ptr(), P(wqkv), P(wsqkv), qkv, T, self.n_qkv, self.H, stream=stream)
        else:
            c.quant(x.data_ptr(), P(self.a1), P(self.s1), T, self.H, stream)
            c.gemm(iu8.W4, P(self.a1), P(self.s1), P(wqkv), P(wsqkv), qkv, T, self.n_qkv, self.H, *map(P, self._ws[0]), stream)
        c.kv_append(qkv, k, k + 2 * self.cache.kv_heads * D, P(self.q), cache, cu, T, self.cache.seqs, self.heads, self.n_qkv, self.q_head,
                    self.n_qkv, P(self.inv_freq), 2 * len(self.inv_freq) if self.inv_freq is not None else 0, self.interleaved,
                    P(self.q_norm), P(self.k_norm), self.eps, stream)
        c.attn(P(self.q), self.n_core, cache, cu, P(self.core), T, self.cache.seqs, self.max_q,
               self.cache.max_kv if max_kv is None else min(max_kv, self.cache.max_kv), self.heads, self.scale, *map(P, self._attn_ws), stream)
        if self.gated:
            c.attn_gate_quant_had(P(self.core), qkv, P(self.a2), P(self.s2), T, self.n_core, D, self.n_qkv, P(self.had_t), stream)
        elif self.fused_o:
            c.linear_fused(iu8.W4, P(self.core), P(wo), P(wso), P(self.out), T, self.H, self.n_core, stream=stream)
            return self.out
        else:
            c.quant(P(self.core), P(self.a2), P(self.s2), T, self.n_core, stream)
        c.gemm(iu8.W4, P(self.a2), P(self.s2), P(wo), P(wso), P(self.out), T, self.H, self.n_core, *map(P, self._ws[1]), stream)
        return self.out
