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


class PagedKvCache:
    """The pages of one layer's sequences. The host deals pages (reserve, release); the table and the counts lie on the device, where
    the kernels read them, so that a captured step follows them; reserve and release write there on torch's current stream. While a step
    runs they must stand still: where steps take another stream than torch's current one, order the two (make it current around reserve, release
    and writes of kv_len, or wait for the step)."""

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
            new = [self._free.pop() for _ in range(want - len(held))]
            self.table[seq, len(held):want] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
            held += new

    def release(self, seq):
        """The sequence's pages back, its count to zero."""
        self._free += reversed(self._held[seq])
        self._held[seq] = []
        self.table[seq] = -1
        self.kv_len[seq] = 0


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
