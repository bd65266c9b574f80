"""The delta-net block of a decoder layer as a launch train over the C ABI: per-token quant -> q, k, v, z and b, a linears -> short causal
convolution -> gated delta rule -> norm, output gate and requant in the Hadamard basis -> o linear.  Every GEMM keeps the iu8 contract; the
train's linears are W4.  torch is used for device memory only.
"""
import torch

from . import iu8
from .attn import _is, current_stream, device_numbers

DIM = 128    # of a head's keys and values


class GdnState:
    """One layer's states and convolution tails, a slot a live sequence. The host deals slots (begin, release); their table lies on the device,
    where the kernels read it, so that a captured step follows it; begin, release and fork write there on torch's current stream. While a step
    runs it must stand still: where steps take another stream than torch's current one, order the two."""

    def __init__(self, seqs, key_heads, heads, slots=None, width=4, device="cuda"):
        """slots: sequences that may be live at once (None: all); a sequence that is not has no slot, and calls pass its rows over."""
        if min(seqs, key_heads, heads) < 1 or heads % key_heads or not 2 <= width <= 4 or slots is not None and slots < 1:
            raise iu8.IU8Error(iu8.E_RULE, f"{seqs} sequences, {heads} heads over {key_heads} key heads, a convolution of {width} inputs, {slots} slots")
        self.seqs, self.key_heads, self.heads, self.width, self.slots = seqs, key_heads, heads, width, slots or seqs
        self.channels = (2 * key_heads + heads) * DIM
        self.state = torch.zeros((self.slots, heads, DIM, DIM), dtype=torch.float32, device=device)
        self.tail = torch.zeros((self.slots, width - 1, self.channels), dtype=torch.int16, device=device)
        self.slot = torch.full((seqs,), -1, dtype=torch.int32, device=device)
        self._free, self._held = list(range(self.slots - 1, -1, -1)), [None] * seqs

    def _take(self, seq):  # (what can fail, on the device, in front of the books)
        self.slot[seq] = self._free[-1]
        self._held[seq] = self._free.pop()

    def begin(self, seq):
        """A slot for the sequence, its state and tail zeros."""
        if self._held[seq] is not None:
            raise iu8.IU8Error(iu8.E_RULE, f"sequence {seq} has a state already")
        if not self._free:
            raise iu8.IU8Error(iu8.E_RULE, f"a state more wanted, none of {self.slots} free")
        self.state[self._free[-1]].zero_()
        self.tail[self._free[-1]].zero_()
        self._take(seq)

    def release(self, seq):
        """The sequence's slot back."""
        if self._held[seq] is not None:
            self.slot[seq] = -1
            self._free.append(self._held[seq])
            self._held[seq] = None

    def fork(self, ctx, src, dsts):
        """Sequence src's memory to each of dsts, which have none yet."""
        if self._held[src] is None or len(set(dsts)) != len(dsts) or any(self._held[d] is not None for d in dsts) or len(dsts) > len(self._free):
            raise iu8.IU8Error(iu8.E_RULE, f"sequence {src} to {list(dsts)}: a source with a state, targets without, and {len(dsts)} of {len(self._free)} free slots")
        if dsts:
            device = self.state.device
            of, to = device_numbers([self._held[src]] * len(dsts), device), device_numbers(self._free[:-len(dsts) - 1:-1], device)
            ctx.gdn_copy(self.state.data_ptr(), self.tail.data_ptr(), self.slots, self.heads, self.channels, self.width, of.data_ptr(), to.data_ptr(), len(dsts),
                         current_stream(device))
            for d in dsts:
                self._take(d)


class GdnLayerIU8:
    def __init__(self, ctx, state, tokens, hidden, max_q=1, eps=1e-6, scale=None):
        """A train for `tokens` rows a call on `state`'s sequences, up to max_q of them a sequence's (1: one row a sequence in order).
        Trains of other sizes (prompts, decode) may share the state; calls on it must not overlap in time. The linears' rows are
        [q | k | v | z] and [b | a]."""
        self.ctx, self.state, self.T, self.H, self.max_q, self.eps = ctx, state, tokens, hidden, max_q, eps
        if max_q == 1 and tokens != state.seqs:
            raise iu8.IU8Error(iu8.E_RULE, f"{tokens} rows of {state.seqs} sequences, one a sequence")
        self.scale = DIM ** -0.5 if scale is None else scale
        device, channels = state.state.device, state.channels
        self.n_core = state.heads * DIM
        self.n_qkvz, self.n_ba = channels + self.n_core, 2 * state.heads
        bf = dict(dtype=torch.int16, device=device)
        self.qkvz, self.ba, self.qkv = (torch.zeros((tokens, n), **bf) for n in (self.n_qkvz, self.n_ba, channels))
        self.core, self.out = torch.zeros((tokens, self.n_core), **bf), torch.zeros((tokens, hidden), **bf)
        self.a1, self.a2 = (torch.zeros(iu8.a_bytes(tokens, n), dtype=torch.uint8, device=device) for n in (hidden, self.n_core))
        self.s1, self.s2 = (torch.zeros(tokens, dtype=torch.float32, device=device) for _ in range(2))
        # a sequence's rows: cu_q[s] .. cu_q[s + 1] - 1, the caller's to fill; with one a sequence there is nothing to say
        self.cu_q = torch.zeros(state.seqs + 1, dtype=torch.int32, device=device) if max_q > 1 else None
        self._ws = [self._workspace(iu8.gemm_workspace(iu8.W4, tokens, n, k)) for n, k in ((self.n_qkvz, hidden), (self.n_ba, hidden), (hidden, self.n_core))]
        n = iu8.gdn_workspace(tokens, state.seqs, max_q, state.key_heads, state.heads)
        self._gdn_ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
        self.paired = tokens <= 32 and self._pairs()

    def _pairs(self):  # the two linears that read the rows in one launch
        try:
            iu8.pair(iu8.resolve(iu8.W4, self.T, self.n_qkvz, self.H), iu8.resolve(iu8.W4, self.T, self.n_ba, self.H))
            return True
        except iu8.IU8Error:
            return False

    def _workspace(self, sizes):  # (scratch, counters: zeroed once, left zero by the kernels)
        device = self.state.state.device
        return tuple(torch.zeros(n // 4, dtype=torch.int32, device=device) if n else None for n in sizes)

    def set_weights(self, wqkvz_frag, wsqkvz, wba_frag, wsba, wo_frag, wso, conv, a_log, dt_bias, norm, had_t, conv_bias=None):
        """gfx950 W4 fragments (uint8) and scales (f32) of the three linears; conv bf16 bits [channels, width], conv_bias [channels] or None; a_log,
        dt_bias f32 [heads]; norm bf16 bits [128]; had_t f32 [heads * 128]: the o linear's weights lie in the Hadamard basis."""
        st, device = self.state, self.state.state.device
        for t, dtype, n, what in ((conv, torch.int16, st.channels * st.width, "conv: bf16 bits"), (a_log, torch.float32, st.heads, "a_log: f32"),
                                  (dt_bias, torch.float32, st.heads, "dt_bias: f32"), (norm, torch.int16, DIM, "norm: bf16 bits"), (had_t, torch.float32, self.n_core, "had_t: f32")):
            if not _is(t, dtype, n, device):
                raise iu8.IU8Error(iu8.E_ARG, f"{what}, {n} of them on {device}")
        if conv_bias is not None and not _is(conv_bias, torch.int16, st.channels, device):
            raise iu8.IU8Error(iu8.E_ARG, f"conv_bias: bf16 bits, {st.channels} of them on {device}")
        self._w = (wqkvz_frag, wsqkvz, wba_frag, wsba, wo_frag, wso)
        self.conv, self.conv_bias, self.a_log, self.dt_bias, self.norm, self.had_t = conv, conv_bias, a_log, dt_bias, norm, had_t

    def _core(self, kept, out, stream):
        c, st, P = self.ctx, self.state, lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        if kept is not None and not _is(kept, torch.int32, st.seqs, st.state.device):
            raise iu8.IU8Error(iu8.E_ARG, f"kept: int32 [{st.seqs}] on {st.state.device}")
        c.gdn_conv(P(self.qkvz), self.n_qkvz, P(self.conv), P(st.tail), st.slots, P(self.qkv), st.channels, self.T, st.seqs, st.channels, st.width, P(self.conv_bias),
                   P(st.slot), P(self.cu_q), P(kept), stream)
        q, keys = P(self.qkv), 2 * st.key_heads * DIM
        c.gdn(q, q + keys, q + 2 * keys, st.channels, P(self.ba) + 2 * st.heads, P(self.ba), self.n_ba, P(self.a_log), P(self.dt_bias), P(st.state), st.slots,
              P(out), self.T, st.seqs, self.max_q, st.key_heads, st.heads, self.scale, self.eps, P(st.slot), P(self.cu_q), P(kept), P(self._gdn_ws), stream)

    def forward(self, x, stream=0, kept=None):
        """x bf16 bits [T, H] (int16 tensor), the newest tokens of the state's sequences; every launch on `stream`. kept (int32 [seqs] on the device): the
        rows by which each sequence's memory moves on, where not by all: zeros for drafted rows, which accept() then counts."""
        if tuple(x.shape) != (self.T, self.H):
            raise iu8.IU8Error(iu8.E_RULE, f"rows of shape {tuple(x.shape)}; the train is made for {(self.T, self.H)}")
        if not _is(x, torch.int16, self.T * self.H, self.state.state.device):
            raise iu8.IU8Error(iu8.E_ARG, f"rows: bf16 bits in one piece on {self.state.state.device}")
        c, T, P = self.ctx, self.T, lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        wqkvz, wsqkvz, wba, wsba, wo, wso = self._w
        c.quant(x.data_ptr(), P(self.a1), P(self.s1), T, self.H, stream)
        if self.paired:
            c.gemm_pair(P(self.a1), P(self.s1), P(wqkvz), P(wsqkvz), P(self.qkvz), self.n_qkvz, P(wba), P(wsba), P(self.ba), self.n_ba, T, self.H, stream)
        else:
            c.gemm(iu8.W4, P(self.a1), P(self.s1), P(wqkvz), P(wsqkvz), P(self.qkvz), T, self.n_qkvz, self.H, *map(P, self._ws[0]), stream)
            c.gemm(iu8.W4, P(self.a1), P(self.s1), P(wba), P(wsba), P(self.ba), T, self.n_ba, self.H, *map(P, self._ws[1]), stream)
        self._core(kept, self.core, stream)
        c.gdn_norm_quant_had(P(self.core), P(self.qkvz) + 2 * self.state.channels, self.n_qkvz, P(self.norm), P(self.a2), P(self.s2), T, self.n_core, self.eps,
                             P(self.had_t), stream)
        c.gemm(iu8.W4, P(self.a2), P(self.s2), P(wo), P(wso), P(self.out), T, self.H, self.n_core, *map(P, self._ws[2]), stream)
        return self.out

    def accept(self, kept, stream=0):
        """Moves the sequences' memory on by the first kept[s] rows of the last forward, which left it where it was (kept of zeros)."""
        self._core(kept, None, stream)
