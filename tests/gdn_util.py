"""A delta-net layer's core from its definition, in 64 bits on the host, with how far a kernel may be off: what the GPU tests compare with."""
import numpy as np
import torch

from tests.attn_util import BF16, F32, f64

D = 128
# Roundings of f32 that one row's update may leave in a column of the state, of the column's length and its value: the sum over the keys (a
# chain of 16 and a tree of 3, or a matrix product's 12 steps of 32), the norm of k (sum, root, quotient, product: 12, twice), the gates
# (exponentials and logarithms of 2 units each, 8), the update itself (3).
ROW = 96
# What enters an answer alone is rounded to f16 in the chunked form (half a step of 2^-11 relative): the state of Q S, both factors of the inner matrix times U
F16 = 2.0 ** -11
# ... and no finer than f16's last step, 2^-24, of the column's unit, which is at most half of the largest value that the column has in the chunk (its
# inputs and the state in front of it): half a step of that, of the 128 values of S under |q^| = 1 (their sum at most sqrt(128)) and of the 64 of U; in the
# state, of those of S under |k^| = 1, and of the 64 rests V - .. and the 64 updates that each chunk splits.
STEP = 2.0 ** -26
FLOOR, STATE_FLOOR = (128 ** 0.5 + 64) * STEP, (128 ** 0.5 + 128) * STEP


def gates(a, b, a_log, dt_bias):
    """decay, beta of rows a, b [n, heads]."""
    with np.errstate(over="ignore"):
        g = -np.exp(a_log) * np.logaddexp(a + dt_bias, 0.0)
        return np.exp(np.maximum(g, -1e4)), 1 / (1 + np.exp(-b))


def rule(q, k, v, a, b, a_log, dt_bias, state, eps, scale, chunked=False):
    """q, k f64 [n, key_heads, 128], v [n, heads, 128], a, b [n, heads], state [heads, 128, 128]. Returns (out, its tolerance, the states
    behind 0 .. n rows, their tolerances [.., heads, 1, 128]).

    The tolerances: a column's error goes through each row's update as the column does, by decay (1 - beta k^ k^T), which lengthens nothing, and each row
    adds ROW roundings of the column's length and its value. An answer has the column's error (|q^| = 1), the same roundings of its own sum,
    in the chunked form f16 factors beside the state in front of the chunk and its updates, and is rounded once. (In chunks: a row's update is
    a sum of at most 64 inputs with weights of at most 1, made with ten roundings of f32 at most, each factor of a product that is f32 taken to 2^-22, four roundings more, or to 2^-25 of the column's
    unit, at most eight times its largest value: 64 roundings of the column's length once over the keys. Their 64-fold is less than what the chunk's rows add up to.)"""
    n, heads = v.shape[:2]
    of = np.arange(heads) // (heads // k.shape[1])
    decay, beta = gates(a, b, a_log, dt_bias)
    s, e = state.copy(), np.zeros((heads, D))
    out, tol, states, tols = np.zeros(v.shape), np.zeros(v.shape), [s.copy()], [e.copy()]
    mass = held = floor = np.zeros((heads, D))
    for i in range(n):
        kh = k[i, of] / np.sqrt((k[i, of] ** 2).sum(-1, keepdims=True) + eps)
        qh = q[i, of] / np.sqrt((q[i, of] ** 2).sum(-1, keepdims=True) + eps)
        length = np.sqrt((s ** 2).sum(1))
        if i % 64 == 0:
            e = e + floor
            floor = STATE_FLOOR * (length + np.abs(v[i:i + 64]).max(0)) * chunked
            start, held, mass = length, length.copy(), np.zeros((heads, D))
        s = s * decay[i][:, None, None]
        u = beta[i][:, None] * (v[i] - np.einsum("hkv,hk->hv", s, kh))
        s = s + kh[:, :, None] * u[:, None, :]
        new = np.sqrt((s ** 2).sum(1))
        e = e * decay[i][:, None] + ROW * F32 * (length + new + np.abs(v[i]))
        held, mass = held * decay[i][:, None], mass * decay[i][:, None] + np.abs(u)
        out[i] = scale * np.einsum("hkv,hk->hv", s, qh)
        slack = e + floor + ROW * F32 * (length + new + np.abs(v[i]))
        if chunked:
            slack += F16 * (held + 2.01 * mass) + FLOOR * (start + np.abs(v[i - i % 64:i - i % 64 + 64]).max(0))
        tol[i] = BF16 * np.abs(out[i]) * 1.01 + abs(scale) * slack + 1e-30
        states.append(s), tols.append(e + floor)
    return out, tol, states, [t[:, None, :] + 1e-30 for t in tols]


def convolved(x, tail, weight, bias):
    """x f64 [n, channels], tail [width - 1, channels], weight [channels, width]: the output and its tolerance (width + 4 roundings of f32 of the sum of
    magnitudes before a function whose slope is at most 1.1, 8 of its own, one rounding to bf16)."""
    n, width = len(x), weight.shape[1]
    every = np.concatenate((tail, x))
    y, size = np.zeros(x.shape), np.zeros(x.shape)
    for w in range(width):
        y += every[w:w + n] * weight[:, w]
        size += np.abs(every[w:w + n] * weight[:, w])
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    out = y / (1 + np.exp(-y))
    return out, BF16 * np.abs(out) * 1.01 + F32 * (1.1 * (width + 4) * size + 8 * np.abs(out)) + 1e-30


def ends(lens, front=0):
    return torch.tensor(front + np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32, device="cuda")


class Rows:
    """Rows, gates, weights and states of a call on the device; what no sequence has is NaN."""

    def __init__(self, key_heads, heads, lens, slots=None, front=0, behind=0, more=0, seed=0, like=0.0, a_at=0.0, old=True):
        """like: how much the keys have in common; a_at: added to the decays' input; more: channels between a row's end and the next's."""
        g = torch.Generator().manual_seed(seed)
        self.kh, self.heads, self.lens, self.seqs = key_heads, heads, list(lens), len(lens)
        self.slots = slots or self.seqs + 2
        live, self.tokens, self.front = sum(lens), front + sum(lens) + behind, front
        self.row = (2 * key_heads + heads) * D + more
        x = torch.randn(live, self.row, generator=g)
        if like:
            x[:, key_heads * D:2 * key_heads * D] = x[:, key_heads * D:2 * key_heads * D] * (1 - like) + like * torch.randn(1, key_heads * D, generator=g)
        self.rows = torch.full((self.tokens, self.row), float("nan"), dtype=torch.bfloat16)
        self.rows[front:front + live] = x.bfloat16()
        self.ab = torch.full((self.tokens, 2 * heads + 3), float("nan"), dtype=torch.bfloat16)
        self.ab[front:front + live] = (torch.randn(live, 2 * heads + 3, generator=g) * 1.5).bfloat16()
        self.ab[front:front + live, :heads] += a_at
        self.a_log = torch.log(torch.rand(heads, generator=g) * 8 + 0.01)
        self.dt_bias = torch.randn(heads, generator=g) - 2
        self.state = torch.randn(self.slots, heads, D, D, generator=g) * (0.3 if old else 0)
        self.slot = torch.randperm(self.slots, generator=g)[:self.seqs].int()
        self.cu = ends(self.lens, front)
        self.out = torch.full((self.tokens, heads, D), 7.0, dtype=torch.bfloat16)
        for n in "rows ab a_log dt_bias state slot out".split():
            setattr(self, n, getattr(self, n).cuda())
        self.eps, self.scale = 1e-6, D ** -0.5

    def call(self, ctx, packed=True, max_q=None, kept=None, workspace=None, out=True, stream=0, tokens=None):
        q = self.rows.data_ptr()
        keys = 2 * self.kh * D
        ctx.gdn(q if out else None, q + keys, q + 2 * keys, self.row, self.ab.data_ptr(), self.ab.data_ptr() + 2 * self.heads, self.ab.shape[1], self.a_log.data_ptr(),
                self.dt_bias.data_ptr(), self.state.data_ptr(), self.slots, self.out.data_ptr() if out else None, tokens or self.tokens, self.seqs,
                max_q or max(self.lens), self.kh, self.heads, self.scale, self.eps, slot=self.slot.data_ptr(), cu_q=self.cu.data_ptr() if packed else None,
                kept=kept.data_ptr() if kept is not None else None, workspace=workspace.data_ptr() if workspace is not None else None, stream=stream)

    def want(self, was, chunked=False):
        """Per sequence (first row, the rule's results) from the states `was`."""
        x, ab = f64(self.rows.float()), f64(self.ab.float())
        t, keys = self.front, self.kh * D
        for s, n in enumerate(self.lens):
            r, p = x[t:t + n], int(self.slot[s])
            if 0 <= p < self.slots:
                yield s, t, p, rule(r[:, :keys].reshape(n, self.kh, D), r[:, keys:2 * keys].reshape(n, self.kh, D), r[:, 2 * keys:2 * keys + self.heads * D].reshape(n, self.heads, D),
                                    ab[t:t + n, :self.heads], ab[t:t + n, self.heads:2 * self.heads], f64(self.a_log), f64(self.dt_bias), was[p], self.eps, self.scale,
                                    chunked)
            t += n
