"""The paged cache and its attention from their definitions, in 64 bits on the host: what the GPU tests compare with."""
import numpy as np
import torch

from saber_engine_amd import iu8

BF16, E4M3 = 2.0 ** -8, 2.0 ** -4      # half a step of a rounding, relative
F32 = 2.0 ** -24


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


class Paged:
    """A cache on the device and, beside it, the positions it holds: pages in no order."""

    def __init__(self, seqs, kv_heads, dim, page, most, e4m3=False, seed=0, pages=None, fill=float("nan")):
        self.seqs, self.h, self.dim, self.page, self.e4m3 = seqs, kv_heads, dim, page, e4m3
        self.stride = -(-most // page)
        g = torch.Generator().manual_seed(seed)
        self.pages = pages or seqs * self.stride
        self.table = torch.randperm(self.pages, generator=g)[: seqs * self.stride].view(seqs, self.stride).int().cuda()
        self.kind = torch.float8_e4m3fn if e4m3 else torch.bfloat16
        self.e = 16 if e4m3 else 8
        shape = (self.pages, kv_heads, page // 16, dim // self.e, 16, self.e)
        # nothing is in it: what a kernel must not look at is NaN
        self.k = torch.full(shape, fill, dtype=torch.bfloat16, device="cuda").to(self.kind)
        self.v = torch.full((self.pages, kv_heads, page, dim), fill, dtype=torch.bfloat16, device="cuda").to(self.kind)
        self.scales = [torch.rand(kv_heads, generator=g).add_(0.5).div_(64).cuda() if e4m3 else None for _ in range(2)]
        self.kv_len = torch.zeros(seqs, dtype=torch.int32, device="cuda")

    def desc(self):
        ks, vs = (s.data_ptr() if s is not None else None for s in self.scales)
        return iu8.KvCache.of(self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(), self.kv_len.data_ptr(), kv_heads=self.h, head_dim=self.dim,
                              page_tokens=self.page, pages=self.pages, table_stride=self.stride, kind=iu8.KV_E4M3 if self.e4m3 else iu8.KV_BF16,
                              k_scale=ks, v_scale=vs)

    def raw(self, t):
        return t.view(torch.uint8 if self.e4m3 else torch.int16)

    def put(self, s, at, k, v):
        """Rows k, v [n, kv_heads, dim] (the cache's type) at positions at .. at + n - 1 of sequence s, element by element's place."""
        pos = torch.arange(at, at + len(k), device="cuda")
        p, o = self.table[s].long()[pos // self.page], pos % self.page
        kk = self.raw(k.contiguous()).view(len(k), self.h, self.dim // self.e, self.e)
        self.raw(self.k)[p, :, o // 16, :, o % 16] = kk
        self.raw(self.v)[p, :, o] = self.raw(v.contiguous())

    def rows(self, s, n):
        """(k, v) f64 [n, kv_heads, dim] of sequence s's first n positions, through the library's offsets' formula; a hole is None's
        mask False."""
        pos = np.arange(n)
        p = self.table[s].cpu().numpy().astype(np.int64)[pos // self.page] if n else np.zeros(0, np.int64)
        there = (p >= 0) & (p < self.pages)
        p = torch.from_numpy(np.where(there, p, 0)).cuda()
        o = torch.from_numpy(pos % self.page).cuda()
        k = self.raw(self.k)[p, :, o // 16, :, o % 16].reshape(n, self.h, self.dim).view(self.kind)
        v = self.raw(self.v)[p, :, o].view(self.kind)
        k, v = f64(k.float()), f64(v.float())
        if self.e4m3:
            k, v = k * f64(self.scales[0])[:, None], v * f64(self.scales[1])[:, None]
        return k, v, there


def random_rows(g, *shape, e4m3=False):
    x = torch.randn(*shape, generator=g)
    return (x * 60).clamp(-448, 448).to(torch.float8_e4m3fn).cuda() if e4m3 else x.to(torch.bfloat16).cuda()


def e4m3_of(x, scale):
    """What an e4m3 cache stores of x (f64, of bf16 or f32 values): the f32 quotient in the e4m3 grid (a step of 2^-9 below 2^-6, of 2^-3 of the
    binade above), to nearest even, saturated."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        y = np.clip((x.astype(np.float32) / np.float32(scale)).astype(np.float64), -448, 448)
        step = 2.0 ** (np.maximum(np.floor(np.log2(np.abs(y))), -6) - 3)
        return np.where(y == 0, 0.0, np.rint(y / step) * step)


def attention(q, k, v, there, scale):
    """q f64 [n, heads, dim], k, v f64 [len, kv_heads, dim]: the n rows are the last positions. Returns the output and how far a
    kernel may be off in each element: the weights rounded to bf16 (half a step of each), the output rounded once, the scores off by
    dim + 4 roundings of f32 of the sum of magnitudes (a relative error of the weight, twice that for numerator and sum), the sums by
    one rounding a key."""
    n, heads, dim = q.shape
    total, kvh = k.shape[0], k.shape[1]
    out, tol = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    for i in range(n):
        sees = there & (np.arange(total) <= total - n + i)
        if not sees.any():
            continue
        kk, vv = k[sees], v[sees]
        for h in range(heads):
            b = h // (heads // kvh)
            s = kk[:, b] @ q[i, h] * scale
            off = (np.abs(kk[:, b]) @ np.abs(q[i, h]) * abs(scale)).max() * (dim + 4) * F32
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv[:, b]
            spread = w @ np.abs(vv[:, b])
            tol[i, h] = BF16 * np.abs(out[i, h]) + spread * (BF16 + 2.5 * off + 2 * (len(w) + 8) * F32) * 1.01 + 1e-30
    return out, tol


def check(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0].tolist()}: {got[bad][0]} for {want[bad][0]} +- {tol[bad][0]}"


class Workspace:
    def __init__(self, seqs, max_q, max_kv, heads, kv_heads, dim):
        pb, cb = iu8.attn_workspace(seqs, max_q, max_kv, heads, kv_heads, dim)
        self.partial = torch.full((pb // 4,), float("nan"), device="cuda") if pb else None
        self.counter = torch.zeros(cb // 4, dtype=torch.int32, device="cuda") if cb else None

    def args(self):
        return tuple(t.data_ptr() if t is not None else None for t in (self.partial, self.counter))
