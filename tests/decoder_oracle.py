"""The decoder operators from their definitions, in 64 bits on the CPU, with the inputs and tolerances of their tests.

A rounding to a type is off by at most half a step, eps / 2 of the value; sums in f32 of n terms are off by at most
n * 2^-23 of the sum of their sizes (2^-24 for a rounded addition, twice that for one that truncates, as the adders of the
tensor cores may)."""
import math

import numpy as np
import torch

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def half_step(kind):
    return torch.finfo(TYPES[kind]).eps / 2


def rounding(kind, y):
    """How far the type's nearest number may be from y: half a step of y's power of two, and of the smallest normal number's
    where y is below it (f16: 2^-14 * 2^-11 = 2^-25; numbers below are as far apart as there)."""
    return half_step(kind) * y.abs().clamp(min=torch.finfo(TYPES[kind]).tiny)


# ---- MatMulNBits ---------------------------------------------------------------------------------
def linear_weights(gen, n, k, group, zero_points, bias):
    blocks = -(-k // group)
    w = {"weights": torch.randint(0, 256, (n, blocks, group // 2), generator=gen, dtype=torch.uint8).numpy(),
         "scales": ((torch.rand(n, blocks, generator=gen) + 0.5) * 0.05).half().float().numpy()}
    if zero_points:
        w["zero_points"] = torch.randint(0, 256, (n, (blocks + 1) // 2), generator=gen, dtype=torch.uint8).numpy()
    if bias:
        w["bias"] = torch.randn(n, generator=gen).numpy()
    return w


def linear_matrix(w, k, rounded=None):
    """The [n][k] matrix in 64 bits; `rounded` to a 16-bit type as many rows take it."""
    codes = w["weights"].astype(np.int64)
    n, blocks = codes.shape[:2]
    q = np.stack((codes & 15, codes >> 4), -1).reshape(n, blocks, -1).astype(np.float64)
    zero = np.full((n, blocks), 8.0)
    if "zero_points" in w:
        z = w["zero_points"].astype(np.int64)
        zero = np.stack((z & 15, z >> 4), -1).reshape(n, -1)[:, :blocks].astype(np.float64)
    m = torch.from_numpy(((q - zero[:, :, None]) * w["scales"].reshape(n, blocks).astype(np.float64)[:, :, None]).reshape(n, -1)[:, :k])
    return m.to(TYPES[rounded]).double() if rounded else m


def linear(x, w, k, rounded=None):
    y = x.double() @ linear_matrix(w, k, rounded).t()
    return y + torch.from_numpy(w["bias"]).double() if "bias" in w else y


def linear_bound(x, w, k, kind, rounded_weights):
    """The result's rounding, the f32 sums (over the inputs, with a product by the scale for each), and for the form that
    multiplies 16-bit matrices the rounding of each weight."""
    size = x.double().abs() @ linear_matrix(w, k).abs().t()
    zero_size = x.double().abs().sum(-1, keepdim=True) * 16 * float(np.abs(w["scales"]).max()) * 2.0**-24  # code - zero is exact, scales of it round once
    h = half_step(kind)
    bias = torch.from_numpy(w["bias"]).double().abs() * 2.0**-23 if "bias" in w else 0.0
    return rounding(kind, linear(x, w, k)) + ((k + 2) * 2.0**-23 + (h if rounded_weights else 0.0)) * (1 + h) * size + zero_size + bias + 1e-30


# ---- paged cache ---------------------------------------------------------------------------------
class Paged:
    """A batch of packed sequences over a paged cache.  `new` rows and `total` lengths of each; pages are handed out in a
    random order; whatever no sequence holds is NaN."""

    def __init__(self, new, total, heads, kv_heads, size, page, kind, seed, behind=0, packed=False, q_kind=None, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.total, self.heads, self.kv_heads, self.size, self.page, self.kind = list(new), list(total), heads, kv_heads, size, page, kind
        self.q_kind = q_kind or kind
        dt, qdt = TYPES[kind], TYPES[self.q_kind]
        tokens = sum(new) + behind
        used = [-(-t // page) for t in total]
        self.pages = sum(used) + 2
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(new), max(max(used), 1) + 1), -7, dtype=torch.int32)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = order[at : at + u]
            at += u
        self.cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
        self.len = torch.tensor(list(total), dtype=torch.int32)
        shape = (self.pages, page, kv_heads, size)
        self.kc, self.vc = torch.full(shape, math.nan, dtype=dt), torch.full(shape, math.nan, dtype=dt)
        for b, t in enumerate(total):
            for j in range(0, t, page):
                n = min(page, t - j)
                p = int(self.table[b, j // page])
                self.kc[p, :n] = (torch.randn(n, kv_heads, size, generator=g) * spread).to(dt)
                self.vc[p, :n] = torch.randn(n, kv_heads, size, generator=g).to(dt)
        self.q = (torch.randn(tokens, heads * size, generator=g) * spread).to(qdt)
        self.k = torch.randn(tokens, kv_heads * size, generator=g).to(qdt)
        self.v = torch.randn(tokens, kv_heads * size, generator=g).to(qdt)
        self.packed = torch.cat((self.q, self.k, self.v), 1) if packed else None

    def rows(self):
        """(row, sequence, position) of every new row that belongs to a sequence."""
        for b, (n, t) in enumerate(zip(self.new, self.total)):
            for i in range(n):
                yield int(self.cu[b]) + i, b, t - n + i

    def held(self, cache, b, upto):
        flat = cache.reshape(-1, self.kv_heads, self.size)
        slots = torch.tensor([int(self.table[b, j // self.page]) * self.page + j % self.page for j in range(upto)], dtype=torch.long)
        return flat[slots].double()


def attend(p, scale=None):
    """Output and its bound, in 64 bits: out = sum_j softmax(scale q k)_j v_j over the row's own and earlier positions.
    Bound: the result's rounding, the rounding of each probability to the 16-bit type, and in f32 the scores (size terms),
    the exponential, and the sums over the keys."""
    scale = 1.0 / math.sqrt(p.size) if scale is None else scale
    q = p.q.to(TYPES[p.kind]).double().reshape(-1, p.heads, p.size)
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    h, group = half_step(p.kind), p.heads // p.kv_heads
    for b, (n, t) in enumerate(zip(p.new, p.total)):
        if t == 0 or n == 0:
            continue
        k, v = p.held(p.kc, b, t), p.held(p.vc, b, t)
        rows = slice(int(p.cu[b]), int(p.cu[b]) + n)
        visible = torch.arange(t)[None, :] <= (t - n + torch.arange(n))[:, None]
        for head in range(p.heads):
            kk, vv = k[:, head // group], v[:, head // group]
            s = (q[rows, head] @ kk.t()) * scale
            size = (q[rows, head].abs() @ kk.abs().t()) * abs(scale)
            s = s.masked_fill(~visible, -math.inf)
            top = s.amax(-1, keepdim=True)
            e = torch.where(visible, torch.exp(s - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
            w = e.sum(-1, keepdim=True)
            prob = torch.where(w > 0, e / w, 0.0)
            out[rows, head] = prob @ vv
            off = (p.size + 4) * 2.0**-23 * torch.where(visible, size, 0.0).amax(-1, keepdim=True)
            mean = prob @ vv.abs()
            # an exponential below 2^-14 (f16's least normal number) of the largest loses up to 2^-25 of the largest instead
            low = 2.0**-24 / w.clamp(min=1.0) * torch.where(visible, 1.0, 0.0) @ vv.abs() if p.kind == "float16" else 0.0
            bound[rows, head] = rounding(p.kind, out[rows, head]) + (h * 2 + 2 * off + (t + 16) * 2.0**-22) * mean + low + 1e-30
    return out.flatten(1), bound.flatten(1)


def rotate(x, cos, sin, position, interleaved):
    """One row [heads][size] in 64 bits, with the bound of its f32 arithmetic."""
    half = cos.shape[1]
    y, off = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    c, s = cos[position].double(), sin[position].double()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    u, v = x[:, a].double(), x[:, b].double()
    y[:, a], y[:, b] = u * c - v * s, v * c + u * s
    off[:, a], off[:, b] = ((u * c).abs() + (v * s).abs()) * 2.0**-23, ((v * c).abs() + (u * s).abs()) * 2.0**-23
    return y, off


def append(p, cos, sin, interleaved):
    """(rotated, its bound), (key cache, its bound), value cache of a Paged batch; NaN stays where nothing was put."""
    h = half_step(p.kind)
    rotated, rb = torch.zeros(p.q.shape, dtype=torch.float64), torch.zeros(p.q.shape, dtype=torch.float64)
    kc, kb, vc = p.kc.double().clone(), torch.zeros(p.kc.shape, dtype=torch.float64), p.vc.clone()
    rounds = p.q_kind != p.kind
    for row, b, position in p.rows():
        if position < 0:
            continue
        at = (int(p.table[b, position // p.page]), position % p.page)
        for src, heads, put in ((p.q, p.heads, "q"), (p.k, p.kv_heads, "k")):
            x = src[row].reshape(heads, p.size)
            y, off = rotate(x, cos, sin, position, interleaved) if cos is not None else (x.double(), torch.zeros(x.shape, dtype=torch.float64))
            turned = torch.zeros(p.size, dtype=torch.bool)
            if cos is not None:
                turned[: 2 * cos.shape[1]] = True
            off = off * (1 + h) + rounding(p.kind, y) * (1.0 if rounds else turned.double())
            if put == "q":
                rotated[row], rb[row] = y.flatten(), off.flatten()
            else:
                kc[at], kb[at] = y, off
        vc[at] = p.v[row].reshape(p.kv_heads, p.size).to(TYPES[p.kind])
    return (rotated, rb), (kc, kb), vc


def angles(positions, half):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    return a.cos().float(), a.sin().float()
