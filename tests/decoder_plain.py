"""Plain forms of the decoder-step operators in 64 bits, the inputs their tests share, and their tolerances.

Tolerances count roundings (u = 2^-24, half a step of fp32; h = half a step of the stored type, 2^-8 for
bf16). A score is a sum of d products scaled and moved to base 2: off by at most (d + 8) u times the sum of
the products' magnitudes, S; its weight is off by that much relatively, and so are the weights' sum and its
logarithm. An output is a sum of n weighted values over the sum of n weights: with A = sum of weight times
|value| it is off by at most (2 (d + 8) u S + 2 (n + 8) u) A, by h A more where the weights are rounded to
bf16 for the product (the tensor-core kernels), and by h |out| for its own rounding. The same bound is
allowed for all kernels of a type. (fp32 on the tensor cores: a factor is a high part of 11 bits, rounded, and an exact rest of at
most 12, of which 11 are used, 2 u of the factor off at most; the product of two rests, at most 4 u, is left out: a product is
off by 8 u. Sums are cut off rather than rounded, 2 u each, in groups of at most 32 products, 4 of them large, that are added
up in fp32: all that stays below d + 8 and n + 8 roundings.)
"""
import math

import torch

U = 2.0 ** -24


class Case:
    """Sequences over a paged cache: `lens` cached positions, of which the last `rows` are the call's rows."""

    def __init__(self, lens, rows, heads=4, kv_heads=2, dim=64, dtype=torch.float32, page=16, layout="heads", seed=0,
                 fill=None, spare_pages=3, device="cuda"):
        self.lens, self.rows, self.heads, self.kv_heads, self.dim, self.page = list(lens), list(rows), heads, kv_heads, dim, page
        self.dtype, self.device = dtype, device
        g = torch.Generator(device=device).manual_seed(seed)
        per = [max(0, (n + page - 1) // page) for n in self.lens]
        pages = sum(per) + spare_pages
        order = torch.randperm(pages, device=device, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(per + [1])), -1, dtype=torch.int32, device=device)
        at = 0
        for s, n in enumerate(per):
            self.table[s, :n] = order[at: at + n]
            at += n
        shape = (2, pages, kv_heads, page, dim) if layout == "heads" else (2, pages, page, kv_heads, dim)
        pool = torch.randn(shape, device=device, generator=g).to(dtype)
        if layout == "heads":
            pool = pool.transpose(2, 3)
        self.k, self.v = pool[0], pool[1]
        if fill is not None:  # what nobody may look at: the slots past the lengths and the spare pages
            seen = torch.zeros(pages, page, dtype=torch.bool, device=device)
            for s, n in enumerate(self.lens):
                j = torch.arange(max(n, 0), device=device)
                seen[self.table[s, j // page].long(), j % page] = True
            self.k[~seen] = fill
            self.v[~seen] = fill
        starts = [0]
        for r in self.rows:
            starts.append(starts[-1] + r)
        self.total = starts[-1]
        self.row_start = torch.tensor(starts, dtype=torch.int32, device=device)
        self.length = torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.max_rows = max(self.rows)
        self.q = torch.randn(self.total, heads, dim, device=device, generator=g).to(dtype)
        self.gen = g

    def cache(self):
        import speech_sampler as ss
        return ss.KvCache(self.k, self.v, self.table)

    def gathered(self, s):
        """Keys and values of sequence s in 64 bits, [positions, kv_heads, dim]."""
        j = torch.arange(max(self.lens[s], 0), device=self.device)
        page = self.table[s, j // self.page].long()
        ok = page >= 0
        k, v = self.k[page.clamp(min=0), j % self.page].double(), self.v[page.clamp(min=0), j % self.page].double()
        k[~ok] = 0.0
        v[~ok] = 0.0
        return k, v


def attend(case, scale, window=0, sinks=0):
    """out, lse and the tolerance of each, by the definition, row by sequence: [rows, heads, dim] and [rows, heads]."""
    d, group, dev = case.dim, case.heads // case.kv_heads, case.device
    half = torch.finfo(case.dtype).eps / 2
    out = torch.zeros(case.total, case.heads, d, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    lse = torch.full((case.total, case.heads), -math.inf, dtype=torch.float64, device=dev)
    lse_tol = torch.zeros_like(lse)
    row = 0
    for s, (n, r) in enumerate(zip(case.lens, case.rows)):
        k, v = case.gathered(s)
        for i in range(r):
            p = n - r + i
            if p >= 0:
                j = torch.arange(p + 1, device=dev)
                if window:
                    j = j[(j > p - window) | (j < sinks)]
                q = case.q[row].double().view(case.kv_heads, group, d)
                kk, vv = k[j], v[j]
                x = scale * torch.einsum("hgd,jhd->hgj", q, kk)
                size = abs(scale) * torch.einsum("hgd,jhd->hgj", q.abs(), kk.abs()).amax(-1)  # S
                w = torch.softmax(x, -1)
                out[row] = torch.einsum("hgj,jhd->hgd", w, vv).reshape(case.heads, d)
                mass = torch.einsum("hgj,jhd->hgd", w, vv.abs()).reshape(case.heads, d)  # A
                lse[row] = torch.logsumexp(x, -1).reshape(-1)
                size = size.reshape(-1)
                weights = half if case.dtype == torch.bfloat16 else 0.0
                tol[row] = (2 * (d + 8) * U * size[:, None] + 2 * (len(j) + 8) * U + weights) * mass + half * out[row].abs()
                lse_tol[row] = (d + 8) * U * size + (len(j) + 8) * U + 4 * U * lse[row].abs()
            row += 1
    return out, lse, tol, lse_tol


def check_attend(case, out, lse, scale, window=0, sinks=0):
    want, want_lse, tol, lse_tol = attend(case, scale, window, sinks)
    off = (out[: case.total].double() - want).abs()
    assert torch.all(off <= tol), (float(off.max()), float((off - tol).max()))
    if lse is not None:
        got = lse[: case.total].double()
        idle = torch.isinf(want_lse)
        assert torch.equal(got[idle], want_lse[idle])
        off = (got - want_lse).abs()[~idle]
        assert torch.all(off <= lse_tol[~idle]), float(off.max())


def norm_rope(x, weight, eps, positions, inv_freq, interleaved):
    """A head row x [rows, heads, dim] normed and rotated in 64 bits, and the bound on fp32's error.

    The norm is a sum of d squares, a root, a division and two products: (d + 8) u relatively. The angle is
    reduced in 64 bits and rounded to fp32 once (at most pi in size: 4 u absolute), its cosine and sine are each
    off by 4 u more; a rotated value is two products and a sum. With M = |a| + |b| of the normed pair (their own
    size where not rotated) all that stays below (d + 24) u M."""
    x = x.double()
    dim = x.shape[-1]
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    r = 2 * len(inv_freq)
    t = positions.double()[:, None, None] * inv_freq
    y, size = x.clone(), x.abs()
    ia = torch.arange(0, r, 2, device=x.device) if interleaved else torch.arange(0, r // 2, device=x.device)
    ib = ia + 1 if interleaved else ia + r // 2
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, (dim + 24) * U * size
