"""The paged-cache operators from their definitions, in float64, with the
error bounds that the tests hold the kernels to.

Bounds (u: half a unit in the last place of the 16-bit type, relative):
a kernel keeps scores, maxima and sums in FP32 and rounds the softmax weights
and the result to 16 bits. With D products per score and n keys per row,

  score         |ds| <= e_s = (D + 8) 2^-24 scale sum|q||k|, at most the row's largest
  weight        relative e_s + 2^-21 (exponential) + |s| 2^-22 (its argument)
  sums over n   relative 2 n 2^-24 (tensor-core accumulation truncates)
  result        |do| <= A (2 e + u) + u |o|, A = sum_j w_j |v_j| over the weights w_j,
                e the sum of the relative errors above

and for float16 weights below its smallest normal number 2^-25 of the row's
largest weight for each key, since a running maximum may scale them down by
less than it could: 2^-25 sum|v| / sum(p).
"""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def attention(q, k_pages, v_pages, table, kv_lens, q_starts, *, scale=None, window=0, sinks=0, out_dtype=None):
    """(out, lse, bound of out, bound of lse, covered tokens) in float64."""
    tokens, heads, dim = q.shape
    pages, kv_heads, page, _ = k_pages.shape
    scale = 1 / math.sqrt(dim) if scale is None else scale
    dev, f8 = q.device, torch.float64
    out = torch.zeros(tokens, heads, dim, dtype=f8, device=dev)
    lse = torch.full((tokens, heads), -math.inf, dtype=f8, device=dev)
    out_tol = torch.zeros_like(out)
    lse_tol = torch.zeros(tokens, heads, dtype=f8, device=dev)
    covered = torch.zeros(tokens, dtype=torch.bool, device=dev)
    starts = q_starts.tolist()
    for b, kv in enumerate(kv_lens.tolist()):
        first, last = starts[b], starts[b + 1]
        n = last - first
        covered[first:last] = True
        if n <= 0 or kv <= 0:
            continue
        j = torch.arange(kv, device=dev)
        where = table[b].long()[j // page]
        there = (where >= 0) & (where < pages)
        pos = kv - n + torch.arange(n, device=dev)[:, None]
        seen = there & (j <= pos)
        if window:
            seen &= (j > pos - window) | (j < sinks)
        at = where.clamp(0, pages - 1)
        for h in range(heads):
            kh = k_pages[at, h // (heads // kv_heads), j % page].to(f8)
            vh = v_pages[at, h // (heads // kv_heads), j % page].to(f8)
            qh = q[first:last, h].to(f8)
            used = seen.any(0)  # rows that no token sees may hold anything
            kh = torch.where(used[:, None], kh, 0)
            vh = torch.where(used[:, None], vh, 0)
            s = torch.where(seen, scale * (qh @ torch.nan_to_num(kh, 0, 0, 0).T), -math.inf)
            # a non-finite key or value counts where it is seen, and nowhere else
            odd_k, odd_v = ~torch.isfinite(kh).all(1), ~torch.isfinite(vh).all(1)
            for jj in torch.nonzero(odd_k)[:, 0].tolist():
                s[seen[:, jj], jj] = scale * (qh[seen[:, jj]] @ kh[jj])
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, 0, m))
            total = p.sum(1, keepdim=True)
            w = torch.where(total == 0, 0, p / total)
            finite_v = torch.where(odd_v[:, None], 0, vh)
            o = w @ finite_v
            for jj in torch.nonzero(odd_v)[:, 0].tolist():
                rows = seen[:, jj]
                o[rows] = o[rows] + w[rows, jj:jj + 1] * vh[jj]
            out[first:last, h] = o
            lse[first:last, h] = (m + torch.log(total))[:, 0]
            absum = scale * (qh.abs() @ torch.nan_to_num(kh, 0, 0, 0).abs().T)
            big = torch.where(seen, absum, 0).amax(1, keepdim=True)
            e = (dim + 8) * 2.0 ** -24 * big + big * 2.0 ** -22 + 2.0 ** -21 + 2 * seen.sum(1, keepdim=True) * 2.0 ** -24
            a = w @ finite_v.abs()
            u_w = UNIT[q.dtype]
            tol = a * (2 * e + u_w) + UNIT[out_dtype or q.dtype] * o.abs() + 2.0 ** -126
            if q.dtype == torch.float16:
                ones = seen.to(f8)
                tol = tol + 2.0 ** -25 * (ones @ finite_v.abs()) / total.clamp(min=1)
                if (out_dtype or q.dtype) == torch.float16:
                    tol = tol + 2.0 ** -25
            out_tol[first:last, h] = tol
            lse_tol[first:last, h] = (e + 2.0 ** -21 * (1 + lse[first:last, h, None].abs().nan_to_num(0, 0, 0)))[:, 0]
    return out, lse, out_tol, lse_tol, covered


def append(q, k, v, cos, sin, positions, slots, k_pages, v_pages, *, q_norm=None, k_norm=None, eps=1e-6, interleaved=False):
    """(q, k_pages, v_pages) in float64 with a bound for each: FP32 arithmetic on a pair (a, b) is off
    by at most 2^-19 (|a| + |b|) (a mean of up to 128 squares, a root, a quotient, two products), then one rounding."""
    f8 = torch.float64
    dtype, page = k_pages.dtype, k_pages.shape[2]
    u = UNIT[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126

    def turned(x, gain):
        x = x.to(f8)
        if gain is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.to(f8)
        size = x.abs()
        if cos is None:
            return x, size
        half = cos.shape[1]
        lo = torch.arange(half, device=x.device) * (2 if interleaved else 1)
        hi = lo + (1 if interleaved else half)
        c, s = (t.to(f8)[positions.long()][:, None] for t in (cos, sin))
        a, b = x[..., lo], x[..., hi]
        y, mag = x.clone(), size.clone()
        y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
        mag[..., lo] = mag[..., hi] = a.abs() + b.abs()
        return y, mag

    def bound(y, mag):
        d = 2.0 ** -19 * mag
        return u * (y.abs() + d) + d + tiny

    qy, qm = turned(q, q_norm)
    pools = []
    ky, km = turned(k, k_norm)
    vy = v.to(f8)
    for pool, y, mag in ((k_pages, ky, km), (v_pages, vy, torch.zeros_like(vy))):
        want, tol = pool.to(f8), torch.zeros(pool.shape, dtype=f8, device=pool.device)
        t = torch.nonzero(slots >= 0)[:, 0]
        at = (slots[t].long() // page, slice(None), slots[t].long() % page)
        want[at], tol[at] = y[t], bound(y, mag)[t]
        pools += [want, tol]
    return (qy, bound(qy, qm)), tuple(pools[:2]), tuple(pools[2:])
