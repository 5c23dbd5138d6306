"""Plain 64-bit CPU implementations of the serving ops, for their tests."""
import math

import torch


def quantise(rows):
    """Rows [...,D] bf16 -> (e4m3 payload as float64 values, scale as float64, scale byte)."""
    x = rows.double()
    finite = torch.where(torch.isfinite(x), x.abs(), 0.0)
    top = finite.amax(-1)
    e = torch.zeros_like(top)
    for i in range(top.numel()):
        t = float(top.view(-1)[i])
        if t > 0:
            k = -124
            while t > 448.0 * 2.0 ** k:
                k += 1
            e.view(-1)[i] = k
    scale = torch.exp2(e)
    y = x / scale[..., None]
    most = torch.where(e == 120, 240.0, 448.0)[..., None]  # 256 * 2^120 is no bf16 number
    y = torch.where(torch.isfinite(y), torch.minimum(torch.maximum(y, -most), most), y)
    payload = torch.where(torch.isfinite(y), y, math.nan).float().to(torch.float8_e4m3fn).double()
    return payload, scale, (e + 127).to(torch.uint8)


def held_rows(cache, scale, pages, n):
    """The first n rows [Hkv,n,D] of a sequence in float64 (CPU tensors)."""
    page = cache.shape[2]
    out = torch.empty(cache.shape[1], n, cache.shape[3], dtype=torch.float64)
    for j in range(n):
        pg = int(pages[j // page])
        row = cache[pg, :, j % page].double()
        if scale is not None:
            row = row * scale.view(torch.uint8)[pg, :, j % page].view(torch.float8_e8m0fnu).double()[:, None]
        out[:, j] = row
    return out


def attention(q, k, v, window=None, softcap=None, scale=None):
    """q [Hq,S,D] (the last S positions), k, v [Hkv,n,D], float64.  Returns (out, bound): bound is what a 32-bit
    kernel's result may differ by before it is rounded to bf16 (see decode_bound)."""
    hq, s, d = q.shape
    g, n = hq // k.shape[0], k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(hq):
        for i in range(s):
            t = n - s + i
            lo = max(0, t - window + 1) if window else 0
            if t < lo:
                continue
            kk, vv = k[h // g, lo:t + 1], v[h // g, lo:t + 1]
            z = kk @ q[h, i] * scale
            size = float((kk.abs() @ q[h, i].abs()).max()) * scale
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            p = torch.softmax(z, 0)
            out[h, i] = p @ vv
            bound[h, i] = decode_bound(d, t + 1 - lo, size, float(z.abs().max()), softcap) * (p @ vv.abs())
    return out, bound


def decode_bound(d, n, size, top, softcap):
    """Relative error of a softmax weight, times two for numerator and denominator.

    A score is a 32-bit sum of d exact products: at most (d + 3) roundings of 2^-24 of the sum of the products' sizes
    (`size`, scaled); the cap adds a division, a tanh good to 2^-21 of the cap (above 128 also to that of a score
    below a sixteenth of the cap; 1 - 2 / (e^2y + 1) alone subtracts numbers near 1, so its error is the cap's), and products.  exp adds 2^-22 for its
    own error, and its argument, a difference of scores times log2(e), three roundings of at most 2 * top.  A weight is split into two bf16 numbers
    for the product with V, which keeps 2^-16 of it, and sums of n terms in 32 bits add at most (n + 16) 2^-24."""
    u = 2.0 ** -24
    reach = min(softcap, 16 * top) if softcap and softcap > 128 else softcap
    score = (d + 3) * u * size + (reach * 2.0 ** -21 + 6 * u * top if softcap else 0.0)
    return 2 * (score + 2.0 ** -22 + 8 * u * top) + 2.0 ** -16 + 2 * (n + 16) * u


def logprobs(x, ids, top):
    """x [N,V] float64 on the CPU."""
    n, v = x.shape
    logp, h = torch.full((n,), math.nan, dtype=torch.float64), torch.full((n,), math.nan, dtype=torch.float64)
    tl = torch.full((n, top), math.nan, dtype=torch.float64)
    ti = torch.full((n, top), -1, dtype=torch.int64)
    for i in range(n):
        r = x[i]
        if torch.isnan(r).any() or (r == math.inf).any() or not torch.isfinite(r).any():
            continue
        lp = torch.log_softmax(r, 0)
        p = lp.exp()
        h[i] = -torch.where(p > 0, p * lp, 0.0).sum()
        if 0 <= int(ids[i]) < v:
            logp[i] = lp[int(ids[i])]
        order = sorted(range(v), key=lambda j: (-float(r[j]), j))[:top]
        ti[i] = torch.tensor(order, dtype=torch.int64)
        tl[i] = lp[ti[i]]
    return logp, h, tl, ti
