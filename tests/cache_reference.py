"""Plain 64-bit implementations of the cache operators, for the tests (any device)."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def e4m3_round(y):
    """Nearest e4m3 value (3 mantissa bits, steps of 2^-9 at least, 448 at most), ties to even; y in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def quantise(x, int8):
    """fp32 rows -> (codes' values in 64 bits, fp32 scale), by the quantiser's fp32 steps."""
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], torch.zeros_like(x), x)
    most = torch.tensor(127.0 if int8 else 448.0, device=x.device)
    scale = torch.maximum(x.abs().amax(-1) / most, torch.tensor(1e-12, device=x.device))
    y = (x / scale[..., None]).double()
    codes = y.round().clamp(-128, 127) if int8 else e4m3_round(y)
    return codes, torch.where(bad, torch.full_like(scale, math.nan), scale)


def rotate(x, pos, freq, magnitude, interleaved, backward=False):
    """x (..., n, d) in 64 bits with positions broadcast over (..., n); freq (rot / 2) in 64 bits."""
    rot = 2 * freq.numel()
    angle = pos.double()[..., None] * freq
    c, s = angle.cos() * magnitude, angle.sin() * magnitude
    if backward:
        s = -s
    y = x.double().clone()
    first = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    second = first + 1 if interleaved else first + rot // 2
    a, b = y[..., first], y[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def values(codes, scale, table, n, d):
    """First n rows of a sequence: codes (pages, H, page, W), scale (pages, H, page), table (width,) -> (H, n, d) in 64
    bits, and whether each row's page exists (n,)."""
    pages, _, page, _ = codes.shape
    ids = table[:-(-n // page)].long() if n else table[:0].long()
    there = (ids >= 0) & (ids < pages)
    at = torch.where(there, ids, torch.zeros_like(ids))
    c = codes.view(torch.uint8)[at].view(codes.dtype).double()
    x = (c * scale[at].double()[..., None]).transpose(0, 1).flatten(1, 2)[:, :n, :d]
    return x, there.repeat_interleave(page)[:n]


def attend(q, k, v, seen, scale):
    """q (t, d), k and v (n, d), seen (t, n): output (t, d) and log-sum-exp (t,) in 64 bits; what is not seen has no part
    in anything, whatever it holds."""
    out = torch.zeros((q.shape[0], v.shape[1]), dtype=torch.float64, device=q.device)
    lse = torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    for i in range(q.shape[0]):
        at = seen[i].nonzero().flatten()
        if at.numel():
            s = (k[at] @ q[i].double()) * scale
            lse[i] = torch.logsumexp(s, 0)
            out[i] = torch.softmax(s, 0) @ v[at]
    return out, lse


def attend_cached(q, cache, table, lens, cu, tree=None, scale=None, shift=None):
    """The whole operator: q (tokens, Hq, d); cache with k_codes .. v_scale; lens and cu lists."""
    tokens, hq, d = q.shape
    hkv = cache.num_kv_heads
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros((tokens, hq, d), dtype=torch.float64, device=q.device)
    lse = torch.full((tokens, hq), -math.inf, dtype=torch.float64, device=q.device)
    for i, n in enumerate(lens):
        t = cu[i + 1] - cu[i]
        if t == 0:
            continue
        k, there = values(cache.k_codes, cache.k_scale, table[i], n, d)
        v, _ = values(cache.v_codes, cache.v_scale, table[i], n, d)
        key, row = torch.arange(n, device=q.device), torch.arange(t, device=q.device)
        ctx = n - t
        if tree is None:
            seen = key[None] <= (ctx + row)[:, None]
        else:
            j = key - ctx
            seen = (j < 0)[None] | (tree[cu[i]:cu[i + 1]][:, j.clamp(0, t - 1)] != 0)
        seen = seen & there[None]
        for h in range(hq):
            o, e = attend(q[cu[i]:cu[i + 1], h], k[h // (hq // hkv)], v[h // (hq // hkv)], seen, scale)
            out[cu[i]:cu[i + 1], h], lse[cu[i]:cu[i + 1], h] = o, e
    if shift is not None:
        lse = lse + scale * torch.einsum("thd,hd->th", q.double(), shift.double().repeat_interleave(hq // hkv, 0))
    return out, lse
