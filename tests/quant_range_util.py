"""Attention over a paged cache in 4 or 8 bits in 64 bits, with a bound on the error of each output dim and
of each mass from the terms that belong to it alone."""
import torch

import quant_util as Q

U = 2.0 ** -23  # an fp32 operation that may truncate


def rows(cache, which, b, n, bits, dh):
    """As Q.rows, where a page that is not in the pool leaves its slots out: (values [heads, n, dh], live [n])."""
    pages, page = cache[0].shape[0], cache[0].shape[2]
    table = cache[3][b]
    live = ((table >= 0) & (table < pages))[torch.arange(n) // page]
    put = (*cache[:3], torch.where((cache[3] >= 0) & (cache[3] < pages), cache[3], 0), cache[4])
    return Q.rows(put, which, b, n, bits, dh), live


def attention(q, cache, bits, scale):
    """(out, tolerance of out before its rounding [B, Hq, 1, Dh], weights and their tolerance per sequence
    [Hkv, n], summed over a kv head's queries) in float64.

    A score is a sum of dh products (exact: q has 8 bits or, fp32, two parts of 22 together, a code 7), in
    fp32 and in any order: off by dh U of the sum of their sizes, groups and scaling by a few U more. A weight
    is 2^x of the difference to the running maximum: off by U of both, and by 2^-22. Sums of n weights or
    products, rescaled as the maximum rises: 2 n U. A weight times its scale enters the second product with
    16 bits at least (bf16) or 22 (fp32). Weights and outputs below 2^-126 may be 0."""
    B, hq, _, dh = q.shape
    hkv = cache[0].shape[1]
    g = hq // hkv
    out = torch.zeros(B, hq, 1, dh, dtype=torch.float64)
    tol, weights, wtol = torch.zeros_like(out), [], []
    part = 2.0 ** -16 if q.dtype == torch.bfloat16 else 2.0 ** -22
    for b in range(B):
        n = int(cache[4][b])
        k, live = rows(cache, 0, b, n, bits, dh)
        v, _ = rows(cache, 1, b, n, bits, dh)
        k, v = k[:, live].repeat_interleave(g, 0), v[:, live].repeat_interleave(g, 0)
        x = q[b, :, 0].double()
        w, t = torch.zeros(hq, n, dtype=torch.float64), torch.zeros(hq, n, dtype=torch.float64)
        if bool(live.any()):
            s = torch.einsum("hd,hnd->hn", x, k) * scale
            size = torch.einsum("hd,hnd->hn", x.abs(), k.abs()) * abs(scale)
            p = torch.softmax(s, -1)
            each = (dh + 12) * U * size + 2 * U * (s.abs() + s.abs().amax(-1, keepdim=True)) + 8 * U
            norm = (p * each).sum(-1, keepdim=True) + (2 * n + 8) * U
            out[b, :, 0] = torch.einsum("hn,hnd->hd", p, v)
            tol[b, :, 0] = 1.1 * (torch.einsum("hn,hnd->hd", p * (each + part + (2 * n + 8) * U), v.abs()) + norm * out[b, :, 0].abs())
            tol[b, :, 0] += 2.0 ** -126 * (1 + v.abs().sum(1))
            w[:, live], t[:, live] = p, 1.1 * p * (each + norm) + 2.0 ** -126
        weights.append(w.view(hkv, g, n).sum(1))
        wtol.append(t.view(hkv, g, n).sum(1))
    return out, tol, weights, wtol


def check_out(out, ref, tol, floor=0.0):
    """The result's dtype rounds it by half a step; floor: what lies below the smallest numbers."""
    d = (out.cpu().double() - ref).abs()
    bound = tol + torch.finfo(out.dtype).eps / 2 * (ref.abs() + tol) + floor
    assert bool((d <= bound).all()), f"{float((d / bound.clamp(min=1e-300)).nan_to_num(1e300).max())} times the bound"


def check_mass(mass, before, weights, wtol, g):
    """The sum of g weights and the mass that was there: rounded g times."""
    want, tol = before.double().clone(), torch.zeros(before.shape, dtype=torch.float64)
    for b, (w, t) in enumerate(zip(weights, wtol)):
        want[b, :, :w.shape[-1]] += w
        tol[b, :, :w.shape[-1]] += t + (g + 1) * 2.0 ** -24 * want[b, :, :w.shape[-1]].abs()
    d = (mass.cpu().double() - want).abs()
    assert bool((d <= tol).all()), f"{float((d / tol.clamp(min=1e-300)).max())} times the bound"
