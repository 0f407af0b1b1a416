"""A paged key-value cache on the CPU and the serving operators' formulas in 64 bits."""
import collections
import math

import torch


def make_cache(lengths, hkv, dh, page, dtype, gen, width=None, spare=2, junk=float("nan")):
    """(k_pages, v_pages, table, lengths): random pages in random order; slots that no sequence uses
    hold `junk`, table entries past a sequence's last page are -1."""
    need = [-(-n // page) for n in lengths]
    width = max(1, max(need)) if width is None else width
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen)
    k = torch.full((total, hkv, page, dh), junk)
    v = torch.full((total, hkv, page, dh), junk)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    used = 0
    for b, n in enumerate(lengths):
        for i in range(need[b]):
            pg, rows = int(order[used]), min(page, n - i * page)
            table[b, i] = pg
            k[pg, :, :rows] = torch.randn(hkv, rows, dh, generator=gen)
            v[pg, :, :rows] = torch.randn(hkv, rows, dh, generator=gen)
            used += 1
    return k.to(dtype), v.to(dtype), table, torch.tensor(lengths, dtype=torch.int32)


def rows(pages, table, b, n):
    """The first n rows of sequence b, [heads, n, dh]."""
    page = pages.shape[2]
    t = torch.arange(n)
    return pages[table[b].long()[t // page], :, t % page].transpose(0, 1)


def attention(q, k_pages, v_pages, table, lengths, scale):
    """(out [B, Hq, 1, Dh], weights per sequence [Hq, n], bound on sum |p v| [B, Hq, 1, Dh], largest
    sum |q k| scale) in float64."""
    B, hq, _, dh = q.shape
    hkv = k_pages.shape[1]
    out = torch.zeros(B, hq, 1, dh, dtype=torch.float64)
    mag = torch.zeros_like(out)
    ps, smax = [], 0.0
    for b in range(B):
        n = int(lengths[b])
        k = rows(k_pages, table, b, n).double().repeat_interleave(hq // hkv, 0)
        v = rows(v_pages, table, b, n).double().repeat_interleave(hq // hkv, 0)
        p = torch.softmax(torch.einsum("hd,hnd->hn", q[b, :, 0].double(), k) * scale, -1)
        if n:
            out[b, :, 0] = torch.einsum("hn,hnd->hd", p, v)
            mag[b, :, 0] = torch.einsum("hn,hnd->hd", p, v.abs())
            smax = max(smax, float(torch.einsum("hd,hnd->hn", q[b, :, 0].double().abs(), k.abs()).max()) * abs(scale))
        ps.append(p)
    return out, ps, mag, smax


def weight_error(n, dh, smax, dtype):
    """Bound on the relative error of a softmax weight and of a weighted sum of n terms computed in
    fp32: a score's sum of dh products is off by at most dh * 2^-24 * sum |q k| (twice that for an
    accumulator that truncates), and that moves a weight by as much, once itself and once in the
    normaliser; sums of n terms by n * 2^-24 (twice, as above); 2^x and the scaling by log2 e by a few
    2^-23 and smax * 2^-23. In bf16 the weights enter the second product as two bf16 parts, which
    leaves 2^-16."""
    u = 2.0 ** -23
    e = 2 * dh * u * smax + 2 * n * u + 4 * u * smax + 16 * u
    return e + (2.0 ** -16 if dtype == torch.bfloat16 else 0.0)


def evict(mass, n, budget, recent, sink):
    """Surviving slots of one (sequence, head), ascending."""
    if n <= budget:
        return list(range(n))
    m = [(-math.inf if math.isnan(x) else x) for x in mass[:n].tolist()]
    # NaN ranks below -inf too
    isn = [math.isnan(x) for x in mass[:n].tolist()]
    middle = sorted(range(sink, n - recent), key=lambda t: (isn[t], -m[t], t))[:budget - sink - recent]
    return sorted(list(range(sink)) + middle + list(range(n - recent, n)))


def rotate(x, cos, sin):
    """x cos + rotate_half(x) sin in float64; cos, sin [B or 1, N, Dh]."""
    h = x.shape[-1] // 2
    x = x.double()
    r = torch.cat([-x[..., h:], x[..., :h]], -1)
    return x * cos.double()[:, None] + r * sin.double()[:, None]


def logits(x, history, starts, rep, pres, freq, bias, allowed):
    """process_logits' formula in float64; rep, pres, freq [B]; allowed bool [B, V] or None."""
    z = x.double().clone()
    B, V = z.shape
    for b in range(B):
        ids = [] if history is None else [int(i) for i in history[b]]
        start = 0 if starts is None else int(starts[b])
        seen = sorted({i for i in ids if 0 <= i < V})
        for t in seen:
            z[b, t] = z[b, t] / float(rep[b]) if z[b, t] > 0 else z[b, t] * float(rep[b])
        for t, c in collections.Counter(i for i in ids[max(start, 0):] if 0 <= i < V).items():
            z[b, t] -= float(freq[b]) * c + float(pres[b])
    if bias is not None:
        z += bias.double()
    if allowed is not None:
        z = z.masked_fill(~allowed, -math.inf)
    return z
