"""A paged cache in 4 or 8 bits on the CPU: quantising, reading and attending by the formulas in 64 bits."""
import torch

GROUP = 32


def groups(dh):
    return -(-dh // GROUP)


def top(bits):
    return 7 if bits == 4 else 127


def close(x, bits):
    """(codes uint8 [.., dh * bits / 8], scales bf16 [.., groups]) of rows x [.., dh], fp32 values."""
    assert x.dtype == torch.float32
    dh, codes, scales = x.shape[-1], [], []
    for at in range(0, dh, GROUP):
        part = x[..., at:at + GROUP].double()
        largest = part.abs().amax(-1, keepdim=True)  # NaN propagates
        scale = (largest / top(bits)).float().bfloat16()
        finite = torch.isfinite(largest)
        there = finite & (scale.double() >= 2.0 ** -100)
        scale = torch.where(finite, torch.where(there, scale, torch.zeros_like(scale)), torch.full_like(scale, float("nan")))
        # torch.round takes halves to the even number
        codes.append(torch.where(there, torch.round(part / torch.where(there, scale, torch.ones_like(scale)).double()), 0.0))
        scales.append(scale)
    u = (torch.cat(codes, -1) + (top(bits) + 1)).to(torch.uint8)
    return (u[..., 0::2] + 16 * u[..., 1::2] if bits == 4 else u), torch.cat(scales, -1)


def open_(codes, scales, bits, dh):
    """The values, float64 [.., dh]."""
    u = torch.stack([codes % 16, codes // 16], -1).flatten(-2) if bits == 4 else codes
    return (u.double() - (top(bits) + 1)) * scales.double().repeat_interleave(GROUP, -1)[..., :dh]


def make_cache(lengths, hkv, dh, page, bits, gen, width=None, spare=2, spread=0.7):
    """(k_pages, v_pages, scales, table, lengths): random pages in random order. Slots that no sequence
    uses hold any bytes and scales of NaN and infinity; table entries past the last page are -1."""
    need = [-(-n // page) for n in lengths]
    width = max(1, max(need, default=0)) if width is None else width
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen)
    row = dh * bits // 8
    k, v = (torch.randint(0, 256, (total, hkv, page, row), generator=gen, dtype=torch.uint8) for _ in range(2))
    scales = torch.full((total, hkv, page, 2, groups(dh)), float("nan")).bfloat16()
    scales[..., 0] = float("inf")
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    used = 0
    for b, n in enumerate(lengths):
        for i in range(need[b]):
            pg, rows = int(order[used]), min(page, n - i * page)
            table[b, i] = pg
            for w, pool in enumerate((k, v)):
                x = torch.randn(hkv, rows, dh, generator=gen) * torch.exp(spread * torch.randn(1, 1, dh, generator=gen))
                pool[pg, :, :rows], scales[pg, :, :rows, w] = close(x, bits)
            used += 1
    return k, v, scales, table, torch.tensor(lengths, dtype=torch.int32)


def rows(cache, which, b, n, bits, dh):
    """The first n keys (0) or values (1) of sequence b, float64 [heads, n, dh]."""
    pool, scales, table = cache[which], cache[2], cache[3]
    t = torch.arange(n)
    pg, at = table[b].long()[t // pool.shape[2]], t % pool.shape[2]
    return open_(pool[pg, :, at], scales[pg, :, at, which], bits, dh).transpose(0, 1)


def attention(q, cache, bits, scale):
    """(out [B, Hq, 1, Dh], weights per sequence [Hq, n], sum |p v|, largest bound on a score's terms) in
    float64. The terms: a product with a code is computed with the offset 8 or 128 added to it and taken
    off the sum, so that its terms reach |q| * 2 * offset * scale."""
    B, hq, _, dh = q.shape
    hkv, zero = cache[0].shape[1], top(bits) + 1
    out = torch.zeros(B, hq, 1, dh, dtype=torch.float64)
    mag, ps, smax = torch.zeros_like(out), [], 0.0
    for b in range(B):
        n = int(cache[4][b])
        k, v = (rows(cache, w, b, n, bits, dh).repeat_interleave(hq // hkv, 0) for w in range(2))
        x = q[b, :, 0].double()
        p = torch.softmax(torch.einsum("hd,hnd->hn", x, k) * scale, -1)
        if n:
            out[b, :, 0] = torch.einsum("hn,hnd->hd", p, v)
            mag[b, :, 0] = torch.einsum("hn,hnd->hd", p, v.abs())
            t = torch.arange(n)
            pg, at = cache[3][b].long()[t // cache[0].shape[2]], t % cache[0].shape[2]
            ks = cache[2][pg, :, at, 0].double().repeat_interleave(GROUP, -1)[..., :dh]  # [n, hkv, dh]
            ks = ks.transpose(0, 1).repeat_interleave(hq // hkv, 0)
            smax = max(smax, float(torch.einsum("hd,hnd->hn", x.abs(), ks).max()) * 2 * zero * abs(scale))
        ps.append(p)
    return out, ps, mag, smax


def weight_error(n, dh, smax, dtype):
    """Bound on the relative error of a softmax weight and of a weighted sum of n terms: a score's sum of
    dh terms is off by at most 2 dh 2^-24 of their bound (an accumulator that truncates: twice that), and
    by 2^-22 of it for q in two fp16 parts (fp32) or below 2^-24 of the row's largest (bf16; less); it
    moves a weight by as much, once itself and once in the normaliser. Sums of n terms: n 2^-23. 2^x and
    the scaling by log2 e: a few 2^-23, and smax 2^-23. In bf16 the weights, times the values' scales,
    enter the second product in fp16, 2^-11; in fp32 in two fp16 parts, 2^-22."""
    u = 2.0 ** -23
    e = 2 * (2 * dh + 4) * u * smax + 2 * n * u + 16 * u
    return e + (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22)
