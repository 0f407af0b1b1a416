"""Cases of the serving operators over a paged key-value cache that is held in 4 or 8 bits, in their
plain form (elementary torch operations in 32 bits, rounded once at the end) and through the engine:

  attend    attention of one new token over the cache (turbo_paged_quant_attention)
  store     rotated keys and values of new tokens quantised into its pages, and read back as the cache
            holds them (turbo_paged_quant_append, turbo_paged_quant_read)
  read      the sequences' keys and values out of the pages, dense (turbo_paged_quant_read)
  evict     survivors by accumulated attention weight into new pages, and read there
            (turbo_paged_quant_evict, turbo_paged_quant_read)

A head's row of Dh values is cut into groups of 32 (the last one may be shorter). A group stands for
scale * code: scale = bf16(max |x| / m) with m = 7 (4 bits) or 127 (8 bits), code = x / scale rounded to
the nearest whole number, halves to the even one. x is the value in fp32 (a rotated key rounded to it
once). Scales below 2^-100 are held as 0, with codes of 0; a group with an infinity or NaN has the
scale NaN, and codes of 0. Codes lie in bytes, 8 added (4 bits; the even dim in the low half) or 128:

  k_pages, v_pages   uint8 [num_pages, kv heads, page size, Dh * bits / 8]
  scales             bf16 [num_pages, kv heads, page size, 2 (key, value), groups]

A block table [B, pages] (int32) names each sequence's pages in order; entries past its last page are
-1. `own` selects the engine's calls.
"""
import functools
import math
import os
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
GROUP = 32


def listed():
    return [
        # one sequence early in its answer, the 140M model's heads: the latency of a call
        dict(name="attend 1 x 200 tokens", op="attend", dt="bf16", bits=4, B=1, hkv=12, g=1, dh=64, page=16, longest=200, mass=False),
        # the 140M model's decode batch, ragged, some sequences not begun
        dict(name="attend 64 x 4096 ragged", op="attend", dt="bf16", bits=4, B=64, hkv=12, g=1, dh=64, page=16, longest=4096, mass=False),
        # few long sequences, query heads sharing key heads: the largest cache
        dict(name="attend 8 x 32768 grouped", op="attend", dt="bf16", bits=4, B=8, hkv=8, g=4, dh=128, page=64, longest=32768, mass=False),
        # a cache in 8 bits that is to be evicted from: weights accumulate; pages that are no power of two
        dict(name="attend 16 x 2500 weights, 8 bits", op="attend", dt="bf16", bits=8, B=16, hkv=4, g=3, dh=64, page=48, longest=2500, mass=True),
        # fp32 models, the tiny configuration's heads
        dict(name="attend 8 x 3001 fp32", op="attend", dt="fp32", bits=4, B=8, hkv=4, g=1, dh=64, page=32, longest=3001, mass=True),
        # the decode step's new token of 256 sequences
        dict(name="store 256 x 1", op="store", dt="bf16", bits=4, B=256, n=1, hkv=12, g=1, dh=64, page=16, start=500, rope=True, mass=True),
        # prompts of different lengths into an empty cache
        dict(name="store 8 x 4096 prompts", op="store", dt="bf16", bits=4, B=8, n=4096, hkv=12, g=1, dh=64, page=16, start=0, rope=True, mass=False),
        # fp32 prompts behind a shared beginning, in 8 bits; heads that are no power of two, small pages
        dict(name="store 5 x 777 fp32, 8 bits", op="store", dt="fp32", bits=8, B=5, n=777, hkv=4, g=2, dh=80, page=8, start=130, rope=True, mass=False),
        # a prompt's cache for a dense pass over it
        dict(name="read 1 x 500, 8 bits", op="read", dt="bf16", bits=8, B=1, hkv=12, dh=64, page=16, longest=500),
        # a batch's whole caches
        dict(name="read 16 x 4096", op="read", dt="bf16", bits=4, B=16, hkv=12, dh=64, page=16, longest=4096),
        # a few sequences that outgrew their budget by a page
        dict(name="evict 4 x 1040 to 1024", op="evict", dt="bf16", bits=4, B=4, hkv=12, dh=64, page=16, longest=1040, budget=1024, recent=256, sink=4),
        # long prompts cut down to a quarter
        dict(name="evict 16 x 8192 to 2048", op="evict", dt="bf16", bits=4, B=16, hkv=12, dh=64, page=16, longest=8192, budget=2048, recent=512, sink=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "store", "read", "evict"])
    dt, bits = rng.choice(["bf16", "bf16", "bf16", "fp32"]), rng.choice([4, 4, 8])
    size = 2 if dt == "bf16" else 4
    hkv, g = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
    dh, page = rng.choice([32, 64, 64, 80, 96, 128]), rng.choice([1, 8, 16, 16, 32, 48, 64, 128])
    b = _log(rng, 1, 256)
    base = dict(op=op, dt=dt, bits=bits, B=b, hkv=hkv, dh=dh, page=page)
    dense, token = hkv * dh * 2 * size, _token(base)  # bytes of one token's keys and values, dense and held
    if op == "attend":
        g = min(g, 64 // hkv or 1)
        longest = max(1, min(_log(rng, 1, 60000), 150000000 // (b * token * max(1, g // 4))))
        return dict(base, g=g, longest=longest, mass=rng.random() < 0.4)
    if op == "store":
        g = min(g, 4)
        n = max(1, min(rng.choice([1, _log(rng, 1, 8000)]), 100000000 // (b * dense * (g + 1))))
        return dict(base, g=g, n=n, start=rng.choice([0, rng.randint(1, 600)]), rope=rng.random() < 0.8, mass=rng.random() < 0.5)
    if op == "read":
        return dict(base, longest=max(1, min(_log(rng, 1, 60000), 200000000 // (b * dense))))
    longest = max(2, min(_log(rng, 16, 60000), 200000000 // (b * token)))
    budget = max(1, min(int(longest * rng.uniform(0.1, 1.05)), 200000000 // (b * dense)))
    recent = int(budget * rng.uniform(0, 0.6))
    return dict(base, longest=longest, budget=budget, recent=recent, sink=min(rng.choice([0, 1, 4, 16]), budget - recent))


def _token(case):
    """Bytes of one token's keys and values in the cache."""
    dh = case["dh"]
    return case["hkv"] * 2 * (dh * case["bits"] // 8 + 2 * -(-dh // GROUP))


# ------------------------------------------------------------------ inputs
def _ragged(b, longest, least=0):
    """Lengths of a batch: the first is the longest, the rest are spread over [least, longest]."""
    return [longest if i == 0 else least + int((i * 0.6180339887) % 1 * (longest - least + 1)) for i in range(b)]


def _tables(pages, width, gen, first=0):
    """Block table [B, width] over the pages first .. in random order, pages[b] of them for sequence b, then -1."""
    n = sum(pages)
    order = (torch.randperm(n, device="cuda", generator=gen) + first).to(torch.int32)
    used = torch.tensor(pages, device="cuda")
    at = torch.arange(width, device="cuda")
    place = (used.cumsum(0) - used)[:, None] + at
    if n == 0:
        return torch.full((len(pages), width), -1, dtype=torch.int32, device="cuda"), 0
    return torch.where(at < used[:, None], order[place.clamp(max=n - 1)], -1).to(torch.int32).contiguous(), n


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    def lens_of(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    dt, b, hkv, dh, page, bits = DT[case["dt"]], case["B"], case["hkv"], case["dh"], case["page"], case["bits"]
    s = dict(case)
    s["starts"] = None
    if case["op"] == "attend":
        lens = _ragged(b, case["longest"])
        width = max(1, -(-case["longest"] // page))
        s["table"], n = _tables([-(-x // page) for x in lens], width, gen)
        s["q"] = normal(b, hkv * case["g"], 1, dh, dtype=dt, scale=1.5)
        s["lengths"] = lens_of(lens)
        s["weights"] = torch.rand(b, hkv, width * page, device="cuda", generator=gen) if case["mass"] else None
    elif case["op"] == "store":
        n_new, start, g = case["n"], case["start"], case["g"]
        counts = _ragged(b, n_new, max(1, n_new // 4))
        starts = _ragged(b, start)
        width = -(-(start + n_new) // page)
        s["table"], n = _tables([-(-(x + c) // page) for x, c in zip(starts, counts)], width, gen)
        s["lengths"], s["after"] = lens_of(starts), lens_of([x + c for x, c in zip(starts, counts)])
        s["counts"] = lens_of(counts) if n_new > 1 else None
        # as projections leave them: [B, N, heads, dim], seen as [B, heads, N, dim]; some channels larger than others
        s["q"], s["k"], s["v"] = ((normal(b, n_new, h, dh) * torch.exp(normal(h, dh, scale=0.5))).to(dt).transpose(1, 2)
                                  for h in (hkv * g, hkv, hkv))
        s["cos"] = s["sin"] = None
        if case["rope"]:
            pos = s["lengths"].double()[:, None] + torch.arange(n_new, device="cuda")
            angle = pos[..., None] * 1e4 ** (-torch.arange(0, dh, 2, device="cuda").double() / dh)
            angle = torch.cat([angle, angle], -1)
            s["cos"], s["sin"] = angle.cos().to(dt), angle.sin().to(dt)
        s["weights"] = torch.rand(b, hkv, width * page, device="cuda", generator=gen) if case["mass"] else None
    elif case["op"] == "read":
        lens = _ragged(b, case["longest"])
        s["table"], n = _tables([-(-x // page) for x in lens], -(-case["longest"] // page), gen)
        s["lengths"], s["n"] = lens_of(lens), case["longest"]
    else:
        lens = _ragged(b, case["longest"], case["longest"] // 2)
        width, to = -(-case["longest"] // page), -(-case["budget"] // page)
        s["table"], n = _tables([-(-x // page) for x in lens], width, gen)
        s["target"], m = _tables([-(-min(x, case["budget"]) // page) for x in lens], to, gen, first=n)
        n += m
        s["lengths"], s["after"] = lens_of(lens), lens_of([min(x, case["budget"]) for x in lens])
        # sums of attention weights: a few large ones, many small ones, some never attended and alike
        w = torch.exp(2.0 * torch.randn(b, hkv, width * page, device="cuda", generator=gen) - 2.0)
        s["weights"] = torch.where(w < 0.02, 0.0, w)
    # codes as normal values leave them
    top, n = 7 if bits == 4 else 127, max(1, n)

    def codes():
        u = (torch.randn(n, hkv, page, dh, device="cuda", generator=gen) * (top / 2.1)).round_().clamp_(-top, top).add_(top + 1).to(torch.uint8)
        return (u[..., 0::2] | u[..., 1::2] << 4).contiguous() if bits == 4 else u
    s["k_pages"], s["v_pages"] = codes(), codes()
    s["scales"] = torch.exp(normal(n, hkv, page, 2, -(-dh // GROUP), scale=0.4)).mul_(2.1 / top).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------ the operators
@functools.lru_cache(maxsize=None)
def _ops():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "medit-one_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from one import turbo_ops
    return turbo_ops


def _open(codes, scales, s):
    """Rows of codes [..., bytes] and their scales [..., groups] as the values they stand for, in fp32."""
    if s["bits"] == 4:
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    else:
        c = codes.float() - 128.0
    return c * scales.float().repeat_interleave(GROUP, -1)[..., :s["dh"]]


def _close(x, s):
    """Codes and scales of rows of fp32 values."""
    dh, top = s["dh"], 7 if s["bits"] == 4 else 127
    groups = -(-dh // GROUP)
    wide = torch.nn.functional.pad(x, (0, groups * GROUP - dh)).unflatten(-1, (groups, GROUP))
    largest = wide.abs().amax(-1)
    scale = (largest / torch.full_like(largest, top)).to(torch.bfloat16).float()  # by a tensor: a quotient, no product with 1 / top
    there = torch.isfinite(largest) & (scale >= 2.0 ** -100)
    scale = torch.where(torch.isfinite(largest), torch.where(there, scale, 0.0), math.nan)
    c = torch.where(there[..., None], torch.round(wide / torch.where(there, scale, 1.0)[..., None]), 0.0)
    u = (c + float(top + 1)).to(torch.uint8).flatten(-2)[..., :dh]
    return (u[..., 0::2] | u[..., 1::2] << 4) if s["bits"] == 4 else u, scale.to(torch.bfloat16)


def _rows(s, which, table):
    """Keys (0) or values (1) of each sequence in order: [B, kv heads, table width * page size, dim]."""
    at = table.clamp(min=0).long()
    codes = s["v_pages" if which else "k_pages"][at].permute(0, 2, 1, 3, 4).flatten(2, 3)
    return _open(codes, s["scales"][:, :, :, which][at].permute(0, 2, 1, 3, 4).flatten(2, 3), s)


def _read(s, table, lengths, starts, n):
    dt = DT[s["dt"]]
    first = torch.zeros_like(lengths) if starts is None else starts
    slot = first[:, None].long() + torch.arange(n, device=table.device)
    live = slot < lengths[:, None]
    slot = torch.where(live, slot, 0)
    page = table.long().gather(1, slot // s["page"]).clamp(min=0)
    out = []
    for which, pool in enumerate((s["k_pages"], s["v_pages"])):
        x = _open(pool[page, :, slot % s["page"]], s["scales"][page, :, slot % s["page"], which], s)
        out.append(torch.where(live[..., None, None], x, 0.0).to(dt).transpose(1, 2).contiguous())
    return out


def _attend(s):
    b, hkv, g, dh = s["B"], s["hkv"], s["g"], s["dh"]
    k, v = _rows(s, 0, s["table"]), _rows(s, 1, s["table"])
    live = torch.arange(k.shape[2], device=k.device) < s["lengths"][:, None]
    q = s["q"].float().view(b, hkv, g, dh)
    scores = torch.matmul(q, k.transpose(-1, -2)) * (dh ** -0.5)
    scores = scores.masked_fill(~live[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, torch.where(live[:, None, :, None], v, 0.0)).view(b, hkv * g, 1, dh).to(s["q"].dtype)
    if s["weights"] is None:
        return out
    s["weights"] += p.sum(2)
    return out, s["weights"]


def _rotate(x, cos, sin):
    """In 64 bits, to the fp32 value: its last bit may decide a code."""
    half = x.shape[-1] // 2
    x = x.double()
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return (x * cos[:, None].double() + turned * sin[:, None].double()).float()


def _store(s):
    n, page = s["n"], s["page"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["cos"] is not None:
        q, k = _rotate(s["q"], s["cos"], s["sin"]), _rotate(s["k"], s["cos"], s["sin"])
    at = torch.arange(n, device=k.device).expand(s["B"], n)
    if s["counts"] is not None:  # tokens behind a row's last one repeat it
        at = torch.minimum(at, s["counts"][:, None].long() - 1)
        pick = at[:, None, :, None].expand_as(k)
        k, v = k.gather(2, pick), v.gather(2, pick)
    slot = s["lengths"][:, None].long() + at
    pages = s["table"].long().gather(1, slot // page)
    for which, (x, pool) in enumerate(((k, s["k_pages"]), (v, s["v_pages"]))):
        codes, scales = _close(x.transpose(1, 2), s)
        pool[pages, :, slot % page] = codes
        s["scales"][pages, :, slot % page, which] = scales
    out = [q.to(s["q"].dtype).contiguous(), *_read(s, s["table"], s["after"], s["lengths"], n), s["scales"]]
    if s["weights"] is not None:
        s["weights"].scatter_(2, slot[:, None].expand(s["B"], s["hkv"], n), 0.0)
        out.append(s["weights"])
    return out


def _evict(s):
    b, hkv, page, budget = s["B"], s["hkv"], s["page"], s["budget"]
    w, lens = s["weights"], s["lengths"].long()[:, None, None]
    slot = torch.arange(w.shape[2], device=w.device)
    kept_always = (slot < s["sink"]) | (slot >= lens - s["recent"])
    rank = torch.where(kept_always, math.inf, w)
    rank = torch.where(slot < lens, rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    top = order[..., :min(budget, w.shape[2])]
    kept = torch.where(top < lens, top, w.shape[2]).sort(-1).values  # slots in order, absent ones last
    kept = torch.where(kept < lens, kept, -1)
    if kept.shape[2] < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[2]), value=-1)
    there = kept >= 0
    src = kept.clamp(min=0)
    to_slot = torch.arange(budget, device=w.device)
    from_page = s["table"].long()[:, None].expand(b, hkv, -1).gather(2, src // page)
    to_page = s["target"].long()[:, None].expand(b, hkv, -1)[:, :, to_slot // page]
    # absent ones repeat the sequence's first survivor, where it goes
    src_page = torch.where(there, from_page, from_page[..., :1])
    src_slot = torch.where(there, src % page, src[..., :1] % page)
    dst_page = torch.where(there, to_page, to_page[..., :1])
    dst_slot = torch.where(there, to_slot % page, 0)
    head = torch.arange(hkv, device=w.device)[:, None]
    for pages in (s["k_pages"], s["v_pages"], s["scales"]):
        pages[dst_page, head, dst_slot] = pages[src_page, head, src_slot]
    weights = torch.where(there, w.gather(2, src), 0.0)
    weights = torch.nn.functional.pad(weights, (0, s["target"].shape[1] * page - budget))
    return [weights, kept.to(torch.int32), *_read(s, s["target"], s["after"], None, budget), s["scales"]]


def run(s):
    op = s["op"]
    if not own:
        if op == "read":
            return _read(s, s["table"], s["lengths"], None, s["n"])
        return {"attend": _attend, "store": _store, "evict": _evict}[op](s)
    ops, dt = _ops(), DT[s["dt"]]
    pools = s["k_pages"], s["v_pages"], s["scales"]
    if op == "attend":
        out = ops.turbo_paged_quant_attention(s["q"], *pools, s["table"], s["lengths"], mass=s["weights"])
        return out if s["weights"] is None else (out, s["weights"])
    if op == "store":
        q = ops.turbo_paged_quant_append(s["k"], s["v"], *pools, s["table"], s["lengths"], cos=s["cos"], sin=s["sin"], q=s["q"],
                                         counts=s["counts"], mass=s["weights"])
        k, v = ops.turbo_paged_quant_read(*pools, s["table"], s["after"], s["n"], s["dh"], starts=s["lengths"], dtype=dt)
        return [q, k, v, s["scales"]] + ([] if s["weights"] is None else [s["weights"]])
    if op == "read":
        return list(ops.turbo_paged_quant_read(*pools, s["table"], s["lengths"], s["n"], s["dh"], dtype=dt))
    weights, kept = ops.turbo_paged_quant_evict(*pools, s["table"], s["target"], s["lengths"], s["weights"], s["budget"],
                                                recent=s["recent"], sink=s["sink"])
    k, v = ops.turbo_paged_quant_read(*pools, s["target"], s["after"], s["budget"], s["dh"], dtype=dt)
    return [weights, kept, k, v, s["scales"]]


def work(case):
    b, size, hkv, dh = case["B"], 2 if case["dt"] == "bf16" else 4, case["hkv"], case["dh"]
    token, dense = _token(case), hkv * dh * 2 * size
    if case["op"] == "attend":
        tokens, hq = sum(_ragged(b, case["longest"])), hkv * case["g"]
        moved = tokens * (token + (8 * hkv if case["mass"] else 0)) + 2 * b * hq * dh * size
        return {"bytes": moved, "flops": 4 * tokens * hq * dh}
    if case["op"] == "store":  # the tokens come, and go into the cache and out as it holds them
        n = case["n"]
        tokens = sum(_ragged(b, n, max(1, n // 4)))
        moved = tokens * (dense + token) + b * n * dense + 2 * b * n * hkv * case["g"] * dh * size
        moved += (2 * b * n * dh * size if case["rope"] else 0) + (4 * tokens * hkv if case["mass"] else 0)
        return {"bytes": moved, "flops": 3 * (tokens + b * n * case["g"]) * hkv * dh if case["rope"] else 0}
    if case["op"] == "read":
        return {"bytes": sum(_ragged(b, case["longest"])) * token + b * case["longest"] * dense, "flops": 0}
    lens = _ragged(b, case["longest"], case["longest"] // 2)
    kept = sum(min(x, case["budget"]) for x in lens)
    return {"bytes": 4 * hkv * sum(lens) + 2 * kept * token + b * case["budget"] * (dense + 8 * hkv), "flops": 0}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    page, lens, dh, bits, hkv = case["page"], s["lengths"].tolist(), case["dh"], case["bits"], case["hkv"]
    pools = s["k_pages"], s["v_pages"]

    def worth(u, sc):
        """Bytes [n, row] and scales [n, groups] -> float64 [n, dh]."""
        n = u.shape[0]
        if bits == 4:
            c = torch.empty(n, dh, dtype=torch.float64, device=u.device)
            c[:, 0::2], c[:, 1::2] = (u % 16).double() - 8, torch.div(u, 16, rounding_mode="floor").double() - 8
        else:
            c = u.double() - 128
        for i in range(sc.shape[1]):
            c[:, 32 * i:32 * i + 32] *= sc[:, i:i + 1].double()
        return c

    def one(which, i, h, n, table=None):
        """The first n rows of sequence i's head h, one after the other."""
        at = (s["table"] if table is None else table)[i, :-(-n // page)].long()
        u = pools[which][at, h].reshape(len(at) * page, -1)[:n]
        return worth(u, s["scales"][at, h, :, which].reshape(len(at) * page, -1)[:n])

    if case["B"] * hkv > 4096:
        return None
    if case["op"] == "attend":
        g = case["g"]
        q = s["q"].double()
        out = torch.zeros_like(q)
        weights = None if s["weights"] is None else s["weights"].double()
        if sum(lens) * hkv * dh > 4e8:
            return None
        for i, n in enumerate(lens):
            for h in range(hkv if n else 0):
                z = q[i, h * g:(h + 1) * g, 0] @ one(0, i, h, n).t() / math.sqrt(dh)
                p = torch.softmax(z, -1)
                out[i, h * g:(h + 1) * g, 0] = p @ one(1, i, h, n)
                if weights is not None:
                    weights[i, h, :n] += p.sum(0)
        return out if weights is None else (out, weights)
    if case["op"] == "read":
        out = [torch.zeros(case["B"], hkv, s["n"], dh, dtype=torch.float64, device="cuda") for _ in range(2)]
        for i, n in enumerate(lens):
            for h in range(hkv if n else 0):
                for which in range(2):
                    out[which][i, h, :n] = one(which, i, h, n)
        return out
    if case["op"] == "store":
        def turn(x):
            if s["cos"] is None:
                return x.double()
            h = dh // 2
            c, sn, y = s["cos"].double()[:, None], s["sin"].double()[:, None], x.double()
            return torch.cat([y[..., :h] * c[..., :h] - y[..., h:] * sn[..., :h], y[..., h:] * c[..., h:] + y[..., :h] * sn[..., h:]], -1)

        def held(x):
            """[hkv, n, dh] as the cache holds it, and its scales."""
            y, sc = torch.zeros_like(x), []
            x = x.float().double()  # the definition's fp32 value
            for at in range(0, dh, 32):
                part = x[..., at:at + 32]
                step = (part.abs().max(-1, keepdim=True).values / (2 ** (bits - 1) - 1)).float().bfloat16().double()
                step[step < 2.0 ** -100] = 0.0
                y[..., at:at + 32] = torch.where(step > 0, torch.round(part / step) * step, 0.0)
                sc.append(step)
            return y, torch.cat(sc, -1)
        q = turn(s["q"]).contiguous()
        new = turn(s["k"]), s["v"].double()
        dense = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in new]
        scales, weights = s["scales"].double(), s["weights"]
        counts = [case["n"]] * case["B"] if s["counts"] is None else s["counts"].tolist()
        for i, (first, n) in enumerate(zip(lens, counts)):
            slots = torch.arange(first, first + n, device="cuda")
            at = s["table"][i].long()[slots // page]
            for which in range(2):
                dense[which][i, :, :n], sc = held(new[which][i, :, :n])
                scales[at, :, slots % page, which] = sc.transpose(0, 1)
            if weights is not None:
                weights[i, :, first:first + n] = 0
        return [q, *dense, scales] + ([] if weights is None else [weights.double()])
    budget, recent, sink = case["budget"], case["recent"], case["sink"]
    weights = torch.zeros(case["B"], hkv, s["target"].shape[1] * page, dtype=torch.float64, device="cuda")
    dense = [torch.zeros(case["B"], hkv, budget, dh, dtype=torch.float64, device="cuda") for _ in range(2)]
    scales = s["scales"].double()
    for i, n in enumerate(lens):
        for h in range(hkv):
            if n <= budget:
                keep = torch.arange(n, device="cuda")
            else:
                middle = s["weights"][i, h, sink:n - recent]
                best = torch.argsort(-middle.double(), stable=True)[:budget - sink - recent] + sink
                edge = torch.arange(n, device="cuda")
                keep = torch.cat([edge[:sink], best.sort().values, edge[n - recent:]])
            m = len(keep)
            weights[i, h, :m] = s["weights"][i, h, keep].double()
            for which in range(2):
                dense[which][i, h, :m] = one(which, i, h, n)[keep]
            to = torch.arange(m, device="cuda")
            src, dst = s["table"][i].long()[keep // page], s["target"][i].long()[to // page]
            scales[dst, h, to % page] = s["scales"][src, h, keep % page].double()
    return weights, None, *dense, scales
