"""Cases of the serving operators over a paged key-value cache and of the logits processor, in their
plain form (elementary torch operations in 32 bits, rounded once at the end) and through the engine:

  append    rotated keys and values of new tokens into the pages of a cache (turbo_paged_append)
  attend    attention of one new token over a paged cache (turbo_paged_attention)
  evict     survivors by accumulated attention weight into new pages (turbo_paged_evict)
  logits    penalties, bias and token mask on a step's logits (one.engine.process_logits)

Pages are [num_pages, kv heads, page size, head dim]; a block table [B, pages] (int32) names each
sequence's pages in order, entries past its last page are -1. `own` selects the engine's calls.
"""
import functools
import math
import os
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one sequence early in its answer, the 140M model's heads: the latency of a call
        dict(name="attend 1 x 200 tokens", op="attend", dt="bf16", B=1, hkv=12, g=1, dh=64, page=16, longest=200, mass=False),
        # the 140M model's decode batch, ragged, some sequences not begun
        dict(name="attend 64 x 4096 ragged", op="attend", dt="bf16", B=64, hkv=12, g=1, dh=64, page=16, longest=4096, mass=False),
        # few long sequences, query heads sharing key heads: the largest cache
        dict(name="attend 8 x 32768 grouped", op="attend", dt="bf16", B=8, hkv=8, g=4, dh=128, page=64, longest=32768, mass=False),
        # a cache that is to be evicted from: weights accumulate; pages that are no power of two
        dict(name="attend 16 x 2500 weights", op="attend", dt="bf16", B=16, hkv=4, g=3, dh=64, page=48, longest=2500, mass=True),
        # fp32 models, the tiny configuration's heads
        dict(name="attend 8 x 3001 fp32", op="attend", dt="fp32", B=8, hkv=4, g=1, dh=64, page=32, longest=3001, mass=True),
        # the decode step's new token of 256 sequences
        dict(name="append 256 x 1", op="append", dt="bf16", B=256, n=1, hkv=12, g=1, dh=64, page=16, start=500, rope=True, mass=True),
        # prompts of different lengths into an empty cache
        dict(name="append 8 x 4096 prompts", op="append", dt="bf16", B=8, n=4096, hkv=12, g=1, dh=64, page=16, start=0, rope=True, mass=False),
        # a few sequences that outgrew their budget by a page
        dict(name="evict 4 x 1040 to 1024", op="evict", dt="bf16", B=4, hkv=12, dh=64, page=16, longest=1040, budget=1024, recent=256, sink=4),
        # long prompts cut down to a quarter
        dict(name="evict 16 x 8192 to 2048", op="evict", dt="bf16", B=16, hkv=12, dh=64, page=16, longest=8192, budget=2048, recent=512, sink=4),
        # one sequence's step with a repetition penalty
        dict(name="logits 1 x 32000", op="logits", dt="bf16", B=1, v=32000, hist=150, bias="none", mask="none"),
        # the decode batch with every penalty and one grammar
        dict(name="logits 256 x 32000", op="logits", dt="bf16", B=256, v=32000, hist=2176, bias="none", mask="shared"),
        # a larger, odd vocabulary in fp32, each request with its own bias and grammar
        dict(name="logits 48 x 50257 fp32", op="logits", dt="fp32", B=48, v=50257, hist=700, bias="rows", mask="rows"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "evict", "logits"])
    dt = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    size = 2 if dt == "bf16" else 4
    if op == "logits":
        v = _log(rng, 500, 160000)
        b = min(_log(rng, 1, 512), max(1, 8000000 // v))
        return dict(op=op, dt=dt, B=b, v=v, hist=_log(rng, 1, 8192), bias=rng.choice(["none", "shared", "rows"]),
                    mask=rng.choice(["none", "shared", "rows"]))
    hkv, g = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
    dh, page = rng.choice([32, 64, 64, 80, 96, 128]), rng.choice([1, 8, 16, 16, 32, 48, 64, 128])
    b = _log(rng, 1, 256)
    token = hkv * dh * 2 * size  # bytes of one token's keys and values
    if op == "attend":
        g = min(g, 64 // hkv or 1)
        longest = max(1, min(_log(rng, 1, 60000), 800000000 // (b * token * max(1, g // 4))))
        return dict(op=op, dt=dt, B=b, hkv=hkv, g=g, dh=dh, page=page, longest=longest, mass=rng.random() < 0.4)
    if op == "append":
        g = min(g, 4)
        n = max(1, min(rng.choice([1, _log(rng, 1, 8000)]), 100000000 // (b * token * (g + 1))))
        return dict(op=op, dt=dt, B=b, n=n, hkv=hkv, g=g, dh=dh, page=page, start=rng.choice([0, rng.randint(1, 600)]),
                    rope=rng.random() < 0.8, mass=rng.random() < 0.5)
    longest = max(2, min(_log(rng, 16, 60000), 400000000 // (b * token)))
    budget = max(1, int(longest * rng.uniform(0.1, 1.05)))
    recent = int(budget * rng.uniform(0, 0.6))
    return dict(op=op, dt=dt, B=b, hkv=hkv, dh=dh, page=page, longest=longest, budget=budget, recent=recent,
                sink=min(rng.choice([0, 1, 4, 16]), budget - recent))


# ------------------------------------------------------------------ inputs
def _ragged(b, longest, least=0):
    """Lengths of a batch: the first is the longest, the rest are spread over [least, longest]."""
    return [longest if i == 0 else least + int((i * 0.6180339887) % 1 * (longest - least + 1)) for i in range(b)]


def _tables(lists, width, gen, first=0):
    """Block table [B, width] over randomly ordered pages first .. : lists[b] pages for sequence b, then -1."""
    n = sum(lists)
    order = torch.randperm(n, device="cuda", generator=gen).to(torch.int32) + first
    table = torch.full((len(lists), width), -1, dtype=torch.int32)
    at = torch.zeros(len(lists), width, dtype=torch.int64)
    used = 0
    for i, k in enumerate(lists):
        table[i, :k] = 0
        at[i, :k] = torch.arange(used, used + k)
        used += k
    live = (table == 0).cuda()
    return torch.where(live, order[at.cuda()] if n else torch.zeros_like(at, dtype=torch.int32).cuda(), -1).to(torch.int32).contiguous(), n


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    dt, b = DT[case["dt"]], case["B"]
    s = dict(case)
    if case["op"] == "logits":
        v, t = case["v"], case["hist"]
        s["logits"] = normal(b, v, dtype=dt, scale=3.0)
        # frequent tokens come again and again; rows are filled behind a history with -1
        ids = (v * torch.rand(b, t, device="cuda", generator=gen) ** 4).to(torch.int64).clamp_(max=v - 1)
        own_len = torch.tensor(_ragged(b, t, t // 3), device="cuda")
        s["history"] = torch.where(torch.arange(t, device="cuda") < own_len[:, None], ids, -1)
        s["starts"] = (own_len // 2).to(torch.int32)
        s["repetition"] = 1.0 + 0.5 * torch.rand(b, device="cuda", generator=gen)
        s["presence"] = torch.rand(b, device="cuda", generator=gen)
        s["frequency"] = 0.2 * torch.rand(b, device="cuda", generator=gen)
        s["bias"] = None if case["bias"] == "none" else normal(*((v,) if case["bias"] == "shared" else (b, v)))
        words = (v + 31) // 32
        s["mask"] = None
        if case["mask"] != "none":
            shape = (words,) if case["mask"] == "shared" else (b, words)
            bits = [torch.randint(-2 ** 31, 2 ** 31, shape, device="cuda", generator=gen, dtype=torch.int64) for _ in range(2)]
            s["mask"] = (bits[0] | bits[1]).to(torch.int32)  # three tokens of four allowed
        return s
    hkv, dh, page = case["hkv"], case["dh"], case["page"]
    if case["op"] == "attend":
        lens = _ragged(b, case["longest"])
        width = max(1, -(-case["longest"] // page))
        s["table"], n = _tables([-(-x // page) for x in lens], width, gen)
        s["q"] = normal(b, hkv * case["g"], 1, dh, dtype=dt, scale=1.5)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["weights"] = torch.rand(b, hkv, width * page, device="cuda", generator=gen) if case["mass"] else None
    elif case["op"] == "append":
        n_new, start, g = case["n"], case["start"], case["g"]
        counts = _ragged(b, n_new, max(1, n_new // 4))
        starts = _ragged(b, start)
        width = -(-(start + n_new) // page)
        s["table"], n = _tables([-(-(x + c) // page) for x, c in zip(starts, counts)], width, gen)
        s["lengths"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda") if n_new > 1 else None
        # as projections leave them: [B, N, heads, dim], seen as [B, heads, N, dim]
        s["q"], s["k"], s["v"] = (normal(b, n_new, h, dh, dtype=dt).transpose(1, 2) for h in (hkv * g, hkv, hkv))
        s["cos"] = s["sin"] = None
        if case["rope"]:
            pos = s["lengths"].double()[:, None] + torch.arange(n_new, device="cuda")
            angle = pos[..., None] * 1e4 ** (-torch.arange(0, dh, 2, device="cuda").double() / dh)
            angle = torch.cat([angle, angle], -1)
            s["cos"], s["sin"] = angle.cos().to(dt), angle.sin().to(dt)
        s["weights"] = torch.rand(b, hkv, width * page, device="cuda", generator=gen) if case["mass"] else None
    else:
        lens = _ragged(b, case["longest"], case["longest"] // 2)
        width, to = -(-case["longest"] // page), -(-case["budget"] // page)
        s["table"], n = _tables([-(-x // page) for x in lens], width, gen)
        s["target"], m = _tables([-(-min(x, case["budget"]) // page) for x in lens], to, gen, first=n)
        n += m
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        # sums of attention weights: a few large ones, many small ones, some never attended and alike
        w = torch.exp(2.0 * torch.randn(b, hkv, width * page, device="cuda", generator=gen) - 2.0)
        s["weights"] = torch.where(w < 0.02, 0.0, w)
    s["k_pages"], s["v_pages"] = (normal(max(1, n), hkv, page, dh, dtype=dt) for _ in range(2))
    return s


# ------------------------------------------------------------------ the operators
@functools.lru_cache(maxsize=None)
def _engine():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "medit-one_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from one import engine, turbo_ops
    return engine, turbo_ops


def _rows(pages, table):
    """The cache of each sequence in order: [B, kv heads, table width * page size, dim]."""
    x = pages[table.clamp(min=0).long()]
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _attend(s):
    b, hkv, g, dh = s["B"], s["hkv"], s["g"], s["dh"]
    k, v = _rows(s["k_pages"], s["table"]).float(), _rows(s["v_pages"], s["table"]).float()
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
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos[:, None].float() + turned * sin[:, None].float()


def _append(s):
    n, page = s["n"], s["page"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["cos"] is not None:
        q, k = _rotate(q, s["cos"], s["sin"]), _rotate(k, s["cos"], s["sin"])
    at = torch.arange(n, device=k.device).expand(s["B"], n)
    if s["counts"] is not None:  # tokens behind a row's last one repeat it
        at = torch.minimum(at, s["counts"][:, None].long() - 1)
        pick = at[:, None, :, None].expand_as(k)
        k, v = k.gather(2, pick), v.gather(2, pick)
    slot = s["lengths"][:, None].long() + at
    pages = s["table"].long().gather(1, slot // page)
    s["k_pages"][pages, :, slot % page] = k.transpose(1, 2).to(s["k_pages"].dtype)
    s["v_pages"][pages, :, slot % page] = v.transpose(1, 2).to(s["v_pages"].dtype)
    out = [q.to(s["q"].dtype).contiguous(), s["k_pages"], s["v_pages"]]
    if s["weights"] is not None:
        s["weights"].scatter_(2, slot[:, None].expand(s["B"], s["hkv"], n), 0.0)
        out.append(s["weights"])
    return out


def _evict(s):
    b, hkv, dh, page, budget = s["B"], s["hkv"], s["dh"], s["page"], s["budget"]
    w, lens = s["weights"], s["lengths"].long()[:, None, None]
    slot = torch.arange(w.shape[2], device=w.device)
    kept_always = (slot < s["sink"]) | (slot >= lens - s["recent"])
    rank = torch.where(kept_always, math.inf, w)
    rank = torch.where(slot < lens, rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    top = order[..., :min(budget, w.shape[2])]
    kept = torch.where(top < lens, top, w.shape[2]).sort(-1).values  # slots in order, absent ones last
    there = kept < lens
    kept = torch.where(there, kept, -1)
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
    for pages in (s["k_pages"], s["v_pages"]):
        pages[dst_page, head, dst_slot] = pages[src_page, head, src_slot]
    weights = torch.where(there, w.gather(2, src), 0.0)
    weights = torch.nn.functional.pad(weights, (0, s["target"].shape[1] * page - budget))
    return weights, kept.to(torch.int32), s["k_pages"], s["v_pages"]


def _logits(s):
    b, v = s["B"], s["v"]
    x = s["logits"].float()
    there = s["history"] >= 0
    ids = s["history"].clamp(min=0)
    late = torch.arange(ids.shape[1], device=x.device) >= s["starts"][:, None]
    seen = torch.zeros(b, v, device=x.device).scatter_add_(1, ids, there.float())
    count = torch.zeros(b, v, device=x.device).scatter_add_(1, ids, (there & late).float())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        word = s["mask"].view(-1, s["mask"].shape[-1])
        tok = torch.arange(v, device=x.device)
        x = x.masked_fill(((word[:, tok // 32] >> (tok % 32)) & 1) == 0, -math.inf)
    return x, x.argmax(-1).to(torch.int32)


def run(s):
    op = s["op"]
    if not own:
        return {"attend": _attend, "append": _append, "evict": _evict, "logits": _logits}[op](s)
    engine, ops = _engine()
    if op == "attend":
        out = ops.turbo_paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], mass=s["weights"])
        return out if s["weights"] is None else (out, s["weights"])
    if op == "append":
        q = ops.turbo_paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], cos=s["cos"],
                                   sin=s["sin"], q=s["q"], counts=s["counts"], mass=s["weights"])
        return [q, s["k_pages"], s["v_pages"]] + ([] if s["weights"] is None else [s["weights"]])
    if op == "evict":
        weights, kept = ops.turbo_paged_evict(s["k_pages"], s["v_pages"], s["table"], s["target"], s["lengths"], s["weights"],
                                              s["budget"], recent=s["recent"], sink=s["sink"])
        return weights, kept, s["k_pages"], s["v_pages"]
    return engine.process_logits(s["logits"], s["history"], output_starts=s["starts"], repetition_penalty=s["repetition"],
                                 presence_penalty=s["presence"], frequency_penalty=s["frequency"], bias=s["bias"],
                                 token_mask=s["mask"], return_argmax=True)


def work(case):
    b, size = case["B"], 2 if case["dt"] == "bf16" else 4
    if case["op"] == "logits":
        v, rows = case["v"], {"none": 0, "shared": 1, "rows": b}
        hist = sum(_ragged(b, case["hist"], case["hist"] // 3))
        moved = b * v * (size + 4) + 4 * v * rows[case["bias"]] + v / 8 * rows[case["mask"]] + 8 * hist + 20 * b
        return {"bytes": moved, "flops": 6 * b * v}
    hkv, dh = case["hkv"], case["dh"]
    token = hkv * dh * 2 * size
    if case["op"] == "attend":
        tokens, hq = sum(_ragged(b, case["longest"])), hkv * case["g"]
        moved = tokens * (token + (8 * hkv if case["mass"] else 0)) + 2 * b * hq * dh * size
        return {"bytes": moved, "flops": 4 * tokens * hq * dh}
    if case["op"] == "append":
        tokens = sum(_ragged(b, case["n"], max(1, case["n"] // 4)))
        moved = 2 * tokens * token + 2 * b * case["n"] * hkv * case["g"] * dh * size
        moved += (2 * b * case["n"] * dh * size if case["rope"] else 0) + (4 * tokens * hkv if case["mass"] else 0)
        return {"bytes": moved, "flops": 3 * (tokens + b * case["n"] * case["g"]) * hkv * dh if case["rope"] else 0}
    lens = _ragged(b, case["longest"], case["longest"] // 2)
    kept = sum(min(x, case["budget"]) for x in lens)
    return {"bytes": 4 * hkv * sum(lens) + 2 * kept * token + 8 * b * hkv * case["budget"], "flops": 0}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        x, hist = s["logits"].double(), s["history"].tolist()
        starts = s["starts"].tolist()
        before, after = torch.zeros(x.shape, dtype=torch.bool), torch.zeros(x.shape, dtype=torch.float64)
        for i, row in enumerate(hist):
            ids = torch.tensor(row)
            late = ids[starts[i]:]
            before[i, ids[ids >= 0]] = True
            after[i] = torch.bincount(late[late >= 0], minlength=case["v"]).double()
        before, after = before.cuda(), after.cuda()
        r = s["repetition"].double()[:, None]
        x = torch.where(before & (x > 0), x / r, torch.where(before, x * r, x))
        x -= s["frequency"].double()[:, None] * after
        x -= s["presence"].double()[:, None] * (after >= 1)
        if s["bias"] is not None:
            x += s["bias"].double()
        if s["mask"] is not None:
            bits = s["mask"].cpu().numpy().view("uint8").reshape(-1, s["mask"].shape[-1] * 4)
            shift = torch.arange(8, dtype=torch.uint8)
            allowed = (torch.from_numpy(bits.copy())[..., None] >> shift & 1).reshape(bits.shape[0], -1)[:, :case["v"]]
            x[(allowed == 0).cuda().expand(x.shape)] = -math.inf
        return x, None
    page, lens = case["page"], s["lengths"].tolist()

    def one(pages, i, h, n):
        """The first n rows of sequence i's head h, one after the other."""
        return pages[s["table"][i, :-(-n // page)].long(), h].reshape(-1, case["dh"])[:n]

    if case["op"] == "attend":
        g = case["g"]
        q = s["q"].double()
        out = torch.zeros_like(q)
        weights = None if s["weights"] is None else s["weights"].double()
        if sum(lens) * case["hkv"] * case["dh"] > 4e8 or case["B"] * case["hkv"] > 4096:
            return None
        for i, n in enumerate(lens):
            for h in range(case["hkv"] if n else 0):
                z = q[i, h * g:(h + 1) * g, 0] @ one(s["k_pages"], i, h, n).double().t() / math.sqrt(case["dh"])
                p = torch.softmax(z, -1)
                out[i, h * g:(h + 1) * g, 0] = p @ one(s["v_pages"], i, h, n).double()
                if weights is not None:
                    weights[i, h, :n] += p.sum(0)
        return out if weights is None else (out, weights)
    if case["op"] == "append":
        def turn(x):
            if s["cos"] is None:
                return x.double()
            h = x.shape[-1] // 2
            c, sn, y = s["cos"].double()[:, None], s["sin"].double()[:, None], x.double()
            return torch.cat([y[..., :h] * c[..., :h] - y[..., h:] * sn[..., :h], y[..., h:] * c[..., h:] + y[..., :h] * sn[..., h:]], -1)
        q, k, v = turn(s["q"]).contiguous(), turn(s["k"]), s["v"].double()
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        weights = s["weights"]
        counts = [case["n"]] * case["B"] if s["counts"] is None else s["counts"].tolist()
        for i, (first, n) in enumerate(zip(lens, counts)):
            slots = torch.arange(first, first + n, device="cuda")
            at = s["table"][i].long()[slots // page]
            kp[at, :, slots % page] = k[i, :, :n].transpose(0, 1)
            vp[at, :, slots % page] = v[i, :, :n].transpose(0, 1)
            if weights is not None:
                weights[i, :, first:first + n] = 0
        return [q, kp, vp] + ([] if weights is None else [weights.double()])
    budget, recent, sink = case["budget"], case["recent"], case["sink"]
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    if case["B"] * case["hkv"] > 4096:
        return None
    weights = torch.zeros(case["B"], case["hkv"], s["target"].shape[1] * page, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        for h in range(case["hkv"]):
            if n <= budget:
                keep = torch.arange(n, device="cuda")
            else:
                middle = s["weights"][i, h, sink:n - recent]
                best = torch.argsort(-middle.double(), stable=True)[:budget - sink - recent] + sink
                edge = torch.arange(n, device="cuda")
                keep = torch.cat([edge[:sink], best.sort().values, edge[n - recent:]])
            m = len(keep)
            weights[i, h, :m] = s["weights"][i, h, keep].double()
            to = torch.arange(m, device="cuda")
            src, dst = s["table"][i].long()[keep // page], s["target"][i].long()[to // page]
            kp[dst, h, to % page] = s["k_pages"][src, h, keep % page].double()
            vp[dst, h, to % page] = s["v_pages"][src, h, keep % page].double()
    return weights, None, kp, vp
