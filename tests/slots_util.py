"""A check that attention over a paged cache counts every slot exactly once.

Keys hold a whole number s of 0 .. -8 in their first dim, queries 1 or 0 there, and the scale is ln 2,
so a slot weighs 2^s (or 1): the softmax is known exactly. The values of a window of Dh slots are the
rows of the identity, all others 0, so that out[d] is the weight of slot w + d alone; the window passes
over the whole length. A slot left out, counted twice or given another's value shifts an output by all
of a weight, whatever the length."""
import math

import torch


class Slots:
    def __init__(self, lens, hkv, g, dh, page, dtype, gen, device="cpu"):
        B, n = len(lens), max(max(lens), 1)
        self.lens, self.g, self.dh, self.dtype = lens, g, dh, dtype
        pages = [-(-x // page) for x in lens]
        order = torch.randperm(sum(pages) + 2, generator=gen)
        self.table = torch.full((B, max(max(pages), 1)), -1, dtype=torch.int32)
        at = 0
        for b, m in enumerate(pages):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.s = -torch.randint(0, 9, (B, hkv, n), generator=gen)
        k = torch.full((sum(pages) + 2, hkv, page, dh), math.nan)
        t = torch.arange(n)
        self.page_of, self.row_of = self.table.long()[:, t // page], t % page
        for b, x in enumerate(lens):
            k[self.page_of[b, :x], :, self.row_of[:x]] = 0.0
            k[self.page_of[b, :x], :, self.row_of[:x], 0] = self.s[b, :, :x].t().float()
        v = torch.where(torch.isnan(k), math.nan, 0.0)
        one = (torch.arange(hkv * g) % 3 != 2).float()  # every third query head weighs all slots alike
        q = torch.zeros(B, hkv * g, 1, dh)
        q[..., 0] = one[:, None]
        w = torch.exp2(self.s.double()).repeat_interleave(g, 1) * one[:, None] + (1 - one[:, None])
        w = torch.where(t < torch.tensor(lens)[:, None, None], w, 0.0)
        self.p = (w / w.sum(-1, keepdim=True).clamp(min=2.0 ** -60)).to(device)  # [B, Hq, n]
        self.lengths = torch.tensor(lens, dtype=torch.int32).to(device)
        self.k, self.v, self.q = (x.to(dtype).to(device) for x in (k, v, q))
        self.table = self.table.to(device)
        # A weight: 2^x to 2^-22, as often as sums are rescaled (8 times here, where the maximum rises)
        # or joined (warps, then parts), in the output and in the normaliser; the normaliser's sum,
        # which a lane takes over a 32nd of the slots or less, to half a step each.
        self.tol = 2 * 11 * 2.0 ** -22 + (n / 32 + 40) * 2.0 ** -24

    def mass(self):
        """Sum of the weights over each kv head's query heads, [B, Hkv, n]."""
        return self.p.unflatten(1, (-1, self.g)).sum(2)

    def check(self, attend):
        """attend(self) -> out [B, Hq, 1, Dh], for each window of values."""
        worst = 0.0
        for w in range(0, max(self.lens), self.dh):
            marks = []
            for b, x in enumerate(self.lens):
                t = torch.arange(min(w, x), min(w + self.dh, x))
                if len(t):
                    marks.append((self.page_of[b, t], self.row_of[t], t - w))
            pg, row, d = (torch.cat(m).to(self.v.device) for m in zip(*marks))
            self.v[pg, :, row, d] = 1.0
            got = attend(self)[:, :, 0].double()
            self.v[pg, :, row, d] = 0.0
            want = torch.zeros_like(got)
            part = self.p[..., w:w + self.dh]
            want[..., :part.shape[-1]] = part
            err = (got - want).abs() - (torch.finfo(self.dtype).eps / 2 + self.tol) * want
            worst = max(worst, float(torch.nan_to_num(err, nan=math.inf).max()))
        assert worst <= 0, f"{worst:.3g} over"


def oracle(s, lost=(), twice=()):
    """Attention in 64 bits, rounded once; the slots `lost` (of sequence 0) do not reach the output, the
    slots `twice` reach it twice."""
    n = s.p.shape[-1]
    out = torch.zeros(s.q.shape, dtype=torch.float64)
    for b, x in enumerate(s.lens):
        p = s.p[b, :, :x].clone()
        if b == 0:
            p[:, list(lost)] = 0.0
            p[:, list(twice)] *= 2.0
        v = s.v[s.page_of[b, :x], :, s.row_of[:x]].double().transpose(0, 1).repeat_interleave(s.g, 0)
        out[b, :, 0] = torch.einsum("hn,hnd->hd", p, v)
    return out.to(s.dtype)
