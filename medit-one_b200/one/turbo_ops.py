"""one.turbo_ops: the reference's turbo entry points (one/turbo_ops.py:96-475), backed by
libone_b200.so. TURBO_MODE is True when the native library loads with every entry point.

There is no CPU fallback: the turbo functions require CUDA tensors and raise otherwise.
"""
from __future__ import annotations

import ctypes
import warnings
from typing import Optional, Tuple

import torch

try:
    from . import _capi as C
    TURBO_MODE = True
except Exception as exc:  # the library is required for every op below
    C = None
    TURBO_MODE = False
    warnings.warn(f"One B200 engine not available ({exc}); turbo ops will raise")


def _need(*ts):
    if not TURBO_MODE:
        raise RuntimeError("libone_b200.so is not built: run `python medit-one_b200/build.py`")
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("the B200 engine has no CPU path: pass CUDA tensors")


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def turbo_flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True,
                          scale_factor: Optional[float] = None) -> torch.Tensor:
    """softmax(q k^T * scale [+ causal mask]) v with an fp32 softmax (one/turbo_ops.py:96-143).
    q [B, H, Nq, Dh], k / v [B, H, Nk, Dh]."""
    _need(q, k, v)
    if scale_factor is None:
        scale_factor = 1.0 / (q.size(-1) ** 0.5)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    B, H, Nq, Dh = q.shape
    out = torch.empty_like(q)
    C.check(C.LIB.one_flash_attention(C.ptr(q), C.ptr(k), C.ptr(v), B, H, Nq, k.shape[2], Dh, 1 if causal else 0,
                                      float(scale_factor), C.dtype_code(q.dtype), C.ptr(out), _stream()),
            "one_flash_attention")
    return out


def turbo_rope_flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                               sin: torch.Tensor, causal: bool = True,
                               scale_factor: Optional[float] = None) -> torch.Tensor:
    """apply_rotary_pos_emb_flash(q, k, cos, sin) (one/flash_attention.py:26-33) followed by
    turbo_flash_attention, as one native call. q, k, v [B, H, N, Dh]; cos, sin [B or 1, N, Dh]
    in q's dtype (OneRotaryEmbedding's output)."""
    _need(q, k, v, cos, sin)
    if scale_factor is None:
        scale_factor = 1.0 / (q.size(-1) ** 0.5)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cos, sin = cos.to(q.dtype).contiguous(), sin.to(q.dtype).contiguous()
    B, H, N, Dh = q.shape
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError("q, k and v must have the same shape [B, H, N, Dh]")
    cb = cos.shape[0] if cos.dim() == 3 else 1
    if cos.shape[-2:] != (N, Dh) or sin.shape != cos.shape or cb not in (1, B):
        raise ValueError(f"cos / sin must be [B or 1, {N}, {Dh}], got {tuple(cos.shape)}")
    dt = C.dtype_code(q.dtype)
    ws = torch.empty(C.LIB.one_rope_flash_attention_workspace_bytes(B, H, N, Dh, dt), dtype=torch.uint8,
                     device=q.device)
    out = torch.empty_like(q)
    C.check(C.LIB.one_rope_flash_attention(C.ptr(q), C.ptr(k), C.ptr(v), C.ptr(cos), C.ptr(sin), cb, B, H, N, Dh,
                                           1 if causal else 0, float(scale_factor), dt, C.ptr(out), C.ptr(ws),
                                           ws.numel(), _stream()),
            "one_rope_flash_attention")
    return out


def ops_error(clear: bool = True) -> Tuple[int, int]:
    """(code, site) of the standalone ops' device error record (0 = none); synchronises."""
    _need()
    where = ctypes.c_int32(0)
    code = C.LIB.one_ops_error(ctypes.byref(where), 1 if clear else 0)
    return int(code), int(where.value)


def turbo_moe_routing(inputs: torch.Tensor, experts_weights: torch.Tensor, top_k: int) -> torch.Tensor:
    """The reference's turbo_moe_routing (one/turbo_ops.py:146-172) returns its inputs: its
    PyTorch path computes a top-k that it discards. Kept as is. The LinearMoE router itself
    is `one.linear_moe.LinearMoE` / the C ABI `one_moe_routing`."""
    _need(inputs)
    return inputs


def turbo_rotary_embedding(x: torch.Tensor, position_ids: torch.Tensor, inv_freq: torch.Tensor
                           ) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos, sin [B, S, dim] in x's dtype (OneRotaryEmbedding.forward, one/modeling_one.py:159-182)."""
    _need(x, position_ids, inv_freq)
    pos = position_ids.to(torch.int64).contiguous()
    inv = inv_freq.to(torch.float32).contiguous()
    B, S = pos.shape
    dim = 2 * inv.numel()
    cos = torch.empty(B, S, dim, dtype=x.dtype, device=x.device)
    sin = torch.empty_like(cos)
    C.check(C.LIB.one_rotary_embedding(C.ptr(pos), B, S, C.ptr(inv), dim, C.dtype_code(x.dtype), C.ptr(cos), C.ptr(sin),
                                       _stream()), "one_rotary_embedding")
    return cos, sin


def turbo_cumsum_and_normalize(x: torch.Tensor, seq_len: int) -> torch.Tensor:
    """fp32 prefix mean over dim 1 (turbo_cumsum_and_normalize_cpu, one/turbo_ops.py:288-310)."""
    _need(x)
    x = x.contiguous()
    b, s, d = x.shape
    n = min(s, int(seq_len))
    out = torch.empty(b, n, d, dtype=x.dtype, device=x.device)
    C.check(C.LIB.one_cumsum_and_normalize(C.ptr(x), b, s, d, int(seq_len), C.dtype_code(x.dtype), C.ptr(out), _stream()),
            "one_cumsum_and_normalize")
    return out


def turbo_combined_rope_attention(single_x, key, value, cos, sin, lin_q, lin_k, lin_v, compute_sequence_len: int):
    """RoPE + three Dh->H projections + softmax(q*k - max) * v (the model's feature attention,
    one/modeling_one.py:515-547; the reference's own CPU version of this entry point raises
    NameError). Inputs [B, H, T, Dh]; cos/sin [B or 1, T, Dh]; returns [B, H, T, H]."""
    _need(single_x, key, value, cos, sin)
    t = int(compute_sequence_len)
    sx = single_x[:, :, -t:].contiguous()
    ky = key[:, :, -t:].contiguous()
    va = value[:, :, -t:].contiguous()
    if cos.dim() == 4:
        cos, sin = cos[:, 0], sin[:, 0]
    cos = cos[:, -t:].contiguous()
    sin = sin[:, -t:].contiguous()
    B, H, T, Dh = sx.shape
    hout = lin_q.weight.shape[0]
    dt = sx.dtype
    ws = [m.weight.to(dt).contiguous() for m in (lin_q, lin_k, lin_v)]
    bs = [None if m.bias is None else m.bias.to(dt).contiguous() for m in (lin_q, lin_k, lin_v)]
    out = torch.empty(B, H, T, hout, dtype=dt, device=sx.device)
    C.check(C.LIB.one_combined_rope_attention(C.ptr(sx), C.ptr(ky), C.ptr(va), C.ptr(cos.to(dt)), C.ptr(sin.to(dt)),
                                              cos.shape[0], C.ptr(ws[0]), C.ptr(bs[0]), C.ptr(ws[1]), C.ptr(bs[1]),
                                              C.ptr(ws[2]), C.ptr(bs[2]), B, H, T, Dh, hout, C.dtype_code(dt), C.ptr(out),
                                              _stream()), "one_combined_rope_attention")
    return out


# ------------------------------------------------------------------ paged key-value cache
# k_pages, v_pages [num_pages, Hkv, page_size, Dh] (pages may lie further apart than their size:
# slices of one pool serve), block_table int32 [B, max_pages] (the pages of each sequence in order),
# lengths int32 [B] (slots in use; no call writes it), mass fp32 [B, Hkv, width >= max_pages *
# page_size] (attention weight that each slot has received). bf16 or fp32, Dh a multiple of 8, at
# most 128, any page size. Page numbers or lengths out of range are recorded (ops_error) and the
# rows that they name left alone.

def _paged(k_pages, v_pages, block_table, lengths, heads_of):
    """Checks a cache; returns its part of the C argument lists and its sizes."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must have the same shape [num_pages, Hkv, page_size, Dh]")
    if block_table.dim() != 2 or lengths.dim() != 1 or block_table.shape[0] != lengths.shape[0]:
        raise ValueError("block_table must be [B, max_pages] and lengths [B]")
    if block_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise ValueError("block_table and lengths must be int32")
    n, hkv, ps, dh = k_pages.shape
    if heads_of.dtype != k_pages.dtype or v_pages.dtype != k_pages.dtype:
        raise ValueError("the cache and the new tokens must have one dtype")
    strides = []
    for p in (k_pages, v_pages):
        s = p.stride()
        if (dh > 1 and s[3] != 1) or (ps > 1 and s[2] != dh) or (hkv > 1 and s[1] != ps * dh):
            raise ValueError("each page must be contiguous [Hkv, page_size, Dh]")
        strides.append(s[0] if n > 1 else hkv * ps * dh)
    b, mp = block_table.shape
    if (mp > 1 and block_table.stride(1) != 1) or (b > 1 and lengths.stride(0) != 1):
        raise ValueError("block_table rows and lengths must be contiguous")
    pools = (k_pages.data_ptr(), v_pages.data_ptr(), strides[0], strides[1], n, ps)
    table = (block_table.data_ptr(), block_table.stride(0) if b > 1 else mp, mp)
    return pools, table, (b, hkv, ps, dh, mp)


def _paged_mass(mass, b, hkv, slots, what="mass"):
    if mass is None:
        return 0, 0
    if mass.dim() != 3 or mass.dtype != torch.float32 or mass.shape[:2] != (b, hkv) or mass.shape[2] < slots:
        raise ValueError(f"{what} must be fp32 [{b}, {hkv}, at least {slots}]")
    if not mass.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return mass.data_ptr(), mass.shape[2]


def _launch(fn, device, *args):
    """Calls a C entry point on `device`'s current stream; every tensor must live on that device."""
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        C.check(rc, fn.__name__)


def _one_device(first, *ts):
    _need(first)
    for t in ts:
        if t is not None and t.device != first.device:
            raise ValueError(f"all tensors must be on one device, got {first.device} and {t.device}")
    return first.device


def _rows_last(t):
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def turbo_paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                       block_table: torch.Tensor, lengths: torch.Tensor, cos: Optional[torch.Tensor] = None,
                       sin: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                       counts: Optional[torch.Tensor] = None, mass: Optional[torch.Tensor] = None
                       ) -> Optional[torch.Tensor]:
    """New tokens into a paged cache. k, v [B, Hkv, N, Dh] (any strides) go to the slots lengths[b]
    .. lengths[b] + counts[b] - 1 (counts int32 [B], default N), k rotated by cos, sin [B or 1, N, Dh]
    (apply_rotary_pos_emb_flash in fp32, rounded once) when they are given; the slots' mass becomes 0.
    Returns q [B, Hq, N, Dh] rotated the same way, or None without q. The caller advances lengths."""
    pools, table, (b, hkv, ps, dh, mp) = _paged(k_pages, v_pages, block_table, lengths, k)
    if k.dim() != 4 or k.shape != v.shape or k.shape[0] != b or k.shape[1] != hkv or k.shape[3] != dh:
        raise ValueError(f"k and v must be [{b}, {hkv}, N, {dh}], got {tuple(k.shape)} and {tuple(v.shape)}")
    n = k.shape[2]
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError("the cache and the new tokens must have one dtype")
    if q is not None and (q.dim() != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (b, n, dh)):
        raise ValueError(f"q must be [{b}, Hq, {n}, {dh}], got {tuple(q.shape)}")
    if counts is not None and (counts.dtype != torch.int32 or counts.shape != (b,) or not counts.is_contiguous()):
        raise ValueError(f"counts must be int32 [{b}]")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    cb = 1
    if cos is not None:
        cb = cos.shape[0] if cos.dim() == 3 else 1
        if cos.shape[-2:] != (n, dh) or sin.shape != cos.shape or cos.dim() not in (2, 3) or cb not in (1, b):
            raise ValueError(f"cos / sin must be [B or 1, {n}, {dh}], got {tuple(cos.shape)}")
    ms = _paged_mass(mass, b, hkv, mp * ps)
    dt = C.dtype_code(k.dtype) if C else 0
    dev = _one_device(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, counts, mass)
    k, v = _rows_last(k), _rows_last(v)
    out, qa, hq = None, (0, 0, 0, 0), 0
    if q is not None:
        q = _rows_last(q)
        hq = q.shape[1]
        out = torch.empty((b, hq, n, dh), dtype=q.dtype, device=dev)
        qs = q.stride()
        qa = (q.data_ptr(), qs[0], qs[1], qs[2])
    if cos is not None:
        cos, sin = cos.to(k.dtype).contiguous(), sin.to(k.dtype).contiguous()
    kst, vst = k.stride(), v.stride()
    _launch(C.LIB.one_paged_append, dev, k.data_ptr(), kst[0], kst[1], kst[2], v.data_ptr(), vst[0], vst[1], vst[2], *qa,
            0 if cos is None else cos.data_ptr(), 0 if sin is None else sin.data_ptr(), cb,
            0 if counts is None else counts.data_ptr(), *pools, *table, lengths.data_ptr(), b, n, hq, hkv, dh, dt, *ms,
            0 if out is None else out.data_ptr())
    return out


def turbo_paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                          lengths: torch.Tensor, scale_factor: Optional[float] = None,
                          mass: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [B, Hq, 1, Dh], over the cached slots below
    lengths[b]: softmax(q k^T * scale) v with an fp32 softmax, scale 1/sqrt(Dh) by default. Hq is a
    multiple of Hkv: query head j reads kv head j // (Hq // Hkv). A sequence without slots gives
    zeros. mass grows by the softmax weights, summed over each kv head's query heads."""
    pools, table, (b, hkv, ps, dh, mp) = _paged(k_pages, v_pages, block_table, lengths, q)
    if q.dim() != 4 or q.shape[0] != b or q.shape[2] != 1 or q.shape[3] != dh or q.shape[1] % hkv:
        raise ValueError(f"q must be [{b}, a multiple of {hkv}, 1, {dh}], got {tuple(q.shape)}")
    hq = q.shape[1]
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous()):
        raise ValueError(f"out must be contiguous {tuple(q.shape)} in {q.dtype}")
    ms = _paged_mass(mass, b, hkv, mp * ps)
    dt = C.dtype_code(q.dtype) if C else 0
    dev = _one_device(q, k_pages, v_pages, block_table, lengths, mass, out)
    q = _rows_last(q)
    if out is None:
        out = torch.empty((b, hq, 1, dh), dtype=q.dtype, device=dev)
    nws = C.LIB.one_paged_attention_workspace_bytes(b, hq, hkv, dh, ps, mp, dt, mass is not None)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev)
    qs = q.stride()
    _launch(C.LIB.one_paged_attention, dev, q.data_ptr(), qs[0], qs[1], *pools, *table, lengths.data_ptr(), b, hq, hkv, dh,
            1.0 / (dh ** 0.5) if scale_factor is None else float(scale_factor), dt, *ms, out.data_ptr(), ws.data_ptr(), nws)
    return out


def turbo_paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                      dst_block_table: torch.Tensor, lengths: torch.Tensor, mass: torch.Tensor, budget: int,
                      recent: int = 0, sink: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Of each (sequence, kv head), at most `budget` slots survive: the first `sink`, the last
    `recent`, and of the rest those with the largest mass (equal ones: the lower slot; NaN counts as
    the smallest). Their keys and values are copied, in slot order, to the pages of the same pools
    that dst_block_table [B, dst pages] names, none of which block_table may use. Returns (mass_out
    [B, Hkv, dst pages * page_size]: the survivors' masses, then 0; kept int32 [B, Hkv, budget]: their
    slots, then -1). The caller goes on with dst_block_table and lengths.clamp(max=budget)."""
    pools, table, (b, hkv, ps, dh, mp) = _paged(k_pages, v_pages, block_table, lengths, k_pages)
    budget, recent, sink = int(budget), int(recent), int(sink)
    if budget < 1 or recent < 0 or sink < 0 or recent + sink > budget:
        raise ValueError("1 <= budget, 0 <= recent, 0 <= sink and recent + sink <= budget")
    d = dst_block_table
    if d.dim() != 2 or d.dtype != torch.int32 or d.shape[0] != b or (d.shape[1] > 1 and d.stride(1) != 1):
        raise ValueError(f"dst_block_table must be int32 [{b}, dst pages] with contiguous rows")
    if d.shape[1] * ps < budget:
        raise ValueError(f"dst_block_table holds {d.shape[1] * ps} slots, fewer than the budget {budget}")
    if d.data_ptr() == block_table.data_ptr():
        raise ValueError("survivors go to other pages: dst_block_table is block_table")
    if mass is None:
        raise ValueError("eviction goes by mass")
    ms = _paged_mass(mass, b, hkv, mp * ps)
    dt = C.dtype_code(k_pages.dtype) if C else 0
    dev = _one_device(k_pages, v_pages, block_table, d, lengths, mass)
    width = d.shape[1] * ps
    mass_out = torch.empty((b, hkv, width), dtype=torch.float32, device=dev)
    kept = torch.empty((b, hkv, budget), dtype=torch.int32, device=dev)
    _launch(C.LIB.one_paged_evict, dev, *pools, *table, d.data_ptr(), d.stride(0) if b > 1 else d.shape[1], d.shape[1],
            lengths.data_ptr(), *ms, b, hkv, dh, dt, budget, recent, sink, mass_out.data_ptr(), width, kept.data_ptr())
    return mass_out, kept


class TurboFlashAttention(torch.nn.Module):
    """one/turbo_ops.py:437-475: returns (output, zero attention weights)."""

    def __init__(self, causal=True, dropout=0.0):
        super().__init__()
        self.causal = causal
        self.dropout = dropout

    def forward(self, q, k, v):
        out = turbo_flash_attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=self.causal)
        return out, torch.zeros((q.size(0), q.size(1), q.size(2), k.size(2)), device=q.device, dtype=q.dtype)
