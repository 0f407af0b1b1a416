"""one.turbo_ops: the reference's turbo entry points (one/turbo_ops.py:96-475), backed by
libone_b200.so. TURBO_MODE is True when the native library loads with every entry point.

There is no CPU fallback: the turbo functions require CUDA tensors and raise otherwise.
"""
from __future__ import annotations

import ctypes
import functools
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

_I32, _F32 = torch.int32, torch.float32
_current_device = torch.cuda.current_device
# current_stream(dev).cuda_stream without the Stream object around it
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _page_stride(p, n, inner):
    """Elements from one page to the next; inner: strides of a contiguous page. Dimensions of size 1
    may have any stride."""
    s = p.stride()
    if s[1:] != inner and any(d > 1 and x != y for d, x, y in zip(p.shape[1:], s[1:], inner)):
        raise ValueError("each page must be contiguous [Hkv, page_size, Dh]")
    return s[0] if n > 1 else p.shape[1] * inner[0]


def _paged(k_pages, v_pages, block_table, lengths, mass, dtype):
    """Checks a cache and packs it for the C entry points: (device, packed, (B, Hkv, page_size, Dh, max_pages))."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must have the same shape [num_pages, Hkv, page_size, Dh]")
    tshape = block_table.shape
    if len(tshape) != 2 or lengths.shape != tshape[:1]:
        raise ValueError("block_table must be [B, max_pages] and lengths [B]")
    if block_table.dtype is not _I32 or lengths.dtype is not _I32:
        raise ValueError("block_table and lengths must be int32")
    if k_pages.dtype is not dtype or v_pages.dtype is not dtype:
        raise ValueError("the cache and the new tokens must have one dtype")
    n, hkv, ps, dh = shape
    b, mp = tshape
    inner = (ps * dh, dh, 1)
    ks, vs = _page_stride(k_pages, n, inner), _page_stride(v_pages, n, inner)
    ts, tc = block_table.stride()
    if (mp > 1 and tc != 1) or not lengths.is_contiguous():
        raise ValueError("block_table rows and lengths must be contiguous")
    dev = k_pages.get_device()
    mptr = mw = 0
    if mass is not None:
        mshape = mass.shape
        if len(mshape) != 3 or mass.dtype is not _F32 or mshape[0] != b or mshape[1] != hkv or mshape[2] < mp * ps:
            raise ValueError(f"mass must be fp32 [{b}, {hkv}, at least {mp * ps}]")
        if not mass.is_contiguous():
            raise ValueError("mass must be contiguous")
        mptr, mw = mass.data_ptr(), mshape[2]
        if mass.get_device() != dev:
            raise ValueError("all tensors must be on one device")
    if v_pages.get_device() != dev or block_table.get_device() != dev or lengths.get_device() != dev:
        raise ValueError("all tensors must be on one device")
    code = C.dtype_code(dtype) if C is not None else 0
    packed = C.PAGED_CACHE(k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, block_table.data_ptr(), ts if b > 1 else mp,
                           lengths.data_ptr(), mptr, mw, n, ps, mp, b, hkv, dh, code) if C is not None else b""
    return dev, packed, (b, hkv, ps, dh, mp)


def _cuda(dev, first):
    """Refuses tensors that are not on a GPU."""
    if dev < 0 or not TURBO_MODE:
        _need(first)


def _launch(fn, dev, *args):
    """Calls a C entry point on the current stream of device `dev`, where every tensor lives."""
    if _current_device() == dev:
        rc = fn(*args, _stream_of(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream_of(dev))
    if rc:
        C.check(rc, fn.__name__)


def _rows_last(t):
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _span(t):
    """[first, last) byte of a tensor with elements."""
    at, es = t.data_ptr(), t.element_size()
    return at, at + es * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _row_starts(t):
    at = torch.zeros(1, dtype=torch.int64)
    for n, s in zip(t.shape[:-1], t.stride()[:-1]):
        at = (at[:, None] + s * torch.arange(n)).flatten()
    return t.data_ptr() + t.element_size() * at


def _rows_overlap(x, y):
    """Whether rows (along the last dimension, each contiguous) of two tensors share memory."""
    if not x.numel() or not y.numel():
        return False
    (x0, x1), (y0, y1) = _span(x), _span(y)
    if x0 >= y1 or y0 >= x1:
        return False
    xs, ys = _row_starts(x), _row_starts(y).sort().values
    wx, wy = x.shape[-1] * x.element_size(), y.shape[-1] * y.element_size()
    i = torch.searchsorted(ys, xs - wy, right=True)  # the first row of y that ends behind the start of x's
    return bool(((i < ys.numel()) & (ys[i.clamp(max=ys.numel() - 1)] < xs + wx)).any())


def turbo_paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                       block_table: torch.Tensor, lengths: torch.Tensor, cos: Optional[torch.Tensor] = None,
                       sin: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                       counts: Optional[torch.Tensor] = None, mass: Optional[torch.Tensor] = None
                       ) -> Optional[torch.Tensor]:
    """New tokens into a paged cache. k, v [B, Hkv, N, Dh] (any strides) go to the slots lengths[b]
    .. lengths[b] + counts[b] - 1 (counts int32 [B], default N), k rotated by cos, sin [B or 1, N, Dh]
    (apply_rotary_pos_emb_flash in fp32, rounded once) when they are given; the slots' mass becomes 0.
    cos and sin are taken in k's dtype or in fp32; other types become fp32.
    Returns q [B, Hq, N, Dh] rotated the same way, or None without q. The caller advances lengths."""
    dt = k.dtype
    dev, cache, (b, hkv, ps, dh, mp) = _paged(k_pages, v_pages, block_table, lengths, mass, dt)
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or shape[0] != b or shape[1] != hkv or shape[3] != dh:
        raise ValueError(f"k and v must be [{b}, {hkv}, N, {dh}], got {tuple(k.shape)} and {tuple(v.shape)}")
    n = shape[2]
    if v.dtype is not dt or (q is not None and q.dtype is not dt):
        raise ValueError("the cache and the new tokens must have one dtype")
    hq = cptr = 0
    if q is not None:
        qshape = q.shape
        if len(qshape) != 4 or qshape[0] != b or qshape[2] != n or qshape[3] != dh:
            raise ValueError(f"q must be [{b}, Hq, {n}, {dh}], got {tuple(qshape)}")
        hq = qshape[1]
        if q.get_device() != dev:
            raise ValueError("all tensors must be on one device")
    if counts is not None:
        if counts.dtype is not _I32 or counts.shape != (b,) or not counts.is_contiguous():
            raise ValueError(f"counts must be int32 [{b}]")
        cptr = counts.data_ptr()
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    cb = 1
    if cos is not None:
        cshape = cos.shape
        cb = cshape[0] if len(cshape) == 3 else 1
        if cshape[-2:] != (n, dh) or sin.shape != cshape or len(cshape) not in (2, 3) or cb not in (1, b):
            raise ValueError(f"cos / sin must be [B or 1, {n}, {dh}], got {tuple(cshape)}")
    for t in (k, v, counts, cos, sin):
        if t is not None and t.get_device() != dev:
            raise ValueError("all tensors must be on one device")
    _cuda(dev, k)
    out, optr, qptr, qs = None, 0, 0, (0, 0, 0, 0)
    if q is not None:
        q = _rows_last(q)
        out = q.new_empty((b, hq, n, dh))
        optr, qptr, qs = out.data_ptr(), q.data_ptr(), q.stride()
    if b == 0 or n == 0:
        return out
    cosp = sinp = 0
    pack, tables = C.PAGED_TOKENS, ()
    if cos is not None:
        if cos.dtype is not dt or sin.dtype is not dt:
            cos, sin = cos.to(_F32), sin.to(_F32)
            pack, tables = C.PAGED_TOKENS_FP32_TABLES, (1,)
        if not cos.is_contiguous() or not sin.is_contiguous():
            cos, sin = cos.contiguous(), sin.contiguous()
        cosp, sinp = cos.data_ptr(), sin.data_ptr()
    k, v = _rows_last(k), _rows_last(v)
    ks, vs = k.stride(), v.stride()
    _launch(C.LIB.one_paged_append, dev, cache,
            pack(k.data_ptr(), v.data_ptr(), qptr, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], qs[0], qs[1], qs[2],
                 cosp, sinp, cptr, optr, n, hq, cb, *tables))
    return out


@functools.lru_cache(maxsize=1024)
def _attention_workspace(*sizes):
    return C.LIB.one_paged_attention_workspace_bytes(*sizes)


def turbo_paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                          lengths: torch.Tensor, scale_factor: Optional[float] = None,
                          mass: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [B, Hq, 1, Dh], over the cached slots below
    lengths[b]: softmax(q k^T * scale) v with an fp32 softmax, scale 1/sqrt(Dh) by default. Hq is a
    multiple of Hkv: query head j reads kv head j // (Hq // Hkv). A sequence without slots gives
    zeros. mass grows by the softmax weights, summed over each kv head's query heads; that takes a
    workspace of 4 bytes per query head and slot of the table. `out` must not overlap q."""
    dt = q.dtype
    dev, cache, (b, hkv, ps, dh, mp) = _paged(k_pages, v_pages, block_table, lengths, mass, dt)
    shape = q.shape
    if len(shape) != 4 or shape[0] != b or shape[2] != 1 or shape[3] != dh or shape[1] % hkv:
        raise ValueError(f"q must be [{b}, a multiple of {hkv}, 1, {dh}], got {tuple(shape)}")
    if q.get_device() != dev or (out is not None and out.get_device() != dev):
        raise ValueError("all tensors must be on one device")
    if out is not None and (out.shape != shape or out.dtype is not dt or not out.is_contiguous()):
        raise ValueError(f"out must be contiguous {tuple(shape)} in {dt}")
    q = _rows_last(q)
    if out is not None and _rows_overlap(q, out):
        raise ValueError("out must not overlap q")
    _cuda(dev, q)
    hq = shape[1]
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    if b == 0:
        return out
    nws = _attention_workspace(b, hq, hkv, dh, ps, mp, C.dtype_code(dt), mass is not None)
    ws = q.new_empty(nws, dtype=torch.uint8) if nws else None
    qs = q.stride()
    _launch(C.LIB.one_paged_attention, dev, cache, q.data_ptr(), qs[0], qs[1], hq,
            dh ** -0.5 if scale_factor is None else float(scale_factor), out.data_ptr(), ws.data_ptr() if nws else 0, nws)
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
    if mass is None:
        raise ValueError("eviction goes by mass")
    dev, cache, (b, hkv, ps, dh, mp) = _paged(k_pages, v_pages, block_table, lengths, mass, k_pages.dtype)
    budget, recent, sink = int(budget), int(recent), int(sink)
    if budget < 1 or recent < 0 or sink < 0 or recent + sink > budget:
        raise ValueError("1 <= budget, 0 <= recent, 0 <= sink and recent + sink <= budget")
    d = dst_block_table
    dshape = d.shape
    if len(dshape) != 2 or d.dtype is not _I32 or dshape[0] != b or (dshape[1] > 1 and d.stride(1) != 1):
        raise ValueError(f"dst_block_table must be int32 [{b}, dst pages] with contiguous rows")
    dp = dshape[1]
    width = dp * ps
    if width < budget:
        raise ValueError(f"dst_block_table holds {width} slots, fewer than the budget {budget}")
    if b and d.data_ptr() == block_table.data_ptr():
        raise ValueError("survivors go to other pages: dst_block_table is block_table")
    if d.get_device() != dev:
        raise ValueError("all tensors must be on one device")
    _cuda(dev, k_pages)
    mass_out = mass.new_empty((b, hkv, width))
    kept = d.new_empty((b, hkv, budget))
    if b == 0:
        return mass_out, kept
    _launch(C.LIB.one_paged_evict, dev, cache, d.data_ptr(), d.stride(0) if b > 1 else dp, dp, budget, recent, sink,
            mass_out.data_ptr(), width, kept.data_ptr())
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
