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


def _table(dev, block_table, lengths, mass, hkv, ps):
    """Checks what says where a batch's slots lie: (B, max_pages, row stride of the table, address of mass, its width)."""
    tshape = block_table.shape
    if len(tshape) != 2 or lengths.shape != tshape[:1]:
        raise ValueError("block_table must be [B, max_pages] and lengths [B]")
    if block_table.dtype is not _I32 or lengths.dtype is not _I32:
        raise ValueError("block_table and lengths must be int32")
    b, mp = tshape
    ts, tc = block_table.stride()
    if (mp > 1 and tc != 1) or not lengths.is_contiguous():
        raise ValueError("block_table rows and lengths must be contiguous")
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
    if block_table.get_device() != dev or lengths.get_device() != dev:
        raise ValueError("all tensors must be on one device")
    return b, mp, ts if b > 1 else mp, mptr, mw


def _paged(k_pages, v_pages, block_table, lengths, mass, dtype):
    """Checks a cache and packs it for the C entry points: (device, packed, (B, Hkv, page_size, Dh, max_pages))."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must have the same shape [num_pages, Hkv, page_size, Dh]")
    if k_pages.dtype is not dtype or v_pages.dtype is not dtype:
        raise ValueError("the cache and the new tokens must have one dtype")
    n, hkv, ps, dh = shape
    inner = (ps * dh, dh, 1)
    ks, vs = _page_stride(k_pages, n, inner), _page_stride(v_pages, n, inner)
    dev = k_pages.get_device()
    if v_pages.get_device() != dev:
        raise ValueError("all tensors must be on one device")
    b, mp, ts, mptr, mw = _table(dev, block_table, lengths, mass, hkv, ps)
    code = _code(dtype)
    packed = C.PAGED_CACHE(k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, block_table.data_ptr(), ts, lengths.data_ptr(),
                           mptr, mw, n, ps, mp, b, hkv, dh, code) if C is not None else b""
    return dev, packed, (b, hkv, ps, dh, mp)


def _code(dtype):
    return C.dtype_code(dtype) if C is not None else 0


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


def _append(dev, cache, dims, k, v, cos, sin, q, counts, quant=None):
    """New tokens into a cache that _paged or, with the tokens' dtype code, _paged_quant has packed."""
    b, hkv, ps, dh, mp = dims
    dt = k.dtype
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
    tokens = pack(k.data_ptr(), v.data_ptr(), qptr, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], qs[0], qs[1], qs[2],
                  cosp, sinp, cptr, optr, n, hq, cb, *tables)
    if quant is None:
        _launch(C.LIB.one_paged_append, dev, cache, tokens)
    else:
        _launch(C.LIB.one_paged_quant_append, dev, cache, tokens, quant)
    return out


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
    return _append(*_paged(k_pages, v_pages, block_table, lengths, mass, k.dtype), k, v, cos, sin, q, counts)


@functools.lru_cache(maxsize=1024)
def _attention_workspace(quantised, *sizes):
    if quantised:
        return C.LIB.one_paged_quant_attention_workspace_bytes(*sizes)
    return C.LIB.one_paged_attention_workspace_bytes(*sizes)


def _attend(dev, cache, dims, q, scale_factor, mass, out, quant=None):
    """Attention over a cache that _paged or, with the dtype code of q, _paged_quant has packed."""
    b, hkv, ps, dh, mp = dims
    dt, shape = q.dtype, q.shape
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
    nws = _attention_workspace(quant is not None, b, hq, hkv, dh, ps, mp, C.dtype_code(dt), mass is not None)
    ws = q.new_empty(nws, dtype=torch.uint8) if nws else None
    qs = q.stride()
    scale = dh ** -0.5 if scale_factor is None else float(scale_factor)
    wptr = ws.data_ptr() if nws else 0
    if quant is None:
        _launch(C.LIB.one_paged_attention, dev, cache, q.data_ptr(), qs[0], qs[1], hq, scale, out.data_ptr(), wptr, nws)
    else:
        _launch(C.LIB.one_paged_quant_attention, dev, cache, q.data_ptr(), qs[0], qs[1], hq, scale, quant, out.data_ptr(), wptr,
                nws)
    return out


def turbo_paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                          lengths: torch.Tensor, scale_factor: Optional[float] = None,
                          mass: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [B, Hq, 1, Dh], over the cached slots below
    lengths[b]: softmax(q k^T * scale) v with an fp32 softmax, scale 1/sqrt(Dh) by default. Hq is a
    multiple of Hkv: query head j reads kv head j // (Hq // Hkv). A sequence without slots gives
    zeros. mass grows by the softmax weights, summed over each kv head's query heads; that takes a
    workspace of 4 bytes per query head and slot of the table. `out` must not overlap q."""
    return _attend(*_paged(k_pages, v_pages, block_table, lengths, mass, q.dtype), q, scale_factor, mass, out)


def _evict(dev, cache, dims, block_table, d, mass, budget, recent, sink, quantised=False):
    """Eviction from a cache that _paged or _paged_quant has packed, into the pages of table d."""
    b, hkv, ps, dh, mp = dims
    budget, recent, sink = int(budget), int(recent), int(sink)
    if budget < 1 or recent < 0 or sink < 0 or recent + sink > budget:
        raise ValueError("1 <= budget, 0 <= recent, 0 <= sink and recent + sink <= budget")
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
    _cuda(dev, d)
    mass_out = mass.new_empty((b, hkv, width))
    kept = d.new_empty((b, hkv, budget))
    if b == 0:
        return mass_out, kept
    _launch(C.LIB.one_paged_quant_evict if quantised else C.LIB.one_paged_evict, dev, cache, d.data_ptr(),
            d.stride(0) if b > 1 else dp, dp, budget, recent, sink, mass_out.data_ptr(), width, kept.data_ptr())
    return mass_out, kept


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
    return _evict(*_paged(k_pages, v_pages, block_table, lengths, mass, k_pages.dtype), block_table, dst_block_table, mass,
                  budget, recent, sink)


# ------------------------------------------------------------------ the same cache in 4 or 8 bits
# k_pages, v_pages uint8 [num_pages, Hkv, page_size, Dh / 2 (4 bits) or Dh (8 bits)], scales bf16
# [num_pages, Hkv, page_size, 2, ceil(Dh / 32)] (a slot's scales of the key, then of the value); Dh a
# multiple of 16, at most 128. Every 32 values of a row (the last ones may be fewer) stand for scale *
# code: scale = bf16(max |x| / m), m = 7 (4 bits) or 127 (8 bits), code = x / scale to the nearest whole
# number, halves to the even one; x is the value in fp32. Scales below 2^-100 are held as 0; a group with
# an infinity or NaN has the scale NaN and reads as NaN. A byte holds code + 128, or two codes, 8 added to
# each, the even dim in the low half. Tables, lengths and masses are those of the cache above.


def turbo_paged_quant_pools(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, bits: int = 4,
                            device="cuda") -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Pools of a quantised cache, (k_pages, v_pages, scales), not initialised."""
    if bits not in (4, 8) or head_dim < 16 or head_dim > 128 or head_dim % 16:
        raise ValueError("4 or 8 bits, and a head_dim that is a multiple of 16, at most 128")
    shape = (num_pages, num_kv_heads, page_size)
    k, v = (torch.empty(*shape, head_dim * bits // 8, dtype=torch.uint8, device=device) for _ in range(2))
    return k, v, torch.empty(*shape, 2, (head_dim + 31) // 32, dtype=torch.bfloat16, device=device)


def _paged_quant(k_pages, v_pages, scales, block_table, lengths, mass, dh):
    """As _paged for a cache in 4 or 8 bits; dh None: whatever the rows hold."""
    shape, sshape = k_pages.shape, scales.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must have the same shape [num_pages, Hkv, page_size, Dh * bits / 8]")
    if k_pages.dtype is not torch.uint8 or v_pages.dtype is not torch.uint8 or scales.dtype is not torch.bfloat16:
        raise ValueError("k_pages and v_pages must be uint8 and scales bf16")
    n, hkv, ps, row = shape
    groups = sshape[-1] if len(sshape) == 5 else 0
    if dh is None:
        dh = 2 * row if groups == (2 * row + 31) // 32 else row
    bits = 4 if dh == 2 * row else 8
    if dh != row * 8 // bits or sshape != (n, hkv, ps, 2, (dh + 31) // 32):
        raise ValueError(f"rows of {row} bytes hold head_dim {2 * row} or {row}, and scales must be [{n}, {hkv}, {ps}, 2, "
                         f"ceil(head_dim / 32)]; got head_dim {dh} and {tuple(sshape)}")
    inner = (ps * row, row, 1)
    ks, vs = _page_stride(k_pages, n, inner), _page_stride(v_pages, n, inner)
    ss = _page_stride(scales, n, (ps * 2 * groups, 2 * groups, groups, 1))
    dev = k_pages.get_device()
    if v_pages.get_device() != dev or scales.get_device() != dev:
        raise ValueError("all tensors must be on one device")
    b, mp, ts, mptr, mw = _table(dev, block_table, lengths, mass, hkv, ps)
    packed = C.PAGED_QUANT_CACHE(k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), ks, vs, ss, block_table.data_ptr(),
                                 ts, lengths.data_ptr(), mptr, mw, n, ps, mp, b, hkv, dh, bits) if C is not None else b""
    return dev, packed, (b, hkv, ps, dh, mp)


def turbo_paged_quant_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                             scales: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                             cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                             q: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                             mass: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """turbo_paged_append into a cache in 4 or 8 bits: keys, rotated when cos and sin are given, and
    values are quantised as they are written."""
    return _append(*_paged_quant(k_pages, v_pages, scales, block_table, lengths, mass, k.shape[-1]), k, v, cos, sin, q, counts,
                   quant=_code(k.dtype))


def turbo_paged_quant_read(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                           lengths: torch.Tensor, n: int, head_dim: int, starts: Optional[torch.Tensor] = None,
                           dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the cache stands for, dense: k, v [B, Hkv, n, head_dim] of the slots
    starts[b] .. starts[b] + n - 1 (starts int32 [B], default 0), scale * code rounded once to dtype (bf16
    or fp32). Slots from lengths[b] on read as zeros."""
    head_dim, n = int(head_dim), int(n)
    dev, cache, (b, hkv, ps, dh, mp) = _paged_quant(k_pages, v_pages, scales, block_table, lengths, None, head_dim)
    if n < 0:
        raise ValueError("n must not be negative")
    sptr = 0
    if starts is not None:
        if starts.dtype is not _I32 or starts.shape != (b,) or not starts.is_contiguous():
            raise ValueError(f"starts must be int32 [{b}]")
        if starts.get_device() != dev:
            raise ValueError("all tensors must be on one device")
        sptr = starts.data_ptr()
    code = _code(dtype)
    _cuda(dev, k_pages)
    k, v = (scales.new_empty((b, hkv, n, dh), dtype=dtype) for _ in range(2))
    if b and n:
        _launch(C.LIB.one_paged_quant_read, dev, cache, sptr, n, code, k.data_ptr(), v.data_ptr())
    return k, v


def turbo_paged_quant_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor,
                                block_table: torch.Tensor, lengths: torch.Tensor, scale_factor: Optional[float] = None,
                                mass: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """turbo_paged_attention over the values that a cache in 4 or 8 bits stands for; q and the result
    in bf16 or fp32."""
    return _attend(*_paged_quant(k_pages, v_pages, scales, block_table, lengths, mass, q.shape[-1]), q, scale_factor, mass, out,
                   quant=_code(q.dtype))


def turbo_paged_quant_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                            dst_block_table: torch.Tensor, lengths: torch.Tensor, mass: torch.Tensor, budget: int,
                            recent: int = 0, sink: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """turbo_paged_evict from a cache in 4 or 8 bits; codes and scales move as they are."""
    if mass is None:
        raise ValueError("eviction goes by mass")
    return _evict(*_paged_quant(k_pages, v_pages, scales, block_table, lengths, mass, None), block_table, dst_block_table, mass,
                  budget, recent, sink, quantised=True)


class TurboFlashAttention(torch.nn.Module):
    """one/turbo_ops.py:437-475: returns (output, zero attention weights)."""

    def __init__(self, causal=True, dropout=0.0):
        super().__init__()
        self.causal = causal
        self.dropout = dropout

    def forward(self, q, k, v):
        out = turbo_flash_attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=self.causal)
        return out, torch.zeros((q.size(0), q.size(1), q.size(2), k.size(2)), device=q.device, dtype=q.dtype)
