"""Cache pages of 8- or 4-bit integers: keys and values quantised as they are written, and read back.

64 channels of one token and head share a bf16 scale; with m = 127 (8 bits) or 7 (4 bits)

    s = bf16(max|x| / m)        c = round(x * (1 / s)), halves to even, in [-m, m]        x ~ c s

products and the reciprocal in FP32.  A group whose largest magnitude is under m 2^-100 holds zeros; one with an
infinity or a NaN reads back as NaN.  Layout, per plane (K and V):

* codes  uint8 [pages, page_size, kv heads, D] (two's complement), or [..., D / 2] with channel 2 i in the low four
  bits of byte i and channel 2 i + 1 in the high ones, each plus 8;
* scales bf16 [pages, kv heads, page_size, D / 64]: the rows that a key head's attention walks lie side by side.

D is a multiple of 64, the page size even.  Unlike the E4M3 pages of ``functional.kv_write_scaled`` a row never
changes once written, and a large row does not coarsen its page.  ``scored.decode_attention`` reads these pages.
CUDA: ``csrc/quant_pages.cu``; on the CPU the formulas above."""
from __future__ import annotations

import torch

from . import native as N
from .scored import current_device, device_of, launch

P, I, L = N.P, N.I, N.L
BF16, F32 = torch.bfloat16, torch.float32
GROUP = 64
N.register_signatures({
    "us_quant_write": (I, [P, P, L, L, L, L, P, I, P, P, P, P, I, I, I, I, I, I, P]),
    "us_quant_prefix": (I, [P, P, P, P, P, I, P, P, I, I, I, I, I, I, I, P, L, I, I, P, P, P, P, P, P]),
    "us_quant_gather": (I, [P, P, P, P, P, I, P, P, I, I, I, I, I, I, I, P, P, L, I, P]),
})


def quant_planes(pages: int, page_size: int, kv_heads: int, dim: int, bits: int, device):
    """(kcache, vcache, k_scale, v_scale) of an empty cache of 8- or 4-bit pages."""
    if bits not in (8, 4) or dim % GROUP or page_size % 2:
        raise ValueError(f"integer pages have 8 or 4 bits, {GROUP}-channel groups and an even page size; got {bits} bits, "
                         f"width {dim}, pages of {page_size}")
    kc, vc = (torch.zeros(pages, page_size, kv_heads, dim * bits // 8, dtype=torch.uint8, device=device) for _ in range(2))
    ks, vs = (torch.zeros(pages, kv_heads, page_size, dim // GROUP, dtype=BF16, device=device) for _ in range(2))
    return kc, vc, ks, vs


def page_bits(kcache, vcache, k_scale, v_scale) -> int:
    """Bits of the codes of an integer cache, whose planes are checked against each other."""
    if not (kcache.is_contiguous() and vcache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError("the planes of an integer cache are contiguous")
    if kcache.dtype != torch.uint8 or vcache.dtype != torch.uint8 or k_scale.dtype != BF16 or v_scale.dtype != BF16:
        raise ValueError(f"an integer cache holds uint8 codes and bfloat16 scales; got {kcache.dtype}, {k_scale.dtype}")
    codes, scales = kcache.shape, k_scale.shape
    if len(codes) != 4 or len(scales) != 4 or codes != vcache.shape or scales != v_scale.shape:
        raise ValueError("K and V planes of an integer cache have the same shape")
    pages, page, heads, width = codes
    dim = scales[3] * GROUP
    if scales[0] != pages or scales[1] != heads or scales[2] != page or (width != dim and width * 2 != dim) or page % 2 or not dim:
        raise ValueError(f"codes {tuple(codes)} and scales {tuple(scales)} are not of one integer cache")
    return 8 if width == dim else 4


# ---------------------------------------------------------------- formulas --
def quantise(x, bits: int):
    """Rows x [..., D] -> (codes as they are stored, bf16 scales [..., D / 64])."""
    m = 127.0 if bits == 8 else 7.0
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    scale = torch.where(top >= m * 2.0 ** -100, (top / m).to(BF16), torch.zeros_like(top, dtype=BF16))
    inv = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(top))
    fine = torch.isfinite(g).all(-1)
    code = torch.round(torch.where(fine[..., None], g * inv[..., None], torch.zeros_like(g)).clamp(-m, m)).flatten(-2)
    scale = torch.where(fine, scale, torch.full_like(scale, float("nan")))
    if bits == 8:
        return code.to(torch.int8).view(torch.uint8), scale
    u = (code + 8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4), scale


def dequantise(codes, scale):
    """FP32 values of codes [..., D or D / 2] under scales [..., D / 64]."""
    if codes.shape[-1] == scale.shape[-1] * GROUP:
        c = codes.view(torch.int8).float()
    else:
        c = torch.stack([(codes & 15).float(), (codes >> 4).float()], -1).flatten(-2) - 8.0
    return (c.unflatten(-1, (-1, GROUP)) * scale.float()[..., None]).flatten(-2)


# ------------------------------------------------------------- entry points --
def kv_write_quant(k, v, slots, kcache, vcache, k_scale, v_scale):
    """Rows k, v [T, Hkv, D] (bf16; any strides) into integer pages at ``slots`` [T] (int32 or int64; page *
    page_size + offset; a negative slot leaves its row out).  The slots of a call are distinct; one outside the cache
    is not written and sets the device status (on the CPU it raises)."""
    bits = page_bits(kcache, vcache, k_scale, v_scale)
    pages, page, heads, _ = kcache.shape
    T, dim = k.shape[0], k_scale.shape[3] * GROUP
    if k.shape != (T, heads, dim) or v.shape != k.shape or k.dtype != BF16 or v.dtype != BF16:
        raise ValueError(f"rows of this cache are bfloat16 [T, {heads}, {dim}]; got {tuple(k.shape)} {k.dtype}, "
                         f"{tuple(v.shape)} {v.dtype}")
    if slots.shape != (T,) or (slots.dtype != torch.int64 and slots.dtype != torch.int32):
        raise ValueError(f"one int32 or int64 slot a row; got {tuple(slots.shape)} {slots.dtype}")
    if not k.is_cuda:
        if T and int(slots.max()) >= pages * page:
            raise IndexError(f"slot {int(slots.max())} is outside a cache of {pages} pages of {page}")
        at = slots[slots >= 0].long()
        for x, cache, scale in ((k, kcache, k_scale), (v, vcache, v_scale)):
            codes, sc = quantise(x[slots >= 0], bits)
            cache[at // page, at % page] = codes
            scale[at // page, :, at % page] = sc
        return
    if device_of((k, v, slots, kcache, vcache, k_scale, v_scale)) != current_device():
        with torch.cuda.device(k.device):
            return kv_write_quant(k, v, slots, kcache, vcache, k_scale, v_scale)
    k, v, slots = _rows16(k), _rows16(v), slots.contiguous()
    a, b, _ = k.stride()
    c, d, _ = v.stride()
    launch("us_quant_write", 1, k.data_ptr(), v.data_ptr(), a, b, c, d, slots.data_ptr(), slots.dtype == torch.int64,
           kcache.data_ptr(), vcache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), T, pages, page, heads, dim, bits)


def _rows16(t):
    """``t`` [rows, heads, D] with dense channels and 16-byte steps, as it is or copied."""
    a, b, c = t.stride()
    return t if c == 1 and a % 8 == 0 and b % 8 == 0 and t.data_ptr() % 16 == 0 else t.contiguous() if t.data_ptr() % 16 == 0 or not t.is_contiguous() else t.clone()


def kv_gather_quant(kcache, vcache, k_scale, v_scale, page_table, cu, total_rows, out=None, out_cu=None):
    """Cached rows of a batch as bf16 (``functional.kv_gather`` for integer pages): sequence s brings its first
    cu[s + 1] - cu[s] positions through ``page_table`` [B, max_pages] to rows [cu[s], cu[s + 1]) of the result
    ([total_rows, Hkv, D] for K and for V), or to the rows from ``out_cu[s]`` on of a larger ``out``.  cu and out_cu
    are int32 on the device, total_rows is at least cu[B]; rows that no sequence brings are left as they were.  A page
    outside the cache is read as zeros and sets the device status, as does a row past total_rows or the end of ``out``,
    which is left out (on the CPU all three raise)."""
    bits = page_bits(kcache, vcache, k_scale, v_scale)
    pages, page, heads, _ = kcache.shape
    dim, B = k_scale.shape[3] * GROUP, page_table.shape[0]
    if page_table.dtype != torch.int32 or cu.dtype != torch.int32 or cu.numel() != B + 1 or not page_table.is_contiguous():
        raise ValueError("page_table is a contiguous int32 [B, max_pages], cu int32 [B + 1]")
    if out_cu is not None and (out is None or out_cu.dtype != torch.int32 or out_cu.numel() < B):
        raise ValueError("out_cu is int32 [B] and goes with an `out`")
    if out is None:
        ko = torch.empty(total_rows, heads, dim, dtype=BF16, device=kcache.device)
        vo = torch.empty_like(ko)
    else:
        ko, vo = out
        if any(t.dtype != BF16 or t.shape[1:] != (heads, dim) or t.stride(2) != 1 or t.stride(1) != dim or t.stride(0) % 8
               for t in out) or ko.stride(0) != vo.stride(0) or (out_cu is None and min(ko.shape[0], vo.shape[0]) < total_rows):
            raise ValueError(f"out is two bfloat16 [>= {total_rows}, {heads}, {dim}] with dense heads and one row pitch")
    if not kcache.is_cuda:
        ends, starts = cu.tolist(), (out_cu if out_cu is not None else cu).tolist()
        if ends[-1] > total_rows:
            raise IndexError(f"{ends[-1]} rows where {total_rows} were told")
        for s in range(B):
            pos = torch.arange(ends[s + 1] - ends[s])
            at = page_table[s, pos // page].long()
            if len(pos) and (int(at.min()) < 0 or int(at.max()) >= pages or starts[s] + len(pos) > ko.shape[0]):
                raise IndexError(f"sequence {s} names a page outside a cache of {pages}, or rows past the end of the output")
            for cache, scale, to in ((kcache, k_scale, ko), (vcache, v_scale, vo)):
                to[starts[s]:starts[s] + len(pos)] = dequantise(cache[at, pos % page], scale[at, :, pos % page]).to(BF16)
        return ko, vo
    if device_of((kcache, vcache, k_scale, v_scale, page_table, cu, ko, vo, out_cu)) != current_device():
        with torch.cuda.device(kcache.device):
            return kv_gather_quant(kcache, vcache, k_scale, v_scale, page_table, cu, total_rows, (ko, vo), out_cu)
    cu, out_cu = cu.contiguous(), None if out_cu is None else out_cu.contiguous()
    launch("us_quant_gather", 1, kcache.data_ptr(), vcache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
           page_table.data_ptr(), page_table.shape[1], cu.data_ptr(), None if out_cu is None else out_cu.data_ptr(), B, total_rows,
           pages, page, heads, dim, bits, ko.data_ptr(), vo.data_ptr(), ko.stride(0), min(ko.shape[0], vo.shape[0]))
    return ko, vo


def expand_prefix(kcache, vcache, k_scale, v_scale, page_table, shared, q):
    """For ``scored.decode_attention``: the shared prefixes of a batch as FP16 rows under a power of two per group and head,
    the queries likewise -> (q, k, v, factors of q's rows, exponents of k and v)."""
    bits = page_bits(kcache, vcache, k_scale, v_scale)
    pages, page, heads, _ = kcache.shape
    B, Hq, D = q.shape
    half, dev, G = torch.float16, q.device, shared.groups
    k, v = (torch.empty(G * shared.max_len, heads, D, dtype=half, device=dev) for _ in range(2))
    qh = torch.empty(B, Hq, D, dtype=half, device=dev)
    back, exps = torch.empty(B * Hq, dtype=F32, device=dev), torch.empty(G * heads, 2, dtype=torch.int32, device=dev)
    launch("us_quant_prefix", 2, kcache.data_ptr(), vcache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
           page_table.data_ptr(), page_table.shape[1], shared.cu_rows.data_ptr(), shared.lens.data_ptr(), G, shared.max_len, pages,
           page, heads, D, bits, q.data_ptr(), q.stride(0), B, Hq, k.data_ptr(), v.data_ptr(), qh.data_ptr(), back.data_ptr(),
           exps.data_ptr())
    return qh, k, v, back, exps
