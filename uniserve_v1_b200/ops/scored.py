"""Softmax attention whose scores are capped, biased by distance or masked.

A row at position p of its sequence (the last row stands at the last key) sees key j under the score

    s = scale q . k_j        s = cap tanh(s / cap)        s -= slope_h |p - j|

where ``ScoreRules`` says so, and out_h = softmax(s) V over the keys that are visible to it, zeros where none is, or where
all of their scores are -inf.

* ``prompt_attention``: packed sequences of rows against packed keys (``attention.varlen_attention`` with rules); a
  mask by documents, by a prefix that every row sees, by a window.  On a GPU ``csrc/scored_flash_tc05.cu``.
* ``decode_attention``: one new row a sequence against cache pages, bf16 or integer (``quant_pages``); sequences may
  share a prefix that is then read once for all of them.  On a GPU ``csrc/scored_decode.cu``, the prefix in
  ``csrc/scored_flash_tc05.cu``.

On the CPU both are FP32 formulas."""
from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple, Optional

import torch

from . import native as N

P, I, L = N.P, N.I, N.L
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
N.register_signatures({
    "us_scored_decode_scratch": (L, [I]),
    "us_scored_decode": (I, [P, L, P, P, P, P, P, I, P, P, P, L, P, P, I, I, I, I, I, I, I, I, N.F, N.F, P, I, P, P, I,
                             P, P, P, P, I, I, I, P]),
    "us_scored_flash": (I, [P, L, P, L, P, L, P, L, P, P, I, I, I, I, I, I, I, I, N.F, N.F, P, I, I, P, P, P, I, I, P, P, P]),
    "us_scored_flash_parts": (I, [I, I, I, I, I]),
    "us_scored_prefix": (I, [P, L, P, L, P, L, P, P, I, I, P, I, I, I, P, P, P, I, I, I, I, I, N.F, N.F, P, P, P, I, I, I, P]),
})

MAX_SEQS = 704             # sequences of one decode launch; larger batches (and ones of huge page tables) go in slices
MAX_KEYS = 1 << 20         # keys of a prompt's sequence
MAX_CAP = 1024.0           # scores under a larger one lose what a tanh near 1, less 1, loses of FP32
_FEW_ROWS = 1 << 15        # rows times heads: more of them have tiles for over half of a GPU
# Blocks of a part of a shared prefix.  The tensor unit cuts each product at some 2^-25 of the sum it is added to: 2^20 values of
# one sign in one sum came out 0.9 % too small, 2^16 lose under 0.1 %.
_LONGEST = 512
# For the same reason prompts of more keys than this (which lose 0.4 % at most) go in parts of so many, as far as the parts have
# room in some memory.  (4,096 rows of 32 heads over 300,000 keys: 19.4 ms in one part, 17.8 so; over 4,096 keys where a max_k of
# 300,000 was told: 165 us, 255.)
_LONG_PROMPT, _LONG_ROOM = 1 << 18, 1 << 32
_TILE = 128                # rows of a tile, keys of a block of the prompt kernel


class ScoreRules(NamedTuple):
    """What happens to a score between scale q.k and the softmax."""
    cap: float = 0.0                            # > 0 (2^-20 to 1024): cap * tanh(score / cap)
    # FP32 [Hq]: - slope * |position - key|.  A negative one that a call uses sets the device status (on the CPU it raises).
    slopes: Optional[torch.Tensor] = None
    window: int = 0                             # > 0: the last `window` keys, the row's own included


@dataclass
class SharedPrefix:
    """Rows [cu_rows[g], cu_rows[g + 1]) of a decode batch share their first lens[g] keys: those are read through the
    page list of the group's first row, once for all its rows.  ``max_rows`` and ``max_len`` bound the groups' sizes
    for the host.  Rows before the first group and past the last one share nothing; rows of a group that begins before
    row 0 or has more rows than told neither, and set the device status (on the CPU the former raises).  A prefix may be longer than some of its rows, which end in it;
    a value in it that is not finite may then reach a shorter row, as one of the row's own group sees it.

    On bf16 pages a shared prefix is read once.  On integer pages it is also expanded to FP16 anew in every call, which pays
    for large groups alone: 64 rows of 32 heads behind two prefixes of 8,200 and 5,740 keys take 51 us on bf16 pages (90
    without a plan), 97 on 8-bit ones (79 without); 96 rows of 64 heads behind one of 16,000 take 96 (328) and 209 (364)."""
    cu_rows: torch.Tensor      # int32 [groups + 1]
    lens: torch.Tensor         # int32 [groups]
    max_rows: int
    max_len: int

    @property
    def groups(self) -> int:
        return self.lens.shape[0]


def device_of(tensors) -> int:
    """The one device that all of `tensors` are on (None is left out)."""
    at = None
    for t in tensors:
        if t is not None:
            i = t.get_device()
            if at is None:
                at = i
            elif i != at:
                raise ValueError("the tensors of a call are on one device")
    return at


current_device = torch._C._cuda_getDevice
_entry: dict = {}


def launch(name: str, launches: int, *args) -> None:
    """``native.call`` with device addresses as plain integers, the entry point looked up once: a decode step of one
    request waits for Python, not for its kernels."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(N.kernels(), name)
    rc = fn(*args, N.stream())
    if rc != 0:
        N.check(rc, name)
    N.launch_count += launches


def _at(t):
    return None if t is None else t.data_ptr()


def _check_rules(rules, Hq, at):
    cap, s, window = rules
    if cap and not 2.0 ** -20 <= cap <= MAX_CAP or not 0 <= window < 1 << 31:
        raise ValueError(f"a cap is 0 (none) or in [2^-20, {MAX_CAP}], a window in [0, 2^31); got {cap}, {window}")
    if s is not None and (s.dtype != F32 or s.shape != (Hq,) or not s.is_contiguous() or s.get_device() != at):
        raise ValueError(f"slopes are a contiguous float32 [{Hq}] beside the queries; got {tuple(s.shape)} {s.dtype}")
    if s is not None and at < 0 and bool((s < 0).any()):
        raise ValueError("slopes are not negative")


def _heads(q, k, v, what):
    a, b = q.shape, k.shape
    if len(a) != 3 or len(b) != 3 or v.shape != b or a[2] != b[2]:
        raise ValueError(f"{what}: q [rows, Hq, D], k and v [keys, Hkv, D]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if not b[1] or not a[1] or a[1] % b[1]:
        raise ValueError(f"{what}: {a[1]} query heads over {b[1]} key heads")


# ----------------------------------------------------------------- prompts --
def prompt_attention(q, k, v, cu_q, cu_k, max_q, max_k, scale, rules: ScoreRules = ScoreRules(), causal=True, docs=None,
                     prefix=None, out=None):
    """q [Tq, Hq, D], k / v [Tk, Hkv, D] bf16 (any strides; D a multiple of 8 up to 128), cu_q / cu_k int32 [n + 1] on the device,
    max_q / max_k at least the longest sequence's rows and keys (more of them than that set the device status, as do
    sequences that leave the tensors: what is there of them is read, and no more).  Row i of a
    sequence with nq rows and nk keys stands at position p = i + nk - nq.  A key j is visible where

        (not causal or j <= p) and (no window or j > p - window),    or j < prefix[sequence],

    and, with ``docs`` (int32 [Tk], a number for every key; a row has that of the key at its position), where both
    belong to the same document.  A row before its sequence's first key (nq > nk) has no document and sees nothing
    under ``docs``.  ``prefix``: int32 [n].  Returns bf16 [Tq, Hq, D]; rows of no sequence (past cu_q[n]) are zeros, and
    left as they were in a given ``out``.  What keys and values hold past a sequence's end never reaches it; a key or value that is not finite
    may reach any row of its own sequence that shares a block of 128 keys with one that sees it.  The tensor unit cuts
    what it adds: a sum of N values of one sign comes out up to N 2^-26 of itself small (N 2^18 at most, unless rows times
    heads have no room for parts of the keys)."""
    _heads(q, k, v, "prompt_attention")
    Tq, Hq, D = q.shape
    Tk, Hkv, _ = k.shape
    at = q.get_device()
    _check_rules(rules, Hq, at)
    n = cu_q.numel() - 1
    if n < 0 or cu_k.numel() != n + 1 or cu_q.dtype != I32 or cu_k.dtype != I32:
        raise ValueError("cu_q and cu_k are int32 [sequences + 1]")
    if docs is not None and (docs.dtype != I32 or docs.shape != (Tk,)):
        raise ValueError("docs is int32, one number a key")
    if prefix is not None and (prefix.dtype != I32 or prefix.numel() != n):
        raise ValueError("prefix is int32, one length a sequence")
    if out is not None and (out.shape != q.shape or out.dtype != BF16):
        raise ValueError("out has the shape of q, in bfloat16")
    if at < 0:
        res = _prompt_cpu(q, k, v, cu_q, cu_k, scale, rules, causal, docs, prefix)
        if out is None:
            return res
        first, end = int(cu_q[0]), int(cu_q[-1])
        out[first:end] = res[first:end]
        return out
    if q.dtype != BF16 or k.dtype != BF16 or v.dtype != BF16:
        raise ValueError(f"scored attention is served in bfloat16; got {q.dtype}, {k.dtype}, {v.dtype}")
    if D % 8 or D > 128 or max_k > MAX_KEYS:
        raise ValueError(f"scored attention serves head widths that are multiples of 8 up to 128, and sequences of up to "
                         f"{MAX_KEYS} keys; got width {D}, {max_k} keys")
    device_of((q, k, v, cu_q, cu_k, docs, prefix, out))
    if at != current_device():
        with torch.cuda.device(at):
            return prompt_attention(q, k, v, cu_q, cu_k, max_q, max_k, scale, rules, causal, docs, prefix, out)
    if D != 64 and D != 128:            # zero channels add nothing to q.k and give zero channels, cut off again
        wide = 64 if D < 64 else 128
        q, k, v = (torch.nn.functional.pad(t, (0, wide - D)) for t in (q, k, v))
        got = prompt_attention(q, k, v, cu_q, cu_k, max_q, max_k, scale, rules, causal, docs, prefix)[..., :D]
        if out is None:
            return got.contiguous()
        rows = torch.arange(Tq, device=q.device)[:, None, None]
        return out.copy_(torch.where((rows >= cu_q[0]) & (rows < cu_q[-1]), got, out))
    q, k, v = _dense_heads(q), _dense_heads(k), _dense_heads(v)
    to = out
    fill = False
    if out is None:        # rows of no sequence: the launch's, unless they may be most of the work
        fill = Tq <= n * max_q
        to = q.new_empty(Tq, Hq, D) if fill else q.new_zeros(Tq, Hq, D)
    elif not _fits(out):
        to = out.contiguous() if not out.is_contiguous() else out.clone()
    if n and Tq and max_q > 0:
        if not Tk:
            k = v = torch.zeros(1, Hkv, D, dtype=BF16, device=q.device)
            docs, Tk = None, 1
        ranges = None
        if docs is not None:
            docs = docs.contiguous()
            ranges = torch.empty(2 * (Tk // _TILE + n + 1), dtype=I32, device=q.device)
        if not (cu_q.is_contiguous() and cu_k.is_contiguous()):
            cu_q, cu_k = cu_q.contiguous(), cu_k.contiguous()
        prefix = None if prefix is None else prefix.contiguous()
        parts, po, pm = 1, None, None
        if max_k > 8 * _TILE:
            rows = n * max_q * Hq
            if rows <= _FEW_ROWS:          # few rows over many keys: the keys in parts
                parts = N.kernels().us_scored_flash_parts(n, max_q, max_k, Hq, Hkv)
            if max_k > _LONG_PROMPT and -(-max_k // _LONG_PROMPT) * rows * D * 4 <= _LONG_ROOM:
                parts = max(parts, -(-max_k // _LONG_PROMPT))
            if parts > 1:
                po = torch.empty(parts * rows * D, dtype=F32, device=q.device)
                pm = torch.empty(parts * rows * 2, dtype=F32, device=q.device)
        launch("us_scored_flash", 1 + (docs is not None) + (parts > 1), q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0),
               v.data_ptr(), v.stride(0), to.data_ptr(), to.stride(0), cu_q.data_ptr(), cu_k.data_ptr(), n, Tq, Tk, Hq, Hkv, D,
               max_q, max_k, scale, rules.cap, _at(rules.slopes), causal, rules.window, _at(docs), _at(prefix), _at(ranges), fill, parts,
               _at(po), _at(pm))
    if out is not None and to is not out:
        return out.copy_(to)
    return to


def _fits(t):
    a, b, c = t.stride()
    return c == 1 and b == t.shape[2] and a % 8 == 0 and t.data_ptr() % 16 == 0


def _dense_heads(t):
    """`t` with dense heads and rows on 16 bytes: as it is, or copied."""
    if _fits(t):
        return t
    return t.clone() if t.is_contiguous() else t.contiguous()


def _prompt_cpu(q, k, v, cu_q, cu_k, scale, rules, causal, docs, prefix):
    out = torch.zeros_like(q)
    G = q.shape[1] // k.shape[1]
    for i in range(cu_q.numel() - 1):
        q0, q1, k0, k1 = int(cu_q[i]), int(cu_q[i + 1]), int(cu_k[i]), int(cu_k[i + 1])
        nq, nk = q1 - q0, k1 - k0
        if nq <= 0 or nk <= 0:
            continue
        p, j = torch.arange(nk - nq, nk)[:, None], torch.arange(nk)[None]
        see = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            see &= j <= p
        if rules.window:
            see &= j > p - rules.window
        if prefix is not None:
            see |= j < int(prefix[i])
        if docs is not None:
            d = docs[k0:k1]
            see &= (d[p[:, 0].clamp(min=0)][:, None] == d[None]) & (p >= 0)
        qq = q[q0:q1].float().unflatten(1, (-1, G))
        s = torch.einsum("qhgd,khd->hgqk", qq, k[k0:k1].float()) * scale
        w = _softmax(s, rules, (p - j).abs(), see)
        out[q0:q1] = torch.einsum("hgqk,khd->qhgd", w, v[k0:k1].float()).flatten(1, 2).to(out.dtype)
    return out


def _softmax(s, rules, distance, see):
    """Weights of scores s [Hkv, G, rows, keys]."""
    if rules.cap:
        s = rules.cap * torch.tanh(s / rules.cap)
    if rules.slopes is not None:
        s = s - rules.slopes.view(s.shape[0], s.shape[1], 1, 1) * distance.float()
    s = s.masked_fill(~see, float("-inf"))
    if not s.numel():
        return s
    w = torch.softmax(s, -1)
    return torch.where(s.amax(-1, keepdim=True) == float("-inf"), torch.zeros_like(w), w)


# ------------------------------------------------------------- single rows --
@dataclass
class DecodeWork:
    """Workspace of ``decode_attention``: one serves every layer and step of a batch size, calls that share it being
    ordered on the device (two captured graphs that may run side by side have one each)."""
    scratch: torch.Tensor
    counters: torch.Tensor                       # zero between calls
    width: int                                   # channels of a head, at most
    prefix_o: Optional[torch.Tensor] = None      # partial results of shared prefixes
    prefix_ml: Optional[torch.Tensor] = None
    own_o: Optional[torch.Tensor] = None         # and of the rest of each row
    own_ml: Optional[torch.Tensor] = None


def _chunks(Hq, Hkv):
    return -(-(Hq // Hkv) // 16)


def _most_seqs(Hq, Hkv, keys):
    """Sequences of a decode launch over page lists of ``keys``: its list of tiles (of 32 keys) is counted in 31 bits."""
    return min(MAX_SEQS, ((1 << 31) - 1) // (Hkv * _chunks(Hq, Hkv) * (-(-keys // 32) + 1)))


def _prefix_plan(shared: SharedPrefix, Hq, Hkv, sms):
    """(tile pairs a group, parts, key blocks a part) of the prefix launch: its CTAs have 256 rows (query heads of a
    key head times sequences) and a share of the prefix's 128-key blocks, as many shares as fill the GPU once, and more where
    one would have more than _LONGEST of them."""
    per = _TILE // (Hq // Hkv)                   # sequences of a tile
    pairs = -(-shared.max_rows // (2 * per))
    blocks = max(1, -(-shared.max_len // _TILE))
    parts = max(1, -(-blocks // _LONGEST), min(sms // max(1, shared.groups * pairs * Hkv), -(-blocks // 2)))
    each = -(-blocks // parts)
    return pairs, -(-blocks // each), each


def _prefix_room(shared: SharedPrefix, Hq, Hkv, sms):
    """Rows of parts that a workspace for prefixes of up to these sizes holds: fewer or shorter groups of fewer rows may be cut
    into more parts, as many as fill the GPU."""
    pairs = _prefix_plan(shared, Hq, Hkv, sms)[0]
    blocks = max(1, -(-shared.max_len // _TILE))
    return max(sms, shared.groups * pairs * Hkv * -(-blocks // _LONGEST)) * 2 * _TILE


_sms: dict = {}


def _sm_count(i: int) -> int:
    if i not in _sms:
        _sms[i] = torch.cuda.get_device_properties(i).multi_processor_count
    return _sms[i]


def decode_work(B, Hq, Hkv, D, device, shared: Optional[SharedPrefix] = None) -> DecodeWork:
    """A workspace for batches of up to ``B`` sequences of these heads (and shared prefixes of up to these sizes)."""
    device = torch.device(device)
    with torch.cuda.device(device):
        bytes_ = N.kernels().us_scored_decode_scratch(D)
        w = DecodeWork(torch.empty(bytes_ // 4, dtype=F32, device=device),
                       torch.zeros(min(B, MAX_SEQS) * Hkv * _chunks(Hq, Hkv), dtype=I32, device=device), D)
        if shared is not None and shared.groups:
            rows = _prefix_room(shared, Hq, Hkv, _sm_count(device.index if device.index is not None else current_device()))
            w.prefix_o = torch.empty(rows * D, dtype=F32, device=device)
            w.prefix_ml = torch.empty(rows * 2, dtype=F32, device=device)
            w.own_o = torch.empty(B * Hq * D, dtype=F32, device=device)
            w.own_ml = torch.empty(B * Hq * 2, dtype=F32, device=device)
    return w


def decode_attention(q, kcache, vcache, page_table, seq_lens, scale, rules: ScoreRules = ScoreRules(), starts=None,
                     k_scale=None, v_scale=None, shared: Optional[SharedPrefix] = None, work: Optional[DecodeWork] = None,
                     out=None):
    """q [B, Hq, D] bf16, D 64 or 128; caches [pages, page_size, Hkv, D] bf16, or integer pages with their scales
    (``quant_pages``); ``page_table`` int32 [B, max_pages], ``seq_lens`` int32 [B] (the new row's key included, so
    the row stands at position length - 1; 0: the row's output is zero).  Keys from max(``starts`` (int32 [B]),
    length - window) on are visible.  ``shared``: see ``SharedPrefix``; it goes with neither ``starts`` nor a window.
    A page outside the cache is read as zeros and sets the device status, as does a length past the page table (which
    is cut there); on the CPU both raise.  Returns bf16 [B, Hq, D]."""
    B, Hq, D = q.shape
    if kcache.dim() != 4 or kcache.shape != vcache.shape:
        raise ValueError("K and V pages have the same shape [pages, page_size, Hkv, D]")
    pages, page, Hkv, width = kcache.shape
    at, bits = q.get_device(), 16
    if k_scale is not None or v_scale is not None:
        if k_scale is None or v_scale is None:
            raise ValueError("integer pages come with the scales of both planes")
        from .quant_pages import GROUP, page_bits
        bits = page_bits(kcache, vcache, k_scale, v_scale)
        width = k_scale.shape[3] * GROUP
    elif kcache.dtype != q.dtype or vcache.dtype != q.dtype:
        raise ValueError(f"queries {q.dtype} over pages {kcache.dtype}")
    if width != D or Hq % Hkv:
        raise ValueError(f"queries [.., {Hq}, {D}] over pages [.., {Hkv}, {width}]")
    _check_rules(rules, Hq, at)
    if page_table.dim() != 2 or page_table.shape[0] < B or seq_lens.numel() < B or page_table.dtype != I32 or seq_lens.dtype != I32:
        raise ValueError("page_table is int32 [B, max_pages], seq_lens int32 [B]")
    if starts is not None and (starts.dtype != I32 or starts.numel() < B):
        raise ValueError("starts is int32 [B]")
    if out is not None and (out.shape != q.shape or out.dtype != BF16):
        raise ValueError("out has the shape of q, in bfloat16")
    if shared is not None:
        if not shared.groups or shared.max_len <= 0:
            shared = None
        elif starts is not None or rules.window:
            raise ValueError("a shared prefix goes with neither starts nor a window")
        elif shared.cu_rows.dtype != I32 or shared.lens.dtype != I32 or shared.cu_rows.shape != (shared.groups + 1,) or shared.lens.dim() != 1:
            raise ValueError("a shared prefix has int32 cu_rows [groups + 1] and lens [groups]")
        elif Hq // Hkv > _TILE or B > MAX_SEQS:
            raise ValueError(f"a shared prefix is served for up to {_TILE} query heads a key head and {MAX_SEQS} sequences")
        elif not (shared.cu_rows.is_contiguous() and shared.lens.is_contiguous()):     # columns of a plan
            shared = SharedPrefix(shared.cu_rows.contiguous(), shared.lens.contiguous(), shared.max_rows, shared.max_len)
    if at < 0:
        res = _decode_cpu(q, kcache, vcache, page_table, seq_lens, scale, rules, starts, k_scale, v_scale, shared)
        return res if out is None else out.copy_(res)
    if q.dtype != BF16 or (D != 128 and D != 64):
        raise ValueError(f"scored decode attention serves bfloat16 queries of width 64 or 128; got {q.dtype}, {D}")
    if not (page_table.is_contiguous() and seq_lens.is_contiguous() and kcache.is_contiguous() and vcache.is_contiguous() and
            (starts is None or starts.is_contiguous())):
        raise ValueError("pages, page table, lengths and starts are contiguous")
    device_of((q, kcache, vcache, k_scale, v_scale, page_table, seq_lens, starts, out,
               shared and shared.cu_rows, shared and shared.lens, work and work.counters))
    if at != current_device():
        with torch.cuda.device(at):
            return decode_attention(q, kcache, vcache, page_table, seq_lens, scale, rules, starts, k_scale, v_scale, shared, work, out)
    keys = page_table.shape[1] * page
    if B > MAX_SEQS or B * Hq * (keys + 64) >= 1 << 36 and B > _most_seqs(Hq, Hkv, keys):
        most = _most_seqs(Hq, Hkv, keys)
        if not most or shared is not None:
            raise ValueError(f"{B} sequences of {Hq} heads over page lists of {page_table.shape[1]} pages of {page} are more than a launch counts")
        out = q.new_empty(B, Hq, D) if out is None else out
        for b in range(0, B, most):
            e = min(B, b + most)
            decode_attention(q[b:e], kcache, vcache, page_table[b:e], seq_lens[b:e], scale, rules,
                             None if starts is None else starts[b:e], k_scale, v_scale, None, work, out[b:e])
        return out
    q = _dense_heads(q)
    to = out
    if out is None or not (out.stride(2) == 1 and out.stride(1) == D and out.stride(0) % 2 == 0 and out.data_ptr() % 4 == 0):
        to = q.new_empty(B, Hq, D)
    if not B:
        return to if out is None else out
    if work is None:
        work = decode_work(B, Hq, Hkv, D, q.device, shared)
    elif work.counters.numel() < B * Hkv * _chunks(Hq, Hkv) or work.width < D:
        raise ValueError("the workspace is of a smaller batch, fewer heads or narrower ones")
    groups, pre = 0, _NO_PREFIX
    if shared is not None:
        pairs, parts, each = _prefix_plan(shared, Hq, Hkv, _sm_count(at))
        groups = shared.groups
        rows = groups * pairs * Hkv * parts * 2 * _TILE
        if work.prefix_o is None or work.prefix_o.numel() < rows * D or work.prefix_ml.numel() < rows * 2 or \
                work.own_o.numel() < B * Hq * D or work.own_ml.numel() < B * Hq * 2:
            raise ValueError("the workspace is of smaller shared prefixes")
        qp, k, v, back, exps, stride = q, kcache, vcache, None, None, 0
        if bits != 16:       # integer pages: the prefix is expanded once for all its readers, as FP16
            from .quant_pages import expand_prefix
            qp, k, v, back, exps = expand_prefix(kcache, vcache, k_scale, v_scale, page_table, shared, q)
            stride = shared.max_len
        elif page < 8 or (_TILE % page and page % _TILE):      # pages that no tile is made of
            from .functional import kv_gather
            stride = shared.max_len
            cu = torch.zeros(groups + 1, dtype=I32, device=q.device)
            torch.cumsum(shared.lens.clamp(0, min(stride, page_table.shape[1] * page)), 0, dtype=I32, out=cu[1:])
            k, v = (torch.empty(groups * stride, Hkv, D, dtype=BF16, device=q.device) for _ in range(2))
            first = page_table.index_select(0, shared.cu_rows[:-1].clamp(0, B - 1))
            bad = (first < 0) | (first >= pages)       # read as zeros; the prefix launch sets the status
            kv_gather(kcache, vcache, first.masked_fill(bad, 0), cu, groups * stride, out=(k, v),
                      out_cu=torch.arange(0, groups * stride, stride, dtype=I32, device=q.device))
            bad = bad.repeat_interleave(page, 1)[:, :stride, None, None]
            for t in (k, v):
                t.view(groups, stride, Hkv, D)[:, :bad.shape[1]].masked_fill_(bad, 0)
        most = min(page_table.shape[1] * page, stride or parts * each * _TILE, 1 << 30)      # keys of a prefix that are read so
        cu_rows, lens, po, pm = shared.cu_rows.data_ptr(), shared.lens.data_ptr(), work.prefix_o.data_ptr(), work.prefix_ml.data_ptr()
        launch("us_scored_prefix", 1, qp.data_ptr(), qp.stride(0), k.data_ptr(), pages, v.data_ptr(), page, _at(back), _at(exps),
               stride, most, page_table.data_ptr(), page_table.shape[1], k.shape[0], B, seq_lens.data_ptr(), cu_rows, lens, groups, Hq,
               Hkv, D, shared.max_rows, scale, rules.cap, _at(rules.slopes), po, pm, pairs, parts, each)
        pre = (cu_rows, lens, most, po, pm, work.own_o.data_ptr(), work.own_ml.data_ptr(), pairs, parts, each)
    launch("us_scored_decode", 2 if groups else 1, q.data_ptr(), q.stride(0), kcache.data_ptr(), vcache.data_ptr(), _at(k_scale),
           _at(v_scale), page_table.data_ptr(), page_table.shape[1], seq_lens.data_ptr(), _at(starts), to.data_ptr(), to.stride(0),
           work.scratch.data_ptr(), work.counters.data_ptr(), B, Hq, Hkv, D, bits, pages, page, rules.window, scale, rules.cap,
           _at(rules.slopes), groups, *pre)
    if out is not None and to is not out:
        return out.copy_(to)
    return to


_NO_PREFIX = (None, None, 0, None, None, None, None, 1, 1, 1)


def _decode_cpu(q, kcache, vcache, page_table, seq_lens, scale, rules, starts, k_scale, v_scale, shared):
    from .quant_pages import dequantise
    B, Hq, D = q.shape
    pages, page, Hkv, _ = kcache.shape
    out = torch.zeros_like(q)
    for b in range(B):
        n = int(seq_lens[b])
        if n > page_table.shape[1] * page:
            raise IndexError(f"sequence {b} has {n} keys, its page list {page_table.shape[1]} pages of {page}")
        if n <= 0:
            continue
        j = torch.arange(n)
        at = page_table[b, j // page].long()
        if shared is not None:
            g = int(torch.searchsorted(shared.cu_rows, b, right=True)) - 1
            if 0 <= g < shared.groups:
                if int(shared.cu_rows[g]) < 0:
                    raise IndexError(f"group {g} begins at row {int(shared.cu_rows[g])}")
                other = page_table[int(shared.cu_rows[g]), j // page].long()
                at = torch.where(j < int(shared.lens[g]), other, at)
        if int(at.min()) < 0 or int(at.max()) >= pages:
            raise IndexError(f"sequence {b} names a page outside a cache of {pages}")
        k, v = kcache[at, j % page], vcache[at, j % page]
        if k_scale is not None:
            k, v = dequantise(k, k_scale[at, :, j % page]), dequantise(v, v_scale[at, :, j % page])
        see = torch.ones(1, n, dtype=torch.bool)
        if starts is not None:
            see &= j >= int(starts[b])
        if rules.window:
            see &= j >= n - rules.window
        s = torch.einsum("hgd,khd->hgk", q[b].float().unflatten(0, (Hkv, -1)), k.float())[:, :, None] * scale
        w = _softmax(s, rules, (n - 1 - j)[None], see)
        out[b] = torch.einsum("hgqk,khd->qhgd", w, v.float()).reshape(Hq, D).to(out.dtype)
    return out
