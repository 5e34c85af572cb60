"""Scored attention and integer pages from their definitions in 64 bits, and how far a kernel with bf16 weights and
results may be from them."""
import torch

F64 = torch.float64
HALF_STEP = torch.finfo(torch.bfloat16).eps / 2


def attend(q, k, v, scale, cap, slopes, p, see, steps=None):
    """q [rows, Hq, D], k / v [keys, Hkv, D], p [rows] positions, see [rows, keys] -> (out, bound), both [rows, Hq, D].

    bound: a weight is rounded to bf16 once (HALF_STEP of it, so HALF_STEP sum w |v| of the result), the result once
    (HALF_STEP of it).  A score errs by its FP32 sum (D + 8 roundings of sum |q k| scale), by the cap's function (2^-16
    of the cap, the kernels' own bound) and by its FP32 size; an error e of all scores changes a normalised weight by 2 e.

    steps: (K's, V's) sizes [keys, Hkv, D] of the offset under which integer codes are multiplied (the step of a code times
    1152 for 8 bits, 72 for 4).  A score is then the sum of D / 16 + 1 products whose running sum is at most sum |q| step,
    each off by at most 2^-22 of it (the tensor unit keeps FP32 sums and cuts off what is below): (D / 16 + 1) 2^-22
    sum |q| step.  A result has, in each tile, four products and one correction of at most sum w step, so 5 x 2^-22 of
    sum w step over all tiles."""
    q, k, v = q.double(), k.double(), v.double()
    share = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    s = torch.einsum("qhd,khd->hqk", q, k) * scale
    err = float((torch.einsum("qhd,khd->hqk", q.abs(), k.abs()) * abs(scale))[:, see].max()) * (q.shape[2] + 8) * 2.0 ** -24 \
        if see.any() else 0.0
    if steps is not None:
        ko, vo = (t.double().repeat_interleave(share, 1) for t in steps)
        if see.any():
            err += float((torch.einsum("qhd,khd->hqk", q.abs(), ko) * abs(scale))[:, see].max()) * (q.shape[2] / 16 + 1) * 2.0 ** -22
    if cap:
        s = cap * torch.tanh(s / cap)
        err += cap * 2.0 ** -16
    if slopes is not None:
        j = torch.arange(k.shape[0], device=q.device)
        s = s - slopes.double()[:, None, None] * (p[:, None] - j[None]).abs()
    s = s.masked_fill(~see, float("-inf"))
    some = see.any(1)
    if some.any():
        err += float(s[:, see].abs().max()) * 2.0 ** -19
    w = torch.where(some[None, :, None], torch.softmax(s, -1), torch.zeros_like(s))
    w = torch.where(see[None], w, torch.zeros_like(w))
    v = torch.where(see.any(0)[:, None, None], v, torch.zeros_like(v))   # what nobody sees weighs nothing
    out = torch.einsum("hqk,khd->qhd", w, v)
    mass = torch.einsum("hqk,khd->qhd", w, v.abs())
    bound = mass * (HALF_STEP + 2 * err + 2.0 ** -20) + out.abs() * HALF_STEP + 1e-30
    if steps is not None:
        bound += torch.einsum("hqk,khd->qhd", w, vo) * 5 * 2.0 ** -22
    return out, bound


def unpack(code, scale):
    """Values of codes [..., D or D / 2] (bytes) under bf16 scales [..., D / 64], in 64 bits."""
    d = scale.shape[-1] * 64
    wide = code.to(torch.int64)
    if code.shape[-1] == d:
        c = wide - 256 * (wide > 127)
    else:
        c = torch.empty(*code.shape[:-1], d, dtype=torch.int64, device=code.device)
        c[..., 0::2], c[..., 1::2] = wide % 16 - 8, wide // 16 - 8
    return (c.double().reshape(*scale.shape, 64) * scale.double()[..., None]).reshape(*scale.shape[:-1], d)


def cached(kc, ks, pages, count):
    """The first `count` rows behind a page list, in 64 bits."""
    if ks is None:
        rows = kc[pages].double()
    else:
        rows = unpack(kc[pages], ks[pages].transpose(1, 2))
    return rows.reshape(-1, *rows.shape[2:])[:count]


def decode(q, kc, vc, table, lens, scale, cap=0.0, slopes=None, window=0, starts=None, ks=None, vs=None, expanded=None):
    """Row by row -> (out, bound) [B, Hq, D].  The first `expanded[b]` keys and values of a row (a shared prefix of integer
    pages) are the cache's rounded to FP16 under a power of two (2^e to 2^(e + 1) holds the prefix's largest scale of the
    head, so products of codes are in reach): its definition of those values."""
    outs, bounds = [], []
    page = kc.shape[1]
    for b, n in enumerate(lens.tolist()):
        if n <= 0:
            outs.append(torch.zeros(q.shape[1:], dtype=F64, device=q.device))
            bounds.append(torch.full(q.shape[1:], 1e-30, dtype=F64, device=q.device))
            continue
        pages = table[b, :-(-n // page)].long()
        k, v = cached(kc, ks, pages, n), cached(vc, vs, pages, n)
        j = torch.arange(n, device=q.device)
        if expanded is not None and expanded[b]:
            m, at = min(expanded[b], n), table[b, :-(-expanded[b] // page)].long()
            kv = []
            for t, sc in ((k, ks), (v, vs)):
                top = sc[at].transpose(1, 2).flatten(0, 1)[:expanded[b]].double().amax((0, 2))
                down = torch.exp2(torch.floor(torch.log2(top)))[None, :, None]
                kv.append(torch.cat([(t[:m] / down).half().double() * down, t[m:]]))
            k, v = kv
        lo = max(n - window if window else 0, int(starts[b]) if starts is not None else 0)
        # keys that are not visible weigh nothing whatever they hold
        k, v = (torch.where((j >= lo)[:, None, None], t, torch.zeros_like(t)) for t in (k, v))
        steps = None
        if ks is not None:
            offset = 1152.0 if kc.shape[3] == q.shape[2] else 72.0
            steps = tuple(torch.where((j >= lo)[:, None, None], t, torch.zeros_like(t)) for t in (
                offset * sc[pages].transpose(1, 2).double().flatten(0, 1)[:n].repeat_interleave(64, -1) for sc in (ks, vs)))
        o, e = attend(q[b:b + 1], k, v, scale, cap, slopes, torch.tensor([n - 1], device=q.device), (j >= lo)[None], steps)
        outs.append(o[0])
        bounds.append(e[0])
    return torch.stack(outs), torch.stack(bounds)


def prompt(q, k, v, cu_q, cu_k, scale, cap=0.0, slopes=None, causal=True, window=0, docs=None, prefix=None):
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    bound = torch.full(q.shape, 1e-30, dtype=F64, device=q.device)
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for i in range(len(cq) - 1):
        nq, nk = cq[i + 1] - cq[i], ck[i + 1] - ck[i]
        if nq <= 0 or nk <= 0:
            continue
        p = torch.arange(nk - nq, nk, device=q.device)
        j = torch.arange(nk, device=q.device)
        see = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            see &= j[None] <= p[:, None]
        if window:
            see &= j[None] > p[:, None] - window
        if prefix is not None:
            see |= j[None] < int(prefix[i])
        if docs is not None:
            d = docs[ck[i]:ck[i + 1]]
            see &= (d[p.clamp(min=0)][:, None] == d[None]) & (p >= 0)[:, None]
        o, e = attend(q[cq[i]:cq[i + 1]], k[ck[i]:ck[i + 1]], v[ck[i]:ck[i + 1]], scale, cap, slopes, p, see)
        out[cq[i]:cq[i + 1]], bound[cq[i]:cq[i + 1]] = o, e
    return out, bound


def check(got, want, bound, what=""):
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite at {torch.nonzero(~torch.isfinite(got))[:4].tolist()}"
    over = (got.double() - want).abs() - bound
    worst = float(over.max()) if over.numel() else 0.0
    if worst > 0:
        i = int(over.argmax())
        raise AssertionError(f"{what}: over its bound by {worst:.3g} at {i} of {tuple(got.shape)} "
                             f"(got {float(got.flatten()[i]):.6g}, want {float(want.flatten()[i]):.6g}, bound {float(bound.flatten()[i]):.3g})")
