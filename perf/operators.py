"""What the speed of the scored attention and of the integer cache is measured on: softmax attention whose scores are
capped, biased by distance or masked, over prompts and over one new token a request; the same for a batch whose
requests share a long prefix; the cache in 8 or 4 bits that decode reads, as it is written and as it is read back.

Head layouts are those of the served configurations (32 query heads over 4 key heads of 128 channels, 64 over 4, 16
over 4) and of their tiny forms (64 channels, one key head for each query head); batches are those of the serving
benchmark (64 requests of 1024 tokens, chunks of 8192 rows, pages of 16).

Formulas.  A row at position p of its sequence (the last row of a sequence stands at its last key) sees key j with the
score s = scale q.k; cap > 0: s = cap tanh(s / cap); slopes: s -= slope[head] |p - j|.  Visible keys: j <= p (causal),
j > p - window, j < prefix (whatever its position), of the same document.  Out: softmax(s) V; zeros where nothing is
visible.  Integer pages: 64 channels of one token and head share a bf16 scale = bf16(max|x| / m), m = 127 or 7, and
hold round(x * (1 / scale)) in -m .. m."""
import math
import random

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
PAGE = 16
MOST_PAIRS = 32 * 8192 * 8192      # scores of a prompt case, over all heads and requests
MOST_FLOPS, MOST_BYTES = 1.6e11, 5.5e8   # about the largest listed cases


def listed():
    return [
        # a short question to a model with capped scores: every launch is in the way of the first token
        _prompt("prompt-cap-one", 16, 4, 128, 1, 190, 0, cap=50.0),
        # what a scheduler hands over when requests arrive, behind the cached history of each conversation
        _prompt("prompt-cap-batch", 32, 4, 128, 5, 5003, 2011, cap=30.0),
        # a long text under a distance bias instead of rotary positions, one key head for each query head
        _prompt("prompt-bias-long", 16, 16, 64, 1, 8191, 0, bias=True),
        # retrieved documents packed into one prompt, each of which sees itself alone
        _prompt("prompt-documents", 32, 4, 128, 1, 8192, 0, mask="documents", size=613, cap=50.0),
        # one user: the next token after a thousand
        _decode("decode-cap-one", 32, 4, 128, 1, 1021, "bf16", cap=50.0),
        # the serving benchmark's batch with grown contexts, distance bias
        _decode("decode-bias-batch", 32, 4, 128, 64, 7001, "bf16", bias=True),
        # the same batch on pages of 8 bits
        _decode("decode-int8-batch", 32, 4, 128, 64, 7001, "int8", cap=50.0),
        # few requests over long documents on pages of 4 bits
        _decode("decode-int4-long", 64, 4, 128, 16, 32001, "int4"),
        # answers sampled side by side from one question
        _shared("shared-samples", 32, 4, 128, 1, 8, 2033, 61, cap=30.0),
        # a service's system prompt and its examples in front of every request; two such services
        _shared("shared-services", 32, 4, 128, 2, 64, 8200, 509),
        # a step's new tokens into the cache, and a short history out of it
        _cache("cache-int4-step", 4, 128, 8, 1, 250, "int4"),
        # a chunk of prompts behind cached histories: written, then read back for its attention
        _cache("cache-int8-chunk", 4, 128, 8, 1021, 7001, "int8"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    hq, hkv, d = rng.choice([(32, 4, 128), (64, 4, 128), (16, 4, 128), (16, 16, 64), (8, 2, 64), (12, 4, 128)])
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    bias = rng.random() < 0.35
    op = rng.choice(["prompt", "prompt", "decode", "decode", "shared", "cache"])
    if op == "prompt":
        n = log(1, 12)
        mask = rng.choice(["causal", "causal", "window", "documents", "prefix", "all"])
        tokens = log(max(n, 33), 8192)
        context = log(16, 4000) if rng.random() < 0.3 else 0
        size = log(17, 2000)

        def drawn(part):
            return _prompt("", hq, hkv, d, n, max(n, int(tokens * part)), int(context * part), mask=mask, size=size,
                           cap=cap, bias=bias)
    elif op == "decode":
        n, longest = log(1, 192), log(1, 33000)
        kv, window = rng.choice(["bf16", "bf16", "int8", "int4"]), log(16, 4096) if rng.random() < 0.2 else 0

        def drawn(part):
            return _decode("", hq, hkv, d, n, max(1, int(longest * part)), kv, cap=cap, bias=bias, window=window)
    elif op == "shared":
        groups = rng.randint(1, 3)
        n, prefix, suffix = max(groups, log(2, 96)), log(100, 16000), log(1, 1500)
        kv = rng.choice(["bf16", "bf16", "int8"])

        def drawn(part):
            return _shared("", hq, hkv, d, groups, n, max(1, int(prefix * part)), suffix, cap=cap, bias=bias, kv=kv)
    else:
        n = log(1, 64)
        new, context, kv = log(1, max(2, 8192 // n)), log(1, 8000), rng.choice(["int8", "int4"])

        def drawn(part):
            return _cache("", hkv, d, n, new, max(1, int(context * part)), kv)
    part = 1.0
    while not _fits(drawn(part)):
        part *= 0.85
    return drawn(part)


def _fits(c):
    w = work(c)
    if w["flops"] > MOST_FLOPS or w["bytes"] > MOST_BYTES:
        return False
    if c["op"] == "prompt":     # the plain form computes the scores of all requests with all
        new, keys = _lengths(c)
        return c["heads"] * sum(new) * sum(keys) <= MOST_PAIRS
    if c["op"] == "decode":     # and a padded batch
        return c["requests"] * c["longest"] * c["kv_heads"] * c["dim"] <= 3e8
    return True


def _named(name, c):
    return {"name": name, **c} if name else c


def _prompt(name, hq, hkv, d, n, tokens, context, mask="causal", size=0, cap=0.0, bias=False):
    return _named(name, {"op": "prompt", "heads": hq, "kv_heads": hkv, "dim": d, "requests": n, "tokens": tokens,
                         "context": context, "mask": mask, "size": size, "cap": cap, "bias": bias})


def _decode(name, hq, hkv, d, n, longest, kv, cap=0.0, bias=False, window=0):
    return _named(name, {"op": "decode", "heads": hq, "kv_heads": hkv, "dim": d, "requests": n, "longest": longest,
                         "kv": kv, "cap": cap, "bias": bias, "window": window})


def _shared(name, hq, hkv, d, groups, n, prefix, suffix, cap=0.0, bias=False, kv="bf16"):
    return _named(name, {"op": "shared", "heads": hq, "kv_heads": hkv, "dim": d, "groups": groups, "requests": n,
                         "prefix": prefix, "suffix": suffix, "kv": kv, "cap": cap, "bias": bias})


def _cache(name, hkv, d, n, new, context, kv):
    return _named(name, {"op": "cache", "kv_heads": hkv, "dim": d, "requests": n, "new": new, "context": context,
                         "kv": kv})


# ------------------------------------------------------------------- sizes --
def _spread(n, longest):
    """Ragged lengths of n requests from about a seventh of the longest to it; the first is the longest."""
    r = random.Random(n * 1000003 + longest)
    return [longest] + [max(1, int(longest * r.uniform(0.15, 1.0))) for _ in range(n - 1)]


def _parts(n, total):
    """`total` cut into n ragged parts of one at least."""
    r = random.Random(n * 7919 + total)
    w = [r.uniform(0.3, 1.7) for _ in range(n)]
    got = [max(1, int(total * x / sum(w))) for x in w]
    got[0] = max(1, got[0] + total - sum(got))
    return got


def _lengths(c):
    """(new rows, keys) of every request of a prompt case."""
    new = _parts(c["requests"], c["tokens"])
    r = random.Random(c["tokens"])
    return new, [x + int(c["context"] * r.uniform(0.4, 1.0)) for x in new]


def _prefixes(c, keys):
    return [min(k, c["size"]) for k in keys]


def _groups(c):
    """(rows, prefix length) of every group, and the length of every request, of a shared case."""
    rows = _parts(c["groups"], c["requests"])
    lens = [max(1, int(c["prefix"] * (1.0 - 0.3 * g))) for g in range(c["groups"])]
    own_keys = _spread(c["requests"], c["suffix"])
    total, at = [], 0
    for n, p in zip(rows, lens):
        total += [p + x for x in own_keys[at:at + n]]
        at += n
    return rows, lens, total


# ------------------------------------------------------------------ inputs --
def _cumulative(counts):
    got = [0]
    for x in counts:
        got.append(got[-1] + x)
    return torch.tensor(got, dtype=torch.int32, device="cuda")


def _normal(gen, shape, gain=1.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=F32)
    return (x * gain).to(BF16)


def _slopes(c):
    """The geometric slopes of a distance bias, one a head."""
    if not c["bias"]:
        return None
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / c["heads"]) for h in range(c["heads"])], device="cuda")


def _pages(gen, c, count):
    """Pages as they are after long use: random rows; integer pages with the scales of rows of unit gain."""
    hkv, d = c["kv_heads"], c["dim"]
    if c["kv"] == "bf16":
        k, v = (torch.randn(count, PAGE, hkv, d, generator=gen, device="cuda", dtype=BF16) for _ in range(2))
        return k, v, None, None
    wide = d if c["kv"] == "int8" else d // 2
    k, v = (torch.randint(0, 256, (count, PAGE, hkv, wide), generator=gen, device="cuda", dtype=torch.uint8)
            for _ in range(2))
    unit = 1.0 / 74.0 if c["kv"] == "int8" else 1.0 / 4.6
    ks, vs = ((torch.rand(count, hkv, PAGE, d // 64, generator=gen, device="cuda") * 0.6 + 0.7).mul(unit).to(BF16)
              for _ in range(2))
    return k, v, ks, vs


def _table(gen, lens, width=None):
    """Page lists of sequences over a pool of which they hold every page, in no order."""
    need = [-(-x // PAGE) for x in lens]
    width = width or max(need)
    order = torch.randperm(sum(need) + 3, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c, "op": c["op"]}
    if c["op"] == "cache":
        lens = _spread(c["requests"], c["context"])
        total = [x + c["new"] for x in lens]
        table, count = _table(gen, total)
        s["kc"], s["vc"], s["ks"], s["vs"] = _pages(gen, c, count)
        rows = c["new"] * c["requests"]
        s["k"], s["v"] = (_normal(gen, (rows, c["kv_heads"], c["dim"])) for _ in range(2))
        at = torch.tensor(lens, device="cuda")[:, None] + torch.arange(c["new"], device="cuda")[None]
        s["slots"] = (torch.gather(table.long(), 1, at // PAGE) * PAGE + at % PAGE).reshape(-1)
        s["table"], s["cu"], s["total"], s["lens"] = table, _cumulative(total), sum(total), total
        return s
    s["scale"] = c["dim"] ** -0.5
    s["slopes"] = _slopes(c)
    gain = 4.0 if c["cap"] else 1.0      # models that cap their scores have large ones
    if c["op"] == "prompt":
        new, keys = _lengths(c)
        s["q"] = _normal(gen, (sum(new), c["heads"], c["dim"]), gain)
        s["k"], s["v"] = (_normal(gen, (sum(keys), c["kv_heads"], c["dim"])) for _ in range(2))
        s["cu_q"], s["cu_k"], s["max_q"], s["max_k"] = _cumulative(new), _cumulative(keys), max(new), max(keys)
        s["docs"] = s["prefix"] = None
        if c["mask"] == "documents":
            s["docs"] = (torch.arange(sum(keys), device="cuda") // c["size"]).to(torch.int32)
        if c["mask"] == "prefix":
            s["prefix"] = torch.tensor(_prefixes(c, keys), dtype=torch.int32, device="cuda")
        s["window"] = c["size"] if c["mask"] == "window" else 0
        s["causal"] = c["mask"] != "all"
        return s
    if c["op"] == "decode":
        lens = _spread(c["requests"], c["longest"])
        table, count = _table(gen, lens)
        s["window"] = c["window"]
    else:
        rows, shared, lens = _groups(c)
        s["window"] = 0
        # the pages below a group's prefix are the same ones for all its rows; what follows is each row's own
        table, count = _table(gen, lens)
        at = 0
        for n, p in zip(rows, shared):
            table[at:at + n, :p // PAGE] = table[at, :p // PAGE].clone()
            if p % PAGE:
                s.setdefault("copies", []).append((at, n, p))
            at += n
        s["cu_rows"], s["shared"] = _cumulative(rows), torch.tensor(shared, dtype=torch.int32, device="cuda")
        s["max_rows"], s["max_shared"] = max(rows), max(shared)
    s["kc"], s["vc"], s["ks"], s["vs"] = _pages(gen, c, count)
    for at, n, p in s.pop("copies", []):   # a prefix that ends inside a page: every row has its own copy of that page
        pages, off = table[at:at + n, p // PAGE].long(), p % PAGE
        for cache in (s["kc"], s["vc"]):
            cache[pages, :off] = cache[pages[0], :off].clone()
        for scale in (s["ks"], s["vs"]):
            if scale is not None:
                scale[pages, :, :off] = scale[pages[0], :, :off].clone()
    s["q"] = _normal(gen, (len(lens), c["heads"], c["dim"]), gain)
    s["table"], s["longest"] = table, max(lens)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------- plain forms --
def _bits(state):
    return 8 if state["case"]["kv"] == "int8" else 4


def _codes(cache, bits):
    """Integers that the bytes of a cache stand for, FP32."""
    if bits == 8:
        return cache.view(torch.int8).float()
    low, high = (cache & 15).float() - 8.0, (cache >> 4).float() - 8.0
    return torch.stack([low, high], -1).flatten(-2)


def _rows_of(cache, scale, table, bits):
    """Cached rows of a padded batch, FP32 [requests, keys, kv heads, channels]."""
    got = cache[table.long()]
    if scale is not None:
        sc = scale[table.long()].float().transpose(2, 3).repeat_interleave(64, -1)
        got = _codes(got, bits) * sc
    return got.float().flatten(1, 2)


def _weights(scores, state, distance, visible):
    """softmax of capped and biased scores [heads..., rows, keys] over what is visible; rows without a key: zeros."""
    cap = state["case"]["cap"]
    if cap:
        scores = cap * torch.tanh(scores / cap)
    if state["slopes"] is not None:
        scores = scores - distance
    scores = scores.masked_fill(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(scores - top)
    return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_prompt(s):
    c = s["case"]
    hq, hkv, d = c["heads"], c["kv_heads"], c["dim"]
    g = hq // hkv
    tq, tk = s["q"].shape[0], s["k"].shape[0]
    rows, keys = torch.arange(tq, device="cuda"), torch.arange(tk, device="cuda")
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    seq_q = torch.searchsorted(cu_q, rows, right=True) - 1
    seq_k = torch.searchsorted(cu_k, keys, right=True) - 1
    pos_k = keys - cu_k[seq_k]
    pos_q = rows - cu_q[seq_q + 1] + (cu_k[seq_q + 1] - cu_k[seq_q])
    away = pos_q[:, None] - pos_k[None]
    visible = torch.ones(tq, tk, dtype=torch.bool, device="cuda")
    if s["causal"]:
        visible &= away >= 0
    if s["window"]:
        visible &= away < s["window"]
    if s["prefix"] is not None:
        visible |= pos_k[None] < s["prefix"].long()[seq_q][:, None]
    visible &= seq_q[:, None] == seq_k[None]
    if s["docs"] is not None:
        visible &= s["docs"][cu_k[seq_q] + pos_q][:, None] == s["docs"][None]
    distance = None
    if s["slopes"] is not None:
        distance = s["slopes"].view(hkv, g, 1, 1) * away.abs().float()
    q = s["q"].float().view(tq, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * tq, d)
    scores = torch.matmul(q, s["k"].float().permute(1, 2, 0)).view(hkv, g, tq, tk) * s["scale"]
    w = _weights(scores, s, distance, visible)
    del scores
    out = torch.matmul(w.view(hkv, g * tq, tk), s["v"].float().transpose(0, 1))
    return out.view(hkv, g, tq, d).permute(2, 0, 1, 3).reshape(tq, hq, d).to(BF16)


def _plain_decode(s):
    c = s["case"]
    hq, hkv, d = c["heads"], c["kv_heads"], c["dim"]
    b = s["q"].shape[0]
    bits = 0 if s["ks"] is None else _bits(s)
    k, v = (_rows_of(x, y, s["table"], bits) for x, y in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
    pos = torch.arange(k.shape[1], device="cuda")
    away = s["lens"].long()[:, None] - 1 - pos[None]
    visible = away >= 0
    if s["window"]:
        visible &= away < s["window"]
    distance = None
    if s["slopes"] is not None:
        distance = s["slopes"].view(1, hkv, hq // hkv, 1) * away.float()[:, None, None]
    q = s["q"].float().view(b, hkv, hq // hkv, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]
    w = _weights(scores, s, distance, visible[:, None, None])
    return torch.matmul(w, v.transpose(1, 2)).reshape(b, hq, d).to(BF16)


def _plain_quantise(x, bits):
    """(bytes, bf16 scales [rows, heads, channels / 64]) of rows."""
    m = 127.0 if bits == 8 else 7.0
    n, h, d = x.shape
    x = x.float().view(n, h, d // 64, 64)
    scale = (x.abs().amax(-1) / m).to(BF16)
    inv = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(scale, dtype=F32))
    code = torch.round(x * inv[..., None]).clamp(-m, m).view(n, h, d)
    if bits == 8:
        return code.to(torch.int8).view(torch.uint8), scale
    u = (code + 8.0).to(torch.uint8).view(n, h, d // 2, 2)
    return u[..., 0] | (u[..., 1] << 4), scale


def _plain_cache(s):
    bits = _bits(s)
    page, off = s["slots"] // PAGE, s["slots"] % PAGE
    got = []
    for x, cache, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        code, sc = _plain_quantise(x, bits)
        cache[page, off] = code
        scale[page, :, off] = sc
        rows = torch.arange(s["total"], device="cuda")
        seq = torch.searchsorted(s["cu"].long(), rows, right=True) - 1
        pos = rows - s["cu"].long()[seq]
        p = s["table"].long()[seq, pos // PAGE]
        value = _codes(cache[p, pos % PAGE], bits) * scale[p, :, pos % PAGE].float().repeat_interleave(64, -1)
        got.append(value.to(BF16))
    return {"k": got[0], "v": got[1], "k_scale": s["ks"], "v_scale": s["vs"]}


def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "prompt":
        return _plain_prompt(s)
    return _plain_cache(s) if s["op"] == "cache" else _plain_decode(s)


def _own(s):
    from uniserve_v1_b200.ops import quant_pages as Q
    from uniserve_v1_b200.ops import scored as S
    if s["op"] == "cache":
        Q.kv_write_quant(s["k"], s["v"], s["slots"], s["kc"], s["vc"], s["ks"], s["vs"])
        k, v = Q.kv_gather_quant(s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["cu"], s["total"])
        return {"k": k, "v": v, "k_scale": s["ks"], "v_scale": s["vs"]}
    rules = S.ScoreRules(cap=s["case"]["cap"], slopes=s["slopes"], window=s["window"])
    if s["op"] == "prompt":
        return S.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["max_q"], s["max_k"], s["scale"],
                                  rules, causal=s["causal"], docs=s["docs"], prefix=s["prefix"])
    shared = None
    if s["op"] == "shared":
        shared = S.SharedPrefix(s["cu_rows"], s["shared"], s["max_rows"], s["max_shared"])
    if "work" not in s:      # a server keeps the workspace of its batch size from step to step
        hkv = s["case"]["kv_heads"]
        s["work"] = S.decode_work(s["q"].shape[0], s["q"].shape[1], hkv, s["q"].shape[2], "cuda", shared)
    return S.decode_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["scale"], rules, k_scale=s["ks"],
                              v_scale=s["vs"], shared=shared, work=s["work"])


# -------------------------------------------------------------------- work --
def _visible_pairs(c):
    new, keys = _lengths(c)
    pairs = at = 0
    for i, (n, k) in enumerate(zip(new, keys)):
        p = torch.arange(k - n, k, dtype=torch.int64)
        first, last = torch.zeros_like(p), p
        if c["mask"] == "all":
            last = torch.full_like(p, k - 1)
        if c["mask"] == "window":
            first = (p - c["size"] + 1).clamp(min=0)
        if c["mask"] == "documents":
            first = ((at + p) // c["size"] * c["size"] - at).clamp(min=0)
        if c["mask"] == "prefix":
            last = p.clamp(min=min(k, c["size"]) - 1)
        pairs += int((last - first + 1).sum())
        at += k
    return pairs


def _row_bytes(c):
    """Bytes of one token's K and V of all key heads."""
    d = c["dim"]
    one = {"bf16": 2 * d, "int8": d + d // 32, "int4": d // 2 + d // 32}[c["kv"]]
    return 2 * c["kv_heads"] * one


def work(case):
    c = case
    if c["op"] == "cache":
        total = sum(_spread(c["requests"], c["context"])) + c["new"] * c["requests"]
        new = c["new"] * c["requests"]
        plain = 4 * c["kv_heads"] * c["dim"]
        return {"bytes": new * (plain + _row_bytes(c) + 8) + total * (plain + _row_bytes(c)) + total / PAGE * 4,
                "flops": 4 * (new + total) * c["kv_heads"] * c["dim"]}
    if c["op"] == "prompt":
        new, keys = _lengths(c)
        return {"bytes": 2 * c["dim"] * (2 * sum(new) * c["heads"] + 2 * sum(keys) * c["kv_heads"]),
                "flops": 4 * c["dim"] * c["heads"] * _visible_pairs(c)}
    if c["op"] == "decode":
        lens = _spread(c["requests"], c["longest"])
        seen = [min(x, c["window"]) if c["window"] else x for x in lens]
        read, pairs = sum(seen), sum(seen)
    else:
        rows, shared, lens = _groups(c)
        pairs = sum(lens)
        read = pairs - sum((n - 1) * p for n, p in zip(rows, shared))
    return {"bytes": read * _row_bytes(c) + 4 * len(lens) * c["heads"] * c["dim"] + read / PAGE * 4,
            "flops": 4 * c["dim"] * c["heads"] * pairs}


# ------------------------------------------------------------ in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "decode": _exact_decode, "shared": _exact_decode, "cache": _exact_cache}[case["op"]](s)


def _attend(q, k, v, s, head, p, visible):
    """One query head of one sequence: q [rows, D], k and v [keys, D] in 64 bits; p: the rows' positions."""
    z = (q @ k.T) * s["scale"]
    cap = s["case"]["cap"]
    if cap:
        z = torch.tanh(z / cap) * cap
    if s["slopes"] is not None:
        away = (p[:, None] - torch.arange(k.shape[0], device="cuda")[None]).abs()
        z = z - s["slopes"][head].double() * away
    z = torch.where(visible, z, torch.full_like(z, -math.inf))
    m = z.max(1, keepdim=True).values
    e = torch.where(visible, torch.exp(z - torch.where(m > -math.inf, m, torch.zeros_like(m))), torch.zeros_like(z))
    n = e.sum(1, keepdim=True)
    return torch.where(n > 0, (e @ v) / torch.where(n > 0, n, torch.ones_like(n)), torch.zeros_like(n))


def _exact_prompt(s):
    c = s["case"]
    new, keys = _lengths(c)
    out = torch.zeros(sum(new), c["heads"], c["dim"], dtype=F64, device="cuda")
    share = c["heads"] // c["kv_heads"]
    rq = rk = 0
    for i, (n, t) in enumerate(zip(new, keys)):
        p = torch.arange(t - n, t, device="cuda")
        j = torch.arange(t, device="cuda")
        see = (j[None] <= p[:, None]) if s["causal"] else torch.ones(n, t, dtype=torch.bool, device="cuda")
        if s["window"]:
            see = see & (j[None] > p[:, None] - s["window"])
        if s["prefix"] is not None:
            see = see | (j[None] < min(t, c["size"]))
        if s["docs"] is not None:
            d = s["docs"][rk:rk + t]
            see = see & (d[p][:, None] == d[None])
        for h in range(c["heads"]):
            k, v = s["k"][rk:rk + t, h // share].double(), s["v"][rk:rk + t, h // share].double()
            out[rq:rq + n, h] = _attend(s["q"][rq:rq + n, h].double(), k, v, s, h, p, see)
        rq, rk = rq + n, rk + t
    return out


def _exact_rows(cache, scale, pages, count, kv):
    """The first `count` rows of a page list in 64 bits: [count, kv heads, channels]."""
    got = cache[pages]
    if kv == "bf16":
        return got.double().reshape(-1, *got.shape[2:])[:count]
    if kv == "int8":
        code = got.to(torch.int64)
        code = code - 256 * (code > 127)
    else:
        wide = got.to(torch.int64)
        code = torch.empty(*got.shape[:-1], 2 * got.shape[-1], dtype=torch.int64, device="cuda")
        code[..., 0::2], code[..., 1::2] = wide % 16 - 8, wide // 16 - 8
    n, page, heads, d = code.shape
    sc = scale[pages].double().permute(0, 2, 1, 3)
    return (code.double().view(n, page, heads, d // 64, 64) * sc[..., None]).reshape(n * page, heads, d)[:count]


def _exact_decode(s):
    c = s["case"]
    share = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // PAGE)].long()
        k, v = (_exact_rows(x, y, pages, n, c["kv"]) for x, y in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        at = torch.tensor([n - 1], device="cuda")
        see = torch.arange(n, device="cuda")[None] > n - 1 - (s["window"] or n)
        for h in range(c["heads"]):
            out[b, h] = _attend(s["q"][b, h].double()[None], k[:, h // share], v[:, h // share], s, h, at, see)[0]
    return out


def _exact_cache(s):
    """The definition on the new rows; the context is read as it stands."""
    c = s["case"]
    m = 127 if c["kv"] == "int8" else 7
    result = {}
    for name, x, cache, scale in (("k", s["k"], s["kc"], s["ks"]), ("v", s["v"], s["vc"], s["vs"])):
        parts = torch.split(x.double(), 64, dim=-1)
        steps = [(p.abs().amax(-1) / m).float().to(BF16) for p in parts]
        whole = [torch.where(t[..., None] > 0, (p / t[..., None].double()).round().clamp(-m, m), torch.zeros_like(p))
                 for p, t in zip(parts, steps)]
        value = torch.cat([w * t[..., None].double() for w, t in zip(whole, steps)], -1)
        rows, at = [], 0
        for b, n in enumerate(s["lens"]):
            old = _exact_rows(cache, scale, s["table"][b, :-(-n // PAGE)].long(), n - c["new"], c["kv"])
            rows += [old, value[at:at + c["new"]]]
            at += c["new"]
        result[name] = torch.cat(rows)
        step = scale.double().clone()
        step[s["slots"] // PAGE, :, s["slots"] % PAGE] = torch.stack(steps, -1).double()
        result[name + "_scale"] = step
    return result
