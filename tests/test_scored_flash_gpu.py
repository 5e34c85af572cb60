"""Scored attention of prompts, and of decode batches that share a prefix, against their definitions in 64 bits."""
import pytest
import torch

import scored_oracle as O
from test_scored_decode_gpu import make, slopes
from uniserve_v1_b200.ops import native as N
from uniserve_v1_b200.ops import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, I32 = torch.bfloat16, torch.int32


def cu(counts):
    return torch.tensor([0] + counts, device=DEV).cumsum(0).to(I32)


def packed(seed, new, keys, Hq, Hkv, D, gain=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (torch.randn(sum(new), Hq, D, generator=g, device=DEV) * gain).to(BF16)
    k, v = (torch.randn(sum(keys), Hkv, D, generator=g, device=DEV).to(BF16) for _ in range(2))
    return q, k, v, cu(new), cu(keys)


PROMPTS = [
    # new rows, keys, Hq, Hkv, D, cap, bias, causal, window, docs, prefix
    ([1], [1], 1, 1, 128, 0.0, False, True, 0, None, None),
    ([190], [190], 16, 4, 128, 50.0, False, True, 0, None, None),
    ([5, 128, 129, 256, 257, 1], [5, 128, 129, 256, 257, 1], 4, 2, 128, 0.0, False, True, 0, None, None),
    ([5, 300, 1], [1005, 300, 777], 4, 2, 128, 30.0, True, True, 0, None, None),
    ([700, 33], [700, 33], 4, 4, 64, 0.0, True, True, 0, None, None),
    ([700, 33], [900, 33], 4, 4, 64, 20.0, True, False, 0, None, None),
    ([700, 33], [900, 1033], 6, 2, 64, 0.0, False, False, 0, None, None),
    ([1000, 33], [1000, 500], 4, 1, 128, 0.0, False, True, 200, None, None),
    ([1000, 33], [1000, 500], 4, 1, 64, 50.0, True, True, 1, None, None),
    ([1000, 33], [1000, 500], 2, 1, 128, 0.0, False, False, 130, None, None),
    ([600, 300], [600, 400], 4, 2, 128, 0.0, False, True, 0, None, [250, 399]),
    ([600, 300], [600, 400], 4, 2, 64, 50.0, True, True, 64, None, [129, 0]),
    ([1500, 100], [1500, 300], 4, 2, 128, 50.0, False, True, 0, 173, None),
    ([1500, 100], [1500, 300], 4, 2, 64, 0.0, True, False, 0, 40, None),
    ([900], [900], 2, 2, 128, 0.0, False, True, 0, "scattered", None),
    ([900, 10], [900, 10], 2, 2, 64, 0.0, False, True, 0, 300, [200, 3]),
    ([300, 40], [100, 0], 4, 2, 128, 0.0, False, True, 0, None, None),     # rows before the first key, no keys
    ([300, 40], [100, 7], 4, 2, 64, 30.0, True, True, 0, 50, [9, 9]),
    ([0, 260, 0], [0, 260, 5], 4, 2, 128, 0.0, False, True, 0, None, None),
    ([130], [130], 3, 1, 96, 50.0, True, True, 0, None, None),
    ([130], [140], 3, 1, 40, 0.0, False, True, 0, None, None),
    ([2100], [2100], 2, 1, 128, 0.0, True, True, 0, None, None),
]


@pytest.mark.parametrize("gain", [1.0, 9.0])
@pytest.mark.parametrize("case", PROMPTS, ids=[str(i) for i in range(len(PROMPTS))])
def test_prompts(case, gain):
    new, keys, Hq, Hkv, D, cap, bias, causal, window, docs, prefix = case
    q, k, v, cu_q, cu_k = packed(11, new, keys, Hq, Hkv, D, gain)
    sl = slopes(Hq) if bias else None
    dd = None
    if docs == "scattered":
        dd = torch.randint(-3, 4, (sum(keys),), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(I32)
    elif docs:
        dd = (torch.arange(sum(keys), device=DEV) // docs).to(I32)
    pre = torch.tensor(prefix, dtype=I32, device=DEV) if prefix else None
    got = S.prompt_attention(q, k, v, cu_q, cu_k, max(new), max(keys), D ** -0.5, S.ScoreRules(cap, sl, window), causal, dd, pre)
    want, bound = O.prompt(q, k, v, cu_q, cu_k, D ** -0.5, cap, sl, causal, window, dd, pre)
    N.raise_on_device_error()
    O.check(got, want, bound)


def test_rows_past_the_last_sequence_stay_and_so_does_what_surrounds_the_output():
    q, k, v, cu_q, cu_k = packed(2, [200, 31], [200, 60], 4, 2, 64)
    more = torch.cat([q, q[:50]])
    out = torch.full((281, 4, 80), 3.0, dtype=BF16, device=DEV)
    res = S.prompt_attention(more, k, v, cu_q, cu_k, 200, 200, 0.125, out=out[:, :, 8:72])
    assert res.data_ptr() == out[:, :, 8:72].data_ptr()
    want, bound = O.prompt(q, k, v, cu_q, cu_k, 0.125)
    O.check(out[:231, :, 8:72], want, bound)
    out[:231, :, 8:72] = 3.0
    assert (out == 3.0).all()


def test_strided_inputs():
    q, k, v, cu_q, cu_k = packed(4, [150], [150], 4, 2, 64)
    want, bound = O.prompt(q, k, v, cu_q, cu_k, 0.125, cap=30.0)
    fused = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    for x in (fused, torch.cat([fused[:, :1], fused], 1)[:, 1:]):      # on 16 bytes, and not
        parts = [t.unflatten(1, (-1, 64)) for t in x.split([256, 128, 128], 1)]
        O.check(S.prompt_attention(*parts, cu_q, cu_k, 150, 150, 0.125, S.ScoreRules(cap=30.0)), want, bound)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    O.check(S.prompt_attention(*turned, cu_q, cu_k, 150, 150, 0.125, S.ScoreRules(cap=30.0)), want, bound)


def test_nothing_of_another_sequence_reaches_a_row():
    q, k, v, cu_q, cu_k = packed(6, [100, 70, 300], [100, 70, 300], 2, 1, 128)
    k[100:170] = float("nan")
    v[100:170] = float("inf")
    got = S.prompt_attention(q, k, v, cu_q, cu_k, 300, 300, 0.09)
    assert not torch.isfinite(got[100:170]).any()
    fine = [torch.cat([t[:100], t[170:]]) for t in (q, k, v)]
    want, bound = O.prompt(*fine, cu([100, 300]), cu([100, 300]), 0.09)
    O.check(torch.cat([got[:100], got[170:]]), want, bound)


def test_large_scores_under_a_cap():
    """Scores far past the cap, where tanh is flat, beside small ones."""
    q, k, v, cu_q, cu_k = packed(8, [300], [300], 2, 1, 128, gain=300.0)
    q[::3] *= 1e-3
    got = S.prompt_attention(q, k, v, cu_q, cu_k, 300, 300, 128 ** -0.5, S.ScoreRules(cap=15.0))
    want, bound = O.prompt(q, k, v, cu_q, cu_k, 128 ** -0.5, cap=15.0)
    O.check(got, want, bound)


# ---------------------------------------------------------- shared prefixes --
SHARED = [
    # rows of the groups, prefixes, rows past the last group, keys behind the prefix, Hq, Hkv, D, page, bits, cap, bias
    ([8], [2033], 0, [61, 1, 0, 16, 17, 40, 3, 9], 32, 4, 128, 16, 16, 30.0, False),
    ([3, 2], [300, 0], 1, [5, 6, 7, 100, 200, 33], 8, 2, 64, 16, 16, 0.0, True),
    ([2, 1, 4], [1, 513, 128], 0, [1, 2, 1, 700, 3, 2, 1], 16, 16, 64, 8, 16, 0.0, False),
    ([20], [700], 2, [30] * 22, 12, 4, 128, 32, 16, 50.0, True),
    ([20], [700], 0, [i % 7 for i in range(20)], 20, 2, 128, 128, 16, 0.0, False),
    ([17], [1000], 0, [1 + i % 300 for i in range(17)], 16, 1, 64, 256, 16, 0.0, False),
    ([5], [333], 0, [10] * 5, 8, 4, 128, 24, 16, 0.0, True),       # pages that no tile is made of
    ([5], [333], 0, [10] * 5, 8, 4, 64, 1, 16, 30.0, False),
    ([9, 5], [1500, 700], 0, [10 + i for i in range(14)], 32, 4, 128, 16, 8, 50.0, False),
    ([9, 5], [1500, 700], 1, [10 + i for i in range(15)], 16, 2, 64, 16, 4, 0.0, True),
    ([70], [260], 0, [1 + i % 50 for i in range(70)], 64, 4, 128, 16, 16, 0.0, False),
    ([2], [100], 0, [40, 90], 71, 1, 64, 16, 16, 0.0, False),
]


def shared_batch(case, seed=3):
    rows, prefixes, rest, behind, Hq, Hkv, D, page, bits, cap, bias = case
    pre = [p for n, p in zip(rows, prefixes) for _ in range(n)] + [0] * rest
    lens = [p + x for p, x in zip(pre, behind)]
    q, kc, vc, ks, vs, table, n = make(seed, lens, Hq, Hkv, D, page, bits, gain=3.0 if cap else 1.0)
    b = 0
    for r, p in zip(rows, prefixes):       # whole pages of the prefix are the same, a page that it ends in is copied
        for i in range(b + 1, b + r):
            table[i, :p // page] = table[b, :p // page]
            if p % page:
                here, there = int(table[b, p // page]), int(table[i, p // page])
                for cache in (kc, vc):
                    cache[there, :p % page] = cache[here, :p % page]
                if ks is not None:
                    for s in (ks, vs):
                        s[there, :, :p % page] = s[here, :, :p % page]
        b += r
    sh = S.SharedPrefix(cu(rows), torch.tensor(prefixes, dtype=I32, device=DEV), max(rows), max(prefixes))
    return q, kc, vc, ks, vs, table, n, sh, cap, slopes(Hq) if bias else None, D ** -0.5


@pytest.mark.parametrize("case", SHARED, ids=[str(i) for i in range(len(SHARED))])
def test_shared_prefixes(case):
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(case)
    rules = S.ScoreRules(cap, sl)
    got = S.decode_attention(q, kc, vc, table, n, scale, rules, k_scale=ks, v_scale=vs, shared=sh)
    N.raise_on_device_error()
    prefixes = [p for r, p in zip(case[0], case[1]) for _ in range(r)] + [0] * case[2]
    O.check(got, *O.decode(q, kc, vc, table, n, scale, cap, sl, ks=ks, vs=vs, expanded=prefixes if ks is not None else None))
    apart = S.decode_attention(q, kc, vc, table, n, scale, rules, k_scale=ks, v_scale=vs)
    O.check(apart, *O.decode(q, kc, vc, table, n, scale, cap, sl, ks=ks, vs=vs))


def test_a_prefix_longer_than_some_of_its_rows():
    """Rows whose length ends inside the prefix, an empty one among them."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([6], [500], 0, [0] * 6, 8, 2, 128, 16, 16, 0.0, True))
    n.copy_(torch.tensor([500, 499, 128, 129, 1, 0], dtype=I32, device=DEV))
    got = S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(slopes=sl), shared=sh)
    want, bound = O.decode(q, kc, vc, table, n, scale, slopes=sl)
    O.check(got, want, bound)


def test_shared_prefixes_in_a_captured_graph():
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(SHARED[0])
    work = S.decode_work(8, 32, 4, 128, DEV, sh)
    out = torch.empty_like(q)

    def call():
        S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(cap), shared=sh, work=work, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    q.copy_(q.flip(0) * 0.5)
    sh.lens.fill_(1000)                    # the pages stay: every row still holds them
    n.sub_(300)
    for _ in range(3):
        out.zero_()
        graph.replay()
    want, bound = O.decode(q, kc, vc, table, n, scale, cap)
    N.raise_on_device_error()
    O.check(out, want, bound)
