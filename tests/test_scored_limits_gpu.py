"""Scored attention at the ends of what its arguments may be, against the definitions in 64 bits."""
import pytest
import torch

import scored_oracle as O
from test_scored_decode_gpu import make, slopes
from test_scored_flash_gpu import cu, packed
from uniserve_v1_b200.ops import native as N
from uniserve_v1_b200.ops import quant_pages as Q
from uniserve_v1_b200.ops import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 300, 1 << 20])
@pytest.mark.parametrize("new,keys", [([10], [5]), ([700, 300], [1500, 40]), ([3], [3])])
def test_a_window_of_all_keys_is_no_window(new, keys, window, causal):
    """Rows that stand before their sequence's first key among them."""
    q, k, v, cu_q, cu_k = packed(21, new, keys, 8, 2, 64)
    sl = slopes(8)
    got = S.prompt_attention(q, k, v, cu_q, cu_k, max(new), max(keys), 0.125, S.ScoreRules(slopes=sl, window=window), causal)
    N.raise_on_device_error()
    O.check(got, *O.prompt(q, k, v, cu_q, cu_k, 0.125, slopes=sl, causal=causal))
    assert torch.equal(got, S.prompt_attention(q, k, v, cu_q, cu_k, max(new), max(keys), 0.125, S.ScoreRules(slopes=sl), causal))


@pytest.mark.parametrize("bits", [16, 8])
def test_a_window_of_all_keys_is_no_window_for_single_rows(bits):
    q, kc, vc, ks, vs, table, n = make(22, [900, 1, 0, 37], 8, 2, 64, 16, bits)
    got = S.decode_attention(q, kc, vc, table, n, 0.125, S.ScoreRules(window=2 ** 31 - 1), k_scale=ks, v_scale=vs)
    N.raise_on_device_error()
    O.check(got, *O.decode(q, kc, vc, table, n, 0.125, ks=ks, vs=vs))


def saturated(rows, keys, Hq, Hkv, D, cap, near, slope):
    """Queries and keys whose scores are all at -cap, a slope under which keys `near` away weigh half a percent of the row's own,
    and values that make up for it: 1 near a row, 100 far from the last one."""
    u = torch.where(torch.arange(D, device=DEV) % 3 == 0, 1.0, -1.0)
    q = u.expand(rows, Hq, D).to(BF16).contiguous()
    k = (-u * (10 * cap * 8 / D)).expand(keys, Hkv, D).to(BF16).contiguous()      # scale 1 / 8: scores of -10 cap
    v = torch.ones(keys, Hkv, D, device=DEV)
    v[:max(0, keys - near)] = 100.0
    return q, k, v.to(BF16), torch.full((Hq,), slope, device=DEV)


@pytest.mark.parametrize("rows", [4000, 20])
@pytest.mark.parametrize("cap,slope,near", [(55.0, 0.004, 1300), (55.4, 0.01, 500), (50.0, 0.03, 170), (28.0, 0.004, 1300)])
def test_far_keys_under_a_cap_and_a_bias_keep_their_weight(rows, cap, slope, near):
    """All scores at the cap's lower end: the weights that stand in for a running maximum start from the smallest."""
    keys = 4000
    q, k, v, sl = saturated(rows, keys, 4, 2, 64, cap, near, slope)
    cu_q, cu_k = (torch.tensor([0, x], dtype=I32, device=DEV) for x in (rows, keys))
    assert rows > 1000 or N.kernels().us_scored_flash_parts(1, rows, keys, 4, 2) > 1
    got = S.prompt_attention(q, k, v, cu_q, cu_k, rows, keys, 0.125, S.ScoreRules(cap, sl))
    N.raise_on_device_error()
    O.check(got, *O.prompt(q, k, v, cu_q, cu_k, 0.125, cap, sl))


@pytest.mark.parametrize("cap,slope,near", [(55.0, 0.004, 1300), (55.4, 0.01, 500)])
def test_a_far_shared_prefix_under_a_cap_and_a_bias_keeps_its_weight(cap, slope, near):
    """Eight rows with `near` keys of their own behind a prefix of 3008."""
    page, prefix, rows = 16, 3008, 8
    lens = [prefix + near + i for i in range(rows)]
    q, kc, vc, _, _, table, n = make(23, lens, 4, 2, 64, page, 16)
    qs, k, v, sl = saturated(rows, prefix + 2 * near, 4, 2, 64, cap, 2 * near, slope)
    for b in range(rows):
        table[b, :prefix // page] = table[0, :prefix // page]
        pos = torch.arange(lens[b], device=DEV)
        kc[table[b, pos // page].long(), pos % page] = k[:lens[b]]
        vc[table[b, pos // page].long(), pos % page] = v[:lens[b]]
    plan = S.SharedPrefix(torch.tensor([0, rows], dtype=I32, device=DEV), torch.tensor([prefix], dtype=I32, device=DEV), rows, prefix)
    got = S.decode_attention(qs, kc, vc, table, n, 0.125, S.ScoreRules(cap, sl), shared=plan)
    N.raise_on_device_error()
    O.check(got, *O.decode(qs, kc, vc, table, n, 0.125, cap, sl))


@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("call", ["prompt", "parts", "single", "single-8", "shared"])
def test_negative_slopes_set_the_status(call, cap):
    """In every launch that reads them; zeros do not."""
    for value, bad in ((-0.25, True), (0.0, False)):
        sl = slopes(8)
        sl[5] = value
        rules = S.ScoreRules(cap, sl)
        N.raise_on_device_error()
        if call in ("prompt", "parts"):
            rows, keys = (300, 300) if call == "prompt" else (9, 5000)
            q, k, v, cu_q, cu_k = packed(24, [rows], [keys], 8, 2, 64)
            got = S.prompt_attention(q, k, v, cu_q, cu_k, rows, keys, 0.125, rules)
        else:
            q, kc, vc, ks, vs, table, n = make(25, [400, 390], 8, 2, 64, 16, 8 if call == "single-8" else 16)
            plan = None
            if call == "shared":
                table[1, :20] = table[0, :20]
                plan = S.SharedPrefix(torch.tensor([0, 2], dtype=I32, device=DEV), torch.tensor([320], dtype=I32, device=DEV), 2, 320)
            got = S.decode_attention(q, kc, vc, table, n, 0.125, rules, k_scale=ks, v_scale=vs, shared=plan)
        if bad:
            with pytest.raises(RuntimeError):
                N.raise_on_device_error()
        else:
            N.raise_on_device_error()
            assert torch.isfinite(got).all()


@pytest.mark.parametrize("D", [128, 64, 40])
@pytest.mark.parametrize("new,keys,before,behind,most", [([200, 31], [200, 60], 0, 50, 200), ([200, 31], [200, 60], 3, 160, 200),
                                                         ([5], [3000], 2, 9, 16), ([5], [3000], 0, 0, 5), ([0, 0], [7, 0], 0, 40, 64),
                                                         ([1, 2], [1, 2], 0, 3000, 2), ([3], [3], 700, 700, 3)])
def test_rows_of_no_sequence(new, keys, before, behind, most, D):
    """Zeros in an output of the call's own, whatever the memory held; as they were in a given one."""
    q, k, v, _, cu_k = packed(26, [before + sum(new) + behind], keys, 4, 2, D)
    cu_q = (torch.tensor([0] + new, device=DEV).cumsum(0) + before).to(I32)
    end = before + sum(new)
    want, bound = O.prompt(q, k, v, cu_q, cu_k, 0.125)
    for _ in range(3):
        soil = [torch.full_like(q, float("nan")) for _ in range(4)]
        del soil
        got = S.prompt_attention(q, k, v, cu_q, cu_k, most, max(keys), 0.125)
        N.raise_on_device_error()
        O.check(got, want, bound)
        assert not got[:before].any() and not got[end:].any()
    out = torch.full_like(q, 7.0)
    S.prompt_attention(q, k, v, cu_q, cu_k, most, max(keys), 0.125, out=out)
    N.raise_on_device_error()
    assert (out[:before] == 7).all() and (out[end:] == 7).all()
    O.check(out[before:end], want[before:end], bound[before:end])


def test_no_sequences_at_all():
    q, k, v, _, _ = packed(27, [20], [5], 4, 2, 64)
    none = torch.zeros(1, dtype=I32, device=DEV)
    soil = torch.full_like(q, float("nan"))
    del soil
    assert not S.prompt_attention(q, k, v, none, none, 0, 0, 0.125).any()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("power", [127, 126, -126, -130])
def test_queries_at_the_ends_of_their_range(bits, power):
    """The largest power of two of bf16 over small keys, and channels under its smallest normal number."""
    lens = [700, 33, 5]
    q, kc, vc, ks, vs, table, n = make(28, lens, 8, 2, 64, 16, bits)
    if bits == 16:
        kc.mul_(2.0 ** -12)
    else:
        ks.mul_(2.0 ** -12)
    q = (q.double().clamp(-1.99, 1.99) * 2.0 ** (power - 1)).to(BF16)
    q[:, :, 7] = 1.5 * 2.0 ** power
    scale = 0.125 * 2.0 ** (12 - power) if power > 0 else 0.125 * 2.0 ** 120
    want, bound = O.decode(q, kc, vc, table, n, scale, ks=ks, vs=vs)
    got = S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs)
    N.raise_on_device_error()
    O.check(got, want, bound)
    if bits == 16:
        return
    table[1:, 0] = table[0, 0]
    plan = S.SharedPrefix(torch.tensor([0, 3], dtype=I32, device=DEV), torch.tensor([5], dtype=I32, device=DEV), 3, 5)
    got = S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=plan)
    N.raise_on_device_error()
    O.check(got, *O.decode(q, kc, vc, table, n, scale, ks=ks, vs=vs, expanded=[5] * 3))


def test_batches_over_huge_page_tables_go_in_slices():
    """Five short sequences whose lists have room for 2^33 keys."""
    q, kc, vc, _, _, table, n = make(29, [700, 33, 0, 300, 65], 32, 4, 64, 16, 16)
    wide = torch.zeros(5, 1 << 28, dtype=I32, device=DEV)
    wide[:, :table.shape[1]] = table
    assert 0 < S._most_seqs(32, 4, (1 << 28) * 16) < 5
    got = S.decode_attention(q, kc, vc, wide, n, 0.125)
    N.raise_on_device_error()
    O.check(got, *O.decode(q, kc, vc, table, n, 0.125))
    plan = S.SharedPrefix(torch.tensor([0, 5], dtype=I32, device=DEV), torch.tensor([8], dtype=I32, device=DEV), 5, 8)
    with pytest.raises(ValueError, match="counts"):
        S.decode_attention(q, kc, vc, wide, n, 0.125, shared=plan)


@pytest.mark.parametrize("more", [0, 512])
@pytest.mark.parametrize("kind", ["plain", "documents", "window", "parts"])
def test_sequences_that_leave_the_tensors_set_the_status(kind, more):
    """The second of two ends behind the last key, or row, or begins before the first; the first one is served.
    (Told of more keys, the plain one goes in parts too.)"""
    rows, keys = ([20, 9], [4000, 3000]) if kind == "parts" else ([300, 200], [300, 700])
    q, k, v, cu_q, cu_k = packed(30, rows, keys, 4, 2, 64)
    docs = (torch.arange(sum(keys), device=DEV) // 50).to(I32) if kind == "documents" else None
    rules = S.ScoreRules(window=100 if kind == "window" else 0)
    want, bound = O.prompt(q, k, v, cu_q, cu_k, 0.125, window=rules.window, docs=docs)
    guard = torch.full((sum(rows) + 200, 4, 64), 7.0, dtype=BF16, device=DEV)
    for which, i, by in (("k", 2, 500), ("k", 2, 100_000), ("q", 2, 60), ("k", 1, -keys[0] - 400), ("q", 1, -rows[0] - 3)):
        a, b = cu_q.clone(), cu_k.clone()
        (a if which == "q" else b)[i] += by
        N.raise_on_device_error()
        guard.fill_(7.0)
        S.prompt_attention(q, k, v, a, b, max(rows), max(keys) + more, 0.125, rules, docs=docs, out=guard[:sum(rows)])
        with pytest.raises(RuntimeError):
            N.raise_on_device_error()
        assert (guard[sum(rows):] == 7).all()
        if i == 2:
            O.check(guard[:rows[0]], want[:rows[0]], bound[:rows[0]])


@pytest.mark.parametrize("rows,Hq,keys", [(600, 64, 1 << 20), (600, 64, 300_000), (9, 64, 1 << 20)])
@pytest.mark.parametrize("window", [0, 700_000])
def test_sums_of_a_million_values_of_one_sign(rows, Hq, keys, window):
    """Products of weights and values that end just under a power of two, where cutting takes most.  A key of the block that is
    walked first weighs e^9.7 times as much as each other."""
    q = torch.ones(rows, Hq, 64, dtype=BF16, device=DEV)
    k, v = torch.zeros(keys, 1, 64, dtype=BF16, device=DEV), torch.full((keys, 1, 64), 127 / 128, dtype=BF16, device=DEV)
    far = 14 * 0.6931471805599453 - 0.0077821404420549    # weights of 129 / 128 2^-14 beside it
    first = torch.full((64,), far / 8, dtype=torch.float64).to(BF16)      # scale 1 / 8, 64 channels
    first[63] = (far * 8 - float(first[:63].double().sum()))
    at = keys - rows - 1            # that every row sees
    k[at], v[at] = first.to(DEV), 0.0
    cu_q, cu_k = (torch.tensor([0, x], dtype=I32, device=DEV) for x in (rows, keys))
    got = S.prompt_attention(q, k, v, cu_q, cu_k, rows, keys, 0.125, S.ScoreRules(window=window))
    N.raise_on_device_error()
    few = [0, rows // 2, rows - 1]
    for i in few:                   # a row as the only one of its sequence: the same keys up to its own
        end = keys - rows + 1 + i
        want, bound = O.prompt(q[i:i + 1, :1], k[:end], v[:end], torch.tensor([0, 1], dtype=I32, device=DEV),
                               torch.tensor([0, end], dtype=I32, device=DEV), 0.125, window=window)
        O.check(got[i:i + 1], want.expand(1, Hq, -1), bound.expand(1, Hq, -1))


@pytest.mark.parametrize("bits,rows", [(8, 40), (4, 40), (8, 20_000)])
def test_reading_back_more_rows_than_told_sets_the_status(bits, rows):
    """Those that were told of are read."""
    planes = Q.quant_planes(rows // 8 + 2, 8, 2, 64, bits, DEV)
    x = torch.randn(rows, 2, 64, device=DEV).to(BF16)
    Q.kv_write_quant(x, x, torch.arange(rows, device=DEV), *planes)
    table = torch.arange(rows // 8 + 2, device=DEV).to(I32)[None]
    whole, _ = Q.kv_gather_quant(*planes, table, cu([rows]), rows)
    N.raise_on_device_error()
    got, _ = Q.kv_gather_quant(*planes, table, cu([rows]), rows - 3)
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()
    assert torch.equal(got, whole[:rows - 3])
