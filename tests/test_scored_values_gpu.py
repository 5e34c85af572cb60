"""Scored attention over values that are not numbers: what they reach is not a number either, however the keys were split,
and they reach nothing else."""
import pytest
import torch

import scored_oracle as O
from test_scored_decode_gpu import make, slopes
from test_scored_flash_gpu import cu, packed, shared_batch
from uniserve_v1_b200.ops import native as N
from uniserve_v1_b200.ops import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, I32 = torch.bfloat16, torch.int32
NAN = float("nan")


def check_but(got, want, bound, lost):
    """`lost` [rows, heads]: rows that are NaN in every channel; the others are within their bounds."""
    assert got[lost].isnan().all(), f"finite where it cannot be: {torch.nonzero(~got[lost].isnan())[:4].tolist()}"
    O.check(got[~lost], want[~lost], bound[~lost])


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (64, 4, 64)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_a_query_that_is_not_a_number_over_many_keys(bits, Hq, Hkv, D, cap):
    """Its pair is spread over many warps and CTAs."""
    q, kc, vc, ks, vs, table, n = make(31, [9000, 33, 4000], Hq, Hkv, D, 16, bits)
    sl = slopes(Hq)
    want, bound = O.decode(q, kc, vc, table, n, 0.1, cap, sl, ks=ks, vs=vs)
    lost = torch.zeros(3, Hq, dtype=torch.bool, device=DEV)
    lost[0, 1] = lost[1, Hq - 1] = lost[2, 0] = True
    q[lost] = NAN
    got = S.decode_attention(q, kc, vc, table, n, 0.1, S.ScoreRules(cap, sl), k_scale=ks, v_scale=vs)
    N.raise_on_device_error()
    check_but(got, want, bound, lost)


@pytest.mark.parametrize("length", [33, 65, 129, 4097])
@pytest.mark.parametrize("D,bits", [(128, 16), (64, 16), (128, 8), (64, 8), (128, 4)])
def test_the_newest_key_is_not_a_number(length, D, bits):
    """It is alone in its tile, and that tile may be a warp's whole range."""
    q, kc, vc, ks, vs, table, n = make(32, [length, 20], 8, 2, D, 16, bits)
    want, bound = O.decode(q, kc, vc, table, n, 0.1, ks=ks, vs=vs)
    page, at = table[0, (length - 1) // 16].long(), (length - 1) % 16
    if bits == 16:
        kc[page, at, 1] = NAN
    else:
        ks[page, 1, at] = NAN
    got = S.decode_attention(q, kc, vc, table, n, 0.1, k_scale=ks, v_scale=vs)
    N.raise_on_device_error()
    lost = torch.zeros(2, 8, dtype=torch.bool, device=DEV)
    lost[0, 4:] = True
    check_but(got, want, bound, lost)


@pytest.mark.parametrize("cap", [0.0, 30.0, 100.0])
def test_prompts_whose_keys_go_in_parts(cap):
    q, k, v, cu_q, cu_k = packed(33, [37, 3], [6000, 3000], 8, 2, 128)
    assert N.kernels().us_scored_flash_parts(2, 37, 6000, 8, 2) > 1
    want, bound = O.prompt(q, k, v, cu_q, cu_k, 0.1, cap)
    lost = torch.zeros(40, 8, dtype=torch.bool, device=DEV)
    lost[0, 3] = lost[36, 0] = lost[39, 7] = True
    q[lost] = NAN
    got = S.prompt_attention(q, k, v, cu_q, cu_k, 37, 6000, 0.1, S.ScoreRules(cap))
    N.raise_on_device_error()
    check_but(got, want, bound, lost)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_shared_prefixes(bits, cap):
    case = ([5, 3], [1500, 700], 1, [40, 1, 0, 200, 17, 5, 9, 1000, 3], 8, 2, 64, 16, bits, cap, False)
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(case)
    want, bound = O.decode(q, kc, vc, table, n, scale, cap, ks=ks, vs=vs, expanded=[1500] * 5 + [700] * 3 + [0] if ks is not None else None)
    lost = torch.zeros(9, 8, dtype=torch.bool, device=DEV)
    lost[1, 2] = lost[2, 5] = lost[8, 0] = True          # one without keys of its own, one that shares nothing
    q[lost] = NAN
    got = S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(cap), k_scale=ks, v_scale=vs, shared=sh)
    N.raise_on_device_error()
    check_but(got, want, bound, lost)


@pytest.mark.parametrize("D,Hq,Hkv,bias,cap", [(128, 4, 2, False, 0.0), (64, 4, 2, False, 0.0), (128, 2, 2, True, 0.0), (64, 2, 1, True, 0.0),
                                               (128, 4, 2, False, 30.0), (64, 2, 1, True, 100.0)])
def test_a_key_that_is_not_a_number_in_every_place_of_a_block(D, Hq, Hkv, bias, cap):
    """256 sequences of 383 to 385 keys, each with one such key: in any place of a block that all rows of a tile see, and that
    comes after the first one.  The rows that see it are NaN, and those before its block are what they were."""
    n = 256
    keys = [383 + i % 3 for i in range(n)]
    q, k, v, cu_q, cu_k = packed(34, keys, keys, Hq, Hkv, D)
    sl = slopes(Hq) if bias else None
    want, bound = O.prompt(q, k, v, cu_q, cu_k, 0.1, cap, sl)
    p = torch.cat([torch.arange(x, device=DEV) for x in keys])
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(keys, device=DEV))
    at = torch.arange(n, device=DEV)                     # the key of sequence s: key s, of its first or second block
    k[cu_k[:-1].long() + at] = NAN
    got = S.prompt_attention(q, k, v, cu_q, cu_k, 385, 385, 0.1, S.ScoreRules(cap, sl))
    N.raise_on_device_error()
    sees, before = p >= at[seq], p < at[seq] // 128 * 128
    assert got[sees].isnan().all(), f"finite where it cannot be: {torch.nonzero(sees & ~got.isnan().flatten(1).all(1))[:4].tolist()}"
    O.check(got[before], want[before], bound[before])


def lose(n, Hq, D, row, heads, group):
    """Outputs that a value of `row`, key head and 64-channel group that is not a number reaches."""
    lost = torch.zeros(n, Hq, D, dtype=torch.bool, device=DEV)
    lost[row, heads, 64 * group:64 * group + 64] = True
    return lost


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("group", [0, 1])
@pytest.mark.parametrize("where", [0, 700, 2999])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (32, 2)])
def test_a_value_that_is_not_a_number_loses_its_own_channels(bits, group, where, Hq, Hkv):
    """The 64 channels that share its scale, and none of the other 64."""
    q, kc, vc, ks, vs, table, n = make(35, [3000, 40], Hq, Hkv, 128, 16, bits)
    want, bound = O.decode(q, kc, vc, table, n, 0.1, ks=ks, vs=vs)
    vs[table[0, where // 16].long(), 1, where % 16, group] = NAN
    got = S.decode_attention(q, kc, vc, table, n, 0.1, k_scale=ks, v_scale=vs)
    N.raise_on_device_error()
    lost = lose(2, Hq, 128, 0, slice(Hq // 2, Hq), group)
    assert torch.equal(got.isnan(), lost)
    O.check(got[~lost], want[~lost], bound[~lost])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("group", [0, 1])
def test_a_value_of_a_shared_prefix_that_is_not_a_number(bits, group):
    case = ([5], [1500], 1, [40, 1, 0, 200, 17, 300], 8, 2, 128, 16, bits, 0.0, False)
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(case)
    want, bound = O.decode(q, kc, vc, table, n, scale, ks=ks, vs=vs, expanded=[1500] * 5 + [0])
    vs[table[0, 30].long(), 1, 3, group] = NAN
    got = S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=sh)
    N.raise_on_device_error()
    lost = lose(6, 8, 128, slice(0, 5), slice(4, 8), group)
    assert torch.equal(got.isnan(), lost)
    O.check(got[~lost], want[~lost], bound[~lost])


@pytest.mark.parametrize("bits", [8, 4])
def test_a_key_of_a_shared_prefix_that_is_not_a_number(bits):
    """Its key head's rows are lost, those of the other one are what they were."""
    case = ([5], [1500], 1, [40, 1, 0, 200, 17, 300], 8, 2, 128, 16, bits, 0.0, False)
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(case)
    want, bound = O.decode(q, kc, vc, table, n, scale, ks=ks, vs=vs, expanded=[1500] * 5 + [0])
    ks[table[0, 30].long(), 1, 3, 0] = NAN
    got = S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=sh)
    N.raise_on_device_error()
    lost = torch.zeros(6, 8, dtype=torch.bool, device=DEV)
    lost[:5, 4:] = True
    check_but(got, want, bound, lost)


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("bits,length", [(16, 20), (16, 5000)])
def test_scores_of_minus_infinity_weigh_nothing(bits, length, cap):
    """A row of them is zeros, as on the CPU; under a cap they are the cap's lower end."""
    q, kc, vc, _, _, table, n = make(36, [length, 70], 8, 2, 64, 16, bits)
    pos = torch.arange(length, device=DEV)
    kc[table[0, pos // 16].long(), pos % 16, :, 0] = 1.0
    q[:, :, 0] = 0.5
    plain, bound = O.decode(q, kc, vc, table, n, 0.1, cap)
    q[0, 3, 0] = float("-inf")
    got = S.decode_attention(q, kc, vc, table, n, 0.1, S.ScoreRules(cap))
    N.raise_on_device_error()
    rest = torch.ones(2, 8, dtype=torch.bool, device=DEV)
    rest[0, 3] = False
    O.check(got[rest], plain[rest], bound[rest])
    if cap:
        mean = vc[table[0, pos // 16].long(), pos % 16, 0].double().mean(0)
        assert (got[0, 3].double() - mean).abs().max() < 2.0 ** -7 * float(vc[table[0, pos // 16].long(), pos % 16, 0].double().abs().mean(0).max())
    else:
        assert not got[0, 3].any()
