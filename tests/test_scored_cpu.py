"""Scored attention and integer pages on the CPU: the formulas against their definitions in 64 bits, and what is refused."""
import pytest
import torch

import scored_oracle as O
from uniserve_v1_b200.ops import quant_pages as Q
from uniserve_v1_b200.ops import scored as S

BF16, I32 = torch.bfloat16, torch.int32


def cu(counts):
    return torch.tensor([0] + counts).cumsum(0).to(I32)


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(BF16)


SLOPES = torch.tensor([0.5, 0.25, 0.125, 0.0625])


@pytest.mark.parametrize("cap,bias,causal,window,docs,prefix", [
    (0.0, False, True, 0, None, None), (5.0, True, True, 0, None, [3, 40]), (5.0, False, False, 9, None, None),
    (0.0, True, True, 0, 7, None), (0.0, False, False, 0, 11, [5, 60])])
def test_prompts(cap, bias, causal, window, docs, prefix):
    new, keys = [20, 5], [33, 5]
    q, k, v = rnd(25, 4, 16), rnd(38, 2, 16, seed=1), rnd(38, 2, 16, seed=2)
    dd = (torch.arange(38) // docs).to(I32) if docs else None
    pre = torch.tensor(prefix, dtype=I32) if prefix else None
    sl = SLOPES if bias else None
    got = S.prompt_attention(q, k, v, cu(new), cu(keys), 20, 33, 0.25, S.ScoreRules(cap, sl, window), causal, dd, pre)
    O.check(got, *O.prompt(q, k, v, cu(new), cu(keys), 0.25, cap, sl, causal, window, dd, pre))


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_single_rows_and_a_shared_prefix(bits):
    page, Hkv, D, pages = 4, 2, 64, 24
    lens = torch.tensor([0, 9, 17, 13], dtype=I32)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(3))[:20].view(4, 5).to(I32)
    table[2:, :2] = table[1, :2]
    q, k, v = rnd(4, 4, D), rnd(pages * page, Hkv, D, seed=1), rnd(pages * page, Hkv, D, seed=2)
    ks = vs = None
    if bits == 16:
        kc, vc = k.view(pages, page, Hkv, D), v.view(pages, page, Hkv, D)
    else:
        kc, vc, ks, vs = Q.quant_planes(pages, page, Hkv, D, bits, "cpu")
        Q.kv_write_quant(k, v, torch.arange(pages * page), kc, vc, ks, vs)
    rules = S.ScoreRules(cap=3.0, slopes=SLOPES)
    want, bound = O.decode(q, kc, vc, table, lens, 0.125, 3.0, SLOPES, ks=ks, vs=vs)
    O.check(S.decode_attention(q, kc, vc, table, lens, 0.125, rules, k_scale=ks, v_scale=vs), want, bound)
    shared = S.SharedPrefix(torch.tensor([1, 4], dtype=I32), torch.tensor([8], dtype=I32), 3, 8)
    table[2:, :2] = 0                       # what the others' lists hold below the prefix is not read
    O.check(S.decode_attention(q, kc, vc, table, lens, 0.125, rules, k_scale=ks, v_scale=vs, shared=shared)[1:], want[1:], bound[1:])
    starts = torch.tensor([0, 3, 17, 12], dtype=I32)
    table[2:, :2] = table[1, :2]
    O.check(S.decode_attention(q, kc, vc, table, lens, 0.125, S.ScoreRules(window=11), starts=starts, k_scale=ks, v_scale=vs),
            *O.decode(q, kc, vc, table, lens, 0.125, window=11, starts=starts, ks=ks, vs=vs))


@pytest.mark.parametrize("bits,most", [(8, 127), (4, 7)])
def test_quantised_rows(bits, most):
    x = rnd(50, 3, 128) * 3
    x[0, 0, :64] = 0
    x[1, 0, :64] = 1e-38
    x[2, 1, 5] = float("inf")
    x[3, 1, 70] = float("nan")
    codes, scale = Q.quantise(x, bits)
    assert codes.shape == (50, 3, 128 * bits // 8) and codes.dtype == torch.uint8 and scale.shape == (50, 3, 2)
    back = Q.dequantise(codes, scale)
    assert torch.equal(back.double().nan_to_num(), O.unpack(codes, scale).nan_to_num())
    fine = torch.isfinite(x.unflatten(-1, (2, 64))).all(-1)
    assert torch.equal(scale.isnan(), ~fine)
    g, b = x.double().unflatten(-1, (2, 64))[fine], back.double().unflatten(-1, (2, 64))[fine]
    step = scale.double()[fine][:, None]
    # half a step off; where the scale was rounded down the largest magnitude is up to most * 2^-8 of a step past the last code
    assert ((g - b).abs() <= step * (0.5 + most * O.HALF_STEP) + 1e-37).all()
    assert (O.unpack(codes, torch.ones_like(scale)).abs() <= most).all()
    assert not back[0, 0, :64].any() and not back[1, 0, :64].any()


def test_rows_are_written_to_their_slots_and_read_back():
    planes = Q.quant_planes(6, 4, 2, 64, 8, "cpu")
    k, v = rnd(5, 2, 64), rnd(5, 2, 64, seed=1)
    Q.kv_write_quant(k, v, torch.tensor([9, -1, 8, 23, 0], dtype=I32), *planes)
    table = torch.tensor([[2, 0], [5, 2]], dtype=I32)
    ko, vo = Q.kv_gather_quant(*planes, table, cu([5, 4]), 9)
    assert torch.equal(ko[0], Q.dequantise(*Q.quantise(k[2], 8)).to(BF16))
    assert torch.equal(ko[1], Q.dequantise(*Q.quantise(k[0], 8)).to(BF16))
    assert torch.equal(vo[4], Q.dequantise(*Q.quantise(v[4], 8)).to(BF16))
    assert torch.equal(ko[8], Q.dequantise(*Q.quantise(k[3], 8)).to(BF16))
    assert not ko[5:8].any()
    out = (torch.full((12, 2, 64), 9.0, dtype=BF16), torch.full((12, 2, 64), 9.0, dtype=BF16))
    Q.kv_gather_quant(*planes, table, cu([5, 4]), 9, out=out, out_cu=torch.tensor([7, 1], dtype=I32))
    assert torch.equal(out[0][7:], ko[:5]) and torch.equal(out[1][1:5], vo[5:]) and (out[0][5:7] == 9).all() and (out[0][0] == 9).all()


# --------------------------------------------------------------- refusals --
def prompt_args(**kw):
    a = dict(q=rnd(4, 4, 16), k=rnd(4, 2, 16), v=rnd(4, 2, 16), cu_q=cu([4]), cu_k=cu([4]), max_q=4, max_k=4, scale=1.0)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(k=rnd(4, 3, 16), v=rnd(4, 3, 16)), dict(v=rnd(3, 2, 16)), dict(k=rnd(4, 2, 8), v=rnd(4, 2, 8)), dict(q=rnd(4, 64)),
    dict(cu_k=cu([2, 2])), dict(cu_q=cu([4]).long()), dict(docs=torch.zeros(3, dtype=I32)), dict(docs=torch.zeros(4)),
    dict(prefix=torch.zeros(2, dtype=I32)), dict(prefix=torch.zeros(1)), dict(rules=S.ScoreRules(cap=-1.0)),
    dict(rules=S.ScoreRules(cap=float("nan"))), dict(rules=S.ScoreRules(cap=float("inf"))), dict(rules=S.ScoreRules(window=-1)),
    dict(rules=S.ScoreRules(slopes=torch.zeros(2))), dict(rules=S.ScoreRules(slopes=torch.zeros(4, dtype=BF16))),
    dict(out=torch.zeros(4, 4, 16)), dict(out=rnd(3, 4, 16))])
def test_prompts_refused(kw):
    with pytest.raises(ValueError):
        S.prompt_attention(**prompt_args(**kw))


def decode_args(bits=16, **kw):
    a = dict(q=rnd(2, 4, 64), kcache=rnd(3, 4, 2, 64), vcache=rnd(3, 4, 2, 64), page_table=torch.zeros(2, 2, dtype=I32),
             seq_lens=torch.ones(2, dtype=I32), scale=1.0)
    if bits != 16:
        a.update(zip(("kcache", "vcache", "k_scale", "v_scale"), Q.quant_planes(3, 4, 2, 64, bits, "cpu")))
    a.update(kw)
    return a


SHARE = S.SharedPrefix(cu([2]), torch.tensor([2], dtype=I32), 2, 2)


@pytest.mark.parametrize("kw", [
    dict(kcache=rnd(3, 4, 2, 32), vcache=rnd(3, 4, 2, 32)), dict(vcache=rnd(2, 4, 2, 64)), dict(kcache=rnd(3, 4, 3, 64), vcache=rnd(3, 4, 3, 64)),
    dict(page_table=torch.zeros(1, 2, dtype=I32)), dict(page_table=torch.zeros(2, 2)), dict(seq_lens=torch.ones(1, dtype=I32)),
    dict(seq_lens=torch.ones(2)), dict(starts=torch.zeros(2)), dict(out=rnd(2, 4, 32)), dict(rules=S.ScoreRules(window=-2)),
    dict(k_scale=torch.ones(3, 2, 4, 1, dtype=BF16)), dict(shared=SHARE, starts=torch.zeros(2, dtype=I32)),
    dict(shared=SHARE, rules=S.ScoreRules(window=3)), dict(shared=S.SharedPrefix(cu([2]).long(), torch.tensor([2], dtype=I32), 2, 2)),
    dict(bits=8, q=rnd(2, 4, 128)), dict(bits=8, k_scale=torch.ones(3, 2, 4, 1)), dict(bits=4, kcache=torch.zeros(3, 4, 2, 48, dtype=torch.uint8)),
    dict(bits=8, v_scale=None), dict(bits=8, kcache=torch.zeros(3, 4, 2, 64, dtype=torch.int8))])
def test_single_rows_refused(kw):
    with pytest.raises(ValueError):
        S.decode_attention(**decode_args(**kw))


def test_bad_pages_and_lengths_raise():
    with pytest.raises(IndexError):
        S.decode_attention(**decode_args(page_table=torch.full((2, 2), 3, dtype=I32)))
    with pytest.raises(IndexError):
        S.decode_attention(**decode_args(page_table=torch.full((2, 2), -1, dtype=I32)))
    with pytest.raises(IndexError):
        S.decode_attention(**decode_args(seq_lens=torch.tensor([1, 9], dtype=I32)))


def test_the_cache_refuses():
    for bad in ((3, 4, 2, 64, 6), (3, 4, 2, 96, 8), (3, 5, 2, 64, 8)):
        with pytest.raises(ValueError):
            Q.quant_planes(*bad, "cpu")
    planes = Q.quant_planes(3, 4, 2, 64, 8, "cpu")
    x, slots = rnd(2, 2, 64), torch.tensor([0, 1])
    for args in ((x.float(), x, slots), (x, rnd(1, 2, 64), slots), (rnd(2, 3, 64), rnd(2, 3, 64), slots), (x, x, slots[:1]),
                 (x, x, slots.to(torch.int16))):
        with pytest.raises(ValueError):
            Q.kv_write_quant(*args, *planes)
    with pytest.raises(IndexError):
        Q.kv_write_quant(x, x, torch.tensor([0, 12]), *planes)
    table = torch.zeros(1, 2, dtype=I32)
    for kw in (dict(page_table=table.long()), dict(cu=cu([1, 1])), dict(out_cu=torch.zeros(1, dtype=I32)),
               dict(out=(torch.zeros(4, 2, 64), torch.zeros(4, 2, 64))), dict(out=(rnd(3, 2, 64), rnd(3, 2, 64)))):
        with pytest.raises(ValueError):
            Q.kv_gather_quant(*planes, **{**dict(page_table=table, cu=cu([4]), total_rows=4), **kw})


@pytest.mark.parametrize("cap", [1e-7, 1025.0, 1e30])
def test_caps_that_single_precision_does_not_carry_are_refused(cap):
    with pytest.raises(ValueError, match="cap"):
        S.prompt_attention(**prompt_args(rules=S.ScoreRules(cap=cap)))
    with pytest.raises(ValueError, match="cap"):
        S.decode_attention(**decode_args(rules=S.ScoreRules(cap=cap)))


def test_a_window_past_32_bits_is_refused():
    with pytest.raises(ValueError, match="window"):
        S.prompt_attention(**prompt_args(rules=S.ScoreRules(window=(1 << 32) + 5)))


def test_reading_back_refuses_bad_pages_and_rows_past_the_output():
    planes = Q.quant_planes(3, 4, 2, 64, 8, "cpu")
    for table, out_cu in ((torch.tensor([[3]], dtype=I32), [0]), (torch.tensor([[-1]], dtype=I32), [0]), (torch.tensor([[0]], dtype=I32), [2])):
        with pytest.raises(IndexError):
            Q.kv_gather_quant(*planes, table, cu([4]), 4, out=(rnd(5, 2, 64), rnd(5, 2, 64)), out_cu=torch.tensor(out_cu, dtype=I32))
    k, v = Q.kv_gather_quant(*planes, torch.zeros(0, 1, dtype=I32), cu([]), 0)
    assert k.shape == v.shape == (0, 2, 64)
    Q.kv_write_quant(rnd(0, 2, 64), rnd(0, 2, 64), torch.zeros(0, dtype=torch.int64), *planes)
