"""Scored decode attention and integer cache pages against their definitions in 64 bits."""
import pytest
import torch

import scored_oracle as O
from uniserve_v1_b200.ops import native as N
from uniserve_v1_b200.ops import quant_pages as Q
from uniserve_v1_b200.ops import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, I32 = torch.bfloat16, torch.int32


def make(seed, lens, Hq, Hkv, D, page, bits, extra_pages=3, width=None, gain=1.0):
    """Queries, pages in no order and whatever integer pages need; pages that nobody holds are full of NaN (bf16)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra_pages
    order = torch.randperm(pages, generator=g, device=DEV).to(I32)
    table = torch.full((len(lens), width or max(1, max(need))), int(order[-1]), dtype=I32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    q = (torch.randn(len(lens), Hq, D, generator=g, device=DEV) * gain).to(BF16)
    rows = [torch.randn(pages, page, Hkv, D, generator=g, device=DEV).to(BF16) for _ in range(2)]
    if bits == 16:
        for t in rows:
            t[order[at:].long()] = float("nan")
            for b, n in enumerate(lens):       # and what lies behind a sequence's end in its last page
                if n % page:
                    t[table[b, need[b] - 1].long(), n % page:] = float("inf")
        return q, rows[0], rows[1], None, None, table, torch.tensor(lens, dtype=I32, device=DEV)
    kc, vc, ks, vs = Q.quant_planes(pages, page, Hkv, D, bits, DEV)
    slots = torch.arange(pages * page, device=DEV)
    Q.kv_write_quant(rows[0].flatten(0, 1), rows[1].flatten(0, 1), slots, kc, vc, ks, vs)
    for s in (ks, vs):
        s[order[at:].long()] = float("nan")
        for b, n in enumerate(lens):
            if n % page:
                s[table[b, need[b] - 1].long(), :, n % page:] = float("nan")
    return q, kc, vc, ks, vs, table, torch.tensor(lens, dtype=I32, device=DEV)


def slopes(Hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV)


CASES = [
    # lens, Hq, Hkv, D, page, bits, cap, bias, window, starts
    ([1], 4, 4, 128, 16, 16, 0.0, False, 0, None),
    ([1000], 32, 4, 128, 16, 16, 50.0, False, 0, None),
    ([0, 1, 127, 128, 129, 4099, 0, 17], 32, 4, 128, 16, 16, 30.0, True, 0, None),
    ([700, 33, 2000], 16, 16, 64, 16, 16, 0.0, True, 0, None),
    ([700, 33, 2000], 12, 4, 128, 5, 16, 0.0, False, 100, None),
    ([300, 299, 7], 20, 4, 64, 1, 16, 50.0, True, 0, [250, 299, 3]),
    ([513, 255, 64], 9, 1, 128, 24, 16, 0.0, False, 0, [0, 300, 63]),
    ([4000, 1], 17, 1, 128, 16, 16, 20.0, False, 0, None),
    ([300, 1], 71, 1, 64, 32, 16, 0.0, True, 64, None),
    ([1000], 32, 4, 128, 16, 8, 50.0, False, 0, None),
    ([0, 1, 127, 257, 255, 4099, 0, 17], 32, 4, 128, 16, 8, 30.0, True, 0, None),
    ([700, 33, 2001], 16, 16, 64, 16, 8, 0.0, True, 0, None),
    ([700, 33, 2000], 40, 4, 64, 6, 8, 0.0, False, 99, None),
    ([1000], 64, 4, 128, 16, 4, 0.0, False, 0, None),
    ([0, 1, 127, 257, 255, 4099, 0, 17], 32, 4, 128, 16, 4, 30.0, True, 0, None),
    ([700, 33, 2001], 8, 2, 64, 16, 4, 0.0, True, 0, None),
    ([700, 33, 2000], 12, 1, 64, 2, 4, 50.0, False, 0, [13, 32, 1999]),
    ([40 + 13 * (i % 9) for i in range(300)], 8, 2, 128, 16, 16, 0.0, False, 0, None),
    ([3 + (i % 5) for i in range(1030)], 4, 2, 64, 4, 8, 0.0, True, 0, None),
    ([100, 30011], 16, 2, 128, 64, 16, 0.0, True, 0, None),
]


@pytest.mark.parametrize("case", CASES, ids=[f"{i}-{c[5]}bit-{c[1]}x{c[2]}x{c[3]}" for i, c in enumerate(CASES)])
def test_single_rows(case):
    lens, Hq, Hkv, D, page, bits, cap, bias, window, starts = case
    q, kc, vc, ks, vs, table, n = make(7, lens, Hq, Hkv, D, page, bits, gain=3.0 if cap else 1.0)
    sl = slopes(Hq) if bias else None
    st = torch.tensor(starts, dtype=I32, device=DEV) if starts else None
    got = S.decode_attention(q, kc, vc, table, n, D ** -0.5, S.ScoreRules(cap, sl, window), starts=st, k_scale=ks, v_scale=vs)
    want, bound = O.decode(q, kc, vc, table, n, D ** -0.5, cap, sl, window, starts, ks, vs)
    N.raise_on_device_error()
    O.check(got, want, bound)
    assert not got[n <= 0].any()


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_a_workspace_serves_call_after_call_and_a_captured_graph(bits):
    lens = [300, 5, 0, 1777]
    q, kc, vc, ks, vs, table, n = make(3, lens, 16, 2, 128, 16, bits)
    work = S.decode_work(4, 16, 2, 128, DEV)
    rules = S.ScoreRules(cap=30.0)

    def call(out=None):
        return S.decode_attention(q, kc, vc, table, n, 0.1, rules, k_scale=ks, v_scale=vs, work=work, out=out)
    first = call()
    again = [call() for _ in range(5)]
    assert all(torch.equal(first, a) for a in again)
    assert not work.counters.any()
    out = torch.empty_like(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for t in (q, table, n):                 # another batch in the same places
        t.copy_(t.flip(0))
    graph.replay()
    want, bound = O.decode(q, kc, vc, table, n, 0.1, 30.0, ks=ks, vs=vs)
    O.check(out, want, bound)


def test_strided_queries_and_outputs():
    q, kc, vc, _, _, table, n = make(5, [200, 31], 8, 2, 64, 16, 16)
    fused = torch.randn(2, 8 * 64 + 40, device=DEV, dtype=BF16)
    fused[:, 8:8 + 512] = q.flatten(1)
    want, bound = O.decode(q, kc, vc, table, n, 0.125)
    O.check(S.decode_attention(fused[:, 8:520].unflatten(1, (8, 64)), kc, vc, table, n, 0.125), want, bound)
    fused[:, 3:515] = q.flatten(1)                      # rows that start on no 16 bytes
    O.check(S.decode_attention(fused[:, 3:515].unflatten(1, (8, 64)), kc, vc, table, n, 0.125), want, bound)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)     # heads outermost
    O.check(S.decode_attention(turned, kc, vc, table, n, 0.125), want, bound)
    wide = torch.full((2, 8, 80), 7.0, device=DEV, dtype=BF16)
    S.decode_attention(q, kc, vc, table, n, 0.125, out=wide[:, :, 8:72])
    O.check(wide[:, :, 8:72], want, bound)
    assert (wide[:, :, :8] == 7).all() and (wide[:, :, 72:] == 7).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_far_positions(bits):
    """A cache of more than 2^31 bytes a plane: the rows at its end."""
    page, Hkv, D = 64, 8, 128
    pages = (1 << 31) // (page * Hkv * D * bits // 8) + 600
    if bits == 16:
        kc, vc = (torch.zeros(pages, page, Hkv, D, device=DEV, dtype=BF16) for _ in range(2))
        ks = vs = None
    else:
        kc, vc, ks, vs = Q.quant_planes(pages, page, Hkv, D, bits, DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    n = 30001
    use = torch.arange(pages - 1, pages - 1 - -(-n // page), -1, device=DEV)
    rows = [torch.randn(use.shape[0] * page, Hkv, D, generator=g, device=DEV).to(BF16) for _ in range(2)]
    slots = (use[:, None] * page + torch.arange(page, device=DEV)).flatten()
    if bits == 16:
        for cache, r in ((kc, rows[0]), (vc, rows[1])):
            cache.view(-1, Hkv, D)[slots] = r
    else:
        Q.kv_write_quant(rows[0], rows[1], slots, kc, vc, ks, vs)
    q = torch.randn(1, 16, D, generator=g, device=DEV).to(BF16)
    table, lens = use[None].to(I32).contiguous(), torch.tensor([n], dtype=I32, device=DEV)
    got = S.decode_attention(q, kc, vc, table, lens, D ** -0.5, k_scale=ks, v_scale=vs)
    want, bound = O.decode(q, kc, vc, table, lens, D ** -0.5, ks=ks, vs=vs)
    N.raise_on_device_error()
    O.check(got, want, bound)


def test_infinite_and_missing_scores():
    q, kc, vc, _, _, table, n = make(9, [150, 60], 4, 2, 64, 16, 16)
    kc[table[0, 1].long(), 3] = float("nan")            # a visible key that is not a number
    got = S.decode_attention(q, kc, vc, table, n, 0.125)
    assert got[0].isnan().all() and torch.isfinite(got[1]).all()
    starts = torch.tensor([20, 0], dtype=I32, device=DEV)     # the same key out of sight
    got = S.decode_attention(q, kc, vc, table, n, 0.125, starts=starts)
    want, bound = O.decode(q, kc, vc, table, n, 0.125, starts=starts)
    O.check(got, want, bound)


# ---------------------------------------------------------------- the cache --
@pytest.mark.parametrize("T,Hkv,D,page,bits,wide", [(1, 1, 64, 2, 8, True), (3, 4, 128, 16, 4, False), (517, 2, 64, 16, 4, True),
                                                     (1000, 4, 128, 16, 8, True), (65, 3, 192, 6, 4, False), (64, 8, 256, 64, 8, False)])
def test_rows_written_and_read_back_are_the_formulas(T, Hkv, D, page, bits, wide):
    g = torch.Generator(device=DEV).manual_seed(T)
    pages = -(-T // page) + 2
    planes = Q.quant_planes(pages, page, Hkv, D, bits, DEV)
    mirror = [t.cpu() for t in planes]
    k, v = ((torch.randn(T, Hkv, D, generator=g, device=DEV) * 10 ** (6 * torch.rand(T, Hkv, 1, generator=g, device=DEV) - 3)).to(BF16)
            for _ in range(2))
    if T > 16:
        k[5, 0, :64] = 0.0
        k[6, 0, 3] = float("inf")
        v[7, 0, 63] = float("nan")
        v[8, 0, :64] = 1e-36
        k[9, 0, :64] = 3e38
        k[10, 0, :64] = -2.5
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:T]
    if T > 20:
        slots[17] = -1
    slots = slots if wide else slots.to(I32)
    Q.kv_write_quant(k, v, slots, *planes)
    Q.kv_write_quant(k.cpu(), v.cpu(), slots.cpu(), *mirror)
    N.raise_on_device_error()
    for a, b in zip(planes, mirror):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) or torch.equal(a.cpu().isnan(), b.isnan()) and \
            torch.equal(a.cpu().nan_to_num(), b.nan_to_num())
    # read back through page lists, as they lie, behind other rows
    lens = [min(page * pages, 1 + page), 0, min(page * pages, 2 * page - 1)]
    table = torch.stack([torch.randperm(pages, generator=g, device=DEV)[:2] for _ in lens]).to(I32)
    cu = torch.tensor([0, lens[0], lens[0], sum(lens)], dtype=I32, device=DEV)
    a = Q.kv_gather_quant(*planes, table, cu, sum(lens))
    b = Q.kv_gather_quant(*mirror, table.cpu(), cu.cpu(), sum(lens))
    for x, y in zip(a, b):
        assert torch.equal(x.cpu().isnan(), y.isnan()) and torch.equal(x.cpu().nan_to_num(), y.nan_to_num())
    out = [torch.full((sum(lens) + 9, Hkv, D), 5.0, dtype=BF16, device=DEV) for _ in range(2)]
    Q.kv_gather_quant(*planes, table, cu, sum(lens), out=tuple(out), out_cu=torch.tensor([2, 0, lens[0] + 5], dtype=I32, device=DEV))
    N.raise_on_device_error()
    for x, y in zip(out, b):
        assert torch.equal(x[2:2 + lens[0]].cpu().nan_to_num(), y[:lens[0]].nan_to_num())
        assert torch.equal(x[lens[0] + 5:lens[0] + 5 + lens[2]].cpu().nan_to_num(), y[lens[0]:].nan_to_num())
        rest = torch.cat([x[:2], x[2 + lens[0]:lens[0] + 5], x[lens[0] + 5 + lens[2]:]])
        assert (rest == 5).all()


def test_rows_of_a_fused_projection_are_written_as_they_lie():
    planes = Q.quant_planes(8, 4, 2, 64, 8, DEV)
    other = Q.quant_planes(8, 4, 2, 64, 8, DEV)
    x = torch.randn(9, 6 * 64 + 8, device=DEV, dtype=BF16)
    slots = torch.arange(20, 29, device=DEV)
    k, v = x[:, 128:256].unflatten(1, (2, 64)), x[:, 257:385].unflatten(1, (2, 64))
    Q.kv_write_quant(k, v, slots, *planes)
    Q.kv_write_quant(k.contiguous(), v.contiguous(), slots, *other)
    assert all(torch.equal(a, b) for a, b in zip(planes, other))
