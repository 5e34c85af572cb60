"""Decode batches with shared prefixes whose plans say more or less than the pages hold."""
import pytest
import torch

import scored_oracle as O
from test_scored_decode_gpu import make, slopes
from test_scored_flash_gpu import shared_batch
from uniserve_v1_b200.ops import native as N
from uniserve_v1_b200.ops import quant_pages as Q
from uniserve_v1_b200.ops import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, I32 = torch.bfloat16, torch.int32


def soiled(work):
    """A workspace as an earlier call may have left it."""
    for t in (work.prefix_o, work.prefix_ml, work.own_o, work.own_ml, work.scratch):
        t.fill_(float("nan"))
    work.prefix_ml[::2] = 3.0          # maxima that look like some
    work.prefix_ml[1::2] = 1.0
    return work


def test_a_prefix_of_more_than_a_million_keys():
    """Its last part counts like its first: values behind key 2^20 stand out."""
    long, rows = 1_500_000, 8
    q, kc, vc, _, _, table, n = make(41, [long] + [1] * (rows - 1), 2, 1, 64, 64, 16)
    vc.view(-1, 1, 64)[(table[0, (1 << 20) // 64:].long()[:, None] * 64 + torch.arange(64, device=DEV)).flatten()] += 4.0
    table = table[:1].expand(rows, -1).contiguous()
    n = torch.tensor([long - i * 7 for i in range(rows)], dtype=I32, device=DEV)
    plan = S.SharedPrefix(torch.tensor([0, rows], dtype=I32, device=DEV), torch.tensor([long - 100], dtype=I32, device=DEV), rows, long - 100)
    work = soiled(S.decode_work(rows, 2, 1, 64, DEV, plan))
    got = S.decode_attention(q, kc, vc, table, n, 0.125, shared=plan, work=work)
    N.raise_on_device_error()
    want, bound = O.decode(q, kc, vc, table, n, 0.125)
    assert float(want.mean()) > 1.0
    O.check(got, want, bound)


@pytest.mark.parametrize("bits,page,told", [(16, 16, 1000), (16, 16, 520), (16, 24, 1000), (8, 16, 1000), (4, 16, 1000), (16, 128, 100_000)])
def test_a_prefix_past_the_page_lists(bits, page, told):
    """Lists of 480 keys, a prefix of `told`: rows of up to 480 keys are whole, and the status says so."""
    lens = [480, 300, 1, 0, 479, 128, 33]
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([7], [480], 0, [0] * 7, 8, 2, 64, page, bits, 0.0, True))
    table = table[:, :480 // page].contiguous() if 480 % page == 0 else table[:, :-(-480 // page)].contiguous()
    n.copy_(torch.tensor(lens, dtype=I32, device=DEV))
    plan = S.SharedPrefix(sh.cu_rows, torch.full_like(sh.lens, told), 7, told)
    work = soiled(S.decode_work(7, 8, 2, 64, DEV, plan))
    N.raise_on_device_error()
    got = S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(slopes=sl), k_scale=ks, v_scale=vs, shared=plan, work=work)
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()
    O.check(got, *O.decode(q, kc, vc, table, n, scale, slopes=sl, ks=ks, vs=vs, expanded=[480] * 7 if ks is not None else None))


@pytest.mark.parametrize("bits,page", [(16, 16), (16, 24), (8, 16)])
def test_the_rest_of_a_prefix_longer_than_told_is_read_row_by_row(bits, page):
    """2000 keys where 600 were told: no key is lost, and the status says so."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([4], [2000], 1, [9, 1, 0, 70, 40], 8, 2, 64, page, bits, 30.0, False))
    plan = S.SharedPrefix(sh.cu_rows, sh.lens, 4, 600)
    work = soiled(S.decode_work(5, 8, 2, 64, DEV, plan))
    N.raise_on_device_error()
    got = S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(cap), k_scale=ks, v_scale=vs, shared=plan, work=work)
    if bits != 16 or page != 16 or S._prefix_plan(plan, 8, 2, S._sm_count(0))[1] * S._prefix_plan(plan, 8, 2, S._sm_count(0))[2] * 128 < 2000:
        with pytest.raises(RuntimeError):
            N.raise_on_device_error()
    O.check(got, *O.decode(q, kc, vc, table, n, scale, cap, ks=ks, vs=vs, expanded=[600] * 4 + [0] if ks is not None else None))


@pytest.mark.parametrize("bits,page,cap", [(16, 16, 0.0), (16, 128, 30.0), (16, 24, 0.0), (8, 16, 0.0), (4, 16, 30.0)])
def test_what_a_prefix_holds_behind_its_rows_reaches_none(bits, page, cap):
    """A prefix of 900 keys over rows of up to 300: behind them the pages hold NaN and infinities."""
    lens = [300, 300, 129, 1, 0, 257]
    q, kc, vc, ks, vs, table, n, sh, _, sl, scale = shared_batch(([6], [900], 0, [0] * 6, 8, 2, 64, page, bits, cap, False))
    n.copy_(torch.tensor(lens, dtype=I32, device=DEV))
    want, bound = O.decode(q, kc, vc, table, n, scale, cap, ks=ks, vs=vs, expanded=[900] * 6 if ks is not None else None)
    pos = torch.arange(300, 900, device=DEV)
    at, off = table[0, pos // page].long(), pos % page
    if bits == 16:
        kc[at, off] = float("nan")
        vc[at, off] = float("inf")
        vc[at[::3], off[::3]] = float("nan")
    else:
        ks[at, :, off] = float("nan")
        vs[at, :, off] = float("nan")
    got = S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(cap), k_scale=ks, v_scale=vs, shared=sh)
    N.raise_on_device_error()
    if ks is not None:          # the largest scale of the prefix may have been behind its rows: another power of two
        want, bound = O.decode(q, kc, vc, table, n, scale, cap, ks=ks.nan_to_num(), vs=vs.nan_to_num(), expanded=[900] * 6)
    O.check(got, want, bound)


@pytest.mark.parametrize("bits,page", [(16, 16), (16, 24), (8, 16)])
def test_a_plan_may_be_columns_of_a_table(bits, page):
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([3, 4], [600, 250], 1, [9, 1, 0, 70, 40, 5, 6, 8], 8, 2, 64, page, bits, 0.0, False))
    plan = torch.stack([sh.cu_rows, torch.cat([sh.lens, sh.lens[:1]])], 1)
    got = S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=S.SharedPrefix(plan[:, 0], plan[:2, 1], 4, 600))
    N.raise_on_device_error()
    assert torch.equal(got, S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=sh))
    O.check(got, *O.decode(q, kc, vc, table, n, scale, ks=ks, vs=vs, expanded=[600] * 3 + [250] * 4 + [0] if ks is not None else None))


@pytest.mark.parametrize("bits,page,cap", [(16, 16, 0.0), (16, 24, 30.0), (8, 16, 0.0), (4, 16, 30.0)])
def test_rows_before_the_first_group_and_past_the_last_share_nothing(bits, page, cap):
    """The lists of rows that do share hold no pages below the prefix, but for the first one's."""
    case = ([1, 1, 3, 4], [0, 0, 600, 250], 2, [700, 33, 1, 0, 70, 40, 5, 6, 300, 90, 513], 8, 2, 64, page, bits, cap, False)
    q, kc, vc, ks, vs, table, n, _, cap, sl, scale = shared_batch(case)
    want, bound = O.decode(q, kc, vc, table, n, scale, cap, ks=ks, vs=vs, expanded=[0] * 2 + [600] * 3 + [250] * 4 + [0] * 2 if ks is not None else None)
    table[3:5, :600 // page] = -1
    table[6:9, :250 // page] = kc.shape[0]
    plan = S.SharedPrefix(torch.tensor([2, 5, 5, 9], dtype=I32, device=DEV), torch.tensor([600, 77, 250], dtype=I32, device=DEV), 4, 600)
    work = soiled(S.decode_work(11, 8, 2, 64, DEV, plan))
    got = S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(cap), k_scale=ks, v_scale=vs, shared=plan, work=work)
    N.raise_on_device_error()
    O.check(got, want, bound)


@pytest.mark.parametrize("bits,page", [(16, 16), (16, 24), (8, 16)])
def test_a_group_that_begins_before_the_batch_shares_nothing(bits, page):
    """Rows 0 and 1 of the first group; the second one is served.  The status says so."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([2, 3], [300, 450], 0, [9, 1, 0, 70, 40], 8, 2, 64, page, bits, 0.0, False))
    plan = S.SharedPrefix(torch.tensor([-3, 2, 5], dtype=I32, device=DEV), sh.lens, 5, 450)
    work = soiled(S.decode_work(5, 8, 2, 64, DEV, plan))
    N.raise_on_device_error()
    got = S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=plan, work=work)
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()
    O.check(got, *O.decode(q, kc, vc, table, n, scale, ks=ks, vs=vs, expanded=[0] * 2 + [450] * 3 if ks is not None else None))


def test_rows_of_a_group_past_those_told_read_their_own_lists():
    """Six rows of 64 query heads a key head, of which two were told and four have room.  The status says so."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([6], [300], 0, [9, 1, 0, 70, 40, 5], 64, 1, 64, 16, 16, 0.0, False))
    plan = S.SharedPrefix(sh.cu_rows, sh.lens, 2, 300)
    work = soiled(S.decode_work(6, 64, 1, 64, DEV, plan))
    N.raise_on_device_error()
    got = S.decode_attention(q, kc, vc, table, n, scale, shared=plan, work=work)
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()
    O.check(got, *O.decode(q, kc, vc, table, n, scale))


def one_key_above(bits, keys, rows, Hq, away, at):
    """Queries and integer pages of a prefix of `keys` that `rows` share: key `at`'s weight is e^away times that of each other;
    values of 1, and 0 there.  Scale 1 / 8, 64 channels."""
    page = 64
    kc, vc, ks, vs = Q.quant_planes(keys // page + 1, page, 1, 64, bits, DEV)
    k, v = torch.zeros(keys, 1, 64, dtype=BF16, device=DEV), torch.ones(keys, 1, 64, dtype=BF16, device=DEV)
    if away:
        k[at], v[at] = away / 8, 0.0
    Q.kv_write_quant(k, v, torch.arange(keys, device=DEV), kc, vc, ks, vs)
    table = torch.arange(keys // page, device=DEV).to(I32).expand(rows, -1).contiguous()
    n = torch.full((rows,), keys, dtype=I32, device=DEV)
    plan = S.SharedPrefix(torch.tensor([0, rows], dtype=I32, device=DEV), torch.tensor([keys], dtype=I32, device=DEV), rows, keys)
    return torch.ones(rows, Hq, 64, dtype=BF16, device=DEV), kc, vc, ks, vs, table, n, plan


@pytest.mark.parametrize("rows,Hq", [(3, 2), (150, 128)])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("keys,away", [(1 << 20, 0.0), (1 << 20, 10.0), (1 << 21, 0.0)])
def test_sums_of_millions_of_values_of_one_sign(keys, away, bits, rows, Hq):
    """For many rows of many heads a prefix would be one part, and each of its sums one chain of products."""
    q, kc, vc, ks, vs, table, n, plan = one_key_above(bits, keys, rows, Hq, away, 777)
    got = S.decode_attention(q, kc, vc, table, n, 0.125, k_scale=ks, v_scale=vs, shared=plan)
    N.raise_on_device_error()
    want, bound = O.decode(q[:1, :1], kc, vc, table[:1], n[:1], 0.125, ks=ks, vs=vs, expanded=[keys])
    O.check(got, want.expand(rows, Hq, -1), bound.expand(rows, Hq, -1))


@pytest.mark.parametrize("rows,Hq", [(3, 2), (150, 128)])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("away", [17.5, 20.0, 24.0])
def test_small_weights_of_an_integer_prefix_add_up(away, bits, rows, Hq):
    """A key near the prefix's end, which is walked first, outweighs each of the others by more than FP16 has room for."""
    q, kc, vc, ks, vs, table, n, plan = one_key_above(bits, 1 << 20, rows, Hq, away, (1 << 20) - 5)
    got = S.decode_attention(q, kc, vc, table, n, 0.125, k_scale=ks, v_scale=vs, shared=plan)
    N.raise_on_device_error()
    want, bound = O.decode(q[:1, :1], kc, vc, table[:1], n[:1], 0.125, ks=ks, vs=vs, expanded=[1 << 20])
    O.check(got, want.expand(rows, Hq, -1), bound.expand(rows, Hq, -1))


@pytest.mark.parametrize("case", [([9, 5], [1500, 700], 1, [10 + i for i in range(15)], 32, 4, 128, 16, 8, 50.0, False),
                                  ([9, 5], [1500, 700], 0, [10 + i for i in range(14)], 16, 2, 64, 16, 4, 0.0, True),
                                  ([40], [4000], 0, [1 + i % 9 for i in range(40)], 8, 1, 128, 16, 8, 0.0, False),
                                  ([6], [300], 0, [9] * 6, 16, 4, 64, 16, 8, 30.0, True)])
def test_integer_prefixes_against_the_values_of_the_pages(case):
    """The definition itself, without the prefix's rounding to FP16 in the oracle.  That rounding moves each key's and value's
    channel by 2^-11 of it (scales here are within 2^10 of the largest, so none is under FP16's normal numbers by more than
    their own last bit): a score by 2^-11 sum |q k| scale, a weight by twice that, a value's share by 2^-11 of it."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(case)
    want, bound = O.decode(q, kc, vc, table, n, scale, cap, sl, ks=ks, vs=vs)
    for b, length in enumerate(n.tolist()):
        pages = table[b, :-(-length // kc.shape[1])].long()
        k, v = (O.cached(c, s, pages, length).repeat_interleave(q.shape[1] // kc.shape[2], 1) for c, s in ((kc, ks), (vc, vs)))
        s = torch.einsum("hd,khd->hk", q[b].double(), k) * scale
        err = torch.einsum("hd,khd->hk", q[b].double().abs(), k.abs()).amax() * scale * 2.0 ** -11
        if cap:
            s = cap * torch.tanh(s / cap)
        if sl is not None:
            s = s - sl.double()[:, None] * (length - 1 - torch.arange(length, device=DEV))
        mass = torch.einsum("hk,khd->hd", torch.softmax(s, -1), v.abs())
        bound[b] += mass * (2 * err + 2.0 ** -11)
    got = S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(cap, sl), k_scale=ks, v_scale=vs, shared=sh)
    N.raise_on_device_error()
    O.check(got, want, bound)


@pytest.mark.parametrize("told", [19_000, 148 * 128])
def test_a_workspace_serves_smaller_plans(told):
    """One for three prefixes of up to `told` keys (three are cut into 22 parts of 148 blocks, one into 74); steps with two, with
    one that is told to be as long, with shorter ones."""
    q, kc, vc, _, _, table, n, sh, _, sl, scale = shared_batch(([6, 2], [2000, 700], 0, [9, 1, 0, 70, 40, 5, 6, 8], 8, 2, 64, 16, 16, 0.0, False))
    work = S.decode_work(8, 8, 2, 64, DEV, S.SharedPrefix(None, torch.zeros(3), 8, told))
    want, bound = O.decode(q, kc, vc, table, n, scale)
    for plan in (S.SharedPrefix(sh.cu_rows[:2], sh.lens[:1], 6, told), sh, S.SharedPrefix(sh.cu_rows[:2], sh.lens[:1], 6, 2000), S.SharedPrefix(sh.cu_rows[1:], sh.lens[1:], 2, 700)):
        O.check(S.decode_attention(q, kc, vc, table, n, scale, shared=plan, work=work), want, bound)
    N.raise_on_device_error()


def test_shared_prefixes_on_two_streams_at_once():
    """Each with its workspace; other launches between them."""
    cases = [([8], [2033], 0, [61, 1, 0, 16, 17, 40, 3, 9], 32, 4, 128, 16, 16, 30.0, False),
             ([9, 5], [1500, 700], 0, [10 + i for i in range(14)], 32, 4, 128, 16, 8, 50.0, False)]
    both = [shared_batch(c, seed=50 + i) for i, c in enumerate(cases)]
    works = [S.decode_work(b[0].shape[0], 32, 4, 128, DEV, b[7]) for b in both]

    def call(i):
        q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = both[i]
        return S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(cap), k_scale=ks, v_scale=vs, shared=sh, work=works[i])
    alone = [call(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in both]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    N.raise_on_device_error()
    for i in range(2):
        assert all(torch.equal(g, alone[i]) for g in got[i])


@pytest.mark.parametrize("bits", [8, 4])
def test_integer_prefixes_in_a_captured_graph(bits):
    """Replayed with other queries, lengths and a shorter prefix: what was expanded before does not stay."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([6], [900], 1, [61, 1, 0, 16, 17, 40, 300], 8, 2, 64, 16, bits, 30.0, False))
    work = S.decode_work(7, 8, 2, 64, DEV, sh)
    out = torch.empty_like(q)

    def call():
        S.decode_attention(q, kc, vc, table, n, scale, S.ScoreRules(cap), k_scale=ks, v_scale=vs, shared=sh, work=work, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for length, less in ((900, 0), (512, 300), (0, 0), (899, 1)):
        q.mul_(-0.75)
        sh.lens.fill_(length)
        n.sub_(less).clamp_(min=0)
        out.fill_(9.0)
        graph.replay()
        N.raise_on_device_error()
        O.check(out, *O.decode(q, kc, vc, table, n, scale, cap, ks=ks, vs=vs, expanded=[length] * 6 + [0]))
