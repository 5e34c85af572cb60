"""Scored attention and integer pages where calls meet: graphs, streams, workspaces, plans that say less than they hold."""
import pytest
import torch

import scored_oracle as O
from test_scored_decode_gpu import make, slopes
from test_scored_flash_gpu import SHARED, cu, packed, shared_batch
from uniserve_v1_b200.ops import native as N
from uniserve_v1_b200.ops import quant_pages as Q
from uniserve_v1_b200.ops import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("with_docs", [False, True])
def test_prompts_in_a_captured_graph_of_a_padded_batch(with_docs):
    """Captured with room for four sequences and 700 rows; replayed with other lengths, one of them empty."""
    q, k, v, cq, ck = packed(1, [300, 130, 170, 100], [300, 130, 170, 100], 4, 2, 128)
    docs = (torch.arange(700, device=DEV) // 90).to(I32) if with_docs else None
    rules = S.ScoreRules(cap=30.0, slopes=slopes(4))
    out = torch.full_like(q, 3.0)

    def call():
        S.prompt_attention(q, k, v, cq, ck, 512, 512, 0.1, rules, docs=docs, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for counts in ([512, 1, 0, 60], [0, 0, 0, 0], [129, 127, 128, 300]):
        cq.copy_(cu(counts))
        ck.copy_(cu(counts))
        q.mul_(-1)
        out.fill_(3.0)
        graph.replay()
        n = sum(counts)
        assert (out[n:] == 3).all()
        if n:
            want, bound = O.prompt(q[:n], k[:n], v[:n], cq, ck, 0.1, 30.0, rules.slopes, docs=None if docs is None else docs[:n])
            O.check(out[:n], want, bound)
    N.raise_on_device_error()


@pytest.mark.parametrize("bits", [16, 8])
def test_two_streams_at_once(bits):
    """Two batches on two streams, each with its workspace, prompts between them."""
    both = [make(s, [900, 0, 77, 3000], 16, 2, 128, 16, bits) for s in (1, 2)]
    works = [S.decode_work(4, 16, 2, 128, DEV) for _ in both]
    p = packed(3, [400], [400], 4, 2, 64)
    alone = S.prompt_attention(*p, 400, 400, 0.1)
    streams = [torch.cuda.Stream() for _ in both]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            q, kc, vc, ks, vs, table, n = both[i]
            with torch.cuda.stream(s):
                got[i].append(S.decode_attention(q, kc, vc, table, n, 0.1, k_scale=ks, v_scale=vs, work=works[i]))
                got[i].append(S.prompt_attention(*p, 400, 400, 0.1))
    torch.cuda.synchronize()
    N.raise_on_device_error()
    for i in range(2):
        q, kc, vc, ks, vs, table, n = both[i]
        O.check(got[i][0], *O.decode(q, kc, vc, table, n, 0.1, ks=ks, vs=vs))
        assert all(torch.equal(a, got[i][0]) for a in got[i][::2]) and all(torch.equal(a, alone) for a in got[i][1::2])


def test_more_sequences_than_a_launch_takes():
    lens = [(37 * i) % 90 for i in range(S.MAX_SEQS + 5)]
    q, kc, vc, ks, vs, table, n = make(4, lens, 4, 2, 64, 16, 8)
    starts = torch.tensor([i % 5 for i in lens], dtype=I32, device=DEV)
    work = S.decode_work(len(lens), 4, 2, 64, DEV)
    got = S.decode_attention(q, kc, vc, table, n, 0.125, starts=starts, k_scale=ks, v_scale=vs, work=work)
    O.check(got, *O.decode(q, kc, vc, table, n, 0.125, starts=starts, ks=ks, vs=vs))


@pytest.mark.parametrize("cap", [2.0 ** -20, 0.01, 1024.0])
def test_the_smallest_and_largest_caps(cap):
    q, k, v, cq, ck = packed(5, [200, 70], [200, 90], 4, 2, 64, 4.0)
    O.check(S.prompt_attention(q, k, v, cq, ck, 200, 200, 0.125, S.ScoreRules(cap)), *O.prompt(q, k, v, cq, ck, 0.125, cap))
    q, kc, vc, _, _, table, n = make(6, [300, 65], 8, 2, 64, 16, 16, gain=4.0)
    O.check(S.decode_attention(q, kc, vc, table, n, 0.125, S.ScoreRules(cap)), *O.decode(q, kc, vc, table, n, 0.125, cap))


def test_a_workspace_of_other_shapes_is_refused():
    """Room for as many channels is not room for as many rows."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([4], [300], 0, [9] * 4, 8, 2, 64, 16, 16, 0.0, False))
    half = S.SharedPrefix(sh.cu_rows, sh.lens, 4, 300)
    for work in (S.decode_work(2, 8, 2, 128, DEV, half), S.decode_work(4, 8, 2, 64, DEV), S.decode_work(1, 8, 2, 64, DEV, sh)):
        with pytest.raises(ValueError, match="workspace"):
            S.decode_attention(q, kc, vc, table, n, scale, shared=sh, work=work)
    wide = S.decode_work(4, 8, 2, 128, DEV, sh)
    wide.own_ml, wide.counters = wide.own_ml[:8], torch.zeros(64, dtype=I32, device=DEV)
    with pytest.raises(ValueError, match="workspace"):
        S.decode_attention(q, kc, vc, table, n, scale, shared=sh, work=wide)


@pytest.mark.parametrize("bits,page", [(8, 16), (4, 16), (16, 24)])
def test_a_prefix_longer_than_told_sets_the_status(bits, page):
    """120 keys where 100 were told: both end in the same block of 128."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([4], [120], 0, [9] * 4, 8, 2, 64, page, bits, 0.0, False))
    N.raise_on_device_error()
    S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=S.SharedPrefix(sh.cu_rows, sh.lens, 4, 100))
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()


@pytest.mark.parametrize("bits", [16, 8])
def test_groups_past_the_batch_share_nothing(bits):
    """A plan of more rows than the batch has."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([4], [120], 0, [9] * 4, 8, 2, 64, 16, bits, 0.0, False))
    plan = S.SharedPrefix(torch.tensor([0, 4, 9, 12], dtype=I32, device=DEV), torch.tensor([120, 64, 64], dtype=I32, device=DEV), 5, 120)
    got = S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=plan)
    N.raise_on_device_error()
    O.check(got, *O.decode(q, kc, vc, table, n, scale, ks=ks, vs=vs, expanded=[120] * 4 if bits == 8 else None))


@pytest.mark.parametrize("bits,page", [(16, 16), (16, 24), (8, 16)])
def test_a_page_outside_the_cache_of_a_shared_prefix(bits, page):
    """It is read as zeros, and the status says so."""
    q, kc, vc, ks, vs, table, n, sh, cap, sl, scale = shared_batch(([4], [192], 0, [9] * 4, 8, 2, 64, page, bits, 0.0, False))
    N.raise_on_device_error()
    held = table[0, 1].long()
    table[:, 1] = kc.shape[0] + 7
    got = S.decode_attention(q, kc, vc, table, n, scale, k_scale=ks, v_scale=vs, shared=sh)
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()
    table[:, 1] = held
    kc[held] = 0
    vc[held] = 0
    O.check(got, *O.decode(q, kc, vc, table, n, scale, ks=ks, vs=vs, expanded=[192] * 4 if bits == 8 else None))


def test_rows_read_back_stay_inside_the_output():
    planes = Q.quant_planes(4, 8, 2, 64, 8, DEV)
    x = torch.randn(32, 2, 64, device=DEV).to(BF16)
    Q.kv_write_quant(x, x, torch.arange(32, device=DEV), *planes)
    table = torch.tensor([[0, 1], [2, 3]], dtype=I32, device=DEV)
    whole = Q.kv_gather_quant(*planes, table, cu([10, 10]), 20)[0]
    N.raise_on_device_error()
    out = [torch.full((40, 2, 64), 5.0, dtype=BF16, device=DEV) for _ in range(2)]
    view = tuple(t[:24] for t in out)
    Q.kv_gather_quant(*planes, table, cu([10, 10]), 20, out=view, out_cu=torch.tensor([0, 18], dtype=I32, device=DEV))
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()
    for t in out:
        assert torch.equal(t[:10], whole[:10]) and torch.equal(t[18:24], whole[10:16]) and (t[10:18] == 5).all() and (t[24:] == 5).all()
    # rows before the first sequence's are nobody's
    out = [torch.full((20, 2, 64), 5.0, dtype=BF16, device=DEV) for _ in range(2)]
    Q.kv_gather_quant(*planes, table, torch.tensor([3, 13, 20], dtype=I32, device=DEV), 20, out=tuple(out))
    N.raise_on_device_error()
    for t in out:
        assert (t[:3] == 5).all() and torch.equal(t[3:13], whole[:10]) and torch.equal(t[13:20], whole[10:17])


def test_a_step_over_integer_pages():
    """Prompts of two sequences, their rows kept as 8 bits, then single rows: written, read back and attended."""
    lens, Hq, Hkv, D, page = [130, 61], 8, 2, 128, 16
    q, k, v, cq, ck = packed(8, lens, lens, Hq, Hkv, D)
    rules = S.ScoreRules(50.0)
    O.check(S.prompt_attention(q, k, v, cq, ck, 130, 130, 0.1, rules), *O.prompt(q, k, v, cq, ck, 0.1, 50.0))
    planes = Q.quant_planes(16, page, Hkv, D, 8, DEV)
    table = torch.randperm(16, device=DEV).view(2, 8).to(I32)
    lens = [100, 61]
    rows = torch.cat([torch.arange(100), 130 + torch.arange(61)]).to(DEV)
    pos = torch.cat([torch.arange(n) for n in lens]).to(DEV)
    seq = torch.repeat_interleave(torch.arange(2), torch.tensor(lens)).to(DEV)
    slots = table[seq, pos // page].long() * page + pos % page
    Q.kv_write_quant(k[rows], v[rows], slots, *planes)
    n = torch.tensor(lens, dtype=I32, device=DEV)
    for step in range(3):
        x = torch.randn(2, 3, max(Hq, Hkv), D, device=DEV).to(BF16)
        at = n.long()
        Q.kv_write_quant(x[:, 1, :Hkv], x[:, 2, :Hkv], table[torch.arange(2, device=DEV), at // page].long() * page + at % page, *planes)
        n += 1
        got = S.decode_attention(x[:, 0, :Hq], planes[0], planes[1], table, n, 0.1, rules, k_scale=planes[2], v_scale=planes[3])
        O.check(got, *O.decode(x[:, 0, :Hq].contiguous(), planes[0], planes[1], table, n, 0.1, 50.0, ks=planes[2], vs=planes[3]))
    N.raise_on_device_error()


@pytest.mark.parametrize("Hq,Hkv,D", [(16, 1, 128), (64, 1, 64), (128, 1, 64), (256, 1, 128), (20, 1, 64), (48, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("kind", ["capped", "biased", "documents", "window", "all"])
def test_few_new_rows_behind_histories(Hq, Hkv, D, kind):
    """Many query heads a key head, and few rows: heads stand side by side in a tile."""
    new, keys = [3, 1, 0, 70, 9], [700, 1, 5, 333, 1001]
    q, k, v, cq, ck = packed(11, new, keys, Hq, Hkv, D)
    kw = {"capped": {}, "biased": {}, "documents": dict(docs=(torch.arange(sum(keys), device=DEV) // 60).to(I32)),
          "window": dict(prefix=torch.tensor([9, 0, 0, 130, 64], dtype=I32, device=DEV)), "all": dict(causal=False)}[kind]
    cap, sl, window = 30.0 if kind in ("capped", "documents") else 0.0, slopes(Hq) if kind in ("biased", "all") else None, 100 if kind == "window" else 0
    got = S.prompt_attention(q, k, v, cq, ck, 128, 1024, D ** -0.5, S.ScoreRules(cap, sl, window), **kw)
    N.raise_on_device_error()
    O.check(got, *O.prompt(q, k, v, cq, ck, D ** -0.5, cap, sl, window=window, **kw))


@pytest.mark.parametrize("case", [
    # new rows, keys, Hq, Hkv, D, cap, bias, causal, window, docs, prefix
    ([1], [5000], 32, 4, 128, 0.0, False, True, 0, None, None),
    ([37], [3001], 32, 4, 128, 50.0, False, True, 0, None, None),
    ([200, 3], [2000, 9000], 4, 1, 64, 0.0, True, True, 0, None, None),
    ([65], [4100], 8, 1, 128, 30.0, True, True, 1000, None, [130]),       # most parts see nothing
    ([30, 0, 9], [2500, 40, 0], 16, 1, 64, 50.0, False, True, 0, 900, None),      # and sequences without rows or keys
    ([100], [1500], 3, 3, 64, 0.0, False, False, 0, None, None),
    ([50], [2600], 4, 2, 128, 0.0, True, False, 0, 500, [700]),
    ([2000], [1500], 1, 1, 128, 30.0, True, True, 0, None, None),         # rows before the first key
])
def test_few_rows_over_many_keys(case):
    """The keys go in parts; rows past the last sequence stay."""
    new, keys, Hq, Hkv, D, cap, bias, causal, window, docs, prefix = case
    q, k, v, cq, ck = packed(12, new + [5], keys, Hq, Hkv, D, 3.0 if cap else 1.0)
    cq = cq[:-1].contiguous()
    n = sum(new)
    assert N.kernels().us_scored_flash_parts(len(new), max(new), max(keys), Hq, Hkv) > 1
    kw = dict(causal=causal, docs=None if docs is None else (torch.arange(sum(keys), device=DEV) // docs).to(I32),
              prefix=None if prefix is None else torch.tensor(prefix, dtype=I32, device=DEV))
    out = torch.full_like(q, 7.0)
    sl = slopes(Hq) if bias else None
    got = S.prompt_attention(q, k, v, cq, ck, max(new), max(keys), D ** -0.5, S.ScoreRules(cap, sl, window), out=out, **kw)
    N.raise_on_device_error()
    assert got is out and (out[n:] == 7).all()
    want, bound = O.prompt(q[:n], k, v, cq, ck, D ** -0.5, cap, sl, window=window, **kw)
    O.check(out[:n], want, bound)
    again = S.prompt_attention(q, k, v, cq, ck, max(new), max(keys), D ** -0.5, S.ScoreRules(cap, sl, window), **kw)
    assert torch.equal(again[:n], out[:n])


@pytest.mark.parametrize("told_q,told_k", [(37, 3000), (60, 1100)])
def test_rows_and_keys_past_what_was_told_set_the_status(told_q, told_k):
    """60 and 12 rows over 3000 and 2000 keys.  Rows that were told of are whole where their keys are."""
    q, k, v, cq, ck = packed(13, [12, 60], [2000, 3000], 32, 4, 128)
    assert N.kernels().us_scored_flash_parts(2, told_q, told_k, 32, 4) > 1
    N.raise_on_device_error()
    guard = torch.full((q.shape[0] + 64, 32, 128), 7.0, dtype=BF16, device=DEV)
    got = S.prompt_attention(q, k, v, cq, ck, told_q, told_k, 0.1, out=guard[:72])
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()
    assert (guard[72:] == 7).all()
    if told_k == 3000:
        want, bound = O.prompt(q, k, v, cq, ck, 0.1)
        for rows in (slice(0, 12), slice(12, 12 + told_q)):
            O.check(got[rows], want[rows], bound[rows])


def test_longer_sequences_than_told_under_documents_set_the_status():
    q, k, v, cq, ck = packed(14, [300], [700], 4, 2, 128)
    docs = (torch.arange(700, device=DEV) // 50).to(I32)
    N.raise_on_device_error()
    S.prompt_attention(q, k, v, cq, ck, 300, 500, 0.1, docs=docs)
    with pytest.raises(RuntimeError):
        N.raise_on_device_error()
    got = S.prompt_attention(q, k, v, cq, ck, 300, 700, 0.1, docs=docs)
    N.raise_on_device_error()
    O.check(got, *O.prompt(q, k, v, cq, ck, 0.1, docs=docs))
