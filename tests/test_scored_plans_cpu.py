"""Plans of shared prefixes and slopes on the CPU: what is refused, and rows that share nothing."""
import random

import pytest
import torch

from test_scored_cpu import cu, decode_args, prompt_args, rnd
from uniserve_v1_b200.ops import quant_pages as Q
from uniserve_v1_b200.ops import scored as S

I32 = torch.int32


@pytest.mark.parametrize("cu_rows,lens", [(torch.tensor([[0], [2]], dtype=I32), torch.tensor([2], dtype=I32)),
                                          (torch.tensor([0, 2], dtype=I32), torch.tensor([[2]], dtype=I32)),
                                          (torch.tensor([0, 1, 2], dtype=I32), torch.tensor([2], dtype=I32))])
def test_plans_of_other_shapes_are_refused(cu_rows, lens):
    with pytest.raises(ValueError, match="cu_rows"):
        S.decode_attention(**decode_args(shared=S.SharedPrefix(cu_rows, lens, 2, 2)))


def test_a_plan_may_be_columns_of_a_table():
    plan = torch.tensor([[0, 3], [1, 2], [2, 9]], dtype=I32)
    args = decode_args(seq_lens=torch.tensor([5, 6], dtype=I32), page_table=torch.tensor([[1, 2], [0, 2]], dtype=I32))
    dense = S.decode_attention(**args, shared=S.SharedPrefix(plan[:, 0].contiguous(), plan[:2, 1].contiguous(), 1, 3))
    assert torch.equal(S.decode_attention(**args, shared=S.SharedPrefix(plan[:, 0], plan[:2, 1], 1, 3)), dense)


def test_rows_before_the_first_group_share_nothing():
    args = decode_args(seq_lens=torch.tensor([5, 6], dtype=I32), page_table=torch.tensor([[1, 2], [0, 2]], dtype=I32))
    alone = S.decode_attention(**args)
    plan = S.SharedPrefix(torch.tensor([1, 2], dtype=I32), torch.tensor([4], dtype=I32), 1, 4)
    assert torch.equal(S.decode_attention(**args, shared=plan), alone)


def test_a_group_that_begins_before_the_batch_raises():
    plan = S.SharedPrefix(torch.tensor([-1, 2], dtype=I32), torch.tensor([2], dtype=I32), 3, 2)
    with pytest.raises(IndexError, match="begins"):
        S.decode_attention(**decode_args(shared=plan))


def test_negative_slopes_are_refused():
    rules = S.ScoreRules(slopes=torch.tensor([0.5, 0.0, -0.25, 0.1]))
    with pytest.raises(ValueError, match="negative"):
        S.prompt_attention(**prompt_args(rules=rules))
    with pytest.raises(ValueError, match="negative"):
        S.decode_attention(**decode_args(rules=rules))


def test_rows_of_no_sequence_before_the_first_and_past_the_last():
    """Zeros, or what a given output held."""
    args = prompt_args(q=rnd(9, 4, 16), cu_q=torch.tensor([2, 6], dtype=I32))
    got = S.prompt_attention(**args)
    assert not got[:2].any() and not got[6:].any() and got[2:6].any()
    out = torch.full_like(got, 5.0)
    S.prompt_attention(**args, out=out)
    assert (out[:2] == 5).all() and (out[6:] == 5).all() and torch.equal(out[2:6], got[2:6])


@pytest.mark.parametrize("Hq,Hkv", [(32, 4), (64, 64), (17, 1), (128, 128), (300, 100)])
@pytest.mark.parametrize("keys", [0, 1, 4096, 1 << 20, 1 << 27, (1 << 31) - 1, 1 << 40])
def test_the_tile_list_of_a_launch_stays_in_31_bits(Hq, Hkv, keys):
    """Tiles of 32 keys of every sequence and key head (or sixteen of its query heads); one more sequence would not fit."""
    most = S._most_seqs(Hq, Hkv, keys)
    tiles = Hkv * -(-(Hq // Hkv) // 16) * max(1, -(-keys // 32))
    assert 0 <= most <= S.MAX_SEQS and most * tiles < 1 << 31
    assert most == S.MAX_SEQS or (most + 1) * (tiles + Hkv * -(-(Hq // Hkv) // 16)) >= 1 << 31
    # (the call's own shorter test never passes what does not fit)
    for B in (1, most, most + 1, 700):
        assert B <= most or B > S.MAX_SEQS or B * Hq * (keys + 64) >= 1 << 36


def test_rows_whose_scores_are_all_minus_infinity_are_zeros():
    """Like rows that see nothing; a score that is no number beside them makes the row none."""
    q, k, v = rnd(3, 2, 16), rnd(3, 1, 16, seed=1), rnd(3, 1, 16, seed=2)
    k[:, :, 0], q[:, :, 0] = 1.0, 0.5
    q[0, 1, 0] = q[1, 0, 0] = float("-inf")
    got = S.prompt_attention(**prompt_args(q=q, k=k, v=v, cu_q=torch.tensor([0, 3], dtype=I32), cu_k=torch.tensor([0, 3], dtype=I32)))
    assert not got[0, 1].any() and not got[1, 0].any() and torch.isfinite(got).all() and got[2].any()
    k[0, 0, 3] = float("nan")
    got = S.prompt_attention(**prompt_args(q=q, k=k, v=v, cu_q=torch.tensor([0, 3], dtype=I32), cu_k=torch.tensor([0, 3], dtype=I32)))
    assert got.isnan().all()


@pytest.mark.parametrize("seed", range(8))
def test_a_workspace_has_room_for_every_plan_of_up_to_its_sizes(seed):
    r = random.Random(seed)
    for _ in range(400):
        Hkv = r.choice([1, 2, 4, 8])
        Hq, groups, rows, longest = Hkv * r.choice([1, 3, 8, 16, 64, 128]), r.randint(1, 9), r.randint(1, 700), r.choice([1, 500, 9000, 70_000, 1 << 21])
        room = S._prefix_room(S.SharedPrefix(None, torch.zeros(groups), rows, longest), Hq, Hkv, 148)
        for _ in range(5):
            small = S.SharedPrefix(None, torch.zeros(r.randint(1, groups)), r.randint(1, rows), r.randint(1, longest))
            pairs, parts, each = S._prefix_plan(small, Hq, Hkv, 148)
            assert small.groups * pairs * Hkv * parts * 256 <= room and parts * each * 128 >= small.max_len and each <= 512


@pytest.mark.parametrize("into", [None, 9])
def test_reading_back_refuses_more_rows_than_told(into):
    planes = Q.quant_planes(3, 4, 2, 64, 8, "cpu")
    out = None if into is None else (rnd(into, 2, 64), rnd(into, 2, 64))
    with pytest.raises(IndexError, match="told"):
        Q.kv_gather_quant(*planes, torch.tensor([[0, 1]], dtype=I32), cu([6]), 5, out=out)
