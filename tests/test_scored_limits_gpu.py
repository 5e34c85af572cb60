"""Scored attention at the ends of what its arguments may be, against the definitions in 64 bits."""
import pytest
import torch

import scored_oracle as O
from test_scored_decode_gpu import make, slopes
from test_scored_flash_gpu import packed
from uniserve_v1_b200.ops import native as N
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
