"""Outputs whose rows or heads share memory are refused: a row could hold any
token's result."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from paged_util import ints, make_cache, starts  # noqa: E402


@pytest.mark.parametrize("shared", ["tokens", "heads"])
def test_shared_outputs(shared):
    k, v, table, _ = make_cache([20, 20], 2, 64, 16, fill=0.0)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    base = torch.zeros(1, 4, 64, device="cuda") if shared == "tokens" else torch.zeros(2, 1, 64, device="cuda")
    out = base.bfloat16().expand(2, 4, 64)
    at = (k, v, table, starts([1, 1]), ints([20, 20]))
    with pytest.raises(ValueError, match="out"):
        ab.paged_attention(q, out, *at, max_q_len=1)
    with pytest.raises(ValueError, match="q_out"):
        ab.qk_norm_rope(torch.zeros(2, 512, device="cuda"), out, *at, torch.zeros(32, 128, device="cuda"))


def test_one_token_and_one_head_may_have_any_stride():
    k, v, table, _ = make_cache([20], 1, 64, 16)
    q = torch.ones(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, 64), (8, 16, 1))
    ab.paged_attention(q, out, k, v, table, starts([1]), ints([20]), max_q_len=1)
    ab.qk_norm_rope(torch.ones(1, 192, device="cuda"), out, k, v, table, starts([1]), ints([20]),
                    torch.ones(32, 128, device="cuda"))
    wide = torch.zeros(5, 3, 64, dtype=torch.bfloat16, device="cuda")[2:3, 1:2]
    ab.paged_attention(q, wide, k, v, table, starts([1]), ints([20]), max_q_len=1)
    assert wide.any()
