"""Steps with nothing in them: no sequences, no tokens, empty lists."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import ints  # noqa: E402


def test_no_sequences():
    c = ab.PagedKVCache(1, 2, 64, 8, slots=4, max_len=64)
    b = c.batch([], [])
    for tokens in (0, 3):
        q = torch.zeros(tokens, 4, 64, dtype=torch.bfloat16, device="cuda")
        out = torch.full_like(q, 7.0)
        ab.paged_attention(q, out, c.k[0], c.v[0], max_q_len=tokens, **b)
        ab.qk_norm_rope(torch.ones(tokens, 512, device="cuda"), out, c.k[0], c.v[0], rope=torch.ones(8, 128, device="cuda"), **b)
        assert (out == 7).all()
    assert not c.k.any() and not c.v.any()
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)


def test_empty_lists():
    c = ab.PagedKVCache(1, 2, 64, 8, slots=4, max_len=64)
    c.update(extend=[(1, 20)])
    c.update(free=[], fork=[], extend=[])
    c.update(fork=torch.empty(0, 2, dtype=torch.int32, device="cuda"))
    assert c.lens.tolist() == [0, 20, 0, 0] and c.check()["free_pages"] == 6
    with pytest.raises((RuntimeError, ValueError)):
        c.update(extend=[1, 2, 3])


def test_no_rows_to_sample():
    ab.sample_tokens(torch.empty(0, 50, device="cuda"), torch.empty(0, device="cuda"), ints([]), torch.empty(0, device="cuda"))
    _lib.context(0).sync_status()
