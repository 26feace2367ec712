"""Broadcast inputs of the paged-serving operators (one row for all): the same
results as their copies row by row."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import ints, make_cache, starts  # noqa: E402


def noise(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [7, 1001, 50000, 400001])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.8), dict(temperature=0.0)])
def test_many_draws_from_one_row(dtype, vocab, kw):
    row = (2 * noise(1, vocab)).to(dtype).cuda()
    u = torch.rand(64, generator=torch.Generator().manual_seed(1)).cuda()
    out = []
    for logits in (row.expand(64, -1), row.expand(64, -1).contiguous()):
        tok, lp = torch.full((64,), -9, dtype=torch.int32, device="cuda"), torch.full((64,), 9.0, device="cuda")
        ab.sample_tokens(logits, u, tok, lp, **kw)
        out.append((tok, lp))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)


def test_draws_from_overlapping_rows():
    flat = noise(900).cuda()
    u = torch.rand(5, generator=torch.Generator().manual_seed(1)).cuda()
    a, b = (torch.empty(5, dtype=torch.int32, device="cuda") for _ in range(2))
    ab.sample_tokens(flat.as_strided((5, 500), (99, 1)), u, a)
    ab.sample_tokens(flat.as_strided((5, 500), (99, 1)).contiguous(), u, b)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_qkv_row_for_every_token(dtype):
    row = noise(1, 8 * 64).to(dtype).cuda()
    rope = torch.rand(64, 128, generator=torch.Generator().manual_seed(2)).cuda()
    out = []
    for qkv in (row.expand(20, -1), row.expand(20, -1).contiguous()):
        k, v, table, _ = make_cache([30, 9], 2, 64, 16, fill=0.0)
        q = torch.zeros(20, 4, 64, dtype=torch.bfloat16, device="cuda")
        ab.qk_norm_rope(qkv, q, k, v, table, starts([15, 5]), ints([30, 9]), rope)
        out.append((q, k, v))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [30, 1, 70]])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_one_page_table_row_for_several_sequences(hd, q_lens):
    """Sequences of different lengths that read one sequence's pages."""
    k, v, table, _ = make_cache([400], 2, hd, 16)
    lens = ints([400, 130, 399])
    q = noise(sum(q_lens), 8, hd).bfloat16().cuda()
    out = []
    for t in (table.expand(3, -1), table.expand(3, -1).contiguous()):
        o = torch.full_like(q, 5.0)
        ab.paged_attention(q, o, k, v, t, starts(q_lens), lens, max_q_len=max(q_lens))
        out.append(o)
    assert torch.equal(*out) and torch.isfinite(out[0].float()).all()
    # and written through: tokens of three sequences at positions of their own
    pages = []
    for t in (table.expand(3, -1), table.expand(3, -1).contiguous()):
        kk, vv = torch.zeros_like(k), torch.zeros_like(v)
        ab.qk_norm_rope(noise(3, 12 * hd).cuda(), torch.empty_like(q[:3]), kk, vv, t, starts([1, 1, 1]), lens,
                        torch.rand(400, 2 * hd, generator=torch.Generator().manual_seed(2)).cuda())
        pages.append((kk, vv))
    assert torch.equal(pages[0][0], pages[1][0]) and torch.equal(pages[0][1], pages[1][1])
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
