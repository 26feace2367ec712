"""Pools and logits of more than 2^31 elements: pages, rows and page copies
past the offsets that fit 32 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import attention_ref, attention_tol, ints, starts  # noqa: E402

PAGES, NKV, PS, HD = 33000, 8, 64, 128   # 2.16e9 elements: the last pages lie past 2^31


@pytest.fixture(scope="module")
def pool():
    k = torch.empty(PAGES, NKV, PS, HD, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    assert k[-200:].storage_offset() > 2 ** 31
    yield k, v
    del k, v
    torch.cuda.empty_cache()


@pytest.mark.parametrize("q_lens", [[1, 1], [90, 3]])
def test_append_and_attend(pool, q_lens):
    k, v = pool
    kv = [400, 130]
    table = torch.full((2, 8), -1, dtype=torch.int32)
    ids = PAGES - 1 - torch.randperm(200, generator=torch.Generator().manual_seed(1))[:10]
    table[0, :7], table[1, :3] = ids[:7].int(), ids[7:].int()
    table = table.cuda()
    g = torch.Generator().manual_seed(2)
    rope = torch.cat([torch.ones(400, HD), torch.zeros(400, HD)], 1).cuda()   # no rotation
    rows, everything = [], []
    for b, n in enumerate(kv):   # every position is written by the operator itself
        x = torch.randn(n, 10 * NKV // 2, HD, generator=g).bfloat16()   # 24 + 8 + 8 heads
        everything.append(x)
        rows.append((x[:, 24:32].transpose(0, 1).double(), x[:, 32:].transpose(0, 1).double()))
        ab.qk_norm_rope(x.view(n, -1).cuda(), torch.empty(n, 24, HD, dtype=torch.bfloat16, device="cuda"), k, v,
                        table[b:b + 1], starts([n]), ints([n]), rope)
    q = torch.cat([x[n - ql:, :24] for x, n, ql in zip(everything, kv, q_lens)]).cuda()
    out = torch.full_like(q, 7.0)
    ab.paged_attention(q, out, k, v, table, starts(q_lens), ints(kv), max_q_len=max(q_lens))
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    ref, mag = attention_ref(q, rows, q_lens, kv)
    assert (np.abs(out.double().cpu().numpy() - ref) <= attention_tol(ref, mag)).all()


def test_page_copies(pool):
    k, v = (t[None] for t in pool)
    last = PAGES - 1
    for t in (k, v):
        t[0, last] = torch.randn(NKV, PS, HD, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    table, lens, refs = ints([last, -1, -1, -1]).view(2, 2), ints([10, 0]), ints([0] * PAGES)
    refs[last] = 1
    refs[:PAGES - 5] += 1   # so that the free pages are the last ones
    ab.update_pages(k, v, table, lens, refs, fork=ints([0, 1]).view(1, 2), extend=ints([1, 1]).view(1, 2))
    new = int(table[1, 0])
    assert new == PAGES - 5 and int(table[0, 0]) == last
    assert torch.equal(k[0, new], k[0, last]) and torch.equal(v[0, new], v[0, last])
    want = k[0, last].clone()
    refs.zero_()
    refs[last] = 1
    table = ints([last]).view(1, 1)
    ab.compact_pages(k, v, table, refs, table, refs)
    assert int(table) == 0 and int(refs[0]) == 1 and torch.equal(k[0, 0], want)
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)


def test_sampling_rows_past_32_bit_offsets():
    rows, vocab = 4200, 512000
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    pick = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(4)).cuda()
    logits.scatter_(1, pick[:, None], 60.0)
    tok = torch.empty(rows, dtype=torch.int32, device="cuda")
    u = torch.full((rows,), 0.5, device="cuda")
    for kw in (dict(), dict(top_k=1), dict(temperature=0.0), dict(top_p=0.5)):
        ab.sample_tokens(logits, u, tok, **kw)
        assert torch.equal(tok.long(), pick)
