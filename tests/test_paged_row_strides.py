"""What the paged-serving wrappers hand to the library for rows that overlap
(one row broadcast over many): the tensor's own row stride, never one that
reaches past its memory.  The library is replaced by a recorder, so this needs
no GPU."""
import types

import pytest

torch = pytest.importorskip("torch")

from alveare_b200 import paged  # noqa: E402


@pytest.fixture
def calls(monkeypatch):
    got = {}

    def entry(name):
        def call(ctx, *args):
            got[name] = args
            return 0
        return call

    names = ("alv_sample", "alv_qk_norm_rope", "alv_paged_attention", "alv_pages_update", "alv_pages_compact")
    ctx = types.SimpleNamespace(lib=types.SimpleNamespace(**{n: entry(n) for n in names}), ptr=None)
    monkeypatch.setattr(paged, "_need", lambda *a: None)
    monkeypatch.setattr(paged, "_device", lambda *a: 0)
    monkeypatch.setattr(paged, "_stream", lambda d: 0)
    monkeypatch.setattr(paged, "context", lambda d: ctx)
    return got


I32 = torch.int32


def cache(batch, width=4):
    k = torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16)
    start = torch.arange(batch + 1, dtype=I32)
    return k, torch.zeros_like(k), start, torch.full((batch,), 5, dtype=I32)


def reach(stride, rows, cols):
    """Elements from the first to one past the last that rows of this stride touch."""
    return (rows - 1) * stride + cols


@pytest.mark.parametrize("logits", [torch.zeros(1, 100).expand(64, -1), torch.zeros(130).as_strided((4, 100), (10, 1)),
                                    torch.zeros(4, 120)[:, :100], torch.zeros(100).as_strided((1, 100), (3, 1))])
def test_logits(calls, logits):
    rows = logits.shape[0]
    paged.sample_tokens(logits, torch.zeros(rows), torch.zeros(rows, dtype=I32))
    stride = paged._SAMPLE.unpack(calls["alv_sample"][0])[1]
    assert rows == 1 or stride == logits.stride(0)
    assert reach(stride, rows, 100) <= logits.untyped_storage().nbytes() // 4


@pytest.mark.parametrize("qkv", [torch.zeros(1, 512).expand(6, -1), torch.zeros(1000).as_strided((6, 512), (8, 1)),
                                 torch.zeros(6, 520)[:, :512], torch.zeros(512).as_strided((1, 512), (3, 1))])
def test_qkv(calls, qkv):
    n = qkv.shape[0]
    k, v, start, lens = cache(n)
    paged.qk_norm_rope(qkv, torch.zeros(n, 4, 64, dtype=torch.bfloat16), k, v, torch.zeros(n, 4, dtype=I32), start, lens,
                       torch.zeros(8, 128))
    stride = paged._NORM_ROPE.unpack(calls["alv_qk_norm_rope"][1])[1]
    assert n == 1 or stride == qkv.stride(0)
    assert stride % 8 == 0 and reach(stride, n, 512) <= qkv.untyped_storage().nbytes() // 4


@pytest.mark.parametrize("table", [torch.zeros(1, 4, dtype=I32).expand(6, -1), torch.zeros(9, dtype=I32).unfold(0, 4, 1),
                                   torch.zeros(6, 9, dtype=I32)[:, :4], torch.zeros(4, dtype=I32).as_strided((1, 4), (2, 1))])
def test_page_table(calls, table):
    n = table.shape[0]
    k, v, start, lens = cache(n)
    q = torch.zeros(n, 4, 64, dtype=torch.bfloat16)
    paged.paged_attention(q, q.clone(), k, v, table, start, lens, max_q_len=1)
    paged.qk_norm_rope(torch.zeros(n, 512), q.clone(), k, v, table, start, lens, torch.zeros(8, 128))
    for name in ("alv_paged_attention", "alv_qk_norm_rope"):
        stride = paged._PAGED.unpack(calls[name][0])[10]
        assert n == 1 or stride == table.stride(0)
        assert reach(stride, n, 4) <= table.untyped_storage().nbytes() // 4


def test_a_pool_s_own_table_must_not_overlap(calls):
    k = torch.zeros(1, 8, 2, 16, 64, dtype=torch.bfloat16)
    refs = torch.zeros(8, dtype=I32)
    for table in (torch.zeros(1, 4, dtype=I32).expand(6, -1), torch.zeros(9, dtype=I32).unfold(0, 4, 1)):
        with pytest.raises(ValueError, match="overlap"):
            paged.update_pages(k, k.clone(), table, torch.zeros(6, dtype=I32), refs)
        with pytest.raises(ValueError, match="overlap"):
            paged.compact_pages(k, k.clone(), table, refs, torch.zeros(6, 4, dtype=I32), refs)
    one = torch.zeros(4, dtype=I32).as_strided((1, 4), (2, 1))
    paged.update_pages(k, k.clone(), one, torch.zeros(1, dtype=I32), refs)
    assert paged._PAGES.unpack(calls["alv_pages_update"][0])[8] >= 4
