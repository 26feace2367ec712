"""Refusals of the paged-serving entry points that need no GPU: tensors that are
not on one, and calls before anything could be launched."""
import pytest
import torch

import alveare_b200
from alveare_b200 import compact_pages, paged_attention, qk_norm_rope, sample_tokens, update_pages


def _cache():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    i32 = torch.int32
    return k, k.clone(), torch.zeros(1, 4, dtype=i32), torch.tensor([0, 1], dtype=i32), torch.ones(1, dtype=i32)


def test_exported():
    for name in ("qk_norm_rope", "paged_attention", "update_pages", "compact_pages", "sample_tokens", "PagedKVCache"):
        assert hasattr(alveare_b200, name)


@pytest.mark.parametrize("bad", ["cpu", "numpy", "none"])
def test_not_a_cuda_tensor(bad):
    make = {"cpu": lambda t: t, "numpy": lambda t: t.float().numpy(), "none": lambda t: None}[bad]
    k, v, table, start, lens = _cache()
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="q must be a torch CUDA tensor"):
        paged_attention(make(q), q, k, v, table, start, lens, max_q_len=1)
    with pytest.raises(TypeError, match="qkv must be a torch CUDA tensor"):
        qk_norm_rope(make(torch.zeros(1, 8 * 64)), q, k, v, table, start, lens, torch.zeros(8, 128))
    with pytest.raises(TypeError, match="logits must be a torch CUDA tensor"):
        sample_tokens(make(torch.zeros(1, 8)), torch.zeros(1), torch.zeros(1, dtype=torch.int32))
    pool = k[None]
    refs = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(TypeError, match="k_pool must be a torch CUDA tensor"):
        update_pages(make(pool), pool, table, lens, refs)
    with pytest.raises(TypeError, match="k_pool must be a torch CUDA tensor"):
        compact_pages(make(pool), pool, table, refs, table, refs)
