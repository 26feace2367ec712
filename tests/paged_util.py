"""Inputs and 64-bit references for the paged-serving tests."""
import math

import numpy as np
import torch

NAN = float("nan")


def make_cache(kv_lens, nkv, hd, ps, *, seed=0, spare=2, fill=NAN, layout="plain", width_extra=1):
    """k, v pages (positions past each length hold `fill`), the page table and
    the sequences' contiguous k, v in float64.  layout "pair": k and v share one
    allocation, "heads": pages stored position-major (strided heads)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // ps) for n in kv_lens]
    pool = sum(need) + spare
    ids = torch.randperm(pool, generator=g)
    width = max(need + [1]) + width_extra
    table = torch.full((len(kv_lens), width), -1, dtype=torch.int32)
    if layout == "pair":
        both = torch.full((pool, 2, nkv, ps, hd), fill, dtype=torch.bfloat16, device="cuda")
        k, v = both[:, 0], both[:, 1]
    elif layout == "heads":
        k = torch.full((pool, ps, nkv, hd), fill, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        v = torch.full((pool, ps, nkv, hd), fill, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    else:
        k = torch.full((pool, nkv, ps, hd), fill, dtype=torch.bfloat16, device="cuda")
        v = torch.full((pool, nkv, ps, hd), fill, dtype=torch.bfloat16, device="cuda")
    rows, at = [], 0
    for b, n in enumerate(kv_lens):
        pages = ids[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = pages.int()
        kk = torch.randn(nkv, n, hd, generator=g).bfloat16()
        vv = torch.randn(nkv, n, hd, generator=g).bfloat16()
        for i, p in enumerate(pages.tolist()):
            m = min(ps, n - i * ps)
            k[p, :, :m] = kk[:, i * ps:i * ps + m].cuda()
            v[p, :, :m] = vv[:, i * ps:i * ps + m].cuda()
        rows.append((kk.double(), vv.double()))
    return k, v, table.cuda(), rows


def starts(q_lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32).cuda()


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32).cuda()


def attention_ref(q, rows, q_lens, kv_lens, *, window=0, sinks=0, scale=None):
    """o and sum_j p_j |v_j| of every token and head, in float64 (numpy)."""
    q = q.double().cpu().numpy()
    tokens, nq, hd = q.shape
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    t = 0
    for (k, v), ql, n in zip(rows, q_lens, kv_lens):
        k, v = k.numpy(), v.numpy()
        g = nq // k.shape[0]
        j = np.arange(n)
        for i in range(ql):
            pos = n - ql + i
            see = j <= pos
            if window:
                see &= (j > pos - window) | (j < sinks)
            if see.any():
                for h in range(k.shape[0]):
                    s = (q[t + i, h * g:(h + 1) * g] @ k[h][see].T) * scale
                    p = np.exp(s - s.max(1, keepdims=True))
                    p /= p.sum(1, keepdims=True)
                    out[t + i, h * g:(h + 1) * g] = p @ v[h][see]
                    mag[t + i, h * g:(h + 1) * g] = p @ np.abs(v[h][see])
        t += ql
    return out, mag


# Output and p are each rounded to bf16 (8 significant bits: 2^-8 relative), so
# |o - ref| <= 2^-8 |o| + 2^-8 sum p |v|; a further 1/16 of that for the fp32
# scores (|s| <= 40 at these inputs: error below 2^-14) and the 2-ulp
# exponential.
def attention_tol(ref, mag):
    return 2.0 ** -8 * (1 + 1 / 16) * (np.abs(ref) + mag) + 1e-30
