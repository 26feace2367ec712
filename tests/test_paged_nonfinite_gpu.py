"""Attention where cached values are not finite: what a token sees of them
gives what the formula gives, what it does not see changes nothing."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import attention_ref, attention_tol, ints, make_cache, starts  # noqa: E402

NAN, INF = float("nan"), float("inf")


def put(pages, table, rows, side, b, j, ps, value, dims=slice(None)):
    """Position j of sequence b, in the pages and in the reference's copy."""
    pages[int(table[b, j // ps]), :, j % ps, dims] = value
    rows[b][side][:, j, dims] = value


def queries(tokens, nq, hd, seed=1):
    return torch.randn(tokens, nq, hd, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


def run(q, k, v, table, q_lens, kv_lens, **kw):
    out = torch.full_like(q, 7.0)
    ab.paged_attention(q, out, k, v, table, starts(q_lens), ints(kv_lens), max_q_len=max(q_lens), **kw)
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    return out.double().cpu().numpy()


def same(got, ref, mag):
    """NaN and infinities where the formula has them, the rest within tolerance."""
    assert np.array_equal(np.isnan(got), np.isnan(ref)), np.argwhere(np.isnan(got) != np.isnan(ref))[:4].tolist()
    inf = np.isinf(ref)
    assert np.array_equal(got[inf], ref[inf]) and not np.isinf(got[~inf]).any()
    fin = np.isfinite(ref)
    assert (np.abs(got[fin] - ref[fin]) <= attention_tol(ref[fin], mag[fin])).all()


Q_LENS = [1, 3, 40, 200]  # row blocks, row blocks of several tokens, one and more query tiles


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q_len", Q_LENS)
def test_a_nan_key_that_every_token_sees(hd, q_len):
    n, ps = 900, 32
    for j in list(range(256, 264)) + [300, 415]:
        k, v, table, rows = make_cache([n], 2, hd, ps, seed=j)
        page = int(table[0, j // ps])
        k[page, 0, j % ps, 5] = NAN   # one kv head: the other's query heads are as ever
        rows[0][0][0, j, 5] = NAN
        q = queries(q_len, 8, hd)
        ref, mag = attention_ref(q, rows, [q_len], [n])
        assert np.isnan(ref[:, :4]).all() and not np.isnan(ref[:, 4:]).any()
        same(run(q, k, v, table, [q_len], [n]), ref, mag)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q_len", Q_LENS)
@pytest.mark.parametrize("value", [INF, -INF])
def test_infinite_scores(hd, q_len, value):
    """A score of +inf leaves nothing defined, one of -inf a weight of zero."""
    n, ps = 700, 16
    for j in [128, 134, 263, n - 1]:
        k, v, table, rows = make_cache([n], 2, hd, ps, seed=j)
        put(k, table, rows, 0, 0, j, ps, value, 0)
        q = queries(q_len, 8, hd)
        q[:, :, 0] = q[:, :, 0].abs() + 0.5
        ref, mag = attention_ref(q, rows, [q_len], [n])
        same(run(q, k, v, table, [q_len], [n]), ref, mag)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_many_chunks_with_keys_that_are_not_finite(hd, value):
    """As above in more chunks than there are SMs, most of them one CTA's alone;
    the marked position of chunk b is 100 + b."""
    batch, q_len, n, ps = 130, 40, 300, 32
    k, v, table, rows = make_cache([n] * batch, 4, hd, ps)
    for b in range(batch):
        put(k, table, rows, 0, b, 100 + b, ps, value, 0)
    q = queries(q_len * batch, 16, hd)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    ref, mag = attention_ref(q, rows, [q_len] * batch, [n] * batch)
    same(run(q, k, v, table, [q_len] * batch, [n] * batch), ref, mag)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q_len", [1, 2, 30])
def test_nothing_but_scores_of_minus_infinity(hd, q_len):
    """Undefined, unlike a row that sees no position, which gives zeros."""
    n, ps = 40, 16
    for kv in (n, q_len - 1):
        if kv == 0:
            continue
        k, v, table, rows = make_cache([kv, n], 2, hd, ps)
        for j in range(kv):
            put(k, table, rows, 0, 0, j, ps, -INF, 3)
        q = queries(q_len + 2, 8, hd)
        q[:, :, 3] = 1.0
        ref, mag = attention_ref(q, rows, [q_len, 2], [kv, n])
        assert np.isnan(ref[max(0, q_len - kv):q_len]).all() and np.isfinite(ref[q_len:]).all()
        same(run(q, k, v, table, [q_len, 2], [kv, n]), ref, mag)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_short_chunks_with_infinite_values(hd):
    """Chunks of one and of two query tiles in turns, each with an infinite value
    that its later tokens see, in more items than there are CTAs."""
    r = np.random.default_rng(hd)
    q_lens = [int(x) for x in np.where(np.arange(200) % 5 == 0, r.integers(33, 64, 200), r.integers(5, 30, 200))]
    kv = [n + int(r.integers(0, 150)) for n in q_lens]
    k, v, table, rows = make_cache(kv, 2, hd, 16)
    for b, (ql, n) in enumerate(zip(q_lens, kv)):
        if b % 3:
            put(v, table, rows, 1, b, n - ql + ql // 2, 16, INF, slice(b % 7, hd, 11))
    q = queries(sum(q_lens), 8, hd)
    ref, mag = attention_ref(q, rows, q_lens, kv)
    same(run(q, k, v, table, q_lens, kv), ref, mag)


# (new tokens, positions, window, first tokens, marked position relative to the first new token)
SEEN_BY_SOME = [
    (6, 306, 0, 0, 3), (6, 306, 150, 0, 2), (6, 306, 150, 0, 3 - 150), (2, 302, 150, 4, 1 - 150),
    (40, 340, 0, 0, 20), (40, 340, 100, 4, 15 - 100), (40, 340, 100, 0, 39),
    (200, 500, 0, 0, 100), (200, 500, 150, 0, 30), (200, 500, 150, 17, 64 - 150), (200, 500, 150, 0, 150 - 150),
    (100, 6000, 0, 0, 50), (100, 6000, 2000, 0, 60 - 2000), (600, 600, 0, 0, 0), (600, 600, 130, 9, 300),
]


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(SEEN_BY_SOME)))
@pytest.mark.parametrize("side,value", [("k", NAN), ("k", INF), ("v", NAN), ("v", INF), ("v", -INF)])
def test_a_position_that_only_some_tokens_see(hd, case, side, value):
    """The tokens that see it get the formula's NaN or infinities, in the dims
    that have them, the others what they would get without it."""
    q_len, n, window, sinks, mark = SEEN_BY_SOME[case]
    j, ps = n - q_len + mark, 16
    k, v, table, rows = make_cache([n], 2, hd, ps, seed=case)
    if side == "k":
        put(k, table, rows, 0, 0, j, ps, value, 0)
    else:
        put(v, table, rows, 1, 0, j, ps, value, slice(0, hd, 3))
        put(v, table, rows, 1, 0, j, ps, -value, slice(1, hd, 3))
    q = queries(q_len, 8, hd, seed=case)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    ref, mag = attention_ref(q, rows, [q_len], [n], window=window, sinks=sinks)
    pos = np.arange(n - q_len, n)
    see = (j <= pos) & ((window == 0) | (j > pos - window) | (j < sinks))
    assert case == 13 or 0 < see.sum() < q_len       # (case 13: position 0 of a whole prompt)
    assert np.isfinite(ref[~see]).all() and not np.isfinite(ref[see]).all(-1).any()
    same(run(q, k, v, table, [q_len], [n], window=window, sinks=sinks), ref, mag)
