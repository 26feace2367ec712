"""Paged attention against the formula in float64: head sizes and groups,
lengths from one position to thousands, pages that end inside a tile, windows
and first tokens, rows that see nothing, strides, and values that are not
finite where they must not matter."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import attention_ref, attention_tol, ints, make_cache, starts  # noqa: E402


def check(q_lens, kv_lens, nq, nkv, hd, ps, *, window=0, sinks=0, scale=None, seed=1, layout="plain", strided=False,
          max_q_len=None):
    k, v, table, rows = make_cache(kv_lens, nkv, hd, ps, seed=seed, layout=layout)
    tokens = sum(q_lens)
    g = torch.Generator().manual_seed(seed + 100)
    q = (2 * torch.randn(tokens, nq, hd, generator=g)).bfloat16().cuda()
    out = torch.full_like(q, 7.0)
    if strided:  # q inside a wider [q | k | v] row, out head-major
        wide = torch.zeros(tokens, nq + 2 * nkv, hd, dtype=torch.bfloat16, device="cuda")
        wide[:, :nq] = q
        q = wide[:, :nq]
        out = torch.full((nq, tokens, hd), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    ab.paged_attention(q, out, k, v, table, starts(q_lens), ints(kv_lens), max_q_len=max_q_len or max(q_lens),
                       window=window, sinks=sinks, scale=scale)
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    ref, mag = attention_ref(q, rows, q_lens, kv_lens, window=window, sinks=sinks, scale=scale)
    got = out.double().cpu().numpy()
    bad = ~(np.abs(got - ref) <= attention_tol(ref, mag))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.nanmax(np.abs(got - ref))))


HEADS = [(1, 1), (8, 8), (4, 1), (6, 2), (10, 2), (14, 2), (32, 8), (16, 1), (40, 2)]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nq,nkv", HEADS)
def test_single_tokens(hd, nq, nkv):
    check([1] * 5, [1, 2, 17, 130, 700], nq, nkv, hd, 16)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ps", [16, 32, 48, 64, 128, 256])
def test_page_sizes(hd, ps):
    check([1, 1, 1], [ps - 1, ps, 3 * ps + 1], 8, 2, hd, ps)
    check([40, 3], [ps + 40, 5 * ps + 7], 8, 2, hd, ps)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nq,nkv", [(4, 4), (8, 2), (6, 2), (10, 2), (16, 1), (20, 1)])
def test_chunks(hd, nq, nkv):
    check([1, 33, 64, 129, 5], [1, 33, 200, 129, 1025], nq, nkv, hd, 32)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (100, 4), (128, 128), (129, 17), (4000, 4), (64, 5000)])
def test_window_and_sinks(hd, window, sinks):
    check([1, 1, 1, 1], [1, 90, 300, 1111], 8, 2, hd, 16, window=window, sinks=sinks)
    check([70, 1, 200], [700, 300, 200], 8, 2, hd, 32, window=window, sinks=sinks)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_long_single_token(hd):
    check([1], [20001], 4, 1, hd, 64)
    check([2, 1], [9000, 3], 4, 2, hd, 16, window=3000, sinks=40)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_few_rows_over_a_long_past(hd):
    check([9], [6000], 16, 2, hd, 64)
    check([70, 70], [3000, 71], 8, 2, hd, 16)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_long_chunk(hd):
    check([700], [1500], 4, 2, hd, 64)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_empty_sequences_and_rows(hd):
    # no new tokens; more new tokens than positions: the first ones see nothing
    check([0, 3, 0, 2, 40], [5, 1, 0, 0, 20], 8, 2, hd, 16)


@pytest.mark.parametrize("layout", ["pair", "heads"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_strides(layout, hd):
    check([1, 1], [50, 333], 8, 2, hd, 16, layout=layout, strided=True)
    check([65, 20], [165, 333], 8, 2, hd, 16, layout=layout, strided=True)


def test_scale_and_slack_in_max_q_len():
    check([3, 1, 8], [30, 10, 500], 8, 2, 64, 16, scale=0.3)
    check([3, 1, 8], [30, 10, 500], 8, 2, 64, 16, scale=-0.05, max_q_len=12)
    check([1, 1, 1], [30, 10, 500], 8, 2, 128, 16, scale=0.0, max_q_len=3)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_sequences(hd):
    r = np.random.default_rng(5)
    kv = r.integers(1, 400, 300)
    check([1] * 300, kv.tolist(), 2, 1, hd, 16)
    q = r.integers(0, 30, 60)
    check(q.tolist(), (q + r.integers(0, 100, 60)).tolist(), 4, 1, hd, 16)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("singles, window, sinks", [(30, 0, 0), (300, 0, 0), (40, 60, 3), (400, 60, 3)])
def test_few_and_many_single_tokens_beside_chunks(hd, singles, window, sinks):
    """A few single tokens beside chunks are taken by the chunks' kernel, many by
    the row blocks'."""
    r = np.random.default_rng(singles)
    q = [1] * singles + [70, 0, 3, 129]
    kv = r.integers(1, 400, singles).tolist() + [300, 0, 500, 129]
    at = r.permutation(len(q))
    check([q[i] for i in at], [kv[i] for i in at], 4, 2, hd, 16, window=window, sinks=sinks)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q_len", [2, 6, 200])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_unseen_values_do_not_matter(hd, q_len, value):
    """A k or v row that a token does not see holds NaN or infinity: the token's
    output is what it is without it (the tokens that see it are not checked)."""
    n, nq, nkv, ps, window = q_len + 300, 4, 2, 32, 150
    k, v, table, rows = make_cache([n], nkv, hd, ps, seed=9)
    q = torch.randn(q_len, nq, hd, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    # a position in the chunk's middle (seen by later tokens only), and one
    # that leaves the window in the middle of the chunk
    marks = [n - q_len + q_len // 2, n - q_len + q_len // 2 - window]
    for j in marks:
        page = int(table[0, j // ps])
        k[page, :, j % ps] = value
        v[page, :, j % ps, ::3] = value
    out = torch.empty_like(q)
    ab.paged_attention(q, out, k, v, table, starts([q_len]), ints([n]), max_q_len=q_len, window=window)
    ref, mag = attention_ref(q, rows, [q_len], [n], window=window)
    got = out.double().cpu().numpy()
    checked = 0
    for i in range(q_len):
        pos = n - q_len + i
        if not any(pos - window < j <= pos for j in marks):
            assert (np.abs(got[i] - ref[i]) <= attention_tol(ref[i], mag[i])).all(), i
            checked += 1
    seen_from = marks[0] - (n - q_len)
    assert not np.isfinite(got[seen_from]).all()  # a token that sees it
    if q_len > 2:
        assert checked >= 0


def test_repeats_bit_for_bit():
    k, v, table, _ = make_cache([5000, 70, 900], 2, 128, 16)
    for q_lens in ([1, 1, 1], [100, 20, 300]):
        q = torch.randn(sum(q_lens), 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
        outs = []
        for _ in range(3):
            out = torch.empty_like(q)
            ab.paged_attention(q, out, k, v, table, starts(q_lens), ints([5000, 70, 900]), max_q_len=max(q_lens))
            outs.append(out)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_runs_on_the_current_stream_and_in_a_graph():
    kv = [300, 1000]
    k, v, table, rows = make_cache(kv, 2, 64, 16)
    q = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    out, lens, st = torch.zeros_like(q), ints(kv), starts([1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ab.paged_attention(q, out, k, v, table, st, lens, max_q_len=1)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ab.paged_attention(q, out, k, v, table, st, lens, max_q_len=1)
    lens.copy_(ints([200, 999]))   # read when the graph runs
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    short = [(a[:, :n], b[:, :n]) for (a, b), n in zip(rows, [200, 999])]
    ref, mag = attention_ref(q, short, [1, 1], [200, 999])
    assert (np.abs(out.double().cpu().numpy() - ref) <= attention_tol(ref, mag)).all()


def test_bad_indices_are_skipped_and_reported():
    k, v, table, rows = make_cache([100, 100], 2, 64, 16)
    q = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    ctx, s = _lib.context(0), torch.cuda.current_stream().cuda_stream
    bad_table = table.clone()
    bad_table[0, 2] = 10 ** 6
    for tab, st, lens in ((bad_table, starts([1, 1]), ints([100, 100])),
                          (table, ints([0, 5, 2]), ints([100, 100])),
                          (table, starts([1, 1]), ints([100, 10 ** 6])),
                          (table, starts([1, 1]), ints([-4, 100]))):
        out = torch.zeros_like(q)
        ab.paged_attention(q, out, k, v, tab, st, lens, max_q_len=1)
        with pytest.raises(_lib.AlvError) as e:
            ctx.sync_status(s)
        assert e.value.code == 1
        ctx.sync_status(s)  # reported once
    # the good sequence of the first call is right all the same
    out = torch.zeros_like(q)
    ab.paged_attention(q, out, k, v, bad_table, starts([1, 1]), ints([100, 100]), max_q_len=1)
    with pytest.raises(_lib.AlvError):
        ctx.sync_status(s)
    ref, mag = attention_ref(q, rows, [1, 1], [100, 100])
    assert (np.abs(out.double().cpu().numpy() - ref) <= attention_tol(ref, mag))[1].all()


def test_refusals():
    k, v, table, _ = make_cache([100], 2, 64, 16, fill=0.0)
    q = torch.zeros(1, 8, 64, dtype=torch.bfloat16, device="cuda")
    a = dict(max_q_len=1)
    st, n = starts([1]), ints([100])
    ok = (q, torch.empty_like(q), k, v, table, st, n)

    def call(i, x, **kw):
        args = list(ok)
        args[i] = x
        ab.paged_attention(*args, **{**a, **kw})

    with pytest.raises(TypeError):
        call(0, q.cpu())
    with pytest.raises(TypeError):
        call(0, q.float())
    with pytest.raises(ValueError):
        call(0, q[0])
    with pytest.raises(ValueError):
        call(1, torch.empty(1, 4, 64, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(TypeError):
        call(2, k.float())
    with pytest.raises(ValueError):
        call(3, v[:, :, ::2])
    with pytest.raises(TypeError):
        call(4, table.long())
    with pytest.raises(ValueError):
        call(5, ints([0, 1, 1]))
    with pytest.raises(ValueError):
        call(0, q, window=-1)
    with pytest.raises(_lib.AlvError):   # heads not a multiple of kv heads
        q3 = q[:, :3]
        ab.paged_attention(q3, torch.empty_like(q3), k, v, table, st, n, max_q_len=1)
    with pytest.raises(_lib.AlvError):   # page size
        ab.paged_attention(q, torch.empty_like(q), k[:, :, :8].contiguous(), v[:, :, :8].contiguous(), table, st, n,
                           max_q_len=1)
    with pytest.raises(_lib.AlvError):   # alignment
        buf = torch.zeros(8 * 64 + 8, dtype=torch.bfloat16, device="cuda")
        call(0, buf[1:1 + 512].view(1, 8, 64))
    with pytest.raises(_lib.AlvError):   # head size
        k32 = torch.zeros(4, 2, 16, 32, dtype=torch.bfloat16, device="cuda")
        q32 = torch.zeros(1, 8, 32, dtype=torch.bfloat16, device="cuda")
        ab.paged_attention(q32, torch.empty_like(q32), k32, k32, table, st, n, max_q_len=1)
    with pytest.raises(_lib.AlvError):
        call(0, q, scale=float("nan"))
    _lib.context(0).sync_status()
