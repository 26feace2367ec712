"""Steps whose token tensors have more rows than the sequences use (a step
captured for its largest batch and replayed with less): every sequence is
computed, the rows past the last one are left alone, nothing is reported."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import attention_ref, attention_tol, ints, make_cache, starts  # noqa: E402


def noise(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def check(out, q, rows, q_lens, kv_lens, **kw):
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    n = sum(q_lens)
    ref, mag = attention_ref(q[:n], rows, q_lens, kv_lens, **kw)
    got = out.double().cpu().numpy()
    assert (np.abs(got[:n] - ref) <= attention_tol(ref, mag)).all()
    assert (got[n:] == 7).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("batch,cap,now", [
    (8, 8, [3] * 8),                                  # a uniform step, replayed with fewer tokens each
    (8, 8, [8] * 8),
    (8, 64, [1, 64, 1, 0, 2, 1, 1, 3]),               # a few chunks among short ones
    (40, 17, [1] * 39 + [17]),
])
@pytest.mark.parametrize("past", [60, 4000])
def test_replayed_with_other_lengths(hd, batch, cap, now, past):
    nq, nkv, ps = 16, 4, 32
    kv = [past + 7 * b for b in range(batch)]
    k, v, table, rows = make_cache(kv, nkv, hd, ps)
    q = noise(batch * cap, nq, hd).bfloat16().cuda()
    out, lens, st = torch.full_like(q, 7.0), ints(kv), starts([cap] * batch)
    call = lambda: ab.paged_attention(q, out, k, v, table, st, lens, max_q_len=cap)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for q_lens in (now, [cap] * batch):
        st.copy_(starts(q_lens))
        out.fill_(7.0)
        graph.replay()
        check(out, q, rows, q_lens, kv)


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_uniform_looking_batches(window, sinks):
    """batch * max_q_len rows, but the sequences are not all that long."""
    kv = [5000] * 60
    k, v, table, rows = make_cache(kv, 2, 64, 16)
    for q_lens in ([1] * 60, [1, 2] * 30, [0] * 59 + [1], [0] * 60):
        q = noise(60 * 5, 8, 64).bfloat16().cuda()
        out = torch.full_like(q, 7.0)
        ab.paged_attention(q, out, k, v, table, starts(q_lens), ints(kv), max_q_len=5, window=window, sinks=sinks)
        check(out, q, rows, q_lens, kv, window=window, sinks=sinks)


@pytest.mark.parametrize("tokens", [9, 3000])
def test_rows_past_the_last_sequence_are_not_an_error(tokens):
    """Norm + rotation + append leaves them alone, as attention does."""
    k, v, table, _ = make_cache([20, 5], 2, 64, 16, fill=0.0)
    qkv = noise(tokens, 8 * 64).cuda()
    rope = torch.rand(32, 128, generator=torch.Generator().manual_seed(2)).cuda()
    got = []
    for x, n in ((qkv, tokens), (qkv[:5], 5)):
        kk, vv = k.clone(), v.clone()
        out = torch.full((n, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        ab.qk_norm_rope(x, out, kk, vv, table, starts([3, 2]), ints([20, 5]), rope)
        _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
        got.append((out, kk, vv))
    (a, ka, va), (b, kb, vb) = got
    assert torch.equal(a[:5], b) and (a[5:] == 7).all()
    assert torch.equal(ka, kb) and torch.equal(va, vb)
    # the first sequence may start past row 0
    out = torch.full((tokens, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ab.qk_norm_rope(qkv, out, k.clone(), v.clone(), table, ints([2, 5, 7]), ints([20, 5]), rope)
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    assert (out[:2] == 7).all() and (out[7:] == 7).all() and (out[2:7] != 7).any(-1).all()
    # starts that are out of order or past the rows still are
    for st in ([0, 3, 2], [0, 3, tokens + 1], [-1, 3, 5]):
        ab.qk_norm_rope(qkv, out, k.clone(), v.clone(), table, ints(st), ints([20, 5]), rope)
        with pytest.raises(_lib.AlvError):
            _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
