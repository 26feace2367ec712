"""Per-head norm + rotation + append against the formula in float64."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import ints, make_cache, starts  # noqa: E402


def table_for(n, rot, dtype):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.cos(), ang.sin(), ang.sin()], 1).to(dtype).cuda()


def reference(x, pos, rope, rot, w, eps):
    """x (tokens, heads, hd) float64; the result and the size of what was added."""
    hd = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    half = rot // 2
    c, s = rope[pos, None, :half], rope[pos, None, rot:rot + half]
    y, mag = x.copy(), np.abs(x)
    a, b = x[..., :half], x[..., half:rot]
    y[..., :half], y[..., half:rot] = a * c - b * s, b * c + a * s
    mag[..., :half], mag[..., half:rot] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    assert hd == y.shape[-1]
    return y, mag


def close(got, ref, mag):
    # one rounding to bf16 (2^-8 relative), fp32 before it: the norm and the
    # rotation are under 300 roundings of 2^-24, mostly of the norm's sum: 2^-18
    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -15 * mag + 1e-30).all()


@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 16), (128, 128), (128, 64), (256, 256), (256, 128), (128, 48)])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (8, 2), (5, 5), (32, 8), (7, 1)])
@pytest.mark.parametrize("norm", [0, 1])
@pytest.mark.parametrize("xdt,rdt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
def test_against_the_formula(hd, rot, nq, nkv, norm, xdt, rdt):
    q_lens, kv_lens, ps = [1, 0, 19, 33, 1], [1, 4, 70, 33, 50], 16
    layout = "pair" if nq == 8 else "heads" if nq == 5 else "plain"
    k, v, table, rows = make_cache(kv_lens, nkv, hd, ps, seed=3, fill=0.0, layout=layout)
    k0, v0 = k.clone(), v.clone()
    tokens = sum(q_lens)
    g = torch.Generator().manual_seed(hd + rot)
    qkv = torch.randn(tokens, (nq + 2 * nkv) * hd + 16, generator=g).to(xdt).cuda()[:, :(nq + 2 * nkv) * hd]
    qw = (1 + 0.3 * torch.randn(hd, generator=g)).cuda() if norm else None
    kw = (1 + 0.3 * torch.randn(hd, generator=g)).cuda() if norm else None
    rope = table_for(80, rot, rdt)
    out = torch.full((tokens, nq, hd), 9.0, dtype=torch.bfloat16, device="cuda")
    ab.qk_norm_rope(qkv, out, k, v, table, starts(q_lens), ints(kv_lens), rope, q_weight=qw, k_weight=kw, eps=1e-5)
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    pos = np.concatenate([np.arange(n - q, n) for q, n in zip(q_lens, kv_lens)])
    seq = np.concatenate([np.full(q, b) for b, q in enumerate(q_lens)])
    x = qkv.double().cpu().numpy().reshape(tokens, nq + 2 * nkv, hd)
    tab = rope.double().cpu().numpy()
    f = lambda w: None if w is None else w.double().cpu().numpy()
    close(out.double().cpu().numpy(), *reference(x[:, :nq], pos, tab, rot, f(qw), 1e-5))
    page = table.cpu().numpy()[seq, pos // ps]
    for cache, before, part, w in ((k, k0, x[:, nq:nq + nkv], kw), (v, v0, x[:, nq + nkv:], None)):
        c = cache.double().cpu().numpy()
        if cache is v:
            close(c[page, :, pos % ps], part, np.abs(part))
        else:
            close(c[page, :, pos % ps], *reference(part, pos, tab, rot, f(w), 1e-5))
        # nothing else in the cache changed
        kept = before.clone()
        kept[torch.tensor(page).cuda().long(), :, torch.tensor(pos % ps).cuda()] = \
            cache[torch.tensor(page).cuda().long(), :, torch.tensor(pos % ps).cuda()]
        assert torch.equal(kept, cache)


def test_zero_rows_and_large_values():
    """A head of zeros stays zeros (eps keeps the norm finite); large fp32 heads stay finite."""
    k, v, table, _ = make_cache([2], 1, 64, 16, fill=0.0)
    qkv = torch.zeros(2, 3 * 64, device="cuda")
    qkv[1] = 1e15
    out = torch.empty(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, device="cuda")
    ab.qk_norm_rope(qkv, out, k, v, table, starts([2]), ints([2]), table_for(4, 64, torch.float32), q_weight=w, k_weight=w)
    assert torch.equal(out[0], torch.zeros_like(out[0]))
    assert torch.isfinite(out[1].float()).all() and float(out[1].float().abs().max()) < 2


def test_many_sequences_find_their_tokens():
    r = np.random.default_rng(1)
    q = r.integers(0, 4, 333)
    kv = q + r.integers(0, 30, 333)
    k, v, table, _ = make_cache(kv.tolist(), 1, 64, 16, fill=0.0)
    tokens = int(q.sum())
    qkv = torch.randn(tokens, 192, generator=torch.Generator().manual_seed(2)).cuda()
    out = torch.empty(tokens, 1, 64, dtype=torch.bfloat16, device="cuda")
    rope = table_for(64, 64, torch.float32)
    ab.qk_norm_rope(qkv, out, k, v, table, starts(q), ints(kv), rope)
    pos = np.concatenate([np.arange(n - m, n) for m, n in zip(q, kv)])
    ref, mag = reference(qkv.double().cpu().numpy().reshape(tokens, 3, 64)[:, :1], pos, rope.double().cpu().numpy(), 64,
                         None, 0)
    close(out.double().cpu().numpy(), ref, mag)


def test_bad_positions_are_skipped_and_reported():
    k, v, table, _ = make_cache([5, 20], 1, 64, 16, fill=0.0)
    qkv = torch.ones(2, 192, device="cuda")
    out = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    rope = table_for(10, 64, torch.float32)   # position 19 is past it
    ab.qk_norm_rope(qkv, out, k, v, table, starts([1, 1]), ints([5, 20]), rope)
    with pytest.raises(_lib.AlvError):
        _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    assert float(out[0].float().abs().sum()) > 0 and float(out[1].float().abs().sum()) == 0


def test_refusals():
    k, v, table, _ = make_cache([5], 1, 64, 16, fill=0.0)
    qkv = torch.ones(1, 192, device="cuda")
    out = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    rope = table_for(10, 64, torch.float32)
    st, n = starts([1]), ints([5])
    with pytest.raises(TypeError):
        ab.qk_norm_rope(qkv.cpu(), out, k, v, table, st, n, rope)
    with pytest.raises(TypeError):
        ab.qk_norm_rope(qkv.half(), out, k, v, table, st, n, rope)
    with pytest.raises(ValueError):
        ab.qk_norm_rope(qkv[:, :128], out, k, v, table, st, n, rope)
    with pytest.raises(TypeError):
        ab.qk_norm_rope(qkv, out.float(), k, v, table, st, n, rope)
    with pytest.raises(ValueError):
        ab.qk_norm_rope(qkv, out, k, v, table, st, n, rope, q_weight=torch.ones(32, device="cuda"))
    with pytest.raises(_lib.AlvError):
        ab.qk_norm_rope(qkv, out, k, v, table, st, n, table_for(10, 8, torch.float32))
    with pytest.raises(_lib.AlvError):
        ab.qk_norm_rope(qkv, out, k, v, table, st, n, table_for(10, 128, torch.float32))
    with pytest.raises(_lib.AlvError):
        ab.qk_norm_rope(qkv, out, k, v, table, st, n, rope, eps=float("nan"))
    ab.qk_norm_rope(qkv[:0], out[:0], k, v, table, ints([0, 0]), n, rope)  # no tokens: nothing to do
    _lib.context(0).sync_status()
