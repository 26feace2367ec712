"""Sampling against the definition: an integer restatement (equal on every
token), the distribution in float64, ties, masks, empty rows, extremes."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402


def draw(logits, u, **kw):
    rows = logits.shape[0]
    tok = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    lp = torch.full((rows,), 7.0, device="cuda")
    ab.sample_tokens(logits, u, tok, lp, **kw)
    return tok.cpu().numpy(), lp.double().cpu().numpy()


def restate(row, u, temp, k, p, min_p):
    """One row, in integers; the weights are the GPU's 32-bit exp."""
    x = row.float()
    if not temp > 0:
        s = torch.where(torch.isnan(x), -math.inf, x)
        return (-1, -math.inf) if s.max() == -math.inf else (int(torch.nonzero(s == s.max())[0]), 0.0)
    s = x / torch.full_like(x, temp)
    s = torch.where(torch.isnan(s), -math.inf, s)
    top = s.max()
    if top == -math.inf:
        return -1, -math.inf
    w = torch.where(s == math.inf, 1.0, 0.0) if top == math.inf else torch.exp(s - top)
    w, s = w.cpu().numpy(), s.cpu().numpy()
    mass = np.floor(w.astype(np.float64) * 2.0 ** 40).astype(np.int64)
    order = np.argsort(-s, kind="stable")
    if 0 < k < order.size:
        order = order[:k]
    if p < 1:
        cum = np.cumsum(mass[order])
        goal = max(1, math.ceil(float(cum[-1]) * float(np.float32(p))))
        order = order[:int(np.searchsorted(cum, goal)) + 1]
    order = np.sort(order[w[order] >= np.float32(min_p)])
    cum = np.cumsum(mass[order])
    total = int(cum[-1])
    goal = min(int(math.floor(float(np.float32(u)) * float(total))), total - 1)
    i = int(np.searchsorted(cum, goal, side="right"))
    return int(order[i]), math.log(mass[order[i]] / total)


def same(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    tok, lp = draw(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    at = lambda v, i: float(v[i]) if isinstance(v, torch.Tensor) else v
    for i in range(logits.shape[0]):
        t, l = restate(logits[i], float(u[i]), at(temperature, i), int(at(top_k, i)), at(top_p, i), at(min_p, i))
        assert tok[i] == t, (i, tok[i], t)
        # the share is an exact ratio; its log is rounded to fp32
        assert l == lp[i] or abs(lp[i] - l) <= 2.0 ** -23 * abs(l) + 1e-12, (i, lp[i], l)


def rand(rows, vocab, dtype=torch.float32, spread=2.5, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(rows, vocab, generator=g)).to(dtype).cuda(), torch.rand(rows, generator=g).cuda()


SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=40, temperature=0.8), dict(top_p=0.9),
            dict(top_p=0.3, temperature=1.7), dict(min_p=0.05), dict(top_k=50, top_p=0.95, min_p=0.02, temperature=0.7),
            dict(top_p=0.0), dict(min_p=1.0), dict(temperature=0.0), dict(top_k=10 ** 6, top_p=2.0), dict(temperature=50.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1025, 32000, 128256, 151937])
@pytest.mark.parametrize("setting", range(len(SETTINGS)))
def test_tokens_match_the_integers(dtype, vocab, setting):
    logits, u = rand(5, vocab, dtype, seed=vocab + setting)
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    same(logits, u, **SETTINGS[setting])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [360449, 400001, 524288])
def test_vocabularies_too_long_to_keep_on_chip(dtype, vocab):
    logits, u = rand(3, vocab, dtype, seed=vocab)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=40, top_p=0.95), dict(top_k=5000, top_p=0.8, min_p=0.001),
               dict(temperature=0.0)):
        same(logits, u, **kw)


@pytest.mark.parametrize("step", [0.0, 0.01, 0.25])
@pytest.mark.parametrize("top_k", [0, 600, 3000])
@pytest.mark.parametrize("top_p", [0.2, 0.7, 0.97])
@pytest.mark.parametrize("min_p", [0.0, 1e-4, 0.03, 0.4])
def test_prefixes_and_floor_together(step, top_k, top_p, min_p):
    """Prefixes that end in ties of any length (logits on a grid), with a floor
    above, inside and below them."""
    logits, u = rand(4, 40000, seed=int(1000 * step) + top_k)
    if step:
        logits = (logits / step).round() * step
    same(logits, u, top_k=top_k, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_keep_the_lowest_indices(dtype):
    logits = torch.zeros(6, 5000, dtype=dtype, device="cuda")
    u = torch.linspace(0, 0.999, 6).cuda()
    for kw in (dict(), dict(top_k=17), dict(top_p=0.01), dict(top_k=2500, top_p=0.5), dict(temperature=0.0)):
        same(logits, u, **kw)
    logits[:, 1000:1010] = 1.0
    logits[:, 4000:] = -1.0
    for kw in (dict(top_k=12), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.5), dict(temperature=0.0)):
        same(logits, u, **kw)


def test_masks_infinities_nan_and_empty_rows():
    logits, u = rand(10, 3000, seed=4)
    logits[0, ::2] = -math.inf
    logits[1] = -math.inf
    logits[2, 7:2990] = float("nan")
    logits[3] = float("nan")
    logits[4, [5, 900]] = math.inf
    logits[5, 1:] = -math.inf
    logits[6] = torch.finfo(torch.float32).min
    logits[7, 100:] = torch.finfo(torch.float32).min
    logits[8, ::3] = 0.0
    logits[8, 1::3] = -0.0
    logits[9] = -1e30
    for kw in (dict(), dict(top_k=5), dict(top_p=0.9), dict(temperature=0.0), dict(top_k=3, top_p=0.5, min_p=0.1)):
        same(logits, u, **kw)
        same(logits.bfloat16(), u, **kw)


def test_per_row_parameters_and_strides():
    wide, u = rand(7, 2000, seed=8)
    logits = wide[:, 3:1704]
    f = lambda *v: torch.tensor(v, device="cuda")
    same(logits, u, temperature=f(0.5, 1.0, 0.0, 2.0, 1e-3, 1.0, 30.0), top_p=f(1.0, 0.5, 0.9, 0.1, 0.99, 0.0, 0.7),
         min_p=f(0.0, 0.1, 0.0, 0.9, 0.0, 0.0, 0.01),
         top_k=torch.tensor([0, 5, 3, -1, 2000, 1701, 100], dtype=torch.int32, device="cuda"))
    same(wide.bfloat16()[:, 1:1500], u, temperature=0.9, top_k=33)


@pytest.mark.parametrize("kw", [dict(temperature=0.8), dict(top_k=6), dict(top_p=0.8), dict(min_p=0.2)])
def test_frequencies_follow_the_distribution(kw):
    """u on an even grid: token i's count is its probability times the grid, to
    within one step at each of its two borders."""
    n = 4096
    row = torch.tensor([0.3, -1.0, 2.0, 1.5, 0.0, 2.0, -3.0, 1.0, 0.7, 1.9, -0.2, 0.1], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tok, lp = draw(row.expand(n, -1).contiguous(), u, **kw)
    x = row.double().cpu().numpy() / kw.get("temperature", 1.0)
    w = np.exp(x - x.max())
    order = np.argsort(-x, kind="stable")
    if "top_k" in kw:
        order = order[:kw["top_k"]]
    if "top_p" in kw:
        cum = np.cumsum(w[order])
        order = order[:int(np.searchsorted(cum, kw["top_p"] * cum[-1])) + 1]
    keep = np.zeros(12)
    keep[order] = 1
    keep *= w >= kw.get("min_p", 0.0)
    prob = w * keep / (w * keep).sum()
    count = np.bincount(tok, minlength=12)
    assert (np.abs(count - prob * n) <= 2).all()
    assert np.allclose(lp, np.log(prob[tok]), rtol=1e-5, atol=1e-6)
    assert (np.diff(tok) >= 0).all()   # index order


def test_same_tokens_every_time_and_in_a_graph():
    logits, u = rand(64, 50000, seed=3)
    a = draw(logits, u, top_p=0.9)
    for _ in range(3):
        b = draw(logits, u, top_p=0.9)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    tok = torch.empty(64, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ab.sample_tokens(logits, u, tok, top_p=0.9)
    graph.replay()
    assert np.array_equal(tok.cpu().numpy(), a[0])


def test_refusals():
    logits, u = rand(3, 100)
    tok = torch.empty(3, dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError):
        ab.sample_tokens(logits.cpu(), u, tok)
    with pytest.raises(TypeError):
        ab.sample_tokens(logits.half(), u, tok)
    with pytest.raises(TypeError):
        ab.sample_tokens(logits, u.double(), tok)
    with pytest.raises(TypeError):
        ab.sample_tokens(logits, u, tok.long())
    with pytest.raises(ValueError):
        ab.sample_tokens(logits, u[:2], tok)
    with pytest.raises(ValueError):
        ab.sample_tokens(logits.t(), u, tok)
    with pytest.raises(TypeError):
        ab.sample_tokens(logits, u, tok, top_k=torch.ones(3, device="cuda"))
    for kw in (dict(temperature=-1.0), dict(top_p=-0.1), dict(min_p=1.5), dict(min_p=float("nan")),
               dict(temperature=float("nan"))):
        with pytest.raises(_lib.AlvError):
            ab.sample_tokens(logits, u, tok, **kw)
    with pytest.raises(_lib.AlvError):
        ab.sample_tokens(torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1], tok[:1])
    ab.sample_tokens(logits[:0], u[:0], tok[:0])
    _lib.context(0).sync_status()
