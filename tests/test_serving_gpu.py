"""PagedLlama (ragged batches over a paged cache) against the CPU oracle and
against itself: chunking, batching, forking and compaction change nothing that
matters."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from alveare_b200 import _lib  # noqa: E402
from alveare_b200.llama import LlamaConfig  # noqa: E402
from alveare_b200.serving import PagedLlama  # noqa: E402
from oracle import llama  # noqa: E402

LOGIT_TOL = 2e-2   # normwise, as the single-sequence decoder's tests


@pytest.fixture(scope="module")
def small():
    cfg = llama.Config(hidden=256, intermediate=512, heads=4, kv_heads=2, head_dim=64, layers=2, vocab=1000,
                       vocab_padded=1024, max_seq=128)
    w, _ = llama.synthetic_weights(cfg, seed=3)
    return cfg, w


def build(cfg, w, **kw):
    c = LlamaConfig(cfg.hidden, cfg.intermediate, cfg.heads, cfg.kv_heads, cfg.head_dim, cfg.layers, cfg.vocab,
                    cfg.max_seq, 1e-5, 0)
    return PagedLlama(w, c, rope_theta=cfg.rope_theta, **{**dict(pages=64, page_size=16, slots=8), **kw})


def normwise(y, ref):
    return float(np.max(np.abs(np.asarray(y, np.float64) - ref)) / np.max(np.abs(ref)))


def test_logits_match_the_oracle(small):
    """A 40-token prompt in uneven chunks beside another sequence, then single
    tokens, teacher-forced."""
    cfg, w = small
    r = np.random.default_rng(1)
    prompt, other = r.integers(0, cfg.vocab, 40).tolist(), r.integers(0, cfg.vocab, 30).tolist()
    orc = llama.LlamaOracle(cfg, w)
    toks, ref = orc.generate(prompt, 6, keep_logits=True)
    m = build(cfg, w)
    m.step([5, 2], [prompt[:7], other[:1]])
    m.step([2, 5], [other[1:25], prompt[7:33]])
    got = [m.step([5], [prompt[33:]])[0]]
    for i, t in enumerate(toks[:5]):
        got.append(m.step([2, 5], [[other[25 + i]], [t]])[1])
    for g, e in zip(got, ref):
        assert normwise(g.float().cpu().numpy(), e) <= LOGIT_TOL
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)


def test_fork_and_compact_change_no_logit(small):
    cfg, w = small
    prompt = np.random.default_rng(2).integers(0, cfg.vocab, 37).tolist()
    m = build(cfg, w)
    m.step([1, 3], [[9] * 50, prompt])
    m.cache.update(fork=[(3, 0), (3, 4)])
    a = m.step([3, 0, 4], [[11], [11], [12]])
    assert torch.equal(a[0], a[1]) and not torch.equal(a[0], a[2])
    b = m.step([3, 0], [[13], [14]])           # the branches part
    m2 = build(cfg, w)
    m2.step([1, 3], [[9] * 50, prompt])
    m2.cache.update(free=[1], fork=[(3, 0)])
    m2.cache.compact()
    assert int((m2.cache.refs > 0).sum()) == int((m2.cache.refs[:3] > 0).sum())
    m2.step([3, 0], [[11], [11]])
    m2.cache.compact()
    assert torch.equal(b, m2.step([3, 0], [[13], [14]]))


def test_generate_greedy_and_sampled(small):
    cfg, w = small
    r = np.random.default_rng(4)
    prompts = [r.integers(0, cfg.vocab, n).tolist() for n in (5, 23, 60)]
    m = build(cfg, w)
    greedy = m.generate(prompts, 5, temperature=0.0, chunk=16)
    alone = [m.generate([p], 5, temperature=0.0)[0] for p in prompts]
    for g, e in zip(greedy, alone):   # the same but for near ties: the first token decides nothing else
        assert g[0][0] == e[0][0]
    s1 = m.generate(prompts[:2], 6, n=3, temperature=0.9, top_k=50, top_p=0.95, seed=7)
    assert s1 == m.generate(prompts[:2], 6, n=3, temperature=0.9, top_k=50, top_p=0.95, seed=7)
    assert len({tuple(b) for b in s1[0]}) > 1
    assert int(m.cache.refs.sum()) == 0


def test_window_sinks_and_norms_run_together(small):
    """A window longer than the text changes nothing; a short one does; unit
    norm weights with per-head norms give finite logits."""
    cfg, w = small
    prompt = np.random.default_rng(5).integers(0, cfg.vocab, 50).tolist()
    full = build(cfg, w).step([0], [prompt])
    assert torch.equal(full, build(cfg, w, window=64).step([0], [prompt]))
    assert not torch.equal(full, build(cfg, w, window=8, sinks=2).step([0], [prompt]))
    ones = [(torch.ones(64, device="cuda"), torch.ones(64, device="cuda"))] * cfg.layers
    assert torch.isfinite(build(cfg, w, qk_norms=ones).step([0], [prompt]).float()).all()


def test_no_room_appends_nothing(small):
    cfg, w = small
    m = build(cfg, w, pages=4)
    m.step([0], [[1] * 40])
    lens = m.cache.lens.clone()
    with pytest.raises(RuntimeError):
        m.step([0, 1], [[2], [3] * 30])
    assert torch.equal(lens, m.cache.lens) and int((m.cache.refs > 0).sum()) == 3
    m.step([0, 1], [[2], [3] * 10])
    with pytest.raises(ValueError):
        m.step([0, 0], [[1], [2]])
    with pytest.raises(ValueError):
        m.step([0], [[cfg.vocab]])
    with pytest.raises(ValueError):
        m.generate([[1]] * 9, 1)
