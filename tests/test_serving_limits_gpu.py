"""PagedLlama at its limits: positions past max_seq, slots that do not exist,
prompts without tokens, sequences of others, steps that fail half way."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from alveare_b200 import PagedKVCache, _lib  # noqa: E402
from alveare_b200.llama import LlamaConfig  # noqa: E402
from alveare_b200.serving import PagedLlama  # noqa: E402
from oracle import llama  # noqa: E402

CFG = llama.Config(hidden=256, intermediate=512, heads=4, kv_heads=2, head_dim=64, layers=2, vocab=1000,
                   vocab_padded=1024, max_seq=100)


@pytest.fixture(scope="module")
def weights():
    return llama.synthetic_weights(CFG, seed=3)[0]


def build(w, max_seq=100, **kw):
    c = LlamaConfig(CFG.hidden, CFG.intermediate, CFG.heads, CFG.kv_heads, CFG.head_dim, CFG.layers, CFG.vocab, max_seq,
                    1e-5, 0)
    return PagedLlama(w, c, rope_theta=CFG.rope_theta, **{**dict(pages=64, page_size=16, slots=8), **kw})


def state(m):
    return [t.clone() for t in (m.cache.table, m.cache.lens, m.cache.refs)]


def unchanged(m, before):
    assert all(torch.equal(a, b) for a, b in zip(state(m), before))
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("slot", [-1, 8, 10 ** 6])
def test_slots_that_do_not_exist(weights, slot):
    m = build(weights)
    m.step([7], [[1] * 20])
    before = state(m)
    with pytest.raises(ValueError, match="slot"):
        m.step([0, slot], [[1], [2]])
    unchanged(m, before)
    with pytest.raises(ValueError, match="slot"):
        m.step([0, 0, 1], [[1], [2]])
    unchanged(m, before)
    with pytest.raises(ValueError, match="slot"):
        m.cache.batch([slot], [1])


def test_batches_that_do_not_match():
    c = PagedKVCache(1, 2, 64, 8, slots=4, max_len=64)
    with pytest.raises(ValueError):
        c.batch([0, 1], [1])
    with pytest.raises(ValueError):
        c.batch([0, 1], [1, -1])


@pytest.mark.parametrize("page_size", [16, 48])
@pytest.mark.parametrize("max_seq", [96, 100])
def test_max_seq(weights, max_seq, page_size):
    """max_seq tokens fit, whatever the page size; one more appends nothing."""
    m = build(weights, max_seq, page_size=page_size)
    m.step([1, 3], [[5] * (max_seq - 1), [6] * 10])
    assert torch.isfinite(m.step([1], [[7]]).float()).all()
    before = state(m)
    with pytest.raises(RuntimeError, match="room"):
        m.step([3, 1], [[8], [9]])
    unchanged(m, before)
    with pytest.raises(RuntimeError, match="room"):
        m.step([3], [[8] * (max_seq - 9)])
    unchanged(m, before)
    assert torch.isfinite(m.step([3], [[8] * (max_seq - 10)]).float()).all()
    _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    with pytest.raises(RuntimeError, match="room"):   # prompt and answer together
        build(weights, max_seq, page_size=page_size).generate([[1] * (max_seq - 2)], 4)


def test_prompts_without_tokens(weights):
    m = build(weights)
    for prompts in ([], [[]], [[1, 2], []]):
        with pytest.raises(ValueError, match="prompt"):
            m.generate(prompts, 3)
    with pytest.raises(ValueError):
        m.generate([[1, 2]], 3, chunk=-4)
    with pytest.raises(ValueError):
        m.generate([[1, 2]], 3, n=0)
    assert m.generate([[1, 2]], 0) == [[[]]]
    assert int(m.cache.refs.sum()) == 0


def test_generate_leaves_other_sequences_alone(weights):
    r = np.random.default_rng(1)
    prompt, more = r.integers(0, CFG.vocab, 30).tolist(), [r.integers(0, CFG.vocab, 11).tolist() for _ in range(2)]
    m = build(weights)
    m.step([0, 2], [prompt, prompt[:9]])
    kept = m.cache.lens.tolist()
    a = m.generate(more, 4, n=2, temperature=0.0, seed=1)
    assert m.cache.lens.tolist() == kept
    after = m.step([0], [[17]])
    alone = build(weights)
    alone.step([0, 2], [prompt, prompt[:9]])
    assert torch.equal(after, alone.step([0], [[17]]))
    assert a == build(weights).generate(more, 4, n=2, temperature=0.0, seed=1)
    with pytest.raises(ValueError, match="slots"):   # six are free
        m.generate([[1]] * 7, 1)


def test_generate_that_fails_gives_its_pages_back(weights):
    m = build(weights, pages=8)
    m.step([5], [[1] * 20])
    before = state(m)
    with pytest.raises(RuntimeError, match="room"):
        m.generate([[1] * 60, [2] * 30], 40)
    after = state(m)
    assert torch.equal(after[1], before[1]) and torch.equal(after[2], before[2])
