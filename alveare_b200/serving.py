"""Many Llama sequences served from one paged cache.

:class:`PagedLlama` runs ragged steps -- chunks of prompts and single tokens of
other sequences in one batch -- over the Q4 matrices (:mod:`alveare_b200.ops`)
and the paged operators (:mod:`alveare_b200.paged`): q/k/v rotated and appended
in one pass, attention over the pages, page bookkeeping with shared prompts,
sampling.  It takes the weights :class:`alveare_b200.llama.LlamaDecoder` takes
(tools/quantize_model.py:39-125) and rounds where the reference's CPU path
rounds (runtime/py/model.py:821-934); LlamaDecoder remains the form for one
greedy sequence.
"""
from __future__ import annotations

import numpy as np

from . import ops
from .llama import LlamaConfig, load_weights_dir, rope_table
from .paged import PagedKVCache, paged_attention, qk_norm_rope, sample_tokens

try:
    import torch
except Exception:  # pragma: no cover
    torch = None


class PagedLlama:
    """``slots`` sequences of up to ``max_len`` tokens over ``pages`` cache
    pages of ``page_size`` positions.  ``window`` / ``sinks`` limit every
    layer's attention (0: none); ``qk_norms`` gives per-layer (q, k) norm
    weights of head_dim float32 values (None: no norm)."""

    def __init__(self, weights, config: LlamaConfig, *, pages: int, page_size: int = 16, slots: int = 16,
                 device: int = 0, rope_theta: float = 500000.0, window: int = 0, sinks: int = 0, qk_norms=None):
        c = self.cfg = config
        self.device = torch.device("cuda", device)
        self.window, self.sinks, self.qk_norms = window, sinks, qk_norms
        if not isinstance(weights, dict):
            weights = load_weights_dir(weights, c.layers)
        host = lambda n: np.asarray(weights[n])
        dev = lambda n, dt: torch.from_numpy(np.array(host(n))).to(self.device, dt)
        nq, nkv = c.heads * c.head_dim, c.kv_heads * c.head_dim

        def q4(rows, *names):  # the first rows of each matrix, stacked
            parts = [host(n)[:r] for n, r in zip(names, rows)]
            cols = parts[0].shape[1] // 20 * 32
            return ops.Q4Weight(np.concatenate(parts), N=sum(rows), K=cols, device=device)

        self.emb = dev("token_embd", torch.float16)
        self.out_norm = dev("output_norm.weight", torch.float32)
        self.lm_head = q4((c.vocab,), "lm_head_packed")
        self.layers = []
        for l in range(c.layers):
            w = lambda p: f"blk.{l}.{p}.weight_packed"
            self.layers.append((dev(f"blk.{l}.attn_norm.weight", torch.float32),
                                q4((nq, nkv, nkv), w("attn_q"), w("attn_k"), w("attn_v")),
                                q4((c.hidden,), w("attn_output")),
                                dev(f"blk.{l}.ffn_norm.weight", torch.float32),
                                q4((c.intermediate, c.intermediate), w("ffn_gate"), w("ffn_up")),
                                q4((c.hidden,), w("ffn_down"))))
        table = rope_table(c.head_dim, c.max_seq, rope_theta).view(np.int16)
        self.rope = torch.from_numpy(table).to(self.device).view(torch.bfloat16)
        self.cache = PagedKVCache(c.layers, c.kv_heads, c.head_dim, pages, page_size=page_size, slots=slots,
                                  max_len=c.max_seq, device=device)

    # -- one ragged step --------------------------------------------------------
    def _gemm(self, w, x):
        y = torch.empty(x.shape[0], w.N, dtype=torch.bfloat16, device=self.device)
        ops.gemm_q_npu(w, x, y, B=x.shape[0], N=w.N, K=w.K)
        return y

    def _norm(self, x, w):
        f = x.float()
        return (f * (1.0 / torch.sqrt((f * f).mean(-1, keepdim=True) + self.cfg.rms_eps)) * w).bfloat16()

    def step(self, slots, tokens):
        """Append ``tokens[i]`` (a list of ids) to sequence ``slots[i]``, all in
        one batch; the bfloat16 logits (len(slots), vocab) after each one's last
        token.  Raises RuntimeError (and appends nothing) when the cache has no
        room for all of them or a sequence would pass ``max_seq`` tokens."""
        c = self.cfg
        lens, slots = [len(t) for t in tokens], [int(s) for s in slots]
        self.cache.check_slots(slots)
        if min(lens, default=0) < 1 or not len(set(slots)) == len(slots) == len(lens):
            raise ValueError("step: every slot once, with at least one token")
        flat = torch.tensor([t for ts in tokens for t in ts], dtype=torch.int64)
        if int(flat.min()) < 0 or int(flat.max()) >= c.vocab:
            raise ValueError("step: token id out of range")
        before = self.cache.snapshot()
        self.cache.update(extend=list(zip(slots, lens)))
        # (pages are whole: the last one may have room past max_seq)
        first_unmet, *held = torch.cat((self.cache.info[3:], self.cache.lens)).tolist()
        if first_unmet >= 0 or any(held[s] > c.max_seq for s in slots):
            self.cache.restore(before)
            raise RuntimeError("step: the cache has no room for these tokens, or max_seq is passed")
        b = self.cache.batch(slots, lens)
        x = self.emb[flat.to(self.device)].bfloat16()
        rows, hd = x.shape[0], c.head_dim
        q = torch.empty(rows, c.heads, hd, dtype=torch.bfloat16, device=self.device)
        attn = torch.empty_like(q)
        for l, (n1, wqkv, wo, n2, wgu, wd) in enumerate(self.layers):
            qw, kw = self.qk_norms[l] if self.qk_norms else (None, None)
            qk_norm_rope(self._gemm(wqkv, self._norm(x, n1)), q, self.cache.k[l], self.cache.v[l], rope=self.rope,
                         q_weight=qw, k_weight=kw, eps=c.rms_eps, **b)
            paged_attention(q, attn, self.cache.k[l], self.cache.v[l], max_q_len=max(lens), window=self.window,
                            sinks=self.sinks, **b)
            x = x + self._gemm(wo, attn.view(rows, -1))
            g, u = self._gemm(wgu, self._norm(x, n2)).float().split(c.intermediate, 1)
            x = x + self._gemm(wd, (g * torch.sigmoid(g) * u).bfloat16())
        last = (b["q_start"][1:] - 1).long()
        return self._gemm(self.lm_head, self._norm(x[last], self.out_norm))

    # -- whole requests -----------------------------------------------------------
    def generate(self, prompts, max_new_tokens: int, *, n: int = 1, chunk: int = 512, seed: int = 0, temperature=1.0,
                 top_k=0, top_p=1.0, min_p=0.0):
        """``n`` continuations of every prompt: prompts in chunks of ``chunk``
        tokens (all sequences' chunks in one batch), their pages shared by the n
        branches, then sampled tokens.  Returns [prompt][branch][token].  Takes
        slots that hold no tokens (ValueError if there are too few) and empties
        them again; other sequences stay as they are."""
        B = len(prompts)
        if B < 1 or min(map(len, prompts)) < 1:
            raise ValueError("generate: every prompt needs at least one token")
        if n < 1 or chunk < 1:
            raise ValueError("generate: n and chunk must be positive")
        slots = [s for s, held in enumerate(self.cache.lens.tolist()) if held == 0][:B * n]
        if len(slots) < B * n:
            raise ValueError(f"generate: {B * n} sequences need as many empty slots (there are {len(slots)})")
        self.cache.update(free=slots)  # (pages that a shortened sequence left)
        try:
            logits = torch.empty(B, self.cfg.vocab, dtype=torch.bfloat16, device=self.device)
            for at in range(0, max(map(len, prompts)), chunk):
                rows = [i for i, p in enumerate(prompts) if at < len(p)]
                logits[rows] = self.step([slots[i * n] for i in rows], [list(prompts[i][at:at + chunk]) for i in rows])
            if n > 1:
                self.cache.update(fork=[(slots[i * n], slots[i * n + j]) for i in range(B) for j in range(1, n)])
            logits = logits.repeat_interleave(n, 0)
            gen = torch.Generator(device=self.device).manual_seed(seed)
            tok = torch.empty(B * n, dtype=torch.int32, device=self.device)
            out = []
            for i in range(max_new_tokens):
                u = torch.rand(B * n, generator=gen, device=self.device)
                sample_tokens(logits, u, tok, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
                out.append(tok.tolist())
                if i + 1 < max_new_tokens:
                    logits = self.step(slots, [[t] for t in out[-1]])
        finally:  # also when a step finds no room half way
            self.cache.update(free=slots)
        return [[[row[i * n + j] for row in out] for j in range(n)] for i in range(B)]
