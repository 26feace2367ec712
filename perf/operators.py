"""The paged-serving operators, measured: per-head q/k norm + rotation + cache
append, attention of new tokens over a paged cache (sliding window, first
tokens that stay visible), page bookkeeping and token sampling.

Every case is made by :func:`prepare` from its seed; :func:`run` makes one
pass, in plain torch operations (``own`` false) or through the library's entry
points (``own`` true); :func:`exact` computes the same from the definitions in
64 bits.
"""
import math

import numpy as np
import torch

own = False

GRID = 2.0 ** 40  # sampling weights are multiples of 2^-40 of the largest


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one user's next token, one layer of the 1B decode model: latency
        dict(name="attn_token_1b", op="attn", nq=32, nkv=8, hd=64, page=16, batch=1, q_lo=1, q_hi=1,
             kv_lo=331, kv_hi=331, window=0, sinks=0),
        # a full decode batch of users at all depths of a conversation: cache bandwidth
        dict(name="attn_token_batch", op="attn", nq=32, nkv=8, hd=128, page=64, batch=64, q_lo=1, q_hi=1,
             kv_lo=200, kv_hi=9000, window=0, sinks=0),
        # a sliding layer with 256-wide heads, long past, first tokens kept
        dict(name="attn_token_window", op="attn", nq=16, nkv=8, hd=256, page=32, batch=32, q_lo=1, q_hi=1,
             kv_lo=900, kv_hi=30000, window=1024, sinks=4),
        # one chunk of a long prompt over what is cached already: tensor cores
        dict(name="attn_chunk_long", op="attn", nq=32, nkv=8, hd=128, page=64, batch=1, q_lo=2048, q_hi=2048,
             kv_lo=16001, kv_hi=16001, window=0, sinks=0),
        # a scheduler's mixed step: single tokens, short continuations and chunks, ragged
        dict(name="attn_mixed_1b", op="attn", nq=32, nkv=8, hd=64, page=16, batch=13, q_lo=1, q_hi=517,
             kv_lo=517, kv_hi=4100, window=0, sinks=0),
        # chunks through a sliding layer with first tokens kept, 256-wide heads
        dict(name="attn_chunk_window", op="attn", nq=16, nkv=8, hd=256, page=32, batch=3, q_lo=700, q_hi=1500,
             kv_lo=1500, kv_hi=9000, window=512, sinks=4),
        # the q/k/v of a few users' next tokens: latency
        dict(name="rope_token", op="rope", nq=32, nkv=8, hd=64, rot=64, page=16, batch=4, q_lo=1, q_hi=1,
             kv_lo=20, kv_hi=1900, norm=0, f32=0),
        # a prompt chunk's q/k/v with per-head norms
        dict(name="rope_chunk_norm", op="rope", nq=32, nkv=8, hd=128, rot=128, page=64, batch=5, q_lo=700, q_hi=2100,
             kv_lo=2100, kv_hi=8000, norm=1, f32=0),
        # best-of-n over shared prompts: drop last round's branches, branch again, one token more each
        dict(name="pages_branch", op="update", nkv=8, hd=64, page=16, layers=4, parents=8, children=7,
             len_lo=50, len_hi=1000, slack=64),
        # a fragmented pool after most users left: live pages move to the front
        dict(name="pages_compact", op="compact", nkv=8, hd=128, page=16, layers=16, pool=1003, seqs=40, live=0.37),
        # one user's next token, the usual chat settings
        dict(name="sample_one", op="sample", rows=1, vocab=128256, f32=0, temp=0.7, top_k=40, top_p=0.95, min_p=0.05,
             spread=3.0),
        # a batch of users, pure nucleus sampling
        dict(name="sample_batch", op="sample", rows=192, vocab=128256, f32=1, temp=1.0, top_k=0, top_p=0.9, min_p=0.0,
             spread=3.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "attn", "rope", "update", "compact", "sample"])
    if op == "attn":
        hd = rng.choice([64, 128, 256])
        nkv = rng.choice([1, 2, 4, 8])
        nq = nkv * rng.choice([1, 2, 3, 4, 5, 8])
        page = rng.choice([16, 32, 64, 128])
        window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 16, 2000), rng.choice([0, 0, 1, 4, 17]))])
        if rng.random() < 0.5:
            batch, q_lo, q_hi = _log(rng, 1, 100), 1, rng.choice([1, 1, 1, 2, 4])
            kv_hi = _log(rng, 8, min(32000, 400000 // batch))
        else:
            batch, q_hi = _log(rng, 1, 8), _log(rng, 5, 1500)
            q_lo = rng.choice([1, q_hi])
            kv_hi = _log(rng, q_hi, max(q_hi, 16000 // batch))
        kv_lo = max(q_hi, min(kv_hi, _log(rng, 1, kv_hi)))
        return dict(op="attn", nq=nq, nkv=nkv, hd=hd, page=page, batch=batch, q_lo=q_lo, q_hi=q_hi, kv_lo=kv_lo,
                    kv_hi=max(kv_lo, kv_hi), window=window, sinks=sinks)
    if op == "rope":
        hd = rng.choice([64, 128, 256])
        nkv = rng.choice([1, 2, 4, 8])
        batch = _log(rng, 1, 64)
        q_hi = _log(rng, 1, max(1, 6000 // batch))
        kv_hi = q_hi + _log(rng, 1, 2000)
        return dict(op="rope", nq=nkv * rng.choice([1, 2, 3, 4, 7]), nkv=nkv, hd=hd, rot=rng.choice([hd, hd, hd // 2]),
                    page=rng.choice([16, 32, 64]), batch=batch, q_lo=rng.choice([1, q_hi]), q_hi=q_hi, kv_lo=q_hi,
                    kv_hi=kv_hi, norm=rng.choice([0, 1]), f32=rng.choice([0, 1]))
    if op == "update":
        return dict(op="update", nkv=rng.choice([1, 4, 8]), hd=rng.choice([64, 128]), page=rng.choice([16, 32, 64]),
                    layers=rng.choice([1, 3, 4]), parents=_log(rng, 1, 12), children=_log(rng, 1, 8), len_lo=1,
                    len_hi=_log(rng, 10, 1500), slack=rng.randrange(0, 40))
    if op == "compact":
        return dict(op="compact", nkv=rng.choice([1, 4, 8]), hd=rng.choice([64, 128]), page=rng.choice([16, 32]),
                    layers=rng.choice([1, 4, 8]), pool=_log(rng, 30, 1000), seqs=_log(rng, 3, 60),
                    live=round(rng.uniform(0.1, 0.9), 3))
    rows = _log(rng, 1, 150)
    return dict(op="sample", rows=rows, vocab=_log(rng, 500, 160000), f32=rng.choice([0, 1]),
                temp=round(rng.uniform(0.4, 1.6), 2), top_k=rng.choice([0, 0, _log(rng, 1, 400)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 3)]), spread=round(rng.uniform(1.0, 4.0), 2))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lens(case):
    """q and kv lengths of each sequence, the case's own: spread over its
    ranges, ends included."""
    r = np.random.default_rng(case["kv_lo"] * 31 + case["kv_hi"] * 7 + case["q_hi"])
    n = case["batch"]

    def pick(lo, hi):
        v = np.exp(r.uniform(np.log(lo), np.log(hi), n)).round().astype(np.int64).clip(lo, hi)
        v[0] = hi
        if n > 1:
            v[1] = lo
        return v[r.permutation(n)] if n > 1 else v

    q = pick(case["q_lo"], case["q_hi"])
    kv = np.maximum(pick(case["kv_lo"], case["kv_hi"]), q)
    return q.tolist(), kv.tolist()


def _paged(case, seed, dev):
    """Lengths, a page table over a shuffled pool and its device forms."""
    q, kv = _lens(case)
    ps = case["page"]
    need = [-(-n // ps) for n in kv]
    pool = sum(need) + 3
    ids = np.random.default_rng(seed + 1).permutation(pool)
    table = np.full((len(kv), max(need)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    t = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
    return dict(q_lens=q, kv_lens=kv, table_host=table, table=t(table), start=t(start), kv=t(kv), pool=pool,
                tokens=int(start[-1]), max_q=max(q))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7 + 1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)
    st = dict(case)
    op = case["op"]
    if op in ("attn", "rope"):
        st.update(_paged(case, seed, dev))
        nq, nkv, hd, ps = case["nq"], case["nkv"], case["hd"], case["page"]
        st["k"] = rnd(st["pool"], nkv, ps, hd).bfloat16()
        st["v"] = rnd(st["pool"], nkv, ps, hd).bfloat16()
        if op == "attn":
            # slots no token was written to hold whatever the memory held
            for b, n in enumerate(st["kv_lens"]):
                if n % ps:
                    last = int(st["table_host"][b, n // ps])
                    st["k"][last, :, n % ps:] = float("nan")
                    st["v"][last, :, n % ps:] = float("nan")
            st["q"] = (2.0 * rnd(st["tokens"], nq, hd)).bfloat16()
            st["out"] = torch.empty_like(st["q"])
        else:
            st["qkv"] = (1.5 * rnd(st["tokens"], (nq + 2 * nkv) * hd)).to(torch.float32 if case["f32"] else torch.bfloat16)
            st["out"] = torch.empty(st["tokens"], nq, hd, dtype=torch.bfloat16, device=dev)
            rot = case["rot"]
            inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
            ang = torch.arange(max(st["kv_lens"]), dtype=torch.float64)[:, None] * inv
            st["rope"] = torch.cat([ang.cos(), ang.cos(), ang.sin(), ang.sin()], 1).to(torch.bfloat16).to(dev)
            st["qw"] = 1.0 + 0.2 * rnd(hd) if case["norm"] else None
            st["kw"] = 1.0 + 0.2 * rnd(hd) if case["norm"] else None
    elif op == "update":
        r = np.random.default_rng(seed)
        P, C, ps = case["parents"], case["children"], case["page"]
        lens = np.geomspace(case["len_lo"], case["len_hi"], P + 2)[1:-1].round().astype(int)
        need = -(-lens // ps)
        pool = int(need.sum() + 2 * P * C + case["slack"])
        ids = r.permutation(pool)
        S = P * (C + 1)
        table = np.full((S, int(need.max()) + 2), -1, np.int32)
        refs = np.zeros(pool, np.int32)
        slots = r.permutation(S)
        at = 0
        for p in range(P):
            table[slots[p], :need[p]] = ids[at:at + need[p]]
            refs[ids[at:at + need[p]]] = 1
            at += need[p]
        full = np.zeros(S, np.int32)
        full[slots[:P]] = lens
        kids = slots[P:]
        t = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
        st.update(table=t(table), lens=t(full), refs=t(refs), free=t(kids),
                  fork=t(np.stack([slots[np.arange(P * C) % P], kids], 1)),
                  extend=t(np.stack([kids, np.ones(P * C)], 1)),
                  k=rnd(case["layers"], pool, case["nkv"], ps, case["hd"]).bfloat16(),
                  v=rnd(case["layers"], pool, case["nkv"], ps, case["hd"]).bfloat16())
    elif op == "compact":
        r = np.random.default_rng(seed)
        pool, S = case["pool"], case["seqs"]
        live = np.sort(r.permutation(pool)[:max(1, int(pool * case["live"]))])
        own_of = r.integers(0, S, live.size)
        order = r.permutation(live.size)
        width = 2 * live.size // S + 8
        table = np.full((S, width), -1, np.int32)
        refs = np.zeros(pool, np.int32)
        fill = np.zeros(S, int)
        for i in order:
            s = own_of[i] if fill[own_of[i]] < width else int(fill.argmin())
            table[s, fill[s]] = live[i]
            fill[s] += 1
            refs[live[i]] = 1
        # a few pages shared by two sequences, as after a fork
        for i in range(S):
            j = (i + 1) % S
            if j != i and fill[i] and fill[j] < width:
                table[j, fill[j]] = table[i, 0]
                fill[j] += 1
                refs[table[i, 0]] += 1
        t = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
        st.update(table=t(table), refs=t(refs), table_out=t(np.zeros_like(table)), refs_out=t(np.zeros_like(refs)),
                  k=rnd(case["layers"], pool, case["nkv"], case["page"], case["hd"]).bfloat16(),
                  v=rnd(case["layers"], pool, case["nkv"], case["page"], case["hd"]).bfloat16())
    else:
        B, V = case["rows"], case["vocab"]
        st["logits"] = (case["spread"] * rnd(B, V)).to(torch.float32 if case["f32"] else torch.bfloat16)
        st["u"] = torch.rand(B, generator=g, device=dev)
        st["tokens"] = torch.empty(B, dtype=torch.int32, device=dev)
        st["logprobs"] = torch.empty(B, dtype=torch.float32, device=dev)
        st["t_temp"] = torch.full((B, 1), case["temp"], device=dev)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    op = st["op"]
    if own:
        import alveare_b200 as ab
        if op == "attn":
            ab.paged_attention(st["q"], st["out"], st["k"], st["v"], st["table"], st["start"], st["kv"],
                               max_q_len=st["max_q"], window=st["window"], sinks=st["sinks"])
            return st["out"]
        if op == "rope":
            ab.qk_norm_rope(st["qkv"], st["out"], st["k"], st["v"], st["table"], st["start"], st["kv"], st["rope"],
                            q_weight=st["qw"], k_weight=st["kw"], eps=1e-6)
            return st["out"], st["k"], st["v"]
        if op == "update":
            ab.update_pages(st["k"], st["v"], st["table"], st["lens"], st["refs"], free=st["free"], fork=st["fork"],
                            extend=st["extend"])
            return st["table"], st["lens"], st["refs"], st["k"], st["v"]
        if op == "compact":
            ab.compact_pages(st["k"], st["v"], st["table"], st["refs"], st["table_out"], st["refs_out"])
            return st["table_out"], st["refs_out"], st["k"], st["v"]
        ab.sample_tokens(st["logits"], st["u"], st["tokens"], st["logprobs"], temperature=st["temp"],
                         top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
        return st["tokens"], st["logprobs"]
    return {"attn": _plain_attn, "rope": _plain_rope, "update": _plain_update, "compact": _plain_compact,
            "sample": _plain_sample}[op](st)


def _visible(pos, j, window, sinks):
    see = j <= pos
    if window:
        see = see & ((j > pos - window) | (j < sinks))
    return see


def _plain_attn(st):
    nq, nkv, hd, ps = st["nq"], st["nkv"], st["hd"], st["page"]
    g = nq // nkv
    out, t0 = st["out"], 0
    for b, (ql, n) in enumerate(zip(st["q_lens"], st["kv_lens"])):
        pages = st["table"][b, :-(-n // ps)].long()
        k = st["k"][pages].transpose(0, 1).reshape(nkv, -1, hd)[:, :n].float()
        v = st["v"][pages].transpose(0, 1).reshape(nkv, -1, hd)[:, :n].float()
        q = st["q"][t0:t0 + ql].float().reshape(ql, nkv, g, hd).permute(1, 2, 0, 3).reshape(nkv, g * ql, hd)
        pos = (n - ql + torch.arange(ql, device=k.device)).repeat(g)[:, None]
        see = _visible(pos, torch.arange(n, device=k.device)[None, :], st["window"], st["sinks"])
        s = torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(hd))
        s = torch.where(see, s, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[t0:t0 + ql] = o.reshape(nkv, g, ql, hd).permute(2, 0, 1, 3).reshape(ql, nq, hd).bfloat16()
        t0 += ql
    return out


def _positions(st):
    seq = torch.cat([torch.full((q,), b, dtype=torch.long) for b, q in enumerate(st["q_lens"])])
    pos = torch.cat([torch.arange(n - q, n) for q, n in zip(st["q_lens"], st["kv_lens"])])
    return seq.to(st["table"].device), pos.to(st["table"].device)


def _plain_rope(st):
    nq, nkv, hd, ps, rot = st["nq"], st["nkv"], st["hd"], st["page"], st["rot"]
    seq, pos = _positions(st)
    x = st["qkv"].float().reshape(-1, nq + 2 * nkv, hd)
    tab = st["rope"][pos].float()[:, None]
    cos, sin = tab[..., :rot], tab[..., rot:]

    def turn(h, w):
        if w is not None:
            h = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w
        a, rest = h[..., :rot], h[..., rot:]
        other = torch.cat([-a[..., rot // 2:], a[..., :rot // 2]], -1)
        return torch.cat([a * cos + other * sin, rest], -1).bfloat16()

    st["out"].copy_(turn(x[:, :nq], st["qw"]))
    page = st["table"][seq, pos // ps].long()
    st["k"][page, :, pos % ps] = turn(x[:, nq:nq + nkv], st["kw"])
    st["v"][page, :, pos % ps] = x[:, nq + nkv:].bfloat16()
    return st["out"], st["k"], st["v"]


def _plain_update(st):
    table, lens, refs, ps = st["table"], st["lens"], st["refs"], st["page"]

    def count(pages, sign):
        pages = pages[pages >= 0].long()
        refs.index_add_(0, pages, torch.full_like(pages, sign, dtype=torch.int32))

    free = st["free"].long()
    count(table[free].reshape(-1), -1)
    table[free] = -1
    lens[free] = 0
    par, kid = st["fork"][:, 0].long(), st["fork"][:, 1].long()
    count(table[kid].reshape(-1), -1)
    table[kid] = table[par]
    lens[kid] = lens[par]
    count(table[kid].reshape(-1), 1)
    seq, more = st["extend"][:, 0].long(), st["extend"][:, 1].long()
    old = lens[seq].long()
    have, want = (old + ps - 1) // ps, (old + more + ps - 1) // ps
    last = table[seq, (have - 1).clamp(min=0)].long()
    cow = (old % ps != 0) & (more > 0) & (refs[last.clamp(min=0)] > 1)
    n_new = want - have + cow.long()
    at = torch.cumsum(n_new, 0) - n_new
    avail = torch.nonzero(refs == 0).reshape(-1)
    if bool(cow.any()):
        src, dst = last[cow], avail[at[cow]]
        st["k"][:, dst] = st["k"][:, src]
        st["v"][:, dst] = st["v"][:, src]
        refs.index_add_(0, src, torch.full_like(src, -1, dtype=torch.int32))
        table[seq[cow], have[cow] - 1] = dst.int()
        refs[dst] = 1
    for i in range(int((want - have).max())):
        m = want - have > i
        page = avail[at[m] + cow[m].long() + i]
        table[seq[m], have[m] + i] = page.int()
        refs[page] = 1
    lens[seq] = (old + more).int()
    return table, lens, refs, st["k"], st["v"]


def _plain_compact(st):
    refs, table = st["refs"], st["table"]
    used = refs > 0
    n = int(used.sum())
    ids = torch.arange(refs.numel(), device=refs.device)
    src, dst = ids[used & (ids >= n)], ids[~used & (ids < n)]
    st["k"][:, dst] = st["k"][:, src]
    st["v"][:, dst] = st["v"][:, src]
    to = ids.clone()
    to[src] = dst
    st["table_out"].copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table))
    st["refs_out"].zero_()
    st["refs_out"][to[used]] = refs[used]
    return st["table_out"], st["refs_out"], st["k"], st["v"]


def _plain_sample(st):
    s = st["logits"].float() / st["t_temp"]
    w = torch.exp(s - s.amax(1, keepdim=True))
    mass = (w * GRID).to(torch.int64)
    order = torch.sort(s, dim=1, descending=True, stable=True).indices
    sorted_mass = mass.gather(1, order)
    V = s.shape[1]
    n = torch.full((s.shape[0], 1), V, device=s.device, dtype=torch.int64)
    if 0 < st["top_k"] < V:
        n.fill_(st["top_k"])
    cum = sorted_mass.cumsum(1)
    if st["top_p"] < 1.0:
        p = torch.tensor(st["top_p"], dtype=torch.float32, device=s.device).double()
        goal = torch.ceil(cum.gather(1, n - 1).double() * p).to(torch.int64).clamp(min=1)
        n = torch.minimum(n, (cum < goal).sum(1, keepdim=True) + 1)
    rank_ok = torch.arange(V, device=s.device)[None, :] < n
    keep = torch.zeros_like(rank_ok).scatter_(1, order, rank_ok)
    keep &= w >= torch.tensor(st["min_p"], dtype=torch.float32, device=s.device)
    mass = torch.where(keep, mass, 0)
    cum = mass.cumsum(1)
    total = cum[:, -1:]
    goal = torch.minimum((st["u"][:, None].double() * total.double()).floor().to(torch.int64), total - 1)
    tok = (cum <= goal).sum(1, keepdim=True)
    st["tokens"].copy_(tok[:, 0])
    st["logprobs"].copy_(torch.log(mass.gather(1, tok).double() / total.double())[:, 0])
    return st["tokens"], st["logprobs"]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "attn":
        nkv, hd, ps = case["nkv"], case["hd"], case["page"]
        g = case["nq"] // nkv
        out = torch.empty(st["tokens"], case["nq"], hd, dtype=torch.float64, device="cuda")
        t0 = 0
        for b, (ql, n) in enumerate(zip(st["q_lens"], st["kv_lens"])):
            slot = torch.arange(n, device="cuda")
            page = st["table"][b].long()[slot // ps]
            for h in range(nkv):
                k = st["k"][page, h, slot % ps].double()
                v = st["v"][page, h, slot % ps].double()
                for i0 in range(0, ql, 512):
                    i1 = min(ql, i0 + 512)
                    q = st["q"][t0 + i0:t0 + i1, h * g:(h + 1) * g].double()
                    s = torch.einsum("qgd,nd->qgn", q, k) / math.sqrt(hd)
                    pos = n - ql + torch.arange(i0, i1, device="cuda")
                    hidden = slot[None, :] > pos[:, None]
                    if case["window"]:
                        hidden |= (slot[None, :] <= pos[:, None] - case["window"]) & (slot[None, :] >= case["sinks"])
                    s.masked_fill_(hidden[:, None, :], float("-inf"))
                    s = s - torch.logsumexp(s, -1, keepdim=True)
                    out[t0 + i0:t0 + i1, h * g:(h + 1) * g] = torch.einsum("qgn,nd->qgd", s.exp_(), v)
            t0 += ql
        return out
    if op == "rope":
        nq, nkv, hd, ps, rot = case["nq"], case["nkv"], case["hd"], case["page"], case["rot"]
        x = st["qkv"].double().view(-1, nq + 2 * nkv, hd)
        k, v = st["k"].double(), st["v"].double()
        q = torch.empty(x.shape[0], nq, hd, dtype=torch.float64, device="cuda")
        half, t0 = rot // 2, 0
        for b, (ql, n) in enumerate(zip(st["q_lens"], st["kv_lens"])):
            pos = torch.arange(n - ql, n, device="cuda")
            c, s = st["rope"][pos, None, :half].double(), st["rope"][pos, None, rot:rot + half].double()
            h = x[t0:t0 + ql].clone()
            for lo, hi, wt in ((0, nq, st["qw"]), (nq, nq + nkv, st["kw"])):
                y = h[:, lo:hi].clone()
                if wt is not None:
                    y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / hd + 1e-6) * wt.double()
                z = y.clone()
                z[..., :half] = y[..., :half] * c - y[..., half:rot] * s
                z[..., half:rot] = y[..., half:rot] * c + y[..., :half] * s
                h[:, lo:hi] = z
            page = st["table"][b].long()[pos // ps]
            q[t0:t0 + ql] = h[:, :nq]
            k[page, :, pos % ps] = h[:, nq:nq + nkv]
            v[page, :, pos % ps] = h[:, nq + nkv:]
            t0 += ql
        return q, k, v
    if op in ("update", "compact"):
        return _exact_pages(st, op)
    return _exact_sample(st, case)


def _exact_pages(st, op):
    table, refs = st["table"].cpu().numpy().copy(), st["refs"].cpu().numpy().copy()
    moves = []
    if op == "compact":
        n = int((refs > 0).sum())
        holes = [p for p in range(n) if refs[p] == 0]
        new = np.zeros_like(refs)
        new[:n] = refs[:n]
        for src in range(n, refs.size):
            if refs[src]:
                dst = holes.pop(0)
                moves.append((src, dst))
                table[table == src] = dst
                new[dst] = refs[src]
        head = (table, new)
    else:
        ps, lens = st["page"], st["lens"].cpu().numpy().copy()

        def drop(row):
            for e in range(table.shape[1]):
                if table[row, e] >= 0:
                    refs[table[row, e]] -= 1
                    table[row, e] = -1
            lens[row] = 0

        for row in st["free"].tolist():
            drop(row)
        for par, kid in st["fork"].tolist():
            drop(kid)
            table[kid], lens[kid] = table[par], lens[par]
            for p in table[kid]:
                if p >= 0:
                    refs[p] += 1
        before = refs.copy()
        fresh = iter([p for p in range(refs.size) if refs[p] == 0])
        for row, more in st["extend"].tolist():
            at = int(lens[row])
            if at % ps and more > 0 and before[table[row, at // ps]] > 1:
                src, dst = int(table[row, at // ps]), next(fresh)
                moves.append((src, dst))
                refs[src] -= 1
                refs[dst] = 1
                table[row, at // ps] = dst
            for e in range(-(-at // ps), -(-(at + more) // ps)):
                table[row, e] = next(fresh)
                refs[table[row, e]] = 1
            lens[row] = at + more
        head = (table, lens, refs)
    for src, dst in moves:
        st["k"][:, dst], st["v"][:, dst] = st["k"][:, src], st["v"][:, src]
    return tuple(torch.from_numpy(a) for a in head) + (st["k"], st["v"])


def _exact_sample(st, case):
    """Tokens and log probabilities row by row.  The definition's weights are
    32-bit values on a grid; an implementation's exp may differ from the true
    one by a last place.  A draw (or a nucleus edge) so close to the border
    of two tokens that such differences decide it has no value here."""
    logits, u = st["logits"].float().cpu().numpy(), st["u"].double().cpu().numpy()
    temp, top_p, min_p = (np.float32(case[f]) for f in ("temp", "top_p", "min_p"))
    tokens, logprobs = [], []
    for row, r in zip(logits, u):
        s = row / temp
        w32 = np.exp((s - s.max()).astype(np.float64)).astype(np.float32)
        w = np.floor(w32.astype(np.float64) * GRID)
        order = np.argsort(-s, kind="stable")
        if 0 < case["top_k"] < row.size:
            order = order[:case["top_k"]]
        cum = np.cumsum(w[order])
        near = 1e-7 * math.sqrt(float(np.square(w[order]).sum()))
        slip = 0.0
        if top_p < 1.0:
            goal = max(math.ceil(cum[-1] * float(top_p)), 1)
            n = min(int(np.searchsorted(cum, goal)), order.size - 1)
            if min(cum[n] - goal, goal - cum[n - 1] if n else cum[-1]) < near:
                slip = float(w[order[n]])
            order = order[:n + 1]
        order = np.sort(order[w32[order] >= min_p])
        cum = np.cumsum(w[order])
        goal = min(math.floor(r * cum[-1]), cum[-1] - 1)
        i = int(np.searchsorted(cum, goal, side="right"))
        if min(cum[i] - goal, goal - cum[i - 1] if i else cum[-1]) < near + slip and order.size > 1:
            return None, None
        tokens.append(int(order[i]))
        logprobs.append(math.log(w[order[i]] / cum[-1]))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "attn":
        q_lens, kv_lens = _lens(case)
        pairs = rows = 0
        for ql, n in zip(q_lens, kv_lens):
            w, s = case["window"], case["sinks"]
            pos = np.arange(n - ql, n)
            if w:
                lo = np.maximum(pos - w + 1, 0)
                pairs += int((pos + 1 - lo + np.minimum(lo, s)).sum())
                rows += n - max(int(lo[0]), 0) + min(int(lo[0]), s)
            else:
                pairs += int((pos + 1).sum())
                rows += n
        io = 2 * sum(q_lens) * case["nq"] * case["hd"] * 2
        return {"bytes": io + rows * case["nkv"] * case["hd"] * 4, "flops": 4 * pairs * case["nq"] * case["hd"]}
    if op == "rope":
        q_lens, _ = _lens(case)
        t, heads, hd = sum(q_lens), case["nq"] + 2 * case["nkv"], case["hd"]
        return {"bytes": t * (heads * hd * ((4 if case["f32"] else 2) + 2) + 4 * case["rot"]),
                "flops": t * (case["nq"] + case["nkv"]) * (3 * case["rot"] + (4 * hd if case["norm"] else 0))}
    if op == "update":
        page = case["layers"] * case["nkv"] * case["page"] * case["hd"] * 2 * 2
        n = case["parents"] * case["children"]
        entries = max(1, (case["len_lo"] + case["len_hi"]) // 2 // case["page"])
        # a child's last page is copied unless it was full
        return {"bytes": int(2 * page * n * (1 - 1 / case["page"])) + n * entries * 16, "flops": n * entries}
    if op == "compact":
        page = case["layers"] * case["nkv"] * case["page"] * case["hd"] * 2 * 2
        n = max(1, int(case["pool"] * case["live"]))
        # a live page sits past the first n with probability 1 - n / pool
        moved = n * (1 - n / case["pool"])
        return {"bytes": int(2 * page * moved) + 8 * n + 8 * case["pool"], "flops": int(case["pool"])}
    size = 4 if case["f32"] else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 12), "flops": 4 * case["rows"] * case["vocab"]}
