"""Performance cases of the serving operators over the Q8_0 paged cache.

Five operators that a speculative or biased decoder needs next to the causal
attention of ``perf/cases.py``:

* ``scored_paged_attention``: scores capped by a tanh, or with a bias that is
  linear in the distance (one slope per query head);
* ``tree_attention``: a tree of drafted tokens over the cached context;
* ``qk_norm_rope_and_cache_q8_kv``: RMS norms of the query and key heads, the
  position rotation and the cache write in one pass;
* ``compact_draft_rows``: the accepted path of a tree moved to the rows right
  behind the context, in every layer's cache;
* ``read_cache_q8_kv``: cached rows back as values.

The plain forms read and write the same planar Q8_0 pages (16-token sub-pages
of 2176 bytes: 128 int8 values a token, then four fp16 scales a token) with
elementary torch operations in 32 bits.  Lengths are ragged and drawn from the
case's own ``lens`` number, so that a case always has the same sizes; block
tables are random permutations of the pool.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128
SUB = 2176                   # bytes of a 16-token sub-page of one kv-head, K or V
ROW = D // 32 * 34           # bytes of a Q8_0 row
SCALE = 1.0 / math.sqrt(D)
EPS = 1e-6
TABLE = 32768                # positions of the rotary table
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HEADS = [(48, 8), (48, 8), (6, 1), (8, 1), (8, 4), (32, 8), (64, 8), (16, 16)]
MOST_SCORES = 3.3e9          # padded scores of a drawn case's plain form, at most


def listed():
    return [
        # The next token of a few short conversations with a distance bias: launches and latency.
        dict(name="alibi_decode_small", kind="scored", prompts=0, len_lo=1, len_hi=1, prior_lo=0, prior_hi=0, decodes=3,
             nq=1, ctx_lo=33, ctx_hi=900, hq=16, hkv=16, bs=16, dtype="f16", cap=0.0, alibi=True, lens=1),
        # A full decode batch with capped scores.
        dict(name="cap_decode_batch", kind="scored", prompts=0, len_lo=1, len_hi=1, prior_lo=0, prior_hi=0, decodes=32,
             nq=1, ctx_lo=2048, ctx_hi=16384, hq=48, hkv=8, bs=16, dtype="bf16", cap=30.0, alibi=False, lens=2),
        # One prompt with capped scores.
        dict(name="cap_prefill", kind="scored", prompts=1, len_lo=8192, len_hi=8192, prior_lo=0, prior_hi=0, decodes=0,
             nq=1, ctx_lo=0, ctx_hi=0, hq=48, hkv=8, bs=16, dtype="bf16", cap=30.0, alibi=False, lens=3),
        # Chunked prefill beside running conversations, with a distance bias.
        dict(name="alibi_mixed", kind="scored", prompts=2, len_lo=700, len_hi=1000, prior_lo=100, prior_hi=4096, decodes=14,
             nq=1, ctx_lo=500, ctx_hi=8191, hq=16, hkv=16, bs=16, dtype="bf16", cap=0.0, alibi=True, lens=4),
        # Two short conversations, each with a small tree of drafts.
        dict(name="tree_small", kind="tree", seqs=2, ctx_lo=200, ctx_hi=900, nodes=7, hq=48, hkv=8, bs=16, dtype="f16",
             cap=0.0, lens=5),
        # A batch of conversations with a wide tree each.
        dict(name="tree_batch", kind="tree", seqs=16, ctx_lo=2048, ctx_hi=8192, nodes=26, hq=48, hkv=8, bs=16,
             dtype="bf16", cap=0.0, lens=6),
        # The projections of one decode step.
        dict(name="norm_rope_decode", kind="norm", tokens=64, hq=48, hkv=8, bs=16, dtype="f16", neox=True, rot=128, lens=7),
        # The projections of a prefill step.
        dict(name="norm_rope_prefill", kind="norm", tokens=8192, hq=48, hkv=8, bs=16, dtype="bf16", neox=True, rot=128,
             lens=8),
        # One layer's cache after a tree step of a few conversations.
        dict(name="compact_layer", kind="compact", layers=1, seqs=7, ctx_lo=20, ctx_hi=300, nodes=13, hkv=8, bs=16, lens=9),
        # Every layer's cache after a tree step of a batch.
        dict(name="compact_model", kind="compact", layers=60, seqs=32, ctx_lo=16, ctx_hi=100, nodes=26, hkv=8, bs=16,
             lens=10),
        # A decode step's rows read back.
        dict(name="read_small", kind="read", tokens=37, hkv=8, bs=16, dtype="f16", lens=11),
        # A long prompt's rows read back, for a transfer.
        dict(name="read_prompt", kind="read", tokens=20001, hkv=8, bs=16, dtype="bf16", lens=12),
    ]


def _between(rng, lo, hi):
    """A whole number, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scored"] * 4 + ["tree"] * 3 + ["norm", "norm", "compact", "compact", "read"])
    hq, hkv = rng.choice(HEADS)
    c = dict(kind=kind, hkv=hkv, bs=rng.choice([16, 16, 32, 64]), lens=rng.randrange(1 << 20))
    if kind != "compact":
        c["dtype"] = rng.choice(["f16", "bf16"])
    if kind == "scored":
        alibi = rng.random() < 0.4
        c.update(hq=hq, alibi=alibi, cap=0.0 if alibi else rng.choice([15.0, 30.0, 50.0]), nq=1, prompts=0, len_lo=1,
                 len_hi=1, prior_lo=0, prior_hi=0, decodes=0, ctx_lo=0, ctx_hi=0)
        how = rng.random()
        if how < 0.6:  # decode and verify steps
            seqs = _between(rng, 1, 64)
            hi = _between(rng, 40, min(65536, max(64, (1 << 21) // (seqs * hkv))))
            c.update(decodes=seqs, nq=rng.choice([1, 1, 2, 5, 8]), ctx_lo=max(16, hi // rng.choice([1, 2, 8])), ctx_hi=hi)
        else:          # prompts, some of them beside decodes
            prompts = _between(rng, 1, 4)
            hi = _between(rng, 20, 6000 // prompts)
            prior = rng.choice([0, 0, _between(rng, 100, 8000 // prompts)])
            c.update(prompts=prompts, len_lo=max(1, hi // rng.choice([1, 3])), len_hi=hi, prior_lo=prior // 2,
                     prior_hi=prior)
            if rng.random() < 0.4:
                c.update(decodes=_between(rng, 1, 8), ctx_lo=64, ctx_hi=_between(rng, 100, 8192))
            while (c["prompts"] + c["decodes"]) * hq * c["len_hi"] * max(c["len_hi"] + c["prior_hi"], c["ctx_hi"]) > MOST_SCORES:
                c.update(len_lo=max(1, c["len_lo"] // 2), len_hi=c["len_hi"] // 2, decodes=c["decodes"] // 2)
    elif kind == "tree":
        seqs = _between(rng, 1, 32)
        hi = _between(rng, 30, min(65536, max(64, (1 << 20) // (seqs * hkv))))
        c.update(hq=hq, seqs=seqs, ctx_lo=max(1, hi // rng.choice([1, 2, 8])), ctx_hi=hi,
                 nodes=rng.choice([1, 3, 5, 8, 13, 26, 40, 64]), cap=rng.choice([0.0, 0.0, 30.0]))
    elif kind == "norm":
        c.update(hq=hq, tokens=_between(rng, 1, 8192 * 56 // (hq + hkv) if hq + hkv > 56 else 8192), neox=rng.random() < 0.7,
                 rot=rng.choice([128, 128, 64, 96, 32]))
    elif kind == "compact":
        c.update(layers=_between(rng, 1, 60), seqs=_between(rng, 1, 32), ctx_lo=1, ctx_hi=_between(rng, 8, 100),
                 nodes=rng.choice([2, 5, 13, 26, 64]))
    else:
        c.update(tokens=_between(rng, 1, 20000 * 8 // max(8, hkv)))
    return c


# --- sizes and inputs ------------------------------------------------------------------------------
def _lens(case):
    """(keys, query tokens) of the case's sequences, prompts first."""
    rng = random.Random(case["lens"])
    if case["kind"] == "scored":
        q = [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(case["prompts"])]
        ctx = [n + rng.randint(case["prior_lo"], case["prior_hi"]) for n in q]
        m = case["nq"]
        more = [max(m, _between(rng, case["ctx_lo"], case["ctx_hi"])) for _ in range(case["decodes"])]
        return ctx + more, q + [m] * len(more)
    if case["kind"] in ("tree", "compact"):
        n = case["nodes"]
        return [_between(rng, case["ctx_lo"], case["ctx_hi"]) + n for _ in range(case["seqs"])], [n] * case["seqs"]
    return [case["tokens"]], [case["tokens"]]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(n):
    s = [0]
    for m in n:
        s.append(s[-1] + m)
    return s


def _raw(case, seed):
    """K and V of every cached token (sequence-major), and the queries."""
    g, td = _gen(seed), TYPES[case["dtype"]]
    ctx, nq = _lens(case)
    k = _randn(g, (sum(ctx), case["hkv"], D), td)
    v = _randn(g, (sum(ctx), case["hkv"], D), td)
    # capped scores are spread wider than plain ones, or the cap would do nothing
    q = (_randn(g, (sum(nq), case["hq"], D), torch.float32) * (2.0 if case["cap"] else 1.0)).to(td)
    return k, v, q


def _pages(g, ctx, bs):
    """Permuted block table and the slot of every cached token."""
    need = [(n + bs - 1) // bs for n in ctx]
    total = sum(need)
    perm = torch.randperm(total + 1, generator=g, device="cuda")[:total]
    bt = torch.full((len(ctx), max(need)), -1, dtype=torch.int32, device="cuda")
    slots, at = [], 0
    for s, (n, m) in enumerate(zip(ctx, need)):
        mine = perm[at:at + m]
        bt[s, :m] = mine.to(torch.int32)
        slots.append((mine[:, None] * bs + torch.arange(bs, device="cuda")).reshape(-1)[:n])
        at += m
    return bt, torch.cat(slots), total + 1


def _blocks(x):
    """Q8_0 blocks of the last dim: int8 values [..., 128] and fp16 scales [..., 4]."""
    b = x.float().view(*x.shape[:-1], 4, 32)
    amax = b.abs().amax(-1, keepdim=True)
    d = amax / torch.full_like(amax, 127.0)
    inv = torch.where(d > 0, torch.ones_like(d) / d, torch.zeros_like(d))
    q = (b * inv).round().clamp(-128, 127).to(torch.int8)
    return q.view(x.shape), d.half().squeeze(-1)


def _new_cache(k, v, slots, nb, bs):
    """The planar cache [pages, 2, kv-heads, bytes] that holds k and v at their slots."""
    hkv, n = k.shape[1], bs // 16
    cache = torch.zeros((nb, 2, hkv, n, SUB), dtype=torch.uint8, device="cuda")
    for plane, x in enumerate((k, v)):
        q, d = _blocks(x)
        pool = torch.zeros((nb * bs, hkv, D), dtype=torch.int8, device="cuda")
        pool[slots] = q
        scale = torch.zeros((nb * bs, hkv, 4), dtype=torch.float16, device="cuda")
        scale[slots] = d
        if plane == 0:  # value d = 64 a + 32 c + 8 g + e of token t at 1024 a + 64 t + 16 g + 8 c + e
            q = pool.view(nb, n, 16, hkv, 2, 2, 4, 8).permute(0, 3, 1, 4, 2, 6, 5, 7)
            d = scale.view(nb, n, 16, hkv, 4).permute(0, 3, 1, 2, 4)
        else:           # value d = 64 a + 16 c + e of token t = 4 u + w at 1024 a + 256 u + 16 e + 4 c + w
            q = pool.view(nb, n, 4, 4, hkv, 2, 4, 16).permute(0, 4, 1, 5, 2, 7, 6, 3)
            d = scale.view(nb, n, 4, 4, hkv, 4).permute(0, 4, 1, 2, 5, 3)
        cache[:, plane, :, :, :2048] = q.reshape(nb, hkv, n, 2048).view(torch.uint8)
        cache[:, plane, :, :, 2048:] = d.reshape(nb, hkv, n, 64).view(torch.uint8)
    return cache.view(nb, 2, hkv, n * SUB)


def _trees(case):
    """For each sequence a random tree: node i's parent is an earlier node, or none."""
    rng = random.Random(case["lens"] + 1)
    return [[rng.randint(-1, i - 1) if rng.random() < 0.7 else i - 1 for i in range(case["nodes"])]
            for _ in range(case["seqs"])]


def _tree_masks(trees):
    """Bit i of a node's mask: it is node i or below it."""
    masks = []
    for tree in trees:
        own_masks = []
        for i, p in enumerate(tree):
            own_masks.append((own_masks[p] if p >= 0 else 0) | 1 << i)
        masks += own_masks
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device="cuda")


def _slopes(heads):
    """Slopes of a distance bias, a geometric sequence over the query heads."""
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    kind = case["kind"]
    if kind == "norm":
        return _prepare_norm(case, seed)
    if kind == "compact":
        return _prepare_compact(case, seed)
    ctx, nq = _lens(case)
    bt, slots, nb = _pages(_gen(seed + 7919), ctx, case["bs"])
    if kind == "read":
        k, v = _raw_read(case, seed)
        return dict(case=case, cache=_new_cache(k, v, slots, nb, case["bs"]), slots=slots)
    k, v, q = _raw(case, seed)
    st = dict(case=case, q=q, cache=_new_cache(k, v, slots, nb, case["bs"]), bt=bt, ctx=_int32(ctx),
              qsl=_int32(_starts(nq)), max_q=max(nq), max_k=max(ctx), mask=None, slopes=None)
    if kind == "tree":
        st["mask"] = _tree_masks(_trees(case))
    elif case["alibi"]:
        st["slopes"] = _slopes(case["hq"])
    return st


def _raw_read(case, seed):
    g, td = _gen(seed), TYPES[case["dtype"]]
    return [_randn(g, (case["tokens"], case["hkv"], D), td) for _ in range(2)]


def _raw_norm(case, seed):
    g, td, t, rot = _gen(seed), TYPES[case["dtype"]], case["tokens"], case["rot"]
    q = _randn(g, (t, case["hq"], D), td)
    k = _randn(g, (t, case["hkv"], D), td)
    v = _randn(g, (t, case["hkv"], D), td)
    wq, wk = ((1 + 0.1 * _randn(g, (D,), torch.float32)).to(td) for _ in range(2))
    inv = 1.0 / (10000.0 ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float32) / rot))
    f = torch.outer(torch.arange(TABLE, device="cuda", dtype=torch.float32), inv)
    table = torch.cat([f.cos(), f.sin()], dim=-1).to(td)
    pos = (torch.arange(t, device="cuda") * 3 + int(seed) % 64) % TABLE
    return q, k, v, wq, wk, table, pos


def _prepare_norm(case, seed):
    q, k, v, wq, wk, table, pos = _raw_norm(case, seed)
    _, slots, nb = _pages(_gen(seed + 7919), [case["tokens"]], case["bs"])
    cache = torch.zeros((nb, 2, case["hkv"], case["bs"] // 16 * SUB), dtype=torch.uint8, device="cuda")
    return dict(case=case, q=q, k=k, v=v, wq=wq, wk=wk, table=table, pos=pos, slots=slots, cache=cache)


def _prepare_compact(case, seed):
    ctx, nq = _lens(case)
    g = _gen(seed)
    bt, _, nb = _pages(_gen(seed + 7919), ctx, case["bs"])
    kv = torch.randint(0, 256, (case["layers"], nb, 2, case["hkv"], case["bs"] // 16 * SUB), generator=g, device="cuda",
                       dtype=torch.uint8)
    # the accepted path of each tree: from a random node up to its root, root first
    rng = random.Random(seed)
    paths = []
    for tree in _trees(case):
        i, path = rng.randrange(len(tree)), []
        while i >= 0:
            path.insert(0, i)
            i = tree[i]
        paths.append(path)
    cols = case["nodes"]
    return dict(case=case, kv=kv, bt=bt, ctx=_int32(ctx), qsl=_int32(_starts(nq)),
                accepted=_int32([p + [-1] * (cols - len(p)) for p in paths]), count=_int32([len(p) for p in paths]))


# --- one pass --------------------------------------------------------------------------------------
def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gfx906-fa-vllm_amd")
    if at not in sys.path:
        sys.path.insert(1, at)
    import gfx906_fa
    return gfx906_fa


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        fa = _framework()
        if kind == "scored":
            return {"out": fa.scored_paged_attention(
                state["q"], state["cache"][:, 0], state["cache"][:, 1], state["bt"], state["ctx"], state["qsl"],
                state["max_q"], state["max_k"], SCALE, soft_cap=case["cap"], alibi_slopes=state["slopes"])}
        if kind == "tree":
            return {"out": fa.tree_attention(
                state["q"], state["cache"][:, 0], state["cache"][:, 1], state["bt"], state["ctx"], state["qsl"],
                state["mask"], state["max_q"], state["max_k"], SCALE, soft_cap=case["cap"])}
        if kind == "norm":
            kp, vp = state["cache"][:, 0], state["cache"][:, 1]
            fa.qk_norm_rope_and_cache_q8_kv(state["pos"], state["q"], state["k"], state["v"], state["wq"], state["wk"], EPS,
                                            state["table"], case["neox"], state["slots"], kp, vp)
            # what the cache now holds, as values
            kr, vr = fa.read_cache_q8_kv(state["slots"], kp, vp, state["k"].dtype)
            return {"key": state["k"], "key_rows": kr, "query": state["q"], "value_rows": vr}
        if kind == "compact":
            fa.compact_draft_rows(state["kv"], state["bt"], state["ctx"], state["qsl"], state["accepted"], state["count"])
            return {"caches": state["kv"]}
        kr, vr = fa.read_cache_q8_kv(state["slots"], state["cache"][:, 0], state["cache"][:, 1], TYPES[case["dtype"]])
        return {"key_rows": kr, "value_rows": vr}
    if kind in ("scored", "tree"):
        return {"out": _plain_attention(state)}
    if kind == "norm":
        return _plain_norm(state)
    if kind == "compact":
        return _plain_compact(state)
    kr, vr = _plain_rows(state["cache"], state["slots"], case["bs"])
    td = TYPES[case["dtype"]]
    return {"key_rows": kr.to(td), "value_rows": vr.to(td)}


def _plain_cached(cache, bt):
    """K and V values [sequences, kv-heads, keys, 128] of the pages in the block table, in 32 bits."""
    b, m = bt.shape
    hkv, n = cache.shape[2], cache.shape[3] // SUB
    pages = cache[bt.clamp_min(0).long()].view(b, m, 2, hkv, n, SUB)
    ints = pages[..., :2048].contiguous().view(torch.int8)
    scales = pages[..., 2048:].contiguous().view(torch.float16)
    k = ints[:, :, 0].view(b, m, hkv, n, 2, 16, 4, 2, 8).permute(0, 2, 1, 3, 5, 4, 7, 6, 8).reshape(b, hkv, m * n * 16, 4, 32)
    ks = scales[:, :, 0].view(b, m, hkv, n, 16, 4).permute(0, 2, 1, 3, 4, 5).reshape(b, hkv, m * n * 16, 4, 1)
    v = ints[:, :, 1].view(b, m, hkv, n, 2, 4, 16, 4, 4).permute(0, 2, 1, 3, 5, 8, 4, 7, 6).reshape(b, hkv, m * n * 16, 4, 32)
    vs = scales[:, :, 1].view(b, m, hkv, n, 4, 4, 4).permute(0, 2, 1, 3, 4, 6, 5).reshape(b, hkv, m * n * 16, 4, 1)
    return (k.float() * ks.float()).flatten(3), (v.float() * vs.float()).flatten(3)


def _plain_attention(st):
    case = st["case"]
    hq, hkv = case["hq"], case["hkv"]
    grp = hq // hkv
    k, v = _plain_cached(st["cache"], st["bt"])
    b, keys = k.shape[0], k.shape[2]
    nq = (st["qsl"][1:] - st["qsl"][:-1]).long()
    j = torch.arange(st["max_q"], device="cuda")
    rows = (st["qsl"][:-1, None] + j).clamp_max(st["q"].shape[0] - 1).long()
    q = st["q"][rows].float().view(b, -1, hkv, grp, D).transpose(1, 2).reshape(b, hkv, -1, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(SCALE).view(b, hkv, -1, grp, keys)
    if case["cap"]:
        s.div_(case["cap"]).tanh_().mul_(case["cap"])
    at = torch.arange(keys, device="cuda")
    before = st["ctx"].long()[:, None] - nq[:, None]      # keys before the step's own tokens
    pos = before + j
    if st["slopes"] is not None:
        away = (at - pos[..., None]).float()               # [sequences, rows, keys]
        s.add_(st["slopes"].view(1, hkv, 1, grp, 1) * away[:, None, :, None])
    seen = at <= pos[..., None]
    if st["mask"] is not None:
        node = at - before[..., None]                      # the key's node of the tree
        bit = (st["mask"][rows][..., None] >> node.clamp(0, 63)) & 1
        seen = seen & ((node < 0) | (bit == 1))
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, hkv, -1, keys), v).view(b, hkv, -1, grp, D)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 2, 1, 3, 4).reshape(b, -1, hq, D)
    mine = (j[None] < nq[:, None])
    return o[mine].to(st["q"].dtype)                       # the sequences' rows, in their order


def _row_bytes(cache, slots, bs):
    """Byte offsets [rows, kv-heads, 2, 136] of cached rows in a layer's cache: 128 values, then four scales."""
    _, _, hkv, page = cache.shape[-4:]
    d = torch.arange(D, device=slots.device)
    pg, off = slots // bs, slots % bs
    t = (off % 16)[:, None]
    k = d // 64 * 1024 + d % 32 // 8 * 16 + d // 32 % 2 * 8 + d % 8 + 64 * t
    v = d // 64 * 1024 + d % 16 * 16 + d // 16 % 4 * 4 + t // 4 * 256 + t % 4
    e = torch.arange(8, device=slots.device)
    ks = 2048 + 8 * t + e
    vs = 2048 + t // 4 * 32 + e // 2 * 8 + t % 4 * 2 + e % 2
    in_sub = torch.stack([torch.cat([k, ks], 1), torch.cat([v, vs], 1)], 1)          # [rows, 2, 136]
    base = (pg * 2 * hkv * page + off // 16 * SUB)[:, None, None, None]
    head = (torch.arange(hkv, device=slots.device) * page)[None, :, None, None]
    plane = (torch.arange(2, device=slots.device) * hkv * page)[None, None, :, None]
    return base + head + plane + in_sub[:, None]


def _plain_rows(cache, slots, bs):
    rows = cache.view(-1)[_row_bytes(cache, slots, bs)]
    q = rows[..., :D].contiguous().view(torch.int8).float().view(*rows.shape[:-1], 4, 32)
    d = rows[..., D:].contiguous().view(torch.float16).float()
    x = (q * d[..., None]).flatten(-2)
    return x[:, :, 0], x[:, :, 1]


def _turned(x, cos, sin, neox, rot):
    """Position rotation of the first `rot` values of each row."""
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    c, s = cos[:, None], sin[:, None]
    u, w = a * c - b * s, b * c + a * s
    y = torch.cat([u, w], -1) if neox else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_norm(st):
    case = st["case"]
    cos, sin = st["table"][st["pos"]].float().chunk(2, dim=-1)

    def turned(x, w):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        return _turned(y, cos, sin, case["neox"], case["rot"]).to(x.dtype)

    st["q"].copy_(turned(st["q"], st["wq"]))
    st["k"].copy_(turned(st["k"], st["wk"]))
    (kq, kd), (vq, vd) = _blocks(st["k"]), _blocks(st["v"])
    q = torch.stack([kq, vq], 2).view(torch.uint8)
    d = torch.stack([kd, vd], 2).view(torch.uint8)
    st["cache"].view(-1)[_row_bytes(st["cache"], st["slots"], case["bs"])] = torch.cat([q, d], -1)
    kr, vr = _plain_rows(st["cache"], st["slots"], case["bs"])
    return {"key": st["k"], "key_rows": kr.to(st["k"].dtype), "query": st["q"], "value_rows": vr.to(st["k"].dtype)}


def _plain_compact(st):
    case, bs = st["case"], st["case"]["bs"]
    before = (st["ctx"] - (st["qsl"][1:] - st["qsl"][:-1])).long()[:, None]
    i = torch.arange(st["accepted"].shape[1], device="cuda")[None]
    moved = (i < st["count"][:, None]).expand_as(st["accepted"])
    src, dst = before + st["accepted"].clamp_min(0), (before + i).expand_as(st["accepted"])
    slot = [(st["bt"].gather(1, x // bs).long() * bs + x % bs)[moved] for x in (src, dst)]
    flat = st["kv"].view(case["layers"], -1)
    flat[:, _row_bytes(st["kv"], slot[1], bs)] = flat[:, _row_bytes(st["kv"], slot[0], bs)]
    return {"caches": st["kv"]}


# --- work ------------------------------------------------------------------------------------------
def work(case):
    kind, hkv = case["kind"], case["hkv"]
    if kind == "norm":
        t, hq = case["tokens"], case["hq"]
        rows = hkv * (2 * ROW + 2 * D * 2)                 # cached rows read back, and their values written
        return {"bytes": t * ((hq + hkv) * D * 4 + hkv * D * 2 + hkv * 2 * ROW + case["rot"] * 2 + 24 + rows), "flops": 0}
    if kind == "read":
        return {"bytes": case["tokens"] * (8 + hkv * (2 * ROW + 2 * D * 2)), "flops": 0}
    if kind == "compact":  # about half of a tree's depth moves: the mean accepted path of its random trees
        rows = 0
        for tree in _trees(case):
            depth = []
            for p in tree:
                depth.append(depth[p] + 1 if p >= 0 else 1)
            rows += sum(depth) / len(depth)
        return {"bytes": rows * case["layers"] * hkv * 4 * ROW, "flops": 0}
    ctx, nq = _lens(case)
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(ctx, nq))
    if kind == "tree":
        pairs = sum(m * (n - m) for n, m in zip(ctx, nq)) + sum(bin(int(x) & (1 << 64) - 1).count("1") for x in _mask_ints(case))
    b = sum(ctx) * hkv * 2 * ROW + 4 * sum((n + case["bs"] - 1) // case["bs"] for n in ctx)
    return {"bytes": b + sum(nq) * case["hq"] * D * 4, "flops": 4 * D * case["hq"] * pairs}


def _mask_ints(case):
    masks = []
    for tree in _trees(case):
        mine = []
        for i, p in enumerate(tree):
            mine.append((mine[p] if p >= 0 else 0) | 1 << i)
        masks += mine
    return masks


# --- the same in 64 bits -----------------------------------------------------------------------------
def _dequantized(x):
    """Q8_0 values of x: blocks of 32 along the last dim, an fp16 scale of amax / 127 each."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    d = top / torch.full_like(top, 127.0)
    inv = torch.where(d > 0, torch.ones_like(d) / d, torch.zeros_like(d))
    return ((b * inv).round().clamp(-128, 127).double() * d.half().double()).flatten(-2)


def _exact_norm(case, seed):
    q, k, v, wq, wk, table, pos = _raw_norm(case, seed)
    angle = table[pos].double()
    half = case["rot"] // 2
    out = []
    for x, w in ((q, wq), (k, wk)):
        y = x.double()
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
        z = y.clone()
        for i in range(half):
            a, b = (i, i + half) if case["neox"] else (2 * i, 2 * i + 1)
            c, s = angle[:, None, i], angle[:, None, half + i]
            z[..., a] = y[..., a] * c - y[..., b] * s
            z[..., b] = y[..., b] * c + y[..., a] * s
        out.append(z)
    # the cache holds the key as it is stored, rounded to its type
    return {"key": out[1], "key_rows": _dequantized(out[1].to(k.dtype)), "query": out[0], "value_rows": _dequantized(v)}


def exact(case, seed):
    kind = case["kind"]
    if kind == "compact":
        return None
    if kind == "norm":
        return _exact_norm(case, seed)
    if kind == "read":
        k, v = _raw_read(case, seed)
        return {"key_rows": _dequantized(k), "value_rows": _dequantized(v)}
    ctx, nq = _lens(case)
    k, v, q = _raw(case, seed)
    hq, hkv = case["hq"], case["hkv"]
    grp = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    masks = _mask_ints(case) if kind == "tree" else None
    slopes = [2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)] if kind == "scored" and case["alibi"] else None
    at = qa = 0
    for n, m in zip(ctx, nq):
        place = torch.arange(n, device="cuda")
        bits = None
        if masks is not None:
            bits = torch.tensor([[mask >> i & 1 for i in range(m)] for mask in masks[qa:qa + m]], dtype=torch.bool, device="cuda")
        for h in range(hkv):
            kd, vd = _dequantized(k[at:at + n, h]), _dequantized(v[at:at + n, h])
            kt = kd.t().contiguous()
            step = max(1, (1 << 26) // n)
            for g in range(h * grp, (h + 1) * grp):
                for a in range(0, m, step):
                    e = min(m, a + step)
                    s = torch.mm(q[qa + a:qa + e, g].double(), kt) * SCALE
                    if case["cap"]:
                        s = case["cap"] * torch.tanh(s / case["cap"])
                    row = torch.arange(n - m + a, n - m + e, device="cuda")[:, None]
                    if slopes is not None:
                        s = s + slopes[g] * (place[None] - row).double()
                    hidden = place[None] > row
                    if bits is not None:
                        hidden[:, n - m:] |= ~bits[a:e]
                    s = s.masked_fill(hidden, -math.inf)
                    p = torch.exp(s - s.amax(-1, keepdim=True))
                    out[qa + a:qa + e, g] = torch.mm(p, vd) / p.sum(-1, keepdim=True)
        at += n
        qa += m
    return {"out": out}
