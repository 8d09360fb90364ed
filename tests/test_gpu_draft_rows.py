"""GPU: accepted draft rows moved behind their context, cached rows read back,
and a whole tree step: norms + rotation + write, tree attention, the kept path,
the next step's attention over it."""
import math

import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from gpu_common import announce, need_gpu, to_np_f32
from oracle import q8_oracle as O
from scored_common import check, eps_of, random_tree, scored_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _tables(rng, lens, bs, extra=2):
    need = [max(1, -(-n // bs)) for n in lens]
    perm = rng.permutation(sum(need) + extra)
    bt = np.full((len(lens), max(need) + 1), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at:at + n]
        at += n
    return bt, sum(need) + extra


def _compact_ref(cache, bt, ctx, nq, accepted, count):
    """cache uint8 [NB, 2, Hkv, X] (numpy, changed in place), one row at a time."""
    bs = cache.shape[3] // 2176 * 16
    old = cache.copy()
    for s in range(len(ctx)):
        for i in range(min(int(count[s]), accepted.shape[1], nq[s])):
            f = int(accepted[s, i])
            if not 0 <= f < nq[s]:
                continue
            src, dst = ctx[s] + f, ctx[s] + i
            for plane in range(2):
                for h in range(cache.shape[2]):
                    q, d = O.planar_read_rows(old, plane, bt[s, src // bs], h, src % bs)
                    O.planar_write_rows(cache, plane, bt[s, dst // bs], h, dst % bs, q, d)


@pytest.mark.parametrize("how", ["stacked", "list"])
@pytest.mark.parametrize("bs,layers,Hkv", [(16, 1, 1), (16, 3, 2), (32, 66, 1), (64, 2, 8)])
def test_compact(bs, layers, Hkv, how):
    need_gpu()
    announce(f"compact bs={bs} layers={layers} Hkv={Hkv} {how}")
    rng = np.random.default_rng(bs + layers)
    ctx, nq = [0, 13, 40, 5, 100], [5, 1, 64, 3, 17]
    bt, nb = _tables(rng, [c + n for c, n in zip(ctx, nq)], bs)
    acc = np.full((5, 64), -1, np.int32)
    acc[0, :3] = [0, 2, 4]
    acc[1, :1] = [0]
    acc[2] = np.arange(64)[::-1]                 # every row a source and a target
    acc[3, :4] = [2, 2, 9, 1]                    # one twice, one past the drafts, and a fourth of three
    acc[4, :5] = [1, -7, 16, 3, 3]
    count = np.array([3, 1, 64, 4, 70], np.int32)
    stack = torch.randint(0, 256, (layers, nb, 2, Hkv, bs // 16 * 2176), dtype=torch.uint8, device=DEV)
    want = stack.cpu().numpy().copy()
    for layer in want:
        _compact_ref(layer, bt, ctx, nq, acc, count)
    kv = stack if how == "stacked" else [(c[:, 0], c[:, 1]) for c in stack]
    t = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    gfx906_fa.compact_draft_rows(kv, t(bt), t([c + n for c, n in zip(ctx, nq)]), t(np.concatenate([[0], np.cumsum(nq)])),
                                 t(acc), t(count))
    torch.cuda.synchronize()
    assert np.array_equal(stack.cpu().numpy(), want)


def test_layers_that_share_a_cache_move_once():
    need_gpu()
    announce("shared layers")
    rng = np.random.default_rng(8)
    ctx, nq, layers = [13, 40], [12, 30], [0, 1, 0, 2, 1, 0]
    bt, nb = _tables(rng, [c + n for c, n in zip(ctx, nq)], 16)
    acc = np.full((2, 8), -1, np.int32)
    acc[0, :4], acc[1] = [0, 2, 3, 9], np.arange(8)[::-1]  # targets that are sources of other rows
    count = np.array([4, 8], np.int32)
    stack = torch.randint(0, 256, (3, nb, 2, 2, 2176), dtype=torch.uint8, device=DEV)
    want = stack.cpu().numpy().copy()
    for layer in want:
        _compact_ref(layer, bt, ctx, nq, acc, count)
    t = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    args = (t(bt), t([c + n for c, n in zip(ctx, nq)]), t(np.concatenate([[0], np.cumsum(nq)])), t(acc), t(count))
    with pytest.raises(RuntimeError):
        gfx906_fa.compact_draft_rows(stack[:1].expand(2, -1, -1, -1, -1), *args)
    gfx906_fa.compact_draft_rows([(stack[i, :, 0], stack[i, :, 1]) for i in layers], *args)
    torch.cuda.synchronize()
    assert np.array_equal(stack.cpu().numpy(), want)


def test_compact_skips_what_it_cannot_reach():
    """Missing pages, short tables and lengths below the drafts move nothing."""
    need_gpu()
    announce("compact unreachable")
    stack = torch.randint(0, 256, (2, 3, 2, 1, 2176), dtype=torch.uint8, device=DEV)
    keep = stack.clone()
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    acc = t([[3, 4, 5]] * 4)
    for bt, lens in ((t([[-1, -1]] * 4), [10] * 4), (t([[99, 7]] * 4), [20] * 4), (t([[0, 1]] * 4), [2, 0, 40, 400])):
        gfx906_fa.compact_draft_rows(stack, bt, t(lens), t([0, 6, 12, 18, 24]), acc, t([3, 3, 3, 3]))
        torch.cuda.synchronize()
        assert torch.equal(stack, keep)
    gfx906_fa.compact_draft_rows(stack, t([[0, 1]] * 4), t([10] * 4), t([0, 6, 12, 18, 24]), acc, t([0, 0, -5, 0]))
    gfx906_fa.compact_draft_rows(stack[:0], t([[0, 1]] * 4), t([10] * 4), t([0, 6, 12, 18, 24]), acc, t([3] * 4))
    gfx906_fa.compact_draft_rows([], t([[0, 1]] * 4), t([10] * 4), t([0, 6, 12, 18, 24]), acc, t([3] * 4))
    torch.cuda.synchronize()
    assert torch.equal(stack, keep)


def test_compact_in_model_pages_and_graph():
    """vLLM's fp16 pages (the planes inside a wider page), captured and
    replayed with other paths."""
    need_gpu()
    announce("compact pages graph")
    from gfx906_fa_paged import q8_planes
    NB, bs, Hkv = 6, 32, 2
    kvs = [torch.randint(0, 256, (NB * 2 * bs * Hkv * 256,), dtype=torch.uint8, device=DEV).view(torch.float16)
           .view(NB, 2, bs, Hkv, 128) for _ in range(3)]
    pairs = [q8_planes(x, Hkv, 128) for x in kvs]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    bt, lens, qsl = t([[4, 2], [0, 5]]), t([40, 50]), t([0, 8, 16])
    acc, cnt = t([[0, 1, 2, 3], [0, 1, 2, 3]]), t([4, 4])
    gfx906_fa.compact_draft_rows(pairs, bt, lens, qsl, acc, cnt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gfx906_fa.compact_draft_rows(pairs, bt, lens, qsl, acc, cnt)
    for path in ([[0, 3, 5, 7], [1, 2, 3, 4]], [[2, 0, 1, 1], [7, 6, 5, 4]], [[0, 1, 2, 7], [-1, 8, 3, 0]]):
        planes = [torch.stack(p, 1) for p in pairs]
        want = [x.cpu().numpy().copy() for x in planes]
        whole = [x.view(torch.uint8).clone() for x in kvs]
        for w in want:
            _compact_ref(w, bt.cpu().numpy(), [32, 42], [8, 8], np.array(path), [4, 4])
        acc.copy_(t(path))
        g.replay()
        torch.cuda.synchronize()
        for p, w, x, old in zip(pairs, want, kvs, whole):
            assert np.array_equal(torch.stack(p, 1).cpu().numpy(), w)
            pk, pv = (y.clone() for y in p)
            a, b = q8_planes(old.view(torch.float16).view(x.shape), Hkv, 128)
            a.copy_(pk)
            b.copy_(pv)
            assert torch.equal(x.view(torch.uint8), old.view(x.view(torch.uint8).shape))  # nothing beside the planes


def test_compact_refusals():
    need_gpu()
    announce("compact refusals")
    stack = torch.zeros((2, 4, 2, 1, 2176), dtype=torch.uint8, device=DEV)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    good = dict(kv_caches=stack, block_table=t([[0, 1]]), seq_lens=t([20]), query_start_loc=t([0, 4]), accepted=t([[0, 1]]),
                num_accepted=t([2]))
    gfx906_fa.compact_draft_rows(**good)
    other = torch.zeros((4, 2, 1, 4352), dtype=torch.uint8, device=DEV)
    for bad in (dict(kv_caches=stack[0]), dict(kv_caches=stack.float()), dict(accepted=t([[0] * 65])),
                dict(accepted=t([[0, 1]]).long()), dict(num_accepted=t([])), dict(num_accepted=t([2]).cpu()),
                dict(query_start_loc=t([0])), dict(block_table=t([[0, 1]]).long()),
                dict(kv_caches=[(stack[0, :, 0], stack[0, :, 1]), (other[:, 0], other[:, 1])]),
                dict(kv_caches=[(stack[0, :, 0].cpu(), stack[0, :, 1].cpu())])):
        with pytest.raises(RuntimeError):
            gfx906_fa.compact_draft_rows(**{**good, **bad})


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,Hkv,bs", [(1, 1, 16), (37, 3, 32), (16, 8, 16), (700, 2, 64)])
@pytest.mark.parametrize("order", ["random", "in_order"])
def test_read_rows(dt, T, Hkv, bs, order):
    """int8 * scale has at most 18 bits: exact in fp32, rounded once below."""
    need_gpu()
    announce(f"read {dt} T={T} Hkv={Hkv} bs={bs} {order}")
    rng = np.random.default_rng(T)
    NB = T // bs + 3
    cache = torch.randint(0, 256, (NB, 2, Hkv, bs // 16 * 2176), dtype=torch.uint8, device=DEV)
    k = torch.from_numpy(rng.standard_normal((NB * bs, Hkv, 128), dtype=np.float32)).to(DEV)
    gfx906_fa.reshape_and_cache_q8_kv(k, k.flip(2).contiguous(), torch.arange(NB * bs, device=DEV), cache[:, 0], cache[:, 1])
    slots = rng.permutation(NB * bs)[:T] if order == "random" else np.arange(5, 5 + T)
    if order == "random" and T > 4:
        slots[1], slots[3], slots[4] = -1, NB * bs, slots[0]
    kr, vr = gfx906_fa.read_cache_q8_kv(torch.from_numpy(slots.astype(np.int64)).to(DEV), cache[:, 0], cache[:, 1], dt)
    kh, vh = O.planar_dequant(cache.cpu().numpy())
    for got, x in ((kr, kh), (vr, vh)):
        x = torch.from_numpy(np.ascontiguousarray(x.reshape(NB * bs, Hkv, 128)[np.clip(slots, 0, NB * bs - 1)]))
        x[(slots < 0) | (slots >= NB * bs)] = 0
        assert torch.equal(got.cpu(), x.to(dt))


def test_read_into_views_and_refusals():
    need_gpu()
    announce("read views")
    cache = gfx906_fa.new_kv_cache(4, 16, 2, device=DEV)
    x = torch.randn((64, 2, 128), dtype=torch.float16, device=DEV)
    n = torch.arange(64, device=DEV)
    gfx906_fa.reshape_and_cache_q8_kv(x, -x, n, cache[:, 0], cache[:, 1])
    k, v = gfx906_fa.read_cache_q8_kv(n, cache[:, 0], cache[:, 1])
    wide = torch.full((64, 2, 2, 256), 9.0, dtype=torch.float16, device=DEV)
    ko, vo = wide[:, 0, :, :128], wide[:, 1, :, 128:]
    r = gfx906_fa.read_cache_q8_kv(n, cache[:, 0], cache[:, 1], k_out=ko, v_out=vo)
    assert r[0] is ko and torch.equal(ko, k) and torch.equal(vo, v)
    assert (wide[:, 0, :, 128:] == 9.0).all() and (wide[:, 1, :, :128] == 9.0).all()
    e = gfx906_fa.read_cache_q8_kv(n[:0], cache[:, 0], cache[:, 1])
    assert e[0].shape == (0, 2, 128)
    for kw in (dict(slot_mapping=n.int()), dict(slot_mapping=n.cpu()), dict(dtype=torch.int8), dict(k_out=ko[:-1]),
               dict(k_out=ko.float()), dict(k_out=torch.empty(64, 2, 132, dtype=torch.float16, device=DEV)[..., 1:129])):
        with pytest.raises(RuntimeError):
            gfx906_fa.read_cache_q8_kv(**{**dict(slot_mapping=n, key_cache=cache[:, 0], value_cache=cache[:, 1]), **kw})


@pytest.mark.parametrize("cap", [0.0, 8.0])
def test_tree_step_from_projection_to_next_token(cap):
    """Two sequences draft a tree each: norms, rotation (a node's position is
    its depth's) and write; attention of the tree; the accepted path kept; one
    more token attends over context and path.  The kept rows are the written
    ones, and both attentions are those of 64 bits over what the cache holds."""
    need_gpu()
    announce(f"tree step cap {cap}")
    rng = np.random.default_rng(6)
    Hq, Hkv, bs, n = 12, 2, 16, 13
    ctx = [41, 128]
    lens = [c + n for c in ctx]
    b = W.build_batch(lens, [n, n], Hq, Hkv, block_size=bs, dtype="bf16", seed=11, device=DEV)
    kp, vp = b.planes()
    trees = [random_tree(rng, n) for _ in ctx]
    depth = [[] for _ in ctx]
    for d, tree in zip(depth, trees):
        for p in tree:
            d.append(d[p] + 1 if p >= 0 else 0)
    pos = torch.tensor([c + x for c, d in zip(ctx, depth) for x in d], device=DEV)
    T = 2 * n
    qkv = torch.randn((T, Hq + 2 * Hkv, 128), device=DEV).to(torch.bfloat16)
    wq, wk = (torch.ones(128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cs = torch.from_numpy(O.rope_cos_sin_cache(512, 128)).to(DEV)
    rows = np.concatenate([np.arange(sum(lens[:s]) + ctx[s], sum(lens[:s + 1])) for s in range(2)])
    slots = b.slot_mapping[torch.from_numpy(rows).to(DEV)]
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    gfx906_fa.qk_norm_rope_and_cache_q8_kv(pos, q, k, v, wq, wk, 1e-6, cs, True, slots, kp, vp)
    b.query = q.contiguous()
    masks = gfx906_fa.tree_masks(trees)
    out = gfx906_fa.tree_attention(q, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, masks.to(DEV), n, max(lens), b.scale,
                                   soft_cap=cap)
    check(out, *scored_oracle(b, cap=cap, masks=masks.numpy(), out_eps=eps_of(torch.bfloat16)))
    # keep the path of each tree's last node
    acc = np.full((2, n), -1, np.int32)
    count = []
    for s, tree in enumerate(trees):
        path, i = [], n - 1
        while i >= 0:
            path.insert(0, i)
            i = tree[i]
        acc[s, :len(path)] = path
        count.append(len(path))
    before = gfx906_fa.read_cache_q8_kv(slots, kp, vp, torch.float32)
    gfx906_fa.compact_draft_rows(b.kv_cache[None], b.block_table, b.seq_lens_t, b.qsl_t, torch.from_numpy(acc).to(DEV),
                                 torch.tensor(count, dtype=torch.int32, device=DEV))
    after = gfx906_fa.read_cache_q8_kv(slots, kp, vp, torch.float32)
    for s in range(2):
        path = torch.from_numpy(acc[s, :count[s]].astype(np.int64)) + s * n
        for x, y in zip(before, after):
            assert torch.equal(y[s * n:s * n + count[s]], x[path])
    # the next token of each sequence
    new = W.Batch(Hq=Hq, Hkv=Hkv, D=128, block_size=bs, seq_lens=np.array([c + m for c, m in zip(ctx, count)], np.int32),
                  q_lens=np.array([1, 1], np.int32), block_table_np=b.block_table_np, num_blocks=b.num_blocks,
                  dtype="bf16", scale=1 / math.sqrt(128), device=torch.device(DEV))
    new.kv_cache, new.query = b.kv_cache, b.query[:2]
    o2 = gfx906_fa.scored_paged_attention(new.query, kp, vp, b.block_table, torch.from_numpy(new.seq_lens).to(DEV),
                                          torch.from_numpy(new.qsl).to(DEV), 1, int(new.seq_lens.max()), new.scale,
                                          soft_cap=cap)
    check(o2, *scored_oracle(new, cap=cap, out_eps=eps_of(torch.bfloat16)))
    assert np.isfinite(to_np_f32(o2)).all()


@pytest.mark.parametrize("n,keep", [(64, 63), (64, 40), (30, 12), (25, 11)])
def test_compact_long_paths(n, keep):
    """Ascending paths of more rows than a wave holds at once, several of them
    a target that a later row's source is next to."""
    need_gpu()
    announce(f"compact long {n} {keep}")
    rng = np.random.default_rng(n + keep)
    ctx, nq = [7, 33, 64], [n] * 3
    bt, nb = _tables(rng, [c + n for c in ctx], 16)
    acc = np.full((3, 64), -1, np.int32)
    for s in range(3):
        acc[s, :keep] = np.sort(rng.permutation(n)[:keep]) if s else np.arange(n - keep, n)
    stack = torch.randint(0, 256, (2, nb, 2, 3, 2176), dtype=torch.uint8, device=DEV)
    want = stack.cpu().numpy().copy()
    for layer in want:
        _compact_ref(layer, bt, ctx, nq, acc, [keep] * 3)
    t = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    gfx906_fa.compact_draft_rows(stack, t(bt), t([c + n for c in ctx]), t(np.arange(4) * n), t(acc), t([keep] * 3))
    torch.cuda.synchronize()
    assert np.array_equal(stack.cpu().numpy(), want)
