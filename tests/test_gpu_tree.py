"""GPU: attention of a tree of drafted tokens over the cache, against 64 bits."""
import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from gpu_common import announce, need_gpu
from scored_common import check, eps_of, random_tree, scored_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
TD = {"f16": torch.float16, "bf16": torch.bfloat16}

# (contexts, nodes of each tree, heads, kv-heads, block size)
SHAPES = {
    "one_node": ([1, 40], [1, 1], 8, 1, 16),
    "no_context": ([0, 0, 5], [1, 7, 7], 8, 1, 16),
    "rows16": ([250, 33, 700], [2, 2, 2], 8, 1, 16),
    "rows30": ([600, 9], [5, 5], 6, 1, 32),
    "rows48_tiles": ([1030] * 8, [8] * 8, 48, 8, 16),
    "rows64": ([333], [64], 4, 4, 16),
    "rows126": ([90, 1000], [21, 21], 6, 1, 16),
    "rows384": ([777, 63], [64, 64], 12, 2, 64),
    "ragged": ([100, 0, 450, 64, 31], [13, 1, 64, 3, 6], 6, 1, 16),
    "long": ([9000], [33], 48, 8, 16),
}


def _batch(name, dt="f16", seed=4):
    ctx, n, hq, hkv, bs = SHAPES[name]
    b = W.build_batch([c + m for c, m in zip(ctx, n)], n, hq, hkv, block_size=bs, dtype=dt, seed=seed, device=DEV,
                      bt_pad_cols=1)
    b.kv_cache.fill_(0xFF)  # NaN scales wherever no key is
    gfx906_fa.reshape_and_cache_q8_kv(b.key, b.value, b.slot_mapping, *b.planes())
    rng = np.random.default_rng(seed)
    return b, gfx906_fa.tree_masks([random_tree(rng, m) for m in n])


def _call(b, masks, **kw):
    kp, vp = b.planes()
    return gfx906_fa.tree_attention(b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, masks.to(DEV),
                                    b.max_query_len, b.max_seq_len, b.scale, **kw)


@pytest.mark.parametrize("cap", [0.0, 4.0])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_tree(name, dt, cap):
    need_gpu()
    announce(f"tree {name} {dt} cap {cap}")
    b, masks = _batch(name, dt)
    out = _call(b, masks, soft_cap=cap)
    check(out, *scored_oracle(b, cap=cap, masks=masks.numpy(), out_eps=eps_of(TD[dt])))


def test_chain_is_causal_attention():
    """A tree that is one chain sees what causal rows see."""
    need_gpu()
    announce("chain")
    for name in ("rows30", "rows126", "ragged"):
        b, _ = _batch(name)
        masks = gfx906_fa.tree_masks([list(range(-1, int(m) - 1)) for m in b.q_lens])
        out = _call(b, masks, out_dtype=torch.float32)
        check(out, *scored_oracle(b))


@pytest.mark.parametrize("name", ["rows30", "rows64", "rows384"])
def test_any_masks(name):
    """Masks that are no tree: bits of later nodes do not count, rows may miss
    their own node, and a row without a bit sees the context alone."""
    need_gpu()
    announce(f"any masks {name}")
    b, _ = _batch(name)
    rng = np.random.default_rng(1)
    masks = torch.from_numpy(rng.integers(-2 ** 63, 2 ** 63, b.num_tokens, dtype=np.int64))
    masks[0], masks[-1] = -1, 0
    out = _call(b, masks, out_dtype=torch.float32)
    check(out, *scored_oracle(b, masks=masks.numpy()))


def test_row_without_a_key_is_zero():
    need_gpu()
    announce("no key")
    for n, hq in ((3, 8), (40, 8)):
        b = W.build_batch([n, n + 9], [n, n], hq, 1, dtype="f16", seed=1, device=DEV)
        masks = torch.zeros(2 * n, dtype=torch.int64)
        out = _call(b, masks)
        assert (out[:n] == 0).all()
        check(out, *scored_oracle(b, masks=masks.numpy(), out_eps=eps_of(torch.float16)))


@pytest.mark.parametrize("name", ["rows16", "rows30", "rows48_tiles", "rows64", "rows126", "rows384"])
def test_hidden_nodes_may_hold_anything(name):
    """Nodes with Inf and NaN keys and values: rows that do not see them are
    as with finite ones."""
    need_gpu()
    announce(f"hidden {name}")
    b, masks = _batch(name)
    bad = [int(b.qsl[s]) + int(b.q_lens[s]) // 2 for s in range(b.num_seqs)]  # a node of each tree
    m = masks.numpy().copy()
    for s, t in enumerate(bad):
        i = t - int(b.qsl[s])
        for r in range(int(b.qsl[s]), int(b.qsl[s + 1])):
            if r != t:
                m[r] &= ~np.int64(1 << i)
    masks = torch.from_numpy(m)
    want = _call(b, masks)
    at = np.cumsum(b.seq_lens) - b.q_lens
    for s, t in enumerate(bad):
        row = int(at[s]) + t - int(b.qsl[s])
        b.key[row] = float("inf")
        b.value[row] = float("nan") if s % 2 else float("inf")
    gfx906_fa.reshape_and_cache_q8_kv(b.key, b.value, b.slot_mapping, *b.planes())
    got = _call(b, masks)
    keep = [t for t in range(b.num_tokens) if t not in bad]
    assert torch.equal(got[keep], want[keep])


def test_rows_behind_the_last_sequence():
    need_gpu()
    announce("rows behind")
    b, masks = _batch("ragged")
    ref = scored_oracle(b, masks=masks.numpy(), out_eps=eps_of(torch.float16))
    T = b.num_tokens
    out = torch.full((T + 5, b.Hq, 128), 5.0, dtype=torch.float16, device=DEV)
    b.query = torch.cat([b.query, b.query[:5]])
    kp, vp = b.planes()
    gfx906_fa.tree_attention(b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t,
                             torch.cat([masks, masks[:5]]).to(DEV), b.max_query_len, b.max_seq_len, b.scale, out=out)
    check(out[:T], *ref)
    assert (out[T:] == 5.0).all()


def test_graph_replay():
    need_gpu()
    announce("tree graph")
    b, masks = _batch("rows126")
    md = masks.to(DEV)
    kp, vp = b.planes()
    ws = gfx906_fa.new_workspace(gfx906_fa.workspace_size(b.num_seqs, b.num_tokens, b.Hq, b.Hkv, b.max_query_len,
                                                          b.max_seq_len), DEV)
    out = torch.zeros((b.num_tokens, b.Hq, 128), dtype=torch.float16, device=DEV)
    call = lambda: gfx906_fa.tree_attention(b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, md,  # noqa: E731
                                            b.max_query_len, b.max_seq_len, b.scale, out=out, workspace=ws)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    rng = np.random.default_rng(8)
    for _ in range(3):
        md.copy_(gfx906_fa.tree_masks([random_tree(rng, int(m)) for m in b.q_lens]))
        want = gfx906_fa.tree_attention(b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, md, b.max_query_len,
                                        b.max_seq_len, b.scale)
        torch.cuda.synchronize()
        out.fill_(2.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals():
    need_gpu()
    announce("tree refusals")
    b, masks = _batch("rows30")
    with pytest.raises(RuntimeError):
        _call(b, masks.int())
    with pytest.raises(RuntimeError):
        _call(b, masks[:-1])
    with pytest.raises(RuntimeError):
        _call(b, masks, soft_cap=-2.0)
    kp, vp = b.planes()
    with pytest.raises(RuntimeError):  # more than 64 nodes
        gfx906_fa.tree_attention(b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, masks.to(DEV), 65, b.max_seq_len,
                                 b.scale)
    with pytest.raises(RuntimeError):
        gfx906_fa.tree_attention(b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, masks, 5, b.max_seq_len, b.scale)
