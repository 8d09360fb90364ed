"""GPU: caps far below the scale, with values on which a wrong score shows and a
bound that the cap limits (tests/test_capped_host.py: zeroed, negated, halved
and misplaced scores are all outside it)."""
import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from capped_common import capped_rows, telling_values
from gpu_common import announce, need_gpu, seq_head_kv, to_np_f32
from scored_common import random_tree, seen_keys

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (keys, query tokens, heads, kv-heads, block size)
SHAPES = {
    "decode": ([33, 257, 900], [1, 1, 1], 16, 2, 16),
    "rows30": ([640, 35], [5, 5], 6, 1, 32),
    "rows48": ([700, 90], [8, 8], 6, 1, 16),
    "rows64": ([500], [8], 8, 1, 16),
    "tiles128": ([700, 130], [12, 12], 8, 1, 16),
    "tiles256": ([500], [60], 12, 2, 16),
    "prompt": ([301], [301], 4, 1, 16),
    "split": ([2100], [50], 6, 1, 32),
    "images": ([1400], [1400], 6, 1, 16),
}
CAPS = [  # cap, scale, the queries' size
    (0.003, 128 ** -0.5, 1500.0), (0.003, 128 ** -0.5, 6.0), (0.003, 128 ** -0.5, 0.01),
    (0.125, 4.0, 0.003), (0.125, 4.0, 1500.0), (1.0, 4.0, 0.02), (1.0, 4.0, 6.0), (0.125, 128 ** -0.5, 0.2),
]


def _run(name, dt, cap, scale, spread, tree):
    sl, nq, hq, hkv, bs = SHAPES[name]
    b = W.build_batch(sl, nq, hq, hkv, block_size=bs, dtype=dt, seed=13, device=DEV)
    b.query = (b.query.float() * spread).clamp(-6000, 6000).to(b.query.dtype)
    q = to_np_f32(b.query).astype(np.float64)
    rng = np.random.default_rng(2)
    masks = gfx906_fa.tree_masks([random_tree(rng, n) for n in nq]) if tree else None
    G, first = hq // hkv, np.concatenate([[0], np.cumsum(sl)])
    V = torch.empty(b.value.shape, dtype=torch.float32)
    for s in range(b.num_seqs):
        rows = np.arange(int(b.qsl[s]), int(b.qsl[s + 1]))[-32:]
        for h in range(hkv):
            K = seq_head_kv(b, s, h)[0].astype(np.float64)
            x = q[rows, h * G:(h + 1) * G].reshape(-1, 128)[-128:]
            V[first[s]:first[s + 1], h] = torch.from_numpy(telling_values(x, K, scale, cap, rng))
    b.value = V.to(b.value.dtype).to(DEV)
    kp, vp = b.planes()
    gfx906_fa.reshape_and_cache_q8_kv(b.key, b.value, b.slot_mapping, kp, vp)
    args = (b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t)
    rest = (b.max_query_len, b.max_seq_len, scale)
    if tree:
        out = gfx906_fa.tree_attention(*args, masks.to(DEV), *rest, soft_cap=cap, out_dtype=torch.float32)
    else:
        out = gfx906_fa.scored_paged_attention(*args, *rest, soft_cap=cap, out_dtype=torch.float32)
    out = to_np_f32(out).astype(np.float64)
    for s in range(b.num_seqs):
        n = int(b.q_lens[s])
        j = np.unique(np.concatenate([np.arange(min(n, 3)), np.arange(max(n - 33, 0), n), rng.integers(0, n, 8)]))
        t = int(b.qsl[s]) + j
        m = None if masks is None else masks.numpy()[t]
        seen = seen_keys(int(sl[s]), n, j, masks=m)
        for h in range(hkv):
            K, v = (x.astype(np.float64) for x in seq_head_kv(b, s, h))
            for e in range(h * G, (h + 1) * G):
                ref, bound = capped_rows(q[t, e], K, v, scale, cap, seen)
                off = np.abs(out[t, e] - ref)
                assert (off <= bound).all(), f"sequence {s} head {e}: {(off / bound).max():.2f} of the bound"


@pytest.mark.parametrize("cap,scale,spread", CAPS)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_capped(name, dt, cap, scale, spread):
    need_gpu()
    announce(f"capped scores {name} {dt} cap {cap} scale {scale:.3f} queries {spread}")
    _run(name, dt, cap, scale, spread, False)


@pytest.mark.parametrize("cap,scale,spread", [CAPS[0], CAPS[3], CAPS[5]])
@pytest.mark.parametrize("name", ["rows30", "rows48", "rows64", "tiles128", "tiles256", "split"])
def test_capped_trees(name, cap, scale, spread):
    need_gpu()
    announce(f"capped tree {name} cap {cap} scale {scale:.3f} queries {spread}")
    _run(name, "f16", cap, scale, spread, True)
