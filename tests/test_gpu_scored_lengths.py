"""GPU: scored decodes whose max_seq_len does not bound the lengths on the
device, or says nothing (0).  Short contexts are taken a segment a workgroup,
without a merge: that must not depend on the lengths being short."""
import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from gpu_common import announce, need_gpu, to_np_f32
from scored_common import U, check, random_tree, scored_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (keys, query tokens, heads, kv-heads)
SHAPES = {
    "decode": ([3000, 1, 700], [1, 1, 1], 16, 4),
    "rows30": ([2500, 40], [5, 5], 6, 1),
    "rows48": ([2100, 8], [8, 8], 6, 1),
    "rows64": ([2000], [8], 8, 1),
    "many": ([2000] + [30] * 31, [1] * 32, 32, 8),
    "mixed": ([1500, 900, 40], [1, 5, 11], 6, 1),
}


@pytest.mark.parametrize("said", [0, 1, 200])
@pytest.mark.parametrize("form", ["cap", "bias", "tree"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_max_seq_len_below_the_lengths(name, form, said):
    need_gpu()
    announce(f"max_seq_len {said} {form} {name}")
    sl, nq, hq, hkv = SHAPES[name]
    b = W.build_batch(sl, nq, hq, hkv, dtype="f16", seed=7, device=DEV)
    args = (b.query, *b.planes(), b.block_table, b.seq_lens_t, b.qsl_t)
    rest = (b.max_query_len, said, b.scale)
    out = torch.full((b.num_tokens, hq, 128), float("nan"), device=DEV)
    if form == "tree":
        m = gfx906_fa.tree_masks([random_tree(np.random.default_rng(1), n) for n in nq])
        gfx906_fa.tree_attention(*args, m.to(DEV), *rest, out=out)
        check(out, *scored_oracle(b, masks=m.numpy()))
    elif form == "cap":
        gfx906_fa.scored_paged_attention(*args, *rest, soft_cap=4.0, out=out)
        check(out, *scored_oracle(b, cap=4.0))
    else:
        slopes = torch.tensor([2.0 ** -(i % 8 + 1) for i in range(hq)], device=DEV)
        gfx906_fa.scored_paged_attention(*args, *rest, alibi_slopes=slopes, out=out)
        check(out, *scored_oracle(b, slopes=slopes.cpu().numpy()))


def test_a_million_keys_said_to_be_one():
    """More keys than the one-piece plan once took: every row is written."""
    need_gpu()
    announce("a million keys, max_seq_len 1")
    n, hq, cap = (1 << 20) + 5000, 2, 3.0
    b = W.build_batch([n], [1], hq, 1, block_size=64, dtype="f16", seed=9, device=DEV, host_values=False)
    kp, vp = b.planes()
    out = torch.full((1, hq, 128), float("nan"), device=DEV)
    gfx906_fa.scored_paged_attention(b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, 1, 1, b.scale, soft_cap=cap,
                                     out=out)
    K, V = (x[:, 0] for x in gfx906_fa.read_cache_q8_kv(b.slot_mapping, kp, vp, torch.float32))  # (exact in fp32)
    q = b.query[0].double()
    ref, bound = np.zeros((1, hq, 128)), np.zeros((1, hq, 128))
    small = n * 2.0 ** -25 * (float(V.abs().max()) + 127)
    for h in range(hq):
        s = (K.double() @ q[h]) * b.scale
        p = torch.softmax(cap * torch.tanh(s / cap), 0)
        ds = U * b.scale * float((K.double().abs() @ q[h].abs()).max())
        ref[0, h] = (p @ V.double()).cpu().numpy()
        bound[0, h] = (2 * ds + 3 * U + 2.0 ** -16) * (1 + 2 * ds) * (p @ V.double().abs()).cpu().numpy() + small
    o = to_np_f32(out)
    assert np.isfinite(o).all()
    assert (np.abs(o - ref) <= bound).all()
