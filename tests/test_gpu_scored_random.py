"""GPU: drawn batches of the scored attention forms against 64 bits: ragged and empty
sequences, more than 64 of them, head groups past a tile, positions before and
behind the keys, query views, rows past the last sequence, loose bounds; and
nothing written behind the workspace or the last sequence's rows."""
import random

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
HEADS = [(48, 8), (6, 1), (8, 4), (8, 1), (16, 16), (5, 1), (9, 3), (32, 1), (20, 1), (96, 1), (64, 8), (2, 2)]


def _draw(rng, tree):
    """(context, new tokens) of each sequence, heads and block size."""
    hq, hkv = rng.choice(HEADS)
    seqs = rng.choice([1, 2, 3, 9, 17, 66, 130])
    sizes = [1, 2, 5, 8, 11, 26, 33, 64] if tree else [1, 1, 1, 2, 5, 8, 17, 40, 130, 300]
    one = rng.choice(sizes)
    nq = [one] * seqs if rng.random() < 0.3 else [rng.choice([rng.choice(sizes), 1, 0]) for _ in range(seqs)]
    while sum(nq) * hq > 40000:
        nq = [n // 2 for n in nq]
    nq[rng.randrange(seqs)] += not sum(nq)
    most = max(1, 40000 // (seqs * hq))
    ctx = [rng.choice([0, 1, rng.randrange(40), rng.randrange(most), rng.randrange(most)]) for _ in nq]
    return ctx, nq, hq, hkv, rng.choice([16, 16, 32, 48, 64, 128])


@pytest.mark.parametrize("form", ["cap", "bias", "tree", "captree"])
@pytest.mark.parametrize("seed", range(8))
def test_drawn_batch(seed, form):
    need_gpu()
    rng, nr = random.Random(f"{seed} {form}"), np.random.default_rng(seed)
    tree = "tree" in form
    ctx, nq, hq, hkv, bs = _draw(rng, tree)
    announce(f"drawn {form} {seed}: {hq}/{hkv} bs {bs} ctx {ctx[:8]} nq {nq[:8]} of {len(nq)}")
    dt = rng.choice(["f16", "bf16"])
    b = W.build_batch([c + n for c, n in zip(ctx, nq)], nq, hq, hkv, block_size=bs, dtype=dt, seed=seed, device=DEV,
                      bt_pad_cols=rng.choice([0, 3]))
    b.kv_cache.fill_(0xFF)
    kp, vp = b.planes()
    gfx906_fa.reshape_and_cache_q8_kv(b.key, b.value, b.slot_mapping, kp, vp)
    T, past = b.num_tokens, rng.choice([0, 0, 5])
    most_q, most_k = b.max_query_len, b.max_seq_len
    if not tree and rng.random() < 0.3:
        most_q, most_k = most_q + rng.randrange(70), most_k + rng.randrange(2000)
    wide = torch.zeros((T + past, hq + 1, 136), dtype=TD[dt], device=DEV)
    wide[:T, :hq, :128] = b.query
    query = wide[:, :hq, :128] if rng.random() < 0.5 else wide[:, :hq, :128].contiguous()
    out_dtype = rng.choice([TD[dt], torch.float32])
    out = torch.full((T + past, hq, 128), 7.0, dtype=out_dtype, device=DEV)
    need = gfx906_fa.workspace_size(b.num_seqs, T + past, hq, hkv, most_q, most_k)
    ws = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device=DEV)
    cap = rng.choice([4.0, 30.0, 900.0]) if "cap" in form else 0.0
    args = (query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t)
    kw = dict(out=out, workspace=ws[:need], soft_cap=cap)
    eps = eps_of(out_dtype)
    if tree:
        masks = gfx906_fa.tree_masks([random_tree(nr, n) for n in nq])
        if rng.random() < 0.3:
            masks = torch.from_numpy(nr.integers(-2 ** 63, 2 ** 63, T, dtype=np.int64))
        m = torch.cat([masks, torch.zeros(past, dtype=torch.int64)]).to(DEV)
        gfx906_fa.tree_attention(*args, m, most_q, most_k, b.scale, **kw)
        want = scored_oracle(b, cap=cap, masks=masks.numpy(), out_eps=eps)
    else:
        causal, q_abs, slopes = rng.random() < 0.85, None, None
        if causal and rng.random() < 0.3:
            q_abs = nr.integers(-5, most_k + 5, b.num_seqs).astype(np.int32)
            kw["q_abs_offset"] = torch.from_numpy(q_abs).to(DEV)
        if form == "bias":
            slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], dtype=torch.float32)
            kw["alibi_slopes"] = slopes.to(DEV)
            slopes = slopes.numpy()
        gfx906_fa.scored_paged_attention(*args, most_q, most_k, b.scale, causal=causal, **kw)
        want = scored_oracle(b, cap=cap, slopes=slopes, q_abs=q_abs, causal=causal, out_eps=eps)
    torch.cuda.synchronize()
    assert (ws[need:] == 0xAB).all() and (out[T:] == 7.0).all()
    check(out[:T], *want)
