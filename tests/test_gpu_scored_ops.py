"""GPU: the scored, tree, norm, draft-row and read functions as torch custom
ops: the same results, declared writes (opcheck), and calls on two streams at
once with a workspace each."""
import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from gpu_common import announce, need_gpu
from scored_common import random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"
OPS = torch.ops.gfx906_fa
CHECKS = ("test_schema", "test_faketensor")


def test_attention_ops():
    need_gpu()
    announce("scored ops")
    b = W.build_batch([70, 33], [5, 5], 6, 1, dtype="f16", seed=3, device=DEV)
    kp, vp = b.planes()
    args = (b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t)
    size = (b.max_query_len, b.max_seq_len, b.scale)
    ws = gfx906_fa.new_workspace(gfx906_fa.workspace_size(2, 10, 6, 1, 5, 70), DEV)
    sl = torch.rand(6, device=DEV)
    masks = gfx906_fa.tree_masks([random_tree(np.random.default_rng(i), 5) for i in range(2)]).to(DEV)
    for cap, slopes in ((2.0, None), (0.0, sl)):
        want = gfx906_fa.scored_paged_attention(*args, *size, cap, slopes)
        assert torch.equal(OPS.scored_paged_attention(*args, *size, cap, slopes, None), want)
        assert torch.equal(OPS.scored_paged_attention(*args, *size, cap, slopes, ws), want)
    assert torch.equal(OPS.tree_attention(*args, masks, *size, 3.0, ws),
                       gfx906_fa.tree_attention(*args, masks, *size, soft_cap=3.0))
    torch.library.opcheck(OPS.scored_paged_attention, (*args, *size, 2.0, None, ws), test_utils=CHECKS)
    torch.library.opcheck(OPS.tree_attention, (*args, masks, *size, 0.0, ws), test_utils=CHECKS)


def test_row_ops():
    need_gpu()
    announce("row ops")
    b = W.build_batch([40, 20], [6, 6], 8, 2, dtype="bf16", seed=3, device=DEV)
    kp, vp = b.planes()
    k, v = OPS.read_cache_q8_kv(b.slot_mapping, kp, vp, torch.float32)
    want = gfx906_fa.read_cache_q8_kv(b.slot_mapping, kp, vp, torch.float32)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    torch.library.opcheck(OPS.read_cache_q8_kv, (b.slot_mapping, kp, vp, torch.bfloat16), test_utils=CHECKS)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    acc, cnt = t([[1, 2, 5], [0, 4, 5]]), t([3, 2])
    one, two = (b.kv_cache[None].clone() for _ in range(2))
    OPS.compact_draft_rows(one, b.block_table, b.seq_lens_t, b.qsl_t, acc, cnt)
    gfx906_fa.compact_draft_rows(two, b.block_table, b.seq_lens_t, b.qsl_t, acc, cnt)
    assert torch.equal(one, two) and not torch.equal(one, b.kv_cache[None])
    torch.library.opcheck(OPS.compact_draft_rows, (one, b.block_table, b.seq_lens_t, b.qsl_t, acc, cnt), test_utils=CHECKS)
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    cs = W.rope_cos_sin_cache(64, 128, torch.bfloat16, DEV)
    pos = torch.arange(12, device=DEV)
    sets = []
    for f in (OPS.qk_norm_rope_and_cache_q8_kv, gfx906_fa.qk_norm_rope_and_cache_q8_kv):
        q, key, value, c = b.query.clone(), b.key[:12].clone(), b.value[:12].clone(), b.kv_cache.clone()
        f(pos, q, key, value, w, w, 1e-5, cs, False, b.slot_mapping[:12], c[:, 0], c[:, 1])
        sets.append((q, key, c))
    assert all(torch.equal(x, y) for x, y in zip(*sets))


def test_two_streams_at_once():
    need_gpu()
    announce("two streams")
    bs = [W.build_batch([900 + i, 64], [7, 7], 12, 2, dtype="bf16", seed=i, device=DEV) for i in range(2)]
    masks = gfx906_fa.tree_masks([random_tree(np.random.default_rng(5), 7)] * 2).to(DEV)
    call = lambda b, **kw: gfx906_fa.tree_attention(b.query, *b.planes(), b.block_table, b.seq_lens_t, b.qsl_t, masks,  # noqa: E731,E501
                                                    7, b.max_seq_len, b.scale, **kw)
    want = [call(b) for b in bs]
    ws = [gfx906_fa.new_workspace(gfx906_fa.workspace_size(2, 14, 12, 2, 7, 901), DEV) for _ in bs]
    outs = [torch.zeros_like(x) for x in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in bs]
    for _ in range(5):
        for st, b, w, o in zip(streams, bs, ws, outs):
            with torch.cuda.stream(st):
                call(b, out=o, workspace=w)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
