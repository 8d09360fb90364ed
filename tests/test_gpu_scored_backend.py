"""GPU: the backend's layers with capped or biased scores, trees of drafts, and
q/k norms, on both cache layouts."""
import math

import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from gpu_common import announce, need_gpu
from scored_common import check, eps_of, random_tree, scored_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _layer(impl_cls, layout, lens, nq, Hq, Hkv, **kw):
    """A batch whose keys lie in a backend cache of the layout, and its metadata."""
    from gfx906_fa_backend import Gfx906FABackend, Gfx906FAMetadata
    from gfx906_fa_paged import q8_planes
    args = dict(alibi_slopes=None, sliding_window=None, kv_cache_dtype="auto" if layout == "auto" else "q8_0")
    impl = impl_cls(Hq, 128, 1 / math.sqrt(128), Hkv, **{**args, **kw})
    b = W.build_batch(lens, nq, Hq, Hkv, block_size=32, dtype="bf16", seed=21, device=DEV)
    shape = Gfx906FABackend.get_kv_cache_shape(b.num_blocks, 32, Hkv, 128, layout)
    kv = torch.zeros(shape, dtype=torch.bfloat16 if layout == "auto" else torch.uint8, device=DEV)
    impl.do_kv_cache_update(None, b.key, b.value, kv, b.slot_mapping)
    md = Gfx906FAMetadata(num_actual_tokens=b.num_tokens, max_query_len=b.max_query_len, max_seq_len=b.max_seq_len,
                          query_start_loc=b.qsl_t, seq_lens=b.seq_lens_t, block_table=b.block_table,
                          slot_mapping=b.slot_mapping)
    kp, vp = q8_planes(kv, Hkv, 128)
    assert torch.equal(kp, b.kv_cache[:, 0]) and torch.equal(vp, b.kv_cache[:, 1])
    return impl, b, kv, md


def _forward(impl, b, kv, md):
    out = torch.empty((b.num_tokens + 2, b.Hq * 128), dtype=torch.bfloat16, device=DEV).fill_(3.0)
    q = torch.cat([b.query, b.query[:2]])  # a padded batch
    impl.forward(None, q, None, None, kv, md, output=out)
    assert (out[b.num_tokens:] == 3.0).all()
    return out[:b.num_tokens].view(b.num_tokens, b.Hq, 128)


@pytest.mark.parametrize("layout", ["auto", "q8_0"])
@pytest.mark.parametrize("form", ["cap", "alibi", "none"])
def test_layer_forward(form, layout):
    need_gpu()
    announce(f"backend {form} {layout}")
    from gfx906_fa_backend import Gfx906FAScoredImpl
    slopes = [2.0 ** -(i + 1) for i in range(8)]
    kw = dict(cap=dict(logits_soft_cap=2.5), alibi=dict(alibi_slopes=slopes), none={})[form]
    impl, b, kv, md = _layer(Gfx906FAScoredImpl, layout, [100, 333, 40], [1, 70, 3], 8, 2, **kw)
    okw = dict(cap=dict(cap=2.5), alibi=dict(slopes=np.array(slopes)), none={})[form]
    check(_forward(impl, b, kv, md), *scored_oracle(b, out_eps=eps_of(torch.bfloat16), **okw))


def test_layer_tree_step_and_kept_path():
    need_gpu()
    announce("backend tree")
    from gfx906_fa_backend import Gfx906FABackend, Gfx906FAImpl
    impl, b, kv, md = _layer(Gfx906FAImpl, "auto", [57, 90], [7, 7], 12, 2)
    rng = np.random.default_rng(2)
    trees = [random_tree(rng, 7) for _ in range(2)]
    masks = gfx906_fa.tree_masks(trees)
    md.tree_mask = torch.cat([masks, masks[:2]]).to(DEV)  # (padded, as the batch)
    check(_forward(impl, b, kv, md), *scored_oracle(b, masks=masks.numpy(), out_eps=eps_of(torch.bfloat16)))
    layers = [kv, kv.clone()]
    acc = torch.tensor([[0, 2, 5, -1], [1, 6, -1, -1]], dtype=torch.int32, device=DEV)
    Gfx906FABackend.keep_accepted_drafts(layers, 2, 128, md, acc, torch.tensor([3, 2], dtype=torch.int32, device=DEV))
    gfx906_fa.compact_draft_rows(b.kv_cache[None], md.block_table, md.seq_lens, md.query_start_loc, acc,
                                 torch.tensor([3, 2], dtype=torch.int32, device=DEV))
    from gfx906_fa_paged import q8_planes
    for x in layers:
        kp, vp = q8_planes(x, 2, 128)
        assert torch.equal(kp, b.kv_cache[:, 0]) and torch.equal(vp, b.kv_cache[:, 1])


def test_layer_norm_rope():
    need_gpu()
    announce("backend norm rope")
    from gfx906_fa_backend import Gfx906FAImpl
    from gfx906_fa_paged import q8_planes
    impl, b, kv, md = _layer(Gfx906FAImpl, "q8_0", [20, 9], [20, 9], 8, 2)
    T = b.num_tokens
    qkv = torch.randn((T + 3, 12 * 128), device=DEV).to(torch.bfloat16)
    w = [torch.rand(128, device=DEV).to(torch.bfloat16) for _ in range(2)]
    cs = W.rope_cos_sin_cache(64, 128, torch.bfloat16, DEV)
    pos = torch.arange(T + 3, device=DEV, dtype=torch.int32)
    mine = qkv.clone()
    impl.do_qk_norm_rope_and_kv_cache_update(None, mine[:, :1024], mine[:, 1024:1280], mine[:, 1280:], pos, *w, 1e-6, cs,
                                             True, kv, b.slot_mapping)
    x = qkv[:T].view(T, 12, 128)
    gfx906_fa.qk_norm_rope_and_cache_q8_kv(pos[:T].long(), x[:, :8], x[:, 8:10], x[:, 10:], *w, 1e-6, cs, True,
                                           b.slot_mapping, *b.planes())
    assert torch.equal(mine, qkv)
    kp, vp = q8_planes(kv, 2, 128)
    assert torch.equal(kp, b.kv_cache[:, 0]) and torch.equal(vp, b.kv_cache[:, 1])


def test_captured_layer_with_slopes():
    """The slopes come to the device before the capture (the profiling forward)."""
    need_gpu()
    announce("backend slopes graph")
    from gfx906_fa_backend import Gfx906FAScoredImpl
    slopes = [0.25] * 8
    impl, b, kv, md = _layer(Gfx906FAScoredImpl, "q8_0", [100, 200], [1, 1], 8, 2, alibi_slopes=slopes)
    out = torch.empty((2, 8 * 128), dtype=torch.bfloat16, device=DEV)
    impl.forward(None, b.query, None, None, kv, None, output=out)
    impl.reserve_workspace(gfx906_fa.workspace_size(2, 2, 8, 2, 1, 200), torch.device("cuda", 0))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        impl.forward(None, b.query, None, None, kv, md, output=out)
    for _ in range(3):
        b.query.mul_(-0.5)
        out.fill_(1.0)
        g.replay()
        torch.cuda.synchronize()
        check(out.view(2, 8, 128), *scored_oracle(b, slopes=np.array(slopes), out_eps=eps_of(torch.bfloat16)))
