"""GPU: tree steps through graphs captured from the metadata builder."""
import types

import numpy as np
import pytest
import torch

import gfx906_fa
from gpu_common import announce, need_gpu
from scored_common import check, eps_of, random_tree, scored_oracle
from test_gpu_scored_backend import _layer

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("cap", [0.0, 3.0])
@pytest.mark.parametrize("heads,n", [((12, 2), 7), ((6, 1), 30), ((8, 8), 1)])
def test_captured_step_replays_the_steps_masks(monkeypatch, heads, n, cap):
    """One captured uniform batch, replayed for trees, for a causal step between
    them, and for other trees: each as its eager step."""
    need_gpu()
    announce(f"tree graph of the builder {heads} {n} cap {cap}")
    from gfx906_fa_backend import Gfx906FAImpl, Gfx906FAMetadataBuilder, Gfx906FAScoredImpl
    from vllm.v1.attention.backend import CommonAttentionMetadata
    from vllm.v1.kv_cache_interface import AttentionSpec
    monkeypatch.setenv("GFX906_FA_TREES", "1")
    monkeypatch.setattr(Gfx906FAImpl, "_limits", None)
    cls, kw = (Gfx906FAScoredImpl, dict(logits_soft_cap=cap)) if cap else (Gfx906FAImpl, {})
    impl, b, kv, md = _layer(cls, "q8_0", [57 + n, 290 + n], [n, n], *heads, **kw)
    cfg = types.SimpleNamespace(scheduler_config=types.SimpleNamespace(max_num_seqs=2, max_num_batched_tokens=64))
    builder = Gfx906FAMetadataBuilder(AttentionSpec(block_size=32), ["l0"], cfg, torch.device("cuda", 0))
    common = CommonAttentionMetadata(query_start_loc=md.query_start_loc, seq_lens=md.seq_lens, num_reqs=2,
                                     num_actual_tokens=2 * n, max_query_len=n, max_seq_len=md.max_seq_len,
                                     block_table_tensor=md.block_table, slot_mapping=md.slot_mapping)
    out = torch.empty((2 * n, b.Hq * 128), dtype=torch.bfloat16, device=DEV)
    captured = builder.build_for_cudagraph_capture(common)
    impl.forward(None, b.query, None, None, kv, captured, output=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        impl.forward(None, b.query, None, None, kv, captured, output=out)
    rng = np.random.default_rng(6)
    for causal in (False, True, False, False, True):
        step = builder.build(0, common)
        masks = None
        if not causal:
            masks = gfx906_fa.tree_masks([random_tree(rng, n) for _ in range(2)])
            step.tree_mask = masks.to(DEV)
        eager = torch.empty_like(out)
        impl.forward(None, b.query, None, None, kv, step, output=eager)
        out.fill_(2.0)
        g.replay()
        torch.cuda.synchronize()
        ref, bound = scored_oracle(b, cap=cap, masks=None if causal else masks.numpy(), out_eps=eps_of(torch.bfloat16))
        check(out.view(2 * n, b.Hq, 128), ref, bound)
        check(eager.view(2 * n, b.Hq, 128), ref, bound)
        if not causal:
            assert torch.equal(out, eager)


def test_causal_sequences_beside_trees():
    """A tree step with a decode, a linear draft and prompt chunks of up to 64
    tokens, whose rows have the mask -1."""
    need_gpu()
    announce("tree step with causal sequences")
    from gfx906_fa_backend import Gfx906FAImpl
    lens, nq = [300, 64, 420, 64, 90], [7, 1, 64, 64, 5]
    impl, b, kv, md = _layer(Gfx906FAImpl, "auto", lens, nq, 12, 2)
    masks = torch.full((sum(nq),), -1, dtype=torch.int64)
    masks[:7] = gfx906_fa.tree_masks(random_tree(np.random.default_rng(4), 7))
    md.tree_mask = masks.to(DEV)
    out = torch.empty((b.num_tokens, b.Hq * 128), dtype=torch.bfloat16, device=DEV)
    impl.forward(None, b.query, None, None, kv, md, output=out)
    out = out.view(b.num_tokens, b.Hq, 128)
    check(out, *scored_oracle(b, masks=masks.numpy(), out_eps=eps_of(torch.bfloat16)))
    ref, bound = scored_oracle(b, out_eps=eps_of(torch.bfloat16))  # causal rows
    check(out[7:], ref[7:], bound[7:])
