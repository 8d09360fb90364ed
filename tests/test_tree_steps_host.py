"""CPU: the metadata of tree steps, and the masks that captured graphs read."""
import copy
import dataclasses
import types

import pytest
import torch

import gfx906_fa
from gfx906_fa_backend import Gfx906FAImpl, Gfx906FAMetadata, Gfx906FAMetadataBuilder
from vllm.v1.attention.backend import CommonAttentionMetadata
from vllm.v1.kv_cache_interface import AttentionSpec

LIMITS = types.SimpleNamespace(scheduler_config=types.SimpleNamespace(max_num_seqs=4, max_num_batched_tokens=40))


@pytest.fixture(autouse=True)
def _flags(monkeypatch):
    monkeypatch.setattr(Gfx906FAImpl, "_captured", Gfx906FAImpl._captured)
    monkeypatch.setattr(Gfx906FAImpl, "_limits", None)


def _builder(cfg=LIMITS):
    return Gfx906FAMetadataBuilder(AttentionSpec(block_size=16), ["l0"], cfg, torch.device("cpu"))


def _step(n, seqs=2):
    return CommonAttentionMetadata(query_start_loc=torch.arange(seqs + 1, dtype=torch.int32) * n,
                                   seq_lens=torch.full((seqs,), 90, dtype=torch.int32), num_reqs=seqs,
                                   num_actual_tokens=seqs * n, max_query_len=n, max_seq_len=90,
                                   block_table_tensor=torch.zeros(seqs, 6, dtype=torch.int32),
                                   slot_mapping=torch.zeros(seqs * n, dtype=torch.int64))


def _masks(n, seqs=2):
    return gfx906_fa.tree_masks([[-1] + [0] * (n - 1)] * seqs)


def test_causal_graphs_refuse_masks(monkeypatch):
    """A graph captured without masks would replay a tree step as a causal one."""
    monkeypatch.delenv("GFX906_FA_TREES", raising=False)
    b = _builder()
    b.build(0, _step(5)).tree_mask = _masks(5)  # nothing captured: eager steps
    assert b.build_for_cudagraph_capture(_step(5)).tree_mask is None
    md = b.build(0, _step(5))
    with pytest.raises(RuntimeError, match="GFX906_FA_TREES"):
        dataclasses.replace(md, tree_mask=_masks(5))
    for step in (md, copy.copy(md), copy.deepcopy(md), dataclasses.replace(md)):
        with pytest.raises(RuntimeError, match="GFX906_FA_TREES"):
            step.tree_mask = _masks(5)
        assert step.tree_mask is None
        step.tree_mask = None
    other = b.build(0, _step(4))  # (no graph of that length: eager)
    other.tree_mask = _masks(4)
    assert torch.equal(other.tree_mask, _masks(4))


def test_graphs_read_the_steps_masks(monkeypatch):
    monkeypatch.setenv("GFX906_FA_TREES", "1")
    b = _builder()
    seen = b.build_for_cudagraph_capture(_step(5)).tree_mask  # what the captured launches read
    assert seen.shape == (10,) and (seen == -1).all()
    md = b.build(0, _step(5))
    assert md.tree_mask is None
    md.tree_mask = torch.cat([_masks(5), _masks(5)[:3]])  # (a padded batch's)
    assert torch.equal(seen, _masks(5)) and md.tree_mask.shape == (13,)
    md.tree_mask = -_masks(5)
    assert torch.equal(seen, -_masks(5))
    dataclasses.replace(md, tree_mask=_masks(5))
    assert torch.equal(seen, _masks(5))
    md = b.build(0, _step(5))  # a causal step after it
    assert (seen == -1).all()
    md.tree_mask = _masks(5)
    md.tree_mask = None
    assert (seen == -1).all()
    short = b.build(0, _step(5, seqs=1))
    short.tree_mask = _masks(5, seqs=1)
    assert torch.equal(seen[:5], _masks(5, seqs=1)) and (seen[5:] == -1).all()
    captured = b.build_for_cudagraph_capture(_step(5))
    assert captured.tree_mask.data_ptr() == seen.data_ptr() and (seen == -1).all()
    md = b.build(0, _step(5))
    md.tree_mask = _masks(5)
    assert dataclasses.replace(captured).tree_mask.data_ptr() == seen.data_ptr() and torch.equal(seen, _masks(5))
    for bad in (_masks(5).int(), _masks(5)[:-1], _masks(5)[None]):
        with pytest.raises(RuntimeError, match="int64"):
            b.build(0, _step(5)).tree_mask = bad
    md = b.build(0, _step(5))
    md.tree_mask = _masks(5)
    with pytest.raises(RuntimeError, match="int64"):  # a refused mask changes nothing
        md.tree_mask = _masks(5).int()
    assert torch.equal(seen, _masks(5)) and torch.equal(md.tree_mask, _masks(5))
    with pytest.raises(RuntimeError, match="max_num_batched_tokens"):
        b.build(0, _step(30)).tree_mask = _masks(30)
    with pytest.raises(RuntimeError, match="max_num_batched_tokens"):
        b.build_for_cudagraph_capture(_step(30))


def test_trees_need_the_limits(monkeypatch):
    monkeypatch.setenv("GFX906_FA_TREES", "1")
    with pytest.raises(ValueError, match="max_num_batched_tokens"):
        _builder(None)


def test_metadata_made_by_hand():
    """Without a builder there are no graphs to reach: the mask is the caller's."""
    args = dict(num_actual_tokens=10, max_query_len=5, max_seq_len=90, query_start_loc=None, seq_lens=None,
                block_table=None, slot_mapping=None)
    m = _masks(5)
    md = Gfx906FAMetadata(**args, tree_mask=m)
    assert md.tree_mask is m
    md.tree_mask = None
    assert md.tree_mask is None
    assert dataclasses.replace(md, tree_mask=m).tree_mask is m


@pytest.mark.parametrize("trees", ["0", "1"])
def test_no_mask_beside_a_longer_chunk(monkeypatch, trees):
    """A row's mask has 64 bits: metadata of longer chunks refuses masks, before
    any layer runs."""
    monkeypatch.setenv("GFX906_FA_TREES", trees)
    step = _step(65, seqs=1)
    cfg = types.SimpleNamespace(scheduler_config=types.SimpleNamespace(max_num_seqs=4, max_num_batched_tokens=400))
    md = _builder(cfg).build(0, step)
    with pytest.raises(RuntimeError, match="64 query tokens"):
        md.tree_mask = torch.full((65,), -1, dtype=torch.int64)
    assert md.tree_mask is None
    assert _builder(cfg).build_for_cudagraph_capture(step).tree_mask is None
    fields = {f.name: getattr(md, f.name) for f in dataclasses.fields(md) if f.name != "graph_masks"}
    with pytest.raises(RuntimeError, match="64 query tokens"):
        Gfx906FAMetadata(**{**fields, "tree_mask": torch.full((65,), -1, dtype=torch.int64)})
