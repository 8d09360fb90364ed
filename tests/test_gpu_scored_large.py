"""GPU: the scored forms, the norm's cache write, rows back and draft rows on pages
past 4 GiB: bit for bit what they give on a small cache.  And sequences of 131072
keys against 64 bits."""
import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from gpu_common import announce, need_gpu
from scored_common import check, eps_of, random_tree, scored_oracle
from test_gpu_large_cache import _relocate

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bs", [16, 64])
def test_attention(bs):
    need_gpu()
    announce(f"large scored attention bs={bs}")
    b = W.build_batch([5, 300, 1500, 700, 33, 4000], [1, 1, 5, 60, 33, 1], 12, 2, block_size=bs, seed=43)
    kp, vp = b.planes()
    big, _, bt, _ = _relocate(b)
    masks = gfx906_fa.tree_masks([random_tree(np.random.default_rng(1), int(n)) for n in b.q_lens]).to(DEV)
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(12)], device=DEV)
    rest = (b.max_query_len, b.max_seq_len, b.scale)
    seqs = (b.seq_lens_t, b.qsl_t)
    for kw in (dict(soft_cap=20.0), dict(alibi_slopes=slopes)):
        out = [gfx906_fa.scored_paged_attention(b.query, k, v, t, *seqs, *rest, **kw)
               for k, v, t in ((kp, vp, b.block_table), (big[:, 0], big[:, 1], bt))]
        assert torch.equal(*out)
    out = [gfx906_fa.tree_attention(b.query, k, v, t, *seqs, masks, *rest)
           for k, v, t in ((kp, vp, b.block_table), (big[:, 0], big[:, 1], bt))]
    assert torch.equal(*out)


def test_rows():
    need_gpu()
    announce("large rows")
    b = W.build_batch([70, 1000, 33], [30, 64, 5], 8, 2, seed=44)
    kp, vp = b.planes()
    big, base, bt, slots = _relocate(b)
    for s in (b.slot_mapping, b.slot_mapping[torch.randperm(b.slot_mapping.shape[0], device=DEV)]):
        small = gfx906_fa.read_cache_q8_kv(s, kp, vp)
        far = gfx906_fa.read_cache_q8_kv(s + base * b.block_size, big[:, 0], big[:, 1])
        assert torch.equal(small[0], far[0]) and torch.equal(small[1], far[1])
    T = b.key.shape[0]
    w = torch.ones(128, dtype=torch.float16, device=DEV)
    cs = W.rope_cos_sin_cache(T, 128, torch.float16, DEV)
    for c, s in ((b.kv_cache, b.slot_mapping), (big, slots)):
        q, k = torch.ones(T, 8, 128, dtype=torch.float16, device=DEV), b.key.clone()
        gfx906_fa.qk_norm_rope_and_cache_q8_kv(torch.arange(T, device=DEV), q, k, b.value, w, w, 1e-6, cs, True, s,
                                               c[:, 0], c[:, 1])
    assert torch.equal(big[base:], b.kv_cache)
    acc = torch.tensor([[0, 2, 3, 11, 29], [63, 1, 0, 7, 5], [1, 2, -1, -1, -1]], dtype=torch.int32, device=DEV)
    count = torch.tensor([5, 5, 2], dtype=torch.int32, device=DEV)
    gfx906_fa.compact_draft_rows([(kp, vp)], b.block_table, b.seq_lens_t, b.qsl_t, acc, count)
    gfx906_fa.compact_draft_rows([(big[:, 0], big[:, 1])], bt, b.seq_lens_t, b.qsl_t, acc, count)
    assert torch.equal(big[base:], b.kv_cache)


def test_layers_past_4gib():
    """A stack of layers whose later ones start past 4 GiB."""
    need_gpu()
    announce("large layers")
    nb, layers = 600_000, 3  # 2.4 GiB a layer
    stack = torch.zeros((layers, nb, 2, 1, 2176), dtype=torch.uint8, device=DEV)
    assert (layers - 1) * stack.stride(0) > 1 << 32
    page = torch.randint(0, 256, (2, 1, 2176), dtype=torch.uint8, device=DEV)
    for c in stack:
        c[0] = c[nb - 1] = page
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    gfx906_fa.compact_draft_rows(stack, t([[nb - 1], [0]]), t([14, 14]), t([0, 11, 22]), t([[0, 4, 6, 9]] * 2), t([4, 4]))
    one = page.clone()[None, None]
    gfx906_fa.compact_draft_rows(one, t([[0]]), t([14]), t([0, 11]), t([[0, 4, 6, 9]]), t([4]))
    assert not torch.equal(one[0, 0], page)
    for c in stack:
        assert torch.equal(c[0], one[0, 0]) and torch.equal(c[nb - 1], one[0, 0])
        assert not c[1].any() and not c[nb - 2].any()


@pytest.mark.parametrize("form", ["cap", "bias", "tree"])
@pytest.mark.parametrize("nq", [1, 11, 60])
def test_long_context(form, nq):
    need_gpu()
    announce(f"long context {form} {nq}")
    b = W.build_batch([131072 - 5, 300], [nq, nq], 3, 1, block_size=16, dtype="bf16", seed=nq, device=DEV)
    args = (b.query, *b.planes(), b.block_table, b.seq_lens_t, b.qsl_t)
    rest = (b.max_query_len, b.max_seq_len, b.scale)
    eps = eps_of(torch.bfloat16)
    if form == "tree":
        masks = gfx906_fa.tree_masks([random_tree(np.random.default_rng(nq), nq) for _ in range(2)])
        out = gfx906_fa.tree_attention(*args, masks.to(DEV), *rest)
        check(out, *scored_oracle(b, masks=masks.numpy(), out_eps=eps))
    elif form == "cap":
        out = gfx906_fa.scored_paged_attention(*args, *rest, soft_cap=30.0)
        check(out, *scored_oracle(b, cap=30.0, out_eps=eps))
    else:
        slopes = torch.tensor([2.0 ** -4, 2.0 ** -12, 2.0 ** -18])  # 16, 4096 and all keys in reach
        out = gfx906_fa.scored_paged_attention(*args, *rest, alibi_slopes=slopes.to(DEV))
        check(out, *scored_oracle(b, slopes=slopes.numpy(), out_eps=eps))
