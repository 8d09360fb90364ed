"""CPU: the scored, tree, norm, draft-row and read entries' checks, tree masks,
and the 64-bit oracle's own visibility rules (no GPU work)."""
import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gfx906_fa

OPS = torch.ops.gfx906_fa


def test_tree_masks():
    m = gfx906_fa.tree_masks([[-1, 0, 0, 2, -1], [-1]])
    assert m.tolist() == [1, 3, 5, 13, 16, 1] and m.dtype == torch.int64
    chain = gfx906_fa.tree_masks(list(range(-1, 63)))
    assert chain[-1] == -1 and chain[62] == 2 ** 63 - 1
    assert gfx906_fa.tree_masks([]).numel() == 0
    for bad in ([0], [-1, 1], [-2], [-1] * 65):
        with pytest.raises(RuntimeError):
            gfx906_fa.tree_masks(bad)
    tree = torch.tensor([-1, 0, 0, 2])
    for same in (tree, tree.numpy(), list(tree.numpy()), [tree], [tree.numpy()], tree[None]):
        assert gfx906_fa.tree_masks(same).tolist() == [1, 3, 5, 13]


def test_oracle_visibility():
    from scored_common import seen_keys
    m = gfx906_fa.tree_masks([-1, 0, 0]).numpy()
    s = seen_keys(5, 3, np.arange(3), masks=m)
    assert s.tolist() == [[True, True, True, False, False], [True, True, True, True, False],
                          [True, True, True, False, True]]
    assert seen_keys(3, 2, np.arange(2), 1).tolist() == [[True, True, False], [True, True, True]]


def _scored(**kw):
    """The C entry with null pointers: refused, or nothing to do, before any GPU work."""
    a = dict(q=None, qdt=1, qts=0, qhs=0, k=None, v=None, cbs=0, chs=0, bt=None, bts=0, sl=None, qsl=None, qa=None, causal=1,
             cap=0.0, slopes=None, tree=None, B=1, T=1, Hq=8, Hkv=1, D=128, bs=16, mq=1, mk=16, scale=0.1, out=None, odt=1,
             ots=0, ohs=0, ws=None, wsb=0, stream=None)
    a.update(kw)
    return gfx906_fa.lib().gfx906_fa_amd_scored_paged_attention(*a.values())


def test_scored_entry_refusals():
    p = ctypes.c_void_p(256)
    assert _scored(T=0, cap=5.0) == 0
    for kw in (dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(cap=1e-44), dict(cap=1025.0), dict(cap=0.003), dict(cap=1.0, scale=1e-5), dict(cap=1.0, scale=float("nan")), dict(cap=2.0, slopes=p),
               dict(slopes=p, tree=p), dict(tree=p, mq=65), dict(tree=p, qa=p), dict(tree=p, causal=0),
               dict(cap=2.0, qdt=0, odt=0), dict(cap=2.0, qdt=1, odt=2), dict(cap=2.0, qdt=2, odt=1), dict(cap=2.0, D=64),
               dict(cap=2.0, bs=24), dict(cap=2.0, Hq=9, Hkv=2), dict(cap=2.0, wsb=128)):
        assert _scored(**kw) == 1, kw


def test_norm_rope_entry_refusals():
    f = gfx906_fa.lib().gfx906_fa_amd_qk_norm_rope_cache_write_kv
    good = [None, None, None, None, None, 1e-6, 1, None, None, 1, 128, 4096, 128, 1, None, None, None, 0, 8, 2, 128, 16,
            4, 0, 0, 0, 0, 0, 0, 0, 0, None]
    assert f(*good) == 0
    for at, value in ((3, ctypes.c_void_p(8)), (4, ctypes.c_void_p(2)), (5, -1.0), (5, float("nan")), (6, 0), (12, 72),
                      (12, 256), (20, 64), (21, 24)):
        bad = list(good)
        bad[at] = value
        assert f(*bad) == 1, (at, value)


def test_row_entries_refusals():
    L = gfx906_fa.lib()
    p = ctypes.c_void_p(256)
    read = [p, p, p, p, p, 1, 0, 1, 128, 16, 4, 4352, 2176, 128, 128, 128, 128, None]
    assert L.gfx906_fa_amd_read_rows(*read) == 0
    for at, value in ((0, ctypes.c_void_p(8)), (3, ctypes.c_void_p(8)), (5, 3), (6, -1), (7, 0), (8, 64), (9, 24), (10, -1),
                      (11, 4), (13, 4)):
        bad = list(read)
        bad[at] = value
        assert L.gfx906_fa_amd_read_rows(*bad) == 1, (at, value)
    comp = [None, None, p, p, 8704, 0, 4352, 2176, 4, p, 2, 2, p, p, p, 4, 4, p, 1, 1, 128, 16, None]
    assert L.gfx906_fa_amd_compact_draft_rows(*comp) == 0   # no layers
    for at, value in ((2, ctypes.c_void_p(8)), (0, (ctypes.c_void_p * 1)(256)), (4, 8), (5, -1), (6, 8), (8, -1), (11, -1),
                      (16, 65), (18, -1), (19, 0), (20, 64), (21, 20)):
        bad = list(comp)
        bad[at] = value
        assert L.gfx906_fa_amd_compact_draft_rows(*bad) == 1, (at, value)


def test_compact_refuses_one_cache_as_two_layers():
    L = gfx906_fa.lib()
    p = ctypes.c_void_p(256)
    rest = [4352, 2176, 4, p, 2, 2, p, p, p, 4, 4, p, 1, 1, 128, 16, None]
    assert L.gfx906_fa_amd_compact_draft_rows(None, None, p, p, 0, 2, *rest) == 1
    planes = lambda *a: (ctypes.c_void_p * len(a))(*a)  # noqa: E731
    far = [1 << 20 | i << 8 for i in range(70)]
    for k, v in (([256, 256], [512, 1024]), ([256, 512], [1024, 1024]), (far[:69] + far[:1], [x + 65536 for x in far])):
        assert L.gfx906_fa_amd_compact_draft_rows(planes(*k), planes(*v), None, None, 0, len(k), *rest) == 1


def test_host_tensors_are_refused():
    q = torch.zeros(1, 8, 128, dtype=torch.float16)
    c = torch.zeros(1, 1, 2176, dtype=torch.uint8)
    i, n = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    w = torch.ones(128, dtype=torch.float16)
    for call in (lambda: gfx906_fa.scored_paged_attention(q, c, c, i[None], i[:1], i, 1, 1, 0.1, soft_cap=1.0),
                 lambda: gfx906_fa.tree_attention(q, c, c, i[None], i[:1], i, n, 1, 1, 0.1),
                 lambda: gfx906_fa.qk_norm_rope_and_cache_q8_kv(n, q, q[:, :1], q[:, :1], w, w, 1e-6, w[None], True, n, c, c),
                 lambda: gfx906_fa.read_cache_q8_kv(n, c, c),
                 lambda: gfx906_fa.compact_draft_rows([(c, c)], i[None], i[:1], i, i[None], i)):
        with pytest.raises(RuntimeError, match="CUDA/HIP"):
            call()
    with pytest.raises(RuntimeError, match="tree_mask"):
        gfx906_fa.tree_attention(q, c, c, i[None], i[:1], i, None, 1, 1, 0.1)


def test_custom_ops():
    writes = {"scored_paged_attention": {"workspace"}, "tree_attention": {"workspace"},
              "qk_norm_rope_and_cache_q8_kv": {"query", "key", "key_cache", "value_cache"}, "read_cache_q8_kv": set(),
              "compact_draft_rows": {"kv_caches"}}
    assert set(gfx906_fa.SCORED_TORCH_OPS) == set(writes)
    for name, want in writes.items():
        schema = getattr(OPS, name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == want
    mode = FakeTensorMode()
    with mode:
        e = lambda shape, dt: torch.empty(shape, dtype=dt, device="cuda")  # noqa: E731
        q, c, i = e((5, 8, 128), torch.bfloat16), e((3, 2, 2, 2176), torch.uint8), e((2,), torch.int32)
        args = (q, c[:, 0], c[:, 1], e((1, 3), torch.int32), i[:1], i)
        o = OPS.scored_paged_attention(*args, 5, 9, 0.1, 3.0, None, None, out_dtype=torch.float32)
        assert o.shape == q.shape and o.dtype == torch.float32
        o = OPS.tree_attention(*args, e((5,), torch.int64), 5, 9, 0.1, 0.0, None)
        assert o.shape == q.shape and o.dtype == torch.bfloat16
        k, v = OPS.read_cache_q8_kv(e((7,), torch.int64), c[:, 0], c[:, 1], torch.float16)
        assert k.shape == v.shape == (7, 2, 128) and k.dtype == torch.float16


def test_backend_takes_the_score_forms(monkeypatch):
    import gfx906_fa_backend as B
    args = dict(num_heads=8, head_size=128, scale=0.1, num_kv_heads=1, alibi_slopes=None, sliding_window=None,
                kv_cache_dtype="auto")
    assert B.Gfx906FAScoredBackend.get_impl_cls() is B.Gfx906FAScoredImpl
    assert B.Gfx906FAScoredImpl(**args, logits_soft_cap=30.0).soft_cap == 30.0
    impl = B.Gfx906FAScoredImpl(**{**args, "alibi_slopes": [0.5] * 8})
    assert impl._slopes(torch.device("cpu")).tolist() == [0.5] * 8 and impl.soft_cap == 0.0
    assert B.Gfx906FAScoredImpl(**args)._slopes(torch.device("cpu")) is None
    for err, kw in ((ValueError, dict(alibi_slopes=[0.5])), (ValueError, dict(logits_soft_cap=-1.0)),
                    (ValueError, dict(logits_soft_cap=float("inf"))),
                    (NotImplementedError, dict(logits_soft_cap=2.0, alibi_slopes=[0.5] * 8)),
                    (NotImplementedError, dict(sliding_window=64)), (NotImplementedError, dict(use_alibi_sqrt=True)),
                    (NotImplementedError, dict(sinks=torch.zeros(8)))):
        with pytest.raises(err):
            B.Gfx906FAScoredImpl(**{**args, **kw})
    names = []
    import vllm.v1.attention.backends.registry as R
    monkeypatch.setattr(R, "register_backend", lambda where, name: names.append(name))
    B.register()
    monkeypatch.setenv("GFX906_FA_SCORES", "1")
    B.register()
    assert [n.rsplit(".", 1)[1] for n in names] == ["Gfx906FABackend", "Gfx906FAScoredBackend"]
