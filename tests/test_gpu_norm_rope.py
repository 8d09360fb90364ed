"""GPU: RMS norms of query and key heads, rotation and cache write in one pass.

Query and key against 64 bits; the cache byte for byte against the write of the
key as stored.  Bound of an element, besides the output's half step: the sum of
128 squares (12 roundings, halved by the root), the reciprocal root (2), the
products with it and the weight (2), the rotation's product and sum (2) and
their slack: 16 * 2^-24 of the values that are combined."""
import numpy as np
import pytest
import torch

import gfx906_fa
from gpu_common import announce, host_bits, need_gpu
from oracle import q8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TD = {"f16": torch.float16, "bf16": torch.bfloat16}


def _inputs(dt, T, Hq, Hkv, rot, cs_dtype, seed, P=4096, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((T, Hq + 2 * Hkv, 128), generator=g) * spread).to(TD[dt]).to(DEV)
    wq, wk = ((1 + 0.3 * torch.randn(128, generator=g)).to(TD[dt]).to(DEV) for _ in range(2))
    cs = torch.from_numpy(O.rope_cos_sin_cache(P, rot)).to(torch.float32 if cs_dtype == "f32" else TD[dt]).to(DEV)
    pos = torch.randint(0, P, (T,), generator=g)
    return qkv, wq, wk, cs, pos


def _ref(x, w, eps, pos, cs, rot, neox):
    """(value, magnitude of what is combined) in 64 bits."""
    x, w, cs = (t.double().cpu() for t in (x, w, cs))
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    ok = (pos >= 0) & (pos < cs.shape[0])
    row = cs[pos.clamp(0, cs.shape[0] - 1)]
    c, s = row[:, None, :rot // 2], row[:, None, rot // 2:rot]
    z, mag = y.clone(), y.abs()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
    u, v = y[..., a], y[..., b]
    z[..., a], z[..., b] = u * c - v * s, v * c + u * s
    mag[..., a] = mag[..., b] = u.abs() + v.abs()
    keep = ok[:, None, None]
    return torch.where(keep, z, y), torch.where(keep, mag, y.abs())


def _assert_rows(out, ref, mag):
    half = torch.finfo(out.dtype).eps / 2
    fp32 = 16 * 2.0 ** -24 * mag
    bound = half * (ref.abs() + fp32) + fp32 + (2.0 ** -25 if out.dtype == torch.float16 else 0.0)
    off = (out.double().cpu() - ref).abs()
    assert (off <= bound).all(), float((off - bound).max())


def _run(dt, T, Hq, Hkv, rot, neox, cs_dtype, bs=16, seed=0, eps=1e-6, spread=2.0, edges=True):
    qkv, wq, wk, cs, pos = _inputs(dt, T, Hq, Hkv, rot, cs_dtype, seed, spread=spread)
    NB = T // bs + 2
    slots = torch.from_numpy(np.random.default_rng(seed).permutation(NB * bs)[:T].astype(np.int64))
    if edges and T > 8:
        pos[2], pos[5], pos[7] = -1, cs.shape[0], 0
        slots[1] = slots[T - 1] = -1
        slots[4] = NB * bs  # past the cache: not written
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]  # views of one projection
    q0, k0, v0 = (t.clone() for t in (q, k, v))
    cache = torch.full((NB, 2, Hkv, bs // 16 * 2176), 0x5A, dtype=torch.uint8, device=DEV)
    gfx906_fa.qk_norm_rope_and_cache_q8_kv(pos.to(DEV), q, k, v, wq, wk, eps, cs, neox, slots.to(DEV), cache[:, 0],
                                           cache[:, 1], rot_dim=rot)
    torch.cuda.synchronize()
    _assert_rows(q, *_ref(q0, wq, eps, pos, cs, rot, neox))
    _assert_rows(k, *_ref(k0, wk, eps, pos, cs, rot, neox))
    assert torch.equal(v, v0)
    exp = np.full(tuple(cache.shape), 0x5A, np.uint8)
    O.planar_cache_write(host_bits(k.contiguous()), host_bits(v0), np.where(slots.numpy() < NB * bs, slots.numpy(), -1), exp)
    assert np.array_equal(cache.cpu().numpy(), exp)


@pytest.mark.parametrize("cs_dtype", ["f32", "model"])
@pytest.mark.parametrize("rot", [128, 96, 64, 16])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_norm_rope(dt, neox, rot, cs_dtype):
    need_gpu()
    announce(f"norm rope {dt} neox={neox} rot={rot} cs={cs_dtype}")
    _run(dt, 45, 8, 2, rot, neox, cs_dtype, seed=rot + neox)


@pytest.mark.parametrize("T,Hq,Hkv,bs", [(1, 6, 1, 16), (3, 5, 5, 16), (9, 48, 8, 32), (300, 40, 8, 64), (17, 64, 1, 16),
                                         (1, 1, 1, 16), (130, 28, 4, 48)])
def test_heads_and_lengths(T, Hq, Hkv, bs):
    need_gpu()
    announce(f"norm rope T={T} {Hq}/{Hkv} bs={bs}")
    _run("bf16", T, Hq, Hkv, 128, True, "model", bs=bs, seed=T)


@pytest.mark.parametrize("T,Hq,Hkv,bs,rot,neox", [(1100, 48, 8, 16, 128, True), (1237, 48, 8, 32, 64, False),
                                                   (2050, 16, 16, 64, 96, True)])
def test_many_tokens(T, Hq, Hkv, bs, rot, neox):
    """From 2048 waves of 16 rows on: 16 rows a wave, nontemporal, a last run of workgroups that is cut."""
    need_gpu()
    announce(f"norm rope T={T} {Hq}/{Hkv} bs={bs}")
    _run("f16", T, Hq, Hkv, rot, neox, "f32", bs=bs, seed=T)


@pytest.mark.parametrize("spread", [1e-4, 300.0])
@pytest.mark.parametrize("eps", [0.0, 1e-5, 1.0])
def test_magnitudes(spread, eps):
    """Rows whose squares are far below and far above eps, and rows of zeros."""
    need_gpu()
    announce(f"norm rope spread {spread} eps {eps}")
    _run("f16", 20, 4, 2, 128, True, "f32", seed=3, eps=eps, spread=spread)
    if eps:
        z = torch.zeros((4, 3, 128), dtype=torch.float16, device=DEV)
        w = torch.ones(128, dtype=torch.float16, device=DEV)
        cs = torch.from_numpy(O.rope_cos_sin_cache(8, 128)).to(DEV)
        cache = gfx906_fa.new_kv_cache(1, 16, 1, device=DEV)
        n = torch.arange(4, device=DEV)
        gfx906_fa.qk_norm_rope_and_cache_q8_kv(n, z[:, :1], z[:, 1:2], z[:, 2:], w, w, eps, cs, False, n, cache[:, 0],
                                               cache[:, 1])
        assert (z == 0).all() and (cache == 0).all()


def test_graph_replay_and_stream():
    need_gpu()
    announce("norm rope graph")
    T, Hq, Hkv = 12, 8, 2
    qkv, wq, wk, cs, pos = _inputs("bf16", T, Hq, Hkv, 128, "model", 4)
    cache = gfx906_fa.new_kv_cache(2, 16, Hkv, device=DEV)
    pos, slots = pos.to(DEV), torch.arange(T, device=DEV)
    buf = qkv.clone()

    def call(x, c):
        gfx906_fa.qk_norm_rope_and_cache_q8_kv(pos, x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], wq, wk, 1e-6, cs, True,
                                               slots, c[:, 0], c[:, 1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(buf, cache)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(buf, cache)
    for i in range(3):
        x = qkv * (i + 1)
        pos.add_(1)
        buf.copy_(x)
        other = torch.zeros_like(cache)
        cache.zero_()
        g.replay()
        torch.cuda.synchronize()
        call(x, other)
        torch.cuda.synchronize()
        assert torch.equal(buf, x) and torch.equal(cache, other)


def test_refusals():
    need_gpu()
    announce("norm rope refusals")
    qkv, wq, wk, cs, pos = _inputs("f16", 4, 4, 1, 128, "model", 9)
    cache = gfx906_fa.new_kv_cache(2, 16, 1, device=DEV)
    n = torch.arange(4, device=DEV)
    good = dict(positions=n, query=qkv[:, :4], key=qkv[:, 4:5], value=qkv[:, 5:6], query_weight=wq, key_weight=wk, eps=1e-6,
                cos_sin_cache=cs, is_neox=True, slot_mapping=n, key_cache=cache[:, 0], value_cache=cache[:, 1])
    gfx906_fa.qk_norm_rope_and_cache_q8_kv(**good)
    for bad in (dict(query_weight=wq.float()), dict(key_weight=wk[:64]), dict(query_weight=wq.cpu()), dict(eps=-1.0),
                dict(eps=float("nan")), dict(rot_dim=72), dict(rot_dim=256), dict(positions=n.int()),
                dict(slot_mapping=n.int()), dict(key=qkv[:, 4:6]), dict(query=qkv[:, :4].float()),
                dict(key_cache=cache[:, 0, :, :100]), dict(query_weight=torch.cat([wq, wq])[4:132])):
        with pytest.raises(RuntimeError):
            gfx906_fa.qk_norm_rope_and_cache_q8_kv(**{**good, **bad})
