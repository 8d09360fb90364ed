"""GPU: cached rows read back in the orders that choose the kernel's two ways:
groups of 16 entries that are a sub-page in order go whole, others row by row.
Against the cache's bytes on the host, bit for bit (int8 * scale has at most 18
bits: exact in fp32, rounded once below)."""
import numpy as np
import pytest
import torch

import gfx906_fa
from gpu_common import announce, need_gpu
from oracle import q8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _cache(NB, Hkv, bs, seed):
    """Every (token, kv-head, block) with a scale of its own."""
    rng = np.random.default_rng(seed)
    n = NB * bs
    x = rng.uniform(-1, 1, (2, n, Hkv, 4, 32)) * np.exp2(rng.uniform(-6, 6, (2, n, Hkv, 4, 1)))
    k, v = torch.from_numpy(x.reshape(2, n, Hkv, 128).astype(np.float32)).to(DEV)
    cache = gfx906_fa.new_kv_cache(NB, bs, Hkv, device=DEV)
    gfx906_fa.reshape_and_cache_q8_kv(k, v, torch.arange(n, device=DEV), cache[:, 0], cache[:, 1])
    return cache


def _orders(T, NB, bs):
    """name -> slots: the first entry a multiple of 16 unless the name says so."""
    n, rng = NB * bs, np.random.default_rng(T)
    whole = np.arange(16, 16 + T)
    broken = whole.copy()  # one group of 16 that is no sub-page: two entries swapped
    if T >= 32:
        broken[[18, 23]] = broken[[23, 18]]
    last = whole.copy()    # a group's last entry elsewhere, and one outside the cache
    last[min(T, 16) - 1] = 3
    if T > 40:
        last[40] = -1
    pages = np.concatenate([np.arange(16) + 16 * p for p in rng.permutation(n // 16)])[:T]
    end = np.arange(n - T, n)  # up to the cache's last slot, and past it below
    over = np.arange((n - T) // 16 * 16 + 16, (n - T) // 16 * 16 + 16 + T)
    return {"whole": whole, "broken": broken, "last": last, "pages": pages, "end": end, "over": over, "shifted": whole - 7,
            "backwards": whole[::-1].copy(), "twice": np.concatenate([whole[:T - T // 2], whole[:T // 2]])}


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,Hkv,bs", [(16, 1, 16), (16, 3, 64), (37, 2, 32), (37, 8, 16), (700, 2, 64), (700, 5, 16)])
def test_read_orders(dt, T, Hkv, bs):
    need_gpu()
    announce(f"read orders {dt} T={T} Hkv={Hkv} bs={bs}")
    NB = (T + 48) // bs + 2
    cache = _cache(NB, Hkv, bs, T + Hkv)
    host = [torch.from_numpy(np.ascontiguousarray(x.reshape(NB * bs, Hkv, 128))) for x in O.planar_dequant(cache.cpu().numpy())]
    for name, slots in _orders(T, NB, bs).items():
        assert slots.shape == (T,)
        bad = torch.from_numpy((slots < 0) | (slots >= NB * bs))
        at = torch.from_numpy(np.clip(slots, 0, NB * bs - 1).astype(np.int64))
        got = gfx906_fa.read_cache_q8_kv(torch.from_numpy(slots.astype(np.int64)).to(DEV), cache[:, 0], cache[:, 1], dt)
        wide = torch.full((T, Hkv, 2, 136), 7.0, dtype=dt, device=DEV)
        gfx906_fa.read_cache_q8_kv(torch.from_numpy(slots.astype(np.int64)).to(DEV), cache[:, 0], cache[:, 1], dt,
                                   k_out=wide[:, :, 0, 8:], v_out=wide[:, :, 1, :128])
        assert (wide[:, :, 0, :8] == 7.0).all() and (wide[:, :, 1, 128:] == 7.0).all()
        for i, x in enumerate(host):
            x = x[at].clone()
            x[bad] = 0
            assert torch.equal(got[i].cpu(), x.to(dt)), (name, "kv"[i])
            view = wide[:, :, i, 8:] if i == 0 else wide[:, :, i, :128]
            assert torch.equal(view.cpu(), x.to(dt)), (name, "kv"[i], "view")
