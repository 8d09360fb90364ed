"""GPU: keys that a row does not see may hold anything, whichever kernel takes
the row: what was written behind the last key of a page, later tokens and
hidden nodes with values past fp16's range.  Outputs are those of finite
hidden values, bit for bit: such a key's weight is 0 in both."""
import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from gpu_common import announce, need_gpu
from scored_common import random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (contexts before the last tokens, those tokens, heads, kv-heads, block size)
SHAPES = {
    "decode": ([32, 899, 256], [1, 1, 1], 16, 4, 16),
    "rows30": ([600, 9], [5, 5], 6, 1, 32),
    "rows64": ([333, 20], [8, 8], 8, 1, 16),
    "tiles128": ([688, 1000], [12, 21], 6, 1, 16),      # 128-row tiles
    "tiles256": ([777, 63], [64, 50], 12, 2, 64),       # 256-row tiles
    "prompts": ([0, 0, 100], [61, 47, 33], 16, 2, 16),
    "split": ([2050], [50], 6, 1, 32),                  # row tiles split over the keys
    "images": ([70], [1330], 6, 1, 16),                 # key tiles dequantized once
}
TREES = [n for n in SHAPES if n != "images"]            # (at most 64 nodes)


def _batch(name, dt):
    ctx, n, hq, hkv, bs = SHAPES[name]
    return W.build_batch([c + m for c, m in zip(ctx, n)], n, hq, hkv, block_size=bs, dtype=dt, seed=11, device=DEV,
                         bt_pad_cols=1)


def _call(b, form):
    kp, vp = b.planes()
    args = (b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t)
    lens = (b.max_query_len, b.max_seq_len, b.scale)
    if form == "plain":
        return gfx906_fa.paged_attention(*args, *lens, out_dtype=torch.float32)
    if form.startswith("tree"):
        rng = np.random.default_rng(3)
        m = gfx906_fa.tree_masks([random_tree(rng, int(n)) for n in b.q_lens])
        return gfx906_fa.tree_attention(*args, m.to(DEV), *lens, soft_cap=4.0 if form == "tree_cap" else 0.0,
                                        out_dtype=torch.float32)
    kw = dict(soft_cap=5.0)
    if form == "bias":
        kw = dict(alibi_slopes=torch.tensor([2.0 ** -(i % 8 + 1) for i in range(b.Hq)], device=DEV))
    return gfx906_fa.scored_paged_attention(*args, *lens, out_dtype=torch.float32, **kw)


def _write(b):
    gfx906_fa.reshape_and_cache_q8_kv(b.key, b.value, b.slot_mapping, *b.planes())


BEHIND = [(f, n) for f in ("plain", "cap", "bias") for n in SHAPES] + [(f, n) for f in ("tree", "tree_cap") for n in TREES]


# (plain decode rows need finite scales there: the scored ones do not)
BYTES = [(f, n, x) for f, n in BEHIND for x in (0x7F, 0x7B, 0x80)
         if not (f == "plain" and n in ("decode", "rows30", "rows64") and x == 0x7F)]


@pytest.mark.parametrize("form,name,byte", BYTES)
def test_bytes_behind_the_keys(form, name, byte):
    """0x7F: int 127 and a NaN scale; 0x7B: int 123 and the scale 61280; 0x80:
    int -128 and a small one."""
    need_gpu()
    announce(f"behind {form} {name} {byte:#x}")
    b = _batch(name, "f16")
    b.kv_cache.zero_()
    _write(b)
    want = _call(b, form)
    assert torch.isfinite(want).all()
    b.kv_cache.fill_(byte)
    _write(b)
    assert torch.equal(_call(b, form), want)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("form,name", [(f, n) for f, n in BEHIND if f != "plain" and n != "decode"])
def test_hidden_tokens_past_fp16(form, name, dt):
    """Each sequence's last token, which only its own row sees, with keys and
    values of +-1e6 (bf16), or fp16's largest: the other rows stay as they were."""
    need_gpu()
    announce(f"hidden {form} {name} {dt}")
    b = _batch(name, dt)
    tok = [int(b.qsl[s]) + int(n) - 1 for s, n in enumerate(b.q_lens)]
    rows = [t for t in range(b.num_tokens) if t not in tok]
    want = _call(b, form)[rows]
    assert torch.isfinite(want).all()
    last = np.cumsum(b.seq_lens) - 1
    big = 1e6 if dt == "bf16" else 65504.0
    for s, r in enumerate(last):
        sign = torch.where(torch.arange(128, device=DEV) % 3 == 0, -1.0, 1.0) * (1 if s % 2 else -1)
        b.value[int(r)] = (big * sign).to(b.value.dtype)
        b.key[int(r)] = (big * sign).to(b.key.dtype)
    _write(b)
    assert torch.equal(_call(b, form)[rows], want)


@pytest.mark.parametrize("form", ["cap", "bias"])
def test_seen_values_past_fp16(form):
    """A value of 1e5 that a row does see: itself for decode rows, fp16's largest
    where the row is of a prefill-shaped sequence."""
    need_gpu()
    announce(f"seen {form}")
    for tokens, want in ((1, 1e5), (90, 65504.0)):
        b = W.build_batch([tokens], [tokens], 8, 1, dtype="bf16", seed=3, device=DEV)
        b.value.zero_()
        b.value[0] = 1e5
        _write(b)
        out = _call(b, form)
        want = min(want, float(b.value[0].max()))  # (bf16 holds 1e5 as 99840)
        # the first row sees this key alone: Q8_0's scale, fp16, is off by 2^-11, p d_v by as much
        assert ((out[0] - want).abs() <= 2.0 ** -10 * want).all()
        assert torch.isfinite(out).all()
