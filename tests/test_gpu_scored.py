"""GPU: attention with capped scores or a distance bias, against 64 bits.

Every kernel the plan can take: one to four 16-row groups a wave, 128- and
256-row tiles, split and whole, batches that mix them."""
import numpy as np
import pytest
import torch

import gfx906_fa
import gfx906_fa_workloads as W
from gpu_common import announce, need_gpu
from scored_common import check, eps_of, scored_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
TD = {"f16": torch.float16, "bf16": torch.bfloat16}

# (keys, query tokens, heads, kv-heads, block size)
SHAPES = {
    "one_key": ([1], [1], 8, 1, 16),
    "decode": ([33, 1, 900, 257], [1, 1, 1, 1], 48, 8, 16),
    "decode_mha": ([17, 700], [1, 1], 5, 5, 32),
    "decode_split": ([1500, 2049], [1, 1], 6, 1, 64),
    "verify30": ([640, 35, 5], [5, 5, 5], 6, 1, 16),
    "verify48_tiles": ([1040] * 8, [8] * 8, 48, 8, 16),
    "verify64": ([300, 8], [8, 8], 8, 1, 16),
    "verify64_short": ([100, 70, 8], [8, 8, 8], 8, 1, 16),
    "verify30_short": ([384, 71, 6], [5, 5, 5], 6, 1, 16),
    "many_short": ([1024] + [100] * 31, [1] * 32, 32, 8, 16),
    "many_verify": ([200] * 16 + [9] * 16, [5] * 32, 48, 8, 16),
    "rows96": ([700, 12], [12, 12], 8, 1, 16),
    "rows360": ([500], [60], 48, 8, 16),
    "prompts": ([77, 301, 130], [77, 301, 130], 8, 2, 16),
    "chunk_split": ([2100], [50], 6, 1, 32),
    "mixed": ([90, 640, 1, 333, 64], [90, 1, 1, 20, 5], 6, 1, 16),
    "mixed_wide": ([200, 90, 700], [1, 1, 3], 20, 1, 16),
    "images": ([1400], [1400], 6, 1, 16),   # 33 row tiles: key tiles dequantized once
}


def _batch(name, dt, spread=1.0, seed=5, poison=True):
    sl, nq, hq, hkv, bs = SHAPES[name]
    b = W.build_batch(sl, nq, hq, hkv, block_size=bs, dtype=dt, seed=seed, device=DEV, bt_pad_cols=2)
    if poison:  # what is not a key of a sequence holds NaN scales and any values
        b.kv_cache.fill_(0xFF)
        gfx906_fa.reshape_and_cache_q8_kv(b.key, b.value, b.slot_mapping, *b.planes())
    if spread != 1.0:
        b.query = (b.query.float() * spread).to(b.query.dtype)
    return b


def _call(b, **kw):
    kp, vp = b.planes()
    return gfx906_fa.scored_paged_attention(b.query, kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, b.max_query_len,
                                            b.max_seq_len, b.scale, **kw)


def _slopes(hq):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], dtype=torch.float32, device=DEV)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_capped(name, dt):
    need_gpu()
    announce(f"capped {name} {dt}")
    b = _batch(name, dt, spread=4.0)
    out = _call(b, soft_cap=5.0)
    check(out, *scored_oracle(b, cap=5.0, out_eps=eps_of(TD[dt])))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_biased(name, dt):
    need_gpu()
    announce(f"biased {name} {dt}")
    b = _batch(name, dt)
    sl = _slopes(b.Hq)
    out = _call(b, alibi_slopes=sl, out_dtype=torch.float32)
    check(out, *scored_oracle(b, slopes=sl.cpu().numpy()))


@pytest.mark.parametrize("cap", [0.003, 1.0, 30.0, 1024.0])
@pytest.mark.parametrize("name", ["decode", "prompts"])
def test_cap_range(name, cap):
    """From a cap that flattens every score to one that changes none."""
    need_gpu()
    announce(f"cap {cap} {name}")
    b = _batch(name, "f16", spread=6.0)
    out = _call(b, soft_cap=cap, out_dtype=torch.float32)
    check(out, *scored_oracle(b, cap=cap))


@pytest.mark.parametrize("spread", [1500.0, 0.01])
@pytest.mark.parametrize("name", ["prompts", "rows96", "decode"])
def test_small_cap_of_large_scores(name, spread):
    """The cap far below the scale, queries far from 1 (the largest about 6000)."""
    need_gpu()
    announce(f"small cap {name} {spread}")
    b = _batch(name, "f16", spread=spread)
    out = _call(b, soft_cap=0.003, out_dtype=torch.float32)
    check(out, *scored_oracle(b, cap=0.003))


@pytest.mark.parametrize("name", ["decode", "verify30", "prompts"])
def test_slopes_of_any_sign_and_size(name):
    need_gpu()
    announce(f"slopes {name}")
    b = _batch(name, "bf16")
    sl = torch.linspace(-0.5, 40.0, b.Hq, device=DEV)
    sl[0] = 0.0
    out = _call(b, alibi_slopes=sl, out_dtype=torch.float32)
    check(out, *scored_oracle(b, slopes=sl.cpu().numpy()))


@pytest.mark.parametrize("how", ["full", "offset", "hidden"])
@pytest.mark.parametrize("form", ["cap", "bias"])
@pytest.mark.parametrize("name", ["decode", "verify30", "prompts"])
def test_visibility(name, form, how):
    """Rows that see every key; a causal offset of their own, also one that
    leaves the first rows (or all) without a key: those are 0."""
    need_gpu()
    announce(f"visibility {name} {form} {how}")
    b = _batch(name, "f16")
    sl = _slopes(b.Hq)
    kw = dict(soft_cap=3.0) if form == "cap" else dict(alibi_slopes=sl)
    okw = dict(cap=3.0) if form == "cap" else dict(slopes=sl.cpu().numpy())
    qa = None
    if how == "full":
        kw["causal"] = okw["causal"] = False
    else:
        qa = [int(s) // 3 for s in b.seq_lens] if how == "offset" else [-3 if i % 2 else -400 for i in range(b.num_seqs)]
        kw["q_abs_offset"] = torch.tensor(qa, dtype=torch.int32, device=DEV)
    out = _call(b, out_dtype=torch.float32, **kw)
    ref, bound = scored_oracle(b, q_abs=qa, **okw)
    check(out, ref, bound)
    if how == "hidden":
        assert (np.abs(ref).max(axis=(1, 2)) == 0).any()


@pytest.mark.parametrize("scale", [1e-4, 4.0])
@pytest.mark.parametrize("name", ["decode", "prompts"])
def test_scale_range(name, scale):
    """Scales far from 1 / sqrt(128) with a cap of the scores' size."""
    need_gpu()
    announce(f"scale {scale} {name}")
    b = _batch(name, "bf16", spread=0.05 / scale if scale < 1 else 0.2)
    b.scale = scale
    out = _call(b, soft_cap=2.0, out_dtype=torch.float32)
    check(out, *scored_oracle(b, cap=2.0))


def test_no_form_is_plain_attention():
    need_gpu()
    announce("no form")
    b = _batch("mixed", "f16", poison=False)
    assert torch.equal(_call(b), W.attention(b))


@pytest.mark.parametrize("name", ["decode", "verify30", "prompts"])
def test_outputs_strides_and_rows_behind(name):
    """Strided query and output views; rows behind the last sequence stay."""
    need_gpu()
    announce(f"strides {name}")
    b = _batch(name, "f16")
    T = b.num_tokens
    ref = scored_oracle(b, cap=4.0, out_eps=eps_of(torch.float16))
    wide = torch.full((T + 3, 2, b.Hq, 256), 7.0, dtype=torch.float16, device=DEV)
    q = torch.zeros((T + 3, b.Hq, 192), dtype=torch.float16, device=DEV)
    q[:T, :, 64:] = b.query
    kp, vp = b.planes()
    out = wide[:, 1, :, 128:]
    r = gfx906_fa.scored_paged_attention(q[..., 64:], kp, vp, b.block_table, b.seq_lens_t, b.qsl_t, b.max_query_len,
                                         b.max_seq_len, b.scale, soft_cap=4.0, out=out)
    assert r is out
    check(out[:T], *ref)
    wide[:T, 1, :, 128:] = 7.0
    assert (wide == 7.0).all()


def test_empty_sequences():
    """Sequences without query tokens, and with neither keys nor tokens."""
    need_gpu()
    announce("empty sequences")
    b = W.build_batch([40, 0, 100, 16], [1, 0, 0, 16], 8, 2, dtype="bf16", seed=2, device=DEV)
    out = _call(b, soft_cap=9.0)
    check(out, *scored_oracle(b, cap=9.0, out_eps=eps_of(torch.bfloat16)))


@pytest.mark.parametrize("form", ["cap", "bias"])
def test_graph_and_streams(form):
    """Captured on a side stream and replayed with other lengths and values,
    with eager calls between; two graphs with a workspace each."""
    need_gpu()
    announce(f"graph {form}")
    b = _batch("verify30", "f16")
    sl = _slopes(b.Hq)
    kw = dict(soft_cap=6.0) if form == "cap" else dict(alibi_slopes=sl)
    ws = gfx906_fa.new_workspace(gfx906_fa.workspace_size(b.num_seqs, b.num_tokens, b.Hq, b.Hkv, b.max_query_len,
                                                          b.max_seq_len), DEV)
    out = torch.zeros((b.num_tokens, b.Hq, 128), dtype=torch.float16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _call(b, out=out, workspace=ws, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _call(b, out=out, workspace=ws, **kw)
    for lens in ([640, 35, 5], [17, 30, 5], [639, 6, 5]):
        b.seq_lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
        b.query.mul_(-1.0)
        eager = _call(b, **kw)
        torch.cuda.synchronize()
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), lens


def test_far_positions():
    """A long context: the bias of near keys keeps its precision at far
    positions."""
    need_gpu()
    announce("far positions")
    b = W.build_batch([20011], [2], 8, 1, dtype="bf16", seed=3, device=DEV, host_values=False)
    sl = torch.tensor([2.0 ** -i for i in range(8)], dtype=torch.float32, device=DEV)
    out = _call(b, alibi_slopes=sl, out_dtype=torch.float32)
    check(out, *scored_oracle(b, slopes=sl.cpu().numpy()))


def test_refusals():
    need_gpu()
    announce("refusals")
    b = _batch("decode", "f16", poison=False)
    sl = _slopes(b.Hq)
    for kw in (dict(soft_cap=-1.0), dict(soft_cap=float("nan")), dict(soft_cap=float("inf")), dict(soft_cap=1e-44), dict(soft_cap=1e-4), dict(soft_cap=1025.0),
               dict(soft_cap=2.0, alibi_slopes=sl), dict(alibi_slopes=sl[:-1]), dict(alibi_slopes=sl.half()),
               dict(alibi_slopes=sl.cpu()), dict(soft_cap=2.0, out_dtype=torch.bfloat16),
               dict(soft_cap=2.0, out=torch.empty(4, 48, 128, dtype=torch.bfloat16, device=DEV)),
               dict(soft_cap=2.0, out=torch.empty(3, 48, 128, dtype=torch.float16, device=DEV))):
        with pytest.raises(RuntimeError):
            _call(b, **kw)
    b.query = b.query.float()
    with pytest.raises(RuntimeError):
        _call(b, soft_cap=2.0)
