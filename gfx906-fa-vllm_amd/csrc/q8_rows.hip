// q8_rows.hip - single rows of the planar Q8_0 cache: read back as values, and
// the rows of accepted draft tokens moved behind their context.
//
// A row (token t of a 16-token sub-page, one kv-head, K or V) is 128 int8
// values and four fp16 scales, value = int8 * scale of its 32-value block.
// K rows are two runs of 64 bytes; V keeps four tokens of a value in a dword,
// so a V row is one byte of each of 128 dwords (q8_common.h has the offsets).
#include <cstdio>

#include "q8_common.h"

using namespace gfa;

namespace {

// ---------------------------------------------------------------------------
// Rows back as values: wave per (row, kv-head), two values per lane.
struct ReadArgs {
    const uint8_t *kc, *vc;
    const int64_t *slot;
    void *ko, *vo;
    int64_t num_rows, num_slots;
    int64_t cbs, chs, kts, khs, vts, vhs;
    int Hkv, block_size;
};

template <int ODT>
__device__ __forceinline__ void store2(void *out, int64_t i, float a, float b) {
    if constexpr (ODT == GFA_DTYPE_F32) {
        *reinterpret_cast<float2 *>(static_cast<float *>(out) + i) = make_float2(a, b);
    } else if constexpr (ODT == GFA_DTYPE_F16) {
        half2_t h = {(half_t)a, (half_t)b};
        *reinterpret_cast<half2_t *>(static_cast<uint16_t *>(out) + i) = h;
    } else {
        const uint32_t lo = __builtin_bit_cast(uint16_t, (__bf16)a), hi = __builtin_bit_cast(uint16_t, (__bf16)b);
        *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(out) + i) = lo | hi << 16;
    }
}

template <int ODT>
__global__ __launch_bounds__(256) void read_rows_kernel(ReadArgs a) {
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t t = w / a.Hkv;
    if (t >= a.num_rows) return;
    const int h = (int)(w - t * a.Hkv);
    const int64_t slot = a.slot[t];
    const int d = 2 * lane;
    float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
    if (slot >= 0 && slot < a.num_slots) {
        const int64_t page = slot / a.block_size;
        const int off = (int)(slot - page * a.block_size);
        const int64_t sub = page * a.cbs + (int64_t)h * a.chs + (int64_t)(off >> 4) * SUBPAGE_BYTES;
        const uint8_t *ks = a.kc + sub, *vs = a.vc + sub;
        const int tt = off & 15, b = d >> 5;
        const int kp = (b >> 1) * 1024 + (4 * tt + ((d >> 3) & 3)) * 16 + (b & 1) * 8 + (d & 7);
        const int vp = (d >> 6) * 1024 + (tt >> 2) * 256 + (d & 15) * 16 + ((d >> 4) & 3) * 4 + (tt & 3);
        const float dk = half_bits_to_f32(*reinterpret_cast<const uint16_t *>(ks + SCALE_OFF + (4 * tt + b) * 2));
        const float dv = half_bits_to_f32(
            *reinterpret_cast<const uint16_t *>(vs + SCALE_OFF + ((tt >> 2) * 4 + b) * 8 + (tt & 3) * 2));
        const uint16_t kq = *reinterpret_cast<const uint16_t *>(ks + kp);
        k0 = (float)(int8_t)(kq & 0xFF) * dk;
        k1 = (float)(int8_t)(kq >> 8) * dk;
        v0 = (float)(int8_t)vs[vp] * dv;
        v1 = (float)(int8_t)vs[vp + 16] * dv;
    }
    store2<ODT>(a.ko, t * a.kts + (int64_t)h * a.khs + d, k0, k1);
    store2<ODT>(a.vo, t * a.vts + (int64_t)h * a.vhs + d, v0, v1);
}

// ---------------------------------------------------------------------------
// Accepted draft rows: sequence s keeps draft tokens accepted[s][0 .. n-1] of
// its n_q; row (context + accepted[s][i]) moves to row (context + i).  Every
// row is read before any is written (a row may be one's source and another's
// target), so one workgroup moves all rows of a (layer, sequence, kv-head,
// plane), through LDS.
constexpr int MAX_DRAFT = 64;
constexpr int LAYERS = 64;  // layers of one launch, given one by one

struct CompactArgs {
    const int32_t *bt, *seq_lens, *qsl, *accepted, *count;
    int64_t bt_stride, acc_stride, cbs, chs, layer_stride, num_blocks;
    int bt_cols, acc_cols, Hkv, block_size, list;
    uint8_t *k[LAYERS], *v[LAYERS];  // list: each layer's planes; else k[0], v[0] + layer * layer_stride
};

// byte offset of position pos of sequence s in a plane (its sub-page), or -1
__device__ __forceinline__ int64_t sub_of(const CompactArgs &a, int s, int h, int64_t pos) {
    if (pos < 0) return -1;
    const int64_t col = pos / a.block_size;
    if (col >= a.bt_cols) return -1;
    const int64_t page = a.bt[(int64_t)s * a.bt_stride + col];
    if (page < 0 || page >= a.num_blocks) return -1;
    const int off = (int)(pos - col * a.block_size);
    return page * a.cbs + (int64_t)h * a.chs + (int64_t)(off >> 4) * SUBPAGE_BYTES;
}

__global__ __launch_bounds__(64) void compact_rows_kernel(CompactArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t rows[];  // [acc_cols][144]: 128 values, 8 bytes of scales
    constexpr int PITCH = 144;
    __shared__ int64_t s_src[MAX_DRAFT], s_dst[MAX_DRAFT];
    __shared__ int s_st[MAX_DRAFT], s_dt[MAX_DRAFT];
    const int lane = threadIdx.x;
    const int s = blockIdx.x / a.Hkv, h = blockIdx.x - s * a.Hkv;
    const bool isv = blockIdx.y & 1;
    const int layer = blockIdx.z;
    uint8_t *const base = a.list ? (isv ? a.v[layer] : a.k[layer]) : (isv ? a.v[0] : a.k[0]) + layer * a.layer_stride;
    const int nq = a.qsl[s + 1] - a.qsl[s];
    const int n = min(min(a.count[s], a.acc_cols), MAX_DRAFT);
    const int64_t ctx = (int64_t)a.seq_lens[s] - nq;
    if (lane < n) {
        const int from = a.accepted[(int64_t)s * a.acc_stride + lane];
        const bool ok = from >= 0 && from < nq && lane < nq && from != lane;
        const int64_t src = ok ? sub_of(a, s, h, ctx + from) : -1, dst = ok ? sub_of(a, s, h, ctx + lane) : -1;
        s_src[lane] = dst < 0 ? -1 : src;
        s_dst[lane] = dst;
        s_st[lane] = (int)((ctx + from) % 16);  // (block sizes are multiples of 16)
        s_dt[lane] = (int)((ctx + lane) % 16);
    }
    __syncthreads();
    // items of a row: 0..31 values (K: dword i of the row; V: the row's bytes of
    // the 16-byte chunk a = i / 16, e = i % 16), 32..35 one scale each
    for (int it = lane; it < n * 36; it += 64) {
        const int r = it / 36, i = it - 36 * r;
        const int64_t src = s_src[r];
        if (src < 0) continue;
        const uint8_t *p = base + src;
        const int t = s_st[r];
        if (i >= 32) {
            const int b = i - 32;
            const uint8_t *sp = p + SCALE_OFF + (isv ? ((t >> 2) * 4 + b) * 8 + (t & 3) * 2 : (4 * t + b) * 2);
            *reinterpret_cast<uint16_t *>(rows + r * PITCH + 128 + 2 * b) = *reinterpret_cast<const uint16_t *>(sp);
        } else if (isv) {
            const u32x4 c = *reinterpret_cast<const u32x4 *>(p + (i >> 4) * 1024 + (t >> 2) * 256 + (i & 15) * 16);
            uint32_t v = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) v |= ((c[e] >> (8 * (t & 3))) & 0xFFu) << (8 * e);
            *reinterpret_cast<uint32_t *>(rows + r * PITCH + 4 * i) = v;
        } else {
            *reinterpret_cast<uint32_t *>(rows + r * PITCH + 4 * i) =
                *reinterpret_cast<const uint32_t *>(p + (i >> 4) * 1024 + t * 64 + (i & 15) * 4);
        }
    }
    __syncthreads();  // every load has completed
    for (int it = lane; it < n * 36; it += 64) {
        const int r = it / 36, i = it - 36 * r;
        if (s_src[r] < 0) continue;
        uint8_t *p = base + s_dst[r];
        const int t = s_dt[r];
        if (i >= 32) {
            const int b = i - 32;
            uint8_t *sp = p + SCALE_OFF + (isv ? ((t >> 2) * 4 + b) * 8 + (t & 3) * 2 : (4 * t + b) * 2);
            *reinterpret_cast<uint16_t *>(sp) = *reinterpret_cast<const uint16_t *>(rows + r * PITCH + 128 + 2 * b);
        } else {
            const uint32_t v = *reinterpret_cast<const uint32_t *>(rows + r * PITCH + 4 * i);
            if (isv) {
                uint8_t *q = p + (i >> 4) * 1024 + (t >> 2) * 256 + (i & 15) * 16 + (t & 3);
#pragma unroll
                for (int e = 0; e < 4; ++e) q[4 * e] = (uint8_t)(v >> (8 * e));
            } else {
                *reinterpret_cast<uint32_t *>(p + (i >> 4) * 1024 + t * 64 + (i & 15) * 4) = v;
            }
        }
    }
}

bool plane_ok(const void *k, const void *v, int64_t cbs, int64_t chs) {
    return (((uintptr_t)k | (uintptr_t)v | (uint64_t)cbs | (uint64_t)chs) & 15u) == 0;
}

}  // namespace

extern "C" hipError_t gfx906_fa_amd_read_rows(
    const uint8_t *k_cache, const uint8_t *v_cache, const int64_t *slot_mapping, void *k_out, void *v_out, int out_dtype,
    int64_t num_rows, int num_kv_heads, int head_size, int block_size, int64_t num_blocks, int64_t cache_block_stride,
    int64_t cache_head_stride, int64_t k_out_row_stride, int64_t k_out_head_stride, int64_t v_out_row_stride,
    int64_t v_out_head_stride, hipStream_t stream) {
    if (head_size != 128 || block_size <= 0 || block_size % SUBPAGE != 0 || num_kv_heads <= 0 || num_rows < 0 ||
        num_blocks < 0 || out_dtype < 0 || out_dtype > 2) {
        fprintf(stderr, "[gfx906_fa_amd] read_rows: need head_size 128, block_size %% 16 == 0 (got %d, %d)\n", head_size,
                block_size);
        return hipErrorInvalidValue;
    }
    const uint64_t os = (uint64_t)(k_out_row_stride | k_out_head_stride | v_out_row_stride | v_out_head_stride);
    const uint64_t align = out_dtype == GFA_DTYPE_F32 ? 15u : 15u;
    if (!plane_ok(k_cache, v_cache, cache_block_stride, cache_head_stride) ||
        (((uintptr_t)k_out | (uintptr_t)v_out) & align) || (os & 7u)) {
        fprintf(stderr, "[gfx906_fa_amd] read_rows: cache and outputs must be 16-byte aligned, output strides multiples "
                        "of 8 elements\n");
        return hipErrorInvalidValue;
    }
    if (num_rows == 0) return hipSuccess;
    const int64_t blocks = (num_rows * num_kv_heads + 3) / 4;
    if (blocks > 0x7FFFFFFF) {
        fprintf(stderr, "[gfx906_fa_amd] read_rows: too many rows\n");
        return hipErrorInvalidValue;
    }
    const ReadArgs a{k_cache, v_cache, slot_mapping, k_out, v_out, num_rows, num_blocks * block_size,
                     cache_block_stride, cache_head_stride, k_out_row_stride, k_out_head_stride, v_out_row_stride,
                     v_out_head_stride, num_kv_heads, block_size};
    switch (out_dtype) {
        case GFA_DTYPE_F32: read_rows_kernel<GFA_DTYPE_F32><<<(unsigned)blocks, 256, 0, stream>>>(a); break;
        case GFA_DTYPE_F16: read_rows_kernel<GFA_DTYPE_F16><<<(unsigned)blocks, 256, 0, stream>>>(a); break;
        default: read_rows_kernel<GFA_DTYPE_BF16><<<(unsigned)blocks, 256, 0, stream>>>(a); break;
    }
    return hipGetLastError();
}

extern "C" hipError_t gfx906_fa_amd_compact_draft_rows(
    uint8_t *const *k_layers, uint8_t *const *v_layers, uint8_t *k_cache, uint8_t *v_cache, int64_t layer_stride,
    int num_layers, int64_t cache_block_stride, int64_t cache_head_stride, int64_t num_blocks, const int32_t *block_table,
    int64_t block_table_stride, int block_table_cols, const int32_t *seq_lens, const int32_t *query_start_loc,
    const int32_t *accepted, int64_t accepted_stride, int accepted_cols, const int32_t *num_accepted, int num_seqs,
    int num_kv_heads, int head_size, int block_size, hipStream_t stream) {
    if (head_size != 128 || block_size <= 0 || block_size % SUBPAGE != 0 || num_kv_heads <= 0 || num_seqs < 0 ||
        num_layers < 0 || num_blocks < 0 || block_table_cols < 0 || accepted_cols < 0 || accepted_cols > MAX_DRAFT) {
        fprintf(stderr, "[gfx906_fa_amd] compact_draft_rows: need head_size 128, block_size %% 16 == 0 and at most %d "
                        "accepted columns (got %d, %d, %d)\n", MAX_DRAFT, head_size, block_size, accepted_cols);
        return hipErrorInvalidValue;
    }
    const bool list = k_layers != nullptr;
    if (list != (v_layers != nullptr)) {
        fprintf(stderr, "[gfx906_fa_amd] compact_draft_rows: k_layers and v_layers go together\n");
        return hipErrorInvalidValue;
    }
    bool ok = list || plane_ok(k_cache, v_cache, layer_stride, 0);
    ok = ok && (((uint64_t)cache_block_stride | (uint64_t)cache_head_stride) & 15u) == 0;
    for (int i = 0; list && i < num_layers; ++i) ok = ok && plane_ok(k_layers[i], v_layers[i], 0, 0);
    if (!ok) {
        fprintf(stderr, "[gfx906_fa_amd] compact_draft_rows: caches must be 16-byte aligned\n");
        return hipErrorInvalidValue;
    }
    if (num_seqs == 0 || num_layers == 0 || accepted_cols == 0) return hipSuccess;
    if ((int64_t)num_seqs * num_kv_heads > 0x7FFFFFFF || num_layers > 65535) {
        fprintf(stderr, "[gfx906_fa_amd] compact_draft_rows: too many sequences or layers\n");
        return hipErrorInvalidValue;
    }
    CompactArgs a{};
    a.bt = block_table;
    a.seq_lens = seq_lens;
    a.qsl = query_start_loc;
    a.accepted = accepted;
    a.count = num_accepted;
    a.bt_stride = block_table_stride;
    a.acc_stride = accepted_stride;
    a.cbs = cache_block_stride;
    a.chs = cache_head_stride;
    a.layer_stride = layer_stride;
    a.num_blocks = num_blocks;
    a.bt_cols = block_table_cols;
    a.acc_cols = accepted_cols;
    a.Hkv = num_kv_heads;
    a.block_size = block_size;
    a.list = list ? 1 : 0;
    const size_t lds = (size_t)accepted_cols * 144;
    for (int l0 = 0; l0 < num_layers; l0 += list ? LAYERS : num_layers) {
        const int nl = list ? min(LAYERS, num_layers - l0) : num_layers;
        for (int i = 0; i < (list ? nl : 1); ++i) {
            a.k[i] = list ? k_layers[l0 + i] : k_cache;
            a.v[i] = list ? v_layers[l0 + i] : v_cache;
        }
        compact_rows_kernel<<<dim3(num_seqs * num_kv_heads, 2, nl), 64, lds, stream>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
