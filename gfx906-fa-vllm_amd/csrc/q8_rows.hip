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
// Rows back as values.  A wave takes 16 consecutive entries of slot_mapping for
// one kv-head.  Where they are a sub-page in order (a prompt's rows), it reads
// the sub-page's 2 x 2176 bytes once, 16 bytes a lane; a lane then holds runs of
// 8 values of a K row, and of a V chunk 4 values of 4 tokens, which go through
// LDS to become rows.  Otherwise 16 lanes take a row, 8 values each: one 8-byte
// K load and 8 dwords of V (each with a byte of the row), four rows at a time.
// 20001 rows at 8 kv-heads, bf16: 46.7 us with a wave per row and a byte load
// per V value, 20.5 us in order (126 MB, 6.1 TB/s: HBM), 38.9 in any order (79 MB
// come in for 44 MB of rows, as a V row's bytes lie in four times as many).
struct ReadArgs {
    const uint8_t *kc, *vc;
    const int64_t *slot;
    void *ko, *vo;
    int64_t num_rows, num_slots;
    int64_t cbs, chs, kts, khs, vts, vhs;
    int Hkv, block_size;
};

template <int ODT>
__device__ __forceinline__ uint16_t out16(float v) {
    if constexpr (ODT == GFA_DTYPE_F16) return f32_to_half_bits(v);
    else return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// 8 values at a 16-byte aligned element offset
template <int ODT>
__device__ __forceinline__ void store8(void *out, int64_t i, const float (&v)[8]) {
    if constexpr (ODT == GFA_DTYPE_F32) {
        float4_t *p = reinterpret_cast<float4_t *>(static_cast<float *>(out) + i);
        p[0] = float4_t{v[0], v[1], v[2], v[3]};
        p[1] = float4_t{v[4], v[5], v[6], v[7]};
    } else {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = out16<ODT>(v[2 * e]) | (uint32_t)out16<ODT>(v[2 * e + 1]) << 16;
        *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(out) + i) = w;
    }
}

__device__ __forceinline__ float byte_f32(uint32_t w, int e) { return (float)(int8_t)(w >> (8 * e)); }

constexpr int RR_PITCH = 132;  // floats of a V row in LDS: rows of a quad of tokens start 4 banks apart

template <int ODT>
__global__ __launch_bounds__(256) void read_rows_kernel(ReadArgs a) {
    __shared__ float sm[4][16][RR_PITCH];
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + wv;
    const int64_t t0 = w / a.Hkv * 16;
    if (t0 >= a.num_rows) return;  // uniform over the wave
    const int h = (int)(w - t0 / 16 * a.Hkv);
    const int n = (int)min((int64_t)16, a.num_rows - t0);
    const int i = lane & 15, g = lane >> 4;
    const int64_t mine = i < n ? a.slot[t0 + i] : -1;
    const int64_t first = ((int64_t)__builtin_amdgcn_readfirstlane((int)(mine >> 32)) << 32) |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)mine);
    if (n == 16 && first >= 0 && (first & 15) == 0 && first + 15 < a.num_slots &&
        __builtin_amdgcn_ballot_w64(mine != first + i) == 0) {  // uniform
        const int64_t page = first / a.block_size;
        const int off = (int)(first - page * a.block_size);
        const int64_t sub = page * a.cbs + (int64_t)h * a.chs + (int64_t)(off >> 4) * SUBPAGE_BYTES;
        const uint8_t *ks = a.kc + sub, *vs = a.vc + sub;
        // K: lane 4 t + q holds values 64 c + 32 b + 8 q .. of token t in dwords 2 b, 2 b + 1 of chunk c
        const u32x4 k0 = *reinterpret_cast<const u32x4 *>(ks + 16 * lane);
        const u32x4 k1 = *reinterpret_cast<const u32x4 *>(ks + 1024 + 16 * lane);
        // V: lane 16 u + e holds values 64 c + 16 m + e of tokens 4 u .. in dword m of chunk c
        const u32x4 v0 = *reinterpret_cast<const u32x4 *>(vs + 16 * lane);
        const u32x4 v1 = *reinterpret_cast<const u32x4 *>(vs + 1024 + 16 * lane);
        const u32x2 kd = *reinterpret_cast<const u32x2 *>(ks + SCALE_OFF + 8 * (lane >> 2));
        const u32x4 d0 = *reinterpret_cast<const u32x4 *>(vs + SCALE_OFF + 32 * g);
        const u32x4 d1 = *reinterpret_cast<const u32x4 *>(vs + SCALE_OFF + 32 * g + 16);
        const int t = lane >> 2;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const u32x4 kq = c ? k1 : k0;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float d = half_bits_to_f32(b ? kd[c] >> 16 : kd[c] & 0xFFFFu);
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = byte_f32(kq[2 * b + (e >> 2)], e & 3) * d;
                store8<ODT>(a.ko, (t0 + t) * a.kts + (int64_t)h * a.khs + 64 * c + 32 * b + 8 * (lane & 3), x);
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const u32x4 vq = c ? v1 : v0, vd = c ? d1 : d0;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // token 4 g + e: scale of block 2 c + m / 2
                    const uint32_t dw = vd[2 * (m >> 1) + (e >> 1)];
                    const float d = half_bits_to_f32(e & 1 ? dw >> 16 : dw & 0xFFFFu);
                    sm[wv][4 * g + e][64 * c + 16 * m + i] = byte_f32(vq[m], e) * d;
                }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // one wave's LDS instructions complete in order
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float4_t *row = reinterpret_cast<const float4_t *>(&sm[wv][4 * r + g][8 * i]);
            const float4_t p = row[0], q = row[1];
            const float x[8] = {p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
            store8<ODT>(a.vo, (t0 + 4 * r + g) * a.vts + (int64_t)h * a.vhs + 8 * i, x);
        }
        return;
    }
    // rows one by one: lane i of 16 takes values 8 i .. of entry 4 r + g
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int at = 4 * r + g;
        if (4 * r >= n) break;  // uniform
        const int64_t slot = ((int64_t)__shfl((int)(mine >> 32), at) << 32) | (uint32_t)__shfl((int)mine, at);
        float k[8] = {}, v[8] = {};
        if (slot >= 0 && slot < a.num_slots) {
            const int64_t page = slot / a.block_size;
            const int off = (int)(slot - page * a.block_size);
            const int64_t sub = page * a.cbs + (int64_t)h * a.chs + (int64_t)(off >> 4) * SUBPAGE_BYTES;
            const uint8_t *ks = a.kc + sub, *vs = a.vc + sub;
            const int tt = off & 15, b = i >> 2, m = i >> 1;
            const u32x2 kq = *reinterpret_cast<const u32x2 *>(ks + (b >> 1) * 1024 + (4 * tt + (i & 3)) * 16 + (b & 1) * 8);
            const uint8_t *vp = vs + (m >> 2) * 1024 + (tt >> 2) * 256 + (i & 1) * 128 + (m & 3) * 4;
            uint32_t vq[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) vq[e] = *reinterpret_cast<const uint32_t *>(vp + 16 * e);
            const float dk = half_bits_to_f32(*reinterpret_cast<const uint16_t *>(ks + SCALE_OFF + (4 * tt + b) * 2));
            const float dv = half_bits_to_f32(
                *reinterpret_cast<const uint16_t *>(vs + SCALE_OFF + ((tt >> 2) * 4 + b) * 8 + (tt & 3) * 2));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k[e] = byte_f32(kq[e >> 2], e & 3) * dk;
                v[e] = byte_f32(vq[e], tt & 3) * dv;
            }
        }
        if (at < n) {
            store8<ODT>(a.ko, (t0 + at) * a.kts + (int64_t)h * a.khs + 8 * i, k);
            store8<ODT>(a.vo, (t0 + at) * a.vts + (int64_t)h * a.vhs + 8 * i, v);
        }
    }
}

// ---------------------------------------------------------------------------
// Accepted draft rows: sequence s keeps draft tokens accepted[s][0 .. n-1] of
// its n_q; row (context + accepted[s][i]) moves to row (context + i), as if
// every row were read before any is written.  Where the rows lie is the same
// for every layer and head: a workgroup works that out once, and its four
// waves then take (layer, kv-head) pairs of the sequence, K and V.
//
// K rows are whole pieces of 16 and 8 bytes.  Of a V row every 16-byte chunk
// holds one byte in four, so V moves by quads of target tokens: a lane loads the
// target's chunk and those of up to four source rows, merges their bytes and
// stores the chunk whole (with byte stores the lines went out in parts: 60
// layers x 32 sequences of 26 drafts at 8 kv-heads, 83 rows moved, 34 us, 20.4
// this way; one layer of 7 sequences 6.2 us, 3.2 of them launch and the rows'
// places).  A path's nodes ascend (a node comes after its parent), so that no
// row is the target of an earlier one, and a wave moves rows and quads in order,
// all loads of a step before its stores.  In any other order all rows go through
// LDS first.  Bound: runs of 64 to 256 bytes all over the caches, 50 MB of lines
// in and out for 22 MB of rows (a V row's 128 bytes lie in 512), at 2.5 TB/s.
constexpr int MAX_DRAFT = 64;
constexpr int LAYERS = 64;  // layers of one launch, given one by one
// Waves from which a wave takes more than one (layer, kv-head) pair (for the
// case above 20.4 us; 8192: 21.5, 16384: 23.6).
constexpr int CR_WAVES = 4096;
constexpr int MAX_QUADS = MAX_DRAFT / 4 + 1;

struct CompactArgs {
    const int32_t *bt, *seq_lens, *qsl, *accepted, *count;
    int64_t bt_stride, acc_stride, cbs, chs, layer_stride, num_blocks;
    int bt_cols, acc_cols, Hkv, block_size, layers, list;
    uint8_t *k[LAYERS], *v[LAYERS];  // list: each layer's planes; else k[0], v[0] + layer * layer_stride
};

// byte offset of position pos of sequence s in a plane (its sub-page, kv-head 0), or -1
__device__ __forceinline__ int64_t sub_of(const CompactArgs &a, int s, int64_t pos) {
    if (pos < 0) return -1;
    const int64_t col = pos / a.block_size;
    if (col >= a.bt_cols) return -1;
    const int64_t page = a.bt[(int64_t)s * a.bt_stride + col];
    if (page < 0 || page >= a.num_blocks) return -1;
    const int off = (int)(pos - col * a.block_size);
    return page * a.cbs + (int64_t)(off >> 4) * SUBPAGE_BYTES;
}

constexpr int CR_PIECES = 8 + 1 + 32 + 2;   // K ints, K scales, V chunks, V scales
constexpr int CR_QUAD = 32 + 2;             // V chunks and scale chunks of a quad of tokens

// Byte offset in its plane's sub-page of piece c of token t, 16-byte aligned.
__device__ __forceinline__ int piece_off(int c, int t) {
    if (c < 8) return (c >> 2) * 1024 + 64 * t + (c & 3) * 16;
    if (c == 8) return SCALE_OFF + (t >> 1) * 16;
    if (c < 41) return ((c - 9) >> 4) * 1024 + (t >> 2) * 256 + ((c - 9) & 15) * 16;
    return SCALE_OFF + (t >> 2) * 32 + (c - 41) * 16;
}

// Stores what piece c holds of token ts at token td of the sub-page p.
__device__ __forceinline__ void piece_store(uint8_t *p, int c, int ts, int td, u32x4 x) {
    uint8_t *const at = p + piece_off(c, td);
    if (c < 8) {
        *reinterpret_cast<u32x4 *>(at) = x;
    } else if (c == 8) {
        *reinterpret_cast<u32x2 *>(at + 8 * (td & 1)) = ts & 1 ? u32x2{x[2], x[3]} : u32x2{x[0], x[1]};
    } else if (c < 41) {  // byte ts % 4 of each dword
#pragma unroll
        for (int e = 0; e < 4; ++e) at[4 * e + (td & 3)] = (uint8_t)(x[e] >> (8 * (ts & 3)));
    } else {  // two blocks, four tokens' scales each
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t w = ts & 2 ? x[2 * b + 1] : x[2 * b];
            *reinterpret_cast<uint16_t *>(at + 8 * b + 2 * (td & 3)) = (uint16_t)(ts & 1 ? w >> 16 : w);
        }
    }
}

// Piece u of the K rows: row u / 9, piece u % 9.
struct KPiece {
    u32x4 x;
    int r, c, tok;
    __device__ __forceinline__ void load(const uint8_t *kb, int u, const int64_t *src, const int *toks) {
        r = u / 9;
        c = u - 9 * r;
        tok = toks[r];
        x = *reinterpret_cast<const u32x4 *>(kb + src[r] + piece_off(c, tok & 15));
    }
    __device__ __forceinline__ void store(uint8_t *kb, const int64_t *dst) const {
        piece_store(kb + dst[r], c, tok & 15, tok >> 8, x);
    }
};

// Chunk u % 34 of target quad u / 34 of V: its 16 bytes, and the four rows' that
// its tokens take (a token without a row takes its own bytes).
struct VQuad {
    u32x4 y[4];
    u32x4 *to;
    int j, t[4];
    __device__ __forceinline__ void load(uint8_t *vb, int u, const int64_t *quad, const int (*row)[4],
                                         const int64_t *src, const int *toks) {
        const int q = u / CR_QUAD;
        j = u - CR_QUAD * q;
        const int at = j < 32 ? (j >> 4) * 1024 + (j & 15) * 16 : SCALE_OFF + (j - 32) * 16;
        const int per = j < 32 ? 256 : 32;  // bytes of a quad
        uint8_t *const own = vb + (quad[q] & ~(int64_t)15) + at + per * (int)(quad[q] & 3);
        to = reinterpret_cast<u32x4 *>(own);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int r = row[q][w];
            t[w] = r < 0 ? w : toks[r] & 15;
            y[w] = *reinterpret_cast<const u32x4 *>(r < 0 ? own : vb + src[r] + at + per * (t[w] >> 2));
        }
    }
    __device__ __forceinline__ void store() const {
        u32x4 x;
        if (j < 32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t v = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) v |= ((y[w][e] >> (8 * (t[w] & 3))) & 0xFFu) << (8 * w);
                x[e] = v;
            }
        } else {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t h[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t d = t[w] & 2 ? y[w][2 * b + 1] : y[w][2 * b];
                    h[w] = t[w] & 1 ? d >> 16 : d & 0xFFFFu;
                }
                x[2 * b] = h[0] | h[1] << 16;
                x[2 * b + 1] = h[2] | h[3] << 16;
            }
        }
        *to = x;
    }
};

__global__ __launch_bounds__(256) void compact_rows_kernel(CompactArgs a) {
    extern __shared__ __attribute__((aligned(16))) u32x4 rows[];  // out of order: [acc_cols][CR_PIECES]
    __shared__ int64_t s_src[MAX_DRAFT], s_dst[MAX_DRAFT];
    __shared__ int s_tok[MAX_DRAFT];  // token in the sub-page: source, target << 8
    __shared__ int64_t s_quad[MAX_QUADS];  // target quads with a row: sub-page, and its quad in it in the low bits
    __shared__ int s_row[MAX_QUADS][4];    // the row that each of its tokens takes, or -1
    __shared__ int s_n, s_nquad, s_ascending;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int s = blockIdx.x;
    if (wv == 0) {
        // (loaded together: the entries past the count are not used)
        const int entry = lane < a.acc_cols ? a.accepted[(int64_t)s * a.acc_stride + lane] : -1;
        const int nq = a.qsl[s + 1] - a.qsl[s];
        const int n = min(min(a.count[s], a.acc_cols), min(nq, MAX_DRAFT));
        const int64_t ctx = (int64_t)a.seq_lens[s] - nq;
        const int from = lane < n ? entry : -1;
        const bool moves = from >= 0 && from < nq && from != lane;
        const int64_t src = moves ? sub_of(a, s, ctx + from) : -1, dst = moves ? sub_of(a, s, ctx + lane) : -1;
        const uint64_t ok = __builtin_amdgcn_ballot_w64(src >= 0 && dst >= 0);
        // quads of targets: lane i is token (ctx + i) & 3 of one; a quad is led by its first lane that moves
        const int tok = (int)((ctx + lane) & 3);
        const int lead = lane - tok;  // the quad's token 0 (before lane 0 in the first quad)
        const uint64_t quad_ok = (lead >= 0 ? ok >> lead : ok << -lead) & 15;  // bit w: token w of the quad moves
        const bool leads = (ok >> lane & 1) && (quad_ok & ((1u << tok) - 1)) == 0;
        const uint64_t leaders = __builtin_amdgcn_ballot_w64(leads);
        if (leads) {
            const int q = __builtin_popcountll(leaders & ((1ull << lane) - 1));
            s_quad[q] = dst | (int)((ctx + lane) >> 2 & 3);
            for (int w = 0; w < 4; ++w)
                s_row[q][w] = quad_ok >> w & 1 ? __builtin_popcountll(ok & ((1ull << (lead + w)) - 1)) : -1;
        }
        if (src >= 0 && dst >= 0) {
            const int at = __builtin_popcountll(ok & ((1ull << lane) - 1));
            s_src[at] = src;
            s_dst[at] = dst;
            s_tok[at] = (int)((ctx + from) & 15) | (int)((ctx + lane) & 15) << 8;  // (block sizes are multiples of 16)
        }
        // no row is read after an earlier one was written over it where every
        // row moves down: its source is behind all targets up to its own
        const bool down = __builtin_amdgcn_ballot_w64(src >= 0 && dst >= 0 && from < lane) == 0;
        if (lane == 0) {
            s_n = __builtin_popcountll(ok);
            s_nquad = __builtin_popcountll(leaders);
            s_ascending = down;
        }
    }
    __syncthreads();
    const int n = s_n, nquad = s_nquad;
    if (n == 0) return;
    const int pairs = a.layers * a.Hkv;
    if (s_ascending) {
        for (int p = blockIdx.y * 4 + wv; p < pairs; p += gridDim.y * 4) {
            const int layer = p / a.Hkv;
            const int64_t head = (int64_t)(p - layer * a.Hkv) * a.chs;
            uint8_t *const kb = (a.list ? a.k[layer] : a.k[0] + layer * a.layer_stride) + head;
            uint8_t *const vb = (a.list ? a.v[layer] : a.v[0] + layer * a.layer_stride) + head;
            // the first pieces' loads all go out before the first store
            KPiece k0;
            VQuad v0, v1;
            const int nk = 9 * n, nv = CR_QUAD * nquad;
            if (lane < nk) k0.load(kb, lane, s_src, s_tok);
            if (lane < nv) v0.load(vb, lane, s_quad, s_row, s_src, s_tok);
            if (lane + 64 < nv) v1.load(vb, lane + 64, s_quad, s_row, s_src, s_tok);
            if (lane < nk) k0.store(kb, s_dst);
            if (lane < nv) v0.store();
            if (lane + 64 < nv) v1.store();
            for (int u = lane + 64; u < nk; u += 64) {
                k0.load(kb, u, s_src, s_tok);
                k0.store(kb, s_dst);
            }
            for (int u = lane + 128; u < nv; u += 64) {
                v0.load(vb, u, s_quad, s_row, s_src, s_tok);
                v0.store();
            }
        }
        return;
    }
    // any order: the workgroup takes one pair at a time, all rows through LDS
    for (int p = blockIdx.y; p < pairs; p += gridDim.y) {
        const int layer = p / a.Hkv;
        const int64_t head = (int64_t)(p - layer * a.Hkv) * a.chs;
        uint8_t *const kb = (a.list ? a.k[layer] : a.k[0] + layer * a.layer_stride) + head;
        uint8_t *const vb = (a.list ? a.v[layer] : a.v[0] + layer * a.layer_stride) + head;
        for (int u = threadIdx.x; u < n * CR_PIECES; u += 256) {
            const int r = u / CR_PIECES, c = u - CR_PIECES * r;
            rows[u] = *reinterpret_cast<const u32x4 *>((c < 9 ? kb : vb) + s_src[r] + piece_off(c, s_tok[r] & 15));
        }
        __syncthreads();
        for (int u = threadIdx.x; u < n * CR_PIECES; u += 256) {
            const int r = u / CR_PIECES, c = u - CR_PIECES * r;
            piece_store((c < 9 ? kb : vb) + s_dst[r], c, s_tok[r] & 15, s_tok[r] >> 8, rows[u]);
        }
        __syncthreads();  // rows[] is filled again
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
    if (!plane_ok(k_cache, v_cache, cache_block_stride, cache_head_stride) ||
        (((uintptr_t)k_out | (uintptr_t)v_out) & 15u) || (os & 7u)) {
        fprintf(stderr, "[gfx906_fa_amd] read_rows: cache and outputs must be 16-byte aligned, output strides multiples "
                        "of 8 elements\n");
        return hipErrorInvalidValue;
    }
    if (num_rows == 0) return hipSuccess;
    const int64_t blocks = ((num_rows + 15) / 16 * num_kv_heads + 3) / 4;
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
    // one cache as two layers would be compacted twice, by waves that race
    bool twice = !list && num_layers > 1 && layer_stride == 0;
    for (int i = 0; list && i < num_layers; ++i)
        for (int j = 0; j < i; ++j) twice = twice || k_layers[i] == k_layers[j] || v_layers[i] == v_layers[j];
    if (twice) {
        fprintf(stderr, "[gfx906_fa_amd] compact_draft_rows: two layers share a cache\n");
        return hipErrorInvalidValue;
    }
    if (num_seqs == 0 || num_layers == 0 || accepted_cols == 0) return hipSuccess;
    if ((int64_t)num_layers * num_kv_heads > (1 << 24)) {
        fprintf(stderr, "[gfx906_fa_amd] compact_draft_rows: too many layers\n");
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
    const size_t lds = (size_t)accepted_cols * CR_PIECES * 16;
    static_assert(MAX_DRAFT * CR_PIECES * 16 + 3 * 512 <= 64 * 1024, "LDS of a workgroup");
    for (int l0 = 0; l0 < num_layers; l0 += list ? LAYERS : num_layers) {
        const int nl = list ? min(LAYERS, num_layers - l0) : num_layers;
        for (int i = 0; i < (list ? nl : 1); ++i) {
            a.k[i] = list ? k_layers[l0 + i] : k_cache;
            a.v[i] = list ? v_layers[l0 + i] : v_cache;
        }
        a.layers = nl;
        // (layer, kv-head) pairs a wave takes: more where they alone fill the device
        const int64_t pairs = (int64_t)nl * num_kv_heads;
        const int64_t each = max((int64_t)1, min((int64_t)8, (pairs * num_seqs + CR_WAVES - 1) / CR_WAVES));
        const int64_t wgs = min((pairs + 4 * each - 1) / (4 * each), (int64_t)65535);
        compact_rows_kernel<<<dim3(num_seqs, (unsigned)wgs), 256, lds, stream>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
