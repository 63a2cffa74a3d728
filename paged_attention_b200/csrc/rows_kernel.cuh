#pragma once
// Rows of q, k and v on their way to the attention: per-head RMS norm and position rotation in one pass, either
// back to dense rows (SINK_DENSE) or with k and v going straight to their pages (the other sinks).  No counterpart
// in the reference, whose append copies K/V that the caller has already normed and rotated.
//
//   n_d = x_d * w_d * rsqrt(mean(x^2) + eps)                                  (with a weight)
//   (y_lo, y_hi) = s * (n_lo cos t - n_hi sin t, n_hi cos t + n_lo sin t)     pairs of the first rotary_dim dims
//   t = position[axis_i] * inv_freq_i
//
// Everything between the load and the one rounding of the store is fp32.  The angle is kept as a fraction of a
// turn in 64-bit fixed point: inv_freq / 2 pi is rounded once to a multiple of 2^-64 turn on the host, and position *
// step mod 2^64 is exact integer arithmetic, so a position of 10^6 is as accurate as position 1 (an fp32 angle would
// be off by 0.03 rad there) and no table of sines has to be read.
//
// A head of 128 dims belongs to 8 lanes with two 16-byte chunks each, chosen so that both members of every rotated
// pair meet in one lane; a warp instruction moves four heads (1 KB).  The sines of a token are computed once per
// warp (two frequencies per lane) and shared by all heads the warp takes.
//
// Bound: memory.  One read of the rows and one write of the results, ~10 instructions per element pair.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace pdk {

constexpr int ROWS_WARPS   = 4;             // warps per CTA: small CTAs spread short calls over the SMs
constexpr int ROWS_THREADS = ROWS_WARPS * 32;
constexpr int ROWS_UNROLL  = 4;             // head groups (1 KB each) a warp has in flight
constexpr int MAX_FREQS    = 64;
constexpr int MAX_BLOCK    = 16;            // tokens that share a scale, at most
// block scales are powers of two in [2^-32, 2^8]: 2^-32 * 448 is below the smallest fp16 number, 2^8 * 448 above the largest
constexpr int MIN_SCALE_EXP = -32, MAX_SCALE_EXP = 8;

constexpr unsigned ST_APPEND_RANGE = 7;     // a token's place lies outside the block table or its page outside the pool

struct RopeArgs {
    unsigned long long step[MAX_FREQS];     // turn fraction per position, 64-bit fixed point
    unsigned char      axis[MAX_FREQS];     // which row of `positions` drives the frequency
    float scale;                            // multiplies sine and cosine
    int   rotary_dim;                       // 0: no rotation
    int   interleaved;                      // pairs (2i, 2i+1) instead of (i, i + rotary_dim/2)
    int   axes;                             // 1 + highest axis
};
struct RowArgs {
    const void *q, *k, *v;                  // [tokens][heads][128], rows *_stride elements apart
    long long q_stride, k_stride, v_stride;
    const void *q_norm, *k_norm;            // [128] or null
    const int* positions;                   // [axes][positions_stride], or null: the token's place in the cache
    long long positions_stride;
    int   tokens, hq, hkv;
    float eps;
    void* q_out;
    long long q_out_stride;
    void* k_out;                            // SINK_DENSE only
    long long k_out_stride;
    int   warps_per_row;
};
struct PageArgs {
    void *k_cache, *v_cache;
    const int* block_table;                 // [num_slots][table_stride]
    const int* start_pos;                   // [batch] tokens of each sequence before this call; null: first_pos for all
    const int* token_begin;                 // [batch + 1] rows of each sequence; null: see one_sequence
    const int* slot_ids;                    // [batch]; null: identity; negative: the sequence is skipped
    const float *k_head_scales, *v_head_scales;
    float* block_scales;                    // [page][kv head][block of the page][K, V]
    const void* const* k_src;               // [batch] per-sequence row bases instead of RowArgs::k / v, or null
    const void* const* v_src;
    unsigned* status;
    float inv_k, inv_v;
    int   table_stride, num_slots, batch, num_pages, page_size, log2_block;
    int   first_pos;
    int   one_sequence;                     // token_begin null: 1 = all rows belong to sequence 0, 0 = row i is sequence i
    int   kv_ctas, window, splits;          // SINK_BLOCKS: CTAs [0, kv_ctas) write pages, each a (window of rows, share of
                                            // the heads); the rest take the q rows
};

enum RowSink { SINK_DENSE = 0, SINK_FP16 = 1, SINK_E4M3 = 2, SINK_BLOCKS = 3 };

template<typename ACT> struct Act;
template<> struct Act<__half> {
    static __device__ __forceinline__ float2 to_f32(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t from_f32(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template<> struct Act<__nv_bfloat16> {
    static __device__ __forceinline__ float2 to_f32(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t from_f32(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template<typename ACT>
__device__ __forceinline__ void unpack8(const uint4& r, float (&x)[16], int at) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = Act<ACT>::to_f32(w[i]);
        x[at + 2 * i] = f.x; x[at + 2 * i + 1] = f.y;
    }
}
template<typename ACT>
__device__ __forceinline__ uint4 pack8(const float (&x)[16], int at) {
    return make_uint4(Act<ACT>::from_f32(x[at], x[at + 1]), Act<ACT>::from_f32(x[at + 2], x[at + 3]),
                      Act<ACT>::from_f32(x[at + 4], x[at + 5]), Act<ACT>::from_f32(x[at + 6], x[at + 7]));
}
// Eight values to e4m3 (round to nearest even, saturating).
__device__ __forceinline__ uint2 quant8(const float (&x)[16], int at, float inv) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[at + 2 * i] * inv, x[at + 2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// The two 16-byte chunks (8 dims) of a head that lane j of its 8 owns.  Adjacent-half pairs: chunk c < R/16 meets
// chunk c + R/16, what is left of the head goes to the other lanes in twos.  (Interleaved pairs lie inside a chunk.)
struct Chunks { int a, b; bool rot_a, rot_b; };
__device__ __forceinline__ Chunks chunks_of(int j, int rotary_dim, bool interleaved) {
    const int half = rotary_dim >> 4;
    Chunks c;
    if (j < half) { c.a = j; c.b = j + half; c.rot_a = c.rot_b = true; }
    else          { c.a = 2 * j; c.b = 2 * j + 1; c.rot_a = c.rot_b = false; }
    if (interleaved) { c.rot_a = 8 * c.a < rotary_dim; c.rot_b = 8 * c.b < rotary_dim; }
    return c;
}
// (cos, sin) of one frequency at one position.
__device__ __forceinline__ float2 cos_sin(const RopeArgs& rope, int freq, int position) {
    const unsigned long long turn = static_cast<unsigned long long>(static_cast<long long>(position)) * rope.step[freq];
    float s, c;
    sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 0x1p-31f, &s, &c);   // top 32 bits: the turn in [-1/2, 1/2)
    return make_float2(c * rope.scale, s * rope.scale);
}
// This lane's eight (cos, sin) out of a token's table: four per chunk (interleaved) or one per pair.
__device__ __forceinline__ void load_cs(const float2* table, const Chunks& ch, bool interleaved, float2 (&cs)[8]) {
    const int fa = interleaved ? 4 * ch.a : 8 * ch.a, fb = interleaved ? 4 * ch.b : 8 * ch.a + 4;
    const float4* ta = reinterpret_cast<const float4*>(table + fa);
    const float4* tb = reinterpret_cast<const float4*>(table + fb);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float4 u = ch.rot_a ? ta[i] : make_float4(1.f, 0.f, 1.f, 0.f);
        const float4 w = ch.rot_b ? tb[i] : make_float4(1.f, 0.f, 1.f, 0.f);
        cs[2 * i] = make_float2(u.x, u.y); cs[2 * i + 1] = make_float2(u.z, u.w);
        cs[4 + 2 * i] = make_float2(w.x, w.y); cs[5 + 2 * i] = make_float2(w.z, w.w);
    }
}
// Rotates the lane's pairs.  Unrotated chunks are skipped, not multiplied by (1, 0): an infinity there must not turn its
// partner into a NaN.
__device__ __forceinline__ void rotate(float (&x)[16], const float2 (&cs)[8], const Chunks& ch, bool interleaved) {
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i < 4 ? ch.rot_a : ch.rot_b) {
                const float lo = x[2 * i], hi = x[2 * i + 1];
                x[2 * i]     = lo * cs[i].x - hi * cs[i].y;
                x[2 * i + 1] = hi * cs[i].x + lo * cs[i].y;
            }
        }
    } else if (ch.rot_a) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float lo = x[i], hi = x[8 + i];
            x[i]     = lo * cs[i].x - hi * cs[i].y;
            x[8 + i] = hi * cs[i].x + lo * cs[i].y;
        }
    }
}
// RMS norm of a head held by 8 neighbouring lanes; the weight (null: none) may differ between the heads of a warp.
template<typename ACT>
__device__ __forceinline__ void norm_head(float (&x)[16], const void* weight, const Chunks& ch, float eps) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!weight) return;
    const float r = rsqrtf(ss * (1.f / 128.f) + eps);
    float w[16];
    unpack8<ACT>(__ldg(static_cast<const uint4*>(weight) + ch.a), w, 0);
    unpack8<ACT>(__ldg(static_cast<const uint4*>(weight) + ch.b), w, 8);
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = x[i] * r * w[i];
}

// The sequence a row belongs to and its place there.  Called by whole warps; every lane gets the answer.
struct Place {
    int seq, slot;      // slot < 0: the row belongs to no sequence, or to a skipped one
    int begin, end;     // the sequence's rows
    int pos;            // the token's position in the sequence, -1 where it is negative or passes 2^31
};
__device__ __forceinline__ Place locate(const PageArgs& t, int row, int tokens, int lane) {
    Place p{-1, -1, 0, 0, 0};
    if (t.token_begin == nullptr) {
        p.seq = t.one_sequence ? 0 : row;
        if (p.seq >= t.batch) return p;
        p.begin = t.one_sequence ? 0 : row;
        p.end   = t.one_sequence ? tokens : row + 1;
    } else {
        // smallest b with token_begin[b + 1] > row, 32 probes at a time
        int lo = 0, n = t.batch;
        for (;;) {
            const int step = (n + 31) >> 5;
            const int last = min(lo + (lane + 1) * step, lo + n);          // token_begin[last] ends this lane's chunk
            const bool over = __ldg(t.token_begin + last) <= row;
            const int skip = __popc(__ballot_sync(0xffffffffu, over)) * step;
            if (skip >= n) return p;                                       // behind the last sequence
            lo += skip;
            n = min(step, n - skip);
            if (step == 1) break;
        }
        p.seq   = lo;
        p.begin = __ldg(t.token_begin + lo);
        p.end   = min(__ldg(t.token_begin + lo + 1), tokens);
        if (row < p.begin) { p.end = p.begin; return p; }                  // rows before the first sequence
    }
    p.slot = t.slot_ids ? __ldg(t.slot_ids + p.seq) : p.seq;
    if (p.slot < 0) return p;
    const int first = t.start_pos ? __ldg(t.start_pos + p.seq) : t.first_pos;
    const long long pos = static_cast<long long>(first) + (row - p.begin);
    p.pos = pos < 0 || pos > 0x7fffffff ? -1 : static_cast<int>(pos);
    return p;
}
// The page of a position, or -1 (reported in the status word): outside the table, or outside the pool.
__device__ __forceinline__ int page_of(const PageArgs& t, const Place& p, int row) {
    const int index = p.pos / t.page_size;
    int page = -1;
    if (p.pos >= 0 && p.slot < t.num_slots && index < t.table_stride) {
        page = __ldg(t.block_table + static_cast<size_t>(p.slot) * t.table_stride + index);
        if (page >= t.num_pages) page = -1;
    }
    if (page < 0) {
        atomicCAS(t.status, 0u, (ST_APPEND_RANGE << 24) | (row & 0xffffffu));
        return -1;
    }
    return page;
}
// Rotation position of frequency `freq` for row `row` (`pos` = its place in the cache).
__device__ __forceinline__ int rope_position(const RowArgs& a, const RopeArgs& rope, int freq, int row, int pos) {
    if (!a.positions) return pos;
    const int axis = rope.axes > 1 ? rope.axis[freq] : 0;
    return __ldg(a.positions + axis * a.positions_stride + row);
}

// k and v of one block of at most 16 tokens: all its new rows meet in one warp per (head, K or V), which finds the
// block's largest magnitude, settles the scale and quantises.  Blocks are written by the CTA whose window of rows holds
// their first new token.  A scale is a power of two, so when a block that was begun by an earlier call needs a
// larger one its other bytes only change exponent: exact while they stay normal, one more rounding of at most half
// a step of the subnormal range below that.  The whole block is re-encoded, slots behind the new tokens included: what a
// byte stands for does not change.
template<typename ACT>
__device__ __forceinline__ void write_blocks(const RowArgs& a, const RopeArgs& rope, const PageArgs& t, float2 (*table)[MAX_FREQS]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sh = lane >> 3, j = lane & 7;
    const int window = blockIdx.x / t.splits, split = blockIdx.x % t.splits;
    const int block = 1 << t.log2_block, per_page = t.page_size >> t.log2_block;
    const bool interleaved = rope.interleaved != 0;
    const Chunks ch = chunks_of(j, rope.rotary_dim, interleaved);
    const int stop = min((window + 1) * t.window, a.tokens);
    for (int row = window * t.window; row < stop;) {
        const Place p = locate(t, row, a.tokens, lane);
        if (p.slot < 0) { row = max(row + 1, p.end); continue; }              // no sequence's row, or a skipped sequence
        const int inside = p.pos & (block - 1);                               // page sizes are multiples of the block
        const int n = min(block - inside, p.end - row);
        const int first_row = row;
        row += max(1, n);
        if (inside != 0 && first_row != p.begin) continue;                    // begun in an earlier window
        const int page = page_of(t, p, first_row);
        if (page < 0) continue;
        const int off = p.pos % t.page_size;
        if (rope.rotary_dim) {
            __syncthreads();                                                  // the previous block's table has been read
            const int freqs = rope.rotary_dim >> 1;
            for (int i = threadIdx.x; i < n * freqs; i += ROWS_THREADS) {
                const int r = i / freqs, f = i - r * freqs;
                table[r][f] = cos_sin(rope, f, rope_position(a, rope, f, first_row + r, p.pos + r));
            }
            __syncthreads();
        }
        for (int u = split * ROWS_WARPS + warp; u < 2 * a.hkv; u += t.splits * ROWS_WARPS) {
            const bool is_v = u >= a.hkv;
            const int h = is_v ? u - a.hkv : u;
            const ACT* src;
            long long stride = is_v ? a.v_stride : a.k_stride;
            if (t.k_src) src = static_cast<const ACT*>((is_v ? t.v_src : t.k_src)[p.seq]) + (first_row - p.begin) * stride;
            else         src = static_cast<const ACT*>(is_v ? a.v : a.k) + first_row * stride;
            src += h * 128;
            float* scale_at = t.block_scales + 2 * ((static_cast<size_t>(page) * a.hkv + h) * per_page + (off >> t.log2_block)) + is_v;
            float old = inside ? *scale_at : 0.f;
            uint4 raw[4][2];
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const int r = 4 * s + sh;
                raw[s][0] = raw[s][1] = make_uint4(0, 0, 0, 0);
                if (r < n) {
                    raw[s][0] = __ldcs(reinterpret_cast<const uint4*>(src + r * stride) + ch.a);
                    raw[s][1] = __ldcs(reinterpret_cast<const uint4*>(src + r * stride) + ch.b);
                }
            }
            float x[4][16], top = 0.f;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                if (4 * s >= n) break;                                        // warp-uniform
                unpack8<ACT>(raw[s][0], x[s], 0);
                unpack8<ACT>(raw[s][1], x[s], 8);
                if (!is_v) {
                    if (a.k_norm) norm_head<ACT>(x[s], a.k_norm, ch, a.eps);
                    if (rope.rotary_dim && 4 * s + sh < n) {
                        float2 cs[8];
                        load_cs(table[4 * s + sh], ch, interleaved, cs);
                        rotate(x[s], cs, ch, interleaved);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; i++) top = fmaxf(top, fabsf(x[s][i]));   // a NaN does not count
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            // smallest power of two with top / scale <= 448 = 1.75 * 2^8
            const unsigned bits = __float_as_uint(top);
            int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
            e = max(MIN_SCALE_EXP, min(MAX_SCALE_EXP, e));
            const float need = __uint_as_float(static_cast<unsigned>(e + 127) << 23);
            old = old > 0.f ? old : 0.f;
            const float scale = fmaxf(old, need), inv = __frcp_rn(scale);
            unsigned char* dst = static_cast<unsigned char*>(is_v ? t.v_cache : t.k_cache)
                + ((static_cast<size_t>(page) * a.hkv + h) * t.page_size + off) * 128;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const int r = 4 * s + sh;
                if (r < n) {
                    *reinterpret_cast<uint2*>(dst + r * 128 + ch.a * 8) = quant8(x[s], 0, inv);
                    *reinterpret_cast<uint2*>(dst + r * 128 + ch.b * 8) = quant8(x[s], 8, inv);
                }
            }
            if (inside && scale > old) {                                      // warp-uniform
                const float ratio = old * inv;
                unsigned char* was = dst - inside * 128;
                for (int r = sh; r < block; r += 4) {
                    if (r >= inside && r < inside + n) continue;              // just written
                    uint4* at = reinterpret_cast<uint4*>(was + r * 128) + j;
                    const uint4 b = *at;
                    const uint32_t in[4] = {b.x, b.y, b.z, b.w};
                    uint32_t out[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(in[i] & 0xffffu), __NV_E4M3);
                        const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(in[i] >> 16), __NV_E4M3);
                        const float2 l = __half22float2(__half2(lo)), g = __half22float2(__half2(hi));
                        out[i] = __nv_cvt_float2_to_fp8x2(make_float2(l.x * ratio, l.y * ratio), __NV_SATFINITE, __NV_E4M3)
                               | (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(g.x * ratio, g.y * ratio), __NV_SATFINITE, __NV_E4M3)) << 16);
                    }
                    *at = make_uint4(out[0], out[1], out[2], out[3]);
                }
            }
            if (lane == 0) *scale_at = scale;
        }
    }
}

// One warp takes warps_per_row-th of a row's heads, four at a time.  Short calls split a row over many warps (latency is
// all that counts there), long ones give each row to one warp, which then computes the row's sines once.
template<typename ACT, int SINK>
__global__ void __launch_bounds__(ROWS_THREADS)
rows_kernel(const __grid_constant__ RowArgs a, const __grid_constant__ RopeArgs rope, const __grid_constant__ PageArgs t)
{
    __shared__ __align__(16) float2 table[SINK == SINK_BLOCKS ? MAX_BLOCK : ROWS_WARPS][MAX_FREQS];
    int cta = blockIdx.x;
    if constexpr (SINK == SINK_BLOCKS) {
        if (cta < t.kv_ctas) { write_blocks<ACT>(a, rope, t, table); return; }
        cta -= t.kv_ctas;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sh = lane >> 3, j = lane & 7;
    const unsigned unit = static_cast<unsigned>(cta) * ROWS_WARPS + warp;
    const int row = static_cast<int>(unit / static_cast<unsigned>(a.warps_per_row));
    const int sub = static_cast<int>(unit % static_cast<unsigned>(a.warps_per_row));
    if (row >= a.tokens) return;
    const bool interleaved = rope.interleaved != 0;
    const Chunks ch = chunks_of(j, rope.rotary_dim, interleaved);
    const int heads = SINK == SINK_BLOCKS ? a.hq : SINK == SINK_DENSE ? a.hq + a.hkv : a.hq + 2 * a.hkv;
    const int groups = (heads + 3) >> 2;
    const ACT* q_row = static_cast<const ACT*>(a.q) + row * a.q_stride;
    const ACT* k_row = static_cast<const ACT*>(a.k) + row * a.k_stride;
    const ACT* v_row = static_cast<const ACT*>(a.v) + row * a.v_stride;
    auto head_ptr = [&](int head) {
        return head < a.hq ? q_row + head * 128 : head < a.hq + a.hkv ? k_row + (head - a.hq) * 128 : v_row + (head - a.hq - a.hkv) * 128;
    };
    uint4 raw[ROWS_UNROLL][2];
    auto fetch = [&](int group) {
#pragma unroll
        for (int u = 0; u < ROWS_UNROLL; u++) {
            const int head = (group + u * a.warps_per_row) * 4 + sh;
            raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
            if (head < heads) {
                const uint4* p = reinterpret_cast<const uint4*>(head_ptr(head));
                raw[u][0] = __ldcs(p + ch.a);
                raw[u][1] = __ldcs(p + ch.b);
            }
        }
    };
    bool from_seq = false;
    if constexpr (SINK == SINK_FP16 || SINK == SINK_E4M3) from_seq = t.k_src != nullptr;
    if (!from_seq) fetch(sub);                      // on their way while the row's place is looked up

    Place p{0, 0, 0, 0, 0};
    size_t base = 0;                                // first element of the token's row of kv head 0
    bool stored = true;
    if constexpr (SINK != SINK_DENSE) {
        p = locate(t, row, a.tokens, lane);
        if (p.slot < 0) return;                     // no sequence's row: left as it is
        if constexpr (SINK != SINK_BLOCKS) {
            const int page = page_of(t, p, row);
            stored = page >= 0;
            base = (static_cast<size_t>(max(page, 0)) * a.hkv * t.page_size + max(p.pos, 0) % t.page_size) * 128;
            if (from_seq) {
                k_row = static_cast<const ACT*>(t.k_src[p.seq]) + (row - p.begin) * a.k_stride;
                v_row = static_cast<const ACT*>(t.v_src[p.seq]) + (row - p.begin) * a.v_stride;
                fetch(sub);
            }
        }
    }
    float2 cs[8];
    if (rope.rotary_dim) {
        for (int f = lane; f < rope.rotary_dim >> 1; f += 32)
            table[warp][f] = cos_sin(rope, f, rope_position(a, rope, f, row, p.pos));
        __syncwarp();
        load_cs(table[warp], ch, interleaved, cs);
    }

    for (int group = sub; group < groups;) {
#pragma unroll
        for (int u = 0; u < ROWS_UNROLL; u++) {
            if ((group + u * a.warps_per_row) * 4 >= heads) break;           // warp-uniform
            const int head = (group + u * a.warps_per_row) * 4 + sh;
            const bool is_q = head < a.hq, is_v = head >= a.hq + a.hkv;
            float x[16];
            unpack8<ACT>(raw[u][0], x, 0);
            unpack8<ACT>(raw[u][1], x, 8);
            if (a.q_norm || a.k_norm) norm_head<ACT>(x, is_v ? nullptr : is_q ? a.q_norm : a.k_norm, ch, a.eps);
            if (rope.rotary_dim && !is_v) rotate(x, cs, ch, interleaved);
            if (head >= heads) continue;
            if (SINK == SINK_DENSE) {
                ACT* dst = is_q ? static_cast<ACT*>(a.q_out) + row * a.q_out_stride + head * 128
                                : static_cast<ACT*>(a.k_out) + row * a.k_out_stride + (head - a.hq) * 128;
                reinterpret_cast<uint4*>(dst)[ch.a] = pack8<ACT>(x, 0);
                reinterpret_cast<uint4*>(dst)[ch.b] = pack8<ACT>(x, 8);
            } else if (is_q) {
                __half* dst = static_cast<__half*>(a.q_out) + row * a.q_out_stride + head * 128;   // what the decode reads
                reinterpret_cast<uint4*>(dst)[ch.a] = pack8<__half>(x, 0);
                reinterpret_cast<uint4*>(dst)[ch.b] = pack8<__half>(x, 8);
            } else if (SINK != SINK_BLOCKS && stored) {
                const int h = head - a.hq - (is_v ? a.hkv : 0);
                const size_t at = base + static_cast<size_t>(h) * t.page_size * 128;
                if (SINK == SINK_FP16) {
                    uint4* dst = reinterpret_cast<uint4*>(static_cast<__half*>(is_v ? t.v_cache : t.k_cache) + at);
                    dst[ch.a] = pack8<__half>(x, 0);
                    dst[ch.b] = pack8<__half>(x, 8);
                } else {
                    const float* hs = is_v ? t.v_head_scales : t.k_head_scales;
                    const float inv = hs ? __frcp_rn(__ldg(hs + h)) : is_v ? t.inv_v : t.inv_k;
                    uint2* dst = reinterpret_cast<uint2*>(static_cast<unsigned char*>(is_v ? t.v_cache : t.k_cache) + at);
                    dst[ch.a] = quant8(x, 0, inv);
                    dst[ch.b] = quant8(x, 8, inv);
                }
            }
        }
        group += ROWS_UNROLL * a.warps_per_row;
        if (group < groups) fetch(group);
    }
}

}  // namespace pdk
