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
// Bound: memory, one read of the rows and one write of the results.  Measured on B200 against that traffic at the
// measured copy rate (6.55 TB/s): 8192 bf16 rows of 40 heads with norm 28.8 us (89 %), 65536 of them 201 us (102 %), 20001
// rows of 72 heads 113 us (99 %), prompts of 33,000 rows of 80 heads into an fp16 cache 206 us (100 %), ragged chunks of
// 12,000 rows into an e4m3 cache 48 us (87 %), of 15,500 into a block-scaled one 65 us (82 %; 87 % at four times the rows); one
// row 2.3 us, a launch.  What is missing at the smaller sizes is 3 us of first loads and last stores.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <type_traits>

namespace pdk {

constexpr int ROWS_WARPS   = 4;             // warps per CTA: small CTAs spread short calls over the SMs
constexpr int ROWS_THREADS = ROWS_WARPS * 32;
constexpr int ROWS_SLOTS   = 4;             // units (four heads, 1 KB) a warp has in flight: 8 measured the same
constexpr int MAX_FREQS    = 64;
constexpr int MAX_BLOCK    = 16;            // tokens that share a scale, at most
// block scales are powers of two in [2^-32, 2^8]: under 2^-32 the smallest fp16 number, 2^-24, is 256; 2^8 * 448 is above the largest
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
    const void* const* k_src;               // SINK_BLOCKS: [batch] per-sequence row bases instead of RowArgs::k / v, or null
    const void* const* v_src;
    unsigned* status;
    float inv_k, inv_v;
    int   table_stride, num_slots, batch, num_pages, page_size, log2_block;
    int   first_pos;
    int   one_sequence;                     // token_begin null: 1 = all rows belong to sequence 0, 0 = row i is sequence i
    int   kv_ctas, window, splits;          // SINK_BLOCKS: so many CTAs write pages, each a (window of rows, share of the
                                            // heads); the rest take the q rows
};

enum RowSink { SINK_DENSE = 0, SINK_FP16 = 1, SINK_E4M3 = 2, SINK_BLOCKS = 3 };

// Two fp32 values in one 64-bit register: sm_100a multiplies and adds them with one instruction, which halves the
// arithmetic of norm and rotation.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pair(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split(F2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ F2 swap(F2 x) { const float2 v = split(x); return pair(v.y, v.x); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

template<typename ACT> struct Act;
template<> struct Act<__half> {
    static __device__ __forceinline__ F2 to_f32(uint32_t w) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        return pair(f.x, f.y);
    }
    static __device__ __forceinline__ uint32_t from_f32(F2 x) {
        const float2 f = split(x);
        const __half2 h = __floats2half2_rn(f.x, f.y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template<> struct Act<__nv_bfloat16> {
    static __device__ __forceinline__ F2 to_f32(uint32_t w) {
        return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t from_f32(F2 x) {
        const float2 f = split(x);
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
// A lane's 16 values: pairs 0..3 are chunk a, 4..7 chunk b.
struct Vals { F2 p[8]; };
struct Raw { uint4 a, b; };
template<typename ACT>
__device__ __forceinline__ Vals unpack(const Raw& r) {
    Vals x;
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; i++) x.p[i] = Act<ACT>::to_f32(w[i]);
    return x;
}
template<typename ACT>
__device__ __forceinline__ uint4 pack8(const Vals& x, int at) {
    return make_uint4(Act<ACT>::from_f32(x.p[at]), Act<ACT>::from_f32(x.p[at + 1]),
                      Act<ACT>::from_f32(x.p[at + 2]), Act<ACT>::from_f32(x.p[at + 3]));
}
__device__ __forceinline__ void scale_by(Vals& x, float s) {
    const F2 s2 = pair(s, s);
#pragma unroll
    for (int i = 0; i < 8; i++) x.p[i] = mul2(x.p[i], s2);
}
// Eight values to e4m3 (round to nearest even, saturating).
__device__ __forceinline__ uint2 quant8(const Vals& x, int at) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __nv_cvt_float2_to_fp8x2(split(x.p[at + i]), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// The two 16-byte chunks (8 dims) of a head that lane j of its 8 owns.  The first R/16 lanes hold the rotated dims, chunk
// j beside chunk j + R/16, which are each other's partners when halves are paired (adjacent pairs lie inside a chunk);
// the other lanes hold the rest.  Both chunks of neighbouring lanes are neighbours in memory (but for one break), so
// both loads of a unit touch whole sectors.
struct Chunks { int a, b; bool rot; };
__device__ __forceinline__ Chunks chunks_of(int j, int rotary_dim) {
    const int half = rotary_dim >> 4;
    return j < half ? Chunks{j, j + half, true} : Chunks{j + half, j + 8, false};
}
// The tables of a RopeArgs that is a kernel parameter, as ordinary pointers.  Every lane of a warp wants another entry, and an
// indexed load from the parameter space serves one entry at a time: 64 turns of a loop per token, a third of all
// instructions of a long append.  Through a generic address the same bytes come with one load.
struct RopeTables { const unsigned long long* step; const unsigned char* axis; };
__device__ __forceinline__ RopeTables rope_tables(const RopeArgs& rope) {
    RopeTables r{rope.step, rope.axis};
    asm volatile("" : "+l"(r.step), "+l"(r.axis));   // keeps the compiler from going back to the parameter space
    return r;
}
// (cos, sin) of one frequency at one position.
__device__ __forceinline__ float2 cos_sin(const RopeTables& tab, float scale, int freq, int position) {
    const unsigned long long turn = static_cast<unsigned long long>(static_cast<long long>(position)) * tab.step[freq];
    float s, c;
    sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 0x1p-31f, &s, &c);   // top 32 bits: the turn in [-1/2, 1/2)
    return make_float2(c * scale, s * scale);
}
// A lane's share of "times the weight, then rotated" as one linear map: y = x * diag + partner * cross, where the
// partner of a value is the other member of its pair.  With w the norm's weight (1 without one):
//   diag = w cos, cross_lo = -w_hi sin, cross_hi = w_lo sin;   outside the rotation diag = w and there is no partner.
struct HeadMap { F2 diag[8], cross[8]; };
template<typename ACT>
__device__ __forceinline__ HeadMap head_map(const float2* table, bool rotary, const Chunks& ch, bool interleaved, const void* weight) {
    HeadMap m;
    Vals w;
#pragma unroll
    for (int i = 0; i < 8; i++) w.p[i] = pair(1.f, 1.f);
    if (weight) {
        const uint4* wp = static_cast<const uint4*>(weight);
        w = unpack<ACT>(Raw{wp[ch.a], wp[ch.b]});
    }
#pragma unroll
    for (int i = 0; i < 8; i++) { m.diag[i] = w.p[i]; m.cross[i] = 0; }
    if (!rotary) return m;
    if (interleaved) {
        // pair (2i, 2i + 1) of a chunk: frequency 4 * chunk + i
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (ch.rot) {
                const float2 cs = table[4 * (i < 4 ? ch.a : ch.b) + (i & 3)], ww = split(w.p[i]);
                m.diag[i]  = pair(ww.x * cs.x, ww.y * cs.x);
                m.cross[i] = pair(-ww.y * cs.y, ww.x * cs.y);
            }
        }
    } else if (ch.rot) {
        const float4* t = reinterpret_cast<const float4*>(table + 8 * ch.a);    // two frequencies at a time
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 u = t[i];
            const float2 lo = split(w.p[i]), hi = split(w.p[4 + i]);
            m.diag[i]      = pair(lo.x * u.x, lo.y * u.z);
            m.diag[4 + i]  = pair(hi.x * u.x, hi.y * u.z);
            m.cross[i]     = pair(-hi.x * u.y, -hi.y * u.w);
            m.cross[4 + i] = pair(lo.x * u.y, lo.y * u.w);
        }
    }
    return m;
}
// Outside the rotation the partner is left out, not multiplied by zero: an infinity there must not become a NaN.
__device__ __forceinline__ void apply_map(Vals& x, const HeadMap& m, bool rotary, const Chunks& ch, bool interleaved) {
    Vals y;
#pragma unroll
    for (int i = 0; i < 8; i++) y.p[i] = mul2(x.p[i], m.diag[i]);
    if (rotary && interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (ch.rot) y.p[i] = fma2(swap(x.p[i]), m.cross[i], y.p[i]);
    } else if (rotary && ch.rot) {
#pragma unroll
        for (int i = 0; i < 8; i++) y.p[i] = fma2(x.p[i ^ 4], m.cross[i], y.p[i]);
    }
    x = y;
}
// 1 / rms of a head held by 8 neighbouring lanes.
__device__ __forceinline__ float inv_rms(const Vals& x, float eps) {
    F2 s2 = mul2(x.p[0], x.p[0]);
#pragma unroll
    for (int i = 1; i < 8; i++) s2 = fma2(x.p[i], x.p[i], s2);
    const float2 s = split(s2);
    float ss = s.x + s.y;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return rsqrtf(ss * (1.f / 128.f) + eps);
}

// What a kernel of this library may just have written - rows, scales, bytes of the pool - is read past L1: the kernel before may
// have brought older lines into the SM's L1 while this grid was already waiting for it (see rows_kernel).  Lists, positions
// and weights come from elsewhere and may use L1; nothing uses the non-coherent path.
__device__ __forceinline__ float load_float(const float* p) {
    float v;
    asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint4 load_16(const void* p) {
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
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
            const bool over = t.token_begin[last] <= row;
            const int skip = __popc(__ballot_sync(0xffffffffu, over)) * step;
            if (skip >= n) return p;                                       // behind the last sequence
            lo += skip;
            n = min(step, n - skip);
            if (step == 1) break;
        }
        p.seq   = lo;
        p.begin = t.token_begin[lo];
        p.end   = min(t.token_begin[lo + 1], tokens);
        if (row < p.begin) { p.end = p.begin; return p; }                  // rows before the first sequence
    }
    p.slot = t.slot_ids ? t.slot_ids[p.seq] : p.seq;
    if (p.slot < 0) return p;
    const int first = t.start_pos ? t.start_pos[p.seq] : t.first_pos;
    const long long pos = static_cast<long long>(first) + (row - p.begin);
    p.pos = pos < 0 || pos > 0x7fffffff ? -1 : static_cast<int>(pos);
    return p;
}
// Where a position's token lies: its page, or -1 (reported in the status word) where that is outside the table or the
// pool, and its place in the page.
struct Spot { int page, off; };
__device__ __forceinline__ Spot spot_of(const PageArgs& t, const Place& p, int row) {
    const unsigned pos = static_cast<unsigned>(max(p.pos, 0)), index = pos / static_cast<unsigned>(t.page_size);
    int page = -1;
    if (p.pos >= 0 && p.slot < t.num_slots && index < static_cast<unsigned>(t.table_stride)) {
        page = t.block_table[static_cast<size_t>(p.slot) * t.table_stride + index];
        if (page < 0 || page >= t.num_pages) page = -1;
    }
    if (page < 0) atomicCAS(t.status, 0u, (ST_APPEND_RANGE << 24) | (row & 0xffffffu));
    return Spot{page, static_cast<int>(pos - index * static_cast<unsigned>(t.page_size))};
}
// Rotation position of frequency `freq` for row `row` (`pos` = its place in the cache).
__device__ __forceinline__ int rope_position(const RowArgs& a, const RopeArgs& rope, const RopeTables& tab, int freq, int row, int pos) {
    if (!a.positions) return pos;
    const int axis = rope.axes > 1 ? tab.axis[freq] : 0;
    return a.positions[axis * a.positions_stride + row];
}

// 16 bytes global -> shared without waiting, past L1.
__device__ __forceinline__ void cp_async16(uint4* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template<int LEFT> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(LEFT) : "memory"); }
__device__ __forceinline__ uint4 load_shared(const uint4* p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))) : "memory");
    return v;
}

struct RowSmem {
    float2 table[ROWS_WARPS][MAX_FREQS];            // a warp's row: (cos, sin)
    uint4  slots[ROWS_WARPS][ROWS_SLOTS][2][32];    // [unit on its way][chunk][lane]
};
struct BlockSmem {
    uint4  map[MAX_BLOCK][8][8];                    // the block's rows: (diag, cross) of a lane's pair i at [row][i][lane of 8]
    uint4  slots[ROWS_WARPS][2][2][2][32];          // [warp][unit on its way][four rows][chunk][lane]
    float  top[ROWS_WARPS / 2][2][2];               // [pair of warps][parity][warp]: largest magnitude of the warp's rows
};

// k and v of one block of at most 16 tokens: all its new rows meet in two warps per (head, K or V), eight rows each, which
// find the block's largest magnitude, settle the scale and quantise what they still hold in registers.  (One warp
// with all 16 rows needs so many registers that it spills or has too little company on its SM.)  A block that gets eight
// rows or fewer, as in a decode step, takes one warp per (head, K or V).  Blocks are written by the CTA whose window of rows holds
// their first new token.  A scale is a power of two, so when a block that was begun by an earlier call needs a
// larger one its other bytes only change exponent: exact while they stay normal, one more rounding of at most half
// a step of the subnormal range below that.  The whole block is re-encoded, slots behind the new tokens included: what a
// byte stands for does not change.
// A K row's weights and sines are the same for all heads: the CTA multiplies them once per block into shared memory.  The
// next unit's rows are on their way while one is worked on.
template<typename ACT, bool HALVES>
__device__ __forceinline__ void write_blocks(const RowArgs& a, const RopeArgs& rope, const PageArgs& t, BlockSmem& sm) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane & 7;
    const int window = blockIdx.x / t.splits, share = blockIdx.x % t.splits;
    const int block = 1 << t.log2_block, per_page = t.page_size >> t.log2_block;
    const bool rotary = HALVES || rope.rotary_dim != 0, interleaved = !HALVES && rope.interleaved != 0;
    const bool mapped = rotary || a.k_norm != nullptr;
    const Chunks ch = HALVES ? Chunks{j, j + 8, true} : chunks_of(j, rope.rotary_dim);
    const int stop = min((window + 1) * t.window, a.tokens);
    int parity = 0;                                                           // of sm.top, over all blocks of the window
    for (int row = window * t.window; row < stop;) {
        const Place p = locate(t, row, a.tokens, lane);
        if (p.slot < 0) { row = max(row + 1, p.end); continue; }              // no sequence's row, or a skipped sequence
        const int inside = p.pos & (block - 1);                               // page sizes are multiples of the block
        const int n = min(block - inside, p.end - row);
        const int first_row = row;
        row += max(1, n);
        if (inside != 0 && first_row != p.begin) continue;                    // begun in an earlier window
        const Spot spot = spot_of(t, p, first_row);
        const int page = spot.page, off = spot.off;
        if (page < 0) continue;

        float* scales = t.block_scales + 2 * (static_cast<size_t>(page) * a.hkv * per_page + (off >> t.log2_block));   // of kv head 0
        const size_t row0 = (static_cast<size_t>(page) * a.hkv * t.page_size + off) * 128;                         // first row, kv head 0
        const bool paired = n > 8;
        const int half = paired ? warp & 1 : 0, mine = 8 * half + (lane >> 3);   // this lane's rows of the block: mine, mine + 4
        const size_t from = t.k_src ? first_row - p.begin : first_row;
        const ACT* k_rows = static_cast<const ACT*>(t.k_src ? t.k_src[p.seq] : a.k) + (from + mine) * a.k_stride + ch.a * 8;
        const ACT* v_rows = static_cast<const ACT*>(t.k_src ? t.v_src[p.seq] : a.v) + (from + mine) * a.v_stride + ch.a * 8;
        const int b_off = (ch.b - ch.a) * 8;
        const int team = paired ? warp >> 1 : warp, teams = paired ? ROWS_WARPS / 2 : ROWS_WARPS, step = t.splits * teams;
        auto fetch = [&](int u, int slot) {                                   // one commit group, empty behind the last unit
            if (u < 2 * a.hkv) {
                const bool is_v = u >= a.hkv;
                const ACT* src = is_v ? v_rows + (u - a.hkv) * 128 : k_rows + u * 128;
                const long long stride = 4 * (is_v ? a.v_stride : a.k_stride);
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    if (4 * s + mine >= n) break;
                    cp_async16(&sm.slots[warp][slot][s][0][lane], src);
                    cp_async16(&sm.slots[warp][slot][s][1][lane], src + b_off);
                    src += stride;
                }
            }
            cp_async_commit();
        };
        // the scale of a begun block, asked for a unit ahead like its rows
        auto begun_scale = [&](int u) {
            const bool is_v = u >= a.hkv;
            return inside && u < 2 * a.hkv ? load_float(scales + (is_v ? u - a.hkv : u) * 2 * per_page + is_v) : 0.f;
        };
        int u = share * teams + team, slot = 0;
        fetch(u, 0);
        float next = begun_scale(u);
        if (mapped) {
            __syncthreads();                                                  // the previous block's map has been read
            const RopeTables tab = rope_tables(rope);
            for (int e = threadIdx.x; e < n * 32; e += ROWS_THREADS) {        // (row, lane of 8, pairs i and i + 4)
                const int r = e >> 5, i = e >> 3 & 3, l = e & 7;
                const Chunks c = HALVES ? Chunks{l, l + 8, true} : chunks_of(l, rope.rotary_dim);
                float2 lo = make_float2(1.f, 1.f), hi = lo;                   // weights of the pairs
                if (a.k_norm) {
                    lo = split(Act<ACT>::to_f32(static_cast<const uint32_t*>(a.k_norm)[c.a * 4 + i]));
                    hi = split(Act<ACT>::to_f32(static_cast<const uint32_t*>(a.k_norm)[c.b * 4 + i]));
                }
                float4 ma = make_float4(lo.x, lo.y, 0.f, 0.f), mb = make_float4(hi.x, hi.y, 0.f, 0.f);
                if (rotary && c.rot) {
                    const int f0 = interleaved ? 4 * c.a + i : 8 * c.a + 2 * i, f1 = interleaved ? 4 * c.b + i : f0 + 1;
                    const float2 t0 = cos_sin(tab, rope.scale, f0, rope_position(a, rope, tab, f0, first_row + r, p.pos + r));
                    const float2 t1 = cos_sin(tab, rope.scale, f1, rope_position(a, rope, tab, f1, first_row + r, p.pos + r));
                    if (interleaved) {
                        ma = make_float4(lo.x * t0.x, lo.y * t0.x, -lo.y * t0.y, lo.x * t0.y);
                        mb = make_float4(hi.x * t1.x, hi.y * t1.x, -hi.y * t1.y, hi.x * t1.y);
                    } else {
                        ma = make_float4(lo.x * t0.x, lo.y * t1.x, -hi.x * t0.y, -hi.y * t1.y);
                        mb = make_float4(hi.x * t0.x, hi.y * t1.x, lo.x * t0.y, lo.y * t1.y);
                    }
                }
                *reinterpret_cast<float4*>(&sm.map[r][i][l])     = ma;
                *reinterpret_cast<float4*>(&sm.map[r][i + 4][l]) = mb;
            }
            __syncthreads();
        }

        auto run = [&](auto is_v_, int end) {                                 // this warp's units of K, then of V
            constexpr bool is_v = decltype(is_v_)::value;
#pragma unroll 1
            for (; u < end; u += step) {
                const int h = is_v ? u - a.hkv : u;
                float* scale_at = scales + h * 2 * per_page + is_v;
                float old = next;
                fetch(u + step, slot ^ 1);
                next = begun_scale(u + step);
                cp_async_wait<1>();
                Vals x[2];
                float top = 0.f;
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    if (8 * half + 4 * s >= n) break;                         // warp-uniform
                    const bool alive = 4 * s + mine < n;
                    Raw raw{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                    if (alive) raw = Raw{load_shared(&sm.slots[warp][slot][s][0][lane]), load_shared(&sm.slots[warp][slot][s][1][lane])};
                    x[s] = unpack<ACT>(raw);
                    if (!is_v && mapped) {
                        const float r = a.k_norm ? inv_rms(x[s], a.eps) : 1.f;
                        if (alive) {
#pragma unroll
                            for (int i = 0; i < 4; i++) {                     // apply_map, four registers of the map at a time
                                const ulonglong2 ma = *reinterpret_cast<const ulonglong2*>(&sm.map[4 * s + mine][i][j]);
                                const ulonglong2 mb = *reinterpret_cast<const ulonglong2*>(&sm.map[4 * s + mine][i + 4][j]);
                                const F2 xa = x[s].p[i], xb = x[s].p[i + 4];
                                F2 ya = mul2(xa, ma.x), yb = mul2(xb, mb.x);
                                if (rotary && ch.rot) {
                                    ya = fma2(interleaved ? swap(xa) : xb, ma.y, ya);
                                    yb = fma2(interleaved ? swap(xb) : xa, mb.y, yb);
                                }
                                x[s].p[i] = ya; x[s].p[i + 4] = yb;
                            }
                        }
                        if (a.k_norm) scale_by(x[s], r);
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {                             // a NaN does not count
                        const float2 f = split(x[s].p[i]);
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                }
                top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));   // not negative: ordered like its bits
                if (paired) {                                                 // both warps of a pair take the same units
                    if (lane == 0) sm.top[team][parity][half] = top;
                    asm volatile("bar.sync %0, 64;" :: "r"(1 + team) : "memory");
                    top = fmaxf(sm.top[team][parity][0], sm.top[team][parity][1]);
                    parity ^= 1;   // the other warp may still be reading; it has done so when the next barrier is passed
                }
                slot ^= 1;
                // smallest power of two with top / scale <= 448 = 1.75 * 2^8
                const unsigned bits = __float_as_uint(top);
                int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
                e = max(MIN_SCALE_EXP, min(MAX_SCALE_EXP, e));
                const float need = __uint_as_float(static_cast<unsigned>(e + 127) << 23);
                old = old > 0.f ? old : 0.f;
                const float scale = fmaxf(old, need), inv = __fdividef(1.f, scale);   // exact for powers of two
                unsigned char* head = static_cast<unsigned char*>(is_v ? t.v_cache : t.k_cache) + row0 + static_cast<size_t>(h) * t.page_size * 128;
                unsigned char* dst = head + mine * 128 + ch.a * 8;
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    if (4 * s + mine >= n) break;
                    scale_by(x[s], inv);
                    *reinterpret_cast<uint2*>(dst + 512 * s)         = quant8(x[s], 0);
                    *reinterpret_cast<uint2*>(dst + 512 * s + b_off) = quant8(x[s], 4);
                }
                if (inside && scale > old) {                                  // warp-uniform
                    const float ratio = old * inv;
                    unsigned char* was = head - inside * 128;
                    for (int r = mine; r < (paired ? min(block, 8 * half + 8) : block); r += 4) {
                        if (r >= inside && r < inside + n) continue;          // just written
                        uint4* at = reinterpret_cast<uint4*>(was + r * 128) + j;
                        const uint4 b = load_16(at);
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
                if (lane == 0 && half == 0) *scale_at = scale;
            }
        };
        run(std::false_type{}, a.hkv);
        run(std::true_type{}, 2 * a.hkv);
        cp_async_wait<0>();                                                   // (empty groups)
    }
}

// One warp takes every warps_per_row-th unit of a row: a unit is up to four heads of q, of k or of v.  Short calls split a
// row over many warps (latency is all that counts there), long ones give each row to one warp, which then computes the
// row's sines once and keeps weights and sines of the heads at hand multiplied together in registers.  Up to ROWS_SLOTS
// units are on their way into the warp's slots of shared memory at any time; every lane reads back only what it
// fetched itself, so nothing has to be synchronised.
// HALVES: the common rotation of the whole head, (i, i + 64), where every lane rotates everything it holds.
template<typename ACT, int SINK, bool HALVES>
__global__ void __launch_bounds__(ROWS_THREADS, SINK == SINK_BLOCKS ? 4 : 5)
rows_kernel(const __grid_constant__ RowArgs a, const __grid_constant__ RopeArgs rope, const __grid_constant__ PageArgs t)
{
    __shared__ __align__(16) unsigned char smem[SINK == SINK_BLOCKS ? sizeof(BlockSmem) : sizeof(RowSmem)];
    auto& table = reinterpret_cast<RowSmem*>(smem)->table;
    auto& slots = reinterpret_cast<RowSmem*>(smem)->slots;
    // A programmatic dependent of whatever is before it in the stream: its CTAs may be placed while that kernel drains, but
    // touch nothing before it has completed.  The same is offered to the kernel behind.  In a stream of calls 8192 rows take
    // 28.9 us instead of 30.8.  (Decode launches are not made this way: their CTAs have to land on the same SMs every time.)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int cta = blockIdx.x;
    if constexpr (SINK == SINK_BLOCKS) {
        // the CTAs that write blocks go first: they take longer (spread evenly over the grid they cost 15 % as its tail)
        if (cta < t.kv_ctas) { write_blocks<ACT, HALVES>(a, rope, t, *reinterpret_cast<BlockSmem*>(smem)); return; }
        cta -= t.kv_ctas;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sh = lane >> 3, j = lane & 7;
    const unsigned index = static_cast<unsigned>(cta) * ROWS_WARPS + warp;
    const int step = a.warps_per_row;
    const int row = step == 1 ? static_cast<int>(index) : static_cast<int>(index / static_cast<unsigned>(step));
    const int sub = static_cast<int>(index) - row * step;
    if (row >= a.tokens) return;
    const bool rotary = HALVES || rope.rotary_dim != 0;
    const bool interleaved = !HALVES && rope.interleaved != 0;
    const Chunks ch = HALVES ? Chunks{j, j + 8, true} : chunks_of(j, rope.rotary_dim);
    const int b_off = (ch.b - ch.a) * 8;            // elements from the lane's first chunk to its second
    // units [0, q_end) are q, [q_end, k_end) k, [k_end, units) v; the bases below are shifted so that all use the unit's number
    const int kv_units = (a.hkv + 3) >> 2;
    const int q_end = (a.hq + 3) >> 2, k_end = q_end + (SINK == SINK_BLOCKS ? 0 : kv_units);
    const int units = k_end + (SINK == SINK_FP16 || SINK == SINK_E4M3 ? kv_units : 0);
    const int mine = sh * 128 + ch.a * 8;           // this lane's first element within a unit's four heads
    const ACT* q_src = static_cast<const ACT*>(a.q) + row * a.q_stride + mine;
    const ACT* k_src = static_cast<const ACT*>(a.k) + row * a.k_stride + mine - q_end * 512;
    const ACT* v_src = static_cast<const ACT*>(a.v) + row * a.v_stride + mine - k_end * 512;
    const int q_live = a.hq - sh, k_live = a.hkv + 4 * q_end - sh, v_live = a.hkv + 4 * k_end - sh;   // a lane's head exists: 4 * unit < ..
    auto fetch = [&](int unit, int slot) {          // one commit group, empty where there is nothing left
        if (unit < units) {
            const bool is_q = unit < q_end, is_k = unit < k_end;
            if (4 * unit < (is_q ? q_live : is_k ? k_live : v_live)) {
                const ACT* p = (is_q ? q_src : is_k ? k_src : v_src) + unit * 512;
                cp_async16(&slots[warp][slot][0][lane], p);
                cp_async16(&slots[warp][slot][1][lane], p + b_off);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int u = 0; u < ROWS_SLOTS; u++) fetch(sub + u * step, u);   // on their way while the row's place is looked up

    Place p{0, 0, 0, 0, 0};
    size_t base = 0;                                // this lane's first element in the token's row of kv heads 0..3
    bool stored = true;
    if constexpr (SINK != SINK_DENSE) {
        p = locate(t, row, a.tokens, lane);
        if (p.slot < 0) {                           // no sequence's row: left as it is
            cp_async_wait<0>();
            return;
        }
        if constexpr (SINK != SINK_BLOCKS) {
            const Spot spot = spot_of(t, p, row);
            stored = spot.page >= 0;
            base = ((static_cast<size_t>(max(spot.page, 0)) * a.hkv + sh) * t.page_size + spot.off) * 128 + ch.a * 8;
        }
    }
    if (rotary) {
        const RopeTables tab = rope_tables(rope);
        for (int f = lane; f < (HALVES ? MAX_FREQS : rope.rotary_dim >> 1); f += 32)
            table[warp][f] = cos_sin(tab, rope.scale, f, rope_position(a, rope, tab, f, row, p.pos));
        __syncwarp();
    }

    int unit = sub, slot = 0;
    // The warp's units of one kind, up to `end`; `put` stores a lane's finished values.
    auto run = [&](auto is_v_, auto quantised_, const void* weight, int end, int live, int first, const float* head_scales, float inv, auto put) {
        constexpr bool is_v = decltype(is_v_)::value, quantised = decltype(quantised_)::value;
        if (unit >= end) return;
        const bool normed = !is_v && weight != nullptr;
        HeadMap map;
        if (!is_v && (normed || rotary)) map = head_map<ACT>(table[warp], rotary, ch, interleaved, weight);
#pragma unroll 1
        for (; unit < end; unit += step) {
            float factor = inv;
            // times the correctly rounded reciprocal, as the append of plain rows does: both leave the same bytes in a cache (a
            // division per value would take 13 % longer: 54.2 us for the ragged chunks above)
            if (quantised && head_scales) factor = __frcp_rn(head_scales[min(4 * (unit - first) + sh, a.hkv - 1)]);
            cp_async_wait<ROWS_SLOTS - 1>();
            Vals x = unpack<ACT>(Raw{load_shared(&slots[warp][slot][0][lane]), load_shared(&slots[warp][slot][1][lane])});
            fetch(unit + ROWS_SLOTS * step, slot);
            slot = (slot + 1) % ROWS_SLOTS;
            if (normed) factor *= inv_rms(x, a.eps);
            if (!is_v && (normed || rotary)) apply_map(x, map, rotary, ch, interleaved);
            if (quantised || normed) scale_by(x, factor);
            put(x, unit, 4 * unit < live);
        }
    };
    using std::false_type;
    using std::true_type;
    if constexpr (SINK == SINK_DENSE) {
        auto put_into = [&](ACT* dst) {
            return [=](const Vals& x, int u, bool alive) {
                if (!alive) return;
                *reinterpret_cast<uint4*>(dst + u * 512)         = pack8<ACT>(x, 0);
                *reinterpret_cast<uint4*>(dst + u * 512 + b_off) = pack8<ACT>(x, 4);
            };
        };
        run(false_type{}, false_type{}, a.q_norm, q_end, q_live, 0, nullptr, 1.f, put_into(static_cast<ACT*>(a.q_out) + row * a.q_out_stride + mine));
        run(false_type{}, false_type{}, a.k_norm, k_end, k_live, q_end, nullptr, 1.f,
            put_into(static_cast<ACT*>(a.k_out) + row * a.k_out_stride + mine - q_end * 512));
    } else {
        __half* q_dst = static_cast<__half*>(a.q_out) + row * a.q_out_stride + mine;      // fp16, what the decode reads
        run(false_type{}, false_type{}, a.q_norm, q_end, q_live, 0, nullptr, 1.f, [=](const Vals& x, int u, bool alive) {
            if (!alive) return;
            *reinterpret_cast<uint4*>(q_dst + u * 512)         = pack8<__half>(x, 0);
            *reinterpret_cast<uint4*>(q_dst + u * 512 + b_off) = pack8<__half>(x, 4);
        });
        if constexpr (SINK == SINK_FP16) {
            auto put_into = [&](void* pool, int first) {
                __half* dst = static_cast<__half*>(pool) + base;
                return [=, &t](const Vals& x, int u, bool alive) {
                    if (!alive || !stored) return;
                    __half* at = dst + static_cast<size_t>(u - first) * t.page_size * 512;
                    *reinterpret_cast<uint4*>(at)         = pack8<__half>(x, 0);
                    *reinterpret_cast<uint4*>(at + b_off) = pack8<__half>(x, 4);
                };
            };
            run(false_type{}, false_type{}, a.k_norm, k_end, k_live, q_end, nullptr, 1.f, put_into(t.k_cache, q_end));
            run(true_type{}, false_type{}, nullptr, units, v_live, k_end, nullptr, 1.f, put_into(t.v_cache, k_end));
        }
        if constexpr (SINK == SINK_E4M3) {
            auto put_into = [&](void* pool, int first) {
                unsigned char* dst = static_cast<unsigned char*>(pool) + base;
                return [=, &t](const Vals& x, int u, bool alive) {
                    if (!alive || !stored) return;
                    unsigned char* at = dst + static_cast<size_t>(u - first) * t.page_size * 512;
                    *reinterpret_cast<uint2*>(at)         = quant8(x, 0);
                    *reinterpret_cast<uint2*>(at + b_off) = quant8(x, 4);
                };
            };
            run(false_type{}, true_type{}, a.k_norm, k_end, k_live, q_end, t.k_head_scales, t.inv_k, put_into(t.k_cache, q_end));
            run(true_type{}, true_type{}, nullptr, units, v_live, k_end, t.v_head_scales, t.inv_v, put_into(t.v_cache, k_end));
        }
    }
}

}  // namespace pdk
