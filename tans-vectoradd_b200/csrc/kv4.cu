// kv4.cu — keys and values in a paged 4-bit cache: append with rotation, read
// back, and attention over the cache.
//
// The cache holds a token's key (and value) of one head as D/2 bytes of e2m1
// codes, two a byte (the even element in the low half), and D/16 bytes of
// e4m3 scales, one per 16 elements: 4.5 bits an element.  Arrays, all dense:
//   codes  u8 [pages][heads][page_size][D/2]
//   scales u8 [pages][heads][page_size][D/16]
// An element is code * scale * gain, gain an optional f32 per head that brings
// a head's range to the scales'.  code * scale has at most 6 significant bits
// and lies in 2^-10 .. 2688, so it is exact in bf16 and in f16.
//
// Quantisation of 16 values x (already divided by the gain):
//   s = e4m3(max|x| / 6), at most 448;  code = e2m1(x / s), 0 where s is 0;
// both round to nearest even.  A NaN makes the block's scale NaN.
//
// Measured on one B200 (8 KV heads of 128, bf16, calls among others in a graph):
// append of 16383 tokens with 32 query heads 71 us = 5.0 TB/s with neighbours
// rotated, 83 with halves (bound by memory latency), their read 15 us = 5.7 TB/s; a
// step of 32 tokens 4.5 us for both.  Attention of 64 sequences up to 8192 tokens,
// group 4: 74 us = 4.1 TB/s; of one with 131071 tokens 46 us with pages of 64 = 3.3
// TB/s, 52 us with pages of 16.

#include "sm100.cuh"

#include <stddef.h>

namespace tans_b200 {
namespace {

struct Cache {
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    const float *k_gain, *v_gain;  // [heads], null: 1
    int64_t pages;
    int32_t heads, page_log2, dim;
};

// Index of (page, head, token in page) in units of one token's head.
__device__ __forceinline__ int64_t token_at(const Cache &c, int64_t page, int head, int at) {
    return (((page * c.heads) + head) << c.page_log2) + at;
}

// e4m3 byte -> f32 (exact; NaN kept)
__device__ __forceinline__ float e4m3_f32(uint32_t b) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)b));
    return __half2float(__ushort_as_half((unsigned short)(h2 & 0xFFFFu)));
}

// e2m1 byte (two codes) -> f16x2, low code in the low half (exact)
__device__ __forceinline__ uint32_t e2m1x2_f16(uint32_t byte) {
    uint32_t h2;
    asm("{\n\t.reg .b8 b, z1, z2, z3;\n\tmov.b32 {b, z1, z2, z3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
        : "=r"(h2)
        : "r"(byte));
    return h2;
}

// ------------------------------------------------------------------- append

struct AppendArgs {
    Cache cache;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;  // elements between tokens; heads are D apart
    void *q_out;                           // [tokens][q_heads][D]
    const int64_t *slots;                  // page * page_size + place; negative: leave the token out
    const int64_t *positions;              // rows of cos and sin
    const float *cos, *sin;                // [max_position][half]
    int64_t max_position;
    int32_t tokens, q_heads, dim, dim_log2, half;  // 2 * half elements of a head are rotated
    int32_t per;                                   // heads of a thread
    bool interleaved;
    int32_t *status;
};

// How a call's rotation lies to a thread's eight elements: none; pairs (i,
// i + half), the partners eight in a row as well (half a multiple of 8); pairs
// of neighbours (interleaved, half a multiple of 4); anything else.
enum Rotation { kNoTurn, kHalves, kNeighbours, kMixed };

// Heads whose loads are in flight together: two with a load for the partners
// (halves, 16383 tokens of 32 + 8 + 8 heads of 128: append 83 us, 94 with four),
// else four (neighbours: 71 us, 80 with two).
template <Rotation R>
constexpr int kBatch = R == kHalves || R == kMixed ? 2 : 4;

// The angles of elements e0 .. e0 + 7 of a head, kept for all heads of a
// token: a rotated element becomes x * c + partner * s, each product and the
// sum rounded (s negative for the first of a pair).
template <Rotation R>
struct Turn {
    float c[8], s[8];
    uint32_t rotated;  // bit i: element i is (all or none but for kMixed)
    int partner;       // kHalves: where the partners lie

    __device__ __forceinline__ void set(const float *cs, const float *sn, int e0, int half, bool interleaved) {
        if (e0 >= 2 * half) return;
        if constexpr (R == kNeighbours) {
            const float4 a = *reinterpret_cast<const float4 *>(cs + e0 / 2), b = *reinterpret_cast<const float4 *>(sn + e0 / 2);
            c[0] = c[1] = a.x, c[2] = c[3] = a.y, c[4] = c[5] = a.z, c[6] = c[7] = a.w;
            s[0] = -b.x, s[1] = b.x, s[2] = -b.y, s[3] = b.y, s[4] = -b.z, s[5] = b.z, s[6] = -b.w, s[7] = b.w;
            rotated = 0xFFu;
        } else if constexpr (R == kHalves) {
            const bool first = e0 < half;
            load8(cs + (first ? e0 : e0 - half), c);
            load8(sn + (first ? e0 : e0 - half), s);
            if (first) {
#pragma unroll
                for (int i = 0; i < 8; i++) s[i] = -s[i];
            }
            partner = first ? half : -half;
            rotated = 0xFFu;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int e = e0 + i;
                if (e < 2 * half) {
                    const bool second = interleaved ? (e & 1) : e >= half;
                    const int pair = interleaved ? e >> 1 : (second ? e - half : e);
                    rotated |= 1u << i;
                    c[i] = cs[pair];
                    s[i] = second ? sn[pair] : -sn[pair];
                }
            }
        }
    }
};

// A thread's eight elements of one head, and their partners.
template <typename T, Rotation R>
struct Loaded {
    Eight<T> own, other;
    __device__ __forceinline__ void load(const T *at, const Turn<R> &t) {
        own = load_eight(at);
        if constexpr (R == kHalves) other = load_eight(at + t.partner);
    }
    // at: where they lie, for kMixed
    __device__ __forceinline__ void turn(const Turn<R> &t, const T *at, int e0, int half, bool interleaved, float (&x)[8]) const {
        own.to(x);
        if constexpr (R == kNoTurn) return;
        float o[8];
        if constexpr (R == kHalves) {
            other.to(o);
        } else if constexpr (R == kNeighbours) {
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = x[i ^ 1];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                o[i] = t.rotated >> i & 1 ? to_f32(at[interleaved ? i ^ 1 : (e0 + i < half ? i + half : i - half)]) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float y = __fadd_rn(__fmul_rn(x[i], t.c[i]), __fmul_rn(o[i], t.s[i]));
            x[i] = (R == kMixed ? t.rotated >> i & 1 : t.rotated) ? y : x[i];
        }
    }
};

// Codes (4 bytes) of eight values and the scale byte of the sixteen of them
// and of the neighbouring lane (lane ^ 1, which runs along).
__device__ __forceinline__ uint32_t quantize(const float (&x)[8], uint32_t &scale) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) amax = max_nan(amax, fabsf(x[i]));
    amax = max_nan(amax, __shfl_xor_sync(3u << (threadIdx.x & 30), amax, 1));
    scale = e4m3x2(amax / 6.f, 0.f) & 0xFFu;
    const float s = e4m3_f32(scale);
    uint32_t w = 0;
    if (s != 0.f) {
        asm("{\n\t.reg .b8 a, b, c, d;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
            "mov.b32 %0, {a, b, c, d};\n\t}"
            : "=r"(w)
            : "f"(x[0] / s), "f"(x[1] / s), "f"(x[2] / s), "f"(x[3] / s), "f"(x[4] / s), "f"(x[5] / s), "f"(x[6] / s),
              "f"(x[7] / s));
    }
    return w;
}

// Heads h0 .. h1 - 1 of keys or values into the cache; src: this thread's
// elements of head 0, at: its group of head 0 in the cache, in units of 8.
template <typename T, Rotation R>
__device__ __forceinline__ void store_heads(const AppendArgs &p, const T *src, int h0, int h1, const Turn<R> &turn, int e0,
                                            const float *gain, uint8_t *codes, uint8_t *scales, int64_t at,
                                            int64_t head_step) {
    src += (int64_t)h0 << p.dim_log2;
    at += h0 * head_step;
    for (int h = h0; h < h1; h += kBatch<R>, src += kBatch<R> * p.dim, at += kBatch<R> * head_step) {
        Loaded<T, R> l[kBatch<R>];
#pragma unroll
        for (int b = 0; b < kBatch<R>; b++)
            if (h + b < h1) l[b].load(src + b * p.dim, turn);
#pragma unroll
        for (int b = 0; b < kBatch<R>; b++) {
            if (h + b >= h1) break;
            float x[8];
            l[b].turn(turn, src + b * p.dim, e0, p.half, p.interleaved, x);
            if (gain) {
                const float d = gain[h + b];
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = x[j] / d;
            }
            uint32_t scale;
            reinterpret_cast<uint32_t *>(codes)[at + b * head_step] = quantize(x, scale);
            if (!(e0 & 8)) scales[(at + b * head_step) / 2] = (uint8_t)scale;
        }
    }
}

// A thread has eight elements of one token, for p.per of its heads (keys,
// values, then queries; blockIdx.y is which), the loads of several at a time to
// keep memory busy; the angles are read once for them.  A warp's lanes lie
// side by side in a head.
template <typename T, Rotation R>
__global__ void __launch_bounds__(256, 4) append_kernel(const AppendArgs p) {
    pdl_enter();
    const int kv = p.cache.heads, heads = 2 * kv + p.q_heads, groups_log2 = p.dim_log2 - 3;
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int token = i >> groups_log2, group = i & ((1 << groups_log2) - 1), e0 = 8 * group;
    if (token >= p.tokens) return;
    const int h0 = (int)blockIdx.y * p.per, h1 = min(heads, h0 + p.per);
    Turn<R> turn;
    turn.rotated = 0;
    turn.partner = 0;
    if (R != kNoTurn && !(h0 >= kv && h1 <= 2 * kv)) {
        const int64_t pos = p.positions[token];
        if (pos < 0 || pos >= p.max_position) {
            if (p.status) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
        } else {
            turn.set(p.cos + pos * p.half, p.sin + pos * p.half, e0, p.half, p.interleaved);
        }
    }
    if (h0 < 2 * kv) {
        const int64_t slot = p.slots[token];
        if (slot >= (p.cache.pages << p.cache.page_log2)) {
            if (p.status) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
        } else if (slot >= 0) {
            const int64_t at = (token_at(p.cache, slot >> p.cache.page_log2, 0, (int)(slot & ((1 << p.cache.page_log2) - 1)))
                                << groups_log2) + group;
            const int64_t head_step = (int64_t)1 << (p.cache.page_log2 + groups_log2);
            if (h0 < kv)
                store_heads<T, R>(p, static_cast<const T *>(p.k) + token * p.k_stride + e0, h0, min(h1, kv), turn, e0,
                                  p.cache.k_gain, p.cache.k_codes, p.cache.k_scales, at, head_step);
            if (h1 > kv)
                store_heads<T, kNoTurn>(p, static_cast<const T *>(p.v) + token * p.v_stride + e0, max(h0 - kv, 0),
                                        min(h1 - kv, kv), Turn<kNoTurn>{}, e0, p.cache.v_gain, p.cache.v_codes,
                                        p.cache.v_scales, at, head_step);
        }
    }
    if (h1 > 2 * kv) {
        const int q0 = max(h0 - 2 * kv, 0), q1 = h1 - 2 * kv;
        const T *src = static_cast<const T *>(p.q) + token * p.q_stride + ((int64_t)q0 << p.dim_log2) + e0;
        T *dst = static_cast<T *>(p.q_out) + (((int64_t)token * p.q_heads + q0) << p.dim_log2) + e0;
        for (int h = q0; h < q1; h += kBatch<R>, src += kBatch<R> * p.dim, dst += kBatch<R> * p.dim) {
            Loaded<T, R> l[kBatch<R>];
#pragma unroll
            for (int b = 0; b < kBatch<R>; b++)
                if (h + b < q1) l[b].load(src + b * p.dim, turn);
#pragma unroll
            for (int b = 0; b < kBatch<R>; b++) {
                if (h + b >= q1) break;
                float x[8];
                l[b].turn(turn, src + b * p.dim, e0, p.half, p.interleaved, x);
                store8(dst + b * p.dim, x);
            }
        }
    }
}

// --------------------------------------------------------------------- read

// Heads h0 .. h1 - 1 of a token's keys or values, this thread's eight elements
// of each (codes and scales: those of head 0), four heads' loads at a time.
template <typename T>
__device__ __forceinline__ void read_heads(const uint8_t *codes, const uint8_t *scales, const float *gain, T *out, int h0,
                                           int h1, int64_t code_step, int dim, bool real) {
    constexpr int kAtATime = 4;
    codes += h0 * code_step;
    scales += h0 * (code_step / 8);
    out += (int64_t)h0 * dim;
    for (int h = h0; h < h1; h += kAtATime) {
        uint32_t w[kAtATime], e[kAtATime];
#pragma unroll
        for (int b = 0; b < kAtATime; b++) {
            w[b] = e[b] = 0;
            if (real && h + b < h1) {
                w[b] = *reinterpret_cast<const uint32_t *>(codes + b * code_step);
                e[b] = scales[b * (code_step / 8)];
            }
        }
#pragma unroll
        for (int b = 0; b < kAtATime; b++) {
            if (h + b >= h1) break;
            const float s = e4m3_f32(e[b]) * (gain ? gain[h + b] : 1.f);
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t h2 = e2m1x2_f16(w[b] >> (8 * j) & 0xFFu);
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h2));
                x[2 * j] = f.x * s;
                x[2 * j + 1] = f.y * s;
            }
            store8(out + b * dim, x);
        }
        codes += kAtATime * code_step;
        scales += kAtATime * (code_step / 8);
        out += kAtATime * dim;
    }
}

// k, v [tokens][heads][D] from the cache's slots; a negative slot gives zeros.
// A thread has eight elements of one token, for `per` of its key and value
// heads (16383 tokens of 8 x 128: 15 us, 5.7 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const Cache c, const int64_t *slots, T *k, T *v, int32_t tokens,
                                                   int32_t groups_log2, int32_t per, int32_t *status) {
    pdl_enter();
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int token = i >> groups_log2, group = i & ((1 << groups_log2) - 1);
    if (token >= tokens) return;
    int64_t slot = slots[token];
    if (slot >= (c.pages << c.page_log2)) {
        if (status) atomicOr(status, TANS_B200_DATA_BAD_INDEX);
        slot = -1;
    }
    // in units of eight elements
    const int64_t at = slot < 0 ? 0
                                : (token_at(c, slot >> c.page_log2, 0, (int)(slot & ((1 << c.page_log2) - 1))) << groups_log2) + group;
    const int64_t code_step = (int64_t)4 << (c.page_log2 + groups_log2), to = (((int64_t)token * c.heads) << groups_log2) + group;
    const int h0 = blockIdx.y * per, h1 = min(2 * c.heads, h0 + per);
    if (h0 < c.heads)
        read_heads(c.k_codes + 4 * at, c.k_scales + at / 2, c.k_gain, k + 8 * to, h0, min(h1, c.heads), code_step, c.dim,
                   slot >= 0);
    if (h1 > c.heads)
        read_heads(c.v_codes + 4 * at, c.v_scales + at / 2, c.v_gain, v + 8 * to, max(h0 - c.heads, 0), h1 - c.heads, code_step,
                   c.dim, slot >= 0);
}

// ---------------------------------------------------------------- attention
//
//   S = q . k / sqrt(D) over the keys a query token sees,  O = softmax(S) V,
//   lse = log(sum(exp(S)));  no visible key: O = 0, lse = -inf.
//
// The rows of one KV head are its new tokens times the query heads that share
// it (row = token * group + head in group); 8 or 16 of them make a tile.
// The keys of a (sequence, head, tile) are cut into units of 128, 32 for each of
// a CTA's four warps, which keep a running maximum and sum each and join at
// the end.
//
// Both products are transposed, S^T = K Q^T and O^T = V^T P^T: the codes are the
// A operand of m16n8k16 MMAs and the rows the N dimension, so few rows cost
// an N of 8 and half the MMAs, sums and exponentials that an M of 16 would
// (64 sequences up to 8192 tokens, group 4: 93 us with rows as M, 76 so).
//
// The codes and the scales of a head lie together in a page, so a unit comes by
// four bulk copies a page, asked for by the warps in turn while the unit before
// it is worked on; with pages under 16 tokens every lane copies a key.  From
// shared memory they go to MMA operands in registers:
//  * S^T: the contraction runs over D in any order, so lane (g, t) takes keys g
//    and g + 8 of 16 and the t-th quarter of their D codes, D/8 contiguous
//    bytes; step j uses codes 4j .. 4j+3 of that quarter, and the Q fragments
//    are laid out in the same order.
//  * P^T: S^T comes out with a key a lane group, P^T goes in with a row a lane
//    group: one 8 x 8 transposition across the warp per eight keys.
//  * O^T: lane (g, t) takes the g-th eighth of D of the four keys of its P^T
//    fragment; merging the nibbles of two keys gives bytes whose conversion is
//    the f16 pair (key, other key) of one element, two elements a MMA.
// code * scale is exact in f16; P enters in f16 relative to 2^-7 of a maximum that
// may lag by up to 2^8: at most 2^15, and a weight errs by at most 2^-32 of the row's
// largest where it is below f16's normal range.  Sums, maxima and O stay in f32
// (sums by an MMA over the rounded P were no faster and cost the lse its last bits).  bf16 queries become
// f16 after a power of two per row that brings their largest element to 2^14: an
// element loses bits only below 2^-28 of that.
//
// Bound: turning codes into operands.  Per 16 keys of D = 128 a warp issues about
// 300 instructions, 64 conversions and 64 multiplications by the scale among
// them; the issue slots are 62 %, the ALU pipe 50 %, memory 63 % busy, and 20
// warps an SM (95 registers, 40 KB of shared memory a CTA) hide the rest.  With
// few long sequences the two launches, the start and the join of the parts
// take about 15 us beside the keys' time.

constexpr int kAttnWarps = 4;
constexpr int kBlockKeys = 32;                  // keys a warp takes at a time
constexpr int kUnit = kBlockKeys * kAttnWarps;  // keys
constexpr int kStages = 2;                      // units in shared memory: one in work, one on its way
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLag = 8.f;       // log2 of what a score may pass the maximum in use by
constexpr float kHeadroom = 7.f;  // log2 of the weight of a score that equals it; kLag + kHeadroom is below f16's 16

struct AttendArgs {
    Cache cache;
    const void *q;       // [tokens][q_heads][D]
    int64_t q_stride;
    const int32_t *table;  // [seqs][table_stride], page of each page_size tokens
    int64_t table_stride;
    const int32_t *lens;   // tokens held, the new ones included
    const int32_t *starts; // [seqs + 1] first new token of each sequence, null: one each
    void *out;             // [tokens][q_heads][D]
    float *lse;            // [tokens][q_heads], may be null
    float *parts;          // workspace of a split launch, else null
    int32_t tokens, seqs, group, max_pages, most_new, window;
    int32_t tile_rows;     // 8 or 16
    float scale;           // softmax scale
    int32_t *status;
};

// A sequence's part in the work.  lo and hi cover the keys of all its rows.
struct Sequence {
    int first, news, len, lo, hi;
    int tiles, units;  // units of one tile; at least one, which writes the zeros of rows that see nothing
    bool refused;      // its rows of q are out of range or too many; it has none then
};

__device__ __forceinline__ Sequence sequence(const AttendArgs &p, int seq) {
    Sequence s{seq, 1, 0, 0, 0, 0, 0, false};
    bool bad = false;
    if (p.starts) {
        s.first = p.starts[seq];
        const int next = p.starts[seq + 1];
        bad = s.refused = s.first < 0 || next < s.first || next - s.first > p.most_new || next > p.tokens;
        s.news = bad ? 0 : next - s.first;
    }
    s.len = p.lens[seq];
    const int64_t room = (int64_t)p.max_pages << p.cache.page_log2;
    if (s.len < 0 || s.len > room) {
        bad = true;
        s.len = s.len < 0 ? 0 : (int)room;
    }
    if (bad && p.status) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
    s.hi = s.len - 1;
    const int last = s.len - s.news;  // the last key of the first new token
    s.lo = p.window > 0 && last + 1 > p.window ? last + 1 - p.window : 0;
    s.tiles = ceil_div(s.news * p.group, p.tile_rows);
    s.units = max(1, ceil_div(s.hi + 1 - (s.lo & ~(kUnit - 1)), kUnit));
    return s;
}

// Asynchronous copy of 4, 8 or 16 bytes; zeros in the place of what is not real (then src is not read).
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const uint8_t *src, bool real) {
    const int n = real ? BYTES : 0;
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n)
                     : "memory");
}

// Bulk copy of `bytes` (a multiple of 16, both ends aligned) into shared memory, counted on `bar`.
__device__ __forceinline__ void copy_bulk(uint32_t dst, const uint8_t *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

constexpr uint32_t kWaitLimit = 1u << 16;  // polls of a wait, 10 us each at most
// Polls of the waits for a unit's copies and for its readers.  A build with 0
// makes them run out at once, which shows that the status says so.
#ifndef TANS_B200_COPY_POLLS
#define TANS_B200_COPY_POLLS kWaitLimit
#endif

// The barriers of a CTA's copies, in shared memory: for each stage the one of its
// copies, then for each the one of its readers.
struct Copies {
    uint64_t bars[2 * kStages];
    uint32_t issued;  // units asked for
    uint32_t failed;  // a wait ran out: no more copies, no more units
};

// Waits for the phase with the given parity of the barrier `at` of the Copies at
// `copies`.  Bounded: false, `failed` and TANS_B200_DATA_TIMEOUT when it has not
// come within 0.66 s, or (looked at every 16 polls) another wait of the CTA has run
// out.  kLast: for what is in flight after that; with it a CTA's waits end
// within three such limits.
template <uint32_t kPolls = TANS_B200_COPY_POLLS, bool kLast = false>
__device__ __forceinline__ bool wait_copies(uint32_t copies, int at, uint32_t parity, int32_t *status) {
#pragma unroll 1
    for (uint32_t i = 0; i < kPolls; i++) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred P1;\n\tmbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2, 10000;\n\t"
            "selp.b32 %0, 1, 0, P1;\n\t}"
            : "=r"(done)
            : "r"(copies + 8u * at), "r"(parity)
            : "memory");
        if (done) return true;
        if (!kLast && (i & 15u) == 15u) {
            uint32_t failed;
            asm volatile("ld.volatile.shared.b32 %0, [%1];"
                         : "=r"(failed)
                         : "r"(copies + (uint32_t)offsetof(Copies, failed))
                         : "memory");
            if (failed) return false;
        }
    }
    if (!kLast)
        asm volatile("st.volatile.shared.b32 [%0], 1;" ::"r"(copies + (uint32_t)offsetof(Copies, failed)) : "memory");
    if (status) atomicOr(status, TANS_B200_DATA_TIMEOUT);
    return false;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}

__device__ __forceinline__ uint32_t h2_of(float lo, float hi) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&r);
}

// two e4m3 bytes -> f16x2 (exact)
__device__ __forceinline__ uint32_t e4m3x2_h2(uint32_t two) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)two));
    return h2;
}

// four bytes of two e2m1 codes each -> four f16x2 (exact), low code in the low half
__device__ __forceinline__ void e2m1x8_h2(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

// 2^x, relative error under 2^-22, results below the normal range flushed to 0
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// NT: 8-row columns of a tile
template <int D, int NT>
struct AttnLayout {
    static constexpr int kRows = 8 * NT;
    static constexpr int kCodes = kUnit * D / 2, kScales = kUnit * D / 16;  // bytes of a unit
    static constexpr int kStage = 2 * (kCodes + kScales);            // K codes, V codes, K scales, V scales
    static constexpr int kRing = kStages * kStage;
    static constexpr int kEighth = D / 8 + 2;                        // floats of an eighth of a row of O
    static constexpr int kRow = 8 * kEighth + 4;                     // of a row: no bank conflicts
    static constexpr int kMerge = kAttnWarps * kRows * (kRow + 2) * 4;  // the warps' O, maxima and sums
    static constexpr int kQ = NT * D * 16;                           // Q fragments
    static constexpr int kBytes = (kRing > kMerge ? kRing : kMerge) + kQ + kRows * 4;
    static constexpr int kCtas = D == 256 ? 2 : (NT == 2 ? 3 : 5);  // resident on an SM
    static constexpr int kPart = kRows * (D + 2);                    // floats of a partial result
    // place of element e in a merged row
    static __device__ int place(int e) { return e / (D / 8) * kEighth + e % (D / 8); }
};

// One piece of a tile's work, in shared memory.
struct Piece {
    Sequence q;
    int seq, head, row0;
    int k0, k1;  // keys, multiples of kUnit
    // keys that some row of the tile sees, and those that every row sees
    int lo_all, hi_all, lo_in, hi_in;
    int hi[16];  // the last key that each row sees
};

__device__ __forceinline__ int first_seen(const AttendArgs &p, int last) {
    return p.window > 0 && last + 1 > p.window ? last + 1 - p.window : 0;
}

// Fills in what follows from q, row0, k0 and k1; called by one whole warp, lane r for row r.
__device__ __forceinline__ void set_rows(const AttendArgs &p, Piece &x) {
    const int lane = threadIdx.x & 31;
    const int end = min(x.row0 + p.tile_rows, x.q.news * p.group) - 1;
    const auto last_key = [&](int row) { return x.q.len - x.q.news + row / p.group; };
    if (lane < 16) x.hi[lane] = last_key(min(x.row0 + lane, end));
    if (lane == 0) {
        x.hi_in = last_key(x.row0);
        x.hi_all = last_key(end);
        x.lo_all = first_seen(p, x.hi_in);
        x.lo_in = first_seen(p, x.hi_all);
        x.k0 = max(x.k0, x.lo_all & ~(kUnit - 1));
        x.k1 = min(x.k1, (x.hi_all & ~(kUnit - 1)) + kUnit);
    }
}

// Runs a piece (set by the caller, before a block barrier).  unit_no counts the
// CTA's units, for their parities.  Afterwards the four warps' results lie in
// `smem` as [warp][kRows][kRow] O, [warp][kRows] maxima and sums.  False if a wait
// ran out: there are no results, and no copies in flight.
template <typename T, int D, int NT>
__device__ __forceinline__ bool attend_piece(const AttendArgs &p, const Piece &x, uint8_t *smem, Copies &s_copies,
                                             uint32_t &unit_no) {
    using L = AttnLayout<D, NT>;
    constexpr int kSteps = D / 16;        // MMA steps of S
    constexpr int kTiles = D / 16;        // MMA row tiles of O
    constexpr int kE = D / 8;             // elements of an eighth of a head
    constexpr int kVS = (D + 127) / 128;  // scales of an eighth
    constexpr int kKS = D / 64;           // scales of a quarter
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int head = x.head, lo_all = x.lo_all;
    int k1 = x.k1;
    const int kend = min(x.hi_all, k1 - 1);  // the piece's last key
    uint4 *qs = reinterpret_cast<uint4 *>(smem + L::kBytes - L::kQ - L::kRows * 4);
    float *factors = reinterpret_cast<float *>(smem + L::kBytes - L::kRows * 4);

    // ---- copies of a unit: lane 4 r + a brings array a (K codes, V codes, K
    // scales, V scales) of the r-th page, or of all keys where a page holds them
    const int page_log2 = p.cache.page_log2, in_page = (1 << page_log2) - 1;
    const bool bulk = page_log2 >= 4;
    const int32_t *table = p.table + (int64_t)x.seq * p.table_stride;
    const uint64_t head_at = (uint64_t)head << page_log2;
    const uint32_t page_tokens = (uint32_t)p.cache.heads << page_log2;
    const uint32_t ring_sa = (uint32_t)__cvta_generic_to_shared(smem), copies_sa = (uint32_t)__cvta_generic_to_shared(&s_copies);
    const int run = min(kUnit, 1 << page_log2), run_at = (lane >> 2) * run;
    const bool copies = bulk && run_at < kUnit;
    // the page of this lane's run of the unit at `base`; keys outside the piece
    // stand for the nearest inside it
    const auto page_of = [&](int unit) -> uint32_t {
        return copies && unit < k1 ? (uint32_t)table[max(lo_all, min(unit + run_at, kend)) >> page_log2] : 0u;
    };
    const auto issue = [&](int unit, uint32_t page, uint32_t no) {  // the no-th unit of this CTA
        const int st = no % kStages;
        // its place was read by all four warps in unit no - 2
        if (no >= kStages &&
            !__all_sync(0xffffffffu, wait_copies(copies_sa, kStages + st, (no / kStages + 1) & 1, p.status)))
            return;
        const uint32_t bar = copies_sa + 8u * st;
        if (lane == 0) {
            s_copies.issued = no + 1;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(L::kStage) : "memory");
        }
        if (copies) {
            if (page >= (uint32_t)p.cache.pages) {
                if (p.status) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
                page = 0;
            }
            const bool codes = !(lane & 2);
            const uint32_t bytes = codes ? D / 2 : D / 16;  // of a key
            const uint8_t *src = codes ? (lane & 1 ? p.cache.v_codes : p.cache.k_codes)
                                       : (lane & 1 ? p.cache.v_scales : p.cache.k_scales);
            copy_bulk(ring_sa + st * L::kStage + (codes ? (lane & 1) * L::kCodes : 2 * L::kCodes + (lane & 1) * L::kScales) +
                          run_at * bytes,
                      src + (head_at + (uint64_t)page * page_tokens + (uint32_t)((unit + run_at) & in_page)) * bytes,
                      run * bytes, bar);
        }
    };
    // pages under 16: a lane copies one of its warp's keys, a unit ahead as well;
    // what is not a key of the piece becomes zeros
    const auto copy_key = [&](int unit, uint32_t page, uint32_t no) {
        if (unit < k1) {
            const int key = unit + kBlockKeys * warp + lane;
            const bool real = key >= lo_all && key <= kend;
            if (page >= (uint32_t)p.cache.pages) {
                if (p.status) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
                page = 0;
            }
            const uint64_t tok = head_at + (uint64_t)page * page_tokens + (uint32_t)(key & in_page);
            const uint32_t to = ring_sa + no % kStages * L::kStage + (kBlockKeys * warp + lane) * (D / 2);
            const uint32_t to_s = ring_sa + no % kStages * L::kStage + 2 * L::kCodes + (kBlockKeys * warp + lane) * (D / 16);
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                copy_async<16>(to + 16 * i, p.cache.k_codes + tok * (D / 2) + 16 * i, real);
                copy_async<16>(to + L::kCodes + 16 * i, p.cache.v_codes + tok * (D / 2) + 16 * i, real);
            }
            copy_async<D / 16>(to_s, p.cache.k_scales + tok * (D / 16), real);
            copy_async<D / 16>(to_s + L::kScales, p.cache.v_scales + tok * (D / 16), real);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const auto key_page = [&](int unit) -> uint32_t {
        const int key = unit + kBlockKeys * warp + lane;
        return unit < k1 && key >= lo_all && key <= kend ? (uint32_t)table[key >> page_log2] : 0u;
    };
    // what was written here by ordinary stores comes before the copies
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    // unit `no` is asked for by warp no % 4, whose pages for it were loaded when
    // it asked for the one before
    const uint32_t first_no = unit_no;
    uint32_t page;
    if (bulk) {
        page = page_of(x.k0 + (int)((warp - first_no) & 3u) * kUnit);
        if (x.k0 < k1 && (first_no & 3u) == (uint32_t)warp) {
            issue(x.k0, page, first_no);
            page = page_of(x.k0 + 4 * kUnit);
        }
    } else {
        copy_key(x.k0, key_page(x.k0), first_no);
        page = key_page(x.k0 + kUnit);
    }

    // ---- Q: steps 2i and 2i + 1, lane (g, t): elements 8i .. 8i + 7 of quarter t of
    // row g.  A row's factor brings its scores to base 2; it is positive: its sign
    // goes into Q, and 0 becomes a number that lifts no score above 2^-20.
    for (int n = warp; n < NT; n += kAttnWarps) {
        const float c = p.scale * kLog2e * (p.cache.k_gain ? p.cache.k_gain[head] : 1.f);
        const int end = min(x.row0 + L::kRows, x.q.news * p.group) - 1, row = min(x.row0 + 8 * n + g, end);
        const T *from = static_cast<const T *>(p.q) + (int64_t)(x.q.first + row / p.group) * p.q_stride +
                        ((int64_t)head * p.group + row % p.group) * D + t * (D / 4);
        uint4 u[kSteps / 2];
#pragma unroll
        for (int i = 0; i < kSteps / 2; i++) u[i] = *reinterpret_cast<const uint4 *>(from + 8 * i);
        float factor = fabsf(c);
        const uint32_t flip = c < 0.f ? 0x80008000u : 0u;
        if constexpr (!std::is_same_v<T, __half>) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps / 2; i++) {
                const T *e = reinterpret_cast<const T *>(&u[i]);
#pragma unroll
                for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(to_f32(e[k])));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            int k = 14 - ((int)(__float_as_uint(top) >> 23) - 127);  // top * 2^k in [2^14, 2^15)
            k = top == 0.f || top > 3.4e38f ? 0 : min(k, 100);
            const float up = __uint_as_float((uint32_t)(127 + k) << 23);
            factor *= __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
            for (int i = 0; i < kSteps / 2; i++) {
                const T *e = reinterpret_cast<const T *>(&u[i]);
                u[i] = make_uint4(h2_of(to_f32(e[0]) * up, to_f32(e[1]) * up), h2_of(to_f32(e[2]) * up, to_f32(e[3]) * up),
                                  h2_of(to_f32(e[4]) * up, to_f32(e[5]) * up), h2_of(to_f32(e[6]) * up, to_f32(e[7]) * up));
            }
        }
#pragma unroll
        for (int i = 0; i < kSteps / 2; i++)
            qs[(n * (kSteps / 2) + i) * 32 + lane] =
                make_uint4(u[i].x ^ flip, u[i].y ^ flip, u[i].z ^ flip, u[i].w ^ flip);
        if (t == 0) factors[8 * n + g] = max_nan(factor, 1e-37f);
    }
    __syncthreads();
    float2 to_log2[NT];  // of this lane's rows 8n + 2t and 8n + 2t + 1
#pragma unroll
    for (int n = 0; n < NT; n++) to_log2[n] = *reinterpret_cast<const float2 *>(factors + 8 * n + 2 * t);
    // blocks that every row sees whole
    const int inner = x.lo_in, inner_span = min(x.hi_in, kend) - (kBlockKeys - 1) - x.lo_in;

    // O^T: row tile j, elements 2j and 2j + 1 of this lane's eighth, rows 2t and 2t + 1
    float o[kTiles][NT][4];
#pragma unroll
    for (int j = 0; j < kTiles; j++)
#pragma unroll
        for (int n = 0; n < NT; n++) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.f;
    // scores up to `limit` need no new maximum; `less`, kHeadroom below the last one, is
    // subtracted; the sums are this lane's keys'
    float limit[NT][2], less[NT][2], sum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) limit[n][i] = -INFINITY, less[n][i] = sum[n][i] = 0.f;
    // Of eight keys the m-th is m ^ (m >> 1 & 1): the V reads of lanes t = 0..3
    // then fall on rows of both parities.
    const int own_key = g ^ (g >> 1 & 1);
#pragma unroll 1
    for (int unit = x.k0; unit < k1; unit += kUnit, unit_no++) {
        const int base = unit + kBlockKeys * warp, st = unit_no % kStages;
        const uint8_t *const stage = smem + st * L::kStage;
        // this warp's keys of the unit: codes and, from `scales` on, scales
        const uint8_t *const blk = stage + warp * kBlockKeys * (D / 2);
        const uint8_t *const scales = stage + 2 * L::kCodes + warp * kBlockKeys * (D / 16);
        if (bulk) {
            if (unit + kUnit < k1 && ((unit_no + 1) & 3u) == (uint32_t)warp) {
                issue(unit + kUnit, page, unit_no + 1);
                page = page_of(unit + 5 * kUnit);
            }
            // (after a wait that ran out the unit's work is done on what lies there, and is the last)
            if (!__all_sync(0xffffffffu, wait_copies(copies_sa, st, unit_no / kStages & 1, p.status))) k1 = unit;
        } else {
            copy_key(unit + kUnit, page, unit_no + 1);
            page = key_page(unit + 2 * kUnit);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
        }
        const bool edge = base < inner || base - inner > inner_span;
        // ---- scores of the keys base + 16 y .., both sixteens worked on together
        float s[2][NT][4];
#pragma unroll
        for (int y = 0; y < 2; y++) {
            uint32_t w[2][D / 32], f[2][kKS];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = 16 * y + 8 * h + own_key;
                const uint8_t *kp = blk + r * (D / 2) + t * (D / 8);
                if constexpr (D == 64) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(kp);
                    w[h][0] = v.x, w[h][1] = v.y;
                } else {
#pragma unroll
                    for (int i = 0; i < D / 128; i++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(kp + 16 * i);
                        w[h][4 * i] = v.x, w[h][4 * i + 1] = v.y, w[h][4 * i + 2] = v.z, w[h][4 * i + 3] = v.w;
                    }
                }
                const uint8_t *sp = scales + r * (D / 16) + t * kKS;
                if constexpr (kKS == 1) {
                    f[h][0] = e4m3x2_h2(*sp * 0x101u);
                } else {
#pragma unroll
                    for (int i = 0; i < kKS; i += 2) {
                        const uint32_t two = e4m3x2_h2(*reinterpret_cast<const uint16_t *>(sp + i));
                        f[h][i] = __byte_perm(two, two, 0x1010);
                        f[h][i + 1] = __byte_perm(two, two, 0x3232);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) s[y][n][0] = s[y][n][1] = s[y][n][2] = s[y][n][3] = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps / 2; i++) {
                uint32_t a[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    e2m1x8_h2(w[h][i], a[h]);
#pragma unroll
                    for (int k = 0; k < 4; k++) a[h][k] = mul_h2(a[h][k], f[h][i / 2]);
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint4 q = qs[(n * (kSteps / 2) + i) * 32 + lane];
                    mma_f16(s[y][n], make_uint4(a[0][0], a[1][0], a[0][1], a[1][1]), q.x, q.y);
                    mma_f16(s[y][n], make_uint4(a[0][2], a[1][2], a[0][3], a[1][3]), q.z, q.w);
                }
            }
        }
        // ---- the running maximum and the weights
        if (edge) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int last = x.hi[8 * n + 2 * t + i], lo = first_seen(p, last), hi = min(last, kend);
#pragma unroll
                    for (int y = 0; y < 2; y++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int key = base + 16 * y + 8 * h + own_key;
                            if (key < lo || key > hi) s[y][n][2 * h + i] = -INFINITY;
                        }
                }
        }
        float m[NT][2];
        bool grew = false;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                m[n][i] = fmaxf(s[0][n][i], s[0][n][2 + i]);
                m[n][i] = fmaxf(m[n][i], fmaxf(s[1][n][i], s[1][n][2 + i]));
                m[n][i] *= i ? to_log2[n].y : to_log2[n].x;
                grew |= m[n][i] > limit[n][i];
            }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float top = limit[n][i] == -INFINITY ? -INFINITY : less[n][i];
                    float v = fmaxf(m[n][i], top + kHeadroom);
#pragma unroll
                    for (int lanes = 4; lanes < 32; lanes *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, lanes));
                    less[n][i] = v == -INFINITY ? 0.f : v - kHeadroom;
                    // (past 2^26 the two sums round, together to as much as f16's end)
                    limit[n][i] = v + kLag - less[n][i] > kLag + kHeadroom ? v : v + kLag;
                    const float f = exp2f(top - less[n][i]);  // nothing to scale yet while top is -inf
                    sum[n][i] *= f;
#pragma unroll
                    for (int j = 0; j < kTiles; j++) {
                        o[j][n][i] *= f;
                        o[j][n][2 + i] *= f;
                    }
                }
        }
        uint32_t pt[2][NT][2];  // P^T fragments
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    s[y][n][c] = exp2_fast(__fmaf_rn(s[y][n][c], c & 1 ? to_log2[n].y : to_log2[n].x, -less[n][c & 1]));
                    sum[n][c & 1] += s[y][n][c];
                }
#pragma unroll
                for (int h = 0; h < 2; h++)
                    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;"
                        : "=r"(pt[y][n][h])
                        : "r"(h2_of(s[y][n][2 * h], s[y][n][2 * h + 1])));
            }
        // ---- values of the lane's four keys of each 16
#pragma unroll
        for (int y = 0; y < 2; y++) {
            uint32_t w[4][(D / 16 + 3) / 4], sc[4][kVS];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int r = 16 * y + 8 * (k >> 1) + ((2 * t + (k & 1)) ^ (t & 1));
                const uint8_t *vp = blk + L::kCodes + r * (D / 2);
                if constexpr (D == 64) {
                    w[k][0] = *reinterpret_cast<const uint32_t *>(vp + 4 * g);
                } else if constexpr (D == 128) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(vp + 8 * g);
                    w[k][0] = v.x, w[k][1] = v.y;
                } else {
                    const uint4 v = *reinterpret_cast<const uint4 *>(vp + 16 * g);
                    w[k][0] = v.x, w[k][1] = v.y, w[k][2] = v.z, w[k][3] = v.w;
                }
#pragma unroll
                for (int i = 0; i < kVS; i++)
                    sc[k][i] = scales[L::kScales + r * (D / 16) + g * kE / 16 + i];
            }
            // Keys outside the piece hold anything: their values count as 0.  A NaN
            // scale on a key that only some rows see must not reach the others
            // as 0 * NaN: its values count as 0 here and are added below.
            uint32_t nan_keys = 0;
            if (edge) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int key = base + 16 * y + 8 * (k >> 1) + ((2 * t + (k & 1)) ^ (t & 1));
                    const bool real = key >= lo_all && key <= kend;
#pragma unroll
                    for (int i = 0; i < kVS; i++) {
                        const bool nan = (sc[k][i] & 0x7Fu) == 0x7Fu;
                        if (nan && real) nan_keys |= 1u << (k * kVS + i);
                        if (nan || !real) sc[k][i] = 0;
                    }
                }
            }
            constexpr int kPer = kE < 16 ? kE : 16;  // elements under one scale here
#pragma unroll
            for (int i = 0; i < kVS; i++) {
                const uint32_t f[2] = {e4m3x2_h2(sc[0][i] | sc[1][i] << 8), e4m3x2_h2(sc[2][i] | sc[3][i] << 8)};
#pragma unroll
                for (int j = 0; j < kPer; j += 8) {
                    const int word = (i * 16 + j) / 8;
                    uint32_t even[2][4], odd[2][4];
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const uint32_t u = w[2 * b][word], v = w[2 * b + 1][word];
                        e2m1x8_h2((u & 0x0F0F0F0Fu) | (v << 4 & 0xF0F0F0F0u), even[b]);
                        e2m1x8_h2((u >> 4 & 0x0F0F0F0Fu) | (v & 0xF0F0F0F0u), odd[b]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint4 a = make_uint4(mul_h2(even[0][e], f[0]), mul_h2(odd[0][e], f[0]),
                                                   mul_h2(even[1][e], f[1]), mul_h2(odd[1][e], f[1]));
#pragma unroll
                        for (int n = 0; n < NT; n++) mma_f16(o[(i * 16 + j) / 2 + e][n], a, pt[y][n][0], pt[y][n][1]);
                    }
                }
            }
            if (edge && __any_sync(0xffffffffu, nan_keys)) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const int last = x.hi[8 * n + g], lo = first_seen(p, last), hi = min(last, kend);
                    uint32_t seen[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int a = base + 16 * y + 8 * h + ((2 * t) ^ (t & 1)), b = a ^ 1;
                        seen[h] = h2_of(a >= lo && a <= hi ? 1.f : 0.f, b >= lo && b <= hi ? 1.f : 0.f);
                    }
#pragma unroll
                    for (int i = 0; i < kVS; i++) {
                        uint32_t flag[2];
#pragma unroll
                        for (int k = 0; k < 2; k++)
                            flag[k] = h2_of(nan_keys >> (2 * k * kVS + i) & 1 ? 1.f : 0.f,
                                            nan_keys >> ((2 * k + 1) * kVS + i) & 1 ? 1.f : 0.f);
                        float v[4] = {};
                        mma_f16(v, make_uint4(flag[0], flag[0], flag[1], flag[1]), seen[0], seen[1]);
#pragma unroll
                        for (int j = 0; j < kPer / 2; j++)
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                if (v[c] > 0.f) o[i * 8 + j][n][c] = NAN;
                    }
                }
            }
        }
        __syncwarp();  // all lanes have read their keys before the place is filled again
        if (bulk && lane == 0)
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(copies_sa + 8u * (kStages + st)) : "memory");
    }

    // ---- the warps' results, side by side
    __syncthreads();
    if (s_copies.failed) {
        if (threadIdx.x == 0)
            for (uint32_t no = s_copies.issued - min(s_copies.issued, (uint32_t)kStages); no < s_copies.issued; no++)
                wait_copies<kWaitLimit, true>(copies_sa, no % kStages, no / kStages & 1, p.status);
        __syncthreads();
        return false;
    }
    float *merge = reinterpret_cast<float *>(smem);
    float *tops = merge + kAttnWarps * L::kRows * L::kRow, *sums = tops + kAttnWarps * L::kRows;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int row = warp * L::kRows + 8 * n + 2 * t + i;
#pragma unroll
            for (int lanes = 4; lanes < 32; lanes *= 2) sum[n][i] += __shfl_xor_sync(0xffffffffu, sum[n][i], lanes);
            if (g == 0) {
                tops[row] = limit[n][i] == -INFINITY ? -INFINITY : less[n][i];
                sums[row] = sum[n][i];
            }
#pragma unroll
            for (int j = 0; j < kTiles; j++)
                *reinterpret_cast<float2 *>(merge + row * L::kRow + g * L::kEighth + 2 * j) =
                    make_float2(o[j][n][i], o[j][n][2 + i]);
        }
    __syncthreads();
    return true;
}

// The factor that brings a part whose weights are relative to `top`, with sum `sum`,
// to the common m (0 where it is -inf); a part that saw nothing has factor 0, one
// whose scores are all NaN keeps its NaN.
__device__ __forceinline__ float part_factor(float top, float sum, float m) {
    return top == -INFINITY && sum == 0.f ? 0.f : exp2f(top - (m == -INFINITY ? 0.f : m));
}

// One row of the output from its sum l and O v, both relative to m; a lane has every 32nd element.
template <typename T, int D>
__device__ __forceinline__ void write_row(const AttendArgs &p, int head, int heads, int64_t token, int in_group, float m,
                                          float l, const float (&v)[D / 32]) {
    const int lane = threadIdx.x & 31;
    const int64_t at = (token * heads + head) * p.group + in_group;
    const float inv = l == 0.f ? 0.f : (p.cache.v_gain ? p.cache.v_gain[head] : 1.f) / l;
#pragma unroll
    for (int i = 0; i < D / 32; i++)
        static_cast<T *>(p.out)[at * D + lane + 32 * i] = from_f32<T>(l == 0.f ? 0.f : v[i] * inv);
    if (p.lse && lane == 0) p.lse[at] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) / kLog2e + logf(l);
}

// Joins the four warps' results of a piece: into the output if the piece is
// the tile's whole range, else into a part of the workspace.
template <typename T, int D, int NT>
__device__ __forceinline__ void join_warps(const AttendArgs &p, const Piece &x, const uint8_t *smem, float *part) {
    const float *merge = reinterpret_cast<const float *>(smem);
    using L = AttnLayout<D, NT>;
    const float *tops = merge + kAttnWarps * L::kRows * L::kRow, *sums = tops + kAttnWarps * L::kRows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = min(L::kRows, x.q.news * p.group - x.row0);
    for (int r = warp; r < rows; r += kAttnWarps) {
        float m = -INFINITY, l = 0.f, f[kAttnWarps], v[D / 32];
#pragma unroll
        for (int w = 0; w < kAttnWarps; w++) m = fmaxf(m, tops[w * L::kRows + r]);
#pragma unroll
        for (int w = 0; w < kAttnWarps; w++) {
            f[w] = part_factor(tops[w * L::kRows + r], sums[w * L::kRows + r], m);
            l += f[w] * sums[w * L::kRows + r];
        }
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; w++)  // (a factor that is 0 still passes on a NaN among the values)
                v[i] += f[w] * merge[(w * L::kRows + r) * L::kRow + L::place(lane + 32 * i)];
        }
        if (part) {
#pragma unroll
            for (int i = 0; i < D / 32; i++) part[r * D + lane + 32 * i] = v[i];
            if (lane == 0) {
                part[L::kRows * D + r] = m;
                part[L::kRows * (D + 1) + r] = l;
            }
        } else {
            const int row = x.row0 + r;
            write_row<T, D>(p, x.head, p.cache.heads, x.q.first + row / p.group, row % p.group, m, l, v);
        }
    }
}

// Called by all threads, before a block barrier.
__device__ __forceinline__ void init_copies(Copies &c) {
    if (threadIdx.x < 2 * kStages)
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(c.bars + threadIdx.x)),
                     "r"(threadIdx.x < kStages ? 1 : kAttnWarps));
    if (threadIdx.x == 0) c.issued = 0, c.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;");
}

// Zeros and -inf in a row of q that sees nothing.
template <typename T, int D>
__device__ __forceinline__ void clear_row(const AttendArgs &p, int64_t i) {
    const int q_heads = p.cache.heads * p.group;
    const int64_t row = i * q_heads;
    uint4 *out = reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + row * D);
    for (int j = threadIdx.x; j < q_heads * (D / 8); j += blockDim.x) out[j] = uint4{};
    for (int j = threadIdx.x; p.lse && j < q_heads; j += blockDim.x) p.lse[row + j] = -INFINITY;
}

// The rows of q that lie before the first sequence's and after the last's, by all CTAs of a launch.
template <typename T, int D>
__device__ __forceinline__ void clear_spare_rows(const AttendArgs &p, int64_t cta, int64_t ctas) {
    if (!p.starts) return;
    const int first = min(max(p.starts[0], 0), p.tokens), last = min(max(p.starts[p.seqs], first), p.tokens);
    for (int64_t i = cta; i < p.tokens - (last - first); i += ctas) clear_row<T, D>(p, i < first ? i : i - first + last);
}

// The rows of a sequence that sequence() refuses, as far as they exist, by one CTA.
template <typename T, int D>
__device__ __forceinline__ void clear_refused_rows(const AttendArgs &p, int seq) {
    const int last = min(p.starts[seq + 1], p.tokens);
    for (int i = max(p.starts[seq], 0); i < last; i++) clear_row<T, D>(p, i);
}

// One CTA a (tile, head, sequence), over all its keys.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAttnWarps * 32, AttnLayout<D, NT>::kCtas) attend_kernel(const AttendArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    pdl_enter();
    __shared__ Piece x;
    __shared__ Copies copies;
    uint32_t unit_no = 0;
    init_copies(copies);
    clear_spare_rows<T, D>(p, blockIdx.x + (int64_t)gridDim.x * (blockIdx.y + (int64_t)gridDim.y * blockIdx.z),
                           (int64_t)gridDim.x * gridDim.y * gridDim.z);
    if (p.seqs == 0) return;
    const Sequence q = sequence(p, blockIdx.z);
    if ((int)blockIdx.x * p.tile_rows >= q.news * p.group) {
        if (q.refused && blockIdx.x == 0 && blockIdx.y == 0) clear_refused_rows<T, D>(p, blockIdx.z);
        return;
    }
    if (threadIdx.x < 32) {
        if (threadIdx.x == 0) {
            x.q = q;
            x.seq = blockIdx.z, x.head = blockIdx.y, x.row0 = blockIdx.x * p.tile_rows;
            x.k0 = q.lo & ~(kUnit - 1);
            x.k1 = x.k0 + q.units * kUnit;
        }
        __syncwarp();
        set_rows(p, x);
    }
    __syncthreads();
    if (attend_piece<T, D, NT>(p, x, smem, copies, unit_no)) join_warps<T, D, NT>(p, x, smem, nullptr);
}

// Split form: the units of all tiles in a row (sequence, head, tile, unit),
// with kTileCost idle ones before each tile for what a tile costs besides its
// keys, cut into equal stretches, one a CTA, whatever the sequences' lengths.
// A CTA's first tile may have begun in an earlier one (part 0 of its
// workspace), its last may go on in the next (part 1); those are joined by
// attend_join_kernel, whose CTA c takes the tile that begins in stretch c
// and does not end there, as `head` describes it.
constexpr int kTileCost = 2;
struct SplitHead {
    int32_t pieces;  // 0: none
    int32_t seq, head, row0, rows, first;
    int32_t refused;  // the rows of some sequence of the call are refused
    int32_t pad;
};

template <int D, int NT>
__host__ __device__ constexpr int64_t split_floats() {
    return sizeof(SplitHead) / 4 + 2 * AttnLayout<D, NT>::kPart;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAttnWarps * 32, AttnLayout<D, NT>::kCtas) attend_split_kernel(const AttendArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int64_t warp_sum[kAttnWarps], found_at, at;
    __shared__ int found_seq, left, take;
    __shared__ bool begins;
    __shared__ Piece x;
    __shared__ Copies copies;
    uint32_t unit_no = 0;
    init_copies(copies);
    constexpr int kThreads = kAttnWarps * 32;
    pdl_enter();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float *mine = p.parts + blockIdx.x * split_floats<D, NT>();
    SplitHead *info = reinterpret_cast<SplitHead *>(mine);
    bool refusals = false;  // this thread's, then the call's
    const auto units_of = [&](int seq) -> int64_t {
        if (seq >= p.seqs) return 0;
        const Sequence s = sequence(p, seq);
        refusals |= s.refused;
        return (int64_t)s.tiles * (s.units + kTileCost) * p.cache.heads;
    };
    // Units of the 128 sequences from b0 on: this thread's own, those before it,
    // and all of them.
    struct Counted {
        int64_t own, before, all;
    };
    const auto count = [&](int b0) {
        Counted c{units_of(b0 + tid), 0, 0};
        int64_t inc = c.own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) warp_sum[warp] = inc;
        refusals = __syncthreads_or(refusals);
        c.before = inc - c.own;
#pragma unroll
        for (int w = 0; w < kAttnWarps; w++) {
            if (w < warp) c.before += warp_sum[w];
            c.all += warp_sum[w];
        }
        return c;
    };
    const Counted first = count(0);
    int64_t total = first.all;
    for (int b0 = kThreads; b0 < p.seqs; b0 += kThreads) {
        __syncthreads();
        total += count(b0).all;
    }
    const int64_t per = ceil_div<int64_t>(total, gridDim.x);
    const int64_t u = per * blockIdx.x;
    const int64_t u_end = u + per < total ? u + per : total;
    if (tid == 0) *info = SplitHead{0, 0, 0, 0, 0, 0, refusals, 0};
    if (u >= u_end) return;
    // the sequence in which unit u lies, and that sequence's first unit
    Counted c = first;
    for (int64_t b0 = 0, from = 0;; b0 += kThreads) {
        if (u >= from + c.before && u < from + c.before + c.own) {
            found_seq = (int)b0 + tid;
            found_at = from + c.before;
        }
        __syncthreads();
        from += c.all;
        if (u < from) break;
        c = count((int)b0 + kThreads);
    }
    if (tid == 0) {
        x.seq = found_seq;
        x.q = sequence(p, x.seq);
        at = u - found_at;  // units from the sequence's first
        left = (int)(u_end - u);
    }
    __syncthreads();
    while (true) {
        if (tid < 32) {
            if (tid == 0) {
                take = 0;
                while (left > 0) {
                    const int span = x.q.units + kTileCost;
                    if (at >= (int64_t)x.q.tiles * span * p.cache.heads) {
                        at -= (int64_t)x.q.tiles * span * p.cache.heads;
                        x.q = sequence(p, ++x.seq);
                        continue;
                    }
                    const int pair = at <= INT32_MAX ? (int)((uint32_t)at / (uint32_t)span) : (int)(at / span);
                    const int pos = (int)(at - (int64_t)pair * span);
                    const int step = min(left, span - pos);
                    at += step;
                    left -= step;
                    const int u0 = max(pos - kTileCost, 0), u1 = pos + step - kTileCost;
                    if (u1 <= 0) continue;
                    take = u1 - u0;
                    begins = u0 == 0;
                    x.head = pair / x.q.tiles;
                    x.row0 = pair % x.q.tiles * p.tile_rows;
                    x.k0 = (x.q.lo & ~(kUnit - 1)) + u0 * kUnit;
                    x.k1 = x.k0 + take * kUnit;
                    if (begins && u1 < x.q.units)
                        *info = SplitHead{1 + (int)ceil_div<int64_t>(x.q.units - u1, per), x.seq, x.head, x.row0,
                                          min(p.tile_rows, x.q.news * p.group - x.row0), x.q.first, refusals, 0};
                    break;
                }
            }
            __syncwarp();
            if (take) set_rows(p, x);
        }
        __syncthreads();
        if (take == 0) return;
        if (!attend_piece<T, D, NT>(p, x, smem, copies, unit_no)) return;
        join_warps<T, D, NT>(p, x, smem,
                         begins && take == x.q.units ? nullptr
                                                     : mine + sizeof(SplitHead) / 4 + (begins ? AttnLayout<D, NT>::kPart : 0));
        // the next piece's copies come after what was written and read here
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
}

// Joins the parts of a tile: part 1 of CTA c, then part 0 of the CTAs after
// it.  A CTA takes four rows, four warps each that take turns at the parts,
// several at a time.
constexpr int kJoinRows = 4, kJoinWarps = 4;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinRows *kJoinWarps * 32) attend_join_kernel(const AttendArgs p) {
    constexpr int kAtATime = 768 / D;  // parts of a warp in flight; twice as many left no room for the next kernel
    __shared__ float tops[kJoinRows][kJoinWarps], sums[kJoinRows][kJoinWarps], o_of[kJoinRows][kJoinWarps][D];
    pdl_enter();
    const float *at = p.parts + blockIdx.x * split_floats<D, NT>();
    const SplitHead h = *reinterpret_cast<const SplitHead *>(at);
    clear_spare_rows<T, D>(p, blockIdx.x + (int64_t)gridDim.x * blockIdx.y, (int64_t)gridDim.x * gridDim.y);
    const int slot = threadIdx.x >> 7, turn = threadIdx.x >> 5 & 3, lane = threadIdx.x & 31;
    const int r = blockIdx.y * kJoinRows + slot;
    if (h.refused && blockIdx.y == 0)
        for (int seq = blockIdx.x; seq < p.seqs; seq += gridDim.x)
            if (sequence(p, seq).refused) clear_refused_rows<T, D>(p, seq);
    if (h.pieces == 0 || (int)blockIdx.y * kJoinRows >= h.rows) return;
    const bool real = r < h.rows;
    float m = -INFINITY, l = 0.f, v[D / 32] = {};
    for (int i0 = turn; real && i0 < h.pieces; i0 += kAtATime * kJoinWarps) {
        float top[kAtATime], sum[kAtATime], o[kAtATime][D / 32];
#pragma unroll
        for (int k = 0; k < kAtATime; k++) {
            const int i = i0 + k * kJoinWarps;
            top[k] = -INFINITY, sum[k] = 0.f;
            if (i < h.pieces) {
                const float *part = at + i * split_floats<D, NT>() + sizeof(SplitHead) / 4 + (i ? 0 : AttnLayout<D, NT>::kPart);
                top[k] = part[8 * NT * D + r];
                sum[k] = part[8 * NT * (D + 1) + r];
#pragma unroll
                for (int e = 0; e < D / 32; e++) o[k][e] = part[r * D + lane + 32 * e];
            }
        }
        float n = m;
#pragma unroll
        for (int k = 0; k < kAtATime; k++) n = fmaxf(n, top[k]);
        const float old = part_factor(m, l, n);
        l *= old;
#pragma unroll
        for (int e = 0; e < D / 32; e++) v[e] *= old;
#pragma unroll
        for (int k = 0; k < kAtATime; k++) {
            const float f = part_factor(top[k], sum[k], n);
            if (top[k] == -INFINITY && sum[k] == 0.f) continue;  // nothing; what is too far below to count may be a NaN
            l += f * sum[k];
#pragma unroll
            for (int e = 0; e < D / 32; e++) v[e] += f * o[k][e];
        }
        m = n;
    }
    if (lane == 0) tops[slot][turn] = m, sums[slot][turn] = l;
#pragma unroll
    for (int e = 0; e < D / 32; e++) o_of[slot][turn][lane + 32 * e] = v[e];
    __syncthreads();
    if (turn || !real) return;
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinWarps; w++) m = fmaxf(m, tops[slot][w]);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < D / 32; e++) v[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; w++) {
        const float f = part_factor(tops[slot][w], sums[slot][w], m);
        l += f * sums[slot][w];
#pragma unroll
        for (int e = 0; e < D / 32; e++) v[e] += f * o_of[slot][w][lane + 32 * e];
    }
    const int row = h.row0 + r;
    write_row<T, D>(p, h.head, p.cache.heads, h.first + row / p.group, row % p.group, m, l, v);
}

// f(<D, NT>) for a head size and a tile's rows.
template <typename F>
auto dispatch_tile(int64_t dim, int tile_rows, F &&f) {
    const auto with = [&](auto d) {
        return tile_rows == 8 ? f(d, std::integral_constant<int, 1>{}) : f(d, std::integral_constant<int, 2>{});
    };
    if (dim == 64) return with(std::integral_constant<int, 64>{});
    if (dim == 128) return with(std::integral_constant<int, 128>{});
    return with(std::integral_constant<int, 256>{});
}

// CTAs of the split form, and floats of its workspace for each; 0 for the
// whole form: ranges of a few units, which are not worth the second launch.
struct Plan {
    int ctas, tile_rows, rows;  // rows of a sequence at most
    int64_t floats;
};
int make_plan(const Cache &c, int64_t q_heads, int64_t max_pages, int64_t seqs, int64_t most_new, int64_t window, Plan *plan) {
    int sms;
    const int rc = current_sms("kv4_attention", &sms);
    if (rc) return rc;
    plan->rows = (int)(most_new * (q_heads / c.heads));
    plan->tile_rows = plan->rows <= 8 ? 8 : 16;
    int64_t keys = max_pages << c.page_log2;
    if (window > 0 && window < keys - most_new) keys = window + most_new;
    const int64_t units = ceil_div<int64_t>(keys, kUnit) + 1;
    const int64_t all = seqs * c.heads * ceil_div(plan->rows, plan->tile_rows) * units;
    dispatch_tile(c.dim, plan->tile_rows, [&](auto d, auto nt) {
        constexpr int D = decltype(d)::value, NT = decltype(nt)::value;
        const int64_t most = AttnLayout<D, NT>::kCtas * (int64_t)sms;
        plan->ctas = units <= 5 ? 0 : (int)(all < most ? all : most);
        plan->floats = plan->ctas * split_floats<D, NT>();
        return 0;
    });
    return TANS_B200_OK;
}

template <typename T, int D, int NT>
int launch_attend(const AttendArgs &p, const Plan &plan, cudaStream_t st) {
    using L = AttnLayout<D, NT>;
    const dim3 block(kAttnWarps * 32);
    if (!plan.ctas) {
        const int rc = allow_smem<attend_kernel<T, D, NT>>("attend_kernel", L::kBytes);
        return rc ? rc
                  : launch_ex(attend_kernel<T, D, NT>, dim3(ceil_div(plan.rows, L::kRows), p.cache.heads, p.seqs ? p.seqs : 1), block,
                              L::kBytes, 1, st, "attend_kernel", p);
    }
    int rc = allow_smem<attend_split_kernel<T, D, NT>>("attend_split_kernel", L::kBytes);
    if (!rc) rc = launch_ex(attend_split_kernel<T, D, NT>, dim3(plan.ctas), block, L::kBytes, 1, st, "attend_split_kernel", p);
    const int rows = plan.rows < L::kRows ? plan.rows : L::kRows;
    return rc ? rc
              : launch_ex(attend_join_kernel<T, D, NT>, dim3(plan.ctas, ceil_div(rows, kJoinRows)),
                          dim3(kJoinRows * kJoinWarps * 32), 0, 1, st, "attend_join_kernel", p);
}

int check_cache(const char *what, const tans_b200_kv4 *c, Cache *out) {
    if (!c || !c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales)
        return fail(TANS_B200_ERR_INVALID, "%s: null cache array", what);
    if (c->pages < 1 || c->pages > INT32_MAX || c->heads < 1 || c->heads > 65535 || c->page_size < 1 || c->page_size > 65536 ||
        (c->page_size & (c->page_size - 1)))
        return fail(TANS_B200_ERR_INVALID, "%s: pages and heads must be positive, page_size a power of two up to 65536",
                    what);
    if (c->dim != 64 && c->dim != 128 && c->dim != 256)
        return fail(TANS_B200_ERR_INVALID, "%s: head size must be 64, 128 or 256", what);
    if (!is_aligned(c->k_codes, 16) || !is_aligned(c->v_codes, 16) || !is_aligned(c->k_scales, 16) ||
        !is_aligned(c->v_scales, 16))
        return fail(TANS_B200_ERR_INVALID, "%s: cache arrays must be 16-byte aligned", what);
    if (!may_hold(4, c->k_gain, c->v_gain)) return fail(TANS_B200_ERR_INVALID, "%s: gains must be 4-byte aligned", what);
    *out = Cache{c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->k_gain, c->v_gain, c->pages,
                 (int32_t)c->heads, __builtin_ctz((unsigned)c->page_size), (int32_t)c->dim};
    return TANS_B200_OK;
}

}  // namespace
}  // namespace tans_b200

using namespace tans_b200;

extern "C" int tans_b200_kv4_append(const tans_b200_kv4 *cache, const void *k, int64_t k_stride, const void *v,
                                    int64_t v_stride, const int64_t *slots, const void *q, int64_t q_stride,
                                    int64_t q_heads, void *q_out, const int64_t *positions, const float *cos,
                                    const float *sin, int64_t max_position, int64_t half, int interleaved,
                                    int64_t tokens, int dtype, int32_t *status, void *stream) {
    clear_error();
    AppendArgs p{};
    int rc = check_cache("kv4_append", cache, &p.cache);
    if (rc) return rc;
    if (tokens < 0 || tokens > INT32_MAX) return fail(TANS_B200_ERR_INVALID, "kv4_append: tokens must be 0..2^31-1");
    if (tokens == 0) return TANS_B200_OK;
    if (!k || !v || !slots || (q && (!q_out || q_heads < 1 || q_heads > 65535)))
        return fail(TANS_B200_ERR_INVALID, "kv4_append: k, v, slots, and q_out with q, are needed");
    if (q && q == q_out) return fail(TANS_B200_ERR_INVALID, "kv4_append: q_out must not be q");
    if (half < 0 || 2 * half > cache->dim || (half && (!positions || !cos || !sin || max_position < 1)))
        return fail(TANS_B200_ERR_INVALID,
                    "kv4_append: half must be 0..dim/2, with positions, cos and sin where it is not 0");
    if (!is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(q, 16) || !is_aligned(q_out, 16) || !is_aligned(cos, 16) || !is_aligned(sin, 16) || k_stride % 8 ||
        v_stride % 8 || (q && q_stride % 8))
        return fail(TANS_B200_ERR_INVALID, "kv4_append: q, k, v, cos and sin must be 16-byte aligned, the strides multiples of 8");
    if (!may_hold(8, slots, positions) || !may_hold(4, status))
        return fail(TANS_B200_ERR_INVALID, "kv4_append: an array is not aligned to its elements");
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_out = q_out;
    p.slots = slots;
    p.positions = positions;
    p.cos = cos;
    p.sin = sin;
    p.max_position = max_position;
    p.tokens = (int32_t)tokens;
    p.q_heads = q ? (int32_t)q_heads : 0;
    p.dim = (int32_t)cache->dim;
    p.half = (int32_t)half;
    p.interleaved = interleaved != 0;
    p.status = status;
    if (dtype != TANS_B200_BF16 && dtype != TANS_B200_F16)
        return fail(TANS_B200_ERR_INVALID, "kv4_append: unsupported element type %d", dtype);
    int sms;
    rc = current_sms("kv4_append", &sms);
    if (rc) return rc;
    // as many heads a thread as leave 1024 threads an SM, at most 16
    const int64_t heads = 2 * (int64_t)p.cache.heads + p.q_heads, groups = p.dim / 8;
    if (tokens * groups > INT32_MAX - 256) return fail(TANS_B200_ERR_INVALID, "kv4_append: too many tokens for one call");
    const int64_t per = tokens * groups * heads / (1024 * (int64_t)sms);
    p.per = (int32_t)(per < 1 ? 1 : (per > 16 ? 16 : per));
    p.dim_log2 = __builtin_ctz((unsigned)p.dim);
    const dim3 grid((unsigned)ceil_div<int64_t>(tokens * groups, 256), (unsigned)ceil_div<int64_t>(heads, p.per));
    if (grid.y > 65535) return fail(TANS_B200_ERR_INVALID, "kv4_append: too many heads");
    const Rotation r = p.half == 0 ? kNoTurn
                                   : (p.interleaved ? (p.half % 4 ? kMixed : kNeighbours) : (p.half % 8 ? kMixed : kHalves));
    return dispatch_half(dtype, "kv4_append", [&](auto t) {
        using T = decltype(t);
        const auto launch = [&](auto kernel) {
            return launch_ex(kernel, grid, dim3(256), 0, 1, (cudaStream_t)stream, "append_kernel", p);
        };
        switch (r) {
            case kNoTurn: return launch(append_kernel<T, kNoTurn>);
            case kHalves: return launch(append_kernel<T, kHalves>);
            case kNeighbours: return launch(append_kernel<T, kNeighbours>);
            default: return launch(append_kernel<T, kMixed>);
        }
    });
}

extern "C" int tans_b200_kv4_read(const tans_b200_kv4 *cache, const int64_t *slots, void *k, void *v, int64_t tokens,
                                  int dtype, int32_t *status, void *stream) {
    clear_error();
    Cache c;
    int rc = check_cache("kv4_read", cache, &c);
    if (rc) return rc;
    if (tokens < 0 || tokens > INT32_MAX) return fail(TANS_B200_ERR_INVALID, "kv4_read: tokens must be 0..2^31-1");
    if (tokens == 0) return TANS_B200_OK;
    if (!slots || !k || !v || !is_aligned(k, 16) || !is_aligned(v, 16))
        return fail(TANS_B200_ERR_INVALID, "kv4_read: slots, and k and v 16-byte aligned, are needed");
    if (!may_hold(8, slots) || !may_hold(4, status))
        return fail(TANS_B200_ERR_INVALID, "kv4_read: an array is not aligned to its elements");
    int sms;
    rc = current_sms("kv4_read", &sms);
    if (rc) return rc;
    const int64_t heads = 2 * (int64_t)c.heads, groups = cache->dim / 8;
    if (tokens * groups > INT32_MAX - 256) return fail(TANS_B200_ERR_INVALID, "kv4_read: too many tokens for one call");
    // as many heads a thread as leave 1024 threads an SM, at most 8
    const int64_t most = tokens * groups * heads / (1024 * (int64_t)sms);
    const int32_t per = (int32_t)(most < 1 ? 1 : (most > 8 ? 8 : most));
    const dim3 grid((unsigned)ceil_div<int64_t>(tokens * groups, 256), (unsigned)ceil_div<int64_t>(heads, per));
    if (grid.y > 65535) return fail(TANS_B200_ERR_INVALID, "kv4_read: too many heads");
    return dispatch_float(dtype, "kv4_read", [&](auto t) {
        using T = decltype(t);
        return launch_ex(read_kernel<T>, grid, dim3(256), 0, 1, (cudaStream_t)stream, "read_kernel", c, slots,
                         static_cast<T *>(k), static_cast<T *>(v), (int32_t)tokens, (int32_t)__builtin_ctz((unsigned)groups),
                         per, status);
    });
}

namespace {

// Checks what the launch form depends on.
int check_attention(const tans_b200_kv4 *cache, Cache *c, int64_t q_heads, int64_t max_pages, int64_t seqs, int64_t tokens,
                    int64_t most_new, int64_t window) {
    int rc = check_cache("kv4_attention", cache, c);
    if (rc) return rc;
    if (seqs < 0 || seqs > 65535 || tokens < 0 || tokens > INT32_MAX || q_heads < 1 || q_heads % c->heads ||
        q_heads > 65535 || most_new < 1 || max_pages < 0 || window < 0)
        return fail(TANS_B200_ERR_INVALID,
                    "kv4_attention: q_heads must be a multiple of the cache's heads, seqs at most 65535, most_new at "
                    "least 1, max_pages and window not negative");
    if (max_pages > INT32_MAX || (max_pages << c->page_log2) > INT32_MAX - 4096 ||
        most_new > INT32_MAX || most_new * (q_heads / c->heads) > (1 << 28))
        return fail(TANS_B200_ERR_INVALID, "kv4_attention: a sequence holds at most 2^31-4097 tokens");
    return TANS_B200_OK;
}

}  // namespace

extern "C" int tans_b200_kv4_attention_workspace_bytes(const tans_b200_kv4 *cache, int64_t q_heads, int64_t max_pages,
                                                       int64_t seqs, int64_t tokens, int64_t most_new,
                                                       int64_t window, int64_t *bytes) {
    clear_error();
    if (!bytes) return fail(TANS_B200_ERR_INVALID, "kv4_attention: null pointer");
    Cache c;
    Plan plan;
    int rc = check_attention(cache, &c, q_heads, max_pages, seqs, tokens, most_new, window);
    if (!rc) rc = make_plan(c, q_heads, max_pages, seqs, most_new, window, &plan);
    if (rc) return rc;
    *bytes = plan.floats * 4;
    return TANS_B200_OK;
}

extern "C" int tans_b200_kv4_attention(const tans_b200_kv4 *cache, const void *q, int64_t q_stride, int64_t q_heads,
                                       const int32_t *table, int64_t table_stride, int64_t max_pages,
                                       const int32_t *lens, const int32_t *starts, int64_t seqs, int64_t tokens,
                                       int64_t most_new, float scale, int64_t window, void *out, float *lse,
                                       void *workspace, int64_t workspace_bytes, int dtype, int32_t *status,
                                       void *stream) {
    clear_error();
    if (tokens == 0) return TANS_B200_OK;
    AttendArgs p{};
    Plan plan;
    int rc = check_attention(cache, &p.cache, q_heads, max_pages, seqs, tokens, most_new, window);
    if (rc) return rc;
    if (!starts && tokens != seqs)
        return fail(TANS_B200_ERR_INVALID, "kv4_attention: one new token a sequence without starts");
    if (!q || !out || (seqs && (!lens || (!table && max_pages))) || !is_aligned(q, 16) || q_stride % 8 || !is_aligned(out, 16))
        return fail(TANS_B200_ERR_INVALID,
                    "kv4_attention: q, out (16-byte aligned, q's stride a multiple of 8), lens and table are needed");
    if (!may_hold(4, table, lens, starts, lse, status))
        return fail(TANS_B200_ERR_INVALID, "kv4_attention: an array is not aligned to its elements");
    rc = make_plan(p.cache, q_heads, max_pages, seqs, most_new, window, &plan);
    if (rc) return rc;
    if (workspace_bytes < plan.floats * 4 || (plan.ctas && (!workspace || !is_aligned(workspace, 16))))
        return fail(TANS_B200_ERR_INVALID, "kv4_attention: the workspace is too small or not 16-byte aligned");
    p.q = q;
    p.q_stride = q_stride;
    p.table = table;
    p.table_stride = table_stride;
    p.lens = lens;
    p.starts = starts;
    p.out = out;
    p.lse = lse;
    p.parts = static_cast<float *>(workspace);
    p.tokens = (int32_t)tokens;
    p.seqs = (int32_t)seqs;
    p.group = (int32_t)(q_heads / p.cache.heads);
    p.max_pages = (int32_t)max_pages;
    p.most_new = (int32_t)most_new;
    p.tile_rows = plan.tile_rows;
    p.window = window > INT32_MAX - 1 ? 0 : (int32_t)window;
    p.scale = scale;
    p.status = status;
    return dispatch_half(dtype, "kv4_attention", [&](auto t) {
        return dispatch_tile(cache->dim, plan.tile_rows, [&](auto d, auto nt) {
            return launch_attend<decltype(t), decltype(d)::value, decltype(nt)::value>(p, plan, (cudaStream_t)stream);
        });
    });
}
