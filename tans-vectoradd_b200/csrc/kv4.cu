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

#include "sm100.cuh"

namespace tans_b200 {
namespace {

struct Cache {
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    const float *k_gain, *v_gain;  // [heads], null: 1
    int64_t pages;
    int32_t heads, page_log2;
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
    int32_t tokens, q_heads, dim, half;    // 2 * half elements of a head are rotated
    bool interleaved;
    int32_t *status;
};

// Sixteen elements e0 .. e0 + 15 of one head, rotated by its token's angle.
// The products and the sum round one by one.
template <typename T>
__device__ __forceinline__ void load_rotated(const T *head, int e0, const float *cs, const float *sn, int half,
                                             bool interleaved, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 8) load8(head + e0 + i, reinterpret_cast<float(&)[8]>(x[i]));
    if (e0 >= 2 * half || !cs) return;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int e = e0 + i;
        if (e < 2 * half) {
            const bool second = interleaved ? (e & 1) : e >= half;
            const int pair = interleaved ? e >> 1 : (second ? e - half : e);
            const int other = interleaved ? e ^ 1 : (second ? e - half : e + half);
            const float o = to_f32(head[other]), c = cs[pair], s = sn[pair];
            x[i] = second ? __fadd_rn(__fmul_rn(x[i], c), __fmul_rn(o, s))
                          : __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(o, s));
        }
    }
}

// Codes (8 bytes) and scale byte of sixteen values.
__device__ __forceinline__ uint2 quantize16(const float (&x)[16], uint32_t &scale) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) amax = max_nan(amax, fabsf(x[i]));
    scale = e4m3x2(amax / 6.f, 0.f);
    scale &= 0xFFu;
    const float s = e4m3_f32(scale);
    uint32_t w[2] = {0u, 0u};
    if (s != 0.f) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            uint32_t b;
            asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\t"
                "mov.b32 %0, {b, 0, 0, 0};\n\t}"
                : "=r"(b)
                : "f"(x[i + 1] / s), "f"(x[i] / s));
            w[i >> 3] |= (b & 0xFFu) << (4 * (i & 7));
        }
    }
    return make_uint2(w[0], w[1]);
}

// One thread per 16 elements: key groups, value groups, then query groups of
// a token.
template <typename T>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs p) {
    pdl_enter();
    const int groups = p.dim / 16;
    const int kv = p.cache.heads * groups, per_token = 2 * kv + (p.q ? p.q_heads * groups : 0);
    const int64_t total = (int64_t)p.tokens * per_token;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int token = (int)(i / per_token);
        int rest = (int)(i - (int64_t)token * per_token);
        const float *cs = nullptr, *sn = nullptr;
        if (p.half && !(rest >= kv && rest < 2 * kv)) {
            const int64_t pos = p.positions[token];
            if (pos < 0 || pos >= p.max_position) {
                if (p.status) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
            } else {
                cs = p.cos + pos * p.half;
                sn = p.sin + pos * p.half;
            }
        }
        float x[16];
        if (rest >= 2 * kv) {
            rest -= 2 * kv;
            const T *head = static_cast<const T *>(p.q) + token * p.q_stride + (int64_t)(rest / groups) * p.dim;
            load_rotated(head, rest % groups * 16, cs, sn, p.half, p.interleaved, x);
            T *out = static_cast<T *>(p.q_out) + ((int64_t)token * p.q_heads * groups + rest) * 16;
#pragma unroll
            for (int j = 0; j < 16; j += 8) store8(out + j, reinterpret_cast<float(&)[8]>(x[j]));
            continue;
        }
        const int64_t slot = p.slots[token];
        if (slot < 0) continue;
        if (slot >= (p.cache.pages << p.cache.page_log2)) {
            if (p.status) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
            continue;
        }
        const bool value = rest >= kv;
        if (value) rest -= kv;
        const int head = rest / groups, g = rest % groups;
        const T *src = static_cast<const T *>(value ? p.v : p.k) + token * (value ? p.v_stride : p.k_stride) +
                       (int64_t)head * p.dim;
        if (value)
            load_rotated(src, g * 16, nullptr, nullptr, 0, false, x);
        else
            load_rotated(src, g * 16, cs, sn, p.half, p.interleaved, x);
        const float *gain = value ? p.cache.v_gain : p.cache.k_gain;
        if (gain) {
            const float d = gain[head];
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = x[j] / d;
        }
        uint32_t scale;
        const uint2 codes = quantize16(x, scale);
        const int64_t at = token_at(p.cache, slot >> p.cache.page_log2, head,
                                    (int)(slot & ((1 << p.cache.page_log2) - 1))) * groups + g;
        reinterpret_cast<uint2 *>(value ? p.cache.v_codes : p.cache.k_codes)[at] = codes;
        (value ? p.cache.v_scales : p.cache.k_scales)[at] = (uint8_t)scale;
    }
}

// --------------------------------------------------------------------- read

// k, v [tokens][heads][D] from the cache's slots; a negative slot gives zeros.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const Cache c, const int64_t *slots, T *k, T *v, int32_t tokens,
                                                   int32_t dim, int32_t *status) {
    pdl_enter();
    const int groups = dim / 16, kv = c.heads * groups;
    const int64_t total = (int64_t)tokens * 2 * kv;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int token = (int)(i / (2 * kv));
        int rest = (int)(i - (int64_t)token * 2 * kv);
        const bool value = rest >= kv;
        if (value) rest -= kv;
        const int head = rest / groups, g = rest % groups;
        const int64_t slot = slots[token];
        float x[16] = {};
        if (slot >= (c.pages << c.page_log2)) {
            if (status) atomicOr(status, TANS_B200_DATA_BAD_INDEX);
        } else if (slot >= 0) {
            const int64_t at =
                token_at(c, slot >> c.page_log2, head, (int)(slot & ((1 << c.page_log2) - 1))) * groups + g;
            const uint2 u = reinterpret_cast<const uint2 *>(value ? c.v_codes : c.k_codes)[at];
            float s = e4m3_f32((value ? c.v_scales : c.k_scales)[at]);
            const float *gain = value ? c.v_gain : c.k_gain;
            if (gain) s *= gain[head];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t h2 = e2m1x2_f16(((j < 4 ? u.x : u.y) >> (8 * (j & 3))) & 0xFFu);
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h2));
                x[2 * j] = f.x * s;
                x[2 * j + 1] = f.y * s;
            }
        }
        T *out = (value ? v : k) + ((int64_t)token * kv + rest) * 16;
#pragma unroll
        for (int j = 0; j < 16; j += 8) store8(out + j, reinterpret_cast<float(&)[8]>(x[j]));
    }
}

// ---------------------------------------------------------------- attention
//
//   S = q . k / sqrt(D) over the keys a query token sees,  O = softmax(S) V,
//   lse = log(sum(exp(S)));  no visible key: O = 0, lse = -inf.
//
// The rows of one KV head are its new tokens times the query heads that share
// it (row = token * group + head in group); a CTA takes 16 of them, the M of
// one m16n8k16 MMA, and its warps take 16-key blocks of the visible range in
// turn.  Codes become MMA operands in registers, with no trip through shared
// memory:
//  * S = Q K^T: the contraction runs over D in any order, so lane (g, t) takes
//    key g of each 8-key half and the t-th quarter of its D codes, D/8
//    contiguous bytes; the k-th step uses codes 4k .. 4k+3 of that quarter, and
//    the Q fragments are loaded in the same order.
//  * O = P V: lane (g, t) takes the g-th eighth of D of keys 2t, 2t+1, 2t+8,
//    2t+9, the keys of its P fragment; merging the nibbles of two keys gives
//    bytes whose conversion is the f16 pair (key, key + 1) of one element.
// code * scale is exact in f16 and bf16, Q enters in its own type, P in f16
// relative to a running maximum; sums, maxima and O stay in f32.

constexpr int kAttnWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

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
    int32_t tokens, group, max_pages, most_new, window;
    float scale;           // softmax scale
    int32_t *status;
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}

__device__ __forceinline__ uint32_t h2_of(float lo, float hi) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&r);
}

// f16x2 whose values are exact in bf16 -> bf16x2
__device__ __forceinline__ uint32_t h2_to_bf2(uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    const __nv_bfloat162 r = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t *>(&r);
}

// e4m3 byte -> f16x2 with the value in both halves (exact)
__device__ __forceinline__ uint32_t e4m3_h2(uint32_t b) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)(b | b << 8)));
    return h2;
}

template <int BYTES>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[BYTES / 4]) {
    if constexpr (BYTES >= 16) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; i++) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p + 16 * i);
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
    } else if constexpr (BYTES == 8) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        w[0] = u.x, w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kAttnWarps * 32) attend_kernel(const AttendArgs p) {
    constexpr int kSteps = D / 16;          // MMA steps of S
    constexpr int kTiles = D / 8;           // MMA column tiles of O
    constexpr int kQ = D / 4, kE = D / 8;   // elements of a quarter and of an eighth of a head
    extern __shared__ float merge[];        // [warps][16][D] O, then [warps][16] maxima and sums
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int seq = blockIdx.z, head = blockIdx.y, row0 = blockIdx.x * 16;
    int first, news;
    if (p.starts) {
        first = p.starts[seq];
        news = p.starts[seq + 1] - first;
        if (first < 0 || news < 0 || news > p.most_new || first > p.tokens - news) {
            if (p.status && threadIdx.x == 0) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
            return;
        }
    } else {
        first = seq;
        news = 1;
    }
    const int rows = news * p.group;
    if (row0 >= rows) return;
    int len = p.lens[seq];
    const int64_t room = (int64_t)p.max_pages << p.cache.page_log2;
    if (len < 0 || len > room) {
        if (p.status && threadIdx.x == 0) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
        len = len < 0 ? 0 : (int)room;
    }
    // keys lo[i] .. hi[i] are those of this lane's two rows; lo_all .. hi_all cover the tile
    const auto last_key = [&](int row) { return len - news + row / p.group; };
    const auto first_key = [&](int last) { return p.window > 0 && last + 1 > p.window ? last + 1 - p.window : 0; };
    const int row_end = min(row0 + 16, rows) - 1;
    const int lo_all = first_key(last_key(row0)), hi_all = last_key(row_end);
    const int lo_in = first_key(last_key(row_end)), hi_in = last_key(row0);  // seen by every row
    int lo[2], hi[2];
    int64_t at_row[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int row = min(row0 + g + 8 * i, row_end);
        hi[i] = last_key(row);
        lo[i] = first_key(hi[i]);
        at_row[i] = (int64_t)(first + row / p.group) * p.q_stride + ((int64_t)head * p.group + row % p.group) * D;
    }

    // Q: step j, lane (g, t): elements 4j..4j+3 of quarter t of rows g and g + 8
    uint32_t qf[kSteps][4];
#pragma unroll
    for (int j = 0; j < kSteps; j++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.q) + at_row[i] + t * kQ + 4 * j);
            qf[j][i] = u.x;
            qf[j][2 + i] = u.y;
        }
    const float to_log2 = p.scale * kLog2e * (p.cache.k_gain ? p.cache.k_gain[head] : 1.f);

    float o[kTiles][4];
#pragma unroll
    for (int j = 0; j < kTiles; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    const int32_t *table = p.table + (int64_t)seq * p.table_stride;
    const int in_page = (1 << p.cache.page_log2) - 1;
    const auto place = [&](int key) -> int64_t {  // where a key's head lies, in token units
        int64_t page = table[key >> p.cache.page_log2];
        if (page < 0 || page >= p.cache.pages) {
            if (p.status) atomicOr(p.status, TANS_B200_DATA_BAD_INDEX);
            page = 0;
        }
        return token_at(p.cache, page, head, key & in_page);
    };

    for (int base = (lo_all & ~15) + 16 * warp; base <= hi_all; base += 16 * kAttnWarps) {
        // ---- scores of 16 keys
        float s[2][4] = {};
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int key = base + 8 * h + g;
            uint32_t w[D / 32] = {};
            uint32_t sc[(D + 63) / 64] = {};
            if (key >= lo_all && key <= hi_all) {
                const int64_t at = place(key);
                load_words<D / 8>(p.cache.k_codes + at * (D / 2) + t * (D / 8), w);
                const uint8_t *sp = p.cache.k_scales + at * (D / 16);
#pragma unroll
                for (int i = 0; i < (D + 63) / 64; i++) sc[i] = sp[t * kQ / 16 + i];
            }
#pragma unroll
            for (int j = 0; j < kSteps; j++) {
                const uint32_t two = w[j / 2] >> (16 * (j & 1));
                const uint32_t f = e4m3_h2(sc[4 * j / 16]);
                uint32_t b0 = mul_h2(e2m1x2_f16(two & 0xFFu), f), b1 = mul_h2(e2m1x2_f16((two >> 8) & 0xFFu), f);
                if constexpr (!std::is_same_v<T, __half>) {
                    b0 = h2_to_bf2(b0);
                    b1 = h2_to_bf2(b1);
                }
                mma16816<T>(s[h], qf[j], b0, b1);
            }
        }
        // ---- the running maximum and the weights
        const bool edge = base < lo_in || base + 15 > hi_in;
        float p_[2][4];
        bool grew = false;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int i = c >> 1, key = base + 8 * h + 2 * t + (c & 1);
                float v = s[h][c] * to_log2;
                if (edge && (key < lo[i] || key > hi[i])) v = -INFINITY;
                s[h][c] = v;
                grew |= v > top[i] + 8.f;
            }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float m = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
                m = fmaxf(m, top[i]);
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const float f = m == -INFINITY ? 1.f : exp2f(top[i] - m);
                top[i] = m;
                sum[i] *= f;
#pragma unroll
                for (int j = 0; j < kTiles; j++) {
                    o[j][2 * i] *= f;
                    o[j][2 * i + 1] *= f;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int i = c >> 1;
                p_[h][c] = exp2f(s[h][c] - (top[i] == -INFINITY ? 0.f : top[i]));
                sum[i] += p_[h][c];
            }
        const uint32_t pf[4] = {h2_of(p_[0][0], p_[0][1]), h2_of(p_[0][2], p_[0][3]), h2_of(p_[1][0], p_[1][1]),
                                h2_of(p_[1][2], p_[1][3])};
        // ---- values of keys 2t, 2t + 1, 2t + 8, 2t + 9
        uint32_t w[4][(D / 16 + 3) / 4] = {};
        uint32_t sc[4][(D + 127) / 128] = {};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int key = base + 2 * t + (k & 1) + 8 * (k >> 1);
            if (key >= lo_all && key <= hi_all) {
                const int64_t at = place(key);
                load_words<D / 16>(p.cache.v_codes + at * (D / 2) + g * (D / 16), w[k]);
                const uint8_t *sp = p.cache.v_scales + at * (D / 16);
#pragma unroll
                for (int i = 0; i < (D + 127) / 128; i++) sc[k][i] = sp[g * kE / 16 + i];
            }
        }
        // A NaN scale on a key that only some rows see must not reach the
        // others as 0 * NaN: its values count as 0 here and are added below.
        bool nan_key = false;
        if (edge) {
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < (D + 127) / 128; i++) nan_key |= (sc[k][i] & 0x7Fu) == 0x7Fu;
            nan_key = __any_sync(0xffffffffu, nan_key);
        }
#pragma unroll
        for (int i = 0; i < (D + 127) / 128; i++) {
            uint32_t f[2];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t lo8 = sc[2 * b][i], hi8 = sc[2 * b + 1][i];
                if (nan_key) {
                    if ((lo8 & 0x7Fu) == 0x7Fu) lo8 = 0;
                    if ((hi8 & 0x7Fu) == 0x7Fu) hi8 = 0;
                }
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f[b]) : "h"((uint16_t)(lo8 | hi8 << 8)));
            }
            constexpr int kPer = kE < 16 ? kE : 16;  // elements under one scale here
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                const int word = (i * 16 + j) / 8, sh = 4 * (j & 6);
                uint32_t b[2];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const uint32_t u = w[2 * x][word] >> sh, v = w[2 * x + 1][word] >> sh;
                    const uint32_t byte = (j & 1) ? ((u >> 4) & 0xFu) | (v & 0xF0u) : (u & 0xFu) | ((v & 0xFu) << 4);
                    b[x] = mul_h2(e2m1x2_f16(byte), f[x]);
                }
                mma16816<__half>(o[i * 16 + j], pf, b[0], b[1]);
            }
        }
        if (nan_key) {
            uint32_t seen[4];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int key = base + 8 * h + 2 * t;
                    seen[2 * h + i] = h2_of(key >= lo[i] && key <= hi[i] ? 1.f : 0.f,
                                            key + 1 >= lo[i] && key + 1 <= hi[i] ? 1.f : 0.f);
                }
#pragma unroll
            for (int i = 0; i < (D + 127) / 128; i++) {
                uint32_t b[2];
#pragma unroll
                for (int x = 0; x < 2; x++)
                    b[x] = h2_of((sc[2 * x][i] & 0x7Fu) == 0x7Fu ? 1.f : 0.f,
                                 (sc[2 * x + 1][i] & 0x7Fu) == 0x7Fu ? 1.f : 0.f);
                float n[4] = {};
                mma16816<__half>(n, seen, b[0], b[1]);
                constexpr int kPer = kE < 16 ? kE : 16;
#pragma unroll
                for (int j = 0; j < kPer; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (n[c] > 0.f) o[i * 16 + j][c] = NAN;
            }
        }
    }

    // ---- join the warps
    float *tops = merge + kAttnWarps * 16 * D, *sums = tops + kAttnWarps * 16;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        if (t == 0) {
            tops[warp * 16 + g + 8 * i] = top[i];
            sums[warp * 16 + g + 8 * i] = sum[i];
        }
    }
    // tile j, column n of the MMA is element (n * kE + j): two columns a lane
#pragma unroll
    for (int j = 0; j < kTiles; j++)
#pragma unroll
        for (int c = 0; c < 4; c++)
            merge[(warp * 16 + g + 8 * (c >> 1)) * D + (2 * t + (c & 1)) * kE + j] = o[j][c];
    __syncthreads();
    const float gain = p.cache.v_gain ? p.cache.v_gain[head] : 1.f;
    for (int r = warp; r <= row_end - row0; r += kAttnWarps) {
        float m = -INFINITY, l = 0.f, f[kAttnWarps];
#pragma unroll
        for (int w = 0; w < kAttnWarps; w++) m = fmaxf(m, tops[w * 16 + r]);
#pragma unroll
        for (int w = 0; w < kAttnWarps; w++) {
            f[w] = tops[w * 16 + r] == -INFINITY && !(sums[w * 16 + r] != sums[w * 16 + r])
                       ? 0.f
                       : exp2f(tops[w * 16 + r] - (m == -INFINITY ? 0.f : m));
            l += f[w] * sums[w * 16 + r];
        }
        const int row = row0 + r;
        const int64_t at = (int64_t)(first + row / p.group) * gridDim.y * p.group + (int64_t)head * p.group + row % p.group;
        const float inv = l == 0.f ? 0.f : gain / l;
        for (int e = lane; e < D; e += 32) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; w++)
                if (f[w] != 0.f) v += f[w] * merge[(w * 16 + r) * D + e];
            static_cast<T *>(p.out)[at * D + e] = from_f32<T>(l == 0.f ? 0.f : v * inv);
        }
        if (p.lse && lane == 0) p.lse[at] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) / kLog2e + logf(l);
    }
}

template <typename T, int D>
int launch_attend(const AttendArgs &p, int seqs, int max_rows, cudaStream_t st) {
    const int smem = (kAttnWarps * 16 * D + 2 * kAttnWarps * 16) * 4;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(attend_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return launch_failed("attend_kernel", e);
    }
    return launch_ex(attend_kernel<T, D>, dim3(ceil_div(max_rows, 16), p.cache.heads, seqs), dim3(kAttnWarps * 32), smem,
                     1, st, "attend_kernel", p);
}

int flat_grid(int64_t total) {
    const int64_t blocks = ceil_div<int64_t>(total, 256);
    return (int)(blocks < (1 << 20) ? blocks : (1 << 20));
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
    *out = Cache{c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->k_gain, c->v_gain, c->pages,
                 (int32_t)c->heads, __builtin_ctz((unsigned)c->page_size)};
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
    if (!is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(q, 16) || !is_aligned(q_out, 16) || k_stride % 8 ||
        v_stride % 8 || (q && q_stride % 8))
        return fail(TANS_B200_ERR_INVALID, "kv4_append: q, k and v must be 16-byte aligned, their strides multiples of 8");
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
    const int64_t total = tokens * (2 * (int64_t)p.cache.heads + p.q_heads) * (p.dim / 16);
    return dispatch_half(dtype, "kv4_append", [&](auto t) {
        return launch_ex(append_kernel<decltype(t)>, dim3(flat_grid(total)), dim3(256), 0, 1, (cudaStream_t)stream,
                         "append_kernel", p);
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
    const int64_t total = tokens * 2 * (int64_t)c.heads * (cache->dim / 16);
    return dispatch_float(dtype, "kv4_read", [&](auto t) {
        using T = decltype(t);
        return launch_ex(read_kernel<T>, dim3(flat_grid(total)), dim3(256), 0, 1, (cudaStream_t)stream, "read_kernel",
                         c, slots, static_cast<T *>(k), static_cast<T *>(v), (int32_t)tokens, (int32_t)cache->dim,
                         status);
    });
}

extern "C" int tans_b200_kv4_attention_workspace_bytes(const tans_b200_kv4 *cache, int64_t q_heads, int64_t max_pages,
                                                       int64_t seqs, int64_t tokens, int64_t most_new,
                                                       int64_t window, int64_t *bytes) {
    clear_error();
    if (!bytes) return fail(TANS_B200_ERR_INVALID, "kv4_attention: null pointer");
    *bytes = 0;
    return TANS_B200_OK;
}

extern "C" int tans_b200_kv4_attention(const tans_b200_kv4 *cache, const void *q, int64_t q_stride, int64_t q_heads,
                                       const int32_t *table, int64_t table_stride, int64_t max_pages,
                                       const int32_t *lens, const int32_t *starts, int64_t seqs, int64_t tokens,
                                       int64_t most_new, float scale, int64_t window, void *out, float *lse,
                                       void *workspace, int64_t workspace_bytes, int dtype, int32_t *status,
                                       void *stream) {
    clear_error();
    AttendArgs p{};
    int rc = check_cache("kv4_attention", cache, &p.cache);
    if (rc) return rc;
    if (seqs < 0 || seqs > 65535 || tokens < 0 || tokens > INT32_MAX || q_heads < 1 ||
        q_heads % p.cache.heads || q_heads > 65535 || most_new < 1 || max_pages < 0 || window < 0)
        return fail(TANS_B200_ERR_INVALID,
                    "kv4_attention: q_heads must be a multiple of the cache's heads, seqs at most 65535, most_new at "
                    "least 1, max_pages and window not negative");
    if (!starts && tokens != seqs)
        return fail(TANS_B200_ERR_INVALID, "kv4_attention: one new token a sequence without starts");
    if (tokens == 0 || seqs == 0) return TANS_B200_OK;
    if (!q || !out || !lens || (!table && max_pages) || !is_aligned(q, 16) || q_stride % 8 || !is_aligned(out, 16))
        return fail(TANS_B200_ERR_INVALID,
                    "kv4_attention: q, out (16-byte aligned, q's stride a multiple of 8), lens and table are needed");
    if ((max_pages << p.cache.page_log2) > INT32_MAX - 64 || most_new * (q_heads / p.cache.heads) > (1 << 28))
        return fail(TANS_B200_ERR_INVALID, "kv4_attention: a sequence holds at most 2^31-65 tokens");
    p.q = q;
    p.q_stride = q_stride;
    p.table = table;
    p.table_stride = table_stride;
    p.lens = lens;
    p.starts = starts;
    p.out = out;
    p.lse = lse;
    p.tokens = (int32_t)tokens;
    p.group = (int32_t)(q_heads / p.cache.heads);
    p.max_pages = (int32_t)max_pages;
    p.most_new = (int32_t)most_new;
    p.window = window > INT32_MAX ? 0 : (int32_t)window;
    p.scale = scale;
    p.status = status;
    const int max_rows = (int)(most_new * p.group);
    return dispatch_half(dtype, "kv4_attention", [&](auto t) {
        using T = decltype(t);
        cudaStream_t st = (cudaStream_t)stream;
        switch (cache->dim) {
            case 64: return launch_attend<T, 64>(p, (int)seqs, max_rows, st);
            case 128: return launch_attend<T, 128>(p, (int)seqs, max_rows, st);
            default: return launch_attend<T, 256>(p, (int)seqs, max_rows, st);
        }
    });
}
