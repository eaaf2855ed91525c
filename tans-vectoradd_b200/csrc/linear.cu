// linear.cu — e4m3 x e4m3 matrix product on tcgen05 with its epilogue.
//
//   y[t][r] = act(xs[t] ws[r] sum_c x[t][c] w[r][c] + bias[r]) * mul[t][r] + residual[t][r]
//
// w is the MMA's A operand (its rows the M dimension, the lanes of tensor
// memory) and the tokens are the N dimension, so one token costs an N of 16
// and not an M of 128, and a thread of the epilogue has one row's scale and
// bias in registers.  Both operands are K-major as they lie in memory: tiles
// of 128 e4m3 columns (one 128-byte swizzle span) come by tensor-map copies,
// which fill ragged edges with zeros, into a ring of shared-memory stages.
//
// Two forms.  linear_split_kernel: a CTA owns 128 rows x up to 128 tokens,
// and a cluster of up to 8 CTAs shares their columns and adds its partial sums
// over distributed shared memory: few tokens read the weight once, bound by
// memory, with enough CTAs to keep it busy.  linear_pair_kernel: CTA pairs
// (cta_group::2) own 256 rows x 256 tokens, stay resident over the tiles and
// write one tile out of tensor memory while they multiply the next: many
// tokens, bound by the tensor cores.
//
// Measured on one B200 (calls among others in a graph): [17408 x 5120], one
// token 17.3 us = 5.2 TB/s of w; [5120 x 17408], 48 tokens with a residual
// 21.5 us; [17408 x 5120], 8192 tokens with bias, GELU and a factor 544-582 us =
// 2.5-2.7 PFLOP/s (a library e4m3 product without any epilogue: 493 us), 634-667
// us in a loop of calls, where the power limit sets the clock.

#include "sm100.cuh"

#include <cuda.h>

namespace tans_b200 {
namespace {

constexpr int kMaxStages = 8;
constexpr uint32_t kWaitLimit = 1u << 16;  // polls per wait
constexpr uint32_t kPollNs = 10000;        // suspend-time hint per poll: bound ~0.66 s
// Polls of the pair form's epilogue for a tile's sums.  A build with 0 makes every
// such wait run out at once, which shows that the status says so.
#ifndef TANS_B200_EPILOGUE_POLLS
#define TANS_B200_EPILOGUE_POLLS kWaitLimit
#endif
constexpr uint32_t kEpiloguePolls = TANS_B200_EPILOGUE_POLLS;
constexpr int kMaxSmem = 225 * 1024;       // dynamic; the barriers' few bytes are static
constexpr uint32_t kTileA = 128 * 128;     // bytes of 128 rows x 128 columns

struct LinearArgs {
    CUtensorMap wmap, xmap;  // boxes of 128 columns x 128 rows / tokens, 128-byte swizzle
    const float *x_scale, *w_scale;
    const void *bias, *mul, *residual;
    void *y;
    int64_t m, rows;
    int32_t chunks;  // of 128 columns
    int32_t bn;      // tokens of a tile
    int32_t stages, act;
    int32_t row_tiles, token_tiles, splits;
    bool vec;        // rows a multiple of 8 and mul, residual and y 16-byte aligned
    int32_t *status;
};

__device__ __forceinline__ uint32_t shared_addr(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
// Wait for the phase of `bar` with the given parity; false when the wait runs
// out or (checked every 16 polls) *failed became non-zero.  kCluster: arrivals
// of the cluster's other CTA are acquired too.
template <bool kCluster = false, uint32_t kPolls = kWaitLimit>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const volatile int32_t *failed) {
    for (uint32_t i = 0; i < kPolls; i++) {
        uint32_t done;
        if constexpr (kCluster)
            asm volatile(
                "{\n\t.reg .pred P1;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P1, [%1], %2, %3;\n\t"
                "selp.b32 %0, 1, 0, P1;\n\t}"
                : "=r"(done)
                : "r"(bar), "r"(parity), "n"(kPollNs)
                : "memory");
        else
            asm volatile(
                "{\n\t.reg .pred P1;\n\tmbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2, %3;\n\t"
                "selp.b32 %0, 1, 0, P1;\n\t}"
                : "=r"(done)
                : "r"(bar), "r"(parity), "n"(kPollNs)
                : "memory");
        if (done) return true;
        if ((i & 15u) == 15u && failed && *failed) return false;
    }
    return false;
}
// K-major, 128-byte-swizzle matrix descriptor: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void copy_box(const CUtensorMap *map, uint32_t dst, uint32_t bar, int32_t col, int32_t row) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(row), "r"(bar)
        : "memory");
}

// act of N values; SiLU is v / (1 + e^-v), and the tanh form of GELU is
// v / (1 + e^(-2 sqrt(2/pi) (v + 0.044715 v^3))) as 1 + tanh(u) = 2 / (1 + e^-2u).
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
    if (act == TANS_B200_ACT_NONE) return;
    if (act == TANS_B200_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = v[i] < 0.f ? 0.f : v[i];
        return;
    }
    // the exponent in base 2
    const bool silu = act == TANS_B200_ACT_SILU;
    constexpr float kSilu = -1.4426950408889634f, kGelu1 = -2.302208198144325f, kGelu3 = -0.1029432395800235f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        float e, r;
        const float u = v[i] * (silu ? kSilu : __fmaf_rn(kGelu3, v[i] * v[i], kGelu1));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(u));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
        v[i] *= r;
    }
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t saddr, uint32_t rank) {
    uint32_t d;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(saddr), "r"(rank));
    return d;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t tmem_columns(uint32_t n) {  // an allocation: a power of two, at least 32
    return n <= 32 ? 32u : (n <= 64 ? 64u : (n <= 128 ? 128u : (n <= 256 ? 256u : 512u)));
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[N]) {
    static_assert(N == 16, "16 columns");
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// The last step of eight rows r .. r + 7 of token t, where p.vec holds: v = act(..)
// becomes v * mul + residual, rounded once.
template <typename T>
struct Operands {
    uint4 mul, residual;  // eight values each, loaded ahead
};
template <typename T>
__device__ __forceinline__ void load_operands(const LinearArgs &p, int64_t at, Operands<T> &o) {
    if (p.vec && p.mul) o.mul = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.mul) + at);
    if (p.vec && p.residual) o.residual = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.residual) + at);
}
template <typename T>
__device__ __forceinline__ void write_eight(const LinearArgs &p, float (&v)[8], int64_t at, const Operands<T> &o) {
    const T *mu = reinterpret_cast<const T *>(&o.mul), *re = reinterpret_cast<const T *>(&o.residual);
    if (p.mul) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] *= to_f32(mu[k]);
    }
    if (p.residual) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] += to_f32(re[k]);
    }
    store8(static_cast<T *>(p.y) + at, v);
}

// The same for one row of N tokens (fewer at the end: the last stands for those
// that are not there, and is not written), where eight rows of a token have no
// common alignment: neighbouring lanes take neighbouring rows (2000 tokens of
// [5121 x 5120]: 54 us, with eight rows a lane 123; of [5120 x 5120] 52).
template <typename T, int N>
struct RowOperands {
    T mul[N], residual[N];
    static __device__ __forceinline__ void load_from(const void *from, int64_t at, int64_t rows, int32_t tokens, T (&to)[N]) {
        const T *e = static_cast<const T *>(from) + at;
#pragma unroll
        for (int k = 0; k < N; k++) {
            to[k] = *e;
            e += k + 1 < tokens ? rows : 0;
        }
    }
    __device__ __forceinline__ void load(const LinearArgs &p, int64_t at, int32_t tokens) {
        if (tokens <= 0) return;
        if (p.mul) load_from(p.mul, at, p.rows, tokens, mul);
        if (p.residual) load_from(p.residual, at, p.rows, tokens, residual);
    }
    __device__ __forceinline__ void write(const LinearArgs &p, float (&v)[N], int64_t at, int32_t tokens) const {
        if (p.mul) {
#pragma unroll
            for (int k = 0; k < N; k++) v[k] *= to_f32(mul[k]);
        }
        if (p.residual) {
#pragma unroll
            for (int k = 0; k < N; k++) v[k] += to_f32(residual[k]);
        }
        T *y = static_cast<T *>(p.y) + at;
#pragma unroll
        for (int k = 0; k < N; k++, y += p.rows)
            if (k < tokens) *y = from_f32<T>(v[k]);
    }
};

// ------------------------------------------------------------ split form
//
// Reads w at 79 % of the copy rate at one token; what is left is the pipeline's
// first and last microsecond, when memory idles.  Asking for w in L2 ahead of the
// kernel before it, more stages and walking the columns from different places
// on were no faster.
//
// Copy warp, MMA warp, and four warps that read tensor memory.  The CTAs of a
// cluster take equal stretches of the chunks; each puts its f32 sums into its
// own shared memory ([token][row]) and, after a cluster barrier, adds the
// stretches' sums of its share of the tokens in rank order.  There a thread
// has the same eight rows of every token it writes; four-row groups of every
// other 32 rows change places in shared memory, so that its two reads of four
// meet no bank twice.
constexpr int kSplitThreads = 192;

template <typename T>
__global__ void __launch_bounds__(kSplitThreads, 2) linear_split_kernel(const __grid_constant__ LinearArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], done;
    __shared__ uint32_t tmem_s;
    __shared__ int32_t failed_s, copied_s;
    volatile int32_t *failed = &failed_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t a_sa = (shared_addr(smem) + 1023u) & ~1023u;
    const uint32_t b_bytes = (uint32_t)p.bn * 128u;
    const uint32_t b_sa = a_sa + (uint32_t)p.stages * kTileA;
    const uint32_t full0 = shared_addr(full), empty0 = shared_addr(empty), done0 = shared_addr(&done);
    const uint32_t ncols = tmem_columns(p.bn);
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            mbar_init(full0 + 8u * s, 1);
            mbar_init(empty0 + 8u * s, 1);
        }
        mbar_init(done0, 1);
        asm volatile("fence.mbarrier_init.release.cluster;");
        failed_s = copied_s = 0;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(&tmem_s)),
                     "r"(ncols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = tmem_s;
    const uint32_t rank = p.splits > 1 ? cluster_rank() : 0u;
    const int32_t r0 = (int32_t)blockIdx.x / p.splits * 128, t0 = (int32_t)blockIdx.y * p.bn;
    const int32_t c0 = (int32_t)((int64_t)p.chunks * rank / p.splits);
    const int32_t n = (int32_t)((int64_t)p.chunks * (rank + 1) / p.splits) - c0;  // at least one
    pdl_enter();
    // what a thread of the last four warps will write: rows r .. r + 7 of every
    // eighth token of its CTA's share
    constexpr int32_t kTokensAtATime = 8;
    const bool writer = warp >= 2;
    const int32_t tokens = p.m - t0 < p.bn ? (int32_t)(p.m - t0) : p.bn;
    // (where p.vec does not hold: row r of every token)
    const int32_t row8 = (threadIdx.x & 15) * 8, row1 = (int32_t)threadIdx.x - 64;
    const int64_t r = r0 + (p.vec ? row8 : row1);
    const int32_t real = p.vec ? (p.rows - r < 8 ? (int32_t)(p.rows - r) : 8) : (int32_t)(r < p.rows);
    const int32_t first = tokens * (int32_t)rank / p.splits + (p.vec ? (int32_t)(threadIdx.x - 64) >> 4 : 0);
    const int32_t last = tokens * (int32_t)(rank + 1) / p.splits;
    float ws[8], bias[8], xs_next = 0.f;
    Operands<T> ops{};
    RowOperands<T, kTokensAtATime> row_ops{};
    if (writer) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            ws[k] = k < real ? p.w_scale[r + k] : 0.f;
            bias[k] = p.bias && k < real ? to_f32(static_cast<const T *>(p.bias)[r + k]) : 0.f;
        }
        if (first < last && real > 0) {
            load_operands<T>(p, (int64_t)(t0 + first) * p.rows + r, ops);
            if (!p.vec) row_ops.load(p, (int64_t)(t0 + first) * p.rows + r, last - first);
            xs_next = p.x_scale[t0 + first];
        }
    }

    if (warp == 0 && lane == 0) {  // ------------------------------ copies
        int s = 0;
        uint32_t ph = 1;  // a fresh stage counts as empty
        for (int32_t c = 0; c < n; c++) {
            if (!mbar_wait(empty0 + 8u * s, ph, failed)) {
                *failed = 1;
                break;
            }
            const uint32_t bar = full0 + 8u * s;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(kTileA + b_bytes)
                         : "memory");
            copy_box(&p.wmap, a_sa + (uint32_t)s * kTileA, bar, (c0 + c) * 128, r0);
            copy_box(&p.xmap, b_sa + (uint32_t)s * b_bytes, bar, (c0 + c) * 128, t0);
            copied_s = c + 1;
            if (++s == p.stages) s = 0, ph ^= 1u;
        }
    } else if (warp == 1 && lane == 0) {  // ----------------------- MMA
        // D f32, A and B e4m3, K-major
        const uint32_t idesc = (1u << 4) | ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int32_t c = 0; c < n; c++) {
            if (!mbar_wait(full0 + 8u * s, ph, failed)) {
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
            for (int j = 0; j < 4; j++)
                asm volatile(
                    "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                    "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(tmem),
                    "l"(smem_desc(a_sa + (uint32_t)s * kTileA + 32u * j)),
                    "l"(smem_desc(b_sa + (uint32_t)s * b_bytes + 32u * j)), "r"(idesc), "r"((uint32_t)(c > 0 || j > 0)),
                    "r"(0u));
            asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                             empty0 + 8u * s)
                         : "memory");
            if (++s == p.stages) s = 0, ph ^= 1u;
        }
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(done0)
                     : "memory");
        if (!mbar_wait(done0, 0, nullptr)) ok = false;
        if (!ok) *failed = 1;
    }
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    if (*failed && threadIdx.x == 0) {  // copies in flight land before the CTA may end
        if (p.status) atomicOr(p.status, TANS_B200_DATA_TIMEOUT);
        for (int32_t c = copied_s > p.stages ? copied_s - p.stages : 0; c < copied_s; c++)
            mbar_wait(full0 + 8u * (c % p.stages), (uint32_t)((c / p.stages) & 1), nullptr);
    }
    float *sums = reinterpret_cast<float *>(smem + (a_sa - shared_addr(smem)));
    if (writer && !*failed) {  // this CTA's sums out of tensor memory
        const int row = 32 * (warp & 3) + lane;
        for (int col = 0; col < tokens; col += 16) {
            uint32_t v[16];
            tmem_load(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)col, v);
#pragma unroll
            for (int k = 0; k < 16; k++) sums[(col + k) * 128 + (row ^ (row >> 3 & 4))] = __uint_as_float(v[k]);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncwarp();
    if (p.splits > 1)
        cluster_sync();
    else
        __syncthreads();
    if (writer && !*failed && real > 0 && !p.vec) {
        for (int32_t col = first; col < last; col += kTokensAtATime) {
            const RowOperands<T, kTokensAtATime> now = row_ops;
            const int64_t at = (int64_t)(t0 + col) * p.rows + r;
            row_ops.load(p, at + kTokensAtATime * p.rows, last - col - kTokensAtATime);
            float v[kTokensAtATime] = {}, xs[kTokensAtATime];
#pragma unroll
            for (int k = 0; k < kTokensAtATime; k++) xs[k] = p.x_scale[t0 + min(col + k, last - 1)];
#pragma unroll 2
            for (int s = 0; s < p.splits; s++) {
                const uint32_t from = cluster_addr(a_sa, s) + (uint32_t)(col * 128 + (row1 ^ (row1 >> 3 & 4))) * 4u;
                float part[kTokensAtATime];  // past the last token: what lies there, within the stages' memory
#pragma unroll
                for (int k = 0; k < kTokensAtATime; k++)
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[k]) : "r"(from + 512u * k) : "memory");
#pragma unroll
                for (int k = 0; k < kTokensAtATime; k++) v[k] += part[k];
            }
#pragma unroll
            for (int k = 0; k < kTokensAtATime; k++) v[k] = __fmaf_rn(v[k] * ws[0], xs[k], bias[0]);
            activate(v, p.act);
            now.write(p, v, at, last - col);
        }
    } else if (writer && !*failed && real > 0) {
        for (int32_t col = first; col < last; col += kTokensAtATime) {
            const Operands<T> now = ops;
            const float xs = xs_next;
            const int64_t at = (int64_t)(t0 + col) * p.rows + r;
            if (col + kTokensAtATime < last) {
                load_operands<T>(p, at + kTokensAtATime * p.rows, ops);
                xs_next = p.x_scale[t0 + col + kTokensAtATime];
            }
            float v[8] = {};
#pragma unroll
            for (int s0 = 0; s0 < 8; s0 += 4) {  // four CTAs' loads at once
                if (s0 >= p.splits) break;
                float4 part[4][2];
#pragma unroll
                for (int s = 0; s < 4; s++)
                    if (s0 + s < p.splits) {
                        const uint32_t from = cluster_addr(a_sa, s0 + s) + (uint32_t)(col * 128 + row8) * 4u;
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(part[s][h].x), "=f"(part[s][h].y), "=f"(part[s][h].z), "=f"(part[s][h].w)
                                         : "r"(from + 16u * (h ^ (row8 >> 5 & 1)))
                                         : "memory");
                    }
#pragma unroll
                for (int s = 0; s < 4; s++)
                    if (s0 + s < p.splits) {
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            v[4 * h] += part[s][h].x, v[4 * h + 1] += part[s][h].y, v[4 * h + 2] += part[s][h].z,
                                v[4 * h + 3] += part[s][h].w;
                    }
            }
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = __fmaf_rn(v[k] * ws[k], xs, bias[k]);
            activate(v, p.act);
            write_eight<T>(p, v, at, now);
        }
    }
    if (p.splits > 1) {
        __syncwarp();
        cluster_sync();  // no CTA leaves while another reads its sums
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(ncols));
    }
}

// ------------------------------------------------------------- pair form
//
// A cluster of two CTAs per tile of 256 rows x bn tokens: each copies its 128
// rows of w and its half of the tokens, all bytes counted on the first CTA's
// `full` barrier, whose MMA thread multiplies for both (M = 256) and frees the
// stage in both.  The accumulator has two places in tensor memory; eight warps
// in each CTA write its 128 rows of one tile while the next is multiplied.
// Tiles are taken in bands of eight token tiles, the row tiles in turn within
// a band, so that the tiles in work at a time share their operands in L2 (8192
// tokens: 562 us with bands of 4, 547 with 8, 540 with 16; 2048 tokens 170, 144
// and 147).  Without its epilogue the kernel takes 482 us for the 8192 tokens.
constexpr int kPairThreads = 320;
constexpr int kBand = 8;
constexpr int kWarpFloats = 16 * 32 + 128;  // an epilogue warp's shared memory: 16 tokens x 32 rows, 128 scales

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1) linear_pair_kernel(const __grid_constant__ LinearArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_s;
    __shared__ int32_t failed_s;
    __shared__ int64_t copied_s;  // stages that this CTA's copy thread has filled
    volatile int32_t *failed = &failed_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t a_sa = (shared_addr(smem) + 1023u) & ~1023u;
    const uint32_t b_bytes = (uint32_t)p.bn * 64u;  // this CTA's half of the tokens
    const uint32_t b_sa = a_sa + (uint32_t)p.stages * kTileA;
    const uint32_t full0 = shared_addr(full), empty0 = shared_addr(empty);
    const uint32_t accf0 = shared_addr(acc_full), acce0 = shared_addr(acc_empty);
    const uint32_t ncols = tmem_columns(2 * p.bn);
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            mbar_init(full0 + 8u * s, 1);
            mbar_init(empty0 + 8u * s, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(accf0 + 8u * i, 1);
            mbar_init(acce0 + 8u * i, 16);  // eight warps in each CTA
        }
        asm volatile("fence.mbarrier_init.release.cluster;");
        failed_s = 0;
    }
    cluster_sync();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(&tmem_s)),
                     "r"(ncols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = tmem_s;
    const int32_t tiles = p.row_tiles * p.token_tiles, pairs = (int32_t)gridDim.x / 2;
    const auto tile_at = [&](int32_t tile, int32_t &r0, int32_t &t0) {
        const int32_t band = tile / (p.row_tiles * kBand), in = tile - band * p.row_tiles * kBand;
        const int32_t width = min(kBand, p.token_tiles - band * kBand);
        r0 = in / width * 256;
        t0 = (band * kBand + in % width) * p.bn;
    };
    const auto give_up = [&] {  // seen by both CTAs
        *failed = 1;
        asm volatile("st.relaxed.cluster.shared::cluster.b32 [%0], 1;" ::"r"(cluster_addr(shared_addr(&failed_s), rank ^ 1u))
                     : "memory");
    };
    pdl_enter();

    if (warp == 0 && lane == 0) {  // ------------------------------ copies
        int s = 0;
        uint32_t ph = 1;
        int64_t copied = 0;
        const uint32_t lead = cluster_addr(full0, 0);
        for (int32_t tile = blockIdx.x / 2; tile < tiles && !*failed; tile += pairs) {
            int32_t r0, t0;
            tile_at(tile, r0, t0);
            r0 += 128 * (int32_t)rank;
            t0 += p.bn / 2 * (int32_t)rank;
            for (int32_t c = 0; c < p.chunks; c++) {
                if (!mbar_wait(empty0 + 8u * s, ph, failed)) {
                    give_up();
                    break;
                }
                if (rank == 0)
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full0 + 8u * s),
                                 "r"(2u * (kTileA + b_bytes))
                                 : "memory");
                const auto box = [&](const CUtensorMap *map, uint32_t dst, int32_t row) {
                    asm volatile(
                        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                        "l"(reinterpret_cast<uint64_t>(map)), "r"(c * 128), "r"(row), "r"(lead + 8u * s)
                        : "memory");
                };
                box(&p.wmap, a_sa + (uint32_t)s * kTileA, r0);
                box(&p.xmap, b_sa + (uint32_t)s * b_bytes, t0);
                copied++;
                if (++s == p.stages) s = 0, ph ^= 1u;
            }
        }
        copied_s = copied;
    } else if (warp == 1 && lane == 0 && rank == 0) {  // ---------- MMA, for both CTAs
        const uint32_t idesc = (1u << 4) | ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
        const auto commit = [&](uint32_t bar) {
            asm volatile(
                "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                "h"((uint16_t)3)
                : "memory");
        };
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        int32_t it = 0;
        for (int32_t tile = blockIdx.x / 2; tile < tiles && ok; tile += pairs, it++) {
            const uint32_t d = tmem + (uint32_t)((it & 1) * p.bn);
            if (!mbar_wait<true>(acce0 + 8u * (it & 1), ((it >> 1) & 1) ^ 1u, failed)) {
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;");
            for (int32_t c = 0; c < p.chunks; c++) {
                if (!mbar_wait<true>(full0 + 8u * s, ph, failed)) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
                for (int j = 0; j < 4; j++)
                    asm volatile(
                        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(d),
                        "l"(smem_desc(a_sa + (uint32_t)s * kTileA + 32u * j)),
                        "l"(smem_desc(b_sa + (uint32_t)s * b_bytes + 32u * j)), "r"(idesc),
                        "r"((uint32_t)(c > 0 || j > 0)), "r"(0u));
                commit(empty0 + 8u * s);
                if (++s == p.stages) s = 0, ph ^= 1u;
            }
            if (!ok) give_up();
            commit(accf0 + 8u * (it & 1));  // what was multiplied is waited for even then
        }
        if (!ok) give_up();
        if (it > 0 && !mbar_wait(accf0 + 8u * ((it - 1) & 1), ((it - 1) >> 1) & 1, nullptr)) give_up();
    } else if (warp >= 2) {  // ------------------------------------ epilogue
        // Rows one a lane out of tensor memory; 16 tokens x 32 rows at a time
        // change places in shared memory, so that four lanes write a token's 32 rows.
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        float *turned = reinterpret_cast<float *>(smem + (b_sa - shared_addr(smem)) + (uint32_t)p.stages * b_bytes) +
                        (warp - 2) * kWarpFloats;
        float *xs = turned + 512;
        int32_t it = 0;
        for (int32_t tile = blockIdx.x / 2; tile < tiles; tile += pairs, it++) {
            int32_t r0, t0;
            tile_at(tile, r0, t0);
            const int64_t r = r0 + 128 * (int32_t)rank + 32 * quarter + lane;
            const bool real = r < p.rows;
            const float ws = real ? p.w_scale[r] : 0.f;
            const float bias = real && p.bias ? to_f32(static_cast<const T *>(p.bias)[r]) : 0.f;
            const int64_t r8 = r - lane + lane % 4 * 8;
            const int32_t real8 = p.rows - r8 < 8 ? (int32_t)(p.rows - r8) : 8;
            const int32_t tokens = p.m - t0 < p.bn ? (int32_t)(p.m - t0) : p.bn;
            const int32_t begin = half * p.bn / 2, end = min(tokens, begin + p.bn / 2);
            // the factor and the residual are asked for 16 tokens ahead, the first before the sums are there
            int64_t at = p.vec ? (int64_t)(t0 + begin + lane / 4) * p.rows + r8 : (int64_t)(t0 + begin) * p.rows + r;
            Operands<T> next[2] = {};
            const auto fetch = [&](int32_t col, int64_t from) {
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (real8 > 0 && col + 8 * h + lane / 4 < end) load_operands<T>(p, from + 8 * h * p.rows, next[h]);
            };
            RowOperands<T, 16> row_next{};
            if (p.vec)
                fetch(begin, at);
            else if (real)
                row_next.load(p, at, end - begin);
            __syncwarp();
            for (int32_t i = lane; i < p.bn / 2; i += 32) xs[i] = begin + i < end ? p.x_scale[t0 + begin + i] : 0.f;
            __syncwarp();
            uint32_t ok = lane ? 1u : (uint32_t)mbar_wait<false, kEpiloguePolls>(accf0 + 8u * (it & 1), (it >> 1) & 1, failed);
            if (!__all_sync(0xffffffffu, ok)) {
                if (lane == 0) give_up();
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;");
            const uint32_t acc = tmem + (uint32_t)((it & 1) * p.bn) + ((uint32_t)(32 * quarter) << 16);
            const auto values = [&](int32_t col, float (&v)[16]) {  // this lane's row, tokens col .. col + 15
                uint32_t raw[16];
                tmem_load(acc + (uint32_t)col, raw);
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(xs + col - begin + k);
                    v[k] = __fmaf_rn(__uint_as_float(raw[k]) * ws, x.x, bias);
                    v[k + 1] = __fmaf_rn(__uint_as_float(raw[k + 1]) * ws, x.y, bias);
                    v[k + 2] = __fmaf_rn(__uint_as_float(raw[k + 2]) * ws, x.z, bias);
                    v[k + 3] = __fmaf_rn(__uint_as_float(raw[k + 3]) * ws, x.w, bias);
                }
                activate(v, p.act);
            };
            if (!p.vec) {
                for (int32_t col = begin; col < end; col += 16, at += 16 * p.rows) {
                    const RowOperands<T, 16> now = row_next;
                    if (real) row_next.load(p, at + 16 * p.rows, end - col - 16);
                    float v[16];
                    values(col, v);
                    if (real) now.write(p, v, at, end - col);
                }
            } else {
                for (int32_t col = begin; col < end; col += 16, at += 16 * p.rows) {
                    const Operands<T> now[2] = {next[0], next[1]};
                    fetch(col + 16, at + 16 * p.rows);
                    float v[16];
                    values(col, v);
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 16; k++) turned[k * 32 + lane] = v[k];
                    __syncwarp();
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float e[8];
                        load8(turned + (8 * h + lane / 4) * 32 + lane % 4 * 8, e);
                        if (real8 > 0 && col + 8 * h + lane / 4 < end) write_eight<T>(p, e, at + 8 * h * p.rows, now[h]);
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;");
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                 cluster_addr(acce0 + 8u * (it & 1), 0))
                             : "memory");
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;");
    // Every role of both CTAs has ended, and both see a wait that ran out in any of
    // them; neither CTA leaves while the other may reach its memory.
    cluster_sync();
    if (*failed) {
        if (threadIdx.x == 0) {
            if (p.status) atomicOr(p.status, TANS_B200_DATA_TIMEOUT);
            if (rank == 0) {  // copies in flight land before the pair may end
                const int64_t mine = copied_s;
                int64_t other;
                asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(other) : "r"(cluster_addr(shared_addr(&copied_s), 1))
                             : "memory");
                const int64_t most = mine > other ? mine : other;
                for (int64_t c = most > p.stages ? most - p.stages : 0; c < most; c++) {
                    const uint32_t bar = full0 + 8u * (uint32_t)(c % p.stages);
                    // a stage that one CTA alone has filled: expect its bytes only
                    if (c >= mine)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(kTileA + b_bytes)
                                     : "memory");
                    else if (c >= other)
                        asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar),
                                     "r"(kTileA + b_bytes)
                                     : "memory");
                    mbar_wait<true>(bar, (uint32_t)(c / p.stages & 1), nullptr);
                }
            }
        }
        __syncwarp();
        cluster_sync();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(ncols));
    }
}

// ------------------------------------------------------------------- host

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, resolved through the runtime (no link against the driver library).
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e =
            cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q);
        return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(f) : nullptr;
    }();
    return fn;
}

// [rows][cols] bytes, boxes of 128 columns x box_rows rows
int e4m3_map(CUtensorMap *map, const uint8_t *p, int64_t rows, int64_t cols, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(TANS_B200_ERR_CUDA, "linear: cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)cols};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(p), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TANS_B200_ERR_CUDA, "linear: tensor map encode failed (%d)", (int)r);
    return TANS_B200_OK;
}

template <typename T>
int launch_linear(const LinearArgs &p, bool pair, int sms, cudaStream_t st) {
    const int smem = 1024 + p.stages * (int)(kTileA + p.bn * (pair ? 64 : 128)) + (pair ? 8 * kWarpFloats * 4 : 0);
    int rc = pair ? allow_smem<linear_pair_kernel<T>>("linear_pair_kernel", kMaxSmem)
                  : allow_smem<linear_split_kernel<T>>("linear_split_kernel", kMaxSmem);
    if (rc) return rc;
    if (pair) {
        const int tiles = p.row_tiles * p.token_tiles, pairs = sms / 2;
        return launch_ex(linear_pair_kernel<T>, dim3(2u * (tiles < pairs ? tiles : pairs)), dim3(kPairThreads), smem, 2, st,
                         "linear_pair_kernel", p);
    }
    return launch_ex(linear_split_kernel<T>, dim3((unsigned)(p.row_tiles * p.splits), (unsigned)p.token_tiles), dim3(kSplitThreads), smem,
                     p.splits, st, "linear_split_kernel", p);
}

}  // namespace
}  // namespace tans_b200

using namespace tans_b200;

extern "C" int tans_b200_linear(const uint8_t *x, const float *x_scale, const uint8_t *w, const float *w_scale,
                                const void *bias, int act, const void *mul, const void *residual, void *y, int64_t m,
                                int64_t rows, int64_t cols, int dtype, int32_t *status, void *stream) {
    clear_error();
    if (m < 0 || m > INT32_MAX / 2 || rows < 1 || rows > INT32_MAX / 2 || cols < 16 || cols % 16 || cols > INT32_MAX / 2)
        return fail(TANS_B200_ERR_INVALID, "linear: rows must be positive and cols a positive multiple of 16");
    if (act < 0 || act > TANS_B200_ACT_GELU_TANH) return fail(TANS_B200_ERR_INVALID, "linear: unknown activation %d", act);
    if (m == 0) return TANS_B200_OK;
    if (!x || !x_scale || !w || !w_scale || !y || !is_aligned(x, 16) || !is_aligned(w, 16))
        return fail(TANS_B200_ERR_INVALID, "linear: x and w (16-byte aligned), their scales and y are needed");
    if (!may_hold(4, x_scale, w_scale, status) || !may_hold(element_bytes(dtype), bias, mul, residual, y))
        return fail(TANS_B200_ERR_INVALID, "linear: an array is not aligned to its elements");
    LinearArgs p{};
    p.x_scale = x_scale;
    p.w_scale = w_scale;
    p.bias = bias;
    p.mul = mul;
    p.residual = residual;
    p.y = y;
    p.m = m;
    p.rows = rows;
    p.chunks = (int32_t)ceil_div<int64_t>(cols, 128);
    p.act = act;
    p.vec = rows % 8 == 0 && is_aligned(mul, 16) && is_aligned(residual, 16) && is_aligned(y, 16);
    p.status = status;
    int sms;
    int rc = current_sms("linear", &sms);
    if (rc) return rc;
    // The split form while its 128 x 128 tiles fit the card one an SM; above, the
    // pair form, except where that needs a second round and the split form still
    // fits two an SM.  Both, us, at K = 5120: [5120 x 5120], 256 tokens 16.7 split,
    // 21.0 pair; [17408 x 5120], 256 tokens 33.6, 28.9; [10240 x 5120], 384 tokens
    // 31.3, 38.2; 512 tokens 54.5, 38.6.
    const int64_t split_tiles = ceil_div<int64_t>(rows, 128) * ceil_div<int64_t>(m, 128);
    const int64_t pair_tiles = ceil_div<int64_t>(rows, 256) * ceil_div<int64_t>(m, 256);
    const bool pair = m > 128 && split_tiles > sms && (pair_tiles <= sms / 2 || 100 * split_tiles > 185 * sms);
    int64_t row_tiles, token_tiles;
    if (pair) {
        p.bn = 256;
        p.splits = 1;
        p.stages = 6;
        row_tiles = ceil_div<int64_t>(rows, 256);
        token_tiles = ceil_div<int64_t>(m, 256);
    } else {
        p.bn = m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : 128));
        row_tiles = ceil_div<int64_t>(rows, 128);
        token_tiles = ceil_div<int64_t>(m, p.bn);
        // Up to 32 tokens: nearly two CTAs an SM, which keep more of w in flight
        // (clusters do not fill every group of SMs: past 1.73 an SM a second round
        // begins, 23 instead of 18 us at [5120 x 17408]).  Above, the exchange of
        // the sums weighs more: about one an SM (64 tokens of [5120 x 5120]: 3
        // splits 10.0 us, 6 12.0), but two splits wherever they fit
        // (128 tokens of [17408 x 5120]: 1 split 26.7 us, 2 23.1).
        const int64_t tiles = row_tiles * token_tiles;
        int64_t splits = (m <= 32 ? 173 : 110) * sms / (100 * tiles);
        if (m > 32 && splits < 2 && 2 * tiles * 100 <= 185 * sms) splits = 2;
        const int32_t least = m <= 32 ? 4 : 8;  // chunks of a split
        if (splits > p.chunks / least) splits = p.chunks / least;
        p.splits = (int32_t)(splits < 1 ? 1 : (splits > 8 ? 8 : splits));
        p.stages = (int32_t)((110 * 1024 - 1024) / (kTileA + p.bn * 128));
        if (p.stages > kMaxStages) p.stages = kMaxStages;
    }
    if (row_tiles * p.splits > INT32_MAX / 4 || token_tiles > 65535 || row_tiles * token_tiles > INT32_MAX / 4)
        return fail(TANS_B200_ERR_INVALID, "linear: m and rows are too large");
    p.row_tiles = (int32_t)row_tiles;
    p.token_tiles = (int32_t)token_tiles;
    rc = e4m3_map(&p.wmap, w, rows, cols, 128);
    if (!rc) rc = e4m3_map(&p.xmap, x, m, cols, pair ? p.bn / 2 : p.bn);
    if (rc) return rc;
    return dispatch_half(dtype, "linear", [&](auto t) { return launch_linear<decltype(t)>(p, pair, sms, (cudaStream_t)stream); });
}
