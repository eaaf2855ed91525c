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

#include "sm100.cuh"

#include <cuda.h>

namespace tans_b200 {
namespace {

constexpr int kMaxStages = 8;
constexpr uint32_t kWaitLimit = 1u << 16;  // polls per wait
constexpr uint32_t kPollNs = 10000;        // suspend-time hint per poll: bound ~0.66 s
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
template <bool kCluster = false>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const volatile int32_t *failed) {
    for (uint32_t i = 0; i < kWaitLimit; i++) {
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

// One output: the epilogue of an accumulator `a` of row r (scale ws, bias) and token t.
template <typename T>
__device__ __forceinline__ void write_out(const LinearArgs &p, float a, float ws, float bias, float xs, int64_t t, int64_t r) {
    float v[1] = {a * ws * xs + bias};
    activate(v, p.act);
    a = v[0];
    const int64_t at = t * p.rows + r;
    if (p.mul) a *= to_f32(static_cast<const T *>(p.mul)[at]);
    if (p.residual) a += to_f32(static_cast<const T *>(p.residual)[at]);
    static_cast<T *>(p.y)[at] = from_f32<T>(a);
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

// ------------------------------------------------------------ split form
//
// Copy warp, MMA warp, four epilogue warps.  With p.splits > 1 the CTAs of a
// cluster take equal stretches of the chunks; each puts
// its f32 sums into its own shared memory ([token][row]) and, after a cluster
// barrier, adds the stretches' sums of its share of the tokens in rank order.
constexpr int kSplitThreads = 192;

template <typename T>
__global__ void __launch_bounds__(kSplitThreads) linear_split_kernel(const __grid_constant__ LinearArgs p) {
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
    const int32_t tokens = p.m - t0 < p.bn ? (int32_t)(p.m - t0) : p.bn;
    if (warp >= 2 && !*failed) {  // this CTA's sums out of tensor memory
        const int row = 32 * (warp & 3) + lane;
        const int64_t r = r0 + row;
        const bool real = r < p.rows;
        const float ws = real ? p.w_scale[r] : 0.f;
        const float bias = real && p.bias ? to_f32(static_cast<const T *>(p.bias)[r]) : 0.f;
        float *sums = reinterpret_cast<float *>(smem + (a_sa - shared_addr(smem)));
        for (int col = 0; col < tokens; col += 16) {
            uint32_t v[16];
            tmem_load(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)col, v);
            if (p.splits > 1) {
#pragma unroll
                for (int k = 0; k < 16; k++) sums[(col + k) * 128 + row] = __uint_as_float(v[k]);
            } else if (real) {
#pragma unroll
                for (int k = 0; k < 16; k++)
                    if (col + k < tokens)
                        write_out<T>(p, __uint_as_float(v[k]), ws, bias, p.x_scale[t0 + col + k], t0 + col + k, r);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncwarp();
    if (p.splits > 1) {
        cluster_sync();
        if (!*failed) {
            const int32_t lo = tokens * (int32_t)rank / p.splits, hi = tokens * (int32_t)(rank + 1) / p.splits;
            for (int32_t i = threadIdx.x; i < (hi - lo) * 128; i += kSplitThreads) {
                const int32_t col = lo + (i >> 7), row = i & 127;
                const int64_t r = r0 + row;
                if (r >= p.rows) continue;
                float a = 0.f;
                for (int s = 0; s < p.splits; s++) {
                    float v;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];"
                                 : "=f"(v)
                                 : "r"(cluster_addr(a_sa, s) + (uint32_t)(col * 128 + row) * 4u));
                    a += v;
                }
                write_out<T>(p, a, p.w_scale[r], p.bias ? to_f32(static_cast<const T *>(p.bias)[r]) : 0.f,
                             p.x_scale[t0 + col], t0 + col, r);
            }
        }
        __syncwarp();
        cluster_sync();  // no CTA leaves while another reads its sums
    } else {
        __syncthreads();
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
// a band, so that the tiles in work at a time share their operands in L2.

// A warp's 32 rows (one a lane) of n tokens from the accumulator columns at
// `acc` on; mul, res and y point to the first token.  The operands of the next
// 16 tokens are loaded while the present ones are worked out.  kFull: n is a
// multiple of 16 and every lane's row is real.
template <typename T, bool kFull>
__device__ __forceinline__ void write_columns(const LinearArgs &p, uint32_t acc, int32_t n, float ws, float bias,
                                              const float *x_scale, const T *mul, const T *res, T *y, bool real) {
    const int lane = threadIdx.x & 31;
    T mu[16], re[16];
    float xs;
    const auto load = [&](int32_t col) {
        xs = col + (lane & 15) < n ? x_scale[col + (lane & 15)] : 0.f;
        if (mul) {
#pragma unroll
            for (int k = 0; k < 16; k++)
                if (kFull || (real && col + k < n)) mu[k] = mul[(int64_t)(col + k) * p.rows];
        }
        if (res) {
#pragma unroll
            for (int k = 0; k < 16; k++)
                if (kFull || (real && col + k < n)) re[k] = res[(int64_t)(col + k) * p.rows];
        }
    };
    load(0);
    for (int32_t col = 0; col < n; col += 16) {
        uint32_t raw[16];
        tmem_load(acc + (uint32_t)col, raw);
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; k++)
            v[k] = __fmaf_rn(__uint_as_float(raw[k]) * ws, __shfl_sync(0xffffffffu, xs, k), bias);
        T mu_now[16], re_now[16];
#pragma unroll
        for (int k = 0; k < 16; k++) mu_now[k] = mu[k], re_now[k] = re[k];
        if (col + 16 < n) load(col + 16);
        activate(v, p.act);
        if (mul) {
#pragma unroll
            for (int k = 0; k < 16; k++) v[k] *= to_f32(mu_now[k]);
        }
        if (res) {
#pragma unroll
            for (int k = 0; k < 16; k++) v[k] += to_f32(re_now[k]);
        }
#pragma unroll
        for (int k = 0; k < 16; k++)
            if (kFull || (real && col + k < n)) y[(int64_t)(col + k) * p.rows] = from_f32<T>(v[k]);
    }
}

constexpr int kPairThreads = 320;
constexpr int kBand = 8;

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1) linear_pair_kernel(const __grid_constant__ LinearArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_s;
    __shared__ int32_t failed_s;
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
        if (*failed && rank == 0)  // copies in flight land before the pair may end
            for (int64_t c = copied > p.stages ? copied - p.stages : 0; c < copied; c++)
                mbar_wait(full0 + 8u * (uint32_t)(c % p.stages), (uint32_t)(c / p.stages & 1), nullptr);
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
            if (ok) commit(accf0 + 8u * (it & 1));
        }
        if (!ok) give_up();
        if (it > 0 && !mbar_wait(accf0 + 8u * ((it - 1) & 1), ((it - 1) >> 1) & 1, nullptr)) give_up();
    } else if (warp >= 2) {  // ------------------------------------ epilogue
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        int32_t it = 0;
        for (int32_t tile = blockIdx.x / 2; tile < tiles; tile += pairs, it++) {
            int32_t r0, t0;
            tile_at(tile, r0, t0);
            const int64_t r = r0 + 128 * (int32_t)rank + 32 * quarter + lane;
            const bool real = r < p.rows;
            const float ws = real ? p.w_scale[r] : 0.f;
            const float bias = real && p.bias ? to_f32(static_cast<const T *>(p.bias)[r]) : 0.f;
            uint32_t ok = lane ? 1u : (uint32_t)mbar_wait(accf0 + 8u * (it & 1), (it >> 1) & 1, failed);
            if (!__all_sync(0xffffffffu, ok)) {
                if (lane == 0) give_up();
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;");
            const int32_t tokens = p.m - t0 < p.bn ? (int32_t)(p.m - t0) : p.bn;
            const int32_t end = min(tokens, (half + 1) * p.bn / 2);
            const int32_t begin = half * p.bn / 2;
            const uint32_t acc = tmem + (uint32_t)((it & 1) * p.bn) + ((uint32_t)(32 * quarter) << 16);
            if (begin < end) {
                const int64_t at = (int64_t)(t0 + begin) * p.rows + r;
                const T *mul = p.mul ? static_cast<const T *>(p.mul) + at : nullptr;
                const T *res = p.residual ? static_cast<const T *>(p.residual) + at : nullptr;
                T *y = static_cast<T *>(p.y) + at;
                if (r - lane + 32 <= p.rows && (end - begin) % 16 == 0)
                    write_columns<T, true>(p, acc + begin, end - begin, ws, bias, p.x_scale + t0 + begin, mul, res, y, true);
                else
                    write_columns<T, false>(p, acc + begin, end - begin, ws, bias, p.x_scale + t0 + begin, mul, res, y, real);
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
    if (*failed && threadIdx.x == 0 && p.status) atomicOr(p.status, TANS_B200_DATA_TIMEOUT);
    asm volatile("tcgen05.fence::before_thread_sync;");
    cluster_sync();  // neither CTA leaves while the other may reach its memory
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
    const int smem = 1024 + p.stages * (int)(kTileA + p.bn * (pair ? 64 : 128));
    const auto kernel = pair ? linear_pair_kernel<T> : linear_split_kernel<T>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return launch_failed("linear_kernel", e);
    if (pair) {
        const int tiles = p.row_tiles * p.token_tiles, pairs = sms / 2;
        return launch_ex(kernel, dim3(2u * (tiles < pairs ? tiles : pairs)), dim3(kPairThreads), smem, 2, st,
                         "linear_pair_kernel", p);
    }
    return launch_ex(kernel, dim3((unsigned)(p.row_tiles * p.splits), (unsigned)p.token_tiles), dim3(kSplitThreads), smem,
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
    p.status = status;
    int dev, sms;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return launch_failed("linear", e);
    const int64_t pair_tiles = ceil_div<int64_t>(rows, 256) * ceil_div<int64_t>(m, 256);
    const bool pair = m > 128 && pair_tiles >= sms / 3;
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
        // two CTAs an SM, each with at least four chunks of columns
        int64_t splits = 2 * sms / (row_tiles * token_tiles);
        if (splits > p.chunks / 4) splits = p.chunks / 4;
        p.splits = (int32_t)(splits < 1 ? 1 : (splits > 8 ? 8 : splits));
        p.stages = (int32_t)((110 * 1024 - 1024) / (kTileA + p.bn * 128));
        if (p.stages > kMaxStages) p.stages = kMaxStages;
    }
    if (row_tiles * p.splits > INT32_MAX / 4 || token_tiles > 65535 || row_tiles * token_tiles > INT32_MAX / 4)
        return fail(TANS_B200_ERR_INVALID, "linear: m and rows are too large");
    p.row_tiles = (int32_t)row_tiles;
    p.token_tiles = (int32_t)token_tiles;
    int rc = e4m3_map(&p.wmap, w, rows, cols, 128);
    if (!rc) rc = e4m3_map(&p.xmap, x, m, cols, pair ? p.bn / 2 : p.bn);
    if (rc) return rc;
    return dispatch_half(dtype, "linear", [&](auto t) { return launch_linear<decltype(t)>(p, pair, sms, (cudaStream_t)stream); });
}
