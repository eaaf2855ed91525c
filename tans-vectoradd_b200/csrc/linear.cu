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

#include "sm100.cuh"

#include <cuda.h>

namespace tans_b200 {
namespace {

constexpr int kMaxStages = 8;
constexpr uint32_t kWaitLimit = 1u << 16;  // polls per wait
constexpr uint32_t kPollNs = 10000;        // suspend-time hint per poll: bound ~0.66 s
constexpr int kThreads = 192;              // copy warp, MMA warp, four epilogue warps

struct LinearArgs {
    CUtensorMap wmap, xmap;  // boxes of 128 columns x 128 rows / bn tokens, 128-byte swizzle
    const float *x_scale, *w_scale;
    const void *bias, *mul, *residual;
    void *y;
    int64_t m, rows;
    int32_t chunks;  // of 128 columns
    int32_t bn, stages, act;
    int32_t *status;
};

__device__ __forceinline__ uint32_t shared_addr(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
// Wait for the phase of `bar` with the given parity; false when the wait runs
// out or (checked every 16 polls) *failed became non-zero.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const volatile int32_t *failed) {
    for (uint32_t i = 0; i < kWaitLimit; i++) {
        uint32_t done;
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

// act(v); SiLU is v / (1 + e^-v), and the tanh form of GELU is
// v / (1 + e^(-2 sqrt(2/pi) (v + 0.044715 v^3))) as 1 + tanh(u) = 2 / (1 + e^-2u).
__device__ __forceinline__ float activate(float v, int act) {
    if (act == TANS_B200_ACT_NONE) return v;
    if (act == TANS_B200_ACT_RELU) return v < 0.f ? 0.f : v;
    const float u = act == TANS_B200_ACT_SILU ? v : 1.5957691216057308f * (v + 0.044715f * v * v * v);
    return __fdividef(v, 1.f + __expf(-u));
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) linear_kernel(const __grid_constant__ LinearArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], done;
    __shared__ uint32_t tmem_s;
    __shared__ int32_t failed_s, copied_s;
    volatile int32_t *failed = &failed_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t a_sa = (shared_addr(smem) + 1023u) & ~1023u;
    const uint32_t a_bytes = 128u * 128u, b_bytes = (uint32_t)p.bn * 128u;
    const uint32_t b_sa = a_sa + (uint32_t)p.stages * a_bytes;
    const uint32_t full0 = shared_addr(full), empty0 = shared_addr(empty), done0 = shared_addr(&done);
    const uint32_t ncols = p.bn <= 32 ? 32u : (p.bn <= 64 ? 64u : (p.bn <= 128 ? 128u : 256u));
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
    const int32_t r0 = (int32_t)blockIdx.x * 128, t0 = (int32_t)blockIdx.y * p.bn;
    pdl_enter();

    if (warp == 0 && lane == 0) {  // ------------------------------ copies
        int s = 0;
        uint32_t ph = 1;  // a fresh stage counts as empty
        for (int32_t c = 0; c < p.chunks; c++) {
            if (!mbar_wait(empty0 + 8u * s, ph, failed)) {
                *failed = 1;
                break;
            }
            const uint32_t bar = full0 + 8u * s;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(a_bytes + b_bytes)
                         : "memory");
            copy_box(&p.wmap, a_sa + (uint32_t)s * a_bytes, bar, c * 128, r0);
            copy_box(&p.xmap, b_sa + (uint32_t)s * b_bytes, bar, c * 128, t0);
            copied_s = c + 1;
            if (++s == p.stages) s = 0, ph ^= 1u;
        }
    } else if (warp == 1 && lane == 0) {  // ----------------------- MMA
        // D f32, A and B e4m3, K-major
        const uint32_t idesc = (1u << 4) | ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int32_t c = 0; c < p.chunks; c++) {
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
                    "l"(smem_desc(a_sa + (uint32_t)s * a_bytes + 32u * j)),
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
    if (*failed) {
        if (threadIdx.x == 0) {  // copies in flight land before the CTA may end
            if (p.status) atomicOr(p.status, TANS_B200_DATA_TIMEOUT);
            for (int32_t c = copied_s > p.stages ? copied_s - p.stages : 0; c < copied_s; c++)
                mbar_wait(full0 + 8u * (c % p.stages), (uint32_t)((c / p.stages) & 1), nullptr);
        }
    } else if (warp >= 2) {  // ------------------------------------- epilogue
        const int quarter = warp & 3;
        const int64_t r = r0 + 32 * quarter + lane;
        const bool real = r < p.rows;
        const float ws = real ? p.w_scale[r] : 0.f;
        const float bias = real && p.bias ? to_f32(static_cast<const T *>(p.bias)[r]) : 0.f;
        for (int col = 0; col < p.bn && t0 + col < p.m; col += 8) {
            uint32_t v[8];
            asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                         : "r"(tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)col));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int64_t t = t0 + col + k;
                if (real && t < p.m) {
                    float a = activate(__uint_as_float(v[k]) * ws * p.x_scale[t] + bias, p.act);
                    if (p.mul) a *= to_f32(static_cast<const T *>(p.mul)[t * p.rows + r]);
                    if (p.residual) a += to_f32(static_cast<const T *>(p.residual)[t * p.rows + r]);
                    static_cast<T *>(p.y)[t * p.rows + r] = from_f32<T>(a);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(ncols));
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
int launch_linear(const LinearArgs &p, cudaStream_t st) {
    const int smem = 1024 + p.stages * (128 + p.bn) * 128;
    const cudaError_t e = cudaFuncSetAttribute(linear_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return launch_failed("linear_kernel", e);
    return launch_ex(linear_kernel<T>, dim3((unsigned)ceil_div<int64_t>(p.rows, 128), (unsigned)ceil_div<int64_t>(p.m, p.bn)),
                     dim3(kThreads), smem, 1, st, "linear_kernel", p);
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
    p.bn = m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : (m <= 128 ? 128 : 256)));
    p.stages = p.bn <= 128 ? 6 : 4;
    int rc = e4m3_map(&p.wmap, w, rows, cols, 128);
    if (!rc) rc = e4m3_map(&p.xmap, x, m, cols, p.bn);
    if (rc) return rc;
    return dispatch_half(dtype, "linear", [&](auto t) { return launch_linear<decltype(t)>(p, (cudaStream_t)stream); });
}
