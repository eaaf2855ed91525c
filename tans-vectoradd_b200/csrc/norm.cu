// norm.cu — residual addition, RMS norm and e4m3 quantisation of token rows.
//
//   s = x + r                        (f32; s = x without a residual)
//   h = rn(s)                        the residual stream, x's type
//   y = s * rsqrt(mean(s^2) + eps) * w
//   scale = max|y| / 448 (1 for a row of zeros, never below the smallest normal f32),
//   q = e4m3(y / scale)
//
// All of it in f32, each output rounded once; the mean square is that of the
// unrounded sum.  max|y| needs no second pass: the factor rsqrt(..) is one
// positive number a row, so max|y| = rsqrt(..) * max|s * w|, and one block
// reduction gives both the sum of squares and that maximum.
//
// One CTA a row, the row in registers between the reduction and the outputs:
// every input is read once and every output written once, so the kernel is
// bound by memory for many rows and by launch and reduction latency for few.
// Measured on one B200, residual and e4m3 output: 16384 x 5120 bf16 95 us =
// 6.2 TB/s (95 % of the copy rate), 16384 x 5121 102 us; 1 x 5120 2.7 us among
// others in a graph.  e4m3 alone, without a norm: 16384 x 5120 57 us, 1 x 5120 2.7-3.0
// us (2.2 with a factor in the divisions' place).
// All loads of a row come before the first use of one: 135 us with the
// residual's after the sums of x began.

#include "sm100.cuh"

namespace tans_b200 {
namespace {

struct NormArgs {
    const void *x, *residual, *weight;  // residual, weight: may be null
    int64_t x_stride, r_stride, h_stride;  // elements between rows
    void *h, *y;     // h: null without a residual; y: null when quantising
    uint8_t *q;
    float *scale;
    int32_t cols;
    float eps;
    bool weight_f32;
    bool weight_vec = false;  // the weight has x's type and begins on a 16-byte boundary
};

// Sum of a and maximum (NaN kept) of b over the block; every thread gets both.
__device__ __forceinline__ void block_reduce(float &a, float &b, float2 *buf) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
    const int warps = blockDim.x >> 5;
    if (warps == 1) return;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    const float2 v = (threadIdx.x & 31) < warps ? buf[threadIdx.x & 31] : make_float2(0.f, 0.f);
    a = v.x;
    b = v.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
}

// From a row's sum of squares and max|s * w|: what brings s * w to y, or to
// y / scale when quantising a norm, and the scale.  There the root cancels, y /
// scale = s * w * 448 / max|s * w|, one rounding less; sizes far out of range (and
// NaN) take the long way.
template <bool kNorm>
__device__ __forceinline__ float row_factor(const NormArgs &p, float sumsq, float amax, float &scale) {
    const float inv = kNorm ? rsqrtf(sumsq / (float)p.cols + p.eps) : 1.f;
    if (!p.q) return inv;
    const float top = amax * inv;
    scale = top == 0.f ? 1.f : max_nan(top / 448.f, 1.17549435e-38f);
    return amax > 1e-30f && amax < 1e30f && top > 1e-30f ? 448.f / amax : inv / scale;
}

// s * w as y, or as y / scale when quantising, from row_factor's f and scale.
// Without a norm y is x, whose few bits make ties of two e4m3 values common: its
// quotient by the scale is rounded once (by a factor 448 / max|x| 317 of 2 million
// bf16 values came out on the other side of a tie).
template <bool kNorm>
__device__ __forceinline__ float scaled(float sw, float f, float scale) {
    return kNorm ? sw * f : sw / scale;
}

// Elements o .. o + 7 of the sixteen in a and b, 0 < o < 8, the same o in all lanes.
template <typename T>
__device__ __forceinline__ Eight<T> window(const Eight<T> &a, const Eight<T> &b, int o) {
    constexpr int kWords = 2 * (int)sizeof(T);
    uint32_t w[2 * kWords];
#pragma unroll
    for (int i = 0; i < kWords; i++) {
        w[i] = reinterpret_cast<const uint32_t *>(a.u)[i];
        w[kWords + i] = reinterpret_cast<const uint32_t *>(b.u)[i];
    }
    if (o & 4) {
#pragma unroll
        for (int i = 0; i < 3 * kWords / 2; i++) w[i] = w[i + kWords / 2];
    }
    if (o & 2) {
#pragma unroll
        for (int i = 0; i < 5 * kWords / 4; i++) w[i] = w[i + kWords / 4];
    }
    if (o & 1) {
#pragma unroll
        for (int i = 0; i < kWords; i++) w[i] = sizeof(T) == 4 ? w[i + 1] : __funnelshift_r(w[i], w[i + 1], 16);
    }
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < kWords; i++) reinterpret_cast<uint32_t *>(r.u)[i] = w[i];
    return r;
}

// Rows by 8-element vectors on 16-byte boundaries: thread t holds vectors t, t +
// blockDim, ...  kShifted: rows begin anywhere, x, residual, h and y alike; the
// vectors are those between the row's first and last boundary, the elements at
// its ends are one each of the block's first 16 threads, and the weight, which lies
// otherwise, is cut out of two of its own vectors (one of another type or off
// its boundary: read one by one).
template <typename T, int VPT, int kMost, bool kShifted, bool kNorm>
__global__ void __launch_bounds__(kMost) norm_vec_kernel(const NormArgs p) {
    __shared__ float2 buf[32];
    pdl_enter();
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *r = kNorm && p.residual ? static_cast<const T *>(p.residual) + row * p.r_stride : nullptr;
    constexpr int kPer = 16 / (int)sizeof(T);
    const int head = kShifted ? min((kPer - (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % kPer)) % kPer, p.cols) : 0;
    const int vecs = (p.cols - head) / 8;
    // this thread's element of the ends, or none
    const int end = (int)threadIdx.x < 8 ? (int)threadIdx.x : head + 8 * vecs + (int)threadIdx.x - 8;
    const bool has_end = kShifted && threadIdx.x < 16 && end < (threadIdx.x < 8 ? head : p.cols);
    const T *wt = static_cast<const T *>(p.weight);
    float at_end = 0.f, w_end = 1.f;
    if (has_end) {
        at_end = to_f32(x[end]);
        if (r) at_end += to_f32(r[end]);
        if (kNorm) w_end = p.weight_f32 ? static_cast<const float *>(p.weight)[end] : to_f32(wt[end]);
    }
    // every load of the row before the first use of one
    Eight<T> xv[VPT], rv[VPT], wv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v < vecs) {
            xv[i] = load_eight(x + head + 8 * v);
            if (r) rv[i] = load_eight(r + head + 8 * v);
            if (!kShifted && kNorm && !p.weight_f32) wv[i] = load_eight(wt + 8 * v);
        }
    }
    float s[VPT][8];
    float sumsq = 0.f, amax = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v < vecs) {
            xv[i].to(s[i]);
            if (r) {
                float a[8];
                rv[i].to(a);
#pragma unroll
                for (int k = 0; k < 8; k++) s[i][k] += a[k];
                store8(static_cast<T *>(p.h) + row * p.h_stride + head + 8 * v, s[i]);
            }
            if (kNorm) {
                float w[8];
                if constexpr (kShifted) {
                    if (p.weight_vec && (head == 0 || 8 * v + 16 <= p.cols)) {
                        Eight<T> e = load_eight(wt + 8 * v);
                        if (head) e = window(e, load_eight(wt + 8 * v + 8), head);
                        e.to(w);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const int e = head + 8 * v + k;
                            w[k] = p.weight_f32 ? static_cast<const float *>(p.weight)[e] : to_f32(wt[e]);
                        }
                    }
                } else if (p.weight_f32) {
                    load8(static_cast<const float *>(p.weight) + 8 * v, w);
                } else {
                    wv[i].to(w);
                }
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    sumsq = __fmaf_rn(s[i][k], s[i][k], sumsq);
                    s[i][k] *= w[k];
                }
            }
            if (p.q) {
#pragma unroll
                for (int k = 0; k < 8; k++) amax = max_nan(amax, fabsf(s[i][k]));
            }
        }
    }
    if (has_end) {
        if (r) static_cast<T *>(p.h)[row * p.h_stride + end] = from_f32<T>(at_end);
        if (kNorm) sumsq = __fmaf_rn(at_end, at_end, sumsq);
        at_end *= w_end;
        if (p.q) amax = max_nan(amax, fabsf(at_end));
    }
    block_reduce(sumsq, amax, buf);
    float scale;
    const float f = row_factor<kNorm>(p, sumsq, amax, scale);
    if (p.q && threadIdx.x == 0) p.scale[row] = scale;
    if (has_end) {
        if (p.q)
            p.q[row * p.cols + end] = (uint8_t)e4m3x2(scaled<kNorm>(at_end, f, scale), 0.f);
        else
            static_cast<T *>(p.y)[row * p.cols + end] = from_f32<T>(at_end * f);
    }
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v < vecs) {
#pragma unroll
            for (int k = 0; k < 8; k++) s[i][k] = scaled<kNorm>(s[i][k], f, scale);
            if (p.q) {
                uint2 u;
                u.x = e4m3x2(s[i][0], s[i][1]) | e4m3x2(s[i][2], s[i][3]) << 16;
                u.y = e4m3x2(s[i][4], s[i][5]) | e4m3x2(s[i][6], s[i][7]) << 16;
                uint8_t *q = p.q + row * p.cols + head + 8 * v;
                if (!kShifted) {
                    *reinterpret_cast<uint2 *>(q) = u;
                } else {  // on a boundary of four
                    reinterpret_cast<uint32_t *>(q)[0] = u.x;
                    reinterpret_cast<uint32_t *>(q)[1] = u.y;
                }
            } else {
                store8(static_cast<T *>(p.y) + row * p.cols + head + 8 * v, s[i]);
            }
        }
    }
}

// Wider rows, and rows of tensors that lie to 16-byte boundaries each in its own
// way: element by element, s * w kept in shared memory (1021 x 4099 f16: 9.7 us
// out of L2, where vectors take 5.3; bound by its 2-byte accesses).
template <typename T, bool kNorm>
__global__ void __launch_bounds__(1024) norm_any_kernel(const NormArgs p) {
    extern __shared__ float srow[];
    __shared__ float2 buf[32];
    pdl_enter();
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *r = kNorm && p.residual ? static_cast<const T *>(p.residual) + row * p.r_stride : nullptr;
    T *h = r ? static_cast<T *>(p.h) + row * p.h_stride : nullptr;
    float sumsq = 0.f, amax = 0.f;
    for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
        float s = to_f32(x[c]);
        if (r) {
            s += to_f32(r[c]);
            h[c] = from_f32<T>(s);
        }
        sumsq += s * s;
        if (kNorm)
            s *= p.weight_f32 ? static_cast<const float *>(p.weight)[c] : to_f32(static_cast<const T *>(p.weight)[c]);
        amax = max_nan(amax, fabsf(s));
        srow[c] = s;
    }
    block_reduce(sumsq, amax, buf);
    float scale;
    const float f = row_factor<kNorm>(p, sumsq, amax, scale);
    if (p.q && threadIdx.x == 0) p.scale[row] = scale;
    for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
        const float y = scaled<kNorm>(srow[c], f, scale);
        if (p.q)
            p.q[row * p.cols + c] = (uint8_t)e4m3x2(y, 0.f);
        else
            static_cast<T *>(p.y)[row * p.cols + c] = from_f32<T>(y);
    }
}

constexpr int kMaxCols = 56 * 1024;  // f32 values of one row that fit a CTA's shared memory

template <typename T, bool kNorm>
int launch_norm(NormArgs p, int64_t rows, cudaStream_t st) {
    p.weight_vec = is_aligned(p.weight, 16) && (!p.weight_f32 || sizeof(T) == 4);
    constexpr int64_t kPer = 16 / (int64_t)sizeof(T);  // elements between boundaries
    const dim3 grid((unsigned)rows);
    // One of x, residual, h and y that exists: do its rows begin where x's do, in
    // every row, relative to 16-byte boundaries?
    const auto as_x = [&](const void *ptr, int64_t stride) {
        return !ptr || ((reinterpret_cast<uintptr_t>(ptr) - reinterpret_cast<uintptr_t>(p.x)) % 16 == 0 &&
                        (stride - p.x_stride) % kPer == 0);
    };
    const bool alike = as_x(p.residual, p.r_stride) && as_x(p.h, p.h_stride) && as_x(p.y, p.cols);
    const bool vec = alike && p.cols % 8 == 0 && p.cols <= 32 * 1024 && is_aligned(p.x, 16) && p.x_stride % kPer == 0 &&
                     is_aligned(p.weight, 16) && is_aligned(p.q, 8);
    // Otherwise by vectors all the same (1021 x 4099 f16, odd rows: 5.3 us, element by
    // element 9.7); the bytes of q then lie to boundaries of four as x's elements do.
    const bool shifted = alike && p.cols < 32 * 1024 + 8 && reinterpret_cast<uintptr_t>(p.x) % sizeof(T) == 0 &&
                         (!p.q || (is_aligned(p.q, 4) && is_aligned(p.x, 16) && (p.x_stride - p.cols) % kPer == 0));
    if (!vec && !shifted) {
        const int threads = p.cols >= 1024 ? 512 : (p.cols >= 256 ? 128 : 32);
        const int smem = p.cols * 4;
        const int rc = allow_smem<norm_any_kernel<T, kNorm>>("norm_any_kernel", kMaxCols * 4);
        if (rc) return rc;
        return launch_ex(norm_any_kernel<T, kNorm>, grid, dim3(threads), smem, 1, st, "norm_any_kernel", p);
    }
    const int vecs = p.cols < 8 ? 1 : p.cols / 8;
    // four vectors a thread: a row's loads are in flight at once, with many rows resident
    const int threads = ceil_div(ceil_div(vecs, 4), 32) * 32;
    const auto launch = [&](auto kernel) {
        return launch_ex(kernel, grid, dim3(threads), 0, 1, st, "norm_vec_kernel", p);
    };
    const auto form = [&](auto shifted) {
        constexpr bool S = decltype(shifted)::value;
        if (vecs <= threads) return launch(norm_vec_kernel<T, 1, 32, S, kNorm>);
        if (vecs <= 2 * threads) return launch(norm_vec_kernel<T, 2, 32, S, kNorm>);
        if (threads <= 256) return launch(norm_vec_kernel<T, 4, 256, S, kNorm>);
        return launch(norm_vec_kernel<T, 4, 1024, S, kNorm>);
    };
    return vec ? form(std::false_type{}) : form(std::true_type{});
}

int check_rows(const char *what, int64_t rows, int64_t cols) {
    if (rows < 0 || rows > INT32_MAX || cols < 1 || cols > kMaxCols)
        return fail(TANS_B200_ERR_INVALID, "%s: rows must be 0..2^31-1 and cols 1..%d", what, kMaxCols);
    return TANS_B200_OK;
}

}  // namespace
}  // namespace tans_b200

using namespace tans_b200;

extern "C" int tans_b200_add_rms_norm(const void *x, int64_t x_stride, const void *residual, int64_t r_stride,
                                      const void *weight, int weight_dtype, float eps, void *h, int64_t h_stride,
                                      void *y, uint8_t *q, float *scale, int64_t rows, int64_t cols, int dtype,
                                      void *stream) {
    clear_error();
    int rc = check_rows("add_rms_norm", rows, cols);
    if (rc) return rc;
    if (rows == 0) return TANS_B200_OK;
    if (!x || !weight || (residual && !h) || (y ? (q || scale) : (!q || !scale)))
        return fail(TANS_B200_ERR_INVALID,
                    "add_rms_norm: x, weight, h with a residual, and either y or q and scale are needed");
    if (weight_dtype != dtype && weight_dtype != TANS_B200_F32)
        return fail(TANS_B200_ERR_INVALID, "add_rms_norm: the weight must have x's type or be f32");
    if (!may_hold(element_bytes(dtype), x, residual, h, y) || !may_hold(element_bytes(weight_dtype), weight) || !may_hold(4, scale))
        return fail(TANS_B200_ERR_INVALID, "add_rms_norm: an array is not aligned to its elements");
    if (residual && rows > 1 && h_stride > -cols && h_stride < cols)
        return fail(TANS_B200_ERR_INVALID, "add_rms_norm: the rows of h overlap");
    if (!(eps >= 0.f)) return fail(TANS_B200_ERR_INVALID, "add_rms_norm: eps must not be negative");
    NormArgs p{x, residual, weight, x_stride, r_stride, h_stride, residual ? h : nullptr, y, q, scale,
               (int32_t)cols, eps, weight_dtype == TANS_B200_F32};
    return dispatch_float(dtype, "add_rms_norm", [&](auto t) {
        return launch_norm<decltype(t), true>(p, rows, (cudaStream_t)stream);
    });
}

extern "C" int tans_b200_quantize_tokens(const void *x, int64_t x_stride, uint8_t *q, float *scale, int64_t rows,
                                         int64_t cols, int dtype, void *stream) {
    clear_error();
    int rc = check_rows("quantize_tokens", rows, cols);
    if (rc) return rc;
    if (rows == 0) return TANS_B200_OK;
    if (!x || !q || !scale) return fail(TANS_B200_ERR_INVALID, "quantize_tokens: null pointer");
    if (!may_hold(element_bytes(dtype), x) || !may_hold(4, scale))
        return fail(TANS_B200_ERR_INVALID, "quantize_tokens: an array is not aligned to its elements");
    NormArgs p{x, nullptr, nullptr, x_stride, 0, 0, nullptr, nullptr, q, scale, (int32_t)cols, 0.f, false};
    return dispatch_float(dtype, "quantize_tokens", [&](auto t) {
        return launch_norm<decltype(t), false>(p, rows, (cudaStream_t)stream);
    });
}
