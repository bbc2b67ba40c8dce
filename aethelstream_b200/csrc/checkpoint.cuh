// checkpoint.cuh -- RMS norm with its input kept in 8 bits, and what the second
// pass does with that checkpoint: restore it, take the norm's gradient at it,
// and the gradient of the linear layer that follows.
//
// Checkpoint of x (rows x d): blocks of 128 features of a row;
//   scale = max|x| / 127 (1 where that maximum is below 2^-119, whose scale's
//           reciprocal fp32 does not hold),
//   code = clamp(round_half_away(x * (1 / scale)), +-127),  x^ = code * scale
// (the formula of the blockwise INT8 state codec).  A block that holds a NaN or
// an infinity gets a NaN scale: it restores to NaN throughout.
//
// Norm: y = s / sqrt(mean s^2 + eps) * gain, s = x (+ residual, rounded to the
// activations' type first: the sum that the next block reads).
// Backward, at x^ with r = 1 / sqrt(mean x^2 + eps):
//   dx = r (dy gain) - x^ r^3 mean(dy gain x^) (+ d_residual)
//   d_gain = sum over rows of dy x^ r
// Sums are fp32.
#pragma once
#include "common.cuh"

namespace aeth {

constexpr int kCkptBlock = 128;

template <typename T>
__device__ __forceinline__ float ck_load(const T* p);
template <>
__device__ __forceinline__ float ck_load<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float ck_load<__half>(const __half* p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float ck_load<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }

template <typename T>
__device__ __forceinline__ T ck_cast(float v);
template <>
__device__ __forceinline__ float ck_cast<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half ck_cast<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 ck_cast<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Scale of a block from its maximum magnitude (NaN where the block held one).
__device__ __forceinline__ float ck_scale(float amax) {
    if (!(amax <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    return amax < 1.504632769e-36f ? 1.0f : __fdiv_rn(amax, 127.0f);
}
__device__ __forceinline__ int8_t ck_encode(float x, float scale) {
    return scale != scale ? (int8_t)0 : lin_encode(x, __fdiv_rn(1.0f, scale));
}

__device__ __forceinline__ float ck_block_sum(float v, float* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[warp] = v;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < nw; ++w) s += sh[w];
    return s;
}

__device__ __forceinline__ float ck_rstd(float sumsq, int d, float eps) {
    return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, (float)d), eps)));
}

template <typename T>
struct CkptStore {
    const T* x;
    int64_t ldx;
    const T* residual;  // or null
    int64_t ldr;
    const void* gain;
    int gain_dtype;
    int64_t rows;
    int d;
    float eps;
    T* sum;  // with residual
    T* y;
    int8_t* codes;
    float* scales;
};

template <typename T>
__global__ void __launch_bounds__(256) ckpt_store_kernel(CkptStore<T> a) {
    __shared__ float sh[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nb = (a.d + kCkptBlock - 1) / kCkptBlock;
    for (int64_t t = blockIdx.x; t < a.rows; t += gridDim.x) {
        const T* x = a.x + t * a.ldx;
        const T* res = a.residual ? a.residual + t * a.ldr : nullptr;
        auto at = [&](int c) {
            float v = ck_load(x + c);
            if (res) v = ck_load<T>(&(const T&)ck_cast<T>(v + ck_load(res + c)));
            return v;
        };
        float ss = 0.0f;
        for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
            const float v = at(c);
            ss += v * v;
            if (res) a.sum[t * a.d + c] = ck_cast<T>(v);
        }
        const float r = ck_rstd(ck_block_sum(ss, sh), a.d, a.eps);
        for (int c = threadIdx.x; c < a.d; c += blockDim.x)
            a.y[t * a.d + c] = ck_cast<T>(at(c) * r * load_as_f32(a.gain, c, a.gain_dtype));
        for (int b = warp; b < nb; b += 8) {
            float v[4], m = 0.0f;
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = b * kCkptBlock + i * 32 + lane;
                v[i] = c < a.d ? at(c) : 0.0f;
                m = fmaxf(m, fabsf(v[i]));
                nan |= v[i] != v[i];
            }
            m = warp_max(m);
            if (__any_sync(0xffffffffu, nan)) m = __int_as_float(0x7fc00000);
            const float s = ck_scale(m);
            if (lane == 0) a.scales[t * nb + b] = s;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = b * kCkptBlock + i * 32 + lane;
                if (c < a.d) a.codes[t * a.d + c] = ck_encode(v[i], s);
            }
        }
    }
}

// x^, or its norm where gain is given.
template <typename T>
__global__ void __launch_bounds__(256) ckpt_decode_kernel(const int8_t* __restrict__ codes,
                                                          const float* __restrict__ scales, int64_t rows, int d,
                                                          const void* __restrict__ gain, int gain_dtype, float eps,
                                                          T* __restrict__ out, int64_t ldo) {
    __shared__ float sh[8];
    const int nb = (d + kCkptBlock - 1) / kCkptBlock;
    for (int64_t t = blockIdx.x; t < rows; t += gridDim.x) {
        auto at = [&](int c) { return (float)codes[t * d + c] * scales[t * nb + c / kCkptBlock]; };
        float r = 1.0f;
        if (gain) {
            float ss = 0.0f;
            for (int c = threadIdx.x; c < d; c += blockDim.x) ss += at(c) * at(c);
            r = ck_rstd(ck_block_sum(ss, sh), d, eps);
        }
        for (int c = threadIdx.x; c < d; c += blockDim.x)
            out[t * ldo + c] = ck_cast<T>(gain ? at(c) * r * load_as_f32(gain, c, gain_dtype) : at(c));
    }
}

template <typename T>
struct CkptBack {
    const T* dy;
    int64_t ld_dy;
    const int8_t* codes;
    const float* scales;
    const void* gain;
    int gain_dtype;
    const T* d_res;  // or null
    int64_t ld_res;
    int64_t rows;
    int d;
    float eps;
    T* dx;
    float* rstd;  // workspace, one per row
};

template <typename T>
__global__ void __launch_bounds__(256) ckpt_back_kernel(CkptBack<T> a) {
    __shared__ float sh[8];
    const int nb = (a.d + kCkptBlock - 1) / kCkptBlock;
    for (int64_t t = blockIdx.x; t < a.rows; t += gridDim.x) {
        auto at = [&](int c) { return (float)a.codes[t * a.d + c] * a.scales[t * nb + c / kCkptBlock]; };
        auto dyw = [&](int c) { return ck_load(a.dy + t * a.ld_dy + c) * load_as_f32(a.gain, c, a.gain_dtype); };
        float ss = 0.0f, dot = 0.0f;
        for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
            const float x = at(c);
            ss += x * x;
            dot += x * dyw(c);
        }
        const float r = ck_rstd(ck_block_sum(ss, sh), a.d, a.eps);
        const float k = r * r * r * (ck_block_sum(dot, sh) / (float)a.d);
        if (threadIdx.x == 0) a.rstd[t] = r;
        for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
            float v = r * dyw(c) - at(c) * k;
            if (a.d_res) v += ck_load(a.d_res + t * a.ld_res + c);
            a.dx[t * a.d + c] = ck_cast<T>(v);
        }
    }
}

// d_gain: each thread sums one column over a range of rows; the ranges are
// added in their order.
template <typename T>
__global__ void __launch_bounds__(128) ckpt_gain_partial_kernel(const T* __restrict__ dy, int64_t ld_dy,
                                                                const int8_t* __restrict__ codes,
                                                                const float* __restrict__ scales,
                                                                const float* __restrict__ rstd, int64_t rows, int d,
                                                                int64_t per, float* __restrict__ part) {
    const int c = blockIdx.x * 128 + threadIdx.x;
    if (c >= d) return;
    const int nb = (d + kCkptBlock - 1) / kCkptBlock;
    const int64_t t0 = blockIdx.y * per, t1 = min(t0 + per, rows);
    float s = 0.0f;
    for (int64_t t = t0; t < t1; ++t)
        s += ck_load(dy + t * ld_dy + c) * ((float)codes[t * d + c] * scales[t * nb + c / kCkptBlock]) * rstd[t];
    part[(int64_t)blockIdx.y * d + c] = s;
}

__global__ void __launch_bounds__(128) ckpt_gain_sum_kernel(const float* __restrict__ part, int np, int d,
                                                            float* __restrict__ d_gain) {
    const int c = blockIdx.x * 128 + threadIdx.x;
    if (c >= d) return;
    float s = 0.0f;
    for (int p = 0; p < np; ++p) s += part[(int64_t)p * d + c];
    d_gain[c] = s;
}

}  // namespace aeth
