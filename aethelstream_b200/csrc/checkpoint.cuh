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

// Eight consecutive features of a row as they lie in memory.
template <typename T>
struct Pack8 {
    static constexpr int kWords = (int)sizeof(T) / 2;
    uint4 w[kWords];
};

template <typename T>
__device__ __forceinline__ float ck_value(const Pack8<T>& p, int i);
template <>
__device__ __forceinline__ float ck_value<float>(const Pack8<float>& p, int i) {
    const uint4 q = p.w[i >> 2];
    return __uint_as_float((i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w);
}
template <>
__device__ __forceinline__ float ck_value<__nv_bfloat16>(const Pack8<__nv_bfloat16>& p, int i) {
    const uint4 q = p.w[0];
    const uint32_t x = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return __uint_as_float((i & 1) ? x & 0xffff0000u : x << 16);
}
template <>
__device__ __forceinline__ float ck_value<__half>(const Pack8<__half>& p, int i) {
    const uint4 q = p.w[0];
    const uint32_t x = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return __half2float(__ushort_as_half((uint16_t)((i & 1) ? x >> 16 : x)));
}

template <typename T>
__device__ __forceinline__ uint32_t ck_pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t ck_pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t ck_pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__device__ __forceinline__ Pack8<T> ck_pack(const float (&v)[8]) {
    Pack8<T> p;
    if constexpr (sizeof(T) == 4) {
        p.w[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        p.w[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
        p.w[0] = make_uint4(ck_pack2<T>(v[0], v[1]), ck_pack2<T>(v[2], v[3]), ck_pack2<T>(v[4], v[5]),
                            ck_pack2<T>(v[6], v[7]));
    }
    return p;
}

// Features c .. c + 7 of a row of d (zero past its end).  VEC: every row
// starts on 16 bytes and d is a multiple of 8; otherwise single elements.
template <typename T, bool VEC>
__device__ __forceinline__ Pack8<T> ck_load8(const T* row, int c, int d) {
    Pack8<T> p;
    if (VEC) {
#pragma unroll
        for (int k = 0; k < Pack8<T>::kWords; ++k)
            p.w[k] = c < d ? __ldg(reinterpret_cast<const uint4*>(row + c) + k) : make_uint4(0, 0, 0, 0);
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < d ? (float)row[c + i] : 0.0f;
        p = ck_pack<T>(v);
    }
    return p;
}
template <typename T, bool VEC>
__device__ __forceinline__ void ck_store8(T* row, int c, int d, const Pack8<T>& p) {
    if (VEC) {
        if (c < d)
#pragma unroll
            for (int k = 0; k < Pack8<T>::kWords; ++k) reinterpret_cast<uint4*>(row + c)[k] = p.w[k];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < d) row[c + i] = (T)ck_value<T>(p, i);
    }
}
template <bool VEC>
__device__ __forceinline__ uint2 ck_load_codes(const int8_t* row, int c, int d) {
    if (VEC) return c < d ? __ldg(reinterpret_cast<const uint2*>(row + c)) : make_uint2(0, 0);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < d) w[i >> 2] |= (uint32_t)(uint8_t)row[c + i] << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}
template <bool VEC>
__device__ __forceinline__ void ck_store_codes(int8_t* row, int c, int d, uint2 q) {
    if (VEC) {
        if (c < d) *reinterpret_cast<uint2*>(row + c) = q;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < d) row[c + i] = (int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
    }
}
__device__ __forceinline__ float ck_code(uint2 q, int i) {
    return (float)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
}

// gain has a type of its own
__device__ __forceinline__ void ck_gain8(const void* gain, int dtype, int c, int d, float (&g)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = c + i < d ? load_as_f32(gain, c + i, dtype) : 0.0f;
}

// Scale of a block from its maximum magnitude (NaN where the block held one).
__device__ __forceinline__ float ck_scale(float amax) {
    if (!(amax <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    return amax < 1.504632769e-36f ? 1.0f : __fdiv_rn(amax, 127.0f);
}

// round_half_away(x / scale's rounded reciprocal): adding a half of x's sign
// with rounding toward zero never carries a value below k - 1/2 up to k, so the
// truncation of that sum is the rounding.  |x| <= 127 scale (1 + 2^-22) in a
// block, so the sum stays below 128 and needs no clamp.
__device__ __forceinline__ int ck_round(float v) {
    return __float2int_rz(__fadd_rz(v, __uint_as_float((__float_as_uint(v) & 0x80000000u) | 0x3f000000u)));
}
__device__ __forceinline__ uint2 ck_encode8(const float (&x)[8], float scale) {
    if (scale != scale) return make_uint2(0, 0);
    const float inv = __frcp_rn(scale);
    int q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = ck_round(__fmul_rn(x[i], inv));
    const uint32_t a = __byte_perm(q[0], q[1], 0x0040), b = __byte_perm(q[2], q[3], 0x0040);
    const uint32_t c = __byte_perm(q[4], q[5], 0x0040), e = __byte_perm(q[6], q[7], 0x0040);
    return make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(c, e, 0x5410));
}

__device__ __forceinline__ float ck_rstd(float sumsq, int d, float eps) {
    return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, (float)d), eps)));
}

// Sums of a row, spread over threadIdx.x (threadIdx.y is the row within the
// CTA).  The order depends on the row's length alone, so a row's result does
// not change with the number of rows in the call: v[k] is the sum of one
// thread's eight features, sixteen lanes join to a block's sum, lane l of every
// warp adds the blocks l and l + 32, and a warp's tree joins the lanes.  One
// barrier a call: `sh` has two halves that alternate.
constexpr int kCkptShared = 64;  // blocks that a CTA holds: 8192 features / 128
template <int N, int VPT>
__device__ __forceinline__ void ck_row_sum(const float (&v)[VPT][N], float* sh, int parity, float (&sum)[N]) {
    const int tx = blockDim.x, blocks = VPT * tx / 16;
    float* s = sh + parity * (N * kCkptShared) + threadIdx.y * blocks * N;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float x = v[k][n];
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            if ((threadIdx.x & 15) == 0) s[((threadIdx.x + k * tx) >> 4) * N + n] = x;
        }
    if (tx == 32) __syncwarp();
    else __syncthreads();
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float x = lane < blocks ? s[lane * N + n] : 0.0f;
        if (lane + 32 < blocks) x += s[(lane + 32) * N + n];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        sum[n] = x;
    }
}

// Every kernel below holds a row in registers: thread x of a row takes the
// features 8 (x + k blockDim.x) .. + 7, k < VPT, so that sixteen neighbouring
// lanes hold a block of 128.  A CTA walks over rows; what depends on the
// feature alone (gain, its gradient's sum) stays in registers meanwhile.
// WIDE: rows longer than a CTA holds, taken in spans of 8 VPT blockDim.x
// features (v then sums a thread's eights over the spans) and read a second
// time after the row's sums are known.
#define CK_SPANS(base, d) for (int base = 0; base < (WIDE ? (d) : 1); base += 8 * VPT * (int)blockDim.x)
#define CK_COLUMN(base, k) ((base) + 8 * (int)(threadIdx.x + (k) * blockDim.x))

// Resident CTAs that the register budget has to allow: two rows of 8192 in
// flight on an SM (VPT 4), one of 1024 threads otherwise.
constexpr int ck_min_ctas(int vpt) { return vpt == 4 ? 2 : 1; }

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

template <typename T, int VPT, bool VEC>
__device__ __forceinline__ void ckpt_input(const CkptStore<T>& a, int64_t t, int base, int d, Pack8<T> (&x)[VPT]) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) x[k] = ck_load8<T, VEC>(a.x + t * a.ldx, CK_COLUMN(base, k), d);
    if (a.residual) {
        Pack8<T> res[VPT];
#pragma unroll
        for (int k = 0; k < VPT; ++k) res[k] = ck_load8<T, VEC>(a.residual + t * a.ldr, CK_COLUMN(base, k), d);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = ck_value<T>(x[k], i) + ck_value<T>(res[k], i);
            x[k] = ck_pack<T>(v);
        }
    }
}

template <typename T, int VPT, bool VEC, bool WIDE>
__global__ void __launch_bounds__(1024 / VPT, ck_min_ctas(VPT)) ckpt_store_kernel(const __grid_constant__ CkptStore<T> a) {
    __shared__ float sh[2 * kCkptShared];
    const int nb = (a.d + kCkptBlock - 1) / kCkptBlock;
    float g[VPT][8];
    if (!WIDE)
#pragma unroll
        for (int k = 0; k < VPT; ++k) ck_gain8(a.gain, a.gain_dtype, CK_COLUMN(0, k), a.d, g[k]);
    int parity = 0;
    for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < a.rows; t0 += (int64_t)gridDim.x * blockDim.y, parity ^= 1) {
        const int64_t t = t0 + threadIdx.y;
        const int d = t < a.rows ? a.d : 0;  // a row past the end holds nothing
        Pack8<T> x[VPT];
        float ss[VPT][1] = {}, sum[1];
        CK_SPANS(base, a.d) {
            ckpt_input<T, VPT, VEC>(a, t, base, d, x);
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = CK_COLUMN(base, k);
                if (a.residual) ck_store8<T, VEC>(a.sum + t * a.d, c, d, x[k]);
                float v[8], m = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[i] = ck_value<T>(x[k], i);
                    ss[k][0] = fmaf(v[i], v[i], ss[k][0]);
                }
#pragma unroll
                for (int i = 0; i < 8; i += 2) m = fmax3_nan(m, fabsf(v[i]), fabsf(v[i + 1]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = fmax3_nan(m, m, __shfl_xor_sync(0xffffffffu, m, o));
                const float s = ck_scale(m);
                if ((threadIdx.x & 15) == 0 && c < d) a.scales[t * nb + c / kCkptBlock] = s;
                ck_store_codes<VEC>(a.codes + t * a.d, c, d, ck_encode8(v, s));
            }
        }
        ck_row_sum<1>(ss, sh, parity, sum);
        const float r = ck_rstd(sum[0], a.d, a.eps);
        CK_SPANS(base, a.d) {
            if (WIDE) {
                ckpt_input<T, VPT, VEC>(a, t, base, d, x);
#pragma unroll
                for (int k = 0; k < VPT; ++k) ck_gain8(a.gain, a.gain_dtype, CK_COLUMN(base, k), a.d, g[k]);
            }
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = ck_value<T>(x[k], i) * r * g[k][i];
                ck_store8<T, VEC>(a.y + t * a.d, CK_COLUMN(base, k), d, ck_pack<T>(v));
            }
        }
    }
}

struct CkptRead {
    const int8_t* codes;
    const float* scales;
    const void* gain;  // null: the activations themselves (decode)
    int gain_dtype;
    int64_t rows;
    int d;
    float eps;
};

// x^ of eight features: the block's scale and the codes.
template <bool VEC>
__device__ __forceinline__ void ck_restore8(const CkptRead& a, int64_t t, int c, int d, uint2& q, float& s) {
    const int nb = (a.d + kCkptBlock - 1) / kCkptBlock;
    q = ck_load_codes<VEC>(a.codes + t * a.d, c, d);
    s = c < d ? __ldg(a.scales + t * nb + c / kCkptBlock) : 0.0f;
}

// The norm of x^, in rows of pitch ldo.
template <typename T, int VPT, bool VEC, bool WIDE>
__global__ void __launch_bounds__(1024 / VPT, ck_min_ctas(VPT))
    ckpt_norm_kernel(const __grid_constant__ CkptRead a, T* __restrict__ out, int64_t ldo) {
    __shared__ float sh[2 * kCkptShared];
    float g[VPT][8];
    if (!WIDE)
#pragma unroll
        for (int k = 0; k < VPT; ++k) ck_gain8(a.gain, a.gain_dtype, CK_COLUMN(0, k), a.d, g[k]);
    int parity = 0;
    for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < a.rows; t0 += (int64_t)gridDim.x * blockDim.y, parity ^= 1) {
        const int64_t t = t0 + threadIdx.y;
        const int d = t < a.rows ? a.d : 0;
        uint2 q[VPT];
        float s[VPT], ss[VPT][1] = {}, sum[1];
        CK_SPANS(base, a.d) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) ck_restore8<VEC>(a, t, CK_COLUMN(base, k), d, q[k], s[k]);
#pragma unroll
            for (int k = 0; k < VPT; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = ck_code(q[k], i) * s[k];
                    ss[k][0] = fmaf(x, x, ss[k][0]);
                }
        }
        ck_row_sum<1>(ss, sh, parity, sum);
        const float r = ck_rstd(sum[0], a.d, a.eps);
        CK_SPANS(base, a.d) {
            if (WIDE)
#pragma unroll
                for (int k = 0; k < VPT; ++k) {
                    ck_restore8<VEC>(a, t, CK_COLUMN(base, k), d, q[k], s[k]);
                    ck_gain8(a.gain, a.gain_dtype, CK_COLUMN(base, k), a.d, g[k]);
                }
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = ck_code(q[k], i) * s[k] * r * g[k][i];
                ck_store8<T, VEC>(out + t * ldo, CK_COLUMN(base, k), d, ck_pack<T>(v));
            }
        }
    }
}

// x^ in rows of pitch ldo; gridDim.y spans of the row.
template <typename T, int VPT, bool VEC>
__global__ void __launch_bounds__(1024 / VPT) ckpt_decode_kernel(const __grid_constant__ CkptRead a, T* __restrict__ out,
                                                                 int64_t ldo) {
    const int base = blockIdx.y * 8 * VPT * blockDim.x;
    for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < a.rows; t0 += (int64_t)gridDim.x * blockDim.y) {
        const int64_t t = t0 + threadIdx.y;
        const int d = t < a.rows ? a.d : 0;
        uint2 q[VPT];
        float s[VPT];
#pragma unroll
        for (int k = 0; k < VPT; ++k) ck_restore8<VEC>(a, t, CK_COLUMN(base, k), d, q[k], s[k]);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = ck_code(q[k], i) * s[k];
            ck_store8<T, VEC>(out + t * ldo, CK_COLUMN(base, k), d, ck_pack<T>(v));
        }
    }
}

template <typename T>
struct CkptBack {
    CkptRead in;
    const T* dy;
    int64_t ld_dy;
    const T* d_res;  // or null
    int64_t ld_res;
    T* dx;
    float* part;  // d_gain of each row group: gridDim.x * blockDim.y rows of d
};

// dx, and each row group's sum of d_gain (ckpt_gain_sum_kernel adds them in
// their order).  WIDE keeps that sum in `part` itself: each element has one
// thread.
template <typename T, int VPT, bool VEC, bool WIDE>
__global__ void __launch_bounds__(1024 / VPT, ck_min_ctas(VPT)) ckpt_back_kernel(const __grid_constant__ CkptBack<T> a) {
    __shared__ float sh[4 * kCkptShared];
    float* part = a.part + ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * a.in.d;
    float g[VPT][8], dg[VPT][8];
    auto gain_of = [&](int base) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) ck_gain8(a.in.gain, a.in.gain_dtype, CK_COLUMN(base, k), a.in.d, g[k]);
    };
    auto sums_to = [&](int base, bool add) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = CK_COLUMN(base, k);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < a.in.d) part[c + i] = dg[k][i] + (add ? part[c + i] : 0.0f);
        }
    };
    if (!WIDE) {
        gain_of(0);
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) dg[k][i] = 0.0f;
    }
    int parity = 0;
    bool first = true;
    for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < a.in.rows;
         t0 += (int64_t)gridDim.x * blockDim.y, parity ^= 1, first = false) {
        const int64_t t = t0 + threadIdx.y;
        const int d = t < a.in.rows ? a.in.d : 0;
        uint2 q[VPT];
        float s[VPT], acc[VPT][2] = {}, sum[2];
        Pack8<T> dy[VPT], res[VPT];
        auto read = [&](int base) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = CK_COLUMN(base, k);
                ck_restore8<VEC>(a.in, t, c, d, q[k], s[k]);
                dy[k] = ck_load8<T, VEC>(a.dy + t * a.ld_dy, c, d);
                if (a.d_res) res[k] = ck_load8<T, VEC>(a.d_res + t * a.ld_res, c, d);
            }
        };
        CK_SPANS(base, a.in.d) {
            if (WIDE) gain_of(base);
            read(base);
#pragma unroll
            for (int k = 0; k < VPT; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = ck_code(q[k], i) * s[k];
                    acc[k][0] = fmaf(x, x, acc[k][0]);
                    acc[k][1] = fmaf(x, ck_value<T>(dy[k], i) * g[k][i], acc[k][1]);
                }
        }
        ck_row_sum<2>(acc, sh, parity, sum);
        const float r = ck_rstd(sum[0], a.in.d, a.in.eps);
        const float f = r * r * r * (sum[1] / (float)a.in.d);
        CK_SPANS(base, a.in.d) {
            if (WIDE) {
                gain_of(base);
                read(base);
            }
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = ck_code(q[k], i) * s[k], e = ck_value<T>(dy[k], i) * r;
                    dg[k][i] = WIDE ? e * x : fmaf(e, x, dg[k][i]);
                    v[i] = fmaf(e, g[k][i], -x * f);
                    if (a.d_res) v[i] += ck_value<T>(res[k], i);
                }
                ck_store8<T, VEC>(a.dx + t * a.in.d, CK_COLUMN(base, k), d, ck_pack<T>(v));
            }
            if (WIDE) sums_to(base, !first);
        }
    }
    if (!WIDE) sums_to(0, false);
}

// d_gain: 32 columns a CTA, its eight warps every eighth row group, then the
// warps in their order.
__global__ void __launch_bounds__(256) ckpt_gain_sum_kernel(const float* __restrict__ part, int np, int d,
                                                            float* __restrict__ d_gain) {
    __shared__ float sh[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < d)
        for (int p = warp; p < np; p += 8) s += part[(int64_t)p * d + c];
    sh[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < d) {
        for (int w = 1; w < 8; ++w) s += sh[w][lane];
        d_gain[c] = s;
    }
}

}  // namespace aeth
