// adamw.cuh -- an AdamW step over many tensors at once, their moments in 32 or
// in 8 bits: what the low-rank step leaves (norm gains, biases, embeddings).
//
//   g = clip g      m = b1 m + (1 - b1) g      v = b2 v + ((1 - b2) g) g
//   p = p - lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + decay p)
//
// in fp32 (1 - b and the bias corrections from 64 bits), p rounded once to its
// type; with a master copy p is that copy's value, and the parameter its
// rounding.  Products and sums round one by one, so the moments' bits are those
// of the formula; the quotient is taken with the approximate square root and
// reciprocal (three units in the last place of an update that is some 1e-3 of p).
//
// The moments of all tensors lie one after the other, each tensor from a whole
// block of 2048 elements on.  8-bit moments are BLOCK_DYNAMIC's (codec.cuh): a
// code per element, a block's largest magnitude as its scale.  A block whose
// maximum is below 2^-126 is kept as zeros; one that holds a NaN or an infinity
// gets a NaN scale and stays NaN, as a 32-bit moment would.
//
// The tensors come as a table in the launch's parameters, so that gradients may
// lie elsewhere in every step and a captured step needs no memory of its own.
// Bound by its bytes: parameters, gradients and moments pass through once.
#pragma once
#include "adam.cuh"
#include "codec.cuh"
#include "pack8.cuh"

namespace aeth {

constexpr int kAdamwBlock = 2048;
// Tensors of one launch: the parameters of a launch take 32764 bytes.  A short
// list has a table of its own, which costs less to hand over.
constexpr int kAdamwTensors = 896, kAdamwFew = 64;
constexpr int64_t kAdamwStepBits = 40;  // of the step's word that count steps; above them, CTAs that have finished

struct AdamwTensor {
    void* p;
    const void* g;
    int64_t n;
    int first;  // of its blocks in this launch's order
    uint8_t p_dtype, g_dtype;
    uint8_t whole;  // p and g start on 16 bytes
    uint8_t decay;
};
template <int CAP>
struct AdamwArgs {
    AdamwTensor t[CAP];
    int at[CAP];  // first of its blocks among all moments
    int count, blocks;
    void *m, *v;
    float *m_scales, *v_scales;
    float* master;
    int64_t* step;
    const float* clip;  // or null: 1
    const float* lr_dev;  // or null
    float lr, eps, decay;
    double beta1, beta2;
    int last;  // of the step's launches: it counts the step
    uint32_t one;
};
static_assert(sizeof(AdamwArgs<kAdamwTensors>) <= 32764, "a launch's parameters");

// Eight elements of any type.  The first `have` exist; whole: 16-byte aligned.
__device__ __forceinline__ void adamw_load8(const void* p, int dtype, bool whole, int64_t i, int have, float (&v)[8]) {
    if (dtype == AETH_DTYPE_F32) {
        const float* q = static_cast<const float*>(p) + i;
        if (whole && have >= 8) {
            const float4 a = *reinterpret_cast<const float4*>(q), b = *reinterpret_cast<const float4*>(q + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < have ? q[k] : 0.0f;
        }
        return;
    }
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
    Pack8<__half> h;
    if (whole && have >= 8) {
        h.w[0] = *reinterpret_cast<const uint4*>(q);
    } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < have) w[k >> 1] |= (uint32_t)q[k] << (16 * (k & 1));
        h.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (dtype == AETH_DTYPE_F16) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ck_value<__half>(h, k);
    } else {
        const Pack8<__nv_bfloat16> b{{h.w[0]}};
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ck_value<__nv_bfloat16>(b, k);
    }
}
__device__ __forceinline__ void adamw_store8(void* p, int dtype, bool whole, int64_t i, int have, const float (&v)[8]) {
    if (dtype == AETH_DTYPE_F32) {
        float* q = static_cast<float*>(p) + i;
        if (whole && have >= 8) {
            *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(q + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < have) q[k] = v[k];
        }
        return;
    }
    const uint4 w = dtype == AETH_DTYPE_F16 ? ck_pack<__half>(v).w[0] : ck_pack<__nv_bfloat16>(v).w[0];
    uint16_t* q = static_cast<uint16_t*>(p) + i;
    if (whole && have >= 8) {
        *reinterpret_cast<uint4*>(q) = w;
    } else {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < have) q[k] = (uint16_t)(x[k >> 1] >> (16 * (k & 1)));
    }
}

// What a step's elements share.
struct AdamwScalars {
    float clip, lr, b1, b2, omb1, omb2, first, second, eps, decay;
};
// 1 / (1 - b^t), b^t by squaring
__device__ __forceinline__ float adamw_correction(double b, int64_t t) {
    double p = 1.0;
    for (; t > 0; t >>= 1, b *= b)
        if (t & 1) p *= b;
    return (float)(1.0 / (1.0 - p));
}
// By all threads of the CTA; ends with a barrier.
template <int CAP>
__device__ __forceinline__ AdamwScalars adamw_scalars(const AdamwArgs<CAP>& a, float* shared2) {
    if (threadIdx.x == 0 || threadIdx.x == 32) {
        const int64_t t = (*(volatile const int64_t*)a.step & ((1ll << kAdamwStepBits) - 1)) + 1;
        shared2[threadIdx.x >> 5] = adamw_correction(threadIdx.x ? a.beta2 : a.beta1, t);
    }
    AdamwScalars s;
    s.clip = a.clip ? *a.clip : 1.0f;
    s.lr = a.lr_dev ? *a.lr_dev : a.lr;
    s.b1 = (float)a.beta1;
    s.b2 = (float)a.beta2;
    s.omb1 = (float)(1.0 - a.beta1);
    s.omb2 = (float)(1.0 - a.beta2);
    s.eps = a.eps;
    s.decay = a.decay;
    __syncthreads();
    s.first = shared2[0];
    s.second = shared2[1];
    return s;
}
// The CTA that ends last counts the step.  Every CTA has read the step's low
// bits before it adds to the high ones.
template <int CAP>
__device__ __forceinline__ void adamw_count(const AdamwArgs<CAP>& a) {
    __syncthreads();
    if (threadIdx.x != 0 || !a.last) return;
    const unsigned long long was = atomicAdd(reinterpret_cast<unsigned long long*>(a.step), 1ull << kAdamwStepBits);
    if ((was >> kAdamwStepBits) == gridDim.x - 1)
        *(volatile int64_t*)a.step = (int64_t)(was & ((1ull << kAdamwStepBits) - 1)) + 1;
}
// The tensor of a block of the launch: the last that starts at or before it.
template <int CAP>
__device__ __forceinline__ int adamw_tensor(const AdamwArgs<CAP>& a, int block) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].first <= block) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ float adamw_sqrt(float x) {
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float adamw_rcp(float x) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void adamw_moments(const AdamwScalars& s, float g, float& m, float& v) {
    g = __fmul_rn(g, s.clip);
    m = __fadd_rn(__fmul_rn(s.b1, m), __fmul_rn(s.omb1, g));
    v = __fadd_rn(__fmul_rn(s.b2, v), __fmul_rn(__fmul_rn(s.omb2, g), g));
}
__device__ __forceinline__ float adamw_param(const AdamwScalars& s, float decay, float p, float m, float v) {
    const float u = m * s.first * adamw_rcp(adamw_sqrt(v * s.second) + s.eps);
    return p - s.lr * (u + decay * p);
}

// Moments in 32 bits: a CTA takes blocks, a thread eight elements of one.
template <int CAP, bool MASTER>
__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ AdamwArgs<CAP> a) {
    __shared__ float corr[2];
    const AdamwScalars s = adamw_scalars(a, corr);
    for (int b = blockIdx.x; b < a.blocks; b += gridDim.x) {
        const int i = adamw_tensor(a, b);
        const AdamwTensor& t = a.t[i];
        const int64_t e = (int64_t)(b - t.first) * kAdamwBlock + threadIdx.x * 8;
        const int64_t o = ((int64_t)a.at[i] + (b - t.first)) * kAdamwBlock + threadIdx.x * 8;
        const int have = (int)min(t.n - e, (int64_t)8);
        if (have <= 0) continue;
        float p[8], g[8], m[8], v[8];
        adamw_load8(t.g, t.g_dtype, t.whole, e, have, g);
        if (MASTER) adamw_load8(a.master, AETH_DTYPE_F32, true, o, 8, p);
        else adamw_load8(t.p, t.p_dtype, t.whole, e, have, p);
        adamw_load8(a.m, AETH_DTYPE_F32, true, o, 8, m);
        adamw_load8(a.v, AETH_DTYPE_F32, true, o, 8, v);
        const float decay = t.decay ? s.decay : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            adamw_moments(s, g[k], m[k], v[k]);
            p[k] = adamw_param(s, decay, p[k], m[k], v[k]);
        }
        if (MASTER) adamw_store8(a.master, AETH_DTYPE_F32, true, o, have, p);
        adamw_store8(t.p, t.p_dtype, t.whole, e, have, p);
        adamw_store8(a.m, AETH_DTYPE_F32, true, o, have, m);
        adamw_store8(a.v, AETH_DTYPE_F32, true, o, have, v);
    }
    adamw_count(a);
}

// Moments in 8 bits.  A CTA is four groups of 256 threads that share the maps
// and the encode's tables (the layout of b2_adam_dyn_kernel: each map entry in
// 32 copies, so that no lookup of a warp meets a bank conflict); a group takes a
// block, a thread eight of its elements.
constexpr int kAdamw8Threads = 1024;
constexpr int kAdamw8Dec = 256 * 256;
constexpr int kAdamw8Shared = kAdamw8Dec + (2 * kDmapLutEntries + kDmapLutUEntries) * 4;

template <int CAP, bool MASTER>
__global__ void __launch_bounds__(kAdamw8Threads, 1) adamw8_kernel(const __grid_constant__ AdamwArgs<CAP> a) {
    extern __shared__ __align__(16) uint8_t adamw_smem[];
    float* dec = reinterpret_cast<float*>(adamw_smem);
    uint32_t* lut_s = reinterpret_cast<uint32_t*>(adamw_smem + kAdamw8Dec);
    uint32_t* lut_u = lut_s + 2 * kDmapLutEntries;
    __shared__ float corr[2];
    __shared__ uint32_t red[4][2][2][8];  // [group][block parity][m, v][warp]: maxima, NaN above all
    for (int i = threadIdx.x; i < 256 * 64; i += blockDim.x)
        dec[i] = (i & 63) < 32 ? c_dmap_signed[i >> 6] : c_dmap_unsigned[i >> 6];
    for (int i = threadIdx.x; i < 2 * kDmapLutEntries; i += blockDim.x) lut_s[i] = g_dmap_lut4_s[i];
    for (int i = threadIdx.x; i < kDmapLutUEntries; i += blockDim.x) lut_u[i] = g_dmap_lut4_u[i];
    const AdamwScalars s = adamw_scalars(a, corr);
    const int grp = threadIdx.x >> 8, tid = threadIdx.x & 255, lane = tid & 31, warp = tid >> 5;
    const uint32_t m1 = a.one << 1, m8 = a.one << 8, m15 = a.one << 15, m16 = a.one << 16;
    const uint32_t dec_base = smem_u32_addr(dec), off_m = (uint32_t)lane * 4u, off_v = off_m + 128u;
    const uint32_t adj_s = smem_u32_addr(lut_s) - (uint32_t)(kDmapLutExpLo << kDmapLutLog2P) * 4u;
    const uint32_t adj_u = smem_u32_addr(lut_u) - (uint32_t)(kDmapLutExpLo << kDmapLutULog2P) * 4u;
    int8_t *m_all = static_cast<int8_t*>(a.m), *v_all = static_cast<int8_t*>(a.v);
    int par = 0;
    for (int b = blockIdx.x * 4 + grp; b < a.blocks; b += gridDim.x * 4, par ^= 1) {
        const int i = adamw_tensor(a, b);
        const AdamwTensor& t = a.t[i];
        const int64_t blk = (int64_t)a.at[i] + (b - t.first);
        const int64_t e = (int64_t)(b - t.first) * kAdamwBlock + tid * 8, o = blk * kAdamwBlock + tid * 8;
        const int have = (int)max(min(t.n - e, (int64_t)8), (int64_t)0);
        const float sm = a.m_scales[blk], sv = a.v_scales[blk];
        const uint2 qm = *reinterpret_cast<const uint2*>(m_all + o), qv = *reinterpret_cast<const uint2*>(v_all + o);
        float p[8], g[8], m[8], v[8], am = 0.0f, av = 0.0f;
        adamw_load8(t.g, t.g_dtype, t.whole, e, have, g);
        if (MASTER) adamw_load8(a.master, AETH_DTYPE_F32, true, o, 8, p);
        else adamw_load8(t.p, t.p_dtype, t.whole, e, have, p);
        const float decay = t.decay ? s.decay : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t sel = 0x5504u | ((uint32_t)(k & 3) << 4);
            m[k] = __fmul_rn(__uint_as_float(lds_u32(dec_base + prmt(k < 4 ? qm.x : qm.y, off_m, sel))), sm);
            v[k] = __fmul_rn(__uint_as_float(lds_u32(dec_base + prmt(k < 4 ? qv.x : qv.y, off_v, sel))), sv);
            adamw_moments(s, g[k], m[k], v[k]);
            p[k] = adamw_param(s, decay, p[k], m[k], v[k]);
            if (k >= have) m[k] = v[k] = 0.0f;  // past the tensor's end: codes of zero
            am = fmax3_nan(am, fabsf(m[k]), 0.0f);
            av = fmax3_nan(av, v[k], 0.0f);
        }
        if (MASTER) adamw_store8(a.master, AETH_DTYPE_F32, true, o, have, p);
        adamw_store8(t.p, t.p_dtype, t.whole, e, have, p);
        // non-negative or NaN (0x7fffffff): their bits order as they do
        const uint32_t wm = __reduce_max_sync(0xffffffffu, __float_as_uint(am));
        const uint32_t wv = __reduce_max_sync(0xffffffffu, __float_as_uint(av));
        if (lane == 0) {
            red[grp][par][0][warp] = wm;
            red[grp][par][1][warp] = wv;
        }
        group_bar(1 + grp);  // the parity's slots are written again two blocks later
        const uint32_t bm = __reduce_max_sync(0xffffffffu, red[grp][par][0][lane & 7]);
        const uint32_t bv = __reduce_max_sync(0xffffffffu, red[grp][par][1][lane & 7]);
        const bool bad_m = bm >= 0x7f800000u, bad_v = bv >= 0x7f800000u;
        const float nm = bad_m || bm < 0x00800000u ? 0.0f : __uint_as_float(bm);
        const float nv = bad_v || bv < 0x00800000u ? 0.0f : __uint_as_float(bv);
        const float im = dyn_inv(nm), iv = dyn_inv(nv);
        uint32_t cm[8], cv[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            cm[k] = dmap_enc4_s(adj_s, nm > 0.0f ? dyn_xn(m[k], im) : 0.0f, m1, m8, m15);
            cv[k] = dmap_enc4_u(adj_u, nv > 0.0f ? dyn_xn(v[k], iv) : 0.0f, m8, m16);
        }
        uint2 om, ov;
        om.x = prmt(prmt(cm[0], cm[1], 0x3340u), prmt(cm[2], cm[3], 0x3340u), 0x5410u);
        om.y = prmt(prmt(cm[4], cm[5], 0x3340u), prmt(cm[6], cm[7], 0x3340u), 0x5410u);
        ov.x = prmt(prmt(cv[0], cv[1], 0x3340u), prmt(cv[2], cv[3], 0x3340u), 0x5410u);
        ov.y = prmt(prmt(cv[4], cv[5], 0x3340u), prmt(cv[6], cv[7], 0x3340u), 0x5410u);
        *reinterpret_cast<uint2*>(m_all + o) = om;
        *reinterpret_cast<uint2*>(v_all + o) = ov;
        if (tid == 0) {
            a.m_scales[blk] = bad_m ? __int_as_float(0x7fc00000) : nm;
            a.v_scales[blk] = bad_v ? __int_as_float(0x7fc00000) : nv;
        }
    }
    adamw_count(a);
}

// 8-bit moments as the values that they stand for: a thread takes 16 codes.
__global__ void __launch_bounds__(256) adamw_decode_kernel(const int8_t* __restrict__ m, const int8_t* __restrict__ v,
                                                           const float* __restrict__ ms, const float* __restrict__ vs,
                                                           int64_t n16, float* __restrict__ m_out, float* __restrict__ v_out) {
    __shared__ float dec[2][256];
    for (int i = threadIdx.x; i < 256; i += 256) {
        dec[0][i] = c_dmap_signed[i];
        dec[1][i] = c_dmap_unsigned[i];
    }
    __syncthreads();
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n16; i += gridDim.x * 256ll) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint4 q = ck_stream(reinterpret_cast<const uint4*>(w ? v : m) + i);
            const float s = (w ? vs : ms)[i / (kAdamwBlock / 16)];
            const uint32_t c[4] = {q.x, q.y, q.z, q.w};
            float4* o = reinterpret_cast<float4*>(w ? v_out : m_out) + i * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                o[k] = make_float4(__fmul_rn(dec[w][c[k] & 255u], s), __fmul_rn(dec[w][c[k] >> 8 & 255u], s),
                                   __fmul_rn(dec[w][c[k] >> 16 & 255u], s), __fmul_rn(dec[w][c[k] >> 24], s));
        }
    }
}

}  // namespace aeth
