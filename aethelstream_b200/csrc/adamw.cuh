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
#include <type_traits>

#include "adam.cuh"
#include "codec.cuh"
#include "pack8.cuh"

namespace aeth {

constexpr int kAdamwBlock = 2048;
// Tensors of one launch, whose parameters take 32764 bytes at most.  Handing a table
// over costs the host 0.5 us a kilobyte (a launch of 161 gains 22.7 us with 29 KB, 7 with 2),
// so short lists have shorter ones.
constexpr int kAdamwTensors = 768, kAdamwSome = 256, kAdamwFew = 64;
constexpr int kAdamwStarts = 888;  // walkers over the blocks (CTAs, or groups of them), at most
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
    uint16_t start[kAdamwStarts];  // the tensor of each walker's first block
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

// N 16-bit elements as floats, and back
template <int N>
__device__ __forceinline__ void adamw_floats(const uint32_t (&w)[N / 2], int dtype, float (&v)[N]) {
    if (dtype == AETH_DTYPE_F16) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[k / 2]));
            v[k] = x.x;
            v[k + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            v[k] = __uint_as_float(w[k / 2] << 16);
            v[k + 1] = __uint_as_float(w[k / 2] & 0xffff0000u);
        }
    }
}
template <int N>
__device__ __forceinline__ void adamw_words(const float (&v)[N], int dtype, uint32_t (&w)[N / 2]) {
    if (dtype == AETH_DTYPE_F16) {
#pragma unroll
        for (int k = 0; k < N; k += 2) w[k / 2] = ck_pack2<__half>(v[k], v[k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 2) w[k / 2] = ck_pack2<__nv_bfloat16>(v[k], v[k + 1]);
    }
}

// N elements (4 or 8) of any type as they lie in memory, the first `have` of which
// exist; whole: they start on as many bytes as they take, 16 at most.  Read and
// turned into floats apart, so that no read waits for another.
template <int N>
struct AdamwRaw {
    uint32_t w[N];
    __device__ __forceinline__ void load(const void* p, int dtype, bool whole, int64_t i, int have) {
        if (dtype == AETH_DTYPE_F32) {
            const uint32_t* q = static_cast<const uint32_t*>(p) + i;
            if (whole && have >= N) {
#pragma unroll
                for (int k = 0; k < N; k += 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(q + k);
                    w[k] = x.x; w[k + 1] = x.y; w[k + 2] = x.z; w[k + 3] = x.w;
                }
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k) w[k] = k < have ? q[k] : 0u;
            }
            return;
        }
        const uint16_t* q = static_cast<const uint16_t*>(p) + i;
        if (whole && have >= N) {
            if constexpr (N == 8) {
                const uint4 x = *reinterpret_cast<const uint4*>(q);
                w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(q);
                w[0] = x.x; w[1] = x.y;
            }
        } else {
#pragma unroll
            for (int k = 0; k < N; k += 2)
                w[k / 2] = (k < have ? (uint32_t)q[k] : 0u) | (k + 1 < have ? (uint32_t)q[k + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ void floats(int dtype, float (&v)[N]) const {
        if (dtype == AETH_DTYPE_F32) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = __uint_as_float(w[k]);
        } else {
            uint32_t x[N / 2];
#pragma unroll
            for (int k = 0; k < N / 2; ++k) x[k] = w[k];
            adamw_floats<N>(x, dtype, v);
        }
    }
};
template <int N>
__device__ __forceinline__ void adamw_load(const void* p, int dtype, bool whole, int64_t i, int have, float (&v)[N]) {
    AdamwRaw<N> r;
    if (dtype == AETH_DTYPE_F32) {
        r.load(p, AETH_DTYPE_F32, whole, i, have);
        r.floats(AETH_DTYPE_F32, v);
    } else {
        r.load(p, AETH_DTYPE_F16, whole, i, have);
        uint32_t x[N / 2];
#pragma unroll
        for (int k = 0; k < N / 2; ++k) x[k] = r.w[k];
        adamw_floats<N>(x, dtype, v);
    }
}
template <int N>
__device__ __forceinline__ void adamw_store(void* p, int dtype, bool whole, int64_t i, int have, const float (&v)[N]) {
    if (dtype == AETH_DTYPE_F32) {
        float* q = static_cast<float*>(p) + i;
        if (whole && have >= N) {
#pragma unroll
            for (int k = 0; k < N; k += 4) *reinterpret_cast<float4*>(q + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (k < have) q[k] = v[k];
        }
        return;
    }
    uint32_t w[N / 2];
    adamw_words<N>(v, dtype, w);
    uint16_t* q = static_cast<uint16_t*>(p) + i;
    if (whole && have >= N) {
        if constexpr (N == 8) *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < have) q[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    }
}

// What a step's elements share.
struct AdamwScalars {
    float clip, lr, b1, b2, omb1, omb2, first, root, eps, decay;  // root: of v's correction
    bool flush;  // eps is so large that root times 2^-63 does not count beside it (2^-23 of it)
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
    s.root = sqrtf(shared2[1]);
    s.flush = a.eps >= 1e-12f * s.root;
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
// The tensor of a block of the launch: the last that starts at or before it.  `i`:
// that of an earlier block, and often of this one too.
template <int CAP>
__device__ __forceinline__ int adamw_tensor(const AdamwArgs<CAP>& a, int block, int i) {
    if (i + 1 >= a.count || a.t[i + 1].first > block) return i;
    int lo = i + 1, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].first <= block) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// 1 / (root sqrt(v) + eps) of two, subnormal numbers flushed to 0 or not.  The correction's
// root, since the corrected v may lie past the largest float, or among the subnormal ones.
template <bool FLUSH>
__device__ __forceinline__ float2 adamw_scale(float x, float y, float2 root, float2 eps) {
    float a, b;
    if (FLUSH) {
        asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(x));
        asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(y));
    } else {
        asm("sqrt.approx.f32 %0, %1;" : "=f"(a) : "f"(x));
        asm("sqrt.approx.f32 %0, %1;" : "=f"(b) : "f"(y));
    }
    float2 r = fma2_rn(make_float2(a, b), root, eps);
    if (FLUSH) {
        asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r.x));
        asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r.y));
    } else {
        asm("rcp.approx.f32 %0, %0;" : "+f"(r.x));
        asm("rcp.approx.f32 %0, %0;" : "+f"(r.y));
    }
    return r;
}
// New moments from the old ones of N elements, in pairs: the products of two in
// one instruction, the sums one by one (common.cuh, add2_sep).
template <int N>
__device__ __forceinline__ void adamw_moments(const AdamwScalars& s, const float (&g)[N], float (&m)[N], float (&v)[N]) {
    const float2 clip = make_float2(s.clip, s.clip), b1 = make_float2(s.b1, s.b1), b2 = make_float2(s.b2, s.b2);
    const float2 omb1 = make_float2(s.omb1, s.omb1), omb2 = make_float2(s.omb2, s.omb2);
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        const float2 gg = mul2_rn(make_float2(g[k], g[k + 1]), clip);
        const float2 mm = add2_sep(mul2_rn(b1, make_float2(m[k], m[k + 1])), mul2_rn(omb1, gg));
        const float2 vv = add2_sep(mul2_rn(b2, make_float2(v[k], v[k + 1])), mul2_rn(mul2_rn(omb2, gg), gg));
        m[k] = mm.x;
        m[k + 1] = mm.y;
        v[k] = vv.x;
        v[k + 1] = vv.y;
    }
}
// The parameters' step from the new moments
template <int N, bool FLUSH>
__device__ __forceinline__ void adamw_params(const AdamwScalars& s, float decay, const float (&m)[N], const float (&v)[N],
                                             float (&p)[N]) {
    const float2 first = make_float2(s.first, s.first), root = make_float2(s.root, s.root), eps = make_float2(s.eps, s.eps);
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        const float2 mm = mul2_rn(make_float2(m[k], m[k + 1]), first);
        const float2 x = adamw_scale<FLUSH>(v[k], v[k + 1], root, eps);
        p[k] -= s.lr * fmaf(mm.x, x.x, decay * p[k]);
        p[k + 1] -= s.lr * fmaf(mm.y, x.y, decay * p[k + 1]);
    }
}
template <int N>
__device__ __forceinline__ void adamw_params(const AdamwScalars& s, float decay, const float (&m)[N], const float (&v)[N],
                                             float (&p)[N]) {
    if (s.flush) adamw_params<N, true>(s, decay, m, v, p);
    else adamw_params<N, false>(s, decay, m, v, p);
}

// Moments in 32 bits: a CTA takes blocks, a thread four elements of each half of
// one, so that a warp's accesses of any type are whole.
template <int CAP>
__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ AdamwArgs<CAP> a) {
    __shared__ float corr[2];
    const AdamwScalars s = adamw_scalars(a, corr);
    int i = a.start[blockIdx.x];
    for (int b = blockIdx.x; b < a.blocks; b += gridDim.x) {
        if (b != (int)blockIdx.x) i = adamw_tensor(a, b, i);
        const AdamwTensor& t = a.t[i];
        const int64_t e0 = (int64_t)(b - t.first) * kAdamwBlock + threadIdx.x * 4;
        const int64_t o0 = ((int64_t)a.at[i] + (b - t.first)) * kAdamwBlock + threadIdx.x * 4;
        AdamwRaw<4> p[2], g[2], m[2], v[2];
        int have[2];
        const int p_dtype = a.master ? AETH_DTYPE_F32 : t.p_dtype;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int64_t e = e0 + q * (kAdamwBlock / 2), o = o0 + q * (kAdamwBlock / 2);
            have[q] = (int)min(t.n - e, (int64_t)4);
            if (have[q] <= 0) continue;
            m[q].load(a.m, AETH_DTYPE_F32, true, o, 4);
            v[q].load(a.v, AETH_DTYPE_F32, true, o, 4);
            p[q].load(a.master ? a.master : t.p, p_dtype, a.master || t.whole, a.master ? o : e, a.master ? 4 : have[q]);
            g[q].load(t.g, t.g_dtype, t.whole, e, have[q]);
        }
        const float decay = t.decay ? s.decay : 0.0f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int64_t e = e0 + q * (kAdamwBlock / 2), o = o0 + q * (kAdamwBlock / 2);
            if (have[q] <= 0) continue;
            float pf[4], gf[4], mf[4], vf[4];
            g[q].floats(t.g_dtype, gf);
            m[q].floats(AETH_DTYPE_F32, mf);
            v[q].floats(AETH_DTYPE_F32, vf);
            p[q].floats(p_dtype, pf);
            adamw_moments<4>(s, gf, mf, vf);
            adamw_params<4>(s, decay, mf, vf, pf);
            if (a.master) adamw_store<4>(a.master, AETH_DTYPE_F32, true, o, have[q], pf);
            adamw_store<4>(t.p, t.p_dtype, t.whole, e, have[q], pf);
            adamw_store<4>(a.m, AETH_DTYPE_F32, true, o, have[q], mf);
            adamw_store<4>(a.v, AETH_DTYPE_F32, true, o, have[q], vf);
        }
    }
    adamw_count(a);
}

// Moments in 8 bits.  A CTA is some groups of 128 threads that share the maps and
// the encode's tables (the layout of b2_adam_dyn_kernel: each map entry in 32
// copies, so that no lookup of a warp meets a bank conflict); a group takes a
// block, a thread eight elements of each of its halves.  A block's 16-bit gradients
// and parameters and its codes are fetched while the one before it is encoded.
// FAST, where all parameters and gradients of the launch are bf16, without a master
// copy: whole blocks go without a branch on types and ends for every eight elements,
// in four groups, whose registers that takes.  Else five, for what is not fetched
// ahead.  2^27 elements: bf16 288 us (4.66 TB/s) fast, 316 in the other; f32 498 in
// the other, 553 in four groups.  Bound by instructions (some 60 an element, issue
// slots 75 % taken), most of them for the two encodes.
template <bool FAST>
constexpr int adamw8_groups() { return FAST ? 4 : 5; }
constexpr int kAdamw8Dec = 256 * 256;
constexpr int kAdamw8Shared = kAdamw8Dec + (2 * kDmapLutEntries + kDmapLutUEntries) * 4;
constexpr int kAdamwHalf = kAdamwBlock / 2;

template <int CAP, bool FAST>
__global__ void __launch_bounds__(128 * adamw8_groups<FAST>(), 1) adamw8_kernel(const __grid_constant__ AdamwArgs<CAP> a) {
    constexpr int kAdamw8Groups = adamw8_groups<FAST>();
    extern __shared__ __align__(16) uint8_t adamw_smem[];
    float* dec = reinterpret_cast<float*>(adamw_smem);
    uint32_t* lut_s = reinterpret_cast<uint32_t*>(adamw_smem + kAdamw8Dec);
    uint32_t* lut_u = lut_s + 2 * kDmapLutEntries;
    __shared__ float corr[2];
    __shared__ uint32_t red[kAdamw8Groups][2][2][4];  // [group][block parity][m, v][warp]: maxima, NaN above all
    for (int i = threadIdx.x; i < 256 * 64; i += blockDim.x)
        dec[i] = (i & 63) < 32 ? c_dmap_signed[i >> 6] : c_dmap_unsigned[i >> 6];
    for (int i = threadIdx.x; i < 2 * kDmapLutEntries; i += blockDim.x) lut_s[i] = g_dmap_lut4_s[i];
    for (int i = threadIdx.x; i < kDmapLutUEntries; i += blockDim.x) lut_u[i] = g_dmap_lut4_u[i];
    const AdamwScalars s = adamw_scalars(a, corr);
    const int grp = threadIdx.x >> 7, tid = threadIdx.x & 127, lane = tid & 31, warp = tid >> 5;
    const uint32_t m1 = a.one << 1, m8 = a.one << 8, m15 = a.one << 15, m16 = a.one << 16;
    const uint32_t dec_base = smem_u32_addr(dec), off_m = (uint32_t)lane * 4u, off_v = off_m + 128u;
    const uint32_t adj_s = smem_u32_addr(lut_s) - (uint32_t)(kDmapLutExpLo << kDmapLutLog2P) * 4u;
    const uint32_t adj_u = smem_u32_addr(lut_u) - (uint32_t)(kDmapLutExpLo << kDmapLutULog2P) * 4u;
    int8_t *m_all = static_cast<int8_t*>(a.m), *v_all = static_cast<int8_t*>(a.v);
    const int walker = blockIdx.x * kAdamw8Groups + grp, step = gridDim.x * kAdamw8Groups;
    int i = a.start[walker], par = 0;
    int64_t e = 0, o = 0, blk = 0;  // this thread's first element, in its tensor and among the moments; its block
    bool p16 = false, g16 = false, fast16 = false;  // fetched ahead; both, by the whole warp, and both bf16
    uint4 pw[2], gw[2];
    uint2 qm[2], qv[2];
    float sm = 0.0f, sv = 0.0f;
    auto fetch = [&](int b) {
        if (b != walker) i = adamw_tensor(a, b, i);
        const AdamwTensor& t = a.t[i];
        const int64_t at = (int64_t)(b - t.first);
        blk = a.at[i] + at;
        e = at * kAdamwBlock + tid * 8;
        o = blk * kAdamwBlock + tid * 8;
        const bool whole = t.whole && e + kAdamwHalf + 8 <= t.n;
        p16 = whole && t.p_dtype != AETH_DTYPE_F32 && !a.master;
        g16 = whole && t.g_dtype != AETH_DTYPE_F32;
        if (FAST) fast16 = __all_sync(0xffffffffu, p16 && g16 && s.flush && t.p_dtype == AETH_DTYPE_BF16 && t.g_dtype == AETH_DTYPE_BF16);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (g16) gw[q] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(t.g) + e + q * kAdamwHalf);
            if (p16) pw[q] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(t.p) + e + q * kAdamwHalf);
            qm[q] = *reinterpret_cast<const uint2*>(m_all + o + q * kAdamwHalf);
            qv[q] = *reinterpret_cast<const uint2*>(v_all + o + q * kAdamwHalf);
        }
        sm = a.m_scales[blk];
        sv = a.v_scales[blk];
    };
    if (walker < a.blocks) fetch(walker);
    for (int b = walker; b < a.blocks; b += step, par ^= 1) {
        const AdamwTensor& t = a.t[i];
        const int64_t oo = o, bb = blk;
        float m[2][8], v[2][8], am = 0.0f, av = 0.0f;
        const float2 sm2 = make_float2(sm, sm), sv2 = make_float2(sv, sv);
        const float decay = t.decay ? s.decay : 0.0f;
        auto update = [&](auto fast) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int64_t eq = e + q * kAdamwHalf;
                const int have = fast.value ? 8 : (int)max(min(t.n - eq, (int64_t)8), (int64_t)0);
                float g[8], p[8];
                if (fast.value || g16) {
                    const uint32_t w[4] = {gw[q].x, gw[q].y, gw[q].z, gw[q].w};
                    adamw_floats<8>(w, fast.value ? (int)AETH_DTYPE_BF16 : t.g_dtype, g);
                } else {
                    adamw_load<8>(t.g, t.g_dtype, t.whole, eq, have, g);
                }
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const uint32_t sel = 0x5504u | ((uint32_t)(k & 3) << 4);
                    const uint32_t wm = k < 4 ? qm[q].x : qm[q].y, wv = k < 4 ? qv[q].x : qv[q].y;
                    const float2 mm = mul2_rn(make_float2(__uint_as_float(lds_u32(dec_base + prmt(wm, off_m, sel))),
                                                          __uint_as_float(lds_u32(dec_base + prmt(wm, off_m, sel + 0x10u)))), sm2);
                    const float2 vv = mul2_rn(make_float2(__uint_as_float(lds_u32(dec_base + prmt(wv, off_v, sel))),
                                                          __uint_as_float(lds_u32(dec_base + prmt(wv, off_v, sel + 0x10u)))), sv2);
                    m[q][k] = mm.x;
                    m[q][k + 1] = mm.y;
                    v[q][k] = vv.x;
                    v[q][k + 1] = vv.y;
                }
                adamw_moments<8>(s, g, m[q], v[q]);
                if (fast.value || p16) {
                    const int dtype = fast.value ? (int)AETH_DTYPE_BF16 : t.p_dtype;
                    uint32_t w[4] = {pw[q].x, pw[q].y, pw[q].z, pw[q].w};
                    adamw_floats<8>(w, dtype, p);
                    if (fast.value) adamw_params<8, true>(s, decay, m[q], v[q], p);
                    else adamw_params<8>(s, decay, m[q], v[q], p);
                    adamw_words<8>(p, dtype, w);
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(t.p) + eq) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    if (a.master) adamw_load<8>(a.master, AETH_DTYPE_F32, true, o + q * kAdamwHalf, 8, p);
                    else adamw_load<8>(t.p, t.p_dtype, t.whole, eq, have, p);
                    adamw_params<8>(s, decay, m[q], v[q], p);
                    if (a.master) adamw_store<8>(a.master, AETH_DTYPE_F32, true, o + q * kAdamwHalf, have, p);
                    adamw_store<8>(t.p, t.p_dtype, t.whole, eq, have, p);
                }
                if (!fast.value && have < 8)  // past the tensor's end: codes of zero
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k >= have) m[q][k] = v[q][k] = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    am = fmax3_nan(am, fabsf(m[q][k]), fabsf(m[q][k + 1]));
                    av = fmax3_nan(av, v[q][k], v[q][k + 1]);
                }
            }
        };
        if (FAST && fast16) update(std::true_type());
        else update(std::false_type());
        if (b + step < a.blocks) fetch(b + step);
        // non-negative or NaN (0x7fffffff): their bits order as they do
        const uint32_t wm = __reduce_max_sync(0xffffffffu, __float_as_uint(am));
        const uint32_t wv = __reduce_max_sync(0xffffffffu, __float_as_uint(av));
        if (lane == 0) {
            red[grp][par][0][warp] = wm;
            red[grp][par][1][warp] = wv;
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");  // the parity's slots are written again two blocks later
        const uint32_t* rm = red[grp][par][0];
        const uint32_t* rv = red[grp][par][1];
        const uint32_t bm = max(max(rm[0], rm[1]), max(rm[2], rm[3])), bv = max(max(rv[0], rv[1]), max(rv[2], rv[3]));
        const bool bad_m = bm >= 0x7f800000u, bad_v = bv >= 0x7f800000u;
        const float nm = bad_m || bm < 0x00800000u ? 0.0f : __uint_as_float(bm);
        const float nv = bad_v || bv < 0x00800000u ? 0.0f : __uint_as_float(bv);
        // 0: codes of zero (of NaN too: the scale says NaN)
        const float im = dyn_inv(nm), iv = dyn_inv(nv);
        const float2 im2 = make_float2(im, im), iv2 = make_float2(iv, iv);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            uint32_t cm[8], cv[8];
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                const float2 mm = mul2_rn(make_float2(m[q][k], m[q][k + 1]), im2);
                const float2 vv = mul2_rn(make_float2(v[q][k], v[q][k + 1]), iv2);
                cm[k] = dmap_enc4_s(adj_s, mm.x, m1, m8, m15);
                cm[k + 1] = dmap_enc4_s(adj_s, mm.y, m1, m8, m15);
                cv[k] = dmap_enc4_u(adj_u, vv.x, m8, m16);
                cv[k + 1] = dmap_enc4_u(adj_u, vv.y, m8, m16);
            }
            uint2 om, ov;
            om.x = prmt(prmt(cm[0], cm[1], 0x3340u), prmt(cm[2], cm[3], 0x3340u), 0x5410u);
            om.y = prmt(prmt(cm[4], cm[5], 0x3340u), prmt(cm[6], cm[7], 0x3340u), 0x5410u);
            ov.x = prmt(prmt(cv[0], cv[1], 0x3340u), prmt(cv[2], cv[3], 0x3340u), 0x5410u);
            ov.y = prmt(prmt(cv[4], cv[5], 0x3340u), prmt(cv[6], cv[7], 0x3340u), 0x5410u);
            *reinterpret_cast<uint2*>(m_all + oo + q * kAdamwHalf) = om;
            *reinterpret_cast<uint2*>(v_all + oo + q * kAdamwHalf) = ov;
        }
        if (tid == 0) {
            a.m_scales[bb] = bad_m ? __int_as_float(0x7fc00000) : nm;
            a.v_scales[bb] = bad_v ? __int_as_float(0x7fc00000) : nv;
        }
    }
    adamw_count(a);
}

// 8-bit moments as the values that they stand for, m's and v's by CTAs of their
// own: a thread takes four codes and sixteen bytes of values, eight times.  Each
// map entry in eight copies (32 would leave no conflict, and cost the CTAs' start).
constexpr int kAdamwDecode = 8;
__global__ void __launch_bounds__(256) adamw_decode_kernel(const int8_t* __restrict__ m, const int8_t* __restrict__ v,
                                                           const float* __restrict__ ms, const float* __restrict__ vs,
                                                           int64_t n4, float* __restrict__ m_out, float* __restrict__ v_out) {
    __shared__ float dec[256 * 8];
    const bool second = blockIdx.y != 0;
    for (int i = threadIdx.x; i < 256 * 8; i += 256) dec[i] = second ? c_dmap_unsigned[i >> 3] : c_dmap_signed[i >> 3];
    __syncthreads();
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(second ? v : m);
    const float* scales = second ? vs : ms;
    float4* out = reinterpret_cast<float4*>(second ? v_out : m_out);
    const float* mine = dec + (threadIdx.x & 7);
    for (int64_t i0 = blockIdx.x * 256ll * kAdamwDecode + threadIdx.x; i0 < n4; i0 += gridDim.x * 256ll * kAdamwDecode) {
        uint32_t c[kAdamwDecode];
        float s[kAdamwDecode];
#pragma unroll
        for (int k = 0; k < kAdamwDecode; ++k) {  // n4 is a multiple of 512
            const int64_t i = i0 + 256 * k;
            c[k] = i < n4 ? __ldcs(codes + i) : 0u;
            s[k] = i < n4 ? __ldg(scales + i / (kAdamwBlock / 4)) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kAdamwDecode; ++k) {
            const int64_t i = i0 + 256 * k;
            if (i < n4)
                out[i] = make_float4(__fmul_rn(mine[(c[k] & 255u) * 8], s[k]), __fmul_rn(mine[(c[k] >> 8 & 255u) * 8], s[k]),
                                     __fmul_rn(mine[(c[k] >> 16 & 255u) * 8], s[k]), __fmul_rn(mine[(c[k] >> 24) * 8], s[k]));
        }
    }
}

}  // namespace aeth
