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
#include "pack8.cuh"
#include "umma.cuh"

namespace aeth {

constexpr int kCkptBlock = 128;

// Eight features from a row in shared memory.
template <typename T>
__device__ __forceinline__ Pack8<T> ck_shared8(const uint8_t* row, int c) {
    Pack8<T> p;
#pragma unroll
    for (int k = 0; k < Pack8<T>::kWords; ++k) p.w[k] = reinterpret_cast<const uint4*>(row + (size_t)c * sizeof(T))[k];
    return p;
}

// Makes the second pass over a row unpack its values again: kept unpacked
// across the barrier they would take two to four times the registers.
__device__ __forceinline__ void ck_opaque(uint2& q) { asm volatile("" : "+r"(q.x), "+r"(q.y)::"memory"); }
template <typename T>
__device__ __forceinline__ void ck_opaque(Pack8<T>& p) {
#pragma unroll
    for (int k = 0; k < Pack8<T>::kWords; ++k)
        asm volatile("" : "+r"(p.w[k].x), "+r"(p.w[k].y), "+r"(p.w[k].z), "+r"(p.w[k].w)::"memory");
}

// Rows that do not start on 16 bytes (odd widths, views): a thread's eight
// elements lie `ck_off` elements into a 16-byte granule, the same for the whole
// row.  They are read as whole granules, one more than they fill, and shifted
// into place; they are written as whole granules too, each lane the one that
// holds the last elements of the lane before it and all but the last of its own.
// A write never leaves the row: its ends, and a warp's, go element by element.
// A read of the row's first or last granule takes in bytes of the rows beside
// it, which are dropped; the matrix's own first and last row (ck_inner) are read
// element by element.  8192 x 8191 bf16, single elements against granules: store
// with residual 435 and 200 us, restored 183 and 70, norm 188 and 89, gradient
// 378 and 224; what is left is each granule's second load, the shifts and the
// registers that these take (8192 x 8184, without them: 108, 43, 47 and 110).
template <typename E>
__device__ __forceinline__ int ck_off(const E* p) {
    constexpr int kGranule = sizeof(E) == 1 ? 8 : 16;
    return (int)((reinterpret_cast<uintptr_t>(p) & (kGranule - 1)) / sizeof(E));
}
// out = the bytes of `in` from m on; G words are a granule, m below its bytes.
template <int W, int G>
__device__ __forceinline__ void ck_shift(uint32_t (&in)[W + G], uint32_t m, uint32_t (&out)[W]) {
    if (G == 4)
#pragma unroll
        for (int i = 0; i < W + 2; ++i) in[i] = m & 8 ? in[(i + 2) % (W + G)] : in[i];
#pragma unroll
    for (int i = 0; i < W + 1; ++i) in[i] = m & 4 ? in[i + 1] : in[i];
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = __funnelshift_r(in[i], in[i + 1], (m & 3) * 8);
}
template <typename E>  // E: int8_t (eight bytes, granules of 8) or a float type
struct CkAny {
    static constexpr int kWords = 2 * sizeof(E), kGranule = sizeof(E) == 1 ? 2 : 4, kElems = 4 * kGranule / sizeof(E);
    using V = std::conditional_t<sizeof(E) == 1, uint2, uint4>;

    // The granules that hold the row's elements c .. c + 7.
    static __device__ __forceinline__ void load(const E* row, int c, int d, uint32_t (&in)[kWords + kGranule]) {
        const int off = ck_off(row + c);
        const V* q = reinterpret_cast<const V*>(row + c - off);
        constexpr int n = kWords / kGranule;
#pragma unroll
        for (int i = 0; i <= n; ++i) {
            V v = {};
            if (c + i * kElems < d + (i > 0 ? off : 0) && (i < n || off)) v = __ldg(q + i);
            *reinterpret_cast<V*>(in + i * kGranule) = v;
        }
    }
    // Those elements, zero past the row's end.
    static __device__ __forceinline__ void place(const E* row, int c, int d, uint32_t (&in)[kWords + kGranule],
                                                 uint32_t (&w)[kWords]) {
        ck_shift<kWords, kGranule>(in, (uint32_t)ck_off(row + c) * sizeof(E), w);
        constexpr int per = 4 / sizeof(E);
        if (c + 8 > d)
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const int have = d - c - i * per;  // elements of this word
                w[i] = have >= per ? w[i] : have <= 0 ? 0u : w[i] & ((1u << (8 * sizeof(E) * have % 32)) - 1u);
            }
    }
    // By all lanes of a warp, whose c are neighbours.  Bit i of the result: the
    // lane still has to write its element i.
    static __device__ __forceinline__ uint32_t store(E* row, int c, int d, const uint32_t (&w)[kWords]) {
        const int off = ck_off(row + c), lane = threadIdx.x & 31;
        alignas(16) uint32_t in[kWords + kGranule], o[kWords];
#pragma unroll
        for (int i = 0; i < kGranule; ++i) in[i] = __shfl_up_sync(0xffffffffu, w[kWords - kGranule + i], 1);
#pragma unroll
        for (int i = 0; i < kWords; ++i) in[kGranule + i] = w[i];
        const bool mine = (off == 0 || lane > 0) && c - off + 8 <= d;
        const bool next = off > 0 && lane < 31 && c - off + 16 <= d;
        if (off) {
            ck_shift<kWords, kGranule>(in, (uint32_t)(kElems - off) * sizeof(E), o);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) o[i] = w[i];
        }
        if (mine) {
            V* q = reinterpret_cast<V*>(row + c - off);
#pragma unroll
            for (int i = 0; i < kWords / kGranule; ++i) q[i] = *reinterpret_cast<const V*>(o + i * kGranule);
        }
        const uint32_t head = 0xffu >> off, exist = c >= d ? 0 : c + 8 <= d ? 0xffu : 0xffu >> (8 - (d - c));
        return exist & ~((mine ? head : 0) | (next ? 0xffu & ~head : 0));
    }
};

// Features c .. c + 7 of a row of d (zero past its end).  VEC: every row
// starts on 16 bytes and d is a multiple of 8.  Stores by whole warps.
template <typename T, bool VEC>
__device__ __forceinline__ Pack8<T> ck_load8(const T* row, int c, int d) {
    Pack8<T> p;
    if (VEC) {
#pragma unroll
        for (int k = 0; k < Pack8<T>::kWords; ++k)
            p.w[k] = c < d ? ck_stream(reinterpret_cast<const uint4*>(row + c) + k) : make_uint4(0, 0, 0, 0);
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
        uint32_t w[CkAny<T>::kWords];
#pragma unroll
        for (int k = 0; k < Pack8<T>::kWords; ++k) {
            w[4 * k] = p.w[k].x;
            w[4 * k + 1] = p.w[k].y;
            w[4 * k + 2] = p.w[k].z;
            w[4 * k + 3] = p.w[k].w;
        }
        if (const uint32_t left = CkAny<T>::store(row, c, d, w))
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (left >> i & 1) row[c + i] = (T)ck_value<T>(p, i);
    }
}
template <bool VEC>
__device__ __forceinline__ uint2 ck_load_codes(const int8_t* row, int c, int d) {
    if (VEC) return c < d ? ck_stream(reinterpret_cast<const uint2*>(row + c)) : make_uint2(0, 0);
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
        const uint32_t w[2] = {q.x, q.y};
        if (const uint32_t left = CkAny<int8_t>::store(row, c, d, w))
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (left >> i & 1) row[c + i] = (int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
    }
}
// The value of code i (the conversion instruction takes a byte of a register).
__device__ __forceinline__ float ck_code(uint2 q, int i) {
    return (float)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
}

// Four features of gain, which has a type of its own.  VEC: it starts on 16
// bytes and d is a multiple of 8.
template <bool VEC>
__device__ __forceinline__ float4 ck_gain4(const void* gain, int dtype, int c, int d) {
    if (VEC) {
        if (c >= d) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (dtype == AETH_DTYPE_F32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(gain) + c));
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(gain) + c));
        if (dtype == AETH_DTYPE_BF16)
            return make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16),
                               __uint_as_float(q.y & 0xffff0000u));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&q.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&q.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    float g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = c + i < d ? load_as_f32(gain, c + i, dtype) : 0.0f;
    return make_float4(g[0], g[1], g[2], g[3]);
}
template <bool VEC>
__device__ __forceinline__ void ck_gain8(const void* gain, int dtype, int c, int d, float (&g)[8]) {
    const float4 a = ck_gain4<VEC>(gain, dtype, c, d), b = ck_gain4<VEC>(gain, dtype, c + 4, d);
    g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w;
    g[4] = b.x; g[5] = b.y; g[6] = b.z; g[7] = b.w;
}

// Eight floats of a thread in shared memory, [k][half][thread of the row], so
// that neighbouring lanes take neighbouring 16 bytes.
__device__ __forceinline__ float4& ck_slot(float4* base, int k, int half) {
    return base[(2 * k + half) * blockDim.x + threadIdx.x];
}
template <int VPT, bool VEC>
__device__ __forceinline__ void ck_gain_to_shared(float4* sg, const void* gain, int dtype, int d) {
    if (threadIdx.y == 0)
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = 8 * (threadIdx.x + k * blockDim.x);
            ck_slot(sg, k, 0) = ck_gain4<VEC>(gain, dtype, c, d);
            ck_slot(sg, k, 1) = ck_gain4<VEC>(gain, dtype, c + 4, d);
        }
    __syncthreads();
}
__device__ __forceinline__ void ck_slot8(float4* base, int k, float (&g)[8]) {
    const float4 a = ck_slot(base, k, 0), b = ck_slot(base, k, 1);
    g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w;
    g[4] = b.x; g[5] = b.y; g[6] = b.z; g[7] = b.w;
}

// Two floats in one 64-bit register, for chains of packed arithmetic.
__device__ __forceinline__ uint64_t f2(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ float2 f2_get(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// Scale of a block from its maximum magnitude (NaN where the block held one).
__device__ __forceinline__ float ck_scale(float amax) {
    if (!(amax <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    return amax < 1.504632769e-36f ? 1.0f : __fdiv_rn(amax, 127.0f);
}

// round_half_away(x * inv): adding a half of x's sign with rounding toward zero
// never carries a value below k - 1/2 up to k, so the truncation of that sum is
// the rounding.  |x * inv| <= 127 (1 + 2^-22) in a block, so the sum stays below
// 128 and needs no clamp; a NaN (the NaN scale's reciprocal) converts to 0.
__device__ __forceinline__ int ck_round(float v) {
    return __float2int_rz(__fadd_rz(v, __uint_as_float((__float_as_uint(v) & 0x80000000u) | 0x3f000000u)));
}
__device__ __forceinline__ uint2 ck_encode8(const float (&x)[8], float inv) {
    int q[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 v = mul2_rn(make_float2(x[i], x[i + 1]), make_float2(inv, inv));
        q[i] = ck_round(v.x);
        q[i + 1] = ck_round(v.y);
    }
    const uint32_t a = __byte_perm(q[0], q[1], 0x0040), b = __byte_perm(q[2], q[3], 0x0040);
    const uint32_t c = __byte_perm(q[4], q[5], 0x0040), e = __byte_perm(q[6], q[7], 0x0040);
    return make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(c, e, 0x5410));
}

// x^ of eight codes
__device__ __forceinline__ void ck_decode8(uint2 q, float s, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 v = mul2_rn(make_float2(ck_code(q, i), ck_code(q, i + 1)), make_float2(s, s));
        x[i] = v.x;
        x[i + 1] = v.y;
    }
}
template <typename T>
__device__ __forceinline__ void ck_unpack(const Pack8<T>& p, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ck_value<T>(p, i);
}
// acc += a b over eight values, in two chains (even and odd features)
__device__ __forceinline__ float ck_dot8(const float (&a)[8], const float (&b)[8]) {
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = fma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), s);
    return s.x + s.y;
}

__device__ __forceinline__ float ck_rstd(float sumsq, float inv_d, float eps) { return rsqrtf(fmaf(sumsq, inv_d, eps)); }

// Joins v[k] of the sixteen lanes that hold a block, for all k at once: with
// four, the first two exchanges halve the blocks that a lane carries on, five
// exchanges instead of sixteen.  Lane l ends with block ck_lane_block<VPT>(l);
// the order of the joins (lanes 8, 4, 2, 1 apart) is the same for every VPT.
struct CkAdd {
    __device__ float operator()(float a, float b) const { return a + b; }
};
struct CkMaxNan {
    __device__ float operator()(float a, float b) const { return fmax3_nan(a, a, b); }
};
template <int VPT, typename Op>
__device__ __forceinline__ float ck_block_tree(const float (&v)[VPT], Op op) {
    const uint32_t all = 0xffffffffu;
    float c;
    if constexpr (VPT == 4) {
        const bool b3 = threadIdx.x & 8, b2 = threadIdx.x & 4;
        const float a0 = op(b3 ? v[1] : v[0], __shfl_xor_sync(all, b3 ? v[0] : v[1], 8));
        const float a1 = op(b3 ? v[3] : v[2], __shfl_xor_sync(all, b3 ? v[2] : v[3], 8));
        c = op(b2 ? a1 : a0, __shfl_xor_sync(all, b2 ? a0 : a1, 4));
    } else if constexpr (VPT == 2) {
        const bool b3 = threadIdx.x & 8;
        c = op(b3 ? v[1] : v[0], __shfl_xor_sync(all, b3 ? v[0] : v[1], 8));
        c = op(c, __shfl_xor_sync(all, c, 4));
    } else {
        static_assert(VPT == 1, "one, two or four blocks a lane");
        c = op(v[0], __shfl_xor_sync(all, v[0], 8));
        c = op(c, __shfl_xor_sync(all, c, 4));
    }
    c = op(c, __shfl_xor_sync(all, c, 2));
    return op(c, __shfl_xor_sync(all, c, 1));
}
template <int VPT>
__device__ __forceinline__ int ck_lane_block() {  // the k whose block this lane ends with
    const int b3 = (threadIdx.x >> 3) & 1, b2 = (threadIdx.x >> 2) & 1;
    return VPT == 4 ? b3 + 2 * b2 : VPT == 2 ? b3 : 0;
}
template <int VPT>
__device__ __forceinline__ float ck_from_block(float c, int k) {  // that block's value, in all its lanes
    static_assert(VPT != 2, "the kernels that need it hold one or four");
    return VPT == 4 ? __shfl_sync(0xffffffffu, c, (threadIdx.x & 16) | ((k & 1) << 3) | ((k & 2) << 1)) : c;
}
template <int VPT>
__device__ __forceinline__ bool ck_block_writer() { return (threadIdx.x & (16 / VPT - 1)) == 0; }

// Sums of a row, spread over threadIdx.x (threadIdx.y is the row within the
// CTA).  The order depends on the row's length alone, so a row's result does
// not change with the number of rows in the call: v[n][k] is the sum of one
// thread's eight features, sixteen lanes join to a block's sum, lane l of every
// warp adds the blocks l and l + 32, and a warp's tree joins the lanes.  One
// barrier a call: `sh` has two halves that alternate.
constexpr int kCkptShared = 64;  // blocks that a CTA holds: 8192 features / 128
template <int N, int VPT, typename Barrier>
__device__ __forceinline__ void ck_row_sum(const float (&v)[N][VPT], float* s, int x0, int tx, float (&sum)[N],
                                           Barrier barrier) {
    const int blocks = VPT * tx / 16;
    const int blk = (x0 >> 4) + ck_lane_block<VPT>() * (tx >> 4);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const float x = ck_block_tree<VPT>(v[n], CkAdd());
        if (ck_block_writer<VPT>()) s[blk * N + n] = x;
    }
    barrier();
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

// The same for the CTA's rows: sh holds two halves that alternate.
template <int N, int VPT>
__device__ __forceinline__ void ck_row_sum(const float (&v)[N][VPT], float* sh, int parity, float (&sum)[N]) {
    const int tx = blockDim.x;
    ck_row_sum<N, VPT>(v, sh + parity * (N * kCkptShared) + threadIdx.y * (VPT * tx / 16) * N, threadIdx.x, tx, sum,
                       [=] {
                           if (tx == 32) __syncwarp();
                           else __syncthreads();
                       });
}

// Every kernel below holds a row in registers: thread x of a row takes the
// features 8 (x + k blockDim.x) .. + 7, k < VPT, so that sixteen neighbouring
// lanes hold a block of 128, and waits for one sum over the row before it can
// write.  What hides that wait is other rows on the SM, so a thread keeps only
// its row's values as they lie in memory; gain (fp32) and the sums of its
// gradient sit in shared memory where a CTA walks over many rows.
// WIDE: rows longer than a CTA holds, taken in spans of 8 VPT blockDim.x
// features (v then sums a thread's eights over the spans) and read a second
// time after the row's sums are known.
#define CK_SPANS(base, d) for (int base = 0; base < (WIDE ? (d) : 1); base += 8 * VPT * (int)blockDim.x)
#define CK_COLUMN(base, k) ((base) + 8 * (int)(threadIdx.x + (k) * blockDim.x))

// A thread's VPT eights of a row.  inner: the matrix goes on before and after
// the row, whose first and last granule may then be read whole.
template <typename T, int VPT, bool VEC>
__device__ __forceinline__ void ck_load_row(const T* row, int base, int d, bool inner, Pack8<T> (&x)[VPT]) {
    if (!VEC && inner) {
        alignas(16) uint32_t in[VPT][CkAny<T>::kWords + CkAny<T>::kGranule];
#pragma unroll
        for (int k = 0; k < VPT; ++k) CkAny<T>::load(row, CK_COLUMN(base, k), d, in[k]);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            uint32_t w[CkAny<T>::kWords];
            CkAny<T>::place(row, CK_COLUMN(base, k), d, in[k], w);
#pragma unroll
            for (int i = 0; i < Pack8<T>::kWords; ++i)
                x[k].w[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < VPT; ++k) x[k] = ck_load8<T, VEC>(row, CK_COLUMN(base, k), d);
    }
}
template <int VPT, bool VEC>
__device__ __forceinline__ void ck_codes_row(const int8_t* row, int base, int d, bool inner, uint2 (&q)[VPT]) {
    if (!VEC && inner) {
        alignas(16) uint32_t in[VPT][4];
#pragma unroll
        for (int k = 0; k < VPT; ++k) CkAny<int8_t>::load(row, CK_COLUMN(base, k), d, in[k]);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            uint32_t w[2];
            CkAny<int8_t>::place(row, CK_COLUMN(base, k), d, in[k], w);
            q[k] = make_uint2(w[0], w[1]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < VPT; ++k) q[k] = ck_load_codes<VEC>(row, CK_COLUMN(base, k), d);
    }
}
// Whether 16 bytes of the matrix lie before row t, and 16 after it.
__device__ __forceinline__ bool ck_inner(int64_t t, int64_t rows, int d) {
    const int n = d < 16 ? 16 : 1;
    return t >= n && t + n < rows;
}

// CTAs that the register budget has to allow on an SM.
constexpr int ck_min_ctas(int vpt, int many) { return vpt == 4 ? many : 1; }

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
    const bool inner = ck_inner(t, a.rows, a.d);
    ck_load_row<T, VPT, VEC>(a.x + t * a.ldx, base, d, inner, x);
    if (a.residual) {
        Pack8<T> res[VPT];
        ck_load_row<T, VPT, VEC>(a.residual + t * a.ldr, base, d, inner, res);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float v[8], w[8];
            ck_unpack(x[k], v);
            ck_unpack(res[k], w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += w[i];
            x[k] = ck_pack<T>(v);
        }
    }
}

// Whether gain is kept in shared memory (dynamic, 4 bytes a feature)
constexpr bool ck_shared_gain(int vpt, bool wide) { return vpt == 4 && !wide; }

// Bound by its writes: 8192 x 8192 bf16 with residual 107 us, 5.7 TB/s in all and
// 3.2 TB/s written, where a copy writes 3.3.  Five of nine bytes an element are
// written (sum, y, code).
template <typename T, int VPT, bool VEC, bool WIDE>
__global__ void __launch_bounds__(1024 / VPT, ck_min_ctas(VPT, VEC && sizeof(T) == 2 ? 4 : 3))
    ckpt_store_kernel(const __grid_constant__ CkptStore<T> a) {
    __shared__ float sh[2 * kCkptShared];
    extern __shared__ float4 ck_dyn[];
    constexpr bool kShared = ck_shared_gain(VPT, WIDE);
    const int nb = (a.d + kCkptBlock - 1) / kCkptBlock;
    const float inv_d = 1.0f / (float)a.d;
    if (kShared) ck_gain_to_shared<VPT, VEC>(ck_dyn, a.gain, a.gain_dtype, a.d);
    int parity = 0;
    for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < a.rows; t0 += (int64_t)gridDim.x * blockDim.y, parity ^= 1) {
        const int64_t t = t0 + threadIdx.y;
        const int d = t < a.rows ? a.d : 0;  // a row past the end holds nothing
        Pack8<T> x[VPT];
        float ss[1][VPT] = {}, sum[1];
        CK_SPANS(base, a.d) {
            ckpt_input<T, VPT, VEC>(a, t, base, d, x);
            float m[VPT];
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                if (a.residual) ck_store8<T, VEC>(a.sum + t * a.d, CK_COLUMN(base, k), d, x[k]);
                float v[8];
                ck_unpack(x[k], v);
                ss[0][k] += ck_dot8(v, v);
                m[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) m[k] = fmax3_nan(m[k], fabsf(v[i]), fabsf(v[i + 1]));
            }
            // a lane scales one of its blocks
            const float scale = ck_scale(ck_block_tree<VPT>(m, CkMaxNan()));
            const float inv = __frcp_rn(scale);
            const int c0 = CK_COLUMN(base, ck_lane_block<VPT>()) / kCkptBlock * kCkptBlock;
            if (ck_block_writer<VPT>() && c0 < d) a.scales[t * nb + c0 / kCkptBlock] = scale;
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                float v[8];
                ck_opaque(x[k]);
                ck_unpack(x[k], v);
                ck_store_codes<VEC>(a.codes + t * a.d, CK_COLUMN(base, k), d, ck_encode8(v, ck_from_block<VPT>(inv, k)));
            }
        }
        ck_row_sum<1, VPT>(ss, sh, parity, sum);
        const float r = ck_rstd(sum[0], inv_d, a.eps);
        CK_SPANS(base, a.d) {
            if (WIDE) ckpt_input<T, VPT, VEC>(a, t, base, d, x);
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                float v[8], g[8];
                ck_opaque(x[k]);
                ck_unpack(x[k], v);
                if (kShared) ck_slot8(ck_dyn, k, g);
                else ck_gain8<VEC>(a.gain, a.gain_dtype, CK_COLUMN(base, k), a.d, g);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float2 y = mul2_rn(mul2_rn(make_float2(v[i], v[i + 1]), make_float2(r, r)),
                                             make_float2(g[i], g[i + 1]));
                    v[i] = y.x;
                    v[i + 1] = y.y;
                }
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

// x^ of a thread's eights: their blocks' scales and the codes.
template <int VPT, bool VEC>
__device__ __forceinline__ void ck_restore_row(const CkptRead& a, int64_t t, int base, int d, uint2 (&q)[VPT],
                                               float (&s)[VPT]) {
    const int nb = (a.d + kCkptBlock - 1) / kCkptBlock;
    auto scales = [&] {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = CK_COLUMN(base, k);
            s[k] = c < d ? __ldg(a.scales + t * nb + c / kCkptBlock) : 0.0f;
        }
    };
    if (!VEC) scales();  // before the codes are waited for
    ck_codes_row<VPT, VEC>(a.codes + t * a.d, base, d, ck_inner(t, a.rows, a.d), q);
    if (VEC) scales();
}

// The norm of x^, in rows of pitch ldo.  8192 x 8192 to bf16: 46 us (writing
// alone takes 41).
template <typename T, int VPT, bool VEC, bool WIDE>
__global__ void __launch_bounds__(1024 / VPT, ck_min_ctas(VPT, VEC || sizeof(T) == 4 ? 4 : 2))
    ckpt_norm_kernel(const __grid_constant__ CkptRead a, T* __restrict__ out, int64_t ldo) {
    __shared__ float sh[2 * kCkptShared];
    extern __shared__ float4 ck_dyn[];
    constexpr bool kShared = ck_shared_gain(VPT, WIDE);
    const float inv_d = 1.0f / (float)a.d;
    pdl_trigger();
    if (kShared) ck_gain_to_shared<VPT, VEC>(ck_dyn, a.gain, a.gain_dtype, a.d);
    int parity = 0;
    for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < a.rows; t0 += (int64_t)gridDim.x * blockDim.y, parity ^= 1) {
        const int64_t t = t0 + threadIdx.y;
        const int d = t < a.rows ? a.d : 0;
        uint2 q[VPT];
        float s[VPT], ss[1][VPT] = {}, sum[1];
        CK_SPANS(base, a.d) {
            ck_restore_row<VPT, VEC>(a, t, base, d, q, s);
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                float x[8];
                ck_decode8(q[k], s[k], x);
                ss[0][k] += ck_dot8(x, x);
            }
        }
        ck_row_sum<1, VPT>(ss, sh, parity, sum);
        const float r = ck_rstd(sum[0], inv_d, a.eps);
        CK_SPANS(base, a.d) {
            if (WIDE) ck_restore_row<VPT, VEC>(a, t, base, d, q, s);
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                float x[8], g[8];
                ck_opaque(q[k]);
                ck_decode8(q[k], s[k], x);
                if (kShared) ck_slot8(ck_dyn, k, g);
                else ck_gain8<VEC>(a.gain, a.gain_dtype, CK_COLUMN(base, k), a.d, g);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float2 y = mul2_rn(mul2_rn(make_float2(x[i], x[i + 1]), make_float2(r, r)),
                                             make_float2(g[i], g[i + 1]));
                    x[i] = y.x;
                    x[i + 1] = y.y;
                }
                ck_store8<T, VEC>(out + t * ldo, CK_COLUMN(base, k), d, ck_pack<T>(x));
            }
        }
    }
}

// x^ of a whole checkpoint whose rows are whole blocks and lie one after the
// other: sixteen codes (one load) at a time, four in flight.  8192 x 8192 to
// bf16: 42 us, 3.2 TB/s written: the write rate bounds it.
template <typename T>
__global__ void __launch_bounds__(256) ckpt_decode_flat_kernel(const uint4* __restrict__ codes,
                                                               const float* __restrict__ scales, int64_t n16,
                                                               T* __restrict__ out) {
    pdl_trigger();
    for (int64_t i0 = (int64_t)blockIdx.x * 1024 + threadIdx.x; i0 < n16; i0 += (int64_t)gridDim.x * 1024) {
        uint4 q[4];
        float s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = i0 + k * 256;
            q[k] = i < n16 ? ck_stream(codes + i) : make_uint4(0, 0, 0, 0);
            s[k] = i < n16 ? __ldg(scales + i / 8) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = i0 + k * 256;
            if (i >= n16) break;
            float v[8];
            ck_decode8(make_uint2(q[k].x, q[k].y), s[k], v);
            ck_store8<T, true>(out + 16 * i, 0, 8, ck_pack<T>(v));
            ck_decode8(make_uint2(q[k].z, q[k].w), s[k], v);
            ck_store8<T, true>(out + 16 * i, 8, 16, ck_pack<T>(v));
        }
    }
}

// x^ in rows of pitch ldo; gridDim.y spans of the row.
template <typename T, int VPT, bool VEC>
__global__ void __launch_bounds__(1024 / VPT) ckpt_decode_kernel(const __grid_constant__ CkptRead a, T* __restrict__ out,
                                                                 int64_t ldo) {
    pdl_trigger();
    const int base = blockIdx.y * 8 * VPT * blockDim.x;
    for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < a.rows; t0 += (int64_t)gridDim.x * blockDim.y) {
        const int64_t t = t0 + threadIdx.y;
        const int d = t < a.rows ? a.d : 0;
        uint2 q[VPT];
        float s[VPT];
        ck_restore_row<VPT, VEC>(a, t, base, d, q, s);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float v[8];
            ck_decode8(q[k], s[k], v);
            ck_store8<T, VEC>(out + t * ldo, CK_COLUMN(base, k), d, ck_pack<T>(v));
        }
    }
}

// A row's sums from eight features: of x^ squared, and of x^ dy gain.  The
// codes' squares are whole numbers; the block's scale goes to the sums.
template <typename T>
__device__ __forceinline__ void ck_back_sums(uint2 q, const Pack8<T>& dy, const uint64_t (&g)[4], float s, float& xx,
                                             float& xd) {
    uint64_t dot = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        dot = f2_fma(f2_mul(f2(ck_value<T>(dy, 2 * i), ck_value<T>(dy, 2 * i + 1)), g[i]),
                     f2(ck_code(q, 2 * i), ck_code(q, 2 * i + 1)), dot);
    const float2 dd = f2_get(dot);
    xx += (float)__dp4a((int)q.y, (int)q.y, __dp4a((int)q.x, (int)q.x, 0)) * s * s;  // in this order: s * s may leave fp32's range
    xd += (dd.x + dd.y) * s;
}
// dx of eight features (dy gain r + x^ f + the residual's) and their addends
// to d_gain's sums.
template <typename T>
__device__ __forceinline__ Pack8<T> ck_back_apply(uint2 q, const Pack8<T>& dy, const Pack8<T>& res, bool with_res,
                                                  const uint64_t (&g)[4], float s, float r, float f, uint64_t (&dg)[4]) {
    const uint64_t fs = f2(f * s, f * s), rs = f2(r * s, r * s), rr = f2(r, r);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t xx = f2(ck_code(q, 2 * i), ck_code(q, 2 * i + 1));
        const uint64_t ee = f2(ck_value<T>(dy, 2 * i), ck_value<T>(dy, 2 * i + 1));
        dg[i] = f2_fma(f2_mul(ee, rs), xx, dg[i]);
        const uint64_t z = with_res ? f2(ck_value<T>(res, 2 * i), ck_value<T>(res, 2 * i + 1)) : 0;
        const float2 o = f2_get(f2_fma(f2_mul(ee, g[i]), rr, f2_fma(xx, fs, z)));
        v[2 * i] = o.x;
        v[2 * i + 1] = o.y;
    }
    return ck_pack<T>(v);
}

template <typename T>
struct CkptBack {
    CkptRead in;
    const T* dy;
    int64_t ld_dy;
    const T* d_res;  // or null
    int64_t ld_res;
    T* dx;
    float* part;  // d_gain of each CTA: gridDim.x rows of d
};

// dx, and each CTA's sum of d_gain (ckpt_gain_sum_kernel adds them in their
// order).  A thread's sums lie in shared memory (dynamic, 4 bytes a
// feature and row of the CTA), those of WIDE in `part` itself; each element has
// one thread.
template <typename T, int VPT, bool VEC, bool WIDE>
__global__ void __launch_bounds__(1024 / VPT, ck_min_ctas(VPT, 2))
    ckpt_back_kernel(const __grid_constant__ CkptBack<T> a) {
    __shared__ float sh[4 * kCkptShared];
    extern __shared__ float4 ck_dyn[];
    pdl_trigger();
    constexpr bool kShared = ck_shared_gain(VPT, WIDE);
    const float inv_d = 1.0f / (float)a.in.d;
    float* part = a.part + (int64_t)blockIdx.x * a.in.d;
    float4* dg = ck_dyn + threadIdx.y * 2 * VPT * blockDim.x;
    float4* sg = ck_dyn + blockDim.y * 2 * VPT * blockDim.x;
    if (!WIDE)
#pragma unroll
        for (int k = 0; k < VPT; ++k) ck_slot(dg, k, 0) = ck_slot(dg, k, 1) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (kShared) ck_gain_to_shared<VPT, VEC>(sg, a.in.gain, a.in.gain_dtype, a.in.d);
    auto gain_of = [&](int base, int k, uint64_t (&p)[4]) {
        float g[8];
        if (kShared) ck_slot8(sg, k, g);
        else ck_gain8<VEC>(a.in.gain, a.in.gain_dtype, CK_COLUMN(base, k), a.in.d, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = f2(g[2 * i], g[2 * i + 1]);
    };
    int parity = 0;
    bool first = true;
    for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < a.in.rows;
         t0 += (int64_t)gridDim.x * blockDim.y, parity ^= 1, first = false) {
        const int64_t t = t0 + threadIdx.y;
        const int d = t < a.in.rows ? a.in.d : 0;
        uint2 q[VPT];
        float s[VPT], acc[2][VPT] = {}, sum[2];
        Pack8<T> dy[VPT], res[VPT];
        auto read = [&](int base) {
            ck_restore_row<VPT, VEC>(a.in, t, base, d, q, s);
            ck_load_row<T, VPT, VEC>(a.dy + t * a.ld_dy, base, d, ck_inner(t, a.in.rows, a.in.d), dy);
        };
        auto read_res = [&](int base) {
            if (a.d_res) ck_load_row<T, VPT, VEC>(a.d_res + t * a.ld_res, base, d, ck_inner(t, a.in.rows, a.in.d), res);
        };
        CK_SPANS(base, a.in.d) {
            read(base);
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                uint64_t g[4];
                gain_of(base, k, g);
                ck_back_sums<T>(q[k], dy[k], g, s[k], acc[0][k], acc[1][k]);
            }
        }
        if (!WIDE) read_res(0);  // arrives during the row's sum
        ck_row_sum<2, VPT>(acc, sh, parity, sum);
        const float r = t < a.in.rows ? ck_rstd(sum[0], inv_d, a.in.eps) : 0.0f;  // no row: nothing for d_gain, at eps 0 too
        const float f = ck_back_factor(r, sum[1] * inv_d);
        CK_SPANS(base, a.in.d) {
            if (WIDE) {
                read(base);
                read_res(base);
            }
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = CK_COLUMN(base, k);
                uint64_t g[4], w[4];
                float p[8];
                ck_opaque(q[k]);
                ck_opaque(dy[k]);
                gain_of(base, k, g);
                if (WIDE && VEC) {
                    const float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    const float4* o = reinterpret_cast<const float4*>(part + c);
                    const float4 p0 = c < a.in.d && !first ? o[0] : z, p1 = c < a.in.d && !first ? o[1] : z;
                    p[0] = p0.x; p[1] = p0.y; p[2] = p0.z; p[3] = p0.w;
                    p[4] = p1.x; p[5] = p1.y; p[6] = p1.z; p[7] = p1.w;
                } else if (WIDE) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) p[i] = c + i < a.in.d && !first ? part[c + i] : 0.0f;
                } else {
                    ck_slot8(dg, k, p);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = f2(p[2 * i], p[2 * i + 1]);
                ck_store8<T, VEC>(a.dx + t * a.in.d, c, d,
                                  ck_back_apply<T>(q[k], dy[k], res[k], a.d_res != nullptr, g, s[k], r, f, w));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = f2_get(w[i]);
                    p[2 * i] = x.x;
                    p[2 * i + 1] = x.y;
                }
                if (WIDE && VEC) {
                    if (c < a.in.d) {
                        float4* o = reinterpret_cast<float4*>(part + c);
                        o[0] = make_float4(p[0], p[1], p[2], p[3]);
                        o[1] = make_float4(p[4], p[5], p[6], p[7]);
                    }
                } else if (WIDE) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c + i < a.in.d) part[c + i] = p[i];
                } else {
                    ck_slot(dg, k, 0) = make_float4(p[0], p[1], p[2], p[3]);
                    ck_slot(dg, k, 1) = make_float4(p[4], p[5], p[6], p[7]);
                }
            }
        }
    }
    if (WIDE) return;
    __syncthreads();
    for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < 2 * VPT * (int)blockDim.x; i += blockDim.x * blockDim.y) {
        const int x = i % (int)blockDim.x, kh = i / (int)blockDim.x;
        const int c = 8 * (x + (kh >> 1) * (int)blockDim.x) + 4 * (kh & 1);
        float4 p = ck_dyn[i];
        for (int y = 1; y < (int)blockDim.y; ++y) {  // the rows of the CTA in their order
            const float4 v = ck_dyn[y * 2 * VPT * blockDim.x + i];
            p = make_float4(p.x + v.x, p.y + v.y, p.z + v.z, p.w + v.w);
        }
        if (VEC) {
            if (c < a.in.d) *reinterpret_cast<float4*>(part + c) = p;
        } else {
            const float w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < a.in.d) part[c + e] = w[e];
        }
    }
}

// The same for many rows of up to 16384 features (d a multiple of 16, every row
// on 16 bytes): one CTA an SM, whose rows come through shared memory by bulk
// copies, so that what is in flight does not depend on the registers or on
// where the row sums stand.  The CTA's threads form groups of tx, each of which
// takes every n-th row of the CTA through a ring of its own: when all its warps
// have reached a row's sum, the row before it is done with and its stage is
// filled again.  A thread's d_gain sums stay in registers; at the end the
// groups' are added in their order.  8192 x 8192 bf16 with the residual's
// gradient: 94 us with the sum over the CTAs, 5.0 TB/s (rows through registers
// instead: 110).  Sixteen warps an SM issue 55 % of the time; what is left is the
// wait between a row's two passes.  (A row ahead, its sums taken before the last
// row's dx is written, costs more in registers and barriers than it hides: 109.)
// WIDE: more than 8192 features, one group.  The residual's gradient goes
// through registers, which leaves the ring room for more rows (for shorter rows
// it costs 4 to 15 %), and a thread's eights join 8192 features apart as the
// spans of ckpt_back_kernel do, so that the row's sums are the same.  4096 x
// 12288 bf16 with it: 85 us (in spans: 164).
struct CkptRing {
    int tx, groups, stages;  // stages a group
    int eights;              // of features a thread holds, 4 at most
    int stage_bytes, res_at, codes_at;  // dy first
    __host__ __device__ int gain_bytes() const { return eights * tx * 8 * 4; }
};
constexpr int kRingThreads = 512, kRingMaxStages = 8;

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRingThreads, 1)
    ckpt_back_ring_kernel(const __grid_constant__ CkptBack<T> a, const CkptRing ring, uint32_t* err) {
    constexpr int VPT = 4, SUMS = WIDE ? 2 : VPT;
    extern __shared__ __align__(128) uint8_t ck_ring[];
    __shared__ float sh[2 * 2 * VPT * kRingThreads / 16];  // [group][parity][block][2]
    __shared__ uint64_t full_s[16 * kRingMaxStages];
    __shared__ int abort_s;
    volatile int* abort = &abort_s;
    const int d = a.in.d, nb = (d + kCkptBlock - 1) / kCkptBlock;
    const int tx = ring.tx, x0 = (int)threadIdx.x % tx, grp = (int)threadIdx.x / tx;
    uint8_t* stages = ck_ring + (size_t)grp * ring.stages * ring.stage_bytes;
    uint64_t* full = full_s + grp * kRingMaxStages;
    // gain: [k][half][thread of the group]
    ulonglong2* sg = reinterpret_cast<ulonglong2*>(ck_ring + (size_t)ring.groups * ring.stages * ring.stage_bytes);
    pdl_trigger();
    if (threadIdx.x == 0) abort_s = 0;
    if (x0 == 0) {
        for (int s = 0; s < ring.stages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    for (int i = threadIdx.x; i < 2 * ring.eights * tx; i += blockDim.x) {
        const int c = 8 * (i % tx + i / (2 * tx) * tx) + 4 * (i / tx % 2);
        const float4 g = ck_gain4<true>(a.in.gain, a.in.gain_dtype, c, d);
        sg[i] = make_ulonglong2(f2(g.x, g.y), f2(g.z, g.w));
    }
    __syncthreads();
    // the group's row j is the CTA's row grp + j * groups, row blockIdx.x + that * gridDim.x of all
    const int64_t step = (int64_t)gridDim.x * ring.groups, row0 = blockIdx.x + (int64_t)grp * gridDim.x;
    const int mine = row0 < a.in.rows ? (int)((a.in.rows - row0 + step - 1) / step) : 0;
    auto copy = [&](int j, int s) {  // row j into stage s, by the group's first thread
        const int64_t t = row0 + j * step;
        const uint32_t row16 = (uint32_t)d * (uint32_t)sizeof(T);
        uint8_t* st = stages + (size_t)s * ring.stage_bytes;
        mbar_arrive_expect_tx(&full[s], row16 * (a.d_res && !WIDE ? 2 : 1) + (uint32_t)d);
        bulk_load(st, a.dy + t * a.ld_dy, row16, &full[s]);
        if (a.d_res && !WIDE) bulk_load(st + ring.res_at, a.d_res + t * a.ld_res, row16, &full[s]);
        bulk_load(st + ring.codes_at, a.in.codes + t * d, (uint32_t)d, &full[s]);
    };
    if (x0 == 0)
        for (int j = 0; j < min(ring.stages, mine); ++j) copy(j, j);
    auto scales_of = [&](int j, float (&s)[VPT]) {
        const int64_t t = row0 + j * step;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = 8 * (x0 + k * tx);
            s[k] = j < mine && c < d ? __ldg(a.in.scales + t * nb + c / kCkptBlock) : 0.0f;
        }
    };
    const float inv_d = 1.0f / (float)d;
    float s[VPT], next[VPT];
    uint64_t dg[VPT][4];  // pairs
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) dg[k][i] = 0;
    scales_of(0, s);
    int j = 0, stage = 0;
    uint32_t phase = 0;
    for (; j < mine; ++j) {
        scales_of(j + 1, next);  // a row ahead
        const int64_t t = row0 + j * step;
        const bool here = mbar_wait(&full[stage], phase, abort, err, DEVERR_TIMEOUT_TMA) && !*abort;
        if (!__all_sync(0xffffffffu, here)) {
            if (tx > 32) named_bar_arrive(1 + grp, tx);  // the group may wait for this warp at the row's sum
            break;
        }
        const uint8_t* st = stages + (size_t)stage * ring.stage_bytes;
        float acc[2][SUMS] = {}, sum[2];
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = 8 * (x0 + k * tx);
            if (c < d) {
                const uint2 q = *reinterpret_cast<const uint2*>(st + ring.codes_at + c);
                const Pack8<T> dy = ck_shared8<T>(st, c);
                const ulonglong2 g0 = sg[2 * k * tx + x0], g1 = sg[(2 * k + 1) * tx + x0];
                const uint64_t g[4] = {g0.x, g0.y, g1.x, g1.y};
                ck_back_sums<T>(q, dy, g, s[k], acc[0][k % SUMS], acc[1][k % SUMS]);
            }
        }
        Pack8<T> held[WIDE ? VPT : 1];
        if (WIDE && a.d_res)  // arrives during the row's sum
#pragma unroll
            for (int k = 0; k < (WIDE ? VPT : 1); ++k) held[k] = ck_load8<T, true>(a.d_res + t * a.ld_res, 8 * (x0 + k * tx), d);
        ck_row_sum<2, SUMS>(acc, sh + (grp * 2 + (j & 1)) * (SUMS * tx / 16) * 2, x0, tx, sum, [=] {
            if (tx == 32) __syncwarp();
            else named_bar(1 + grp, tx);
        });
        if (x0 == 0 && j > 0 && j - 1 + ring.stages < mine)
            copy(j - 1 + ring.stages, stage > 0 ? stage - 1 : ring.stages - 1);
        const float r = ck_rstd(sum[0], inv_d, a.in.eps);
        const float f = ck_back_factor(r, sum[1] * inv_d);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = 8 * (x0 + k * tx);
            if (c < d) {
                uint2 q = *reinterpret_cast<const uint2*>(st + ring.codes_at + c);
                Pack8<T> dy = ck_shared8<T>(st, c), res;
                ck_opaque(q);
                ck_opaque(dy);
                if (WIDE) res = held[WIDE ? k : 0];
                else if (a.d_res) res = ck_shared8<T>(st + ring.res_at, c);
                const ulonglong2 g0 = sg[2 * k * tx + x0], g1 = sg[(2 * k + 1) * tx + x0];
                const uint64_t g[4] = {g0.x, g0.y, g1.x, g1.y};
                ck_store8<T, true>(a.dx + t * d, c, d,
                                   ck_back_apply<T>(q, dy, res, a.d_res != nullptr, g, s[k], r, f, dg[k]));
            }
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) s[k] = next[k];
        if (++stage == ring.stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    // a wait gave up: the copies in flight get a last, bounded chance to land
    if (j < mine && x0 == 0)
        for (int i = 0; i < ring.stages && j + i < mine; ++i)
            for (int n = 0, w = stage + i < ring.stages ? stage + i : stage + i - ring.stages;
                 n < 1000 && !mbar_try_wait(&full[w], stage + i < ring.stages ? phase : phase ^ 1u); ++n) {}
    __syncthreads();
    if (*abort) return;
    // the groups' sums, added in their order
    float* all = reinterpret_cast<float*>(ck_ring);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = 8 * (x0 + k * tx);
        if (c < d) {
            ulonglong2* o = reinterpret_cast<ulonglong2*>(all + (size_t)grp * d + c);
            o[0] = make_ulonglong2(dg[k][0], dg[k][1]);
            o[1] = make_ulonglong2(dg[k][2], dg[k][3]);
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
        float v = all[c];
        for (int g = 1; g < ring.groups; ++g) v += all[(size_t)g * d + c];
        a.part[(int64_t)blockIdx.x * d + c] = v;
    }
}

// d_gain: 32 columns a CTA, its 32 warps every 32nd of the sums, then the warps
// in their order.
__global__ void __launch_bounds__(1024) ckpt_gain_sum_kernel(const float* part, int np, int d, float* d_gain) {
    __shared__ float sh[32][33];
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < d)
#pragma unroll 8
        for (int p = warp; p < np; p += 32) s += part[(int64_t)p * d + c];
    sh[warp][lane] = s;
    __syncthreads();
    s = sh[lane][warp];  // column `warp` of the 32, its 32 sums over the lanes
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0 && blockIdx.x * 32 + warp < d) d_gain[blockIdx.x * 32 + warp] = s;
}

}  // namespace aeth
