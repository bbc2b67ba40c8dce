// rotary.cuh -- the position rotation of queries and keys, alone and behind a
// norm of each head, and the gradients of both.
//
// Head row x of D features, the first R of which turn in R / 2 pairs (u, v):
// (x_p, x_{p + R/2}) ("half") or (x_2p, x_{2p+1}) ("interleaved").  At position t
//   u' = a (u cos - v sin)   v' = a (v cos + u sin)   of the angle t f_p,
// the rest of the row stays.  The gradient turns back: sin with the other sign.
// Norm first: x becomes x r w, r = 1 / sqrt(mean x^2 + eps) over the D features.
// Its gradient, with g the turned-back gradient of the output:
//   dx = r (w g) - x r^3 mean(w g x)      dw = sum over rows of g x r
//
// Angles: f_p comes in turns, as a fraction of 2^64.  t f_p in whole numbers
// modulo 2^64 is then the angle without its whole turns, exact whatever the
// position: far positions lose nothing, and neither a table of cosines nor
// 64-bit floating point is needed.  The nearest quarter is taken off in whole
// numbers too, so that 32 bits hold the rest to 3e-8 of a radian.
//
// Rows are read and written once, which bounds every form.  A warp has rows of
// D / 16 lanes (a power of two; lanes past it idle): a lane holds eight features
// at 8 c and the eight R / 2 further on, which are eight pairs in either layout,
// so a row needs no exchange but the norm's sums.  A CTA takes a stretch of the
// (token, head) rows, all SMs one to three waves of them (rot_waves); its tokens'
// cosines go to shared memory first, each for all the heads of q and k.  A lane's rows to come are on
// their way to shared memory by asynchronous copies of its own, which it alone
// reads: bytes in flight without registers, and no barrier.  8192 tokens x (64 + 8)
// heads x 128 bf16: rotation 52 us (5.8 TB/s), with the norm 58 (5.2), the gradient
// 86 (5.3), where a copy of as many bytes takes 50, 50 and 73.  What is left is
// the instructions of a row (issue slots half taken) and a CTA's first microsecond,
// its table; with rows straight from global memory to registers it took 66, 82 and
// 162 us, with q's rows and k's in CTAs of their own 72, 78 and 123.
#pragma once
#include <type_traits>

#include "pack8.cuh"

namespace aeth {

constexpr int kRotThreads = 256;
constexpr int kRotTableBytes = 32 * 1024;  // cosines and sines of a CTA's tokens, at most
constexpr int kRotMaxHead = 1024;          // features of a head

struct RotaryRows {  // one of q and k
    const void* x;   // the rows; of the norm's gradient: its input
    int64_t ld_t, ld_h;
    const void* dy;  // the norm's gradient only
    int64_t ld_dt, ld_dh;
    void* out;       // contiguous
    const void* gain;
    float* part;     // the norm's gradient: D sums for each of the CTAs
    int heads;
    uint32_t magic;  // of rot_quotient
    int64_t rows;    // tokens x heads
    int stretch;     // not rotary_kernel: rows of a stretch, of which a CTA takes every ctas-th
    unsigned ctas;   // CTAs that have rows of it (not rotary_kernel: for it alone)
};
struct RotaryArgs {
    RotaryRows s[2];  // q, k
    const void* pos;  // int64 or int32, one for each of `period` tokens, over and over
    int pos32;
    int64_t period;
    const uint64_t* freq;  // R / 2: 2^64 turns a position
    float amp;             // a, negative sign of `flip` apart
    int flip;              // the other way round
    int D, R, gain_dtype;
    float eps;
    int table_bytes;  // not rotary_kernel: shared memory before the sums
};

__device__ __forceinline__ float2 rot_angle(uint64_t t, float amp, bool flip) {
    const uint64_t near = t + (1ull << 61);
    const int quarter = (int)(near >> 62);
    const int64_t rest = (int64_t)(t - ((uint64_t)quarter << 62));  // +-2^61: an eighth of a turn
    float s, c;
    sincospif((float)(int)(rest >> 30) * 0x1p-33f, &s, &c);
    const float x = quarter & 1 ? -s : c, y = quarter & 1 ? c : s;
    const float cs = quarter & 2 ? -x : x, sn = quarter & 2 ? -y : y;
    return make_float2(cs * amp, (flip ? -sn : sn) * amp);
}
// n / heads for n below heads + a stretch (512): a product with 2^32 / heads, rounded
// up, is exact there up to 32768 heads; with more the quotient is 0 or 1.
__device__ __forceinline__ int rot_quotient(int n, int heads, uint32_t magic) {
    return heads == 1 ? n : heads > 32768 ? (n >= heads ? 1 : 0) : (int)__umulhi((uint32_t)n, magic);
}
__device__ __forceinline__ int64_t rot_position(const RotaryArgs& a, int64_t token) {
    const int64_t i = token < a.period ? token : token % a.period;
    return a.pos32 ? (int64_t)static_cast<const int*>(a.pos)[i] : static_cast<const int64_t*>(a.pos)[i];
}

// The cosines and sines of tokens t0 .. t0 + count - 1: place(p) is where pair
// p's cosine lies among a token's R / 2; the sines follow.  A thread keeps its pair.
template <typename Place>
__device__ __forceinline__ void rot_table(const RotaryArgs& a, float* table, int64_t t0, int count, Place place) {
    const int half = a.R / 2, side = half < kRotThreads ? kRotThreads / half : 1;  // tokens side by side
    const int mine = half < kRotThreads ? threadIdx.x / half : 0;
    if (mine >= side) return;
    for (int p = threadIdx.x - mine * half; p < half; p += kRotThreads) {
        const uint64_t f = a.freq[p];
        float* o = table + place(p);
#pragma unroll 2
        for (int tok = mine; tok < count; tok += side) {
            const float2 cs = rot_angle((uint64_t)rot_position(a, t0 + tok) * f, a.amp, a.flip);
            o[tok * a.R] = cs.x;
            o[tok * a.R + half] = cs.y;
        }
    }
}

// Eight features of a row and the eight beside them, from shared or to global memory.
template <typename T>
__device__ __forceinline__ void rot_get(const uint4* p, int pitch, float2 (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        const uint4 a = p[0], b = p[pitch];
        v[0] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y));
        v[1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
        v[2] = make_float2(__uint_as_float(b.x), __uint_as_float(b.y));
        v[3] = make_float2(__uint_as_float(b.z), __uint_as_float(b.w));
    } else {
        const uint4 a = p[0];
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>)
                v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            else
                v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        }
    }
}
template <typename T>
__device__ __forceinline__ void rot_put(T* p, const float2 (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(ck_pack2<T>(v[0].x, v[0].y), ck_pack2<T>(v[1].x, v[1].y),
                                                  ck_pack2<T>(v[2].x, v[2].y), ck_pack2<T>(v[3].x, v[3].y));
    }
}
__device__ __forceinline__ void rot_copy(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32_addr(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void rot_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void rot_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Four values of a table [four of a lane][lane], as two pairs.
__device__ __forceinline__ void rot_four(const float4* p, float2& a, float2& b) {
    const float4 x = *p;
    a = make_float2(x.x, x.y);
    b = make_float2(x.z, x.w);
}
// Turns a lane's eight low and eight high features by its eight pairs' cosines
// and sines ([cosines 0-3, 4-7, sines 0-3, 4-7][lane]).
template <bool INTER>
__device__ __forceinline__ void rot_turn(float2 (&lo)[4], float2 (&hi)[4], const float4* t, int pitch) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float2 c[2], s[2];
        rot_four(t + k * pitch, c[0], c[1]);
        rot_four(t + (k + 2) * pitch, s[0], s[1]);
        if (INTER) {  // a pair of features is a pair
            float2(&x)[4] = k ? hi : lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ci = i & 1 ? c[i / 2].y : c[i / 2].x, si = i & 1 ? s[i / 2].y : s[i / 2].x;
                x[i] = make_float2(x[i].x * ci - x[i].y * si, x[i].y * ci + x[i].x * si);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 u = lo[2 * k + i], v = hi[2 * k + i], ns = make_float2(-s[i].x, -s[i].y);
                lo[2 * k + i] = fma2_rn(v, ns, mul2_rn(u, c[i]));
                hi[2 * k + i] = fma2_rn(u, s[i], mul2_rn(v, c[i]));
            }
        }
    }
}
__device__ __forceinline__ float rot_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

enum RotaryOp { ROT_TURN = 0, ROT_NORM = 1, ROT_NORM_BACK = 2 };

// What a lane copies of its rows to come: 16-byte pieces of the low features, the
// high ones, and those of dy.
template <typename T, int OP>
constexpr int rot_pieces() { return (int)sizeof(T) / 2 * (OP == ROT_NORM_BACK ? 4 : 2); }
// Stages of the ring: 32 KB a CTA, 48 KB of the gradient's (at 8192 x (64 + 8) x 128
// bf16, rotation 56 to 58 us with 4 to 8 stages, gradient 96, 92 and 93 with 2, 3 and 4).
template <typename T, int OP>
constexpr int rot_stages() {
    constexpr int s = (OP == ROT_NORM_BACK ? 12 : 8) / rot_pieces<T, OP>();
    return s > 2 ? s : 2;
}
template <typename T, int OP>
constexpr int rot_ring_bytes() { return rot_pieces<T, OP>() * rot_stages<T, OP>() * kRotThreads * 16; }

// r / heads
__device__ __forceinline__ int64_t rot_token(int64_t r, int heads) {
    return r <= 0xffffffffll ? (int64_t)((uint32_t)r / (uint32_t)heads) : r / heads;
}

// lanes: of a row, the power of two from D / 16 on.  held: tokens of the table, at
// most.  sums_at: where the gradient's groups x D sums lie in shared memory.
// Of q's rows and of k's a CTA takes the same share, so that its table serves both.
template <typename T, bool INTER, int OP, int CTAS>
__global__ void __launch_bounds__(kRotThreads, CTAS) rotary_kernel(const __grid_constant__ RotaryArgs a, int lanes, int held, int sums_at) {
    constexpr int P = rot_pieces<T, OP>(), S = rot_stages<T, OP>(), Q = (int)sizeof(T) / 2;  // Q: pieces of eight features
    extern __shared__ float4 rot_sh[];  // ring [stage][piece][thread]; q's and k's gain [low 0-3, 4-7, high 0-3, 4-7][lane]; table
    uint4* ring = reinterpret_cast<uint4*>(rot_sh) + threadIdx.x;
    float4* gains = rot_sh + rot_ring_bytes<T, OP>() / 16;
    float4* table = gains + (OP == ROT_TURN ? 0 : a.D / 2);
    const int c = threadIdx.x & (lanes - 1), turning = a.R / 16, all = a.D / 16;
    const int group = threadIdx.x / lanes, groups = kRotThreads / lanes;
    const bool turns = c < turning, mine = c < all;
    const int lo = turns ? 8 * c : a.R + 16 * (c - turning), hi = turns ? a.R / 2 + 8 * c : lo + 8;
    if (OP != ROT_TURN)
        for (int i = threadIdx.x; i < 2 * a.D; i += kRotThreads) {
            const int which = i >= a.D ? 1 : 0, d = i - which * a.D, half = a.R / 2;
            // feature d: of lane l its e-th, low or high
            const bool high = d < a.R ? d >= half : (d - a.R) & 8;
            const int l = d < a.R ? (high ? d - half : d) / 8 : turning + (d - a.R) / 16, e = (d < a.R && high ? d - half : d) & 7;
            if (a.s[which].rows > 0)
                reinterpret_cast<float*>(gains)[which * a.D + (((high ? 2 : 0) + (e >> 2)) * all + l) * 4 + (e & 3)] =
                    load_as_f32(a.s[which].gain, d, a.gain_dtype);
        }
    auto begin_of = [&](int which, unsigned cta) { return a.s[which].rows * cta / gridDim.x; };
    int64_t base = 0, until = 0;  // the table's first token, and the one past its last
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const RotaryRows& s = a.s[which];
        const int64_t begin = begin_of(which, blockIdx.x), end = begin_of(which, blockIdx.x + 1);
        // this lane's first row; a step of `groups` rows is step_t tokens and step_h heads
        const int step_t = groups / s.heads, step_h = groups - step_t * s.heads;
        const int64_t first = begin + group, token = rot_token(first, s.heads);
        int h = (int)(first - token * s.heads), tok = 0;
        // rows on their way to the ring: how many are left, the next one's head and place
        int left = (int)(end - first), ahead_h = h, fill = 0, use = 0;
        const T* px = static_cast<const T*>(s.x) + token * s.ld_t + h * s.ld_h;
        const T* pd = OP == ROT_NORM_BACK ? static_cast<const T*>(s.dy) + token * s.ld_dt + h * s.ld_dh : nullptr;
        const int64_t move = step_t * s.ld_t + step_h * s.ld_h, wrap = s.ld_t - s.heads * s.ld_h;
        const int64_t move_d = step_t * s.ld_dt + step_h * s.ld_dh, wrap_d = s.ld_dt - s.heads * s.ld_dh;
        auto fetch = [&] {
            if (left > 0 && mine) {
                uint4* r = ring + fill * P * kRotThreads;
#pragma unroll
                for (int k = 0; k < Q; ++k) {
                    rot_copy(r + k * kRotThreads, px + lo + k * 4);
                    rot_copy(r + (Q + k) * kRotThreads, px + hi + k * 4);
                    if (OP == ROT_NORM_BACK) {
                        rot_copy(r + (2 * Q + k) * kRotThreads, pd + lo + k * 4);
                        rot_copy(r + (3 * Q + k) * kRotThreads, pd + hi + k * 4);
                    }
                }
            }
            rot_commit();
            left -= groups;
            fill = fill + 1 == S ? 0 : fill + 1;
            ahead_h += step_h;
            const bool over = ahead_h >= s.heads;
            if (over) ahead_h -= s.heads;
            px += move + (over ? wrap : 0);
            if (OP == ROT_NORM_BACK) pd += move_d + (over ? wrap_d : 0);
        };
#pragma unroll 1
        for (int i = 0; i < S - 1; ++i) fetch();
        const float4* gain = gains + (which ? a.D / 4 : 0);
        float2 wl[4], wh[4];  // gradient: the sums of the gain's
        if (OP == ROT_NORM_BACK)
#pragma unroll
            for (int i = 0; i < 4; ++i) wl[i] = wh[i] = make_float2(0.0f, 0.0f);
        T* out = static_cast<T*>(s.out) + first * a.D;
        int64_t row_until = begin;  // rows whose tokens the table holds
        for (int64_t r = begin; r < end; r += groups) {  // the same for all lanes of the CTA
            if (min(r + groups, end) > row_until) {
                const int64_t from = rot_token(r, s.heads), to = rot_token(end - 1, s.heads) + 1;
                if (from < base || min(to, from + held) > until) {
                    base = from;
                    until = min(to, from + held);
                    if (which == 0 && until - base < held && a.s[1].rows > 0)  // k's rows may reach one token further
                        until = min(until + 1, a.s[1].rows / a.s[1].heads);
                    __syncthreads();
                    rot_table(a, reinterpret_cast<float*>(table), base, (int)(until - base), [&](int p) {
                        // a lane's pairs: eight in a row, or four at its low and four at its high features
                        const int q = a.R / 4, l = INTER ? (p < q ? p : p - q) / 4 : p / 8;
                        const int e = INTER ? (p & 3) + (p < q ? 0 : 4) : p & 7;
                        return ((e >> 2) * turning + l) * 4 + (e & 3);
                    });
                    __syncthreads();
                }
                row_until = until * s.heads;
                tok = (int)(rot_token(r + group, s.heads) - base);
            }
            fetch();  // into the stage that the row before took
            rot_wait<S - 1>();
            const uint4* in = ring + use * P * kRotThreads;
            if (++use == S) use = 0;
            const bool here = r + group < end && mine;
            const float4* t = table + tok * (a.R / 4) + c;
            float2 l[4], u[4];
            rot_get<T>(in, kRotThreads, l);
            rot_get<T>(in + Q * kRotThreads, kRotThreads, u);
            if (!here)
#pragma unroll
                for (int e = 0; e < 4; ++e) l[e] = u[e] = make_float2(0.0f, 0.0f);
            float rinv = 1.0f;
            if (OP != ROT_TURN) {
                float2 sq = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int e = 0; e < 4; ++e) sq = fma2_rn(u[e], u[e], fma2_rn(l[e], l[e], sq));
                rinv = rsqrtf(rot_sum(sq.x + sq.y, lanes) / (float)a.D + a.eps);
            }
            if (OP == ROT_NORM && here) {
                const float2 rr = make_float2(rinv, rinv);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float2 g[4];
                    rot_four(gain + k * all + c, g[0], g[1]);
                    rot_four(gain + (k + 2) * all + c, g[2], g[3]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        l[2 * k + e] = mul2_rn(mul2_rn(l[2 * k + e], rr), g[e]);
                        u[2 * k + e] = mul2_rn(mul2_rn(u[2 * k + e], rr), g[2 + e]);
                    }
                }
            }
            if (OP != ROT_NORM_BACK && here && turns) rot_turn<INTER>(l, u, t, turning);
            if (OP == ROT_NORM_BACK) {
                float2 dl[4], dh[4], dot2 = make_float2(0.0f, 0.0f);
                const float2 rr = make_float2(rinv, rinv);
                rot_get<T>(in + 2 * Q * kRotThreads, kRotThreads, dl);
                rot_get<T>(in + 3 * Q * kRotThreads, kRotThreads, dh);
                if (here) {
                    if (turns) rot_turn<INTER>(dl, dh, t, turning);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float2 g[4];
                        rot_four(gain + k * all + c, g[0], g[1]);
                        rot_four(gain + (k + 2) * all + c, g[2], g[3]);
#pragma unroll
                        for (int e = 2 * k; e < 2 * k + 2; ++e) {
                            wl[e] = fma2_rn(dl[e], mul2_rn(l[e], rr), wl[e]);
                            wh[e] = fma2_rn(dh[e], mul2_rn(u[e], rr), wh[e]);
                            dl[e] = mul2_rn(dl[e], g[e - 2 * k]);
                            dh[e] = mul2_rn(dh[e], g[2 + e - 2 * k]);
                            dot2 = fma2_rn(dh[e], u[e], fma2_rn(dl[e], l[e], dot2));
                        }
                    }
                }
                const float dot = ck_back_factor(rinv, rot_sum(dot2.x + dot2.y, lanes) / (float)a.D);
                const float2 nd = make_float2(dot, dot);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    l[e] = fma2_rn(l[e], nd, mul2_rn(dl[e], rr));
                    u[e] = fma2_rn(u[e], nd, mul2_rn(dh[e], rr));
                }
            }
            if (here) {
                rot_put<T>(out + lo, l);
                rot_put<T>(out + hi, u);
            }
            out += (int64_t)groups * a.D;
            h += step_h;
            tok += step_t + (h >= s.heads ? 1 : 0);
            if (h >= s.heads) h -= s.heads;
        }
        rot_wait<0>();
        if (OP == ROT_NORM_BACK && s.rows > 0) {  // the groups' sums, one after the other
            float* sums = reinterpret_cast<float*>(rot_sh) + sums_at;
            __syncthreads();
            if (mine)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    *reinterpret_cast<float2*>(sums + group * a.D + lo + 2 * e) = wl[e];
                    *reinterpret_cast<float2*>(sums + group * a.D + hi + 2 * e) = wh[e];
                }
            __syncthreads();
            for (int d = threadIdx.x; d < a.D; d += kRotThreads) {
                float t = 0.0f;
                for (int g = 0; g < groups; ++g) t += sums[g * a.D + d];
                s.part[(int64_t)blockIdx.x * a.D + d] = t;
            }
        }
    }
}

// Heads that 16 features or 16 bytes do not divide: a warp takes a row, a lane
// every 32nd pair and feature of the rest, one element at a time.  The second
// pass over a row finds it in L1.  For the rotation and heads above 256 features.
template <typename T, bool INTER, int OP>
__global__ void __launch_bounds__(kRotThreads) rotary_any_kernel(const __grid_constant__ RotaryArgs a) {
    extern __shared__ float4 rot_sh[];
    float* table = reinterpret_cast<float*>(rot_sh);
    constexpr int kWarps = kRotThreads / 32;
    float* sums = table + a.table_bytes / 4;  // [warp][D]
    const int which = blockIdx.x >= a.s[0].ctas ? 1 : 0;
    const RotaryRows& s = a.s[which];
    const unsigned cta = blockIdx.x - (which ? a.s[0].ctas : 0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = a.R / 2;
    if (OP == ROT_NORM_BACK)
        for (int d = lane; d < a.D; d += 32) sums[warp * a.D + d] = 0.0f;
    for (int64_t r0 = (int64_t)cta * s.stretch; r0 < s.rows; r0 += (int64_t)s.ctas * s.stretch) {
        const int64_t t0 = r0 / s.heads;
        const int h0 = (int)(r0 - t0 * s.heads), count = (int)min((int64_t)s.stretch, s.rows - r0);
        __syncthreads();
        rot_table(a, table, t0, (h0 + count - 1) / s.heads + 1, [](int p) { return p; });
        __syncthreads();
        for (int i = warp; i < count; i += kWarps) {
            const int tok = rot_quotient(h0 + i, s.heads, s.magic), h = h0 + i - tok * s.heads;
            const T* x = static_cast<const T*>(s.x) + (t0 + tok) * s.ld_t + h * s.ld_h;
            const T* dy = OP == ROT_NORM_BACK ? static_cast<const T*>(s.dy) + (t0 + tok) * s.ld_dt + h * s.ld_dh : nullptr;
            T* o = static_cast<T*>(s.out) + (r0 + i) * a.D;
            const float *cs = table + tok * a.R, *sn = cs + half;
            auto gain = [&](int d) { return load_as_f32(s.gain, d, a.gain_dtype); };
            auto at = [&](int p, int& u, int& v) {
                u = INTER ? 2 * p : p;
                v = INTER ? u + 1 : p + half;
            };
            float r = 1.0f, dot = 0.0f;
            if (OP != ROT_TURN) {
                float sq = 0.0f;
                for (int d = lane; d < a.D; d += 32) sq += (float)x[d] * (float)x[d];
                r = rsqrtf(rot_sum(sq, 32) / (float)a.D + a.eps);
            }
            if (OP == ROT_NORM_BACK) {
                for (int p = lane; p < half; p += 32) {
                    int u, v;
                    at(p, u, v);
                    const float gu = (float)dy[u] * cs[p] - (float)dy[v] * sn[p], gv = (float)dy[v] * cs[p] + (float)dy[u] * sn[p];
                    sums[warp * a.D + u] += gu * ((float)x[u] * r);
                    sums[warp * a.D + v] += gv * ((float)x[v] * r);
                    dot += gain(u) * gu * (float)x[u] + gain(v) * gv * (float)x[v];
                }
                for (int d = a.R + lane; d < a.D; d += 32) {
                    sums[warp * a.D + d] += (float)dy[d] * ((float)x[d] * r);
                    dot += gain(d) * (float)dy[d] * (float)x[d];
                }
                dot = ck_back_factor(r, rot_sum(dot, 32) / (float)a.D);
            }
            for (int p = lane; p < half; p += 32) {
                int u, v;
                at(p, u, v);
                const T* src = OP == ROT_NORM_BACK ? dy : x;
                float xu = (float)src[u], xv = (float)src[v];
                if (OP == ROT_NORM) {
                    xu = xu * r * gain(u);
                    xv = xv * r * gain(v);
                }
                float yu = xu * cs[p] - xv * sn[p], yv = xv * cs[p] + xu * sn[p];
                if (OP == ROT_NORM_BACK) {
                    yu = r * (yu * gain(u)) + (float)x[u] * dot;
                    yv = r * (yv * gain(v)) + (float)x[v] * dot;
                }
                o[u] = (T)yu;
                o[v] = (T)yv;
            }
            for (int d = a.R + lane; d < a.D; d += 32) {
                if (OP == ROT_TURN) o[d] = x[d];
                else if (OP == ROT_NORM) o[d] = (T)((float)x[d] * r * gain(d));
                else o[d] = (T)(r * ((float)dy[d] * gain(d)) + (float)x[d] * dot);
            }
        }
    }
    if (OP == ROT_NORM_BACK) {
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += kRotThreads) {
            float t = 0.0f;
            for (int w = 0; w < kWarps; ++w) t += sums[w * a.D + d];
            s.part[(int64_t)cta * a.D + d] = t;
        }
    }
}

// The norms of such heads up to 256 features and their gradients: a lane has NP pairs
// at most, whose gains and sums of the gains' gradient stay in registers, and the row
// after is on its way meanwhile.  Features that do not turn make pairs of neighbours;
// the last may lack its second.  2047 x (32 + 8) x 80, 40 turning, bf16: norm 24 us,
// gradient 44 (rotary_any_kernel 29 and 91); 8192 x (32 + 32) x 80, 20 turning: 126 and
// 208 (202 and 793).  The rotation alone is no faster so (19 us, 18; 106, 98), nor is
// the norm of 513 features with nine pairs a lane (63, 39).
template <typename T, bool INTER, int OP, int NP>
__global__ void __launch_bounds__(kRotThreads) rotary_pairs_kernel(const __grid_constant__ RotaryArgs a) {
    extern __shared__ float4 rot_sh[];
    float* table = reinterpret_cast<float*>(rot_sh);
    constexpr int kWarps = kRotThreads / 32;
    constexpr bool kBack = OP == ROT_NORM_BACK;
    float* sums = table + a.table_bytes / 4;  // [warp][D]
    const int which = blockIdx.x >= a.s[0].ctas ? 1 : 0;
    const RotaryRows& s = a.s[which];
    const unsigned cta = blockIdx.x - (which ? a.s[0].ctas : 0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = a.R / 2, pairs = half + (a.D - a.R + 1) / 2;
    auto each = [&](auto f) {  // f(j, its features, whether both are there) of the lane's pairs
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int p = 32 * j + lane;
            const int d = p >= half ? a.R + 2 * (p - half) : INTER ? 2 * p : p, e = p >= half || INTER ? d + 1 : d + half;
            if (p < pairs) f(j, d, e, e < a.D);
        }
    };
    float gu[NP], gv[NP], wu[NP], wv[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) gu[j] = gv[j] = wu[j] = wv[j] = 0.0f;
    each([&](int j, int d, int e, bool both) {
        gu[j] = load_as_f32(s.gain, d, a.gain_dtype);
        gv[j] = both ? load_as_f32(s.gain, e, a.gain_dtype) : 0.0f;
    });
    auto load = [&](const T* x, T (&u)[NP], T (&v)[NP]) {
#pragma unroll
        for (int j = 0; j < NP; ++j) u[j] = v[j] = T(0.0f);
        each([&](int j, int d, int e, bool both) {
            u[j] = x[d];
            if (both) v[j] = x[e];
        });
    };
    for (int64_t r0 = (int64_t)cta * s.stretch; r0 < s.rows; r0 += (int64_t)s.ctas * s.stretch) {
        const int64_t t0 = r0 / s.heads;
        const int h0 = (int)(r0 - t0 * s.heads), count = (int)min((int64_t)s.stretch, s.rows - r0);
        __syncthreads();
        rot_table(a, table, t0, (h0 + count - 1) / s.heads + 1, [](int p) { return p; });
        __syncthreads();
        T xu[NP], xv[NP], du[NP], dv[NP];
        auto fetch = [&](int i) {  // row i of the stretch
            if (i >= count) return;
            const int tok = rot_quotient(h0 + i, s.heads, s.magic), h = h0 + i - tok * s.heads;
            load(static_cast<const T*>(s.x) + (t0 + tok) * s.ld_t + h * s.ld_h, xu, xv);
            if (kBack) load(static_cast<const T*>(s.dy) + (t0 + tok) * s.ld_dt + h * s.ld_dh, du, dv);
        };
        fetch(warp);
        for (int i = warp; i < count; i += kWarps) {
            T* o = static_cast<T*>(s.out) + (r0 + i) * a.D;
            const float* cs = table + rot_quotient(h0 + i, s.heads, s.magic) * a.R;
            float u[NP], v[NP], eu[NP], ev[NP], sq = 0.0f;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                u[j] = (float)xu[j];
                v[j] = (float)xv[j];
                eu[j] = kBack ? (float)du[j] : 0.0f;
                ev[j] = kBack ? (float)dv[j] : 0.0f;
                sq = fmaf(v[j], v[j], fmaf(u[j], u[j], sq));
            }
            fetch(i + kWarps);
            const float r = rsqrtf(rot_sum(sq, 32) / (float)a.D + a.eps);
            auto turn = [&](float (&x)[NP], float (&y)[NP]) {
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int p = 32 * j + lane;
                    if (p >= half) continue;
                    const float co = cs[p], si = cs[half + p], was = x[j];
                    x[j] = x[j] * co - y[j] * si;
                    y[j] = y[j] * co + was * si;
                }
            };
            if (kBack) {
                float dot = 0.0f;
                turn(eu, ev);
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    wu[j] = fmaf(eu[j], u[j] * r, wu[j]);
                    wv[j] = fmaf(ev[j], v[j] * r, wv[j]);
                    eu[j] *= gu[j];
                    ev[j] *= gv[j];
                    dot = fmaf(ev[j], v[j], fmaf(eu[j], u[j], dot));
                }
                dot = ck_back_factor(r, rot_sum(dot, 32) / (float)a.D);
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    u[j] = r * eu[j] + u[j] * dot;
                    v[j] = r * ev[j] + v[j] * dot;
                }
            } else {
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    u[j] = u[j] * r * gu[j];
                    v[j] = v[j] * r * gv[j];
                }
                turn(u, v);
            }
            each([&](int j, int d, int e, bool both) {
                o[d] = (T)u[j];
                if (both) o[e] = (T)v[j];
            });
        }
    }
    if (kBack) {
        each([&](int j, int d, int e, bool both) {
            sums[warp * a.D + d] = wu[j];
            if (both) sums[warp * a.D + e] = wv[j];
        });
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += kRotThreads) {
            float t = 0.0f;
            for (int w = 0; w < kWarps; ++w) t += sums[w * a.D + d];
            s.part[(int64_t)cta * a.D + d] = t;
        }
    }
}

// The gain's gradients: the CTAs' sums added up, warp w of 32 every 32nd and
// then the warps, in an order that the grid alone decides.  Lane = feature.
struct RotaryGain {
    const float* part[2];
    float* out[2];
    int groups[2];
    int D;
};
__global__ void __launch_bounds__(1024) rotary_gain_kernel(const RotaryGain a) {
    __shared__ float sh[32][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = blockIdx.x * 32 + lane, which = blockIdx.y;
    pdl_wait();
    float t = 0.0f;
    if (d < a.D)
        for (int g = warp; g < a.groups[which]; g += 32) t += a.part[which][(int64_t)g * a.D + d];
    sh[warp][lane] = t;
    __syncthreads();
    if (warp == 0 && d < a.D) {
        t = 0.0f;
#pragma unroll
        for (int w = 0; w < 32; ++w) t += sh[w][lane];
        a.out[which][d] = t;
    }
}

}  // namespace aeth
