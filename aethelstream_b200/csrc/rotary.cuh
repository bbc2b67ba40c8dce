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
// (token, head) rows; its tokens' cosines go to shared memory first, each for
// all the heads.
#pragma once
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
    int64_t rows;    // tokens x heads
    int stretch;     // rows of a CTA's stretch; a CTA takes every ctas-th stretch
    unsigned ctas;   // of the grid
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
    int table_bytes;  // shared memory before the gain (any: before the sums)
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
__device__ __forceinline__ int64_t rot_position(const RotaryArgs& a, int64_t token) {
    const int64_t i = a.period == 1 ? 0 : token % a.period;
    return a.pos32 ? (int64_t)static_cast<const int*>(a.pos)[i] : static_cast<const int64_t*>(a.pos)[i];
}

// The cosines and sines of tokens t0 .. t0 + count - 1: place(p) is where pair
// p's cosine lies among a token's R / 2; the sines follow.
template <typename Place>
__device__ __forceinline__ void rot_table(const RotaryArgs& a, float* table, int64_t t0, int count, Place place) {
    const int half = a.R / 2;
    for (int i = threadIdx.x; i < count * half; i += kRotThreads) {
        const int tok = i / half, p = i - tok * half;
        const float2 cs = rot_angle((uint64_t)rot_position(a, t0 + tok) * a.freq[p], a.amp, a.flip);
        float* o = table + tok * a.R + place(p);
        o[0] = cs.x;
        o[half] = cs.y;
    }
}

// Turns a lane's sixteen features by its eight pairs' cosines and sines.
template <bool INTER>
__device__ __forceinline__ void rot_turn(float (&lo)[8], float (&hi)[8], const float (&c)[8], const float (&s)[8]) {
    if (INTER) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float u = lo[2 * e], v = lo[2 * e + 1], x = hi[2 * e], y = hi[2 * e + 1];
            lo[2 * e] = u * c[e] - v * s[e];
            lo[2 * e + 1] = v * c[e] + u * s[e];
            hi[2 * e] = x * c[4 + e] - y * s[4 + e];
            hi[2 * e + 1] = y * c[4 + e] + x * s[4 + e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float u = lo[e], v = hi[e];
            lo[e] = u * c[e] - v * s[e];
            hi[e] = v * c[e] + u * s[e];
        }
    }
}
template <typename T>
__device__ __forceinline__ void rot_unpack(const Pack8<T>& p, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ck_value<T>(p, i);
}
template <typename T>
__device__ __forceinline__ Pack8<T> rot_load(const T* p) {
    Pack8<T> v;
#pragma unroll
    for (int k = 0; k < Pack8<T>::kWords; ++k) v.w[k] = ck_stream(reinterpret_cast<const uint4*>(p) + k);
    return v;
}
template <typename T>
__device__ __forceinline__ void rot_store(T* p, const Pack8<T>& v) {
#pragma unroll
    for (int k = 0; k < Pack8<T>::kWords; ++k) reinterpret_cast<uint4*>(p)[k] = v.w[k];
}
__device__ __forceinline__ void rot_four(const float4* p, float* v) {
    const float4 x = *p;
    v[0] = x.x;
    v[1] = x.y;
    v[2] = x.z;
    v[3] = x.w;
}
__device__ __forceinline__ float rot_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

enum RotaryOp { ROT_TURN = 0, ROT_NORM = 1, ROT_NORM_BACK = 2 };

// lanes: of a row, the power of two from D / 16 on.  U: rows that a lane has in flight.
template <typename T, bool INTER, int OP, int U>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryArgs a, int lanes) {
    extern __shared__ float4 rot_sh[];  // a token's table: [cos 0-3, cos 4-7, sin 0-3, sin 4-7 of the lane][lane]; gain; sums
    const int which = blockIdx.x >= a.s[0].ctas ? 1 : 0;
    const RotaryRows& s = a.s[which];
    const unsigned cta = blockIdx.x - (which ? a.s[0].ctas : 0);
    const int c = threadIdx.x & (lanes - 1), turning = a.R / 16, all = a.D / 16;
    const int group = threadIdx.x / lanes, groups = kRotThreads / lanes;
    const bool turns = c < turning, mine = c < all;
    const int lo = turns ? 8 * c : a.R + 16 * (c - turning), hi = turns ? a.R / 2 + 8 * c : lo + 8;
    float4* gain = rot_sh + a.table_bytes / 16;  // [lo 0-3, lo 4-7, hi 0-3, hi 4-7][lane]
    float wl[8], wh[8];                           // gradient: the sums of the gain's
    if (OP == ROT_NORM_BACK)
#pragma unroll
        for (int i = 0; i < 8; ++i) wl[i] = wh[i] = 0.0f;
    if (OP != ROT_TURN && group == 0 && mine)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = (i < 2 ? lo : hi) + 4 * (i & 1);
            gain[i * all + c] = make_float4(load_as_f32(s.gain, at, a.gain_dtype), load_as_f32(s.gain, at + 1, a.gain_dtype),
                                            load_as_f32(s.gain, at + 2, a.gain_dtype), load_as_f32(s.gain, at + 3, a.gain_dtype));
        }
    const T *x = static_cast<const T*>(s.x), *dy = static_cast<const T*>(s.dy);
    T* out = static_cast<T*>(s.out);
    for (int64_t r0 = (int64_t)cta * s.stretch; r0 < s.rows; r0 += (int64_t)s.ctas * s.stretch) {
        const int64_t t0 = r0 / s.heads;
        const int h0 = (int)(r0 - t0 * s.heads), count = (int)min((int64_t)s.stretch, s.rows - r0);
        __syncthreads();
        rot_table(a, reinterpret_cast<float*>(rot_sh), t0, (h0 + count - 1) / s.heads + 1, [&](int p) {
            // a lane's pairs: eight in a row, or four at its low and four at its high features
            const int q = a.R / 4, l = INTER ? (p < q ? p : p - q) / 4 : p / 8;
            const int e = INTER ? (p & 3) + (p < q ? 0 : 4) : p & 7;
            return ((e >> 2) * turning + l) * 4 + (e & 3);
        });
        __syncthreads();
        for (int i0 = group; i0 - group < count; i0 += U * groups) {  // the same for all lanes of a warp
            Pack8<T> xl[U], xh[U], gl[U], gh[U];
            int tok[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * groups;
                tok[u] = (h0 + i) / s.heads;
                if (i < count && mine) {
                    const int64_t t = t0 + tok[u];
                    const int h = h0 + i - tok[u] * s.heads;
                    const T* p = x + t * s.ld_t + h * s.ld_h;
                    xl[u] = rot_load(p + lo);
                    xh[u] = rot_load(p + hi);
                    if (OP == ROT_NORM_BACK) {
                        const T* q = dy + t * s.ld_dt + h * s.ld_dh;
                        gl[u] = rot_load(q + lo);
                        gh[u] = rot_load(q + hi);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * groups;
                const bool here = i < count && mine;
                float l[8], h[8], cs[8], sn[8];
                if (here) {
                    rot_unpack(xl[u], l);
                    rot_unpack(xh[u], h);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) l[e] = h[e] = 0.0f;
                }
                if (here && turns) {
                    const float4* t = rot_sh + tok[u] * (a.R / 4) + c;
                    rot_four(t, cs);
                    rot_four(t + turning, cs + 4);
                    rot_four(t + 2 * turning, sn);
                    rot_four(t + 3 * turning, sn + 4);
                }
                T* o = out + (r0 + i) * a.D;
                if (OP == ROT_TURN) {
                    if (here && turns) rot_turn<INTER>(l, h, cs, sn);
                } else {
                    float sq = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sq += l[e] * l[e] + h[e] * h[e];
                    const float r = rsqrtf(rot_sum(sq, lanes) / (float)a.D + a.eps);
                    float gnl[8], gnh[8];
                    if (here) {
                        rot_four(gain + c, gnl);
                        rot_four(gain + all + c, gnl + 4);
                        rot_four(gain + 2 * all + c, gnh);
                        rot_four(gain + 3 * all + c, gnh + 4);
                    }
                    if (OP == ROT_NORM) {
                        if (here) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                l[e] = l[e] * r * gnl[e];
                                h[e] = h[e] * r * gnh[e];
                            }
                            if (turns) rot_turn<INTER>(l, h, cs, sn);
                        }
                    } else {
                        float dl[8], dh[8], dot = 0.0f;
                        if (here) {
                            rot_unpack(gl[u], dl);
                            rot_unpack(gh[u], dh);
                            if (turns) rot_turn<INTER>(dl, dh, cs, sn);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                wl[e] += dl[e] * (l[e] * r);
                                wh[e] += dh[e] * (h[e] * r);
                                dl[e] *= gnl[e];
                                dh[e] *= gnh[e];
                                dot += dl[e] * l[e] + dh[e] * h[e];
                            }
                        }
                        dot = rot_sum(dot, lanes) / (float)a.D * (r * r * r);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            l[e] = r * dl[e] - l[e] * dot;
                            h[e] = r * dh[e] - h[e] * dot;
                        }
                    }
                }
                if (here) {
                    rot_store(o + lo, ck_pack<T>(l));
                    rot_store(o + hi, ck_pack<T>(h));
                }
            }
        }
    }
    if (OP == ROT_NORM_BACK) {  // the groups' sums, one after the other
        float* sums = reinterpret_cast<float*>(rot_sh);
        __syncthreads();
        if (mine)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sums[group * a.D + lo + e] = wl[e];
                sums[group * a.D + hi + e] = wh[e];
            }
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += kRotThreads) {
            float t = 0.0f;
            for (int g = 0; g < groups; ++g) t += sums[g * a.D + d];
            s.part[(int64_t)cta * a.D + d] = t;
        }
    }
}

// Heads that 16 features or 16 bytes do not divide: a warp takes a row, a lane
// every 32nd pair and feature of the rest, one element at a time.  The second
// pass over a row finds it in L1.
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
            const int tok = (h0 + i) / s.heads, h = h0 + i - tok * s.heads;
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
                dot = rot_sum(dot, 32) / (float)a.D * (r * r * r);
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
                    yu = r * (yu * gain(u)) - (float)x[u] * dot;
                    yv = r * (yv * gain(v)) - (float)x[v] * dot;
                }
                o[u] = (T)yu;
                o[v] = (T)yv;
            }
            for (int d = a.R + lane; d < a.D; d += 32) {
                if (OP == ROT_TURN) o[d] = x[d];
                else if (OP == ROT_NORM) o[d] = (T)((float)x[d] * r * gain(d));
                else o[d] = (T)(r * ((float)dy[d] * gain(d)) - (float)x[d] * dot);
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
