// head_loss.cuh -- softmax cross entropy at the language model's head, in
// pieces of the vocabulary, without keeping the logits (the device form of
// doublepass/src/loss.rs:83-377, streaming_cut_ce).
//
//   s = H W^T                      H: tokens x d, W: vocab x d
//   lse_t = log sum_v exp s_tv     loss_t = lse_t - s_t,label
//   G = g_t (exp(s - lse_t) - onehot(label_t))
//   dH = G W                       dW = G^T H
//
// Tokens whose label is ignore_index are left out before the first product:
// the live rows of H are gathered (head_pack_kernel) and every product runs
// over their count, which stays on the device.  What masked rows hold (NaN
// too) therefore reaches nothing.
//
// Forward: one product whose epilogue keeps, per row and column range, the
// running maximum and the sum of exponentials; head_loss_kernel joins them.
// Backward: per vocabulary piece, the same product again, its epilogue writing
// G in 16 bits; then dW of the piece and the piece's share of dH (fp32).
#pragma once
#include "pair_gemm.cuh"

namespace aeth {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kHeadIgnored = -1, kHeadBad = -2;  // pos[] of a token that takes no part

// G is held relative to the largest token weight (|G| <= 1) and times 2^k, the
// power folded into the exponent of p: with k = 15 f16 keeps eleven bits down
// to p = 2e-9 (6e-5 without); with k = 32 what fp32's and bf16's range cuts off
// is p < 2^-158, not 2^-126.
__host__ __device__ constexpr float head_g_bits(bool bf16) { return bf16 ? 32.0f : 15.0f; }
__host__ __device__ constexpr float head_g_scale(bool bf16) { return bf16 ? 4294967296.0f : 32768.0f; }

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

struct HeadRows {
    const int64_t* labels;
    int64_t n;
    int64_t ignore_index;
    int vocab;
    int* rows;   // live row -> token
    int* pos;    // token -> live row, kHeadIgnored or kHeadBad
    int* lab;    // live row -> label
    int* count;  // live rows
    // backward only (coef != null)
    const float* lse;   // per token
    const float* grad;  // per token, or null: 1 / count
    float scale, g_bits, g_scale;  // g_scale = 2^g_bits
    float* coef;       // live row -> g_t / max|g|
    float* lse2;       // live row -> lse * log2(e) - g_bits
    float* out_scale;  // max|g| / g_scale
};

// One CTA numbers the live tokens in order (a scan over the labels) and
// gathers what the epilogues need per live row.
__global__ void __launch_bounds__(1024) head_rows_kernel(HeadRows a, uint32_t* err) {
    __shared__ int wsum[32];
    __shared__ float wmax[32];
    __shared__ int base_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int base = 0;
    float gmax = 0.0f;
    bool gnan = false;
    for (int64_t t0 = 0; t0 < a.n; t0 += 1024) {
        const int64_t t = t0 + tid;
        bool live = false, bad = false;
        int64_t lab = 0;
        if (t < a.n) {
            lab = a.labels[t];
            live = lab != a.ignore_index;
            bad = live && (lab < 0 || lab >= a.vocab);
            if (bad) { live = false; report_dev_error(err, DEVERR_BAD_ARG); }
        }
        const uint32_t m = __ballot_sync(0xffffffffu, live);
        if (lane == 0) wsum[warp] = __popc(m);
        __syncthreads();
        if (warp == 0) {
            int v = wsum[lane], s = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += x;
            }
            wsum[lane] = s - v;
            if (lane == 31) base_s = s;
        }
        __syncthreads();
        if (t < a.n) {
            const int i = base + wsum[warp] + __popc(m & ((1u << lane) - 1));
            a.pos[t] = live ? i : bad ? kHeadBad : kHeadIgnored;
            if (live) {
                a.rows[i] = (int)t;
                a.lab[i] = (int)lab;
                if (a.coef) {
                    a.lse2[i] = fmaf(a.lse[t], kLog2e, -a.g_bits);
                    if (a.grad) {
                        const float g = a.grad[t] * a.scale;
                        a.coef[i] = g;
                        gmax = fmaxf(gmax, fabsf(g));
                        gnan |= g != g;
                    }
                }
            }
        }
        base += base_s;
        __syncthreads();
    }
    if (tid == 0) *a.count = base;
    if (!a.coef) return;
    if (a.grad) {
        gmax = warp_max(gmax);
        gnan = __any_sync(0xffffffffu, gnan);
        if (lane == 0) wmax[warp] = gnan ? __int_as_float(0x7fc00000) : gmax;
        __syncthreads();
        gmax = 0.0f;
        for (int w = 0; w < 32; ++w) gmax = wmax[w] != wmax[w] || gmax != gmax ? __int_as_float(0x7fc00000) : fmaxf(gmax, wmax[w]);
        for (int i = tid; i < base; i += 1024) a.coef[i] = gmax == 0.0f ? 0.0f : a.coef[i] / gmax;
    } else {
        const float g = a.scale / (float)max(base, 1);
        gmax = fabsf(g);
        for (int i = tid; i < base; i += 1024) a.coef[i] = gmax == 0.0f ? 0.0f : g / gmax;
    }
    if (tid == 0) *a.out_scale = gmax / a.g_scale;
}

// Live rows of H, gathered to a pitch that TMA takes; rows from the count up
// to the next multiple of 256 are zero (the products' last tiles read them;
// past row n TMA itself fills with zero, without reading).
__global__ void __launch_bounds__(256) head_pack_kernel(const uint16_t* __restrict__ h, int64_t ld, int64_t n, int d,
                                                        const int* __restrict__ rows, const int* __restrict__ count,
                                                        uint16_t* __restrict__ out, int64_t ldo) {
    const int live = *count;
    const int64_t padded = min((int64_t)max((live + 255) / 256 * 256, 256), n);
    const bool whole = (ld % 8) == 0 && (d % 8) == 0 && (reinterpret_cast<uintptr_t>(h) & 15) == 0;
    for (int64_t i = blockIdx.x; i < padded; i += gridDim.x) {
        const uint16_t* src = h + (i < live ? (int64_t)rows[i] * ld : 0);
        uint16_t* dst = out + i * ldo;
        if (i >= live) {
            for (int c = threadIdx.x; c < d; c += blockDim.x) dst[c] = 0;
        } else if (whole) {
            for (int c = threadIdx.x; c < d / 8; c += blockDim.x)
                reinterpret_cast<uint4*>(dst)[c] = reinterpret_cast<const uint4*>(src)[c];
        } else {
            for (int c = threadIdx.x; c < d; c += blockDim.x) dst[c] = src[c];
        }
    }
}

// Epilogue of the forward product: per row, over this warp's columns, the
// largest logit (times log2 e) and the sum of 2^(logit log2 e - that), and the
// label's logit where it lies here.
struct HeadStats {
    const int* lab;
    float* label_logit;
    float2* part;  // [2 * n_tile + half][row]
    int64_t ld_part;
    static constexpr int kChunk = 8;  // the loss is an fp32 result: see pair_gemm.cuh
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
        const int row = t.row0 + t.lane;
        const bool in = row < t.M;
        const int at = in ? lab[row] - t.col0 - t.c_begin : -1;
        float mx = -INFINITY, sum = 0.0f;  // mx in units of log2
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int left = min(t.c_end, t.N - t.col0) - t.c_begin - 32 * c;  // columns of this chunk that exist
            if (left > 0) {
                float m = -INFINITY;
                if (left >= 32) {
#pragma unroll
                    for (int i = 0; i < 32; i += 2) m = fmax3(m, acc[32 * c + i], acc[32 * c + i + 1]);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (i < left) m = fmaxf(m, acc[32 * c + i]);
                }
                const float nm = fmaxf(mx, m * kLog2e);
                const float off = nm == -INFINITY ? 0.0f : nm;
                sum *= ex2(mx - off);
                float s0 = 0.0f, s1 = 0.0f;
                if (left >= 32) {
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        s0 += ex2(fmaf(acc[32 * c + i], kLog2e, -off));
                        s1 += ex2(fmaf(acc[32 * c + i + 1], kLog2e, -off));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (i < left) s0 += ex2(fmaf(acc[32 * c + i], kLog2e, -off));
                }
                sum += s0 + s1;
                mx = nm;
                const int k = at - 32 * c;
                if (__any_sync(0xffffffffu, k >= 0 && k < 32)) {
                    float x = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) x = k == i ? acc[32 * c + i] : x;
                    if (k >= 0 && k < 32) label_logit[row] = x;
                }
            }
        }
        if (in) part[(int64_t)(2 * t.n_tile + t.half) * ld_part + row] = make_float2(mx, sum);
    }
};

// Joins the column ranges' maxima and sums.  A CTA takes 32 live rows (lane =
// row), its warps every eighth range.
__global__ void __launch_bounds__(256) head_loss_kernel(const float2* __restrict__ part, int64_t ld_part, int np,
                                                        const float* __restrict__ label_logit,
                                                        const int* __restrict__ rows, const int* __restrict__ count,
                                                        float* __restrict__ losses, float* __restrict__ lse) {
    __shared__ float2 sh[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int live = *count;
    for (int64_t r0 = (int64_t)blockIdx.x * 32; r0 < live; r0 += (int64_t)gridDim.x * 32) {
        const int64_t row = r0 + lane;
        float mx = -INFINITY, sum = 0.0f;
        if (row < live) {
            for (int p = warp; p < np; p += 8) {
                const float2 x = part[p * ld_part + row];
                const float nm = fmaxf(mx, x.x), off = nm == -INFINITY ? 0.0f : nm;
                sum = sum * ex2(mx - off) + x.y * ex2(x.x - off);
                mx = nm;
            }
        }
        sh[warp][lane] = make_float2(mx, sum);
        __syncthreads();
        if (warp == 0 && row < live) {
            for (int w = 1; w < 8; ++w) mx = fmaxf(mx, sh[w][lane].x);
            const float off = mx == -INFINITY ? 0.0f : mx;
            sum = 0.0f;
            for (int w = 0; w < 8; ++w) sum += sh[w][lane].y * ex2(sh[w][lane].x - off);
            const float l = off * kLn2 + logf(sum);
            const int t = rows[row];
            lse[t] = l;
            losses[t] = l - label_logit[row];
        }
        __syncthreads();
    }
}

// Losses of the tokens that take no part (0; NaN for a label outside the
// vocabulary) and the mean over the live ones, summed in one fixed order.
__global__ void __launch_bounds__(1024) head_mean_kernel(const int* __restrict__ pos, int64_t n,
                                                         const int* __restrict__ count, float* __restrict__ losses,
                                                         float* __restrict__ lse, float* __restrict__ loss) {
    __shared__ double ws[32];
    double s = 0.0;
    for (int64_t t = threadIdx.x; t < n; t += 1024) {
        const int p = pos[t];
        if (p < 0) {
            losses[t] = lse[t] = p == kHeadBad ? __int_as_float(0x7fc00000) : 0.0f;
            if (p == kHeadBad) s += (double)__int_as_float(0x7fc00000);
        } else {
            s += (double)losses[t];
        }
    }
    s = warp_sum_d(s);
    if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = warp_sum_d(ws[threadIdx.x]);
        if (threadIdx.x == 0) *loss = (float)(s / (double)max(*count, 1));
    }
}

// Epilogue of the backward's product: G of the piece in 16 bits.  G is rounded
// once, from fp32; rows from the count to the tile's end (or n) become zero.
template <bool BF16>
struct HeadGrad {
    static constexpr int kChunk = 0;
    const int* lab;
    const float* coef;
    const float* lse2;
    uint16_t* g;
    int64_t ldg;
    int n;   // rows of g: the tokens
    int v0;  // first vocabulary entry of the piece
    __device__ __forceinline__ void tile(const PairTile& t) const {
        const int row = t.row0 + t.lane;
        const bool in = row < t.M;
        const float f = in ? coef[row] : 0.0f, l2 = in ? lse2[row] : 0.0f;
        const int lab_c = in ? lab[row] - v0 - t.col0 : -1;
        for (int c = t.c_begin; c < t.c_end; c += 64) {
            if (t.col0 + c >= t.N || t.row0 >= n) break;
            uint32_t w[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[32];
                if (c + 32 * h < t.c_end) {
                    tmem_ld32<0>(t.tmem + (uint32_t)(c + 32 * h), v);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = ex2(fmaf(v[i], kLog2e, -l2));
                const int k = lab_c - c - 32 * h;
                if (__any_sync(0xffffffffu, k >= 0 && k < 32)) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = k == i ? v[i] - head_g_scale(BF16) : v[i];
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) w[16 * h + i] = pack16<BF16>(v[2 * i] * f, v[2 * i + 1] * f);
            }
            pair_store16(t, w, c, g, ldg, n, min(t.N, t.col0 + t.c_end));
        }
    }
};

// dH of every token from the slabs (in their order), in 16 bits; zero for the
// tokens that took no part.
template <bool BF16>
__global__ void __launch_bounds__(256) head_dh_kernel(const float* __restrict__ slab, int64_t ld, int64_t split_stride,
                                                      int splits, const int* __restrict__ pos, int64_t n, int d,
                                                      const float* __restrict__ scale, uint16_t* __restrict__ out,
                                                      int64_t ldo) {
    const float a = *scale;
    for (int64_t t = blockIdx.x; t < n; t += gridDim.x) {
        const int p = pos[t];
        for (int c = threadIdx.x; c < d; c += blockDim.x) {
            float v = 0.0f;
            if (p >= 0) {
                for (int s = 0; s < splits; ++s) v += slab[s * split_stride + p * ld + c];
                v *= a;
            }
            out[t * ldo + c] = (uint16_t)pack16<BF16>(v, 0.0f);
        }
    }
}

}  // namespace aeth
