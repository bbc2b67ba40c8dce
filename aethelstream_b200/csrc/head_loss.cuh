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
// Forward and backward are bound by their products (four of 2 n V d operations;
// pair_gemm.cuh) down to some 300 tokens, below by the weight, read three times,
// and the writing of dW: 64 tokens x 4096 x 32000 58 + 177 us, of which the
// weight's bytes take 3 x 40 and dW's 62.
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
// to p = 2e-9 of the largest weight (6e-5 without); with k = 32 what fp32's and
// bf16's range cuts off is p < 2^-158, not 2^-126.
// f16 with token weights: what a token of 1e-6 of the largest weight has in G is
// cut off at p = 1e-6, which its row of dH may need.  dH is then taken from a
// second G without the weights, which multiply dH's rows at the end; dW, where
// the tokens are added up, keeps the first (each entry within 2^-40 of the
// largest weight).
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
    unsigned* done;  // zeroed: CTAs of head_loss_kernel that have finished
    // backward only (coef != null)
    const float* lse;   // per token
    const float* grad;  // per token, or null: 1 / count
    float scale, g_bits, g_scale;  // g_scale = 2^g_bits
    float* coef;       // live row -> g_t / max|g|
    float* lse2;       // live row -> lse * log2(e) - g_bits
    float* out_scale;  // max|g| / g_scale
    float* row_scale;  // live row -> |g_t| / g_scale
    // the live rows of H, gathered to a pitch that TMA takes
    const uint16_t* h;
    int64_t ld;
    int d;
    uint16_t* out;
    int64_t ldo;
};

// Copies rows of H (row r of the caller's list from `from(r)` to `to(r)`, zeros
// where from(r) < 0) with all threads of the CTA, four loads in flight.
template <typename From, typename To>
__device__ __forceinline__ void head_copy_rows(const HeadRows& a, int64_t nrows, From from, To to) {
    const bool whole = (a.ld % 8) == 0 && (a.d % 8) == 0 && (reinterpret_cast<uintptr_t>(a.h) & 15) == 0;
    if (whole) {
        const int nv = a.d / 8;
        for (int64_t i0 = threadIdx.x; i0 < nrows * nv; i0 += 4 * blockDim.x) {
            uint4 v[4];
            uint4* o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t i = i0 + (int64_t)k * blockDim.x;
                o[k] = nullptr;
                if (i < nrows * nv) {
                    const int64_t r = i / nv;
                    const int c = (int)(i - r * nv);
                    const int64_t src = from(r), dst = to(r);
                    v[k] = src >= 0 ? __ldg(reinterpret_cast<const uint4*>(a.h + src * a.ld) + c) : make_uint4(0, 0, 0, 0);
                    if (dst >= 0) o[k] = reinterpret_cast<uint4*>(a.out + dst * a.ldo) + c;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (o[k]) *o[k] = v[k];
        }
    } else {
        for (int64_t i = threadIdx.x; i < nrows * a.d; i += blockDim.x) {
            const int64_t r = i / a.d, src = from(r), dst = to(r);
            const int c = (int)(i - r * a.d);
            if (dst >= 0) a.out[dst * a.ldo + c] = src >= 0 ? a.h[src * a.ld + c] : (uint16_t)0;
        }
    }
}
// The products' last tiles read rows from the count up to the next multiple of
// 256: they are zero (past row n TMA itself fills with zero, without reading).
__device__ __forceinline__ int64_t head_padded(int live, int64_t n) {
    return min((int64_t)max((live + 255) / 256 * 256, 256), n);
}

// Numbers the live tokens in order (a scan over the labels, 8192 at a time, so
// that their loads are in flight together) and gathers what the epilogues need
// per live row.  CTA 0 writes that.  PACK (up to 8192 tokens): every CTA makes
// the scan for itself and then gathers its share of H's rows; more tokens take
// one CTA and head_pack_kernel behind it.
constexpr int kHeadScan = 8192;
template <bool PACK>
__global__ void __launch_bounds__(1024) head_rows_kernel(const __grid_constant__ HeadRows a, uint32_t* err) {
    constexpr int kItems = kHeadScan / 1024;
    __shared__ int wsum[kItems * 32];
    __shared__ float wmax[32];
    __shared__ int base_s;
    __shared__ int spos[PACK ? kHeadScan : 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool writes = blockIdx.x == 0;
    pdl_trigger();
    int base = 0;
    float gmax = 0.0f;
    for (int64_t t0 = 0; t0 < a.n; t0 += kHeadScan) {
        int64_t lab[kItems];
        float lse[kItems], grad[kItems];
        uint32_t m[kItems];
        const bool per_row = writes && a.coef;
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int64_t t = t0 + k * 1024 + tid;
            lab[k] = t < a.n ? a.labels[t] : a.ignore_index;
            lse[k] = per_row && t < a.n ? a.lse[t] : 0.0f;
            grad[k] = per_row && a.grad && t < a.n ? a.grad[t] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const bool live = lab[k] != a.ignore_index && lab[k] >= 0 && lab[k] < a.vocab;
            m[k] = __ballot_sync(0xffffffffu, live);
            if (lane == 0) wsum[k * 32 + warp] = __popc(m[k]);
        }
        __syncthreads();
        if (warp == 0) {  // exclusive scan of the 256 warp counts: eight a lane
            int v[kItems], s = 0;
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
                v[k] = s;
                s += wsum[lane * kItems + k];
            }
            int x = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
#pragma unroll
            for (int k = 0; k < kItems; ++k) wsum[lane * kItems + k] = x - s + v[k];
            if (lane == 31) base_s = x;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int64_t t = t0 + k * 1024 + tid;
            if (t >= a.n) continue;
            const bool live = (m[k] >> lane) & 1u;
            const int i = base + wsum[k * 32 + warp] + __popc(m[k] & ((1u << lane) - 1));
            if (PACK) spos[k * 1024 + tid] = live ? i : kHeadIgnored;
            if (!writes) continue;
            if (!live) {
                const bool bad = lab[k] != a.ignore_index;
                if (bad) report_dev_error(err, DEVERR_BAD_ARG);
                a.pos[t] = bad ? kHeadBad : kHeadIgnored;
                continue;
            }
            a.pos[t] = i;
            a.rows[i] = (int)t;
            a.lab[i] = (int)lab[k];
            if (a.coef) {
                a.lse2[i] = fmaf(lse[k], kLog2e, -a.g_bits);
                if (a.grad) {
                    const float g = grad[k] * a.scale;
                    a.coef[i] = g;
                    a.row_scale[i] = fabsf(g) / a.g_scale;
                    if (fabsf(g) <= 3.402823466e38f) gmax = fmaxf(gmax, fabsf(g));  // what is not finite stays its token's
                }
            }
        }
        base += base_s;
        __syncthreads();
    }
    if (PACK) {
        const int64_t g = gridDim.x, b = blockIdx.x, first = base + b;
        head_copy_rows(a, (a.n - b + g - 1) / g, [&](int64_t r) { return b + r * g; },
                       [&](int64_t r) { return (int64_t)spos[b + r * g]; });
        const int64_t padded = head_padded(base, a.n);
        if (first < padded)
            head_copy_rows(a, (padded - first + g - 1) / g, [](int64_t) { return (int64_t)-1; },
                           [&](int64_t r) { return first + r * g; });
    }
    if (!writes) return;
    if (tid == 0) {
        *a.count = base;
        *a.done = 0;
    }
    if (!a.coef) return;
    if (a.grad) {
        gmax = warp_max(gmax);
        if (lane == 0) wmax[warp] = gmax;
        __syncthreads();
        gmax = warp_max(wmax[lane]);
        for (int i = tid; i < base; i += 1024) {
            const float g = a.coef[i];
            a.coef[i] = g == 0.0f ? 0.0f : g / gmax;
        }
    } else {
        const float g = a.scale / (float)max(base, 1);
        gmax = fabsf(g);
        for (int i = tid; i < base; i += 1024) a.coef[i] = g == 0.0f ? 0.0f : g / gmax;
    }
    if (tid == 0) *a.out_scale = gmax / a.g_scale;
}

// The gathering alone, after the scan (more than kHeadScan tokens).
__global__ void __launch_bounds__(1024) head_pack_kernel(const __grid_constant__ HeadRows a) {
    pdl_wait();
    pdl_trigger();
    const int live = *a.count;
    const int64_t padded = head_padded(live, a.n), g = gridDim.x, b = blockIdx.x;
    if (b < padded)
        head_copy_rows(a, (padded - b + g - 1) / g,
                       [&](int64_t r) { return b + r * g < live ? (int64_t)a.rows[b + r * g] : -1; },
                       [&](int64_t r) { return b + r * g; });
}

// Joins two (maximum, sum) pairs.
__device__ __forceinline__ float2 head_join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), off = m == -INFINITY ? 0.0f : m;
    return make_float2(m, a.y * ex2(a.x - off) + b.y * ex2(b.x - off));
}
__device__ __forceinline__ float head_lse(float2 a) {
    return (a.x == -INFINITY ? 0.0f : a.x) * kLn2 + logf(a.y);
}

// Joins 32 logits (the first `left` of them) to a running maximum, in units of
// log2, and sum of 2^(logit log2 e - maximum).
__device__ __forceinline__ void head_stats32(const float (&v)[32], int left, float2& st) {
    float m = -INFINITY;
    if (left >= 32) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) m = fmax3(m, v[i], v[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < left) m = fmaxf(m, v[i]);
    }
    const float nm = fmaxf(st.x, m * kLog2e);
    const float off = nm == -INFINITY ? 0.0f : nm;
    float s0 = 0.0f, s1 = 0.0f;
    if (left >= 32) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            s0 += ex2(fmaf(v[i], kLog2e, -off));
            s1 += ex2(fmaf(v[i + 1], kLog2e, -off));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < left) s0 += ex2(fmaf(v[i], kLog2e, -off));
    }
    st = make_float2(nm, st.y * ex2(st.x - off) + (s0 + s1));
}
// v[k] where some lane's k lies in the 32
__device__ __forceinline__ void head_label32(const float (&v)[32], int k, float* out) {
    if (!__any_sync(0xffffffffu, k >= 0 && k < 32)) return;
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) x = k == i ? v[i] : x;
    if (k >= 0 && k < 32) *out = x;
}
__device__ __forceinline__ void head_slice(const float (&acc)[128], int c, float (&v)[32]) {  // c known when unrolled
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = acc[32 * c + i];
}

// Epilogue of the forward product: per row, over this warp's columns, the
// maximum and sum, and the label's logit where it lies here.
struct HeadStats {
    static constexpr int kChunk = 8;  // the loss is an fp32 result: see pair_gemm.cuh
    static constexpr bool kLiveN = false;
    const int* lab;
    float* label_logit;
    float2* part;  // [2 * n_tile + half][row]
    int64_t ld_part;
    __device__ static void give_up(const PairTile&) {}
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
        const int row = t.row0 + t.lane;
        const bool in = row < t.M;
        const int at = in ? lab[row] - t.col0 - t.c_begin : -1;
        float2 st = make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int left = min(t.c_end, t.N - t.col0) - t.c_begin - 32 * c;  // columns of this chunk that exist
            if (left > 0) {
                float v[32];
                head_slice(acc, c, v);
                head_stats32(v, left, st);
                head_label32(v, at - 32 * c, label_logit + row);
            }
        }
        if (in) part[(int64_t)(2 * t.n_tile + t.half) * ld_part + row] = st;
    }
};

// The same with tokens as the tile's columns (few live rows) and vocabulary
// entries as its rows: a warp has 32 entries; the four warps of a column half
// join theirs through shared memory.
struct HeadStatsT {
    static constexpr int kChunk = 8;
    static constexpr bool kLiveN = true;
    const int* lab;
    float* label_logit;
    float2* part;  // [2 * m_tile + CTA of the pair][row]
    int64_t ld_part;
    // The two barriers of finish(), each with an id of its own: a barrier counts
    // arrivals, so two at one id could both fall into its first wait.  A warp that
    // leaves waits for nobody, since the others may never come to its next tile's.
    __device__ static void give_up(const PairTile& t) {
        named_bar_arrive(1 + t.half, 128);
        named_bar_arrive(3 + t.half, 128);
    }
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
        const int left = t.M - t.row0;  // entries of this warp that exist
        float2 st[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            st[c] = make_float2(-INFINITY, 0.0f);
            const int token = t.col0 + t.c_begin + 32 * c + t.lane;
            if (t.c_begin + 32 * c < t.c_end && left > 0) {
                float v[32];
                head_slice(acc, c, v);
                pair_transpose(t, v);
                head_stats32(v, left, st[c]);
                const int k = token < t.N ? lab[token] - t.row0 : -1;
                head_label32(v, k < left ? k : -1, label_logit + token);
            }
        }
        float2* mine = reinterpret_cast<float2*>(t.staging);
#pragma unroll
        for (int c = 0; c < 4; ++c) mine[32 * c + t.lane] = st[c];
        named_bar(1 + t.half, 128);
        // warp `e` of the half takes its 32 columns c = e
        const int e = t.warp & 3;
        const float2* all = reinterpret_cast<const float2*>(t.staging - e * kPairStaging);
        float2 x = all[32 * e + t.lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) x = head_join(x, all[w * (kPairStaging / 8) + 32 * e + t.lane]);
        const int col = t.c_begin + 32 * e + t.lane;
        if (col < t.c_end && t.col0 + col < t.N)
            part[(int64_t)(2 * t.m_tile + (t.tile_row >> 7)) * ld_part + t.col0 + col] = x;
        named_bar(3 + t.half, 128);
    }
};

// Joins the column ranges' maxima and sums.  A CTA takes 8 live rows (lane % 8),
// its 64 quarter-warps every 64th range, four loads in flight; then a tree.
// The CTA that finishes last settles the tokens that take no part (loss 0; NaN
// for a label outside the vocabulary) and the mean over the live ones, summed
// in one fixed order.
struct HeadLoss {
    const float2* part;
    int64_t ld_part;
    int np;
    const float* label_logit;
    const int *rows, *pos, *count;
    unsigned* done;
    int64_t n;
    float *losses, *lse, *loss;
};
__global__ void __launch_bounds__(512) head_loss_kernel(const HeadLoss a) {
    __shared__ float2 sh[16][8];
    __shared__ double ws[16];
    __shared__ bool last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    const int live = *a.count;
    for (int64_t r0 = (int64_t)blockIdx.x * 8; r0 < live; r0 += (int64_t)gridDim.x * 8) {
        const int64_t row = r0 + (lane & 7);
        float2 x = make_float2(-INFINITY, 0.0f);
        for (int p0 = warp * 4 + (lane >> 3); p0 < a.np; p0 += 256) {
            float2 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v[k] = p0 + 64 * k < a.np && row < live ? a.part[(p0 + 64 * k) * a.ld_part + row]
                                                        : make_float2(-INFINITY, 0.0f);
            x = head_join(x, head_join(head_join(v[0], v[1]), head_join(v[2], v[3])));
        }
#pragma unroll
        for (int o = 8; o < 32; o <<= 1)
            x = head_join(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
        if (lane < 8) sh[warp][lane] = x;
        __syncthreads();
        if (warp == 0) {
            x = sh[lane >> 3][lane & 7];
#pragma unroll
            for (int w = 4; w < 16; w += 4) x = head_join(x, sh[w + (lane >> 3)][lane & 7]);
#pragma unroll
            for (int o = 8; o < 32; o <<= 1)
                x = head_join(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
            if (lane < 8 && row < live) {
                const float l = head_lse(x);
                const int t = a.rows[row];
                a.lse[t] = l;
                a.losses[t] = l - a.label_logit[row];
            }
        }
        __syncthreads();
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(a.done, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    double s = 0.0;
    for (int64_t t = threadIdx.x; t < a.n; t += 512) {
        const int p = a.pos[t];
        if (p < 0) {
            const float v = p == kHeadBad ? __int_as_float(0x7fc00000) : 0.0f;
            a.losses[t] = a.lse[t] = v;
            s += (double)v;
        } else {
            s += (double)__ldcg(a.losses + t);
        }
    }
    s = warp_sum_d(s);
    if (lane == 0) ws[warp] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = warp_sum_d(threadIdx.x < 16 ? ws[threadIdx.x] : 0.0);
        if (threadIdx.x == 0) *a.loss = (float)(s / (double)max(live, 1));
    }
}

// Forward of one to four tokens: a product that reads the weight once and does
// little else, so the bytes in flight and their order in DRAM decide.  A warp
// takes two vocabulary entries at a time, each a row read from its start to its
// end (512 bytes an instruction, sixteen in flight), against the tokens' hidden
// states in shared memory; it keeps their running maximum and sum and leaves
// one pair per token and CTA.  One token x 4096 x 32000: 46 us a call, 5.7 TB/s
// (6.3 at 2048 x 131071); the tile product takes 57, its columns of 128 bytes
// and its launches included.
constexpr int kHeadVecTokens = 4, kHeadVecThreads = 512;

struct HeadVec {
    const uint16_t* hidden;
    int64_t ld_h;
    const uint16_t* weight;
    int64_t ld_w;
    const int64_t* labels;
    int d, vocab;
    int64_t ignore_index;
    float* label_logit;  // [token]
    float2* part;        // [CTA][token]
};

// Weight rows are read once, in order: past L1, 256 bytes at a time into L2
// (plain loads: 52 us where this takes 44, one token at 4096 x 32000).
__device__ __forceinline__ uint4 head_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
template <bool BF16>
__device__ __forceinline__ float2 head_pair(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <bool BF16, int NT>
__global__ void __launch_bounds__(kHeadVecThreads, 1) head_vec_kernel(const HeadVec a) {
    constexpr int R = 2, U = 8;  // entries a warp, loads in flight an entry
    extern __shared__ uint4 head_sh[];  // [token][eight of features]
    __shared__ float2 red[kHeadVecThreads / 32][NT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, eights = (a.d + 7) / 8;
    const int64_t first = (int64_t)R * (blockIdx.x * (kHeadVecThreads / 32) + warp);
    // the warp's first entries are on their way to L2 while the hidden states are staged
    for (int r = 0; r < R; ++r)
        for (int b = lane * 128; b < 2 * a.d && first + r < a.vocab; b += 4096)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(a.weight + (first + r) * a.ld_w) + b));
    uint16_t* sh16 = reinterpret_cast<uint16_t*>(head_sh);
    for (int i = threadIdx.x; i < NT * eights * 8; i += kHeadVecThreads) {
        const int t = i / (eights * 8), c = i - t * eights * 8;
        sh16[i] = c < a.d ? a.hidden[t * a.ld_h + c] : (uint16_t)0;
    }
    int lab[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t l = a.labels[t];
        lab[t] = l != a.ignore_index && l >= 0 && l < a.vocab ? (int)l : -1;
    }
    __syncthreads();
    float2 st[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) st[t] = make_float2(-INFINITY, 0.0f);
    pdl_trigger();
    const int warps = gridDim.x * (kHeadVecThreads / 32);
    for (int64_t v0 = first; v0 < a.vocab; v0 += (int64_t)R * warps) {
        const uint16_t* row[R];
#pragma unroll
        for (int r = 0; r < R; ++r) row[r] = a.weight + min(v0 + r, (int64_t)a.vocab - 1) * a.ld_w;
        float2 acc[R][NT];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[r][t] = make_float2(0.0f, 0.0f);
        for (int e0 = lane; e0 < eights; e0 += 32 * U) {
            uint4 w[R][U];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    w[r][u] = e0 + 32 * u < eights ? head_stream(reinterpret_cast<const uint4*>(row[r]) + e0 + 32 * u)
                                                   : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int e = e0 + 32 * u;
                if (e >= eights) break;
                if (8 * e + 8 > a.d) {  // the row's last eight: nothing past its end
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        uint32_t* x = reinterpret_cast<uint32_t*>(&w[r][u]);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (8 * e + i >= a.d) x[i >> 1] &= (i & 1) ? 0x0000ffffu : 0xffff0000u;
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint4 h = head_sh[t * eights + e];
                    const uint32_t hw[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const uint32_t ww[4] = {w[r][u].x, w[r][u].y, w[r][u].z, w[r][u].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[r][t] = fma2_rn(head_pair<BF16>(ww[i]), head_pair<BF16>(hw[i]), acc[r][t]);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float x = acc[r][t].x + acc[r][t].y;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                if (v0 + r < a.vocab) {
                    st[t] = head_join(st[t], make_float2(x * kLog2e, 1.0f));
                    if (lab[t] == v0 + r && lane == 0) a.label_logit[t] = x;
                }
            }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
        if (lane == 0) red[warp][t] = st[t];
    __syncthreads();
    if (threadIdx.x < NT) {
        float2 x = red[0][threadIdx.x];
        for (int w = 1; w < kHeadVecThreads / 32; ++w) x = head_join(x, red[w][threadIdx.x]);
        a.part[(int64_t)blockIdx.x * NT + threadIdx.x] = x;
    }
}

// One warp a token joins the CTAs' pairs; then losses and mean.
__global__ void __launch_bounds__(32 * kHeadVecTokens)
    head_vec_loss_kernel(const HeadVec a, int n, int ctas, float* losses, float* lse, float* loss, uint32_t* err) {
    __shared__ float sl[kHeadVecTokens];
    __shared__ int sc[kHeadVecTokens];
    const int t = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    float2 x = make_float2(-INFINITY, 0.0f);
    for (int p0 = lane; p0 < ctas; p0 += 128) {
        float2 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            v[k] = p0 + 32 * k < ctas ? a.part[(int64_t)(p0 + 32 * k) * n + t] : make_float2(-INFINITY, 0.0f);
        x = head_join(x, head_join(head_join(v[0], v[1]), head_join(v[2], v[3])));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        x = head_join(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
    if (lane == 0) {
        const int64_t lab = a.labels[t];
        const bool in = lab != a.ignore_index, bad = in && (lab < 0 || lab >= a.vocab);
        const float l = in ? head_lse(x) : 0.0f;
        lse[t] = bad ? __int_as_float(0x7fc00000) : l;
        losses[t] = sl[t] = bad ? __int_as_float(0x7fc00000) : in ? l - a.label_logit[t] : 0.0f;
        sc[t] = in && !bad;
        if (bad) report_dev_error(err, DEVERR_BAD_ARG);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        int count = 0;
        for (int i = 0; i < n; ++i) {
            s += (double)sl[i];
            count += sc[i];
        }
        *loss = (float)(s / (double)max(count, 1));
    }
}

// A token weight's part in the G without weights: its sign (NaN and 0 stay).
__device__ __forceinline__ float head_unit(float f) { return f > 0.0f ? 1.0f : f < 0.0f ? -1.0f : f; }

// Epilogue of the backward's product: G of the piece in 16 bits, as the tensor
// cores take it for dW and dH.  G is rounded once, from fp32, which a sum over many
// tokens or entries evens out (against 64 bits 1.9e-3 in bf16, 1.7e-3 of it the
// output's own rounding); in dW of one token, all but an outer product, it stands
// beside that rounding.  Rows from the count to the tile's end (or n) become zero.  The
// logits are added up as in the forward, so that they are those that lse came
// from: taken whole, one of 30 made of 8192 products is 2.3e-4 too small, which
// is all of p - 1 for a label known with p = 0.9998.  That costs 1.4 to 2.4 % of a
// large backward (8192 x 8192 x 32000: 10.03 -> 10.18 ms, power-capped; 3584 x 4096
// x 32000: 2.13 -> 2.19) and 6 to 13 us of one of 130 to 311 tokens (160 to 260 us).
// UNIT (f16): the G without token weights, beside the other where that is wanted
// (3584 x 4096 x 32000 with weights: 2.26 -> 2.42 ms, 64 tokens 178 -> 183 us).
template <bool BF16, bool UNIT>
struct HeadGrad {
    static constexpr int kChunk = 8;
    static constexpr bool kLiveN = false;
    const int* lab;
    const float* coef;
    const float* lse2;
    uint16_t* g;       // with UNIT: or null
    uint16_t* g_unit;  // with UNIT
    int64_t ldg;
    int n;   // rows of g: the tokens
    int v0;  // first vocabulary entry of the piece
    __device__ static void give_up(const PairTile&) {}
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
        const int row = t.row0 + t.lane;
        const bool in = row < t.M;
        const float f = in ? coef[row] : 0.0f, u = head_unit(f), l2 = in ? lse2[row] : 0.0f;
        const int lab_c = in ? lab[row] - v0 - t.col0 - t.c_begin : -1;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int c = t.c_begin + 64 * b;
            if (c < t.c_end && t.col0 + c < t.N && t.row0 < n) {
                uint32_t w[32], w1[32];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[32];
                    head_slice(acc, 2 * b + h, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = ex2(fmaf(v[i], kLog2e, -l2));
                    const int k = lab_c - 64 * b - 32 * h;
                    if (__any_sync(0xffffffffu, k >= 0 && k < 32)) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = k == i ? v[i] - head_g_scale(BF16) : v[i];
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        w[16 * h + i] = pack16<BF16>(v[2 * i] * f, v[2 * i + 1] * f);
                        if (UNIT) w1[16 * h + i] = pack16<BF16>(v[2 * i] * u, v[2 * i + 1] * u);
                    }
                }
                const int cols = min(t.N, t.col0 + t.c_end);
                if (!UNIT || g) pair_store16(t, w, c, g, ldg, n, cols);
                if (UNIT) pair_store16(t, w1, c, g_unit, ldg, n, cols);
            }
        }
    }
};

// The same with tokens as the tile's columns: each 32 x 32 block is turned over,
// so that a thread has a token and 32 entries.
template <bool BF16, bool UNIT>
struct HeadGradT {
    static constexpr int kChunk = 8;
    static constexpr bool kLiveN = true;
    const int* lab;
    const float* coef;
    const float* lse2;
    uint16_t* g;
    uint16_t* g_unit;
    int64_t ldg;
    int n;
    int v0;
    __device__ static void give_up(const PairTile&) {}
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int c = t.c_begin + 32 * b;
            if (c >= t.c_end || t.row0 >= t.M || t.col0 + c >= n) continue;
            float v[32];
            head_slice(acc, b, v);
            pair_transpose(t, v);
            const int token = t.col0 + c + t.lane;
            const bool in = token < t.N;
            const float f = in ? coef[token] : 0.0f, u = head_unit(f), l2 = in ? lse2[token] : 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = ex2(fmaf(v[i], kLog2e, -l2));
            const int k = in ? lab[token] - v0 - t.row0 : -1;
            if (__any_sync(0xffffffffu, k >= 0 && k < 32)) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = k == i ? v[i] - head_g_scale(BF16) : v[i];
            }
            uint32_t w[16], w1[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[i] = pack16<BF16>(v[2 * i] * f, v[2 * i + 1] * f);
                if (UNIT) w1[i] = pack16<BF16>(v[2 * i] * u, v[2 * i + 1] * u);
            }
            if (!UNIT || g) store(t, w, c, g);
            if (UNIT) store(t, w1, c, g_unit);
        }
    }
    // 32 tokens (columns c .. of the tile) x 32 entries, thread = token
    __device__ __forceinline__ void store(const PairTile& t, const uint32_t (&w)[16], int c, uint16_t* out) const {
        const bool whole = (ldg % 8) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
        // 64 bytes a token; piece p (16 bytes) of token r lies at p ^ (r / 2) % 4
#pragma unroll
        for (int p = 0; p < 4; ++p)
            *reinterpret_cast<uint4*>(t.staging + t.lane * 64 + ((p ^ ((t.lane >> 1) & 3)) * 16)) =
                make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (t.lane >> 2), p = t.lane & 3;
            const int gr = t.col0 + c + r, gc = t.row0 + p * 8;
            const uint4 x = *reinterpret_cast<const uint4*>(t.staging + r * 64 + ((p ^ ((r >> 1) & 3)) * 16));
            if (gr < n && gc < t.M) {
                uint16_t* o = out + (int64_t)gr * ldg + gc;
                if (whole && gc + 8 <= t.M) {
                    *reinterpret_cast<uint4*>(o) = x;
                } else {
                    const uint32_t xx[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (gc + q < t.M) o[q] = (uint16_t)(xx[q >> 1] >> (16 * (q & 1)));
                }
            }
        }
        __syncwarp();
    }
};

// dH of every token in 16 bits: the slab's row, plus the further K ranges of
// the tail's tiles in their order; zero for the tokens that took no part.  A
// CTA takes 1024 columns of tokens, TOKENS of them in flight.
struct HeadDh {
    const float* slab;
    int64_t ld;
    const float* extra;
    int pairs, tail_kb, live_n;  // live_n: tokens were the product's columns
    const int *pos, *count;
    int64_t n;
    int d;
    const float* scale;      // one for all, or null
    const float* row_scale;  // else a live row's
    uint16_t* out;
    int64_t ldo;
};
template <bool BF16, int TOKENS>
__global__ void __launch_bounds__(128) head_dh_kernel(const HeadDh a) {
    __shared__ int sh[5];
    pdl_wait();
    if (threadIdx.x < 32) {
        const int count = *a.count, tiles_d = (a.d + 255) / 256;
        const int bt = a.live_n ? pair_live_bn(count) : 256, tiles_t = max((count + bt - 1) / bt, 1);
        const PairTail t(tiles_t * tiles_d, a.pairs, a.tail_kb);
        sh[0] = bt;
        sh[1] = tiles_t;
        sh[2] = t.full;
        sh[3] = t.rest;
        sh[4] = t.splits;
    }
    __syncthreads();
    const int bt = sh[0], tiles_t = sh[1], full = sh[2], rest = sh[3], splits = sh[4], tiles_d = (a.d + 255) / 256;
    const float scale_all = a.scale ? *a.scale : 0.0f;
    const int c = (blockIdx.y * 128 + threadIdx.x) * 8;
    if (c >= a.d) return;
    const bool whole = (a.ldo % 8) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && c + 8 <= a.d;
    for (int64_t t0 = blockIdx.x; t0 < a.n; t0 += TOKENS * (int64_t)gridDim.x) {
        float4 v[TOKENS][2];
        int p[TOKENS];
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
            const int64_t t = t0 + (int64_t)k * gridDim.x;
            p[k] = t < a.n ? a.pos[t] : kHeadIgnored;
#pragma unroll
            for (int h = 0; h < 2; ++h)  // ld is a multiple of 8
                v[k][h] = p[k] >= 0 ? *reinterpret_cast<const float4*>(a.slab + p[k] * a.ld + c + 4 * h)
                                    : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
            const int64_t t = t0 + (int64_t)k * gridDim.x;
            if (t >= a.n) break;
            if (p[k] >= 0) {
                const int i = (a.live_n ? pair_tile_index(c / 256, p[k] / bt, tiles_d, tiles_t)
                                        : pair_tile_index(p[k] / bt, c / 256, tiles_t, tiles_d)) - full;
                if (i >= 0) {
                    const float* e = a.extra + ((int64_t)i * 256 + p[k] % bt) * 256 + c % 256;
#pragma unroll(TOKENS == 1 ? 12 : 4)
                    for (int s = 0; s + 1 < splits; ++s)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float4 x = *reinterpret_cast<const float4*>(e + (int64_t)s * rest * 65536 + 4 * h);
                            v[k][h] = make_float4(v[k][h].x + x.x, v[k][h].y + x.y, v[k][h].z + x.z, v[k][h].w + x.w);
                        }
                }
            }
            uint32_t w[4] = {0, 0, 0, 0};
            const float scale = a.scale || p[k] < 0 ? scale_all : a.row_scale[p[k]];
            if (p[k] >= 0)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    w[2 * h] = pack16<BF16>(v[k][h].x * scale, v[k][h].y * scale);
                    w[2 * h + 1] = pack16<BF16>(v[k][h].z * scale, v[k][h].w * scale);
                }
            uint16_t* o = a.out + t * a.ldo + c;
            if (whole) {
                *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (c + q < a.d) o[q] = (uint16_t)(w[q >> 1] >> (16 * (q & 1)));
            }
        }
    }
}

}  // namespace aeth
