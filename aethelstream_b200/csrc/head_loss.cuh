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
    int* count;  // live rows; of the gradient of log probabilities also, after it, rows that a token has
    unsigned* done;  // zeroed: CTAs of head_loss_kernel that have finished
    // backward only (coef != null)
    const float* lse;   // per token
    const float* grad;  // per token, or null: 1 / count
    float scale, g_bits, g_scale;  // g_scale = 2^g_bits
    float* coef;       // live row -> g_t / max|g|
    float* lse2;       // live row -> lse * log2(e) - g_bits
    float* out_scale;  // max|g| / g_scale
    float* row_scale;  // live row -> |g_t| / g_scale
    // the gradient of log probabilities and entropies in its place (head_probs.cuh; row != null)
    const float *entropy, *grad_entropy;
    float bound;  // of |p (log p + entropy)|
    float4* row;
    int64_t room;  // rows of G (the loss: tokens)
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

// A live row of the gradient of a log p_y + b entropy: its weight w = |a| + c |b|
// (returned, and for now in row[].w) and, of a / w and b / w, what an entry takes
// (HeadRowGrad).
__device__ __forceinline__ float head_probs_row(const HeadRows& a, int64_t t, int i, int lab) {
    const float ga = a.grad ? a.grad[t] : 0.0f, gb = a.grad_entropy ? a.grad_entropy[t] : 0.0f;
    const float w = fmaf(a.bound, fabsf(gb), fabsf(ga));
    const float ua = w == 0.0f ? 0.0f : ga / w, ub = w == 0.0f ? 0.0f : gb / w, gamma = ub * kLn2;
    a.lab[i] = lab;
    a.lse2[i] = a.lse[t];
    a.row_scale[i] = w / a.g_scale;
    a.row[i] = make_float4(ua * a.g_scale, fmaf(-gamma, a.g_bits, fmaf(ub, a.entropy[t], ua)), gamma, w);
    return w;
}

// Up to how many live tokens the gradient of log probabilities has two rows of G for
// each (HeadGrad says what that gives and costs).  By the live ones, whose number is
// known on the device alone, so that a padded batch has the gradient of its tokens.
constexpr int kHeadTwice = 128;

// Numbers the live tokens in order (a scan over the labels, 8192 at a time, so
// that their loads are in flight together) and gathers what the epilogues need
// per live row.  CTA 0 writes that.  PROBS: for a gradient of log probabilities and
// entropies (head_probs_row).  PACK (up to 8192 tokens): every CTA makes
// the scan for itself and then gathers its share of H's rows; more tokens take
// one CTA and head_pack_kernel behind it.  Live token i has row i of what it writes,
// or rows 2 i and 2 i + 1 (kHeadTwice).
constexpr int kHeadScan = 8192;
template <bool PACK, bool PROBS>
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
            if (!PROBS) a.lab[i] = (int)lab[k];
            if (PROBS) {
                const float w = head_probs_row(a, t, i, (int)lab[k]);
                if (w <= 3.402823466e38f) gmax = fmaxf(gmax, w);
            } else if (a.coef) {
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
    const bool twice = PROBS && base <= kHeadTwice;
    const int count = twice ? 2 * base : base;
    if (PACK) {
        const int64_t g = gridDim.x, b = blockIdx.x, first = count + b;
        const int64_t mine = (a.n - b + g - 1) / g;
        auto from = [&](int64_t r) { return b + r * g; };
        if (twice) {
            head_copy_rows(a, 2 * mine, [&](int64_t r) { return from(r / 2); }, [&](int64_t r) {
                const int64_t to = spos[from(r / 2)];
                return to >= 0 ? 2 * to + r % 2 : to;
            });
        } else {
            head_copy_rows(a, mine, from, [&](int64_t r) { return (int64_t)spos[from(r)]; });
        }
        const int64_t padded = head_padded(count, a.room);
        if (first < padded)
            head_copy_rows(a, (padded - first + g - 1) / g, [](int64_t) { return (int64_t)-1; },
                           [&](int64_t r) { return first + r * g; });
    }
    if (!writes) return;
    if (tid == 0) {
        a.count[0] = count;
        if (PROBS) a.count[1] = twice ? 2 : 1;
        *a.done = 0;
    }
    if (PROBS) {
        gmax = warp_max(gmax);
        if (lane == 0) wmax[warp] = gmax;
        __syncthreads();
        gmax = warp_max(wmax[lane]);
        if (tid == 0) *a.out_scale = gmax / a.g_scale;
        if (!twice) {
            for (int i = tid; i < base; i += 1024) {
                const float w = a.row[i].w;
                a.row[i].w = w == 0.0f ? 0.0f : w / gmax;
            }
            return;
        }
        const bool mine = tid < base;  // base <= kHeadTwice < 1024
        float4 row = mine ? a.row[tid] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const int label = mine ? a.lab[tid] : 0;
        const float row_lse = mine ? a.lse2[tid] : 0.0f, scale = mine ? a.row_scale[tid] : 0.0f;
        row.w = row.w == 0.0f ? 0.0f : row.w / gmax;
        __syncthreads();
        if (mine) {
            a.pos[a.rows[tid]] = 2 * tid;
            for (int r = 2 * tid; r < 2 * tid + 2; ++r) {
                a.row[r] = row;
                a.lab[r] = label;
                a.lse2[r] = row_lse;
                a.row_scale[r] = scale;
            }
        }
        return;
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
    const int live = *a.count, half = a.row && a.count[1] == 2 ? 1 : 0;
    const int64_t padded = head_padded(live, a.room), g = gridDim.x, b = blockIdx.x;
    if (b < padded)
        head_copy_rows(a, (padded - b + g - 1) / g,
                       [&](int64_t r) { return b + r * g < live ? (int64_t)a.rows[(b + r * g) >> half] : -1; },
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

// What the forward's epilogues keep of a row and range: the loss's maximum and sum
// of exponentials.  `Sums` of the epilogues; head_probs.cuh has another.
struct HeadLossSums {
    using Sum = float2;
    float2* part;  // [range][row]
    int64_t ld_part;
    __device__ static Sum none() { return make_float2(-INFINITY, 0.0f); }
    // what a row's 128 logits are added to, the first `left` of which exist
    __device__ static Sum before(const float (&)[128], int) { return none(); }
    // whether a row's sums are good, or its logits are added once more the other way
    __device__ static bool good(Sum) { return true; }
    __device__ static Sum join(Sum a, Sum b) { return head_join(a, b); }
    __device__ __forceinline__ static void add32(const float (&v)[32], int left, Sum& st) { head_stats32(v, left, st); }
    __device__ __forceinline__ static void again32(const float (&v)[32], int left, Sum& st) { head_stats32(v, left, st); }
    __device__ __forceinline__ void put(int range, int row, Sum x) const { part[(int64_t)range * ld_part + row] = x; }
    // 32 columns of the warp's rows, and 32 entries of a token (none of them kept)
    __device__ __forceinline__ void rows(const PairTile&, const float (&)[32], int) const {}
    __device__ __forceinline__ void token(int, int, int, const float (&)[32]) const {}
};

// Epilogue of the forward product: per row, over this warp's columns, the
// maximum and sum, and the label's logit where it lies here.
template <class Sums>
struct HeadStats {
    static constexpr int kChunk = 8;  // the loss is an fp32 result: see pair_gemm.cuh
    static constexpr bool kLiveN = false;
    const int* lab;
    float* label_logit;
    int v0;  // first entry of the product's columns
    Sums sums;  // range: 2 * n_tile + half
    __device__ static void give_up(const PairTile&) {}
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
        const int row = t.row0 + t.lane;
        const bool in = row < t.M;
        const int at = in ? lab[row] - v0 - t.col0 - t.c_begin : -1;
        const int all = min(t.c_end, t.N - t.col0) - t.c_begin;  // columns that exist
        typename Sums::Sum st = Sums::before(acc, all);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int left = all - 32 * c;
            if (left > 0) {
                float v[32];
                head_slice(acc, c, v);
                Sums::add32(v, left, st);
                head_label32(v, at - 32 * c, label_logit + row);
                sums.rows(t, v, t.c_begin + 32 * c);
            }
        }
        if (__any_sync(0xffffffffu, !Sums::good(st))) {
            typename Sums::Sum other = Sums::none();
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (all - 32 * c > 0) {
                    float v[32];
                    head_slice(acc, c, v);
                    Sums::again32(v, all - 32 * c, other);
                }
            if (!Sums::good(st)) st = other;
        }
        if (in) sums.put(2 * t.n_tile + t.half, row, st);
    }
};

// The same with tokens as the tile's columns (few live rows) and vocabulary
// entries as its rows: a warp has 32 entries; the four warps of a column half
// join theirs through shared memory.
template <class Sums>
struct HeadStatsT {
    static constexpr int kChunk = 8;
    static constexpr bool kLiveN = true;
    const int* lab;
    float* label_logit;
    int v0;
    Sums sums;  // range: 2 * m_tile + CTA of the pair
    // The two barriers of finish(), each with an id of its own: a barrier counts
    // arrivals, so two at one id could both fall into its first wait.  A warp that
    // leaves waits for nobody, since the others may never come to its next tile's.
    __device__ static void give_up(const PairTile& t) {
        named_bar_arrive(1 + t.half, 128);
        named_bar_arrive(3 + t.half, 128);
    }
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
        using Sum = typename Sums::Sum;
        const int left = t.M - t.row0;  // entries of this warp that exist
        Sum st[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            st[c] = Sums::none();
            const int token = t.col0 + t.c_begin + 32 * c + t.lane;
            if (t.c_begin + 32 * c < t.c_end && left > 0) {
                float v[32];
                head_slice(acc, c, v);
                pair_transpose(t, v);
                Sums::again32(v, left, st[c]);
                const int k = token < t.N ? lab[token] - v0 - t.row0 : -1;
                head_label32(v, k < left ? k : -1, label_logit + token);
                if (token < t.N) sums.token(token, t.row0, left, v);
            }
        }
        Sum* mine = reinterpret_cast<Sum*>(t.staging);
#pragma unroll
        for (int c = 0; c < 4; ++c) mine[32 * c + t.lane] = st[c];
        named_bar(1 + t.half, 128);
        // warp `e` of the half takes its 32 columns c = e
        const int e = t.warp & 3;
        const Sum* all = reinterpret_cast<const Sum*>(t.staging - e * kPairStaging);
        Sum x = all[32 * e + t.lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) x = Sums::join(x, all[w * (kPairStaging / (int)sizeof(Sum)) + 32 * e + t.lane]);
        const int col = t.c_begin + 32 * e + t.lane;
        if (col < t.c_end && t.col0 + col < t.N) sums.put(2 * t.m_tile + (t.tile_row >> 7), t.col0 + col, x);
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

// Stages the hidden states ([token][eight of features]), calls begin() behind a
// barrier and then logit(token, entry, its place, its logit) with all lanes of a
// warp, for the entries that are the warp's: two in turn, from 2 (CTA's warps +
// warp) on.  place: the entry's among the CTA's.
template <bool BF16, int NT, typename Begin, typename Logit>
__device__ __forceinline__ void head_vec_walk(const HeadVec& a, uint4* head_sh, Begin begin, Logit logit) {
    constexpr int R = 2, U = 8;  // entries a warp, loads in flight an entry
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
    begin();
    __syncthreads();
    pdl_trigger();
    const int warps = gridDim.x * (kHeadVecThreads / 32);
    int place = R * warp;
    for (int64_t v0 = first; v0 < a.vocab; v0 += (int64_t)R * warps, place += R * kHeadVecThreads / 32) {
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
                if (v0 + r < a.vocab) logit(t, (int)(v0 + r), place + r, x);
            }
    }
}
// The label of token t where it takes part, else -1.
__device__ __forceinline__ int head_vec_label(const HeadVec& a, int t) {
    const int64_t l = a.labels[t];
    return l != a.ignore_index && l >= 0 && l < a.vocab ? (int)l : -1;
}

template <bool BF16, int NT>
__global__ void __launch_bounds__(kHeadVecThreads, 1) head_vec_kernel(const HeadVec a) {
    extern __shared__ uint4 head_sh[];
    __shared__ float2 red[kHeadVecThreads / 32][NT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int lab[NT];
    float2 st[NT];
    head_vec_walk<BF16, NT>(
        a, head_sh,
        [&] {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                lab[t] = head_vec_label(a, t);
                st[t] = make_float2(-INFINITY, 0.0f);
            }
        },
        [&](int t, int entry, int, float x) {
            st[t] = head_join(st[t], make_float2(x * kLog2e, 1.0f));
            if (lab[t] == entry && lane == 0) a.label_logit[t] = x;
        });
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

// A row of G before the token's weight, from 32 logits of it: 2^k (p - 1[label]),
// or with PROBS 2^k (alpha 1[label] - p (beta + gamma x)), x = log2 p.
template <bool BF16, bool PROBS>
struct HeadRowGrad {
    // the token's weight, that of the G without weights, and the log-sum-exp: in units of log2 and - k, PROBS as it is
    float f, u, l2;
    float alpha, beta, gamma;
    __device__ __forceinline__ HeadRowGrad(bool in, int r, const float* coef, const float* lse2, const float4* row) {
        l2 = in ? lse2[r] : 0.0f;
        if (PROBS) {
            const float4 x = in ? row[r] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            f = x.w;
            u = 1.0f;
            alpha = x.x;
            beta = x.y;
            gamma = x.z;
        } else {
            f = in ? coef[r] : 0.0f;
            u = head_unit(f);
        }
    }
    // k: the label's place among the 32
    __device__ __forceinline__ void values(float (&v)[32], int k) const {
        constexpr float kBits = head_g_bits(BF16);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if (PROBS) {
                const float x = fmax3_nan(fmaf(v[i] - l2, kLog2e, kBits), -300.0f, -300.0f);  // finite where p is 0
                v[i] = -(ex2(x) * fmaf(gamma, x, beta));
            } else {
                v[i] = ex2(fmaf(v[i], kLog2e, -l2));
            }
        }
        if (__any_sync(0xffffffffu, k >= 0 && k < 32)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = k == i ? v[i] + (PROBS ? alpha : -head_g_scale(BF16)) : v[i];
        }
    }
};

// N numbers, times f, in 16 bits; `left`: what that rounding leaves, in 16 bits.
template <bool BF16, int N>
__device__ __forceinline__ void head_round(const float (&v)[N], float f, bool left, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack16<BF16>(v[2 * i] * f, v[2 * i + 1] * f);
    if (!left) return;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float2 r = BF16 ? make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u))
                              : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        w[i] = pack16<BF16>(fmaf(v[2 * i], f, -r.x), fmaf(v[2 * i + 1], f, -r.y));
    }
}

// Epilogue of the backward's product: G of the piece in 16 bits, as the tensor
// cores take it for dW and dH.  G is rounded once, from fp32, which stands beside
// the outputs' own rounding whatever the number of terms (a sum's error grows as the
// sum does, and a label's entry is most of a row): with token weights 2.4e-3 against
// 64 bits in both gradients where the outputs' rounding makes 1.7e-3 (f16 2.3e-4 to
// 3.1e-4 and 2.1e-4), with 129 tokens as with 4096.  Without them a label's entry of
// the loss's is a power of two but for p: 1.7e-3.  Rows from the count to the tile's end (or n) become zero.  The
// logits are added up as in the forward, so that they are those that lse came
// from: taken whole, one of 30 made of 8192 products is 2.3e-4 too small, which
// is all of p - 1 for a label known with p = 0.9998.  That costs 1.4 to 2.4 % of a
// large backward (8192 x 8192 x 32000: 10.03 -> 10.18 ms, power-capped; 3584 x 4096
// x 32000: 2.13 -> 2.19) and 6 to 13 us of one of 130 to 311 tokens (160 to 260 us).
// UNIT (f16): the G without token weights, beside the other where that is wanted
// (3584 x 4096 x 32000 with weights: 2.26 -> 2.42 ms, 64 tokens 178 -> 183 us).
// PROBS: the gradient of log probability and entropy (head_probs.cuh), whose rows
// have coefficients of their own in `row`.  Up to kHeadTwice live tokens each has two
// rows: G's rounding and, in the odd ones, what that left, good together to 2^-16 (f16:
// to 2^-20, and to 2^-40 of the largest weight), so that the outputs' rounding
// alone is left.  All products have twice the rows: at 4096 x 32000 bf16, one row and
// two, one token 188 and 190 us, 64 190 and 203, 128 199 and 225, 256 216 and 331, 1024
// 570 and 1170, 4096 2620 and 5250.
template <bool BF16, bool UNIT, bool PROBS>
struct HeadGrad {
    static constexpr int kChunk = 8;
    static constexpr bool kLiveN = false;
    const int* lab;
    const float* coef;
    const float* lse2;
    uint16_t* g;       // with UNIT: or null
    uint16_t* g_unit;  // with UNIT
    int64_t ldg;
    int n;   // rows of g
    int v0;  // first vocabulary entry of the piece
    const float4* row;  // with PROBS
    const int* each;    // with PROBS: rows that a token has
    __device__ static void give_up(const PairTile&) {}
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
        const int r = t.row0 + t.lane;
        const bool in = r < t.M;
        const HeadRowGrad<BF16, PROBS> a(in, r, coef, lse2, row);
        const bool left = PROBS && *each == 2 && (r & 1);
        const int lab_c = in ? lab[r] - v0 - t.col0 - t.c_begin : -1;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int c = t.c_begin + 64 * b;
            if (c < t.c_end && t.col0 + c < t.N && t.row0 < n) {
                uint32_t w[32], w1[32];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[32];
                    head_slice(acc, 2 * b + h, v);
                    a.values(v, lab_c - 64 * b - 32 * h);
                    head_round<BF16>(v, a.f, left, w + 16 * h);
                    if (UNIT) head_round<BF16>(v, a.u, left, w1 + 16 * h);
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
template <bool BF16, bool UNIT, bool PROBS>
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
    const float4* row;
    const int* each;
    __device__ static void give_up(const PairTile&) {}
    __device__ __forceinline__ void finish(const PairTile& t, const float (&acc)[128]) const {
        const bool twice = PROBS && *each == 2;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int c = t.c_begin + 32 * b;
            if (c >= t.c_end || t.row0 >= t.M || t.col0 + c >= n) continue;
            float v[32];
            head_slice(acc, b, v);
            pair_transpose(t, v);
            const int token = t.col0 + c + t.lane;
            const bool in = token < t.N;
            const HeadRowGrad<BF16, PROBS> a(in, token, coef, lse2, row);
            a.values(v, in ? lab[token] - v0 - t.row0 : -1);
            uint32_t w[16], w1[16];
            head_round<BF16>(v, a.f, twice && (token & 1), w);
            if (UNIT) head_round<BF16>(v, a.u, twice && (token & 1), w1);
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
// CTA takes 1024 columns of tokens, TOKENS of them in flight.  PROBS: or one, where
// tokens have two rows, which are added up.
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
template <bool BF16, int TOKENS, bool TWICE>
__device__ __forceinline__ void head_dh(const HeadDh& a, int* sh) {
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
        constexpr int R = TWICE ? 2 : 1;
        float4 v[TOKENS][2 * R];
        int p[TOKENS];
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
            const int64_t t = t0 + (int64_t)k * gridDim.x;
            p[k] = t < a.n ? a.pos[t] : kHeadIgnored;
#pragma unroll
            for (int h = 0; h < 2 * R; ++h)  // ld is a multiple of 8
                v[k][h] = p[k] >= 0 ? *reinterpret_cast<const float4*>(a.slab + (p[k] + h / 2) * a.ld + c + 4 * (h & 1))
                                    : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
            const int64_t t = t0 + (int64_t)k * gridDim.x;
            if (t >= a.n) break;
            if (p[k] >= 0) {
                const int i = (a.live_n ? pair_tile_index(c / 256, p[k] / bt, tiles_d, tiles_t)
                                        : pair_tile_index(p[k] / bt, c / 256, tiles_t, tiles_d)) - full;
                if (i >= 0) {  // of two rows too: they are in one tile, whose width is even
                    const float* e = a.extra + ((int64_t)i * 256 + p[k] % bt) * 256 + c % 256;
#pragma unroll(TOKENS == 1 ? 12 : 4)
                    for (int s = 0; s + 1 < splits; ++s)
#pragma unroll
                        for (int h = 0; h < 2 * R; ++h) {
                            const float4 x = *reinterpret_cast<const float4*>(e + (int64_t)s * rest * 65536 + 256 * (h / 2) + 4 * (h & 1));
                            v[k][h] = make_float4(v[k][h].x + x.x, v[k][h].y + x.y, v[k][h].z + x.z, v[k][h].w + x.w);
                        }
                }
            }
            if (TWICE)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 x = v[k][2 * R - 2 + h];
                    v[k][h] = make_float4(v[k][h].x + x.x, v[k][h].y + x.y, v[k][h].z + x.z, v[k][h].w + x.w);
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
template <bool BF16, int TOKENS, bool PROBS>
__global__ void __launch_bounds__(128) head_dh_kernel(const HeadDh a) {
    __shared__ int sh[5];
    pdl_wait();
    if (PROBS && a.count[1] == 2) head_dh<BF16, 1, true>(a, sh);
    else head_dh<BF16, TOKENS, false>(a, sh);
}

}  // namespace aeth
