// head_probs.cuh -- log probabilities of given tokens at the language model's
// head, with the entropy of their distribution and the likeliest alternatives,
// the logits kept for a piece of the vocabulary at most.
//
//   s = H W^T    lse = log sum_v exp s_v    log p_y = s_y - lse
//   entropy = lse - sum_v p_v s_v           alternatives: the largest s_v - lse
//
// One pass of the head's product (head_loss.cuh: rows that take no part are left
// out before it).  A range of the vocabulary leaves its maximum m, the sum s of
// 2^x and u, the sum of 2^x x, of x = (logit - m) log2 e; two ranges join as sums
// do after both are taken to the larger maximum, and
//   lse = m + ln s     entropy = ln s - ln 2 u / s.
//
// Alternatives: of a row's k best entries none lies outside the k ranges (128
// entries each) whose maxima are the best, the lower range before the other on
// equal ones: each of these holds an entry before any of another range.  The
// product therefore leaves its logits in fp32, a piece of the vocabulary at a time
// (256 MiB), and a warp a row reads the maxima of a piece and then such ranges
// alone (head_top).  The best so far lie in its lanes, one each, which bounds k by
// 32.  Equal logits: the lower entry first.
//
// Gradient of a log p_y + b entropy, with q = log p:
//   G_v = a 1[v = y] - p_v (a + b (q_v + entropy))
// taken as the loss's is (head_loss.cuh), whose weight is one number a token, here
// w = |a| + c |b|: c = ln(vocab) / 4 + 1/2 bounds |p (q + entropy)|.
#pragma once
#include "head_loss.cuh"

namespace aeth {

constexpr int kHeadTop = 32;         // alternatives, at most
constexpr int kHeadRange = 128;      // entries of a range where alternatives are wanted
constexpr float kHeadNone = -200.0f;  // of log2: 2^-200 is 0, and finite times 0 too

// (maximum, s, u) of a range
struct alignas(16) HeadSums {
    float m, s, u, unused;
};
__device__ __forceinline__ HeadSums head_no_sums() { return {-INFINITY, 0.0f, 0.0f, 0.0f}; }
// What logits are taken against: a maximum, or 0 where there is none.  They are
// subtracted before they are scaled, so that no finite logit overflows.
__device__ __forceinline__ float head_base(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ float head_log2(float v, float base) { return fmax3_nan((v - base) * kLog2e, kHeadNone, kHeadNone); }
// a's sums against a larger base
__device__ __forceinline__ void head_rebase(const HeadSums& a, float base, float& s, float& u) {
    const float d = head_log2(a.m, base), w = ex2(d);
    s += a.s * w;
    u += fmaf(a.s, d, a.u) * w;
}
__device__ __forceinline__ HeadSums head_join3(const HeadSums& a, const HeadSums& b) {
    HeadSums r{fmaxf(a.m, b.m), 0.0f, 0.0f, 0.0f};
    const float base = head_base(r.m);
    head_rebase(a, base, r.s, r.u);
    head_rebase(b, base, r.s, r.u);
    return r;
}
__device__ __forceinline__ HeadSums head_shuffle(const HeadSums& a, int o) {
    return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o), 0.0f};
}
// ln s and the entropy.  A whole row's s is 1 at least (the maximum's own term) and its
// entropy 0, but for rounding, which may not make a log probability positive or an
// entropy negative; s = 0 is a row of -infinity alone.
__device__ __forceinline__ float head_log_sum(const HeadSums& a) { return a.s < 1.0f && a.s > 0.5f ? 0.0f : logf(a.s); }
__device__ __forceinline__ float head_entropy(const HeadSums& a) {
    const float e = head_log_sum(a) - kLn2 * (a.u / a.s);
    return e < 0.0f ? 0.0f : e;
}

// Joins 32 logits, the first `left` of them, whatever they are.
__device__ __forceinline__ void head_sums32(const float (&v)[32], int left, HeadSums& st) {
    float m = st.m;
#pragma unroll
    for (int i = 0; i < 32; i += 2)
        m = left >= 32 ? fmax3(m, v[i], v[i + 1]) : fmaxf(i < left ? fmaxf(m, v[i]) : m, i + 1 < left ? v[i + 1] : m);
    const float base = head_base(m);
    float s0 = 0.0f, s1 = 0.0f, u0 = 0.0f, u1 = 0.0f;
    head_rebase(st, base, s0, u0);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float x0 = head_log2(v[i], base), x1 = head_log2(v[i + 1], base);
        const float e0 = left >= 32 || i < left ? ex2(x0) : 0.0f, e1 = left >= 32 || i + 1 < left ? ex2(x1) : 0.0f;
        if (left >= 32 || i < left) {
            s0 += e0;
            u0 = fmaf(e0, x0, u0);
        }
        if (left >= 32 || i + 1 < left) {
            s1 += e1;
            u1 = fmaf(e1, x1, u1);
        }
    }
    st = {m, s0 + s1, u0 + u1, 0.0f};
}
// The same in two and a half instructions a logit, against a maximum that is known
// (`unused` holds it in units of log2): fused multiply-adds of pairs.  The maximum's
// rounding in those units, half a step of it, is one factor of all sums, which
// head_fast_end takes out; up to 2^24 that is 2^0.5 at most.  Rows beyond, whose
// sums it could overflow, and those with a logit of -infinity, which makes u NaN, go
// the other way.
__device__ __forceinline__ void head_fast32(const float (&v)[32], int left, HeadSums& st) {
    const float2 l2 = make_float2(kLog2e, kLog2e), nb = make_float2(-st.unused, -st.unused);
    float2 s = make_float2(st.s, 0.0f), u = make_float2(st.u, 0.0f);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float2 x = fma2_rn(make_float2(v[i], v[i + 1]), l2, nb);
        const float2 e = make_float2(left >= 32 || i < left ? ex2(x.x) : 0.0f, left >= 32 || i + 1 < left ? ex2(x.y) : 0.0f);
        s = add2_rn(s, e);
        u = fma2_rn(e, x, u);
    }
    st.s = s.x + s.y;
    st.u = u.x + u.y;
}
__device__ __forceinline__ HeadSums head_fast_begin(const float (&acc)[128], int left) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 128; i += 2)
        m = left >= 128 ? fmax3(m, acc[i], acc[i + 1]) : fmaxf(i < left ? fmaxf(m, acc[i]) : m, i + 1 < left ? acc[i + 1] : m);
    return {m, 0.0f, 0.0f, m * kLog2e};
}
__device__ __forceinline__ bool head_fast_good(const HeadSums& st) { return fabsf(st.unused) < 0x1p24f && st.u == st.u; }
// Takes the base's rounding d = m log2 e - base out: s 2^-d and, of x - d, u.
__device__ __forceinline__ HeadSums head_fast_end(const HeadSums& st) {
    const float d = fmaf(st.m, kLog2e, -st.unused), w = ex2(-d);
    return {st.m, st.s * w, fmaf(-st.s, d, st.u) * w, 0.0f};
}

// What the product's epilogues (HeadStats, HeadStatsT) keep: the sums and, with
// TOP, the logits.
template <bool TOP>
struct HeadProbsSums {
    using Sum = HeadSums;
    HeadSums* part;  // [row][range]; TOP: ranges of 128 entries, of all pieces
    int ranges, first;
    float* logits;  // [row][entry of the piece], a multiple of 8 of them
    int64_t ld;
    __device__ static Sum none() { return head_no_sums(); }
    __device__ static Sum join(const Sum& a, const Sum& b) { return head_join3(a, b); }
    __device__ __forceinline__ static Sum before(const float (&acc)[128], int left) { return head_fast_begin(acc, left); }
    __device__ __forceinline__ static void add32(const float (&v)[32], int left, Sum& st) { head_fast32(v, left, st); }
    __device__ static bool good(const Sum& st) { return head_fast_good(st); }
    __device__ __forceinline__ static void again32(const float (&v)[32], int left, Sum& st) { head_sums32(v, left, st); }
    __device__ __forceinline__ void put(int range, int row, const Sum& x) const {
        part[(int64_t)row * ranges + first + range] = x.unused != 0.0f ? head_fast_end(x) : x;
    }
    // A row's 32 logits go out from their thread, a sector (eight) at a time: through
    // shared memory, in whole lines, they took the epilogue so long that the products
    // waited for it.
    __device__ __forceinline__ void store(float* o, const float (&v)[32], int left) const {
#pragma unroll
        for (int i = 0; i < 32; i += 8)
            if (i < left)  // ld is a multiple of 8
                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o + i), "f"(v[i]), "f"(v[i + 1]),
                             "f"(v[i + 2]), "f"(v[i + 3]), "f"(v[i + 4]), "f"(v[i + 5]), "f"(v[i + 6]), "f"(v[i + 7])
                             : "memory");
    }
    __device__ __forceinline__ void rows(const PairTile& t, const float (&v)[32], int c) const {
        const int row = t.row0 + t.lane, col = t.col0 + c;
        if (TOP && row < t.M) store(logits + (int64_t)row * ld + col, v, t.N - col);
    }
    __device__ __forceinline__ void token(int token, int entry, int left, const float (&v)[32]) const {
        if (TOP) store(logits + (int64_t)token * ld + entry, v, left);
    }
};

// The best entries so far, lane i the i-th: larger logits first, the lower entry
// first among equal ones.
struct HeadBest {
    float v;
    int i;
    __device__ static bool before(float a, int i, float b, int j) { return a > b || (a == b && i < j); }
    // Takes (x, j) in; all lanes with the same arguments.
    __device__ __forceinline__ void insert(float x, int j) {
        const int lane = threadIdx.x & 31;
        const int at = __popc(__ballot_sync(0xffffffffu, before(v, i, x, j)));
        const float up = __shfl_up_sync(0xffffffffu, v, 1);
        const int ui = __shfl_up_sync(0xffffffffu, i, 1);
        if (lane > at) {
            v = up;
            i = ui;
        } else if (lane == at) {
            v = x;
            i = j;
        }
    }
    // Takes in what the lanes hold, where it comes before the k-th.
    __device__ __forceinline__ void offer(float x, int j, int k) {
        uint32_t left = __ballot_sync(0xffffffffu,
                                      before(x, j, __shfl_sync(0xffffffffu, v, k - 1), __shfl_sync(0xffffffffu, i, k - 1)));
        while (left) {
            const int from = __ffs(left) - 1;
            left &= left - 1;
            const float y = __shfl_sync(0xffffffffu, x, from);
            const int l = __shfl_sync(0xffffffffu, j, from);
            if (before(y, l, __shfl_sync(0xffffffffu, v, k - 1), __shfl_sync(0xffffffffu, i, k - 1))) insert(y, l);
        }
    }
    __device__ static HeadBest none() { return {-INFINITY, 0x7fffffff}; }
};

// What a token gets; warps of a CTA take tokens.  With alternatives one launch
// for each piece of the vocabulary, the last of which joins the ranges.
struct HeadProbsOut {
    const HeadSums* part;
    int ranges;              // of the whole vocabulary
    const float* label_logit;
    const int* pos;
    int64_t n;
    float *log_probs, *entropy, *lse;
    // alternatives
    int top;
    const float* logits;
    int64_t ld;
    int first, count, v0, vp;  // the piece's ranges, first entry and entries
    int is_first, is_last;
    float2* best;              // [row][32], between pieces: (value, index's bits)
    float* top_log_probs;      // [token][top]
    int64_t* top_ids;
};

__device__ __forceinline__ void head_probs_write(const HeadProbsOut& a, int64_t t, int lane, bool bad, bool live, HeadSums x,
                                                 float label_logit, const HeadBest& best) {
    const float nan = __int_as_float(0x7fc00000);
    // one lane's: in the others the same sums were added the other way round
    const float m = __shfl_sync(0xffffffffu, bad ? nan : live ? head_base(x.m) : 0.0f, 0);
    const float log_s = __shfl_sync(0xffffffffu, live ? head_log_sum(x) : 0.0f, 0), lse = m + log_s;
    // from a logit's distance to the maximum: without the rounding of a large lse
    auto log_prob = [&](float v) { return (v - m) - log_s; };
    if (lane == 0) {
        a.lse[t] = lse;
        a.log_probs[t] = bad ? nan : live ? log_prob(label_logit) : 0.0f;
        a.entropy[t] = bad ? nan : live ? head_entropy(x) : 0.0f;
    }
    if (lane < a.top) {
        const bool known = live && !isnan(lse) && best.i != 0x7fffffff;
        a.top_log_probs[t * a.top + lane] = known ? log_prob(best.v) : bad || live ? nan : 0.0f;
        a.top_ids[t * a.top + lane] = known ? best.i : -1;
    }
}

// Joins a row's ranges, by a warp: eight loads of a lane in flight, each brought to
// the largest maximum so far.
__device__ __forceinline__ HeadSums head_join_ranges(const HeadSums* p, int ranges) {
    const int lane = threadIdx.x & 31;
    HeadSums x = head_no_sums();
    for (int r0 = 0; r0 < ranges; r0 += 256) {
        HeadSums y[8];
        float m = x.m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = r0 + 32 * j + lane;
            y[j] = r < ranges ? p[r] : head_no_sums();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, y[j].m);
        const float base = head_base(m);
        float s = 0.0f, u = 0.0f;
        head_rebase(x, base, s, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) head_rebase(y[j], base, s, u);
        x = {m, s, u, 0.0f};
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = head_join3(x, head_shuffle(x, o));
    return x;
}

// The place of (x, i) among values in shared memory: how many come before it.
template <typename At>
__device__ __forceinline__ int head_place(float x, int i, int count, At at) {
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) {
        const float2 y = at(j);
        place += HeadBest::before(y.x, __float_as_int(y.y), x, i) ? 1 : 0;
    }
    return place;
}

// A float's place in the order of floats
__device__ __forceinline__ uint32_t head_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float head_unkey(uint32_t k) { return __uint_as_float(k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u)); }

// What a warp needs to take a row's best entries of a piece.
constexpr int kTopRanges = 256, kTopList = 128;
struct HeadTopShared {
    float2 list[kTopList], out[kHeadTop];
    uint16_t ranges[kTopRanges];
    int count;
};

// A row's ranges of a piece, or some of them
struct HeadPiece {
    const HeadSums* p;
    const float* s;
    int count, v0, vp;  // ranges, first entry, entries
    __device__ HeadPiece(const HeadProbsOut& a, int row, int from, int to)
        : p(a.part + (int64_t)row * a.ranges + a.first + from), s(a.logits + (int64_t)row * a.ld + from * kHeadRange),
          count(to - from), v0(a.v0 + from * kHeadRange), vp(min(a.vp, to * kHeadRange) - from * kHeadRange) {}
};

// The slow way, whatever the logits: one range and one entry after the other.
__device__ __noinline__ HeadBest head_top_slow(const HeadPiece& a, int top, HeadBest best) {
    const int lane = threadIdx.x & 31;
    HeadBest at = HeadBest::none();
    for (int r0 = 0; r0 < a.count; r0 += 32) {
        const int r = r0 + lane;
        at.offer(r < a.count ? a.p[r].m : -INFINITY, r < a.count ? r : 0x7fffffff, top);
    }
    for (int k = 0; k < top; ++k) {
        const float m = __shfl_sync(0xffffffffu, at.v, k);
        const int r = __shfl_sync(0xffffffffu, at.i, k);
        if (r == 0x7fffffff || !HeadBest::before(m, a.v0 + r * kHeadRange, __shfl_sync(0xffffffffu, best.v, top - 1),
                                                 __shfl_sync(0xffffffffu, best.i, top - 1)))
            break;
        const int e0 = r * kHeadRange + 4 * lane;
        const float4 v = e0 < a.vp ? *reinterpret_cast<const float4*>(a.s + e0) : make_float4(0, 0, 0, 0);
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            best.offer(e0 + i < a.vp ? x[i] : -INFINITY, e0 + i < a.vp ? a.v0 + e0 + i : 0x7fffffff, top);
    }
    return best;
}

// A row's best entries, of a piece and those before it: a warp, lane i gets the
// i-th.  A bound that `top` entries reach comes from the maxima of 256 groups (of
// ranges, or of entries where there are few ranges), by halving the interval that
// it lies in; the ranges whose maxima reach it are read, eight at a time, and the
// entries that do are counted into their places.  With equal logits by the hundred,
// which a bound cannot part, the slow way.
__device__ __forceinline__ HeadBest head_top(const HeadPiece& a, int top, HeadBest best, HeadTopShared& sh) {
    const int lane = threadIdx.x & 31;
    const HeadSums* p = a.p;
    const float* s = a.s;
    const bool few = 2 * a.count < 3 * top;
    uint32_t key[8] = {};
    if (few) {
        for (int e0 = 0; e0 < a.vp; e0 += 1024)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = e0 + 128 * j + 4 * lane;
                if (e >= a.vp) continue;
                const float4 v = *reinterpret_cast<const float4*>(s + e);
                float m = fmaxf(-INFINITY, v.x);
                if (e + 1 < a.vp) m = fmaxf(m, v.y);
                if (e + 2 < a.vp) m = fmaxf(m, v.z);
                if (e + 3 < a.vp) m = fmaxf(m, v.w);
                key[j] = max(key[j], head_key(m));
            }
    } else {
        for (int r0 = 0; r0 < a.count; r0 += 256)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = r0 + 32 * j + lane;
                if (r < a.count) key[j] = max(key[j], head_key(p[r].m));
            }
    }
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, key[j]);
    // the least of the lanes' maxima is reached by 32 of them
    uint32_t lo = __reduce_min_sync(0xffffffffu, most), hi = __reduce_max_sync(0xffffffffu, most);
    for (int i = 0; i < 14 && lo < hi; ++i) {
        const uint32_t mid = hi - (hi - lo) / 2;
        int n = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) n += key[j] >= mid ? 1 : 0;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n >= top) lo = mid;
        else hi = mid - 1;
        if (n == top) break;
    }
    const int last = __shfl_sync(0xffffffffu, best.i, top - 1);
    const float last_v = __shfl_sync(0xffffffffu, best.v, top - 1);
    if (last != 0x7fffffff) lo = max(lo, head_key(last_v));
    const float bound = lo <= head_key(-INFINITY) ? -INFINITY : head_unkey(lo);  // below: no float, and no group either
    int count = a.count;
    if (!few) {
        count = 0;
        for (int r0 = 0; r0 < a.count; r0 += 256) {
            bool in[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = r0 + 32 * j + lane;
                in[j] = r < a.count && (a.count <= 256 ? head_unkey(key[j]) : p[r].m) >= bound;  // 256: a group is a range
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t who = __ballot_sync(0xffffffffu, in[j]);
                const int at = count + __popc(who & ((1u << lane) - 1));
                if (in[j] && at < kTopRanges) sh.ranges[at] = (uint16_t)(r0 + 32 * j + lane);
                count += __popc(who);
            }
        }
        if (count > kTopRanges) return head_top_slow(a, top, best);
    }
    sh.out[lane] = make_float2(-INFINITY, __int_as_float(0x7fffffff));
    if (lane == 0) sh.count = 0;
    __syncwarp();
    auto take = [&](float x, int i) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kTopList) sh.list[at] = make_float2(x, __int_as_float(i));
    };
    for (int q0 = 0; q0 < count; q0 += 8) {
        float4 v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int e = q0 + q < count ? (few ? q0 + q : (int)sh.ranges[q0 + q]) * kHeadRange + 4 * lane : a.vp;
            v[q] = e < a.vp ? *reinterpret_cast<const float4*>(s + e) : make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (q0 + q >= count) break;
            const int e = (few ? q0 + q : (int)sh.ranges[q0 + q]) * kHeadRange + 4 * lane;
            const float x[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (x[i] >= bound && e + i < a.vp) take(x[i], a.v0 + e + i);
        }
    }
    if (lane < top && best.i != 0x7fffffff && best.v >= bound) take(best.v, best.i);
    __syncwarp();
    const int n = sh.count;
    if (n > kTopList) return head_top_slow(a, top, best);
    for (int q = lane; q < n; q += 32) {
        const float2 x = sh.list[q];
        const int place = head_place(x.x, __float_as_int(x.y), n, [&](int j) { return sh.list[j]; });
        if (place < kHeadTop) sh.out[place] = x;
    }
    __syncwarp();
    const float2 x = sh.out[lane];
    __syncwarp();
    return {x.x, __float_as_int(x.y)};
}

// A warp a token, or with SPLIT the eight warps of a CTA: each takes an eighth of
// the ranges, and their best entries are counted into their places.
template <bool TOP, bool SPLIT>
__global__ void __launch_bounds__(256) head_probs_kernel(const HeadProbsOut a) {
    __shared__ HeadTopShared sh[TOP ? 8 : 1];
    __shared__ float2 all[SPLIT && TOP ? 8 * kHeadTop : 1], out[SPLIT && TOP ? kHeadTop : 1];
    __shared__ HeadSums sums[SPLIT ? 8 : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_trigger();
    for (int64_t t = SPLIT ? blockIdx.x : blockIdx.x * 8ll + warp; t < a.n; t += gridDim.x * (SPLIT ? 1ll : 8ll)) {
        const int row = a.pos[t];
        HeadBest best = HeadBest::none();
        if (TOP && row >= 0) {
            if (!a.is_first && (!SPLIT || warp == 0)) {
                const float2 b = a.best[(int64_t)row * 32 + lane];
                best = {b.x, __float_as_int(b.y)};
            }
            const int from = SPLIT ? a.count * warp / 8 : 0, to = SPLIT ? a.count * (warp + 1) / 8 : a.count;
            if (from < to) best = head_top(HeadPiece(a, row, from, to), a.top, best, sh[TOP ? warp : 0]);
            if (SPLIT) {
                if (lane < a.top) all[warp * a.top + lane] = make_float2(best.v, __int_as_float(best.i));
                if (warp == 0) out[lane] = make_float2(-INFINITY, __int_as_float(0x7fffffff));
                __syncthreads();
                if (lane < a.top && best.i != 0x7fffffff) {
                    const int place = head_place(best.v, best.i, 8 * a.top, [&](int j) { return all[j]; });
                    if (place < a.top) out[place] = make_float2(best.v, __int_as_float(best.i));
                }
                __syncthreads();
                best = {out[lane].x, __float_as_int(out[lane].y)};
            }
            if (!a.is_last && (!SPLIT || warp == 0)) a.best[(int64_t)row * 32 + lane] = make_float2(best.v, __int_as_float(best.i));
        }
        HeadSums x = head_no_sums();
        if (row >= 0 && (!TOP || a.is_last)) {
            const int from = SPLIT ? a.ranges * warp / 8 : 0, to = SPLIT ? a.ranges * (warp + 1) / 8 : a.ranges;
            x = head_join_ranges(a.part + (int64_t)row * a.ranges + from, to - from);
            if (SPLIT) {
                if (lane == 0) sums[warp] = x;
                __syncthreads();
                x = sums[lane & 7];
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) x = head_join3(x, head_shuffle(x, o));
            }
        }
        if (SPLIT) __syncthreads();  // the shared places are the next token's
        if ((!TOP || a.is_last) && (!SPLIT || warp == 0))
            head_probs_write(a, t, lane, row == kHeadBad, row >= 0, x, row >= 0 ? a.label_logit[row] : 0.0f, best);
    }
}

// One to four tokens: the weight by rows, as head_vec_kernel.  A CTA keeps its
// logits in shared memory and takes everything from there at the end: its sums, and
// its best entries in their order.  An entry's place is the number of those before
// it, so that no thread waits for another; to be counted among few, it must come no
// later than the `top`-th of the best of 64 groups.  One token x 4096 x 32000 with
// twenty alternatives: 47.5 us, 43 without, 2048 x 131071 85 and 79.5 (107 where all of a
// CTA's entries are counted); with sums per entry and one warp that joins the CTAs'
// entries one by one 57.
struct HeadVecProbs {
    HeadVec v;
    HeadSums* part;  // [token][CTA]
    float2* cand;    // [token][CTA][top]: (logit, entry's bits)
    int top, slots;  // logits that a CTA has for a token, at most
};
template <bool BF16, int NT>
__global__ void __launch_bounds__(kHeadVecThreads, 1) head_vec_probs_kernel(const HeadVecProbs a) {
    extern __shared__ uint4 head_sh[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, each = 2 * kHeadVecThreads / 32;  // entries of a round
    float* logits = reinterpret_cast<float*>(head_sh + NT * ((a.v.d + 7) / 8));  // [token][place]
    const int round = each * gridDim.x, mine = each * blockIdx.x;  // entry = round's first + mine + place in the round
    head_vec_walk<BF16, NT>(a.v, head_sh, [] {}, [&](int t, int, int place, float x) {
        if (lane == 0) logits[t * a.slots + place] = x;
    });
    // none, where there are fewer entries than alternatives, or NaN (which has no place) takes others' places
    for (int i = threadIdx.x; i < NT * a.top; i += kHeadVecThreads)
        a.cand[((int64_t)(i / a.top) * gridDim.x + blockIdx.x) * a.top + i % a.top] =
            make_float2(-INFINITY, __int_as_float(0x7fffffff));
    __syncthreads();
    // whole rounds, and what the last one has here
    const int last = a.v.vocab / round, have = last * each + max(min(a.v.vocab - last * round - mine, each), 0);
    for (int t = warp; t < NT; t += kHeadVecThreads / 32) {
        const float* l = logits + t * a.slots;
        float m = -INFINITY;
        for (int i = lane; i < have; i += 32) m = fmaxf(m, l[i]);
        HeadSums x{warp_max(m), 0.0f, 0.0f, 0.0f};
        const float base = head_base(x.m);
        for (int i = lane; i < have; i += 32) {
            const float z = head_log2(l[i], base), e = ex2(z);
            x.s += e;
            x.u = fmaf(e, z, x.u);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            x.s += __shfl_xor_sync(0xffffffffu, x.s, o);
            x.u += __shfl_xor_sync(0xffffffffu, x.u, o);
        }
        if (lane == 0) {
            a.part[(int64_t)t * gridDim.x + blockIdx.x] = x;
            const int lab = head_vec_label(a.v, t), in = lab % round - mine;
            if (lab >= 0 && in >= 0 && in < each) a.v.label_logit[t] = l[lab / round * each + in];
        }
    }
    if (a.top == 0) return;
    // 128 threads a token
    constexpr int kGroups = 64;
    __shared__ float2 maxima[kHeadVecTokens][kGroups], bound[kHeadVecTokens];
    __shared__ int count[kHeadVecTokens];
    const int t = threadIdx.x >> 7, j = threadIdx.x & 127;
    const bool takes = t < NT;
    const float* l = logits + (takes ? t : 0) * a.slots;
    uint16_t* places = reinterpret_cast<uint16_t*>(logits + NT * a.slots) + (takes ? t : 0) * a.slots;
    if (takes && j < kGroups) {
        float x = -INFINITY;
        int at = 0x7fffffff;
        for (int i = j; i < have; i += kGroups)
            if (HeadBest::before(l[i], i, x, at)) {
                x = l[i];
                at = i;
            }
        maxima[t][j] = make_float2(x, __int_as_float(at));
        if (j == 0) {
            bound[t] = make_float2(-INFINITY, __int_as_float(0x7fffffff));
            count[t] = 0;
        }
    }
    __syncthreads();
    if (takes && j < kGroups) {
        const float2 x = maxima[t][j];
        if (__float_as_int(x.y) != 0x7fffffff &&
            head_place(x.x, __float_as_int(x.y), kGroups, [&](int k) { return maxima[t][k]; }) == a.top - 1)
            bound[t] = x;
    }
    __syncthreads();
    if (takes)
        for (int i = j; i < have; i += 128)
            if (!HeadBest::before(bound[t].x, __float_as_int(bound[t].y), l[i], i)) places[atomicAdd(&count[t], 1)] = (uint16_t)i;
    __syncthreads();
    if (takes)
        for (int q = j; q < count[t]; q += 128) {
            const int i = places[q];
            const int place = head_place(l[i], i, count[t], [&](int k) { return make_float2(l[places[k]], __int_as_float((int)places[k])); });
            if (place < a.top)
                a.cand[((int64_t)t * gridDim.x + blockIdx.x) * a.top + place] =
                    make_float2(l[i], __int_as_float(i / each * round + mine + i % each));
        }
}

// A CTA a token: takes the best of the CTAs' best while its last warp joins their
// sums.
constexpr int kHeadVecJoin = 512;
__global__ void __launch_bounds__(kHeadVecJoin)
    head_vec_probs_join_kernel(const HeadVecProbs a, int ctas, const HeadProbsOut o, uint32_t* err) {
    __shared__ float2 heads[kHeadVecJoin], best[kHeadTop * kHeadTop], top[kHeadTop], last;
    __shared__ int list[kHeadTop], count;
    __shared__ HeadSums sums;
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const float2 none = make_float2(-INFINITY, __int_as_float(0x7fffffff));
    pdl_wait();
    const float2* cand = a.cand + (int64_t)t * ctas * a.top;
    if (tid < kHeadTop) {
        list[tid] = -1;
        top[tid] = none;
        if (tid == 0) {
            last = none;
            count = 0;
        }
    }
    if (a.top > 0)
        for (int i = tid; i < ctas; i += kHeadVecJoin) heads[i] = cand[(int64_t)i * a.top];
    if (tid >= kHeadVecJoin - 32) {
        const HeadSums x = head_join_ranges(a.part + (int64_t)t * ctas, ctas);
        if (lane == 0) sums = x;
    }
    __syncthreads();
    if (a.top > 0) {
        // the CTAs whose best entries are the best: no other has one of the first `top`
        for (int i = tid; i < ctas; i += kHeadVecJoin) {
            const float2 x = heads[i];
            if (__float_as_int(x.y) == 0x7fffffff) continue;
            const int place = head_place(x.x, __float_as_int(x.y), ctas, [&](int j) { return heads[j]; });
            if (place < a.top) list[place] = i;
            if (place == a.top - 1) last = x;
        }
        __syncthreads();
        // of their entries, those up to the last one's best
        for (int i = tid; i < a.top * a.top; i += kHeadVecJoin) {
            const int from = list[i / a.top];
            const float2 x = from >= 0 ? cand[(int64_t)from * a.top + i % a.top] : none;
            if (__float_as_int(x.y) != 0x7fffffff && !HeadBest::before(last.x, __float_as_int(last.y), x.x, __float_as_int(x.y)))
                best[atomicAdd(&count, 1)] = x;
        }
        __syncthreads();
        for (int i = tid; i < count; i += kHeadVecJoin) {
            const float2 x = best[i];
            const int place = head_place(x.x, __float_as_int(x.y), count, [&](int j) { return best[j]; });
            if (place < a.top) top[place] = x;
        }
        __syncthreads();
    }
    if (tid >= 32) return;
    const int64_t lab = a.v.labels[t];
    const bool in = lab != a.v.ignore_index, bad = in && (lab < 0 || lab >= a.v.vocab);
    if (bad && lane == 0) report_dev_error(err, DEVERR_BAD_ARG);
    head_probs_write(o, t, lane, bad, in && !bad, sums, in && !bad ? a.v.label_logit[t] : 0.0f,
                     HeadBest{top[lane].x, __float_as_int(top[lane].y)});
}

}  // namespace aeth
