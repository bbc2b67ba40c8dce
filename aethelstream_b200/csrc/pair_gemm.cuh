// pair_gemm.cuh -- the matrix product of the training operators: a persistent
// tcgen05 GEMM on CTA pairs, D (M x N) = A (M x K) B (K x N), 16-bit operands,
// fp32 accumulation in TMEM, the epilogue a functor.
//
// Unit = 256 x bn tile of D (or a K range of one, see PairTail); each CTA of the pair holds its 128 rows
// of A and half of the tile's bn columns of B per 64-deep k-block, CTA 0 issues
// the pair's MMAs (M = 256, N = bn) and its commits reach both CTAs' barriers.
// 256 x 256 is the largest tile whose accumulator fits TMEM twice (2 x 256
// columns), so the epilogue of one tile runs under the MMAs of the next; each
// CTA then loads 32 KB per k-block of 512 MMA cycles.  Warps: 0 = TMEM
// allocation + TMA producer, 1 = MMA issuer, 2..9 = epilogue (warp w reads TMEM
// lane quarter w % 4; warps 2-5 take the first half of the columns, 6-9 the
// second), 10 and 11 = TMA producers too.  Three producers share the k-blocks
// in turn: one thread's wait, expect and two to four copies take 480 to 640
// cycles (measured, whatever the copies' sizes), which alone would hold a
// k-block of 512 MMA cycles at about 720.
//
// Every wait on a barrier is bounded (mbar_wait); an epilogue with barriers of
// its own says in give_up() how a warp that leaves settles them.
//
// An epilogue may take the accumulator in pieces of kChunk k-blocks and add
// them up in registers (Epi::kChunk > 0).  The tensor cores cut every partial
// sum off toward zero, which shrinks a sum of K products by about K * 1e-9 of
// itself (measured in bf16: 3.8e-6 at K = 4096); pieces of 512 keep that at 4e-7 to
// 7e-7 (2.6e-6 in f16, whose products have more bits to cut).  The
// logits are taken so, in the loss and in its gradient; sums that end in 16 bits
// (over tokens or the vocabulary) are taken whole: 8e-6 at 8192 terms.  Tiles
// of at most 160 columns have TMEM for three or four accumulators instead of two,
// so that the MMAs go on while the epilogue ends a tile (300 and 512 tokens x 4096
// x 32000, forward: 88.5 -> 86 and 117 -> 109 us).
//
// Measured, 3584 x 4096 x 32000 bf16: 568-608 us a product (1.54-1.65 PF/s at the
// 1.5 GHz that the power cap leaves), tensor pipe 97-98 % active: the clock
// bounds it (92 % where G is written: its epilogue outlasts the two accumulators
// that the MMAs are ahead).  With the issuer and one producer behind `lane == 0` 688 us, 71 %.
//
// M, N or K may be held on the device (`live`): the number of rows that a mask
// leaves.  Operand rows past it, up to the next multiple of 256, must be zero.
//
// Few live rows are taken as N, not M: M comes in tiles of 256 only, N in
// multiples of 32, so 311 rows cost two tiles of 160 and not two of 256, and a
// handful of rows leaves a product bound by the other operand's bytes.  Their
// smaller stages make up to nine of six: a k-block of 320 MMA cycles (N = 160)
// took 530 with six stages, whose copies were not far enough ahead of the MMAs
// (tensor pipe 52 % active, DRAM 44 %; 300 x 4096 x 32000, forward and backward:
// 95 + 274 us with six, 89 + 257 with seven; 16 tokens, nine: 63 + 176 and 58 +
// 170; before the gradient took its logits in pieces).  The
// tile's columns are then the rows of the result, and epilogues turn each
// 32 x 32 block over in shared memory (pair_transpose).
// Tiles are walked in groups of row tiles so that the tiles in flight
// share their operands in L2.
#pragma once
#include <algorithm>

#include "tmap.cuh"
#include "umma.cuh"

namespace aeth {

constexpr int kPairEpiWarps = 8;
constexpr int kPairProducers = 3;
constexpr int kPairThreads = 32 * (1 + kPairProducers + kPairEpiWarps);
constexpr int kPairStages = 6;
constexpr int kPairOperand = 128 * 64 * 2;                  // one operand of one stage and CTA
constexpr int kPairStage = 2 * kPairOperand;
// Of narrow tiles, whose B takes less: 64 columns at least (pair_live_bn).
constexpr int kPairMaxStages = kPairStages * kPairStage / (kPairOperand + 32 * 128);
static_assert(kPairMaxStages == 9, "stages of a tile of 64 columns");
// The producers take the k-blocks in turn, whatever the number of stages S (6 to
// 9), so a stage has k-blocks of several producers.  A wait looks at a barrier's
// parity alone: before its k-block i a producer waits for the end of k-block i - S,
// and must not take that of i - 2 S for it.  It cannot, having waited for the end
// of k-block i - 3 - S, which comes after i - 2 S.
static_assert(kPairProducers < kPairStages, "a producer's last wait covers the stage's use before last");
constexpr int kPairMaxAcc = 4;  // accumulators in TMEM
constexpr int kPairStaging = 32 * 128;                      // per epilogue warp: 32 rows x 128 bytes
constexpr int kPairBar = 256;
constexpr int kPairSmem = 1024 + kPairStages * kPairStage + kPairEpiWarps * kPairStaging + kPairBar;
// Row tiles of a group.  A group reads all of B once; few row tiles are one
// group.  Head forward + backward under the power cap, 14 row tiles (3584 x 4096
// x 32000): one group 665 + 2056 us, groups of 8 687 + 2072, of 4 723 + 2119;
// 32 row tiles (8192 x 8192 x 32000): of 8 3215 + 9481, of 16 3248 + 9841, of 4
// 3361 + 9764.
__host__ __device__ inline int pair_group(int tiles_m) { return tiles_m <= 16 ? tiles_m : 8; }
constexpr int kLiveBox = 64;  // rows of B a copy with a live N (boxes of 16 alone took 20 to 40 % longer)

enum PairLive { PAIR_LIVE_NONE = 0, PAIR_LIVE_M = 1, PAIR_LIVE_K = 2, PAIR_LIVE_N = 3 };

struct PairGemm {
    CUtensorMap tmA;  // K-major: box 64 (K) x 128; MN-major: box 64 (M) x 64 (K)
    CUtensorMap tmB;  // K-major: box 64 (K) x bn / 2, or x kLiveBox with a live N; MN-major: box 64 (N) x 64 (K)
    CUtensorMap tmB16;  // with a live N: box 64 (K) x 16
    const int* live;  // device count that replaces M, N or K
    int live_dim;     // PairLive
    int M, N, K;
    int bn;           // columns per tile: a multiple of 32 (128 where B is MN-major), at most 256;
                      // chosen on the device for a live N
    int tail_kb;      // > 0: the last wave's tiles are split along K (PairTail of that many k-blocks)
    uint32_t idesc;   // without N
};

// Tile width for a live N: as few tiles as 256 columns allow, of equal width;
// together they cover N rounded up to 64 (the k-blocks of a product over them).
__host__ __device__ inline int pair_live_bn(int n) {
    const int n64 = (n > 1 ? n + 63 : 64) / 64 * 64, tiles = (n64 + 255) / 256;
    return ((n64 + tiles - 1) / tiles + 31) / 32 * 32;
}

// Tiles that do not fill a wave of CTA pairs.  `full` tiles run whole; the
// `rest` (fewer than a wave) are split into `splits` K ranges each, what makes
// their time least: in k-blocks, waves * ceil(kb / splits), and a fifth of one
// for each range's output, which is written and added up.  A range is 8 k-blocks
// at least.  The first range of a tile goes where whole tiles go, the others to
// buffers of their own ((splits - 1) * rest <= 2 pairs of them).  In whole
// numbers, so that host and device agree; on the device by whole warps.
struct PairTail {
    int full, rest, splits;
    __host__ __device__ static uint32_t cost(int s, int rest, int pairs, int kb) {  // and s in the low 8 bits
        if (s > 1 && (s * 8 > kb || (s - 1) * rest > 2 * pairs)) return 0xffffffffu;
        const int per = ((kb < 1 << 19 ? kb : 1 << 19) + s - 1) / s;
        return (uint32_t)(5 * ((rest * s + pairs - 1) / pairs) * per + s * rest) * 256u + (uint32_t)s;
    }
    __host__ __device__ static int most(int pairs) { return pairs < 255 ? pairs : 255; }
    __host__ __device__ PairTail(int tiles, int pairs, int kb) {
        full = tiles / pairs * pairs;
        rest = tiles - full;
        splits = 1;
        if (rest > 0) {
            uint32_t least = 0xffffffffu;
#ifdef __CUDA_ARCH__
            for (int s = 1 + (int)(threadIdx.x & 31); s <= most(pairs); s += 32) least = min(least, cost(s, rest, pairs, kb));
            least = __reduce_min_sync(0xffffffffu, least);
#else
            for (int s = 1; s <= most(pairs) && (s == 1 || s * 8 <= kb); ++s) least = std::min(least, cost(s, rest, pairs, kb));
#endif
            splits = (int)(least & 255u);
        }
        const int per = (kb + splits - 1) / splits;
        splits = (kb + per - 1) / per;  // no empty range
    }
};
// Tile r in the order in which tiles are walked.
__device__ __forceinline__ void pair_tile_at(int r, int tiles_m, int tiles_n, int group, int& m, int& n) {
    const int grp = r / (group * tiles_n);
    const int first = grp * group;
    const int gm = min(group, tiles_m - first);
    const int rr = r - grp * group * tiles_n;
    n = rr / gm;
    m = first + rr - n * gm;
}
// Position of tile (m, n) in that order.
__host__ __device__ inline int pair_tile_index(int m, int n, int tiles_m, int tiles_n) {
    const int group = pair_group(tiles_m), first = m / group * group;
    const int gm = tiles_m - first < group ? tiles_m - first : group;
    return first * tiles_n + n * gm + (m - first);
}

// The part of D that an epilogue call covers: this warp's 32 rows, its columns.
struct PairTile {
    uint32_t tmem;     // address of (this warp's lane quarter, the tile's first column)
    int row0;          // first of the warp's 32 rows of D
    int col0;          // first column of the tile
    int c_begin, c_end;  // this warp's columns within the tile (multiples of 32)
    int m_tile, n_tile, half;
    int part;          // 0: the tile's own place; k > 0: buffer k - 1 of the tail
    int rest;          // of a split tile: its number among them, else -1
    int tile_row;      // row0 within the tile
    int M, N;          // live sizes
    uint8_t* staging;  // kPairStaging bytes of this warp alone, the warps' one after the other
    int lane, warp;    // warp: of the epilogue's
};

struct PairUnit {
    int m0, n0, n_tile, part, rest, kb0, kb1;
};

struct PairShape {
    int M, N, K, bn, tiles_m, tiles_n, kb, total;
    int full, rest, splits, group;
    __device__ explicit PairShape(const PairGemm& g) {
        M = g.M;
        N = g.N;
        K = g.K;
        bn = g.bn;
        if (g.live_dim == PAIR_LIVE_M) M = *g.live;
        if (g.live_dim == PAIR_LIVE_K) K = *g.live;
        if (g.live_dim == PAIR_LIVE_N) {
            N = *g.live;
            bn = pair_live_bn(N);
        }
        tiles_m = max((M + 255) / 256, 1);
        // Few tiles: narrower ones, where a wave takes them all (they too cover N
        // rounded up to 64; 300 x 4096 x 2000 bf16, log probabilities and their gradient
        // 35 + 56 -> 27 + 48 us, the loss and its 32 to 38 + 57 to 69 -> 27 to 31 + 50 to 63;
        // 64 and 300 x 4096 x 32000 as before).  A split product's stay as its reader knows them.
        if (g.live_dim == PAIR_LIVE_N && g.tail_kb == 0)
            for (int narrow = 64; narrow < bn; narrow += 64)
                if (tiles_m * ((N + narrow - 1) / narrow) <= (int)gridDim.x / 2) bn = narrow;
        tiles_n = max((N + bn - 1) / bn, 1);
        kb = max((K + 63) / 64, 1);
        group = pair_group(tiles_m);
        full = tiles_m * tiles_n;
        rest = 0;
        splits = 1;
        if (g.tail_kb > 0) {
            const PairTail t(full, (int)gridDim.x / 2, g.tail_kb);
            full = t.full;
            rest = t.rest;
            splits = t.splits;
        }
        total = full + rest * splits;
    }
    __device__ PairUnit unit(int u) const {
        PairUnit t;
        int r = u, split = 0, per = kb;
        t.part = 0;
        t.rest = -1;
        if (u >= full) {
            split = (u - full) / rest;
            r = u - split * rest;
            per = (kb + splits - 1) / splits;
            if (splits > 1) t.rest = r - full;
            t.part = split > 0 ? (split - 1) * rest + (r - full) + 1 : 0;
        }
        int m;
        pair_tile_at(r, tiles_m, tiles_n, group, m, t.n_tile);
        t.m0 = m * 256;
        t.n0 = t.n_tile * bn;
        t.kb0 = min(split * per, kb);  // a K shorter than the tail's plan leaves its last ranges empty
        t.kb1 = min(t.kb0 + per, kb);
        return t;
    }
};

// acc += the accumulator's columns of this warp, thread = row.
__device__ __forceinline__ void pair_accumulate(const PairTile& t, float (&acc)[128]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (t.c_begin + 16 * i < t.c_end) {
            float v[16];
            tmem_ld16<0>(t.tmem + (uint32_t)(t.c_begin + 16 * i), v);
            tmem_wait_ld_bind(v);
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[16 * i + k] += v[k];
        }
    }
}

template <class Epi, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kPairThreads, 1) pair_gemm_kernel(const __grid_constant__ PairGemm g, const Epi epi,
                                                                     uint32_t* err) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // stays a shared pointer
    uint8_t* sA = base;
    uint8_t* staging = base + kPairStages * kPairStage;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + kPairEpiWarps * kPairStaging);
    uint64_t* empty = full + kPairMaxStages;
    uint64_t* acc_full = empty + kPairMaxStages;
    uint64_t* acc_empty = acc_full + kPairMaxAcc;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + kPairMaxAcc);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((2 * kPairMaxStages + 2 * kPairMaxAcc) * 8 + 8 <= kPairBar, "barriers must fit the barrier area");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int crank = (int)cluster_ctarank();
    const int ustart = (int)(blockIdx.x >> 1), ustep = (int)(gridDim.x >> 1);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairMaxStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        // acc_empty (CTA 0): one arrival per epilogue warp of both CTAs
        for (int b = 0; b < kPairMaxAcc; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * kPairEpiWarps); }
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 0) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();
    const PairShape sh(g);
    constexpr int kStep = Epi::kChunk > 0 ? Epi::kChunk : 1 << 30;  // k-blocks per accumulator
    // Rows of B a stage: with a live N in boxes of 64 (a rest of 48 too) and of 16;
    // what they leave free makes more stages.
    constexpr bool kLive = Epi::kLiveN;
    const int half_n = sh.bn / 2;
    const int rows64 = kLive ? (half_n + 16) / kLiveBox * kLiveBox : half_n, rows_b = max(rows64, half_n);
    const int b_bytes = kLive ? rows_b * 128 : kPairOperand;
    const int stages = kLive ? kPairStages * kPairStage / (kPairOperand + b_bytes) : kPairStages;
    uint8_t* sB = base + stages * kPairOperand;
    const int acc_cols = kLive ? sh.bn : 256, accs = kLive ? min(512 / acc_cols, kPairMaxAcc) : 2;

    if (warp == 0 || warp >= 2 + kPairEpiWarps) {
        if (elect_one()) {
            const int me = warp == 0 ? 0 : warp - 1 - kPairEpiWarps;
            const uint32_t bytes = 2u * (uint32_t)(kPairOperand + rows_b * 64 * 2);  // both CTAs
            int s = me, lag = me, issued = 0;  // this producer's next stage; k-blocks until its next turn
            uint32_t ph = 1;
            for (int u = ustart; u < sh.total && !*abort; u += ustep) {
                const PairUnit t = sh.unit(u);
                const int m0 = t.m0 + crank * 128, n0 = t.n0 + crank * half_n;
                int kb = t.kb0 + lag;
                for (; kb < t.kb1; kb += kPairProducers) {
                    if (!mbar_wait(&empty[s], ph, abort, err, DEVERR_TIMEOUT_TMA)) break;
                    if (crank == 0) mbar_arrive_expect_tx(&full[s], bytes);
                    uint8_t* a = sA + s * kPairOperand;
                    uint8_t* b = sB + s * b_bytes;
                    if (A_MN) {
                        tma_load_2d_pair(a, &g.tmA, &full[s], m0, kb * 64);
                        tma_load_2d_pair(a + 8192, &g.tmA, &full[s], m0 + 64, kb * 64);
                    } else {
                        tma_load_2d_pair(a, &g.tmA, &full[s], kb * 64, m0);
                    }
                    if (B_MN) {
                        for (int c = 0; c < half_n; c += 64)
                            tma_load_2d_pair(b + c * 128, &g.tmB, &full[s], n0 + c, kb * 64);
                    } else if (kLive) {
                        for (int c = 0; c < rows64; c += kLiveBox) tma_load_2d_pair(b + c * 128, &g.tmB, &full[s], kb * 64, n0 + c);
                        for (int c = rows64; c < half_n; c += 16) tma_load_2d_pair(b + c * 128, &g.tmB16, &full[s], kb * 64, n0 + c);
                    } else {
                        tma_load_2d_pair(b, &g.tmB, &full[s], kb * 64, n0);
                    }
                    ++issued;
                    if ((s += kPairProducers) >= stages) {
                        s -= stages;
                        ph ^= 1u;
                    }
                }
                lag = kb - t.kb1;
            }
            // a wait gave up: the loads in flight get a last, bounded chance to land
            if (*abort && crank == 0)
                for (int i = max(issued - (stages + kPairProducers - 1) / kPairProducers, 0); i < issued; ++i) {
                    const int kb = me + i * kPairProducers;  // of all that this pair went through
                    for (int n = 0; n < 1000 && !mbar_try_wait(&full[kb % stages], (uint32_t)(kb / stages) & 1u); ++n) {}
                }
        }
    } else if (warp == 1) {
        if (crank == 0 && elect_one()) {
            const uint32_t idesc = g.idesc | ((uint32_t)(sh.bn >> 3) << 17);
            // descriptors of stage 0; a stage and a step of 16 in K are constants further
            const uint64_t da0 = sdesc_sw128(smem_u32(sA), A_MN ? 8192 : 16, 1024);
            const uint64_t db0 = sdesc_sw128(smem_u32(sB), B_MN ? 8192 : 16, 1024);
            constexpr uint64_t kStepA = (A_MN ? 2048 : 32) / 16, kStepB = (B_MN ? 2048 : 32) / 16;
            int s = 0, b = 0;
            uint32_t ph = 0, acc_ph = 1;
            for (int u = ustart; u < sh.total && !*abort; u += ustep) {
                const PairUnit t = sh.unit(u);
                for (int kb0 = t.kb0; kb0 < t.kb1 && !*abort; kb0 += kStep) {
                    const int kb1 = min(kb0 + kStep, t.kb1);
                    if (!mbar_wait(&acc_empty[b], acc_ph, abort, err, DEVERR_TIMEOUT_MMA)) break;
                    tc_fence_after();
                    const uint32_t d = tmem + (uint32_t)(b * acc_cols);
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!mbar_wait(&full[s], ph, abort, err, DEVERR_TIMEOUT_MMA)) break;
                        tc_fence_after();
                        const uint64_t da = da0 + (uint64_t)(s * (kPairOperand / 16));
                        const uint64_t db = db0 + (uint64_t)(s * (b_bytes / 16));
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            umma_f16_ss_pair(d, da + kk * kStepA, db + kk * kStepB, idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
                        umma_commit_pair(&empty[s]);
                        if (++s == stages) {
                            s = 0;
                            ph ^= 1u;
                        }
                    }
                    umma_commit_pair(&acc_full[b]);
                    if (++b == accs) {
                        b = 0;
                        acc_ph ^= 1u;
                    }
                }
            }
        }
    } else {
        const int ew = warp - 2;
        const int q = warp & 3;
        const int mid = (sh.bn / 32 + 1) / 2 * 32;  // columns of the first half: a multiple of 32
        PairTile tile;
        tile.half = ew >> 2;
        tile.c_begin = tile.half ? mid : 0;
        tile.c_end = tile.half ? sh.bn : mid;
        tile.M = sh.M;
        tile.N = sh.N;
        tile.staging = staging + ew * kPairStaging;
        tile.lane = lane;
        tile.warp = ew;
        int b = 0;
        uint32_t acc_ph = 0;
        auto next = [&] {  // waits for the next accumulator
            const bool here = mbar_wait(&acc_full[b], acc_ph, abort, err, DEVERR_TIMEOUT_EPI) && !*abort;
            if (!__all_sync(0xffffffffu, here)) return false;
            tc_fence_after();
            tile.tmem = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * acc_cols);
            return true;
        };
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(smem_leader(&acc_empty[b]));
            if (++b == accs) {
                b = 0;
                acc_ph ^= 1u;
            }
        };
        bool ok = true;
        for (int u = ustart; u < sh.total && ok; u += ustep) {
            const PairUnit t = sh.unit(u);
            tile.row0 = t.m0 + crank * 128 + q * 32;
            tile.col0 = t.n0;
            tile.m_tile = t.m0 / 256;
            tile.n_tile = t.n_tile;
            tile.part = t.part;
            tile.rest = t.rest;
            tile.tile_row = crank * 128 + q * 32;
            if constexpr (Epi::kChunk > 0) {
                float acc[128];
#pragma unroll
                for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
                for (int kb0 = t.kb0; kb0 < t.kb1; kb0 += kStep) {
                    if (!(ok = next())) break;
                    pair_accumulate(tile, acc);
                    release();
                }
                if (ok) epi.finish(tile, acc);
                // a warp that gave up arrives where the others may wait for it; they see
                // `abort` before their next tile
                else Epi::give_up(tile);
            } else if (t.kb0 < t.kb1) {
                if (!(ok = next())) break;
                epi.tile(tile);
                release();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the pair's MMAs and both epilogues are done with TMEM
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// Turns a 32 x 32 block over: in, thread = row, v = its 32 columns; out, thread
// = column, v = its 32 rows.  Word j of row r lies at j ^ r, so both ways are
// free of bank conflicts.
__device__ __forceinline__ void pair_transpose(const PairTile& t, float (&v)[32]) {
    float* s = reinterpret_cast<float*>(t.staging);
#pragma unroll
    for (int j = 0; j < 32; ++j) s[t.lane * 32 + (j ^ t.lane)] = v[j];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = s[j * 32 + (t.lane ^ j)];
    __syncwarp();
}

// Writes 32 columns of the warp's 32 rows (thread = row, v = its values, times
// alpha) as 16-bit values: through the warp's staging area, so that each row's
// 64 bytes go out as four 16-byte pieces of neighbouring lanes.  ld and out
// decide the piece: whole pieces where every row starts on 16 bytes, else
// single values.
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// out16: element (r, c) of a matrix with row pitch ld; rows < rows, columns < cols are written.
__device__ __forceinline__ void pair_store16(const PairTile& t, const uint32_t (&w)[32], int c, uint16_t* out,
                                             int64_t ld, int rows, int cols) {
    // 64 columns: 32 words per row, chunk k (16 bytes) of row r at k ^ (r & 7)
    const int row = t.lane;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        *reinterpret_cast<uint4*>(t.staging + row * 128 + ((k ^ (row & 7)) * 16)) =
            make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    __syncwarp();
    const bool whole = (ld % 8) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (t.lane >> 3), k = t.lane & 7;
        const int gr = t.row0 + r, gc = t.col0 + c + k * 8;
        const uint4 v = *reinterpret_cast<const uint4*>(t.staging + r * 128 + ((k ^ (r & 7)) * 16));
        if (gr < rows && gc < cols) {
            uint16_t* o = out + (int64_t)gr * ld + gc;
            if (whole && gc + 8 <= cols) {
                *reinterpret_cast<uint4*>(o) = v;
            } else {
                const uint32_t ww[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (gc + e < cols) o[e] = (uint16_t)(ww[e >> 1] >> (16 * (e & 1)));
            }
        }
    }
    __syncwarp();
}

// Epilogue: D times a device scale, in 16 bits.
template <bool BF16>
struct PairOut16 {
    static constexpr int kChunk = 0;
    static constexpr bool kLiveN = false;
    uint16_t* out;
    int64_t ld;
    const float* scale;  // device; null: 1
    __device__ __forceinline__ void tile(const PairTile& t) const {
        const float a = scale ? *scale : 1.0f;
        for (int c = t.c_begin; c < t.c_end; c += 64) {
            if (t.col0 + c >= t.N || t.row0 >= t.M) break;
            uint32_t w[32];
            float v[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (c + 32 * h < t.c_end) {
                    tmem_ld32<0>(t.tmem + (uint32_t)(c + 32 * h), v);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) w[16 * h + i] = pack16<BF16>(v[2 * i] * a, v[2 * i + 1] * a);
            }
            pair_store16(t, w, c, out, ld, t.M, min(t.N, t.col0 + t.c_end));
        }
    }
};

// Writes 32 columns of the warp's 32 rows (thread = row) in fp32 to out, whose
// row 0 is the warp's first: rows below `rows`, columns c .. below `cols` (both a
// multiple of 4), over what is there or added to it.
__device__ __forceinline__ void pair_store32(const PairTile& t, const float (&v)[32], int c, float* out, int64_t pitch,
                                             int rows, int cols, bool over) {
    const int row = t.lane;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        *reinterpret_cast<float4*>(t.staging + row * 128 + ((k ^ (row & 7)) * 16)) =
            make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (t.lane >> 3), k = t.lane & 7;
        const int gc = c + k * 4;
        float4 x = *reinterpret_cast<const float4*>(t.staging + r * 128 + ((k ^ (r & 7)) * 16));
        if (r < rows && gc < cols) {
            float4* o = reinterpret_cast<float4*>(out + r * pitch + gc);
            if (!over) {
                const float4 p = *o;
                x = make_float4(p.x + x.x, p.y + x.y, p.z + x.z, p.w + x.w);
            }
            *o = x;
        }
    }
    __syncwarp();
}

// Epilogue: D in 16 bits; the ranges of a split tile in fp32, each to a buffer
// of 256 x 256 of its own, for pair_join_kernel.
template <bool BF16>
struct PairSplit16 {
    static constexpr int kChunk = 0;
    static constexpr bool kLiveN = false;
    PairOut16<BF16> whole;
    float* buffers;  // range s of split tile i: s * rest + i
    int rest;
    __device__ __forceinline__ void tile(const PairTile& t) const {
        if (t.rest < 0) {
            whole.tile(t);
            return;
        }
        float* out = buffers + (int64_t)(t.part ? t.part - 1 + rest : t.rest) * 65536 + t.tile_row * 256;
        for (int c = t.c_begin; c < t.c_end; c += 32) {
            if (t.col0 + c >= t.N || t.row0 >= t.M) break;
            float v[32];
            tmem_ld32<0>(t.tmem + (uint32_t)c, v);
            tmem_wait_ld();
            pair_store32(t, v, c, out, 256, t.M - t.row0, 256, true);
        }
    }
};

// Adds up a split tile's ranges in their order: 8 rows a CTA, a warp a row.
struct PairJoin {
    const float* buffers;
    int full, rest, splits;  // PairTail's
    int M, N;
    uint16_t* out;
    int64_t ld;
};
template <bool BF16>
__global__ void __launch_bounds__(256) pair_join_kernel(const PairJoin a) {
    pdl_wait();
    const int i = (int)blockIdx.x >> 5, row = ((int)blockIdx.x & 31) * 8 + ((int)threadIdx.x >> 5);
    const int col = ((int)threadIdx.x & 31) * 8;
    const int tiles_m = (a.M + 255) / 256, tiles_n = (a.N + 255) / 256;
    int m, n;
    pair_tile_at(a.full + i, tiles_m, tiles_n, pair_group(tiles_m), m, n);
    const int gr = m * 256 + row, gc = n * 256 + col;
    if (gr >= a.M || gc >= a.N) return;
    const float* p = a.buffers + (int64_t)i * 65536 + row * 256 + col;
    float v[8] = {};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
        const float4* q = reinterpret_cast<const float4*>(p + (int64_t)s * a.rest * 65536);
        const float4 x = q[0], y = q[1];
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = pack16<BF16>(v[2 * k], v[2 * k + 1]);
    uint16_t* o = a.out + (int64_t)gr * a.ld + gc;
    if (a.ld % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && gc + 8 <= a.N) {
        *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (gc + k < a.N) o[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    }
}

// Epilogue: D in fp32, stored by the first K range of a sum over launches and
// added by the later ones; a tail's further ranges go to `extra`, 256 x 256
// each.  Each element has one writer per launch, so the order of a sum is the
// order of the launches.
struct PairSlab {
    static constexpr int kChunk = 0;
    static constexpr bool kLiveN = false;
    float* slab;
    int64_t ld;  // a multiple of 4
    float* extra;
    int first;
    __device__ __forceinline__ void tile(const PairTile& t) const {
        float* out = t.part ? extra + (int64_t)(t.part - 1) * 65536 + t.tile_row * 256
                            : slab + (int64_t)t.row0 * ld + t.col0;
        const int64_t pitch = t.part ? 256 : ld;
        const int cols = t.part ? 256 : (int)min((int64_t)256, ld - t.col0);
        for (int c = t.c_begin; c < t.c_end; c += 32) {
            if (t.col0 + c >= t.N || t.row0 >= t.M) break;
            float v[32];
            tmem_ld32<0>(t.tmem + (uint32_t)c, v);
            tmem_wait_ld();
            pair_store32(t, v, c, out, pitch, t.M - t.row0, cols, first);
        }
    }
};

// The same where the tile's columns are the rows of the result (live N): slab
// row = column of D.  A tail's further ranges go to `extra`, 256 columns of D
// by 256 rows each.
struct PairSlabT {
    static constexpr int kChunk = 0;
    static constexpr bool kLiveN = true;
    float* slab;
    int64_t ld;  // at least M
    float* extra;
    int first;
    __device__ __forceinline__ void tile(const PairTile& t) const {
        float* out = t.part ? extra + (int64_t)(t.part - 1) * 65536 : slab + (int64_t)t.col0 * ld + t.row0 - t.tile_row;
        const int64_t pitch = t.part ? 256 : ld;
        const bool in = t.row0 + t.lane < t.M;
        for (int c = t.c_begin; c < t.c_end; c += 32) {
            if (t.col0 + c >= t.N || t.row0 >= t.M) break;
            float v[32];
            tmem_ld32<0>(t.tmem + (uint32_t)c, v);
            tmem_wait_ld();
            // a column's 32 rows (the warp's lanes) are 128 bytes of a slab row
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (in && t.col0 + c + j < t.N) {
                    float* o = out + (int64_t)(c + j) * pitch + t.tile_row + t.lane;
                    *o = first ? v[j] : *o + v[j];
                }
        }
    }
};

// ---- host ----
struct PairOperand {
    const void* ptr;
    int64_t ld;    // row pitch in elements
    int64_t rows;  // rows that may be read (K rows where MN-major, M or N rows where K-major)
    int64_t cols;
};

inline int pair_count() { return num_sms() / 2; }

template <class Epi, bool A_MN, bool B_MN>
int pair_gemm_launch(PairOperand A, PairOperand B, int M, int N, int K, const int* live, int live_dim, int bn,
                     int tail_kb, bool bf16, const Epi& epi, cudaStream_t st) {
    DeviceRuntime* rt = nullptr;
    AETH_TRY(runtime_for_current(&rt));
    PairGemm g;
    AETH_TRY(make_tmap_16b(&g.tmA, A.ptr, (uint64_t)A.cols, (uint64_t)A.rows, A.ld, 64, A_MN ? 64 : 128, bf16));
    constexpr bool live_n = Epi::kLiveN;
    if (live_n != (live_dim == PAIR_LIVE_N)) return AETH_ERR_ARG;
    AETH_TRY(make_tmap_16b(&g.tmB, B.ptr, (uint64_t)B.cols, (uint64_t)B.rows, B.ld, 64,
                           B_MN ? 64 : live_n ? kLiveBox : bn / 2, bf16));
    if (live_n) AETH_TRY(make_tmap_16b(&g.tmB16, B.ptr, (uint64_t)B.cols, (uint64_t)B.rows, B.ld, 64, 16, bf16));
    g.live = live;
    g.live_dim = live_dim;
    g.M = M;
    g.N = N;
    g.K = K;
    g.bn = bn;
    g.tail_kb = tail_kb;
    g.idesc = idesc_f16(256, 0, bf16, A_MN, B_MN);
    auto kern = pair_gemm_kernel<Epi, A_MN, B_MN>;
    static std::atomic<bool> allowed[kMaxDevices] = {};
    AETH_TRY(allow_shared(kern, kPairSmem, allowed));
    const int64_t units = (int64_t)((M + 255) / 256) * (live_n ? (N + 63) / 64 : (N + bn - 1) / bn);
    const unsigned pairs = (unsigned)(tail_kb > 0 ? pair_count() : std::min<int64_t>(units, pair_count()));
    AETH_CUDA(launch_after(kern, dim3(2 * pairs), dim3(kPairThreads), kPairSmem, st, 2, g, epi, rt->err_word));
    return AETH_OK;
}

}  // namespace aeth
