// aeth_train.cu -- libaeth_galore: the training operators around the optimizer
// step (section 3b of include/aeth_galore.h): the head's loss and gradient, the
// RMS norm whose input is kept in 8 bits, and the weight gradient taken from
// that checkpoint.
#include <algorithm>
#include <type_traits>

#include "checkpoint.cuh"
#include "common.cuh"
#include "head_loss.cuh"
#include "pair_gemm.cuh"

using namespace aeth;

namespace {

bool is16(int dtype) { return dtype == AETH_DTYPE_BF16 || dtype == AETH_DTYPE_F16; }
bool known_dtype(int dtype) { return dtype == AETH_DTYPE_F32 || is16(dtype); }
int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Carves a workspace into 256-byte aligned parts.
struct Carver {
    uint8_t* base;
    size_t used = 0;
    explicit Carver(void* p) : base(static_cast<uint8_t*>(p)) {}
    template <typename T>
    T* take(int64_t count) {
        T* p = reinterpret_cast<T*>(base + used);
        used += (size_t)up(count * (int64_t)sizeof(T), 256);
        return p;
    }
};

// ---------------------------------------------------------------------------
// Head loss
// ---------------------------------------------------------------------------
constexpr int64_t kHeadMaxDim = 1ll << 30;       // token, feature and vocabulary counts (tile coordinates are int)
constexpr int64_t kHeadPieceBytes = 256ll << 20;  // scratch of a vocabulary piece: its G's, and the buffers of dH's tail

// Columns per tile for a product of `cols` columns (B K-major) with `tiles_m`
// row tiles: what makes the last wave of tiles over the 74 CTA pairs least
// wasteful.  A wave lasts about bn columns plus a share that does not shrink
// with bn (32 columns' worth of time).
int head_bn(int64_t tiles_m, int64_t cols) {
    int best = 256;
    int64_t least = INT64_MAX;
    for (int bn = 256; bn >= 64; bn -= 32) {
        const int64_t units = tiles_m * ((cols + bn - 1) / bn), pairs = num_sms() / 2;
        const int64_t cost = (units + pairs - 1) / pairs * (bn + 32);
        if (cost < least) {
            least = cost;
            best = bn;
        }
    }
    return best;
}

// Whether the tokens are the products' columns (pair_gemm.cuh): where tiles of
// 256 rows would be a tenth larger than the columns that cover the tokens, and
// masks may leave fewer still.  Measured at d 4096, vocabulary 32000, forward
// and backward, rows against columns: 16 tokens 66.5 + 189 and 58.5 + 173
// us; 300: 104 + 309 and 91 + 273; but 256: 69 + 237 and 72 + 250 (the blocks
// are turned over in the epilogue), 512: 117 + 410 and 137 + 397.
bool head_tokens_as_columns(int64_t n) {
    if (n > 1024) return false;
    const int64_t bn = pair_live_bn((int)n);
    return 10 * up(n, 256) >= 11 * ((n + bn - 1) / bn * bn);
}

struct HeadPlan {
    int64_t n_pad, dp, piece, ldg;
    bool live_n;  // tokens as the products' columns (see pair_gemm.cuh)
    int bn;      // tile columns of the forward otherwise
    int np;      // column ranges of the forward's statistics
    int tail_kb;    // k-blocks of a piece's dH product
    int64_t extra;  // buffers of its tail
    int gs;         // G's of a piece: a second one without the token weights (head_loss.cuh)

    HeadPlan(int64_t n, int64_t d, int64_t vocab, int gs_ = 1) : gs(gs_) {
        n_pad = up(std::max<int64_t>(n, 1), 256);
        dp = up(d, 8);
        live_n = head_tokens_as_columns(n);
        bn = head_bn(n_pad / 256, vocab);
        np = 2 * (int)((vocab + (live_n ? 256 : bn) - 1) / (live_n ? 256 : bn));
        // buffers that a dH product's tail may need: two waves of tiles at most
        const int64_t pairs = pair_count(), tiles_m = n_pad / 256;
        const int64_t most = std::min<int64_t>(pairs, (vocab + 511) / 512) - 1;  // ranges of 8 k-blocks past the first
        extra = std::min<int64_t>(2 * pairs, most * std::min<int64_t>(tiles_m * ((d + 255) / 256), pairs));
        // a piece is a number of 256-entry tiles whose G's fit beside them; of those, from the
        // largest down to half of it (64 are looked at), the one with the fewest waves of tiles over all pieces
        const int64_t all = (vocab + 255) / 256;
        const int64_t fit = std::max<int64_t>((kHeadPieceBytes - extra * 262144) / (512 * n_pad * gs), 1);
        int64_t best = fit, least = INT64_MAX;
        auto waves = [&](int64_t tiles) { return (tiles * tiles_m + pairs - 1) / pairs; };
        for (int64_t p = fit; p >= std::max((fit + 1) / 2, fit - 64) && fit < all; --p) {
            const int64_t cost = all / p * waves(p) + waves(all % p);
            if (cost < least) {
                least = cost;
                best = p;
            }
        }
        piece = std::min(256 * best, up(vocab, 8));
        ldg = up(piece, 8);
        tail_kb = (int)((piece + 63) / 64);
    }
};

// The forward of a few tokens reads the weight by rows (head_vec_kernel).
constexpr int kHeadVecShared = 96 * 1024;
bool head_vec_fits(int64_t n, int64_t d) { return n <= kHeadVecTokens && n * up(d, 8) * 2 <= kHeadVecShared; }

struct HeadWork {
    int *rows, *pos, *lab, *count;
    unsigned* done;
    uint16_t* h;
    // forward
    float* label_logit;
    float2* part;
    // backward
    float *coef, *lse2, *out_scale, *row_scale, *slab, *extra;
    uint16_t *g, *g_unit;
    size_t bytes;

    HeadWork(const HeadPlan& p, int64_t n, bool backward, void* ws) {
        Carver c(ws);
        rows = c.take<int>(p.n_pad);
        pos = c.take<int>(std::max<int64_t>(n, 1));
        lab = c.take<int>(p.n_pad);
        count = c.take<int>(1);
        done = c.take<unsigned>(1);
        h = c.take<uint16_t>(p.n_pad * p.dp);
        label_logit = nullptr;
        part = nullptr;
        coef = lse2 = out_scale = row_scale = slab = extra = nullptr;
        g = g_unit = nullptr;
        if (!backward) {
            label_logit = c.take<float>(p.n_pad);
            part = c.take<float2>(std::max<int64_t>((int64_t)p.np * p.n_pad, num_sms() * kHeadVecTokens));
        } else {
            coef = c.take<float>(p.n_pad);
            lse2 = c.take<float>(p.n_pad);
            row_scale = c.take<float>(p.n_pad);
            out_scale = c.take<float>(1);
            g = c.take<uint16_t>(p.n_pad * p.ldg);
            g_unit = p.gs > 1 ? c.take<uint16_t>(p.n_pad * p.ldg) : g;
            slab = c.take<float>(p.n_pad * p.dp);
            extra = c.take<float>(p.extra * 65536);
        }
        bytes = c.used;
    }
};

int head_check(const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight, int dtype,
               const int64_t* labels, int64_t n, int64_t d, int64_t vocab) {
    if (n < 0 || d <= 0 || vocab <= 0 || !weight || ld_weight < d) return AETH_ERR_ARG;
    if (n > 0 && (!hidden || !labels || ld_hidden < d)) return AETH_ERR_ARG;
    if (!known_dtype(dtype)) return AETH_ERR_ARG;
    if (!is16(dtype)) return AETH_ERR_UNSUPPORTED;
    if (n > kHeadMaxDim || d > kHeadMaxDim || vocab > kHeadMaxDim) return AETH_ERR_UNSUPPORTED;
    const int64_t tn = (n + 255) / 256, tv = (vocab + 63) / 64, td = (d + 255) / 256;  // tiles of the products
    if (tn * tv > kHeadMaxDim || tn * td > kHeadMaxDim || tv * td > kHeadMaxDim) return AETH_ERR_UNSUPPORTED;
    if (!aligned16(weight) || ld_weight % 8) return AETH_ERR_UNSUPPORTED;  // TMA reads the weight in place
    return AETH_OK;
}

// Fills in what every call gives, numbers the live tokens and gathers their rows.
int head_rows(HeadRows a, const int64_t* labels, int64_t n, int64_t d, int64_t vocab, int64_t ignore_index,
              const void* hidden, int64_t ld, const HeadPlan& p, const HeadWork& w, cudaStream_t st) {
    DeviceRuntime* rt = nullptr;
    AETH_TRY(runtime_for_current(&rt));
    a.labels = labels;
    a.n = n;
    a.ignore_index = ignore_index;
    a.vocab = (int)vocab;
    a.rows = w.rows;
    a.pos = w.pos;
    a.lab = w.lab;
    a.count = w.count;
    a.done = w.done;
    a.h = static_cast<const uint16_t*>(hidden);
    a.ld = ld;
    a.d = (int)d;
    a.out = w.h;
    a.ldo = p.dp;
    const unsigned ctas = (unsigned)std::min<int64_t>(n, num_sms());
    if (n <= kHeadScan) {
        head_rows_kernel<true><<<ctas, 1024, 0, st>>>(a, rt->err_word);
        AETH_LAUNCH_CHECK();
    } else {
        head_rows_kernel<false><<<1, 1024, 0, st>>>(a, rt->err_word);
        AETH_LAUNCH_CHECK();
        AETH_CUDA(launch_after(head_pack_kernel, dim3(ctas), dim3(1024), 0, st, 1, a));
    }
    return AETH_OK;
}

template <bool BF16>
int head_vec(const HeadVec& a, int64_t n, int ctas, float* losses, float* lse, float* loss, cudaStream_t st) {
    DeviceRuntime* rt = nullptr;
    AETH_TRY(runtime_for_current(&rt));
    auto kern = n == 1 ? head_vec_kernel<BF16, 1> : n == 2 ? head_vec_kernel<BF16, 2>
              : n == 3 ? head_vec_kernel<BF16, 3> : head_vec_kernel<BF16, 4>;
    const int smem = (int)(n * up(a.d, 8) * 2);
    static std::atomic<bool> allowed[kHeadVecTokens][kMaxDevices] = {};
    AETH_TRY(allow_shared(kern, kHeadVecShared, allowed[n - 1]));
    kern<<<ctas, kHeadVecThreads, smem, st>>>(a);
    AETH_LAUNCH_CHECK();
    AETH_CUDA(launch_after(head_vec_loss_kernel, dim3(1), dim3(32 * (unsigned)n), 0, st, 1, a, (int)n, ctas, losses, lse,
                           loss, rt->err_word));
    return AETH_OK;
}

// UNIT: d_hidden comes from a G without the token weights
template <bool BF16, bool UNIT>
int head_backward(const HeadPlan& p, const HeadWork& w, const void* weight, int64_t ld_weight, int64_t n, int64_t d,
                  int64_t vocab, void* d_hidden, int64_t ld_dh, void* d_weight, int64_t ld_dw, cudaStream_t st) {
    const uint16_t* W = static_cast<const uint16_t*>(weight);
    uint16_t *g = UNIT && !d_weight ? nullptr : w.g, *g_unit = UNIT ? w.g_unit : nullptr;
    for (int64_t v0 = 0; v0 < vocab; v0 += p.piece) {
        const int64_t vp = std::min(p.piece, vocab - v0);
        const PairOperand H{w.h, p.dp, n, d}, Wp{W + v0 * ld_weight, ld_weight, vp, d};
        const PairOperand G{w.g, p.ldg, n, vp}, Gh{UNIT ? w.g_unit : w.g, p.ldg, n, vp};
        if (p.live_n) {
            HeadGradT<BF16, UNIT> eg{w.lab, w.coef, w.lse2, g, g_unit, p.ldg, (int)n, (int)v0};
            AETH_TRY((pair_gemm_launch<HeadGradT<BF16, UNIT>, false, false>(Wp, H, (int)vp, (int)n, (int)d, w.count,
                                                                            PAIR_LIVE_N, 256, 0, BF16, eg, st)));
        } else {
            HeadGrad<BF16, UNIT> eg{w.lab, w.coef, w.lse2, g, g_unit, p.ldg, (int)n, (int)v0};
            AETH_TRY((pair_gemm_launch<HeadGrad<BF16, UNIT>, false, false>(H, Wp, (int)n, (int)vp, (int)d, w.count, PAIR_LIVE_M,
                                                                           head_bn(p.n_pad / 256, vp), 0, BF16, eg, st)));
        }
        if (d_weight) {
            PairOut16<BF16> ew{static_cast<uint16_t*>(d_weight) + v0 * ld_dw, ld_dw, w.out_scale};
            AETH_TRY((pair_gemm_launch<PairOut16<BF16>, true, true>(G, H, (int)vp, (int)d, (int)n, w.count, PAIR_LIVE_K,
                                                                    256, 0, BF16, ew, st)));
        }
        if (d_hidden) {
            if (p.live_n) {
                PairSlabT es{w.slab, p.dp, w.extra, v0 == 0};
                AETH_TRY((pair_gemm_launch<PairSlabT, true, false>(Wp, Gh, (int)d, (int)n, (int)vp, w.count, PAIR_LIVE_N,
                                                                   256, p.tail_kb, BF16, es, st)));
            } else {
                PairSlab es{w.slab, p.dp, w.extra, v0 == 0};
                AETH_TRY((pair_gemm_launch<PairSlab, false, true>(Gh, Wp, (int)n, (int)d, (int)vp, w.count, PAIR_LIVE_M,
                                                                  256, p.tail_kb, BF16, es, st)));
            }
        }
    }
    if (d_hidden && n > 0) {
        const HeadDh a{w.slab, p.dp, w.extra, pair_count(), p.tail_kb, p.live_n, w.pos, w.count, n, (int)d,
                       UNIT ? nullptr : w.out_scale, w.row_scale, static_cast<uint16_t*>(d_hidden), ld_dh};
        const unsigned cols = (unsigned)((d + 1023) / 1024);
        const int64_t rows = std::max<int64_t>(16 * num_sms() / cols, 1);
        // few tokens: one at a time, and more of its parts
        if (n <= rows) AETH_CUDA(launch_after(head_dh_kernel<BF16, 1>, dim3((unsigned)n, cols), dim3(128), 0, st, 1, a));
        else AETH_CUDA(launch_after(head_dh_kernel<BF16, 4>, dim3((unsigned)std::min((n + 3) / 4, rows), cols), dim3(128), 0,
                                    st, 1, a));
    }
    return AETH_OK;
}

// ---------------------------------------------------------------------------
// Checkpoints
// ---------------------------------------------------------------------------
constexpr int64_t kCkptMaxDim = 1ll << 30;

int ckpt_dims(int64_t rows, int64_t d, int dtype) {
    if (rows < 0 || d <= 0 || !known_dtype(dtype)) return AETH_ERR_ARG;
    if (rows > kCkptMaxDim || d > kCkptMaxDim) return AETH_ERR_UNSUPPORTED;
    return AETH_OK;
}

// How a kernel that holds rows in registers is laid out: vpt eights of
// features a thread, tx threads a row, ty rows a CTA.
struct RowPlan {
    int vpt, tx, ty;
    bool wide;
    unsigned grid;

    // per_sm: CTAs an SM is given (they walk over the rows); 0: those that its registers hold
    RowPlan(int64_t rows, int64_t d, int per_sm) {
        const int64_t nv = (d + 7) / 8;
        wide = nv > 1024;
        // A row spread over four times the threads has the shorter chain of loads, which
        // counts when there are too few rows to fill the SMs; and a row of 32 eights or fewer
        // has one for each lane of a warp (6206 x 135 f16: store 8.5 us for 16.5, gradient 10 for 22).
        vpt = wide || (rows > 2 * num_sms() && nv > 32) ? 4 : 1;
        const int most = 1024 / vpt;
        tx = wide ? most : (int)((nv + vpt - 1) / vpt + 31) / 32 * 32;
        ty = (int)std::max<int64_t>(std::min<int64_t>(256 / tx, rows), 1);
        if (per_sm == 0) per_sm = std::max(65536 / ((vpt == 4 ? 128 : 64) * tx * ty), 1);
        grid = (unsigned)std::min<int64_t>((rows + ty - 1) / ty, (int64_t)num_sms() * per_sm);
    }
    dim3 block() const { return dim3(tx, ty); }
    // dynamic shared memory: rows of 4 bytes a feature (gain where it is kept there, and `more`)
    int shared(int more = 0) const {
        return ((ck_shared_gain(vpt, wide) ? 1 : 0) + (wide ? 0 : more)) * vpt * tx * 32;
    }
};
constexpr int kStorePerSm = 8, kBackPerSm = 0;

// The ring's layout for rows of d features: groups of tx threads that hold a
// row in four eights each, as many stages as shared memory takes beside gain.
// Taken for many rows (each SM walks over several) that bulk copies can move
// and of which a group has room for two (f32: up to 15968 features).
constexpr int kRingShared = 220 * 1024;
CkptRing ring_plan(int64_t d, int size, bool res) {
    CkptRing r;
    const bool wide = d > 8192;
    r.tx = wide ? kRingThreads : (int)((d + 1023) / 1024) * 32;
    r.eights = (int)((d + 8 * r.tx - 1) / (8 * r.tx));
    r.groups = kRingThreads / r.tx;
    const int row = (int)up(d * size, 128);
    r.res_at = row;
    r.codes_at = row * (res && !wide ? 2 : 1);
    r.stage_bytes = r.codes_at + (int)up(d, 128);
    const int room = kRingShared - r.gain_bytes();
    while (r.groups > 1 && room / r.stage_bytes / r.groups < 2) r.groups /= 2;  // two stages a group at least
    r.stages = std::min(room / r.stage_bytes / r.groups, kRingMaxStages);
    return r;
}
bool ring_fits(int64_t rows, int64_t d, int size, bool res) {
    return rows > 2 * num_sms() && d % 16 == 0 && d >= 256 && d <= 16384 && ring_plan(d, size, res).stages >= 2;
}

template <typename F>
int by_type(int dtype, F f) {
    if (dtype == AETH_DTYPE_F32) return f((float*)nullptr);
    if (dtype == AETH_DTYPE_F16) return f((__half*)nullptr);
    return f((__nv_bfloat16*)nullptr);
}

template <int V>
using Int = std::integral_constant<int, V>;

// f(type tag, vpt, vec, wide) with the last three as compile-time constants
template <typename F>
int by_row(int dtype, const RowPlan& p, bool vec, F f) {
    return by_type(dtype, [&](auto* tag) {
        if (p.wide) return vec ? f(tag, Int<4>(), Int<1>(), Int<1>()) : f(tag, Int<4>(), Int<0>(), Int<1>());
        if (p.vpt > 1) return vec ? f(tag, Int<4>(), Int<1>(), Int<0>()) : f(tag, Int<4>(), Int<0>(), Int<0>());
        return vec ? f(tag, Int<1>(), Int<1>(), Int<0>()) : f(tag, Int<1>(), Int<0>(), Int<0>());
    });
}

// Whether rows of pitch ld at p can be taken in eights of `size` bytes each
bool vec_rows(const void* p, int64_t ld, int size) {
    const int bytes = std::min(8 * size, 16);
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * size % bytes == 0;
}
int type_size(int dtype) { return dtype == AETH_DTYPE_F32 ? 4 : 2; }

int decode(const CkptRead& a, void* out, int64_t ld_out, int dtype, cudaStream_t st) {
    const bool vec = a.d % 8 == 0 && vec_rows(a.codes, a.d, 1) && vec_rows(out, ld_out, type_size(dtype)) &&
                     (!a.gain || aligned16(a.gain));
    RowPlan p(a.rows, a.d, kStorePerSm);
    return by_row(dtype, p, vec, [&](auto* tag, auto vpt, auto v, auto wide) {
        using T = std::remove_pointer_t<decltype(tag)>;
        T* o = static_cast<T*>(out);
        if (a.gain) {
            ckpt_norm_kernel<T, vpt.value, v.value, wide.value><<<p.grid, p.block(), p.shared(), st>>>(a, o, ld_out);
        } else if (vec && a.d % kCkptBlock == 0 && ld_out == a.d && aligned16(a.codes) && aligned16(out)) {
            const int64_t n16 = a.rows * a.d / 16;
            ckpt_decode_flat_kernel<T><<<(unsigned)std::min<int64_t>((n16 + 1023) / 1024, 1 << 20), 256, 0, st>>>(
                reinterpret_cast<const uint4*>(a.codes), a.scales, n16, o);
        } else {
            const unsigned spans = (unsigned)((a.d + 8 * p.vpt * p.tx - 1) / (8 * p.vpt * p.tx));
            ckpt_decode_kernel<T, vpt.value, v.value><<<dim3(p.grid, spans), p.block(), 0, st>>>(a, o, ld_out);
        }
        AETH_LAUNCH_CHECK();
        return (int)AETH_OK;
    });
}

// The weight gradient's tiles that do not fill a wave are split along the tokens
// where that takes 32 k-blocks or more (8 us) off the product; a kernel of its
// own then adds up the ranges, for 5 us and a launch.  A call without and with
// the split: 8170 x (216 x 952) 65 and 26 us (4 tiles), 8192 x (1024 x 1024) 51
// and 31, 8192 x (5120 x 5120) 321 and 316; with 24 k-blocks less 2048 x (512 x
// 2048) 22 and 28.
struct GradTail {
    int full = 0, rest = 0, splits = 1;
    int64_t buffers() const { return splits > 1 ? (int64_t)rest * splits : 0; }
};
constexpr int kGradTailBlocks = 32;
GradTail grad_tail(int64_t rows, int64_t m, int64_t d) {
    GradTail g;
    const int64_t tiles = (m + 255) / 256 * ((d + 255) / 256), kb = (rows + 63) / 64;
    if (kb < 1 || tiles > kCkptMaxDim) return g;
    const PairTail t((int)tiles, pair_count(), (int)kb);
    const int64_t waves = ((int64_t)t.rest * t.splits + pair_count() - 1) / pair_count();
    if (t.splits < 2 || kb - waves * ((kb + t.splits - 1) / t.splits) < kGradTailBlocks) return g;
    g.full = t.full;
    g.rest = t.rest;
    g.splits = t.splits;
    return g;
}

template <bool BF16>
int grad_product(const PairOperand& A, const PairOperand& B, int64_t m, int64_t d, int64_t rows, const GradTail& tail,
                 float* buffers, void* d_weight, int64_t ld_dw, cudaStream_t st) {
    uint16_t* out = static_cast<uint16_t*>(d_weight);
    const PairSplit16<BF16> e{{out, ld_dw, nullptr}, buffers, tail.rest};
    const int tail_kb = tail.splits > 1 ? (int)((rows + 63) / 64) : 0;
    AETH_TRY((pair_gemm_launch<PairSplit16<BF16>, true, true>(A, B, (int)m, (int)d, (int)rows, nullptr, PAIR_LIVE_NONE, 256,
                                                              tail_kb, BF16, e, st)));
    if (tail.splits == 1) return AETH_OK;
    const PairJoin j{buffers, tail.full, tail.rest, tail.splits, (int)m, (int)d, out, ld_dw};
    AETH_CUDA(launch_after(pair_join_kernel<BF16>, dim3(32u * (unsigned)tail.rest), dim3(256), 0, st, 1, j));
    return AETH_OK;
}

}  // namespace

extern "C" {

int aeth_cut_ce_workspace(int64_t n, int64_t d, int64_t vocab, int backward, size_t* bytes) {
    if (n < 0 || d <= 0 || vocab <= 0 || !bytes) return set_err(AETH_ERR_ARG);
    if (n > kHeadMaxDim || d > kHeadMaxDim || vocab > kHeadMaxDim) return set_err(AETH_ERR_UNSUPPORTED);
    *bytes = HeadWork(HeadPlan(n, d, vocab), n, backward != 0, nullptr).bytes;
    if (backward) *bytes = std::max(*bytes, HeadWork(HeadPlan(n, d, vocab, 2), n, true, nullptr).bytes);
    return AETH_OK;
}

int aeth_cut_ce_forward(const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight, int dtype,
                        const int64_t* labels, int64_t n, int64_t d, int64_t vocab, int64_t ignore_index,
                        float* losses, float* lse, float* loss, void* workspace, size_t workspace_bytes,
                        aeth_stream_t stream) {
    AETH_TRY(head_check(hidden, ld_hidden, weight, ld_weight, dtype, labels, n, d, vocab));
    if (!loss || (n > 0 && (!losses || !lse || !workspace))) return set_err(AETH_ERR_ARG);
    cudaStream_t st = to_stream(stream);
    if (n == 0) {
        AETH_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), st));
        return AETH_OK;
    }
    const bool bf16 = dtype == AETH_DTYPE_BF16;
    const HeadPlan p(n, d, vocab);
    const HeadWork w(p, n, false, workspace);
    if (workspace_bytes < w.bytes || !aligned16(workspace)) return set_err(AETH_ERR_ARG);
    if (head_vec_fits(n, d)) {
        const HeadVec a{static_cast<const uint16_t*>(hidden), ld_hidden, static_cast<const uint16_t*>(weight), ld_weight,
                        labels, (int)d, (int)vocab, ignore_index, w.label_logit, w.part};
        const int ctas = num_sms();
        return bf16 ? head_vec<true>(a, n, ctas, losses, lse, loss, st) : head_vec<false>(a, n, ctas, losses, lse, loss, st);
    }
    AETH_TRY(head_rows({}, labels, n, d, vocab, ignore_index, hidden, ld_hidden, p, w, st));
    const PairOperand H{w.h, p.dp, n, d}, W{weight, ld_weight, vocab, d};
    if (p.live_n) {
        HeadStatsT es{w.lab, w.label_logit, w.part, p.n_pad};
        AETH_TRY((pair_gemm_launch<HeadStatsT, false, false>(W, H, (int)vocab, (int)n, (int)d, w.count, PAIR_LIVE_N, 256, 0,
                                                             bf16, es, st)));
    } else {
        HeadStats es{w.lab, w.label_logit, w.part, p.n_pad};
        AETH_TRY((pair_gemm_launch<HeadStats, false, false>(H, W, (int)n, (int)vocab, (int)d, w.count, PAIR_LIVE_M, p.bn, 0,
                                                            bf16, es, st)));
    }
    const HeadLoss l{w.part, p.n_pad, p.np, w.label_logit, w.rows, w.pos, w.count, w.done, n, losses, lse, loss};
    AETH_CUDA(launch_after(head_loss_kernel, dim3((unsigned)std::min<int64_t>((n + 7) / 8, 4 * num_sms())), dim3(512), 0, st,
                           1, l));
    return AETH_OK;
}

int aeth_cut_ce_backward(const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight, int dtype,
                         const int64_t* labels, int64_t n, int64_t d, int64_t vocab, int64_t ignore_index,
                         const float* lse, const float* grad_losses, float scale, void* d_hidden, int64_t ld_dh,
                         void* d_weight, int64_t ld_dw, void* workspace, size_t workspace_bytes,
                         aeth_stream_t stream) {
    AETH_TRY(head_check(hidden, ld_hidden, weight, ld_weight, dtype, labels, n, d, vocab));
    if (!d_hidden && !d_weight) return set_err(AETH_ERR_ARG);
    if ((d_hidden && ld_dh < d) || (d_weight && ld_dw < d)) return set_err(AETH_ERR_ARG);
    if (n > 0 && (!lse || !workspace)) return set_err(AETH_ERR_ARG);
    cudaStream_t st = to_stream(stream);
    if (n == 0) {
        if (d_weight)
            AETH_CUDA(cudaMemset2DAsync(d_weight, (size_t)ld_dw * 2, 0, (size_t)d * 2, (size_t)vocab, st));
        return AETH_OK;
    }
    const bool bf16 = dtype == AETH_DTYPE_BF16;
    const bool unit = !bf16 && grad_losses && d_hidden;
    const HeadPlan p(n, d, vocab, unit ? 2 : 1);
    const HeadWork w(p, n, true, workspace);
    if (workspace_bytes < w.bytes || !aligned16(workspace)) return set_err(AETH_ERR_ARG);
    HeadRows a = {};
    a.lse = lse;
    a.grad = grad_losses;
    a.scale = scale;
    a.g_bits = head_g_bits(bf16);
    a.g_scale = head_g_scale(bf16);
    a.coef = w.coef;
    a.lse2 = w.lse2;
    a.out_scale = w.out_scale;
    a.row_scale = w.row_scale;
    AETH_TRY(head_rows(a, labels, n, d, vocab, ignore_index, hidden, ld_hidden, p, w, st));
    auto run = bf16 ? head_backward<true, false> : unit ? head_backward<false, true> : head_backward<false, false>;
    return run(p, w, weight, ld_weight, n, d, vocab, d_hidden, ld_dh, d_weight, ld_dw, st);
}

int aeth_rms_norm_checkpoint(const void* x, int64_t ld_x, const void* residual, int64_t ld_residual, const void* gain,
                             int gain_dtype, int dtype, int64_t rows, int64_t d, float eps, void* sum_out, void* y,
                             int8_t* codes, float* scales, aeth_stream_t stream) {
    AETH_TRY(ckpt_dims(rows, d, dtype));
    if (!gain || !known_dtype(gain_dtype)) return set_err(AETH_ERR_ARG);
    if (rows == 0) return AETH_OK;
    if (!x || !y || !codes || !scales || ld_x < d || (residual && (!sum_out || ld_residual < d)))
        return set_err(AETH_ERR_ARG);
    cudaStream_t st = to_stream(stream);
    const int sz = type_size(dtype);
    const bool vec = d % 8 == 0 && aligned16(gain) && vec_rows(x, ld_x, sz) && vec_rows(y, d, sz) && vec_rows(codes, d, 1) &&
                     (!residual || (vec_rows(residual, ld_residual, sz) && vec_rows(sum_out, d, sz)));
    const RowPlan p(rows, d, kStorePerSm);
    return by_row(dtype, p, vec, [&](auto* tag, auto vpt, auto v, auto wide) {
        using T = std::remove_pointer_t<decltype(tag)>;
        CkptStore<T> a{static_cast<const T*>(x), ld_x, static_cast<const T*>(residual), ld_residual, gain, gain_dtype,
                       rows, (int)d, eps, static_cast<T*>(sum_out), static_cast<T*>(y), codes, scales};
        ckpt_store_kernel<T, vpt.value, v.value, wide.value><<<p.grid, p.block(), p.shared(), st>>>(a);
        AETH_LAUNCH_CHECK();
        return (int)AETH_OK;
    });
}

int aeth_checkpoint_decode(const int8_t* codes, const float* scales, int64_t rows, int64_t d, const void* gain,
                           int gain_dtype, float eps, void* out, int64_t ld_out, int dtype, aeth_stream_t stream) {
    AETH_TRY(ckpt_dims(rows, d, dtype));
    if (gain && !known_dtype(gain_dtype)) return set_err(AETH_ERR_ARG);
    if (rows == 0) return AETH_OK;
    if (!codes || !scales || !out || ld_out < d) return set_err(AETH_ERR_ARG);
    return decode({codes, scales, gain, gain_dtype, rows, (int)d, eps}, out, ld_out, dtype, to_stream(stream));
}

int aeth_rms_norm_checkpoint_backward_workspace(int64_t rows, int64_t d, size_t* bytes) {
    AETH_TRY(ckpt_dims(rows, d, AETH_DTYPE_F32));
    if (!bytes) return set_err(AETH_ERR_ARG);
    const RowPlan p(std::max<int64_t>(rows, 1), d, kBackPerSm);
    Carver c(nullptr);
    c.take<float>(std::max<int64_t>((int64_t)p.grid, num_sms()) * d);
    *bytes = c.used;
    return AETH_OK;
}

int aeth_rms_norm_checkpoint_backward(const void* dy, int64_t ld_dy, const int8_t* codes, const float* scales,
                                      const void* gain, int gain_dtype, const void* d_residual, int64_t ld_residual,
                                      int dtype, int64_t rows, int64_t d, float eps, void* dx, float* d_gain,
                                      void* workspace, size_t workspace_bytes, aeth_stream_t stream) {
    AETH_TRY(ckpt_dims(rows, d, dtype));
    if (!gain || !known_dtype(gain_dtype) || !d_gain) return set_err(AETH_ERR_ARG);
    cudaStream_t st = to_stream(stream);
    if (rows == 0) {
        AETH_CUDA(cudaMemsetAsync(d_gain, 0, sizeof(float) * (size_t)d, st));
        return AETH_OK;
    }
    if (!dy || !codes || !scales || !dx || ld_dy < d || (d_residual && ld_residual < d) || !workspace)
        return set_err(AETH_ERR_ARG);
    const RowPlan p(rows, d, kBackPerSm);
    Carver c(workspace);
    float* part = c.take<float>(std::max<int64_t>((int64_t)p.grid, num_sms()) * d);
    if (workspace_bytes < c.used || !aligned16(workspace)) return set_err(AETH_ERR_ARG);
    const int sz = type_size(dtype);
    const bool vec = d % 8 == 0 && aligned16(gain) && vec_rows(dy, ld_dy, sz) && vec_rows(dx, d, sz) && vec_rows(codes, d, 1) &&
                     (!d_residual || vec_rows(d_residual, ld_residual, sz));
    DeviceRuntime* rt = nullptr;
    AETH_TRY(runtime_for_current(&rt));
    auto gain_sum = [&](int groups) -> int {
        AETH_CUDA(launch_after(ckpt_gain_sum_kernel, dim3((unsigned)((d + 31) / 32)), dim3(1024), 0, st, 1, part, groups,
                               (int)d, d_gain));
        return AETH_OK;
    };
    return by_row(dtype, p, vec, [&](auto* tag, auto vpt, auto v, auto wide) {
        using T = std::remove_pointer_t<decltype(tag)>;
        CkptBack<T> a{{codes, scales, gain, gain_dtype, rows, (int)d, eps}, static_cast<const T*>(dy), ld_dy,
                      static_cast<const T*>(d_residual), ld_residual, static_cast<T*>(dx), part};
        if (vec && ring_fits(rows, d, sz, d_residual != nullptr) && aligned16(codes)) {
            const CkptRing r = ring_plan(d, sz, d_residual != nullptr);
            const int smem = r.groups * r.stages * r.stage_bytes + r.gain_bytes();
            static std::atomic<bool> allowed[kMaxDevices] = {};
            auto kern = ckpt_back_ring_kernel<T, wide.value>;
            AETH_TRY(allow_shared(kern, kRingShared, allowed));
            kern<<<num_sms(), r.groups * r.tx, smem, st>>>(a, r, rt->err_word);
            AETH_LAUNCH_CHECK();
            return gain_sum(num_sms());
        }
        auto kern = ckpt_back_kernel<T, vpt.value, v.value, wide.value>;
        const int smem = p.shared(p.ty);
        static std::atomic<bool> allowed[kMaxDevices] = {};
        AETH_TRY(allow_shared(kern, 64 * 1024, allowed));  // 8192 features: their sums and gain
        kern<<<p.grid, p.block(), smem, st>>>(a);
        AETH_LAUNCH_CHECK();
        return gain_sum((int)p.grid);
    });
}

int aeth_checkpoint_weight_grad_workspace(int64_t rows, int64_t m, int64_t d, size_t* bytes) {
    AETH_TRY(ckpt_dims(rows, d, AETH_DTYPE_F32));
    if (m <= 0 || !bytes) return set_err(AETH_ERR_ARG);
    if (m > kCkptMaxDim) return set_err(AETH_ERR_UNSUPPORTED);
    Carver c(nullptr);
    c.take<uint16_t>(std::max<int64_t>(rows, 1) * up(d, 8));
    c.take<float>(grad_tail(rows, m, d).buffers() * 65536);
    *bytes = c.used;
    return AETH_OK;
}

int aeth_checkpoint_weight_grad(const void* dy, int64_t ld_dy, const int8_t* codes, const float* scales,
                                const void* gain, int gain_dtype, float eps, int dtype, int64_t rows, int64_t m,
                                int64_t d, void* d_weight, int64_t ld_dw, void* workspace, size_t workspace_bytes,
                                aeth_stream_t stream) {
    AETH_TRY(ckpt_dims(rows, d, dtype));
    if (m <= 0 || !d_weight || ld_dw < d || (gain && !known_dtype(gain_dtype))) return set_err(AETH_ERR_ARG);
    if (!is16(dtype) || m > kCkptMaxDim) return set_err(AETH_ERR_UNSUPPORTED);
    if ((m + 255) / 256 * ((d + 255) / 256) > kCkptMaxDim) return set_err(AETH_ERR_UNSUPPORTED);
    cudaStream_t st = to_stream(stream);
    if (rows == 0) {
        AETH_CUDA(cudaMemset2DAsync(d_weight, (size_t)ld_dw * 2, 0, (size_t)d * 2, (size_t)m, st));
        return AETH_OK;
    }
    if (!dy || !codes || !scales || !workspace || ld_dy < m) return set_err(AETH_ERR_ARG);
    if (!aligned16(dy) || ld_dy % 8) return set_err(AETH_ERR_UNSUPPORTED);  // TMA reads dY in place
    Carver c(workspace);
    const int64_t dp = up(d, 8);
    uint16_t* xr = c.take<uint16_t>(rows * dp);
    const GradTail tail = grad_tail(rows, m, d);
    float* buffers = c.take<float>(tail.buffers() * 65536);
    if (workspace_bytes < c.used || !aligned16(workspace)) return set_err(AETH_ERR_ARG);
    AETH_TRY(decode({codes, scales, gain, gain_dtype, rows, (int)d, eps}, xr, dp, dtype, st));
    const PairOperand A{dy, ld_dy, rows, m}, B{xr, dp, rows, d};
    return dtype == AETH_DTYPE_BF16 ? grad_product<true>(A, B, m, d, rows, tail, buffers, d_weight, ld_dw, st)
                                    : grad_product<false>(A, B, m, d, rows, tail, buffers, d_weight, ld_dw, st);
}

}  // extern "C"
