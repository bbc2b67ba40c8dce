// aeth_rotary.cu -- libaeth_galore: rotary positions of queries and keys, and
// their per-head norms with the rotation in the same pass (section 3c of
// include/aeth_galore.h).
#include <algorithm>

#include "rotary.cuh"
#include "tmap.cuh"

using namespace aeth;

namespace {

constexpr int64_t kRotMaxRows = 1ll << 38;

bool rot_dtype(int dtype) { return dtype == AETH_DTYPE_F32 || dtype == AETH_DTYPE_F16 || dtype == AETH_DTYPE_BF16; }
int rot_size(int dtype) { return dtype == AETH_DTYPE_F32 ? 4 : 2; }
int64_t rot_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

struct RotaryIn {
    const void* data;
    int64_t ld_t, ld_h;
    int heads;
};
struct RotaryCall {  // what every entry point has
    const AethRotaryPlan* plan;
    const void* positions;
    int bits;
    int64_t period;
    RotaryIn q, k;
    int64_t tokens;
    int head_dim, dtype;
    void *q_out, *k_out;
};

int rot_heads(const RotaryIn& h, int64_t tokens, const void* out) {
    if (h.heads == 0 || tokens == 0) return AETH_OK;
    return h.data && out && h.ld_t >= 0 && h.ld_h >= 0 ? AETH_OK : AETH_ERR_ARG;
}
int rot_check(const RotaryCall& c) {
    const AethRotaryPlan* p = c.plan;
    const int hq = c.q.heads, hk = c.k.heads;
    if (!p || c.tokens < 0 || c.head_dim <= 0 || hq < 0 || hk < 0 || (hq == 0 && hk == 0) || !rot_dtype(c.dtype)) return AETH_ERR_ARG;
    if (p->rotary_dim < 2 || p->rotary_dim % 2 || p->rotary_dim > c.head_dim || !p->freq) return AETH_ERR_ARG;
    if ((c.bits != 32 && c.bits != 64) || (c.tokens > 0 && (!c.positions || c.period <= 0))) return AETH_ERR_ARG;
    if (c.head_dim > kRotMaxHead || c.tokens > kRotMaxRows || hq > (1 << 20) || hk > (1 << 20)) return AETH_ERR_UNSUPPORTED;
    if (c.tokens > kRotMaxRows / ((int64_t)hq + hk)) return AETH_ERR_UNSUPPORTED;
    AETH_TRY(rot_heads(c.q, c.tokens, c.q_out));
    return rot_heads(c.k, c.tokens, c.k_out);
}

// Whether every head row can be taken in 16-byte pieces
bool rot_whole(const RotaryIn& h, int64_t tokens, int size) {
    if (h.heads == 0) return true;
    return reinterpret_cast<uintptr_t>(h.data) % 16 == 0 && (tokens == 1 || h.ld_t * size % 16 == 0) &&
           (h.heads == 1 || h.ld_h * size % 16 == 0);
}
bool rot_whole(const RotaryCall& c) {
    const int size = rot_size(c.dtype);
    return rot_whole(c.q, c.tokens, size) && rot_whole(c.k, c.tokens, size) && reinterpret_cast<uintptr_t>(c.q_out) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(c.k_out) % 16 == 0;
}

// Rows of a stretch and CTAs of rotary_any_kernel's and rotary_pairs_kernel's grid.  A stretch is what gives
// every SM six CTAs, 512 rows at most and what the table of its tokens holds;
// `most`: CTAs that q and k may have together (0: one for each stretch).
void rot_grid(RotaryArgs& a, int64_t tokens, int step, int most) {
    const int held = kRotTableBytes / (4 * a.R);  // tokens; 8 at least
    const int64_t all = a.s[0].rows + a.s[1].rows;
    int64_t rows = rot_up((all + 6 * num_sms() - 1) / (6 * num_sms()), step);
    rows = std::min<int64_t>(rows, 512);
    int64_t table = 0;
    for (RotaryRows& s : a.s) {
        if (s.rows == 0) {
            s.stretch = 1;
            s.ctas = 0;
            continue;
        }
        s.stretch = (int)std::min<int64_t>(rows, (int64_t)(held - 2) * s.heads + 1);
        int64_t n = (s.rows + s.stretch - 1) / s.stretch;
        if (most > 0) n = std::min<int64_t>(n, std::max<int64_t>(s.rows * most / all, 1));
        s.ctas = (unsigned)std::min<int64_t>(n, 1 << 30);
        table = std::max<int64_t>(table, std::min<int64_t>((s.stretch + s.heads - 2) / s.heads + 1, tokens) * a.R * 4);
    }
    a.table_bytes = (int)rot_up(table, 16);
}

// CTAs of an SM, and how many waves of them.  A CTA's start (its table, the first
// rows' way) is hidden behind the others' rows where they start apart, and costs
// issue slots: the rotation, which has these to spare, 63, 58, 56 and 60 us in one, two,
// three and four waves of three, the norm 62.7, 62.1, 67 and the gradient (two of an
// SM: 126 registers) 92, 102 and 110 in one, two and three.
template <int OP>
constexpr int rot_per_sm() { return OP == ROT_NORM_BACK ? 2 : 3; }
// Whole waves, whose CTAs have twelve passes (of all their groups) at least where there
// are several: with 18 passes of one wave's CTAs, 8192 x (32 + 8) x 128 bf16, one wave takes
// 32 and 34 us (rotation, norm), 2.3 and 2 waves 33 and 39, 1.15 waves 35 and 41; with
// 9 and 13 passes (4096 and 6000 tokens) one wave 15 and 21, 21 and 27, two of half as
// many 18 and 24, 25 and 33; with 37 (8192 x (64 + 8)) three waves 52, 1.15 waves 58.
constexpr int kRotPasses = 12;
template <int OP>
constexpr int rot_waves() { return OP == ROT_TURN ? 3 : OP == ROT_NORM ? 2 : 1; }
// CTAs of the gradient, each of which leaves sums of the gains', at most: rotary_kernel
// has two an SM, the others four
int rot_back_ctas() { return 4 * num_sms(); }

template <typename T, bool INTER, int OP>
int rot_launch(RotaryArgs& a, int64_t tokens, bool whole, cudaStream_t st) {
    static std::atomic<bool> allowed[4][kMaxDevices] = {};
    if (whole && a.D % 16 == 0 && a.R % 16 == 0 && a.D <= 512) {
        int lanes = 1;
        while (lanes < a.D / 16) lanes *= 2;
        const int groups = kRotThreads / lanes, held = kRotTableBytes / (4 * a.R);
        const int64_t rows = std::max(a.s[0].rows, a.s[1].rows);
        const int64_t passes = (rows + groups - 1) / groups, wave = (int64_t)rot_per_sm<OP>() * num_sms();
        const int64_t waves = std::clamp<int64_t>(passes / (kRotPasses * wave), 1, rot_waves<OP>());
        const unsigned ctas = (unsigned)std::min(passes, waves * wave);
        int64_t most = 0;  // tokens that a CTA's rows have, and one more
        for (RotaryRows& s : a.s) {
            s.ctas = s.rows > 0 ? ctas : 0;
            most = std::max<int64_t>(most, ((s.rows + ctas - 1) / ctas + s.heads - 2) / s.heads + 2);
        }
        const int sums = rot_ring_bytes<T, OP>() + (OP == ROT_TURN ? 0 : a.D * 8) + (int)std::min<int64_t>(most, held) * a.R * 4;
        const int smem = sums + (OP == ROT_NORM_BACK ? groups * a.D * 4 : 0);
        auto kern = rotary_kernel<T, INTER, OP, rot_per_sm<OP>()>;
        AETH_TRY(allow_shared(kern, rot_ring_bytes<T, OP>() + 512 * 8 + kRotTableBytes + 16 * kRotThreads * 4, allowed[0]));
        kern<<<ctas, kRotThreads, smem, st>>>(a, lanes, held, sums / 4);
    } else {
        rot_grid(a, tokens, kRotThreads / 32, OP == ROT_NORM_BACK ? rot_back_ctas() : 0);
        const int smem = a.table_bytes + (OP == ROT_NORM_BACK ? kRotThreads / 32 * a.D * 4 : 0);
        auto kern = rotary_any_kernel<T, INTER, OP>;
        int one = 1;
        if constexpr (OP != ROT_TURN)
            if (a.D <= 256) {
                kern = a.D <= 128 ? rotary_pairs_kernel<T, INTER, OP, 2> : rotary_pairs_kernel<T, INTER, OP, 4>;
                one = a.D <= 128 ? 2 : 3;
            }
        AETH_TRY(allow_shared(kern, 2 * kRotTableBytes, allowed[one]));
        kern<<<a.s[0].ctas + a.s[1].ctas, kRotThreads, smem, st>>>(a);
    }
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

template <int OP>
int rot_typed(RotaryArgs& a, int64_t tokens, int dtype, bool inter, bool whole, cudaStream_t st) {
    if (dtype == AETH_DTYPE_F32)
        return inter ? rot_launch<float, true, OP>(a, tokens, whole, st) : rot_launch<float, false, OP>(a, tokens, whole, st);
    if (dtype == AETH_DTYPE_F16)
        return inter ? rot_launch<__half, true, OP>(a, tokens, whole, st) : rot_launch<__half, false, OP>(a, tokens, whole, st);
    return inter ? rot_launch<__nv_bfloat16, true, OP>(a, tokens, whole, st)
                 : rot_launch<__nv_bfloat16, false, OP>(a, tokens, whole, st);
}

RotaryArgs rot_args(const RotaryCall& c, bool flip) {
    RotaryArgs a = {};
    const RotaryIn* h[2] = {&c.q, &c.k};
    void* out[2] = {c.q_out, c.k_out};
    for (int i = 0; i < 2; ++i) {
        RotaryRows& s = a.s[i];
        s.x = h[i]->data;
        s.ld_t = h[i]->ld_t;
        s.ld_h = h[i]->ld_h;
        s.out = out[i];
        s.heads = std::max(h[i]->heads, 1);
        s.magic = (uint32_t)(((1ull << 32) + s.heads - 1) / s.heads);
        s.rows = c.tokens * h[i]->heads;
    }
    a.pos = c.positions;
    a.pos32 = c.bits == 32;
    a.period = c.period;
    a.freq = c.plan->freq;
    a.amp = c.plan->amplitude;
    a.flip = flip;
    a.D = c.head_dim;
    a.R = c.plan->rotary_dim;
    return a;
}
template <int OP>
int rot_run(RotaryArgs& a, const RotaryCall& c, bool whole, cudaStream_t st) {
    return rot_typed<OP>(a, c.tokens, c.dtype, c.plan->interleaved != 0, whole, st);
}

}  // namespace

extern "C" {

int aeth_rotary(const AethRotaryPlan* plan, const void* positions, int position_bits, int64_t period, const void* q,
                int64_t ld_q_token, int64_t ld_q_head, int q_heads, const void* k, int64_t ld_k_token, int64_t ld_k_head,
                int k_heads, int64_t tokens, int head_dim, int dtype, int inverse, void* q_out, void* k_out,
                aeth_stream_t stream) {
    const RotaryCall c{plan, positions, position_bits, period, {q, ld_q_token, ld_q_head, q_heads},
                       {k, ld_k_token, ld_k_head, k_heads}, tokens, head_dim, dtype, q_out, k_out};
    AETH_TRY(rot_check(c));
    if (tokens == 0) return AETH_OK;
    RotaryArgs a = rot_args(c, inverse != 0);
    return rot_run<ROT_TURN>(a, c, rot_whole(c), to_stream(stream));
}

int aeth_qk_norm_rotary(const AethRotaryPlan* plan, const void* positions, int position_bits, int64_t period, const void* q,
                        int64_t ld_q_token, int64_t ld_q_head, int q_heads, const void* k, int64_t ld_k_token,
                        int64_t ld_k_head, int k_heads, const void* q_gain, const void* k_gain, int gain_dtype, float eps,
                        int64_t tokens, int head_dim, int dtype, void* q_out, void* k_out, aeth_stream_t stream) {
    const RotaryCall c{plan, positions, position_bits, period, {q, ld_q_token, ld_q_head, q_heads},
                       {k, ld_k_token, ld_k_head, k_heads}, tokens, head_dim, dtype, q_out, k_out};
    AETH_TRY(rot_check(c));
    if (!rot_dtype(gain_dtype) || (q_heads && !q_gain) || (k_heads && !k_gain)) return set_err(AETH_ERR_ARG);
    if (tokens == 0) return AETH_OK;
    RotaryArgs a = rot_args(c, false);
    a.s[0].gain = q_gain;
    a.s[1].gain = k_gain;
    a.gain_dtype = gain_dtype;
    a.eps = eps;
    return rot_run<ROT_NORM>(a, c, rot_whole(c), to_stream(stream));
}

int aeth_qk_norm_rotary_backward_workspace(int head_dim, size_t* bytes) {
    if (head_dim <= 0 || !bytes) return set_err(AETH_ERR_ARG);
    if (head_dim > kRotMaxHead) return set_err(AETH_ERR_UNSUPPORTED);
    *bytes = (size_t)(rot_back_ctas() + 1) * 2 * (size_t)head_dim * sizeof(float);
    return AETH_OK;
}

int aeth_qk_norm_rotary_backward(const AethRotaryPlan* plan, const void* positions, int position_bits, int64_t period,
                                 const void* dq, int64_t ld_dq_token, int64_t ld_dq_head, const void* dk,
                                 int64_t ld_dk_token, int64_t ld_dk_head, const void* q, int64_t ld_q_token,
                                 int64_t ld_q_head, int q_heads, const void* k, int64_t ld_k_token, int64_t ld_k_head,
                                 int k_heads, const void* q_gain, const void* k_gain, int gain_dtype, float eps,
                                 int64_t tokens, int head_dim, int dtype, void* dq_out, void* dk_out, float* d_q_gain,
                                 float* d_k_gain, void* workspace, size_t workspace_bytes, aeth_stream_t stream) {
    const RotaryCall c{plan, positions, position_bits, period, {q, ld_q_token, ld_q_head, q_heads},
                       {k, ld_k_token, ld_k_head, k_heads}, tokens, head_dim, dtype, dq_out, dk_out};
    AETH_TRY(rot_check(c));
    const RotaryIn dy[2] = {{dq, ld_dq_token, ld_dq_head, q_heads}, {dk, ld_dk_token, ld_dk_head, k_heads}};
    AETH_TRY(rot_heads(dy[0], tokens, dq_out));
    AETH_TRY(rot_heads(dy[1], tokens, dk_out));
    if (!rot_dtype(gain_dtype) || (q_heads && (!q_gain || !d_q_gain)) || (k_heads && (!k_gain || !d_k_gain)))
        return set_err(AETH_ERR_ARG);
    cudaStream_t st = to_stream(stream);
    if (tokens == 0) {
        if (q_heads) AETH_CUDA(cudaMemsetAsync(d_q_gain, 0, sizeof(float) * (size_t)head_dim, st));
        if (k_heads) AETH_CUDA(cudaMemsetAsync(d_k_gain, 0, sizeof(float) * (size_t)head_dim, st));
        return AETH_OK;
    }
    size_t need = 0;
    AETH_TRY(aeth_qk_norm_rotary_backward_workspace(head_dim, &need));
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16) return set_err(AETH_ERR_ARG);
    RotaryArgs a = rot_args(c, true);
    for (int i = 0; i < 2; ++i) {
        a.s[i].dy = dy[i].data;
        a.s[i].ld_dt = dy[i].ld_t;
        a.s[i].ld_dh = dy[i].ld_h;
        a.s[i].part = static_cast<float*>(workspace) + (int64_t)i * (rot_back_ctas() + 1) * head_dim;
    }
    a.s[0].gain = q_gain;
    a.s[1].gain = k_gain;
    a.gain_dtype = gain_dtype;
    a.eps = eps;
    const int size = rot_size(dtype);
    AETH_TRY(rot_run<ROT_NORM_BACK>(a, c, rot_whole(c) && rot_whole(dy[0], tokens, size) && rot_whole(dy[1], tokens, size), st));
    RotaryGain g{{a.s[0].part, a.s[1].part}, {d_q_gain, d_k_gain}, {(int)a.s[0].ctas, (int)a.s[1].ctas}, head_dim};
    if (!q_heads) {  // k's alone
        g.part[0] = g.part[1];
        g.out[0] = g.out[1];
        g.groups[0] = g.groups[1];
    }
    AETH_CUDA(launch_after(rotary_gain_kernel, dim3((unsigned)(head_dim + 31) / 32, q_heads && k_heads ? 2 : 1), dim3(1024), 0, st,
                           1, g));
    return AETH_OK;
}

}  // extern "C"
