// The Gated DeltaNet mixer over a tree of drafted tokens (qlm_deltanet_tree) and
// the states' advance along the accepted path (qlm_deltanet_tree_commit).
//
// A node t follows its parent p: S_t = a_t S_p + k_t w_t^T with w_t = b_t (v_t -
// a_t S_p^T k_t), o_t = S_t^T q_t / sqrt(d). No node's state is formed: with g_t
// the product of the a over t's line (itself and all above it),
//   S_t = g_t S + sum over s on t's line of (g_t / g_s) k_s w_s^T,
// S the sequence's state, so that
//   (I + A) W = R,  A_ts = b_t (g_t / g_s) k_t . k_s  for s strictly above t,
//                   R_t  = b_t (v_t - g_t S^T k_t)
//   o_t = (g_t S^T q_t + sum over s on t's line of (g_t / g_s) (q_t . k_s) w_s) / sqrt(d).
// Parents come before their children, so A is strictly lower triangular and W
// follows by substitution; a chain is a tree like any other. The state is read
// once and, in a verification, not written.
//
// A workgroup takes one head of one sequence and 16 NC of its 128 value
// columns. Products run on the fp32 matrix cores. Logarithms of the decays are
// summed in 64 bits along each line: a ratio of two products far below the fp32
// range is as good as any other.
//
// Bound by the phases that wait for each other, of which a workgroup a CU overlaps
// none: 16 trees of up to 64 nodes, 16 heads, take 46 us, a quarter of that the
// state's products; their 36 MB alone would take 8. One tree of 16 nodes 14 us, 16
// accepted paths' commit 16.

#include "paged.hpp"
#include "silu.hpp"

namespace {

constexpr int kD = 128;
constexpr int kThreads = 512, kNW = kThreads / QLM_WAVE;  // two waves a SIMD: LDS holds one workgroup
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct TreeArgs {
    const float* proj;
    const float* conv;  // [B, 3, 3 H d], read, or advanced (commit)
    const float* wt;    // [4, 3 H d]
    const float* A_log;
    const float* dt_bias;
    const float* norm_w;
    float* state;  // read, or advanced (commit)
    float* raw;    // outputs before their head norm [rows, H d]
    float* out;
    const int *path, *accepted;  // commit: the rows to advance along
    long long ldp, ldo;
    int H, ld_path;
    int above;  // a launch takes the sequences of more nodes than this
    qlm_row_batch bt;
};

template <int TM, int NC>
struct TreeShared {
    static constexpr int QS = kD + 4, TS = TM + 4, WS = 16 * NC + 4;  // row strides
    // conv inputs, behind the nodes' the ring's three; then outputs after SiLU
    // (not normalised)
    float q[TM + 3][QS];
    float k[TM + 3][QS];
    float w[TM + 3][WS];  // the same of v, then R, then W
    float at[TM][TS];     // A transposed: at[s][t]
    float m[TM][TS];      // (g_t / g_s) (q_t . k_s) / sqrt(d), s on t's line (tiles up to t's)
    double c[TM];         // log g
    unsigned long long line[TM];
    int tap[TM][4];       // rows of q, k, w that a node's conv reads, oldest first
    float beta[TM], sq[TM], sk[TM];  // b; 1 / |q| and 1 / |k|
    int row[TM];          // proj rows
    int bad;              // >= 0: outputs that did not come out finite
};

// SiLU of a convolution's sum (silu_f's expf and division were half of the
// convolutions' instructions). Below kDeepGate 0, less than 2e-33 off; of -inf, as
// silu_f has it, NaN.
__device__ __forceinline__ float silu_conv(float x) {
    const float y = silu_fast(x);
    return x < kDeepGate ? x * 0.0f : y;
}

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// 32 floats of a row: an operand's elements 32 qd .. + 31 (step s: element 32 qd + s)
__device__ __forceinline__ void load32(float (&d)[32], const float* p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(p + 4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[4 * j + i] = x[i];
    }
}

__device__ __forceinline__ f32x4 dot32(const float (&a)[32], const float (&b)[32]) {
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x;
#pragma unroll
    for (int s = 0; s < 32; s += 2) {
        x = mfma4(a[s], b[s], x);
        y = mfma4(a[s + 1], b[s + 1], y);
    }
    return x + y;
}

// lane n of this lane's 16-lane row
template <int n>
__device__ __forceinline__ float row_lane(float v) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + n, 0xf, 0xf, false));
}

// Forward substitution: lane (r, j) = (l % 16, l / 16) holds rows RP r .. of
// columns NC of its own; step t takes w_t from lane t / RP and leaves
// A_{t', t} w_t out of every later row's rest.
template <int TM, int NC, int T0>
__device__ __forceinline__ void solve_from(const float (&at)[TM][TM + 4],
                                           float (&x)[NC][TM / 16], int nodes) {
    constexpr int RP = TM / 16;
    if constexpr (T0 < 16) {
        if (T0 * RP >= nodes) return;
        const int r = threadIdx.x & 15;
#pragma unroll
        for (int i = 0; i < RP; ++i) {
            float a[RP];
#pragma unroll
            for (int e = 0; e < RP; ++e) a[e] = at[T0 * RP + i][RP * r + e];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float w = row_lane<T0>(x[c][i]);
#pragma unroll
                for (int e = 0; e < RP; ++e) x[c][e] = fmaf(-a[e], w, x[c][e]);
            }
        }
        solve_from<TM, NC, T0 + 1>(at, x, nodes);
    }
}

// A sequence's accepted path: its length, and in lane i its row i. It ends
// where it does not rise to another row of the sequence.
__device__ __forceinline__ int path_of(const TreeArgs& a, int b, const SeqRows& sq, int& p) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const int want = min(max(a.accepted[b], 0), min(a.ld_path, QLM_TREE_MAX));
    p = lane < want ? a.path[(size_t)b * a.ld_path + lane] : -1;
    const int last = __shfl_up(p, 1);
    const unsigned long long ends = __ballot(p < 0 || p >= sq.n || (lane > 0 && p <= last));
    return ends ? __ffsll((long long)ends) - 1 : QLM_WAVE;
}

// Decay's logarithm and b from a row's two gate inputs.
__device__ __forceinline__ void gates(float ga, float gb, float dt_bias, float A_log, double& alpha,
                                      float& beta) {
    const float dt = ga + dt_bias;
    const float sp = dt > 20.0f ? dt : log1pf(expf(dt));
    const float x = -expf(A_log) * sp;
    alpha = x < -1e4f ? -1e4 : (double)x;  // (0 in fp32 long before)
    beta = sigmoid_f(gb);
}

// Head norm and SiLU(z) gate of a row's head, a wave: o0, o1 its elements lane
// and lane + 64 (not normalised). A row outside the tree: 0.
__device__ __forceinline__ void put_head(const TreeArgs& a, int row, int h, bool live, float o0,
                                         float o1, float z0, float z1) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    float* to = a.out + (size_t)row * a.ldo + h * kD + lane;
    const float sn = 1.0f / sqrtf(wave_sum(fmaf(o0, o0, o1 * o1)) / (float)kD + 1e-6f);
    to[0] = live ? (o0 * sn) * a.norm_w[lane] * silu_f(z0) : 0.0f;
    to[64] = live ? (o1 * sn) * a.norm_w[lane + 64] * silu_f(z1) : 0.0f;
}

// A channel of a sequence's ring (cs): the last three of (the ring's three, the
// path's T inputs), put where position ctx_len + accepted expects them.
template <typename F>
__device__ __forceinline__ void advance_ring(const TreeArgs& a, float* cs, int C, int ctx, int T,
                                             int ch, F row_of) {
    float x[3];
#pragma unroll
    for (int j = 0; j < 3; ++j)  // place T + j of that line
        x[j] = T + j >= 3 ? a.proj[(size_t)row_of(T + j - 3) * a.ldp + ch]
                          : cs[(size_t)((ctx % 3 + T + j) % 3) * C];
#pragma unroll
    for (int j = 0; j < 3; ++j) cs[(size_t)((ctx % 3 + T + j) % 3) * C] = x[j];
}

template <int TM, int NC, bool COMMIT>
__global__ __launch_bounds__(kThreads) void k_dn_tree(TreeArgs a) {
    using SH = TreeShared<TM, NC>;
    constexpr int CW = 16 * NC, SPLIT = kD / CW, RT = TM / 16;
    constexpr float kScale = 0.08838834764831845f;  // 1 / sqrt(d)
    __shared__ __align__(16) SH sh;
    const int h = blockIdx.x / SPLIT, c0 = blockIdx.x % SPLIT * CW, b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, qd = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid / QLM_WAVE);
    const int HD = a.H * kD, C = 3 * HD;
    const SeqRows sq = seq_rows(a.bt, b);

    // ---- the nodes: rows, lines, decays (a lane a node, every wave alike) ----
    int T, row = sq.first, parent;
    if constexpr (COMMIT) {
        int p;
        T = path_of(a, b, sq, p);
        row += lane < T ? p : 0;
        parent = lane < T ? lane - 1 : -2;
    } else {
        T = min(sq.n, QLM_TREE_MAX);
        row += lane < T ? lane : 0;
        parent = tree_parent(a.bt, sq, lane);
    }
    T = __builtin_amdgcn_readfirstlane(T);
    if (T <= a.above || T > TM) return;  // nothing to do, or another launch's
    // gate inputs, used when the lines are known (a lane a node)
    const float* gp = a.proj + (size_t)row * a.ldp + 4 * (size_t)HD + h;
    const float gb = gp[0], ga = gp[a.H], gdt = a.dt_bias[h], galog = a.A_log[h];
    // ---- conv inputs: a channel of q or k a thread, every other node ----
    const int qk = tid & 255, hf = wave >> 2;
    const int ch = (qk >> 7) * HD + h * kD + (qk & 127);
    const float* cs = a.conv + (size_t)b * 3 * C;
    float* const col = qk < kD ? &sh.q[0][qk] : &sh.k[0][qk - kD];
    float w4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w4[j] = a.wt[(size_t)j * C + ch];
    col[(TM + hf) * SH::QS] = cs[(size_t)hf * C + ch];
    if (hf == 0) col[(TM + 2) * SH::QS] = cs[(size_t)2 * C + ch];
    // v: a column a thread, nodes VG apart
    constexpr int VG = kThreads / CW, VN = TM > VG ? TM / VG : 1;
    const int vc = tid % CW, vg = tid / CW, vch = 2 * HD + h * kD + c0 + vc;
    const bool v_on = TM >= VG || vg < TM;
    float vw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vw[j] = a.wt[(size_t)j * C + vch];
    if (vg < 3) sh.w[TM + vg][vc] = cs[(size_t)vg * C + vch];
#pragma unroll 1
    for (int i0 = 0; i0 < T; i0 += 16) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = a.proj[(size_t)__builtin_amdgcn_readlane(row, i0 + 2 * i + hf) * a.ldp + ch];
#pragma unroll
        for (int i = 0; i < 8; ++i) col[(i0 + 2 * i + hf) * SH::QS] = x[i];
    }
#pragma unroll
    for (int j = 0; j < VN; ++j) {
        const int i = vg + j * VG;
        const int r = __shfl(row, i & 63);  // (every lane active; past the last node the first row)
        const float x = a.proj[(size_t)r * a.ldp + vch];
        if (v_on) sh.w[i][vc] = i < T ? x : 0.0f;
    }
    // ---- who multiplies what with the state: WC waves over the column tiles, the
    // others over the row tiles, or over keys and queries ----
    constexpr int WC = NC < kNW ? NC : kNW, CPW = NC / WC, WR = kNW / WC;
    constexpr int WT = WR < RT ? WR : RT, TPW = RT / WT;  // waves over row tiles, tiles of one
    const int cw = wave % WC, tw = wave / WC % WT, role = wave / (WC * WT);
    const bool do_k = WR <= RT || role == 0, do_q = !COMMIT && (WR <= RT || role == 1);
    const float* S = a.state + ((size_t)b * a.H + h) * kD * kD + c0;
    float sb[CPW][32];
    if (do_k || do_q) {
#pragma unroll
        for (int c = 0; c < CPW; ++c)
#pragma unroll
            for (int s = 0; s < 32; ++s)
                sb[c][s] = S[(size_t)(32 * qd + s) * kD + 16 * (cw + c * WC) + n];
    }
    // the output gates of the rows that this wave will finish
    constexpr int ZN = NC == 8 && !COMMIT ? TM / kNW : 1;
    float z0[ZN], z1[ZN];
    if constexpr (NC == 8 && !COMMIT) {
#pragma unroll
        for (int k = 0; k < ZN; ++k) {
            const float* z = a.proj +
                             (size_t)__builtin_amdgcn_readlane(row, wave + k * kNW) * a.ldp +
                             3 * (size_t)HD + h * kD + lane;
            z0[k] = z[0];
            z1[k] = z[64];
        }
    }
    for (int i = tid; i < TM * SH::TS; i += kThreads) (&sh.at[0][0])[i] = 0.0f;
    if (tid == 0) sh.bad = -1;
    // a node's inputs: itself and three above; behind the root the ring
    const unsigned long long line = tree_line(parent);
    int up = line ? parent : -1;
    int tap[4] = {0, 0, 0, lane};
    {
        int at = lane, old = 3;
#pragma unroll
        for (int j = 2; j >= 0; --j) {
            const int p = __shfl(up, max(at, 0));
            at = at >= 0 ? p : -1;
            if (at < 0) --old;
            tap[j] = at >= 0 ? at : TM + (sq.ctx % 3 + old) % 3;
        }
    }
    if (wave == 0) {
        double alpha = 0.0;
        float beta = 0.0f;
        if (line && lane < T) gates(ga, gb, gdt, galog, alpha, beta);
        double c = alpha;
        while (__ballot(up >= 0)) {
            const int from = up >= 0 ? up : lane;
            const double x = __shfl(c, from);
            const int next = __shfl(up, from);
            if (up >= 0) {
                c += x;
                up = next;
            }
        }
        if (lane < TM) {
            sh.line[lane] = lane < T ? line : 0;
            sh.c[lane] = c;
            sh.beta[lane] = beta;
            sh.row[lane] = row;
#pragma unroll
            for (int j = 0; j < 4; ++j) sh.tap[lane][j] = tap[j];
        }
    }
    __syncthreads();
    // q, k and v in place: every read before the first write
    {
        float y[TM / 2], yv[VN];
#pragma unroll
        for (int i0 = 0; i0 < TM / 2; i0 += 8) {
            if (2 * i0 < T) {
                float x[8][4];
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[i][j] =
                            col[__builtin_amdgcn_readlane(tap[j], 2 * (i0 + i) + hf) * SH::QS];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float acc = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc = fmaf(x[i][j], w4[j], acc);
                    y[i0 + i] = 2 * (i0 + i) + hf < T ? silu_conv(acc) : 0.0f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i0 + i] = 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < VN; ++j) {
            const int i = min(vg + j * VG, TM - 1);
            const int4 tp = *reinterpret_cast<const int4*>(sh.tap[i]);
            float acc = sh.w[tp.x][vc] * vw[0];
            acc = fmaf(sh.w[tp.y][vc], vw[1], acc);
            acc = fmaf(sh.w[tp.z][vc], vw[2], acc);
            acc = fmaf(sh.w[tp.w][vc], vw[3], acc);
            yv[j] = i < T ? silu_conv(acc) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TM / 2; ++i) col[(2 * i + hf) * SH::QS] = y[i];
#pragma unroll
        for (int j = 0; j < VN; ++j)
            if (v_on) sh.w[vg + j * VG][vc] = yv[j];
    }
    __syncthreads();
    // ---- norms: four threads a node. Vectors are normalised in their products, but
    // those so long that a product of two might leave the range at once (an infinite
    // length leaves 0) ----
    constexpr float kShort = 1e-15f;
    static_assert(kThreads / 4 >= QLM_TREE_MAX, "every node");
    if (const int i = tid / 4; i < TM) {
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int at = 4 * (4 * e + (tid & 3));
            const f32x4 x = *reinterpret_cast<const f32x4*>(&sh.q[i][at]);
            const f32x4 y = *reinterpret_cast<const f32x4*>(&sh.k[i][at]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s0 = fmaf(x[j], x[j], s0);
                s1 = fmaf(y[j], y[j], s1);
            }
        }
        s0 = group_sum<4>(s0);
        s1 = group_sum<4>(s1);
        s0 = 1.0f / sqrtf(s0 + 1e-6f);
        s1 = 1.0f / sqrtf(s1 + 1e-6f);
        if (s0 < kShort || s1 < kShort) {
            auto shorten = [&](float* x, float& by) {
                if (!(by < kShort)) return;
                for (int e = tid & 3; e < kD; e += 4) x[e] *= by;
                by = 1.0f;
            };
            shorten(sh.q[i], s0);
            shorten(sh.k[i], s1);
        }
        if ((tid & 3) == 0) {
            sh.sq[i] = s0;
            sh.sk[i] = s1;
        }
    }
    __syncthreads();
    // ---- products of keys and queries with keys: pairs of 16-node tiles in turn ----
    const int tiles = (T + 15) / 16;
    constexpr int KINDS = COMMIT ? 1 : 2;  // keys, queries
#pragma unroll 1
    for (int job = wave; job < tiles * (tiles + 1) / 2 * KINDS; job += kNW) {
        const int p = job / KINDS, kind = job % KINDS;
        const int ti = p >= 6 ? 3 : p >= 3 ? 2 : p >= 1 ? 1 : 0, si = p - ti * (ti + 1) / 2;
        float ra[32], kb[32];
        load32(kb, &sh.k[16 * si + n][32 * qd]);
        load32(ra, kind ? &sh.q[16 * ti + n][32 * qd] : &sh.k[16 * ti + n][32 * qd]);
        const f32x4 prod = dot32(ra, kb);
        const int s = 16 * si + n;
        const double cs_ = sh.c[s];
        const float ks = sh.sk[s];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 16 * ti + 4 * qd + i;
            const bool on = sh.line[t] >> s & 1ull;
            const float d = on ? expf((float)(sh.c[t] - cs_)) * ks : 0.0f;
            if (kind)
                sh.m[t][s] = on ? sh.sq[t] * kScale * d * prod[i] : 0.0f;
            else
                sh.at[s][t] = on && s != t ? sh.beta[t] * sh.sk[t] * d * prod[i] : 0.0f;
        }
    }
    // ---- products with the state; R in place of v ----
    f32x4 o[TPW][CPW];
#pragma unroll
    for (int k = 0; k < TPW; ++k) {
        const int ti = tw + k * WT;
#pragma unroll
        for (int c = 0; c < CPW; ++c) o[k][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (ti >= tiles) break;
        float ka[32];
        if (do_k) {
            load32(ka, &sh.k[16 * ti + n][32 * qd]);
#pragma unroll
            for (int c = 0; c < CPW; ++c) {
                const f32x4 ks = dot32(ka, sb[c]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 16 * ti + 4 * qd + i;
                    float* r = &sh.w[t][16 * (cw + c * WC) + n];
                    const float g = expf((float)sh.c[t]) * sh.sk[t];
                    *r = sh.line[t] ? sh.beta[t] * (*r - g * ks[i]) : 0.0f;
                }
            }
        }
        if (do_q) {
            load32(ka, &sh.q[16 * ti + n][32 * qd]);
#pragma unroll
            for (int c = 0; c < CPW; ++c) {
                o[k][c] = dot32(ka, sb[c]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 16 * ti + 4 * qd + i;
                    o[k][c][i] *= expf((float)sh.c[t]) * sh.sq[t] * kScale;
                }
            }
        }
    }
    __syncthreads();
    // ---- W by substitution: four columns a wave, or NC / 2 times four ----
    {
        constexpr int RP = TM / 16, NCW = NC * 4 > kNW ? NC * 4 / kNW : 1;
        if (NC * 4 >= kNW || wave < NC * 4) {
            float x[NCW][RP];
#pragma unroll
            for (int c = 0; c < NCW; ++c)
#pragma unroll
                for (int e = 0; e < RP; ++e) x[c][e] = sh.w[RP * n + e][4 * (NCW * wave + c) + qd];
            solve_from<TM, NCW, 0>(sh.at, x, T);
            const double end = sh.c[T - 1];
#pragma unroll
            for (int e = 0; e < RP; ++e) {
                float f = 1.0f;  // commit: what is left of a node at the path's end
                const int t = RP * n + e;
                if constexpr (COMMIT) f = t < T ? expf((float)(end - sh.c[t])) * sh.sk[t] : 0.0f;
#pragma unroll
                for (int c = 0; c < NCW; ++c) sh.w[t][4 * (NCW * wave + c) + qd] = f * x[c][e];
            }
        }
    }
    __syncthreads();
    if constexpr (COMMIT) {
        // S' = g S + sum of k_s w_s^T: 16-row tiles of the state, two a wave
        const float g = expf((float)sh.c[T - 1]);
        float* Sw = a.state + ((size_t)b * a.H + h) * kD * kD + c0;
#pragma unroll 1
        for (int ri = wave; ri < kD / 16; ri += kNW) {
            float kc[TM / 4];
#pragma unroll
            for (int s = 0; s < TM / 4; ++s) kc[s] = sh.k[4 * s + qd][16 * ri + n];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                f32x4 x;
                float* at = Sw + (size_t)(16 * ri + 4 * qd) * kD + 16 * c + n;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = g * at[(size_t)i * kD];
#pragma unroll
                for (int s = 0; s < TM / 4; ++s)
                    x = mfma4(kc[s], sh.w[4 * s + qd][16 * c + n], x);
#pragma unroll
                for (int i = 0; i < 4; ++i) at[(size_t)i * kD] = x[i];
            }
        }
        if constexpr (NC == 8) {  // nobody else reads these channels of the ring
            static_assert(3 * kD <= kThreads, "a thread a channel");
            const int own = (tid / kD) * HD + h * kD + tid % kD;
            if (tid < 3 * kD)
                advance_ring(a, const_cast<float*>(cs) + own, C, sq.ctx, T, own,
                             [&](int i) { return sh.row[i]; });
        }
        return;
    }
    // ---- outputs: the state's part, and what the nodes above have added ----
    if (do_q) {
        bool fine = true;
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
            const int ti = tw + k * WT;
            if (ti >= tiles) break;
#pragma unroll 1
            for (int si = 0; si <= ti; ++si)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int at = 16 * si + 4 * s + qd;
                    const float m = sh.m[16 * ti + n][at];
#pragma unroll
                    for (int c = 0; c < CPW; ++c)
                        o[k][c] = mfma4(m, sh.w[at][16 * (cw + c * WC) + n], o[k][c]);
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 16 * ti + 4 * qd + i;
                const bool live = sh.line[t] != 0;
#pragma unroll
                for (int c = 0; c < CPW; ++c) {
                    if (live) fine &= fabsf(o[k][c][i]) < INFINITY;
                    if (NC < 8 && t < T)
                        a.raw[(size_t)sh.row[t] * HD + h * kD + c0 + 16 * (cw + c * WC) + n] =
                            live ? o[k][c][i] : 0.0f;
                }
            }
        }
        if (!fine) sh.bad = 0;
    }
    __syncthreads();
    // where the whole head is here: its norm and gate, a row a wave, and rows past
    // the tree's last
    auto finish = [&](auto of) {
#pragma unroll
        for (int k = 0; k < ZN; ++k) {
            const int t = wave + k * kNW;
            if (t >= T) break;
            float o0, o1;
            of(t, o0, o1);
            put_head(a, sh.row[t], h, sh.line[t] != 0, o0, o1, z0[k], z1[k]);
        }
        for (int t = QLM_TREE_MAX + wave; t < sq.n; t += kNW)
            put_head(a, sq.first + t, h, false, 0.0f, 0.0f, 0.0f, 0.0f);
    };
    if constexpr (NC == 8) {
        if (sh.bad < 0) {
#pragma unroll
            for (int k = 0; k < TPW; ++k) {
                if (tw + k * WT >= tiles) break;
#pragma unroll
                for (int c = 0; c < CPW; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sh.w[16 * (tw + k * WT) + 4 * qd + i][16 * (cw + c * WC) + n] = o[k][c][i];
            }
            __syncthreads();
            finish([&](int t, float& o0, float& o1) {
                o0 = sh.w[t][lane];
                o1 = sh.w[t][lane + 64];
            });
            return;
        }
    }
    if (sh.bad < 0) return;
    // ---- some output is not finite: every node again, along its own line ----
    // (a node's NaN has reached others through products with 0). Thread (i, j)
    // keeps rows 8 i .. + 7 of columns j, j + 16, ..; the sums over rows meet in
    // sh.m, which nothing reads any more.
    float* red = &sh.m[0][0];  // [16][16]
    const int j = tid & 15, i8 = (tid >> 4) & 15;  // (the second 256 threads do the same again)
#pragma unroll 1
    for (int t = 0; t < T; ++t) {
        const unsigned long long line = sh.line[t];
        if (!line) continue;
#pragma unroll 1
        for (int c = 0; c < NC; ++c) {
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = S[(size_t)(8 * i8 + e) * kD + 16 * c + j];
            double was = 0.0;
            for (unsigned long long left = line; left; left &= left - 1) {
                const int u = __ffsll((long long)left) - 1;
                const float dec = expf((float)(sh.c[u] - was));
                was = sh.c[u];
                float kv = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    s[e] *= dec;
                    kv = fmaf(sh.k[u][8 * i8 + e] * sh.sk[u], s[e], kv);
                }
                __syncthreads();
                red[i8 * 16 + j] = kv;
                __syncthreads();
                float sum = 0.0f;
                for (int e = 0; e < 16; ++e) sum += red[e * 16 + j];
                // v again: its place holds W
                const int vch = 2 * HD + h * kD + c0 + 16 * c + j;
                float acc = 0.0f;
                for (int e = 0; e < 4; ++e) {
                    const int tp = sh.tap[u][e];
                    const float x = tp < TM ? a.proj[(size_t)sh.row[tp] * a.ldp + vch]
                                            : cs[(size_t)(tp - TM) * C + vch];
                    acc = fmaf(x, a.wt[(size_t)e * C + vch], acc);
                }
                const float w = sh.beta[u] * (silu_conv(acc) - sum);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] = fmaf(sh.k[u][8 * i8 + e] * sh.sk[u], w, s[e]);
            }
            float y = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) y = fmaf(sh.q[t][8 * i8 + e], s[e], y);
            __syncthreads();
            red[i8 * 16 + j] = y;
            __syncthreads();
            float sum = 0.0f;
            for (int e = 0; e < 16; ++e) sum += red[e * 16 + j];
            if (i8 == 0)
                a.raw[(size_t)sh.row[t] * HD + h * kD + c0 + 16 * c + j] = sum * sh.sq[t] * kScale;
        }
    }
    if constexpr (NC == 8) {
        __syncthreads();
        finish([&](int t, float& o0, float& o1) {
            const float* r = a.raw + (size_t)sh.row[t] * HD + h * kD + lane;
            o0 = r[0];
            o1 = r[64];
        });
    }
}

// Head norm and gate where a head's columns are several workgroups'.
constexpr int kNormThreads = 256, kNormWaves = kNormThreads / QLM_WAVE;
__global__ __launch_bounds__(kNormThreads) void k_dn_tree_norm(TreeArgs a) {
    const int row = blockIdx.x, lane = threadIdx.x & 63, b = seq_of_row(a.bt, row);
    if (b < 0) return;
    const SeqRows sq = seq_rows(a.bt, b);
    const int i = row - sq.first, HD = a.H * kD;
    if (i < 0 || i >= sq.n) return;
    const unsigned long long mine = tree_line(tree_parent(a.bt, sq, lane));
    const bool live = __ballot(mine != 0) >> min(i, QLM_TREE_MAX - 1) & 1ull && i < QLM_TREE_MAX;
    for (int h = blockIdx.y * kNormWaves + threadIdx.x / QLM_WAVE; h < a.H;
         h += gridDim.y * kNormWaves) {
        const float* o = a.raw + (size_t)row * HD + h * kD + lane;
        const float* z = a.proj + (size_t)row * a.ldp + 3 * (size_t)HD + h * kD + lane;
        put_head(a, row, h, live, live ? o[0] : 0.0f, live ? o[64] : 0.0f, z[0], z[64]);
    }
}

// The rings' advance where a head's columns are several workgroups': after
// k_dn_tree, whose workgroups all read the old ring.
__global__ __launch_bounds__(kThreads) void k_dn_tree_ring(TreeArgs a) {
    const int b = blockIdx.y, C = 3 * a.H * kD;
    const SeqRows sq = seq_rows(a.bt, b);
    int p;
    const int T = path_of(a, b, sq, p);
    if (T == 0) return;
    int row[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) row[j] = sq.first + __shfl(p, max(T + j - 3, 0));
    const int ch = blockIdx.x * kThreads + threadIdx.x;
    if (ch < C)
        advance_ring(a, const_cast<float*>(a.conv) + (size_t)b * 3 * C + ch, C, sq.ctx, T, ch,
                     [&](int i) { return row[i - T + 3]; });
}

template <int TM, int NC, bool COMMIT>
int launch_tree(const TreeArgs& a, hipStream_t st) {
    static_assert(sizeof(TreeShared<TM, NC>) <= 160 * 1024, "fits a CU");
    hipLaunchKernelGGL((k_dn_tree<TM, NC, COMMIT>), dim3(a.H * (kD / (16 * NC)), a.bt.B),
                       dim3(kThreads), 0, st, a);
    return qlm_launch_status();
}

// Column tiles of a workgroup: the fewest that need no more workgroups than CUs,
// since all of a head repeat its convolutions and its nodes' products (16 heads,
// trees of 64, us with 1, 2, 4 and 8: 2 sequences 27, 27, 33, 44; 4 50, 30, 35, 44;
// 8 94, 56, 39, 46; 16 182, 106, 73, 50).
int columns_of(long long heads) {
    return heads > 128 ? 8 : heads > 64 ? 4 : heads > 32 ? 2 : 1;
}

template <int TM, bool COMMIT>
int launch_columns(const TreeArgs& a, hipStream_t st) {
    switch (columns_of((long long)a.H * a.bt.B)) {
        case 8: return launch_tree<TM, 8, COMMIT>(a, st);
        case 4: return launch_tree<TM, 4, COMMIT>(a, st);
        case 2: return launch_tree<TM, 2, COMMIT>(a, st);
        default: return launch_tree<TM, 1, COMMIT>(a, st);
    }
}

// LDS for 64 nodes leaves a CU one workgroup, for 16 it has room for four. No
// sequence has more nodes than the call has rows; where that does not bound
// them and 16 are likely to do (the accepted path of a tree; short trees on
// average), sequences of up to 16 have a launch of their own. What that gives and
// costs (16 heads, us with it and without): 16 trees of 16 18 and 20; of up to 36, 18
// on average, 47 and 33, since the larger ones' workgroups then begin later; of up
// to 64, 27 on average, which the rule leaves in one launch, 59 and 46.
template <bool COMMIT>
int launch_nodes(TreeArgs a, hipStream_t st) {
    if (a.bt.rows <= 16) return launch_columns<16, COMMIT>(a, st);
    if (COMMIT || a.bt.rows <= 20LL * a.bt.B) {
        const int rc = launch_columns<16, COMMIT>(a, st);
        if (rc != QLM_OK) return rc;
        a.above = 16;
    }
    if (a.bt.rows <= 32) return launch_columns<32, COMMIT>(a, st);
    return launch_columns<64, COMMIT>(a, st);
}

int check_tree(const float* proj, int ldp, const qlm_row_batch* batch, int H, int d) {
    const int rc = check_row_batch(batch);
    if (rc != QLM_OK) return rc;
    if (!proj || H <= 0) return QLM_ERR_ARG;
    if (d != kD || H > 4096) return QLM_ERR_SHAPE;
    return ldp < 4 * H * d + 2 * H ? QLM_ERR_SHAPE : QLM_OK;
}

}  // namespace

extern "C" size_t qlm_deltanet_tree_workspace_bytes(int rows, int H, int d) {
    if (rows <= 0 || rows > kMaxBatchRows || H <= 0 || H > 4096 || d != kD) return 0;
    return (size_t)rows * H * d * sizeof(float);
}

extern "C" int qlm_deltanet_tree(const float* proj, int ldp, const qlm_row_batch* batch,
                                 const float* conv_state, const float* conv_w_t,
                                 const float* A_log, const float* dt_bias, const float* norm_w,
                                 const float* state, float* out, int ldo, int H, int d, void* work,
                                 size_t work_bytes, void* stream) {
    const int rc = check_tree(proj, ldp, batch, H, d);
    if (rc != QLM_OK) return rc;
    if (!conv_state || !conv_w_t || !A_log || !dt_bias || !norm_w || !state || !out || !work)
        return QLM_ERR_ARG;
    if (work_bytes < qlm_deltanet_tree_workspace_bytes(batch->rows, H, d)) return QLM_ERR_ARG;
    if (ldo < H * d || ((uintptr_t)work & 15u)) return QLM_ERR_SHAPE;
    if (proj == out) return QLM_ERR_ARG;  // heads read what others would have written
    const TreeArgs a{proj,   conv_state, conv_w_t, A_log, dt_bias, norm_w, const_cast<float*>(state),
                     reinterpret_cast<float*>(work), out, nullptr, nullptr, ldp, ldo, H, 0, 0, *batch};
    hipStream_t st = as_stream(stream);
    const int r = launch_nodes<false>(a, st);
    if (r != QLM_OK || columns_of((long long)H * batch->B) == 8) return r;
    hipLaunchKernelGGL(k_dn_tree_norm, dim3(batch->rows, (H + kNormWaves - 1) / kNormWaves),
                       dim3(kNormThreads), 0, st, a);
    return qlm_launch_status();
}

extern "C" int qlm_deltanet_tree_commit(const float* proj, int ldp, const qlm_row_batch* batch,
                                        const int* path, int ld_path, const int* accepted,
                                        float* conv_state, const float* conv_w_t,
                                        const float* A_log, const float* dt_bias, float* state,
                                        int H, int d, void* stream) {
    const int rc = check_tree(proj, ldp, batch, H, d);
    if (rc != QLM_OK) return rc;
    if (!path || !accepted || !conv_state || !conv_w_t || !A_log || !dt_bias || !state ||
        ld_path <= 0)
        return QLM_ERR_ARG;
    const TreeArgs a{proj,  conv_state, conv_w_t, A_log,    dt_bias, nullptr, state, nullptr,
                     nullptr, path,     accepted, ldp, 0, H, ld_path, 0, *batch};
    hipStream_t st = as_stream(stream);
    const int r = launch_nodes<true>(a, st);
    if (r != QLM_OK || columns_of((long long)H * batch->B) == 8) return r;
    hipLaunchKernelGGL(k_dn_tree_ring, dim3((3 * H * d + kThreads - 1) / kThreads, batch->B),
                       dim3(kThreads), 0, st, a);
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_deltanet_tree() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(k_dn_tree_norm));
}
