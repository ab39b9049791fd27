// New rows into a paged KV cache (qlm_paged_append) and the end of a greedy
// verification of drafted trees (qlm_tree_commit).
//
// Append, a head of a row:  r = x / sqrt(mean(x^2) + eps) * (1 + gain), then
// for each pair (j, j + rot / 2) of its first rot elements
//   (r_j, r_j+h) -> (r_j cos - r_j+h sin, r_j+h cos + r_j sin)
// with the angle of the row's position on the pair's axis. Queries go to their
// own array, keys and values (as they are) to the row's slot. Every value is
// read once and written once.

#include "paged.hpp"

namespace {

// vectors of four aligned to one element only: rows of any stride
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kAppendThreads = 256;
constexpr int kScalarAxes = 4;  // axes whose positions are read ahead

struct AppendArgs {
    const float* qkv;
    const float *qn, *kn;  // gains, NULL: that head is not normalised
    const float *cos_tab, *sin_tab;
    const int *positions, *pair_axis;
    float* q_out;
    long long ldqkv, ldq, ld_pos;
    int n_pos, rot, n_axes, n_q, q_stride;
    qlm_row_batch bt;
    qlm_kv_pages pg;
};

// Groups of HD / 4 lanes take K heads each of the row blockIdx.x, four elements a
// lane: query heads first, then keys, then values. Few rows: K = 1, a workgroup
// for each few heads. Many: K = 3, all requested before the row's sequence is
// looked up, which three heads then share (16 + 2 x 4 heads of 128 into a bf16
// cache, one axis, K = 1 and 3: 340 rows 5.2 and 6.1 us, 600 7.2 and 7.0, 2048 15.8
// and 12.2, 46 MB at 3.7 TB/s; positions of three axes 12.8).
template <int HD, typename KV, int K>
__global__ __launch_bounds__(kAppendThreads) void k_paged_append(AppendArgs a) {
    constexpr int LPH = HD / 4, HPB = kAppendThreads / LPH;  // lanes a head, heads at once
    __shared__ __align__(16) float sh[HPB][HD];
    const int grp = threadIdx.x / LPH, l = threadIdx.x % LPH, e0 = 4 * l;
    const int row = blockIdx.x, n_kv = a.pg.n_kv, heads = a.n_q + 2 * n_kv;
    const float* xr = a.qkv + (size_t)row * a.ldqkv;
    // vector loads come back in order: what leads to the angles is asked for ahead of
    // the row, or through the scalar cache
    const int half = a.rot / 2;
    const int start0 = a.bt.row_start[min((int)(threadIdx.x & (QLM_WAVE - 1)), a.bt.B)];
    // (and none of them under a branch, behind which the compiler waits for all that
    // the shortest way there has asked for: something else is read instead)
    const bool has_axis = a.positions && a.pair_axis && half > 0;
    const int* const axes = has_axis ? a.pair_axis : a.bt.row_start;
    int pair[4], axis[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = max(min(e0 + j, a.rot - 1), 0);
        pair[j] = e < half ? e : e - half;
        axis[j] = axes[has_axis ? pair[j] : 0];
    }
    __builtin_amdgcn_sched_barrier(0);
    f32x4u v[K], gn[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        // groups past the last head do its work, unstored
        const int hc = min((int)(blockIdx.y * K + k) * HPB + grp, heads - 1);
        const size_t at = hc < a.n_q ? (size_t)hc * a.q_stride
                                     : (size_t)a.n_q * a.q_stride + (size_t)(hc - a.n_q) * HD;
        v[k] = __builtin_nontemporal_load(reinterpret_cast<const f32x4u*>(xr + at + e0));
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int hc = min((int)(blockIdx.y * K + k) * HPB + grp, heads - 1);
        const float* gain = hc < a.n_q ? a.qn : a.kn;
        gn[k] = *reinterpret_cast<const f32x4u*>((gain ? gain : xr) + e0);
    }
    __builtin_amdgcn_sched_barrier(0);
    int at_axis[kScalarAxes];
    if (a.positions) {
#pragma unroll
        for (int x = 0; x < kScalarAxes; ++x)
            at_axis[x] = uniform_load(a.positions, (size_t)min(x, a.n_axes - 1) * a.ld_pos + row);
    }
    const int b = __builtin_amdgcn_readfirstlane(seq_of_row(a.bt, row, start0));
    if (b < 0) return;  // the whole workgroup
    const int first = min(max(uniform_load(a.bt.row_start, b), 0), a.bt.rows);
    const int end = min(max(uniform_load(a.bt.row_start, b + 1), 0), a.bt.rows);
    const int ctx = min(max(uniform_load(a.bt.ctx_len, b), 0), 1 << 30);
    const SeqRows sq{first, max(end - first, 0), ctx};
    const int i = row - sq.first;
    if (i < 0 || i >= sq.n) return;
    const int slot_page = page_of(a.pg, b, sq.ctx + i);
    bool live = true;
    int depth = i;
    if (a.bt.parent) {
        const unsigned long long line = tree_line(tree_parent(a.bt, sq, threadIdx.x & 63));
        const int at = min(i, QLM_TREE_MAX - 1);
        const unsigned long long mine = (unsigned long long)__shfl((unsigned)(line >> 32), at) << 32 |
                                        __shfl((unsigned)line, at);
        live = i < QLM_TREE_MAX && mine != 0;
        depth = __popcll(mine) - 1;
    }
    // the angles of this lane's elements, the same for every head
    float c4[4], s4[4];
    if (half > 0) {
        int pos[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) pos[j] = sq.ctx + depth;
        if (a.positions) {
            bool there[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                axis[j] = has_axis ? axis[j] : 0;
                there[j] = axis[j] >= 0 && axis[j] < a.n_axes;
                pos[j] = at_axis[0];
#pragma unroll
                for (int x = 1; x < kScalarAxes; ++x) pos[j] = axis[j] == x ? at_axis[x] : pos[j];
            }
            if (a.n_axes > kScalarAxes) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    pos[j] = a.positions[(size_t)(there[j] ? axis[j] : 0) * a.ld_pos + row];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) pos[j] = there[j] ? pos[j] : -1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const size_t at = (size_t)min(max(pos[j], 0), a.n_pos - 1) * half + pair[j];
            c4[j] = a.cos_tab[at];
            s4[j] = a.sin_tab[at];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (pos[j] < 0 || pos[j] >= a.n_pos) c4[j] = s4[j] = NAN;  // no angle
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int head = (int)(blockIdx.y * K + k) * HPB + grp, hc = min(head, heads - 1);
        const bool is_q = hc < a.n_q, is_v = hc >= a.n_q + n_kv;
        f32x4u x = v[k];
        float ss = fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(x.z, x.z, x.w * x.w)));
        ss = group_sum<LPH>(ss);
        if (is_q ? a.qn != nullptr : !is_v && a.kn) {
            const float s = 1.0f / sqrtf(ss / (float)HD + 1e-6f);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = (x[j] * s) * (1.0f + gn[k][j]);
        }
        if (half > 0) {
            // a pair's other element is some lane's of the same group, so of the
            // same wave
            *reinterpret_cast<f32x4u*>(&sh[grp][e0]) = x;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (!is_v && e0 < a.rot) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = e0 + j;
                    if (e >= a.rot) break;
                    const bool low = e < half;
                    const float y = sh[grp][low ? e + half : e - half];
                    x[j] = low ? nc_mul_sub(x[j], c4[j], y, s4[j])
                               : nc_mul_add2(x[j], c4[j], y, s4[j]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        if (head >= heads) continue;
        if (is_q) {
            if (!live) x = f32x4u{0.0f, 0.0f, 0.0f, 0.0f};
            *reinterpret_cast<f32x4u*>(a.q_out + (size_t)row * a.ldq + (size_t)head * HD + e0) = x;
            continue;
        }
        if (!live || slot_page < 0) continue;
        const int g = is_v ? hc - a.n_q - n_kv : hc - a.n_q;
        KV* to = reinterpret_cast<KV*>(is_v ? a.pg.v : a.pg.k) +
                 slot_at(a.pg, slot_page, g, sq.ctx + i) + e0;
        if constexpr (sizeof(KV) == 4) {
            *reinterpret_cast<float4*>(to) = make_float4(x.x, x.y, x.z, x.w);
        } else {
            unsigned w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = (unsigned)__builtin_bit_cast(unsigned short, (__bf16)x[j]);
            *reinterpret_cast<uint2*>(to) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
        }
    }
}

// ---- commit ------------------------------------------------------------------
// The walk: from row 0 to the first row that follows the last accepted one and
// holds its pick, a row a lane, one ballot a step. Every workgroup of a sequence
// walks for itself (a handful of steps) and so needs no other launch.
// The move: row path[i] -> slot ctx + i. Rows of a path are in rising order and
// path[i] >= i, so that a place is only written once the row it held has been
// read, if one thread moves its 16 bytes of every row of the path in order. Bound
// by the walk's dependent reads: 64 trees of up to 64 rows, 9 layers of 4 heads of
// 128 in bf16, take 5 us, one tree of 16 takes 4.
constexpr int kCommitThreads = 256;
constexpr int kMoveBatch = 8;  // rows in flight a thread

struct CommitArgs {
    const int *tokens, *picks;
    int *path, *accepted, *next, *new_len;
    int ld_path, layers, pieces;  // pieces: 16 bytes each, of a slot of a head
    long long layer_bytes;
    qlm_row_batch bt;
    qlm_kv_pages pg;
};

__global__ __launch_bounds__(kCommitThreads) void k_tree_commit(CommitArgs a) {
    __shared__ long long from[QLM_TREE_MAX], to[QLM_TREE_MAX];  // bytes, -1: not there
    __shared__ int moves;
    const int b = blockIdx.y, lane = threadIdx.x & (QLM_WAVE - 1);
    if (threadIdx.x < QLM_WAVE) {
        const SeqRows sq = seq_rows(a.bt, b);
        const bool there = lane < sq.n;
        const int parent = tree_parent(a.bt, sq, lane);
        const int token = there ? a.tokens[sq.first + lane] : 0;
        const int pick = there ? a.picks[sq.first + lane] : 0;
        int mine = -1, count = 0, next = -1;
        int cur = __ballot(parent == -1) & 1ull ? 0 : -1;
        while (cur >= 0) {
            if (lane == count) mine = cur;
            ++count;
            next = __shfl(pick, cur);
            const unsigned long long c = __ballot(parent == cur && lane > cur && token == next);
            cur = c ? __ffsll((long long)c) - 1 : -1;
        }
        if (blockIdx.x == 0) {
            int* path = a.path + (size_t)b * a.ld_path;
            for (int i = lane; i < a.ld_path; i += QLM_WAVE) path[i] = i < QLM_WAVE ? mine : -1;
            if (lane == 0) {
                a.accepted[b] = count;
                a.next[b] = next;
                if (a.new_len) a.new_len[b] = sq.ctx + count;
            }
        }
        // the rows that move, of those whose slots are there
        const bool move = lane < count && mine != lane;
        const int fp = move ? page_of(a.pg, b, sq.ctx + mine) : -1;
        const int tp = move ? page_of(a.pg, b, sq.ctx + lane) : -1;
        const bool both = fp >= 0 && tp >= 0;
        const unsigned long long who = __ballot(both);
        if (both) {
            const int at = __popcll(who & ((1ull << lane) - 1ull));
            const long long size = a.pg.dtype == 0 ? 4 : 2;
            from[at] = (long long)slot_at(a.pg, fp, 0, sq.ctx + mine) * size;
            to[at] = (long long)slot_at(a.pg, tp, 0, sq.ctx + lane) * size;
        }
        if (lane == 0) moves = __popcll(who);
    }
    __syncthreads();
    const int n = moves;
    // this thread's piece: of a layer, a pool and a head
    long long p = (long long)blockIdx.x * kCommitThreads + threadIdx.x;
    const int piece = (int)(p % a.pieces);
    p /= a.pieces;
    const int g = (int)(p % a.pg.n_kv);
    p /= a.pg.n_kv;
    if (n == 0 || p >= 2LL * a.layers) return;
    char* pool = reinterpret_cast<char*>(p & 1 ? a.pg.v : a.pg.k) + (p >> 1) * a.layer_bytes +
                 (size_t)g * a.pg.page_size * a.pieces * 16 + piece * 16;
    for (int i0 = 0; i0 < n; i0 += kMoveBatch) {
        u32x4 v[kMoveBatch];
#pragma unroll
        for (int i = 0; i < kMoveBatch; ++i)
            v[i] = *reinterpret_cast<const u32x4*>(pool + from[min(i0 + i, n - 1)]);
#pragma unroll
        for (int i = 0; i < kMoveBatch; ++i)
            if (i0 + i < n) *reinterpret_cast<u32x4*>(pool + to[i0 + i]) = v[i];
    }
}

template <int HD, typename KV>
void launch_append(const AppendArgs& a, hipStream_t st) {
    const int per = kAppendThreads / (HD / 4), heads = a.n_q + 2 * a.pg.n_kv;
    const int rounds = (heads + per - 1) / per;
    if ((long long)a.bt.rows * rounds <= 1024)
        hipLaunchKernelGGL((k_paged_append<HD, KV, 1>), dim3(a.bt.rows, rounds),
                           dim3(kAppendThreads), 0, st, a);
    else
        hipLaunchKernelGGL((k_paged_append<HD, KV, 3>), dim3(a.bt.rows, (rounds + 2) / 3),
                           dim3(kAppendThreads), 0, st, a);
}

}  // namespace

extern "C" int qlm_paged_append(const float* qkv, int ldqkv, const float* q_norm,
                                const float* k_norm, const float* cos_tab, const float* sin_tab,
                                int n_pos, int rot_dim, const int* positions, int ld_pos,
                                const int* pair_axis, int n_axes, const qlm_row_batch* batch,
                                const qlm_kv_pages* pages, float* q_out, int ldq, int n_q,
                                int gated, void* stream) {
    int rc = check_row_batch(batch);
    if (rc == QLM_OK) rc = check_kv_pages(pages);
    if (rc != QLM_OK) return rc;
    if (!qkv || !q_out || qkv == q_out || n_q <= 0) return QLM_ERR_ARG;
    if (rot_dim > 0 && (!cos_tab || !sin_tab || n_pos <= 0)) return QLM_ERR_ARG;
    if (positions && (ld_pos < batch->rows || n_axes <= 0)) return QLM_ERR_ARG;
    const int hd = pages->hd;
    if (rot_dim < 0 || rot_dim > hd || rot_dim % 2 != 0) return QLM_ERR_SHAPE;
    if (n_q > 8192) return QLM_ERR_SHAPE;
    const int q_stride = gated ? 2 * hd : hd;
    if (ldqkv < n_q * q_stride + 2 * pages->n_kv * hd || ldq < n_q * hd) return QLM_ERR_SHAPE;
    const AppendArgs a{qkv, q_norm, k_norm, cos_tab, sin_tab, positions, pair_axis, q_out, ldqkv,
                       ldq, ld_pos, n_pos, rot_dim, n_axes, n_q, q_stride, *batch, *pages};
    hipStream_t st = as_stream(stream);
    if (hd == 128)
        pages->dtype == 0 ? launch_append<128, float>(a, st) : launch_append<128, uint16_t>(a, st);
    else
        pages->dtype == 0 ? launch_append<256, float>(a, st) : launch_append<256, uint16_t>(a, st);
    return qlm_launch_status();
}

extern "C" int qlm_tree_commit(const int* tokens, const int* picks, const qlm_row_batch* batch,
                               const qlm_kv_pages* pages, int layers, long long layer_stride,
                               int* path, int ld_path, int* accepted, int* next_token,
                               int* new_len, void* stream) {
    int rc = check_row_batch(batch);
    if (rc == QLM_OK) rc = check_kv_pages(pages);
    if (rc != QLM_OK) return rc;
    if (!tokens || !picks || !path || !accepted || !next_token || !batch->parent || layers <= 0)
        return QLM_ERR_ARG;
    if (new_len == batch->ctx_len || ld_path < QLM_TREE_MAX) return QLM_ERR_ARG;
    const long long pool = (long long)pages->n_pages * pages->n_kv * pages->page_size * pages->hd;
    if (layer_stride < 0 || (layers > 1 && layer_stride < pool)) return QLM_ERR_ARG;
    const long long size = pages->dtype == 0 ? 4 : 2;
    if (layers > 4096 || layer_stride > 1LL << 48) return QLM_ERR_SHAPE;
    if (layers > 1 && layer_stride * size % 16 != 0) return QLM_ERR_SHAPE;
    const int pieces = (int)(pages->hd * size / 16);
    const CommitArgs a{tokens, picks, path, accepted, next_token, new_len, ld_path, layers, pieces,
                       layer_stride * size, *batch, *pages};
    const long long threads = 2LL * layers * pages->n_kv * pieces;
    hipLaunchKernelGGL(k_tree_commit,
                       dim3((unsigned)((threads + kCommitThreads - 1) / kCommitThreads), batch->B),
                       dim3(kCommitThreads), 0, as_stream(stream), a);
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_paged() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(k_tree_commit));
}
