// Log probabilities of given tokens, entropy and the top alternatives of rows
// of logits, each logit read once:
//   M = max l,  z = sum exp(l - M),  u = sum (l - M) exp(l - M)
//   log p(i) = (l_i - M) - log z,   H = log z - u / z
// k_logprob_part: a workgroup takes a slice of a row and keeps a running
//   (M, z, u), rescaled when M grows. M is uniform over a wave (the maximum of
//   each 256-logit chunk that a wave reads is needed anyway), so the rescaling
//   is a uniform branch that is hardly ever taken after the first chunks. For
//   the alternatives it stores the chunk's maximum and nothing else.
// k_logprob_finish: a workgroup a row joins the slices' (M, z, u) in order,
//   and selects the alternatives: any token among the first k of a row lies in
//   one of the k chunks with the largest maxima (equal maxima: the earlier
//   chunk), since each of those holds a token that precedes it. So a threshold
//   over the chunk maxima (bisection over the floats' bits) names about k
//   chunks of 1 KB, which are read again (1 % of a 152 K row for k = 5); their
//   logits that reach the threshold, little more than k, are ranked by counting.
//   Where too many reach it (few chunks, equal logits) the threshold is
//   bisected over the logits themselves, and logits equal to it are taken in
//   order. No input is slower than that path.
// Bound by the one read of the logits.

#include "common.hpp"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / QLM_WAVE;
constexpr int kChunk = 4 * QLM_WAVE;  // logits of a chunk: a vector of four a lane
constexpr int kUnroll = 4;            // chunks a wave keeps in flight
constexpr int kMaxTop = 64;
constexpr int kSlack = 8;             // chunks beyond k that a threshold may name
constexpr int kCand = 512;            // logits that are ranked by counting
constexpr int kMaxVocab = 1 << 21;    // chunk maxima of a row fit 32 KB of LDS
constexpr int kMaxRows = 1 << 23;     // a launch's threads fit 32 bits
constexpr float kFloor = -200.0f;     // exp(kFloor) is 0 in fp32

struct Part {
    float m, z, u;
};

// Both arguments as parts of one whole; the first one's tokens come first.
// An empty part (all logits -inf) has z = 0; a NaN in z or u stays.
__device__ __forceinline__ Part join(Part a, Part b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return Part{m, a.z + b.z, a.u + b.u};
    // a part without tokens contributes 0 (its m - m would be -inf)
    const float da = fmaxf(a.m - m, kFloor), db = fmaxf(b.m - m, kFloor);
    const float ea = expf(da), eb = expf(db);
    return Part{m, a.z * ea + b.z * eb, ea * (a.u + da * a.z) + eb * (b.u + db * b.z)};
}

struct LpArgs {
    const float* logits;
    long long ldl;
    int n, rows, slices, nchunk;
    const int* ids;
    int n_ids;
    float* id_lp;
    float* entropy;
    int top;
    int* top_ids;
    float* top_lp;
    Part* part;      // [rows, slices]
    float* maxima;   // [rows, nchunk]
};

// A lane's four logits of chunk c (-inf past the row's end).
__device__ __forceinline__ f32x4u load_chunk(const float* row, int n, int c) {
    const int i = c * kChunk + 4 * (int)(threadIdx.x & (QLM_WAVE - 1));
    if (i + 4 <= n) return *reinterpret_cast<const f32x4u*>(row + i);
    f32x4u v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < n ? row[i + j] : -INFINITY;
    return v;
}

__global__ __launch_bounds__(kThreads) void k_logprob_part(LpArgs a) {
    const int row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
    const int lane = threadIdx.x & (QLM_WAVE - 1), wave = threadIdx.x / QLM_WAVE;
    const float* lr = a.logits + (size_t)row * a.ldl;
    const int per = (a.nchunk + a.slices - 1) / a.slices;
    const int c0 = slice * per, c1 = min(a.nchunk, c0 + per);
    Part p{-INFINITY, 0.0f, 0.0f};
    for (int c = c0 + wave; c < c1; c += kWaves * kUnroll) {
        f32x4u v[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j)
            v[j] = load_chunk(lr, a.n, min(c + j * kWaves, c1 - 1));
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int cj = c + j * kWaves;
            if (cj >= c1) break;
            const float mx = wave_max(fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
            if (a.maxima && lane == 0) a.maxima[(size_t)row * a.nchunk + cj] = mx;
            if (mx > p.m) {
                const float d = fmaxf(p.m - mx, kFloor), e = expf(d);
                p.u = e * (p.u + d * p.z);
                p.z *= e;
                p.m = mx;
            }
            if (p.m == -INFINITY) {
                // nothing but masked tokens so far, or NaN, which maxima drop
                const float s = (v[j].x + v[j].y) + (v[j].z + v[j].w);
                if (s != s) p.z = NAN;
                continue;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float d = v[j][k] - p.m;
                const float e = __expf(d);  // NaN and +inf - inf stay NaN
                p.z += e;
                p.u = fmaf(fmaxf(d, kFloor), e, p.u);
            }
        }
    }
    p.z = wave_sum(p.z);
    p.u = wave_sum(p.u);
    __shared__ Part parts[kWaves];
    if (lane == 0) parts[wave] = p;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWaves; ++w) p = join(p, parts[w]);
        a.part[(size_t)row * a.slices + slice] = p;
    }
}

// Floats as integers in their order, -0 as +0, NaN as -inf.
constexpr int kLowest = (int)0xff800000 ^ 0x7fffffff;  // order of -inf
constexpr int kPast = 0x7f800001;                      // above the order of +inf
__device__ __forceinline__ int order_of(float v) {
    const int b = __float_as_int(v + 0.0f);
    return v != v ? kLowest : b < 0 ? b ^ 0x7fffffff : b;
}
// Between lo and hi, lo < mid < hi, where hi - lo > 1.
__device__ __forceinline__ int mid_of(int lo, int hi) { return (lo & hi) + ((lo ^ hi) >> 1); }

// Sum of an int over the workgroup, for every thread.
__device__ __forceinline__ int block_count(int v, int* red) {
#pragma unroll
    for (int m = 1; m < QLM_WAVE; m <<= 1) v += __shfl_xor(v, m, QLM_WAVE);
    __syncthreads();
    if ((threadIdx.x & (QLM_WAVE - 1)) == 0) red[threadIdx.x / QLM_WAVE] = v;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) t += red[w];
    return t;
}

struct TopShared {
    int red[kWaves];
    int nsel, ncand;
    int sel[kMaxTop + kSlack];
    int cand_o[kCand];
    int cand_i[kCand];
};

// The first `top` tokens of a row by (logit, then lower id). `mx`: the row's
// chunk maxima in LDS. Called by the whole workgroup. emit(rank, id, logit).
template <typename Emit>
__device__ void select_top(const float* row, int n, int nchunk, int top, const float* mx,
                           TopShared& sh, Emit emit) {
    const int lane = threadIdx.x & (QLM_WAVE - 1), wave = threadIdx.x / QLM_WAVE;
    const unsigned long long below = (1ull << lane) - 1;
    // Every wave finds the same threshold `lo` over the chunk maxima:
    // count(>= lo) >= top, and as near to top as the slack, unless maxima tie.
    int lo = kLowest, spare = 0x7fffffff;  // spare: chunks equal to lo that are taken
    int named = nchunk;
    if (nchunk > top) {
        int hi = kPast, above = 0;  // count(>= hi) = above < top
        while (hi - (long long)lo > 1 && named > top + kSlack) {
            const int m = mid_of(lo, hi);
            int cnt = 0;
            for (int c = lane; c < nchunk + lane; c += QLM_WAVE)
                cnt += (int)__popcll(__ballot(c < nchunk && order_of(mx[min(c, nchunk - 1)]) >= m));
            if (cnt >= top) {
                lo = m;
                named = cnt;
            } else {
                hi = m;
                above = cnt;
            }
        }
        if (named > top + kSlack) spare = top - above;
    }
    // The chunks, in order, into LDS (wave 0).
    const bool listed = nchunk > top;
    if (threadIdx.x == 0) sh.ncand = 0;
    if (listed && wave == 0) {
        int at = 0, left = spare;
        for (int c0 = 0; c0 < nchunk; c0 += QLM_WAVE) {
            const int c = c0 + lane;
            const int o = order_of(mx[min(c, nchunk - 1)]);
            const bool over = c < nchunk && o > lo, same = c < nchunk && o == lo;
            const unsigned long long bs = __ballot(same);
            const bool take = over || (same && (int)__popcll(bs & below) < left);
            const unsigned long long bt = __ballot(take);
            if (take) sh.sel[at + (int)__popcll(bt & below)] = c;
            at += (int)__popcll(bt);
            left -= min(left, (int)__popcll(bs));
        }
        if (lane == 0) sh.nsel = at;
    }
    __syncthreads();
    const int nsel = listed ? sh.nsel : nchunk;
    auto chunk_at = [&](int s) { return listed ? sh.sel[s] : s; };
    auto count_from = [&](int from) {
        int cnt = 0;
        for (int s = wave; s < nsel; s += kWaves) {
            const int c = chunk_at(s);
            const f32x4u v = load_chunk(row, n, c);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                cnt += c * kChunk + 4 * lane + j < n && order_of(v[j]) >= from;
        }
        return block_count(cnt, sh.red);
    };
    int from = lo;
    auto gather = [&]() {
        for (int s = wave; s < nsel; s += kWaves) {
            const int c = chunk_at(s);
            const f32x4u v = load_chunk(row, n, c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = c * kChunk + 4 * lane + j;
                const int o = order_of(v[j]);
                const bool in = i < n && o >= from;
                const unsigned long long b = __ballot(in);
                if (b == 0) continue;
                int base = 0;
                if (lane == 0) base = atomicAdd(&sh.ncand, (int)__popcll(b));
                base = __builtin_amdgcn_readfirstlane(base) + (int)__popcll(b & below);
                if (in && base < kCand) {
                    sh.cand_o[base] = o;
                    sh.cand_i[base] = i;
                }
            }
        }
    };
    gather();
    __syncthreads();
    int nc = sh.ncand;
    bool tied = false;
    if (nc > kCand) {
        // bisect over the logits: count(>= from) >= top, <= kCand
        int a = from, hi = kPast, cnt = nc;
        while (hi - (long long)a > 1 && cnt > kCand) {
            const int m = mid_of(a, hi);
            const int k = count_from(m);
            if (k >= top) {
                a = m;
                cnt = k;
            } else {
                hi = m;
            }
        }
        from = a;
        tied = cnt > kCand;
        __syncthreads();
        if (threadIdx.x == 0) sh.ncand = 0;
        __syncthreads();
        if (!tied) gather();
        __syncthreads();
        nc = sh.ncand;
    }
    if (tied && wave == 0) {
        // fewer than `top` logits lie above `from`; those equal to it follow
        // in order of their ids
        int over = 0, same = 0;
        for (int pass = 0; pass < 2; ++pass) {
            for (int s = 0; s < nsel && (pass == 0 || over + same < top); ++s) {
                const int c = chunk_at(s);
                const f32x4u v = load_chunk(row, n, c);
                int o[4];
                bool in[4];
                int mine = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = c * kChunk + 4 * lane + j;
                    o[j] = order_of(v[j]);
                    in[j] = i < n && (pass == 0 ? o[j] > from : o[j] == from);
                    mine += in[j];
                }
                // exclusive prefix over the lanes: ids ascend with the lane
                int pre = mine;
#pragma unroll
                for (int m = 1; m < QLM_WAVE; m <<= 1) {
                    const int up = __shfl_up(pre, m, QLM_WAVE);
                    if (lane >= m) pre += up;
                }
                const int total = __shfl(pre, QLM_WAVE - 1, QLM_WAVE);
                int at = over + same + pre - mine;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (in[j]) {
                        if (at < kCand) {
                            sh.cand_o[at] = o[j];
                            sh.cand_i[at] = c * kChunk + 4 * lane + j;
                        }
                        ++at;
                    }
                (pass == 0 ? over : same) += total;
            }
        }
        if (lane == 0) sh.ncand = min(over + same, kCand);
    }
    __syncthreads();
    nc = sh.ncand;
    for (int i = threadIdx.x; i < nc; i += kThreads) {
        const int o = sh.cand_o[i], id = sh.cand_i[i];
        int rank = 0;
        for (int j = 0; j < nc; ++j) {
            const int oj = sh.cand_o[j];
            rank += oj > o || (oj == o && sh.cand_i[j] < id);
        }
        if (rank < top) emit(rank, id, row[id]);
    }
}

__global__ __launch_bounds__(kThreads) void k_logprob_finish(LpArgs a) {
    extern __shared__ float mx[];
    __shared__ TopShared sh;
    const int row = blockIdx.x;
    const float* lr = a.logits + (size_t)row * a.ldl;
    if (a.top)
        for (int c = threadIdx.x; c < a.nchunk; c += kThreads)
            mx[c] = a.maxima[(size_t)row * a.nchunk + c];
    // the slices in order, by every thread alike
    Part p = a.part[(size_t)row * a.slices];
    for (int s = 1; s < a.slices; ++s) p = join(p, a.part[(size_t)row * a.slices + s]);
    // no distribution: every logit masked, a NaN, or +inf among them
    if (!(p.z > 0.0f)) p.z = NAN;
    const float lz = logf(p.z);
    if (a.entropy && threadIdx.x == 0) a.entropy[row] = lz - p.u / p.z;
    for (int j = threadIdx.x; j < a.n_ids; j += kThreads) {
        const int id = a.ids[(size_t)row * a.n_ids + j];
        // an id outside the row is not read
        a.id_lp[(size_t)row * a.n_ids + j] = id >= 0 && id < a.n ? (lr[id] - p.m) - lz : NAN;
    }
    if (!a.top) return;
    __syncthreads();
    select_top(lr, a.n, a.nchunk, a.top, mx, sh, [&](int rank, int id, float v) {
        a.top_ids[(size_t)row * a.top + rank] = id;
        a.top_lp[(size_t)row * a.top + rank] = (v - p.m) - lz;
    });
}

int chunks_of(int n) { return (n + kChunk - 1) / kChunk; }

// Workgroups a row: enough in all to fill the GPU, each with work for every
// wave's loads in flight.
int slices_of(int rows, int n) {
    const int most = (chunks_of(n) + kWaves * kUnroll - 1) / (kWaves * kUnroll);
    const int want = (2048 + rows - 1) / rows;
    return want < most ? want : most;
}

size_t round16(size_t b) { return (b + 15) / 16 * 16; }

}  // namespace

extern "C" size_t qlm_token_logprobs_workspace_bytes(int rows, int n, int top) {
    if (rows <= 0 || n <= 0 || n > kMaxVocab || top < 0) return 0;
    return round16((size_t)rows * slices_of(rows, n) * sizeof(Part)) +
           (top ? (size_t)rows * chunks_of(n) * sizeof(float) : 0);
}

extern "C" int qlm_token_logprobs(const float* logits, int ldl, int n, int rows, const int* ids,
                                  int n_ids, float* id_logprobs, float* entropy, int top,
                                  int* top_ids, float* top_logprobs, void* work,
                                  size_t work_bytes, void* stream) {
    if (!logits || !work || rows <= 0 || n <= 0 || ldl < n) return QLM_ERR_ARG;
    if (n_ids < 0 || top < 0 || (n_ids > 0 && (!ids || !id_logprobs))) return QLM_ERR_ARG;
    if (top > 0 && (!top_ids || !top_logprobs || top > n)) return QLM_ERR_ARG;
    if (n_ids == 0 && top == 0 && !entropy) return QLM_ERR_ARG;
    if (n > kMaxVocab || top > kMaxTop || rows > kMaxRows) return QLM_ERR_SHAPE;
    if ((uintptr_t)work & 15u) return QLM_ERR_SHAPE;
    if (work_bytes < qlm_token_logprobs_workspace_bytes(rows, n, top)) return QLM_ERR_ARG;
    LpArgs a{logits, ldl, n, rows, slices_of(rows, n), chunks_of(n), ids, n_ids, id_logprobs,
             entropy, top, top_ids, top_logprobs, reinterpret_cast<Part*>(work), nullptr};
    if (top)
        a.maxima = reinterpret_cast<float*>(
            reinterpret_cast<char*>(work) +
            round16((size_t)rows * a.slices * sizeof(Part)));
    hipStream_t st = as_stream(stream);
    hipLaunchKernelGGL(k_logprob_part, dim3((unsigned)(a.slices * rows)), dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL(k_logprob_finish, dim3(rows), dim3(kThreads),
                       top ? (size_t)a.nchunk * sizeof(float) : 0, st, a);
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_logprobs() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(k_logprob_part));
}
