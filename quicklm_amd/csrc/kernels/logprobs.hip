// Log probabilities of given tokens, entropy and the top alternatives of rows
// of logits, each logit read once:
//   M = max l,  z = sum exp(l - M),  u = sum (l - M) exp(l - M)
//   log p(i) = (l_i - M) - log z,   H = log z - u / z
// A workgroup takes a slice of a row and keeps a running (M, z, u), rescaled
// when M grows. M is uniform over a wave (the maximum of each 256-logit chunk
// that a wave reads is needed anyway), so the rescaling is a uniform branch
// that is hardly ever taken after the first chunks. For the alternatives it
// keeps the chunk's maximum and nothing else.
// Selection: any token among the first k of a row lies in one of the k chunks
// with the largest maxima (equal maxima: the earlier chunk), since each of
// those holds a token that precedes it. So a threshold over the chunk maxima
// (bisection over the floats' bits, the maxima in registers) names about k
// chunks of 1 KB, which are read again (1 % of a 152 K row for k = 5); their
// logits that reach the threshold, little more than k, are ranked by counting.
// Where too many reach it (few chunks, equal or masked logits) the threshold
// is bisected over the logits held, and logits equal to it are taken in order.
// One workgroup a row does all of it (k_logprob<.., true>) where the rows fill
// the GPU; otherwise slices leave (M, z, u) and their maxima to
// k_logprob_finish. Bound by the one read of the logits.

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
constexpr int kRegMax = 16;           // chunk maxima a lane holds in registers
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
    Part* part;   // [rows, slices], where a row is sliced
    int* maxima;  // [rows, nchunk], orders of the chunks' maxima, likewise
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

// Floats as integers in their order, -0 as +0, NaN as -inf.
constexpr int kLowest = (int)0xff800000 ^ 0x7fffffff;  // order of -inf
constexpr int kPast = 0x7f800001;                      // above the order of +inf
__device__ __forceinline__ int order_of(float v) {
    const int b = __float_as_int(v + 0.0f);
    return v != v ? kLowest : b < 0 ? b ^ 0x7fffffff : b;
}
// Between lo and hi, lo < mid < hi, where hi - lo > 1.
__device__ __forceinline__ int mid_of(int lo, int hi) { return (lo & hi) + ((lo ^ hi) >> 1); }

// The workgroup's share of a row: chunks c0 .. c1 - 1, joined over the waves
// into every thread's result. keep(c, order of chunk c's maximum), by one lane.
template <typename Keep>
__device__ __forceinline__ Part stream_row(const float* lr, int n, int c0, int c1, Part* parts,
                                           bool want_max, Keep keep) {
    const int lane = threadIdx.x & (QLM_WAVE - 1), wave = threadIdx.x / QLM_WAVE;
    Part p{-INFINITY, 0.0f, 0.0f};
    for (int c = c0 + wave; c < c1; c += kWaves * kUnroll) {
        f32x4u v[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j)
            v[j] = load_chunk(lr, n, min(c + j * kWaves, c1 - 1));
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int cj = c + j * kWaves;
            if (cj >= c1) break;
            const float mx = wave_max(fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
            if (want_max && lane == 0) keep(cj, order_of(mx));
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
    if (lane == 0) parts[wave] = p;
    __syncthreads();
    p = parts[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) p = join(p, parts[w]);
    return p;
}

struct TopShared {
    int red[kWaves];
    int nsel, ncand;
    int sel[kMaxTop + kSlack];
    int same[kMaxTop + kSlack];
    int cand_o[kCand];
    int cand_i[kCand];
};

// Sum of an int over the workgroup, for every thread.
__device__ __forceinline__ int block_count(int v, int* red) {
    __syncthreads();
    if ((threadIdx.x & (QLM_WAVE - 1)) == 0) red[threadIdx.x / QLM_WAVE] = v;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) t += red[w];
    return t;
}

// The first `top` tokens of a row by (logit, then lower id). `mx`: the orders
// of the row's chunk maxima in LDS, `most` the largest of them. CPW: chunks a
// wave can hold, kWaves CPW >= top + kSlack. Called by the whole workgroup.
// emit(rank, id, logit).
template <int CPW, typename Emit>
__device__ void select_top(const float* row, int n, int nchunk, int top, const int* mx, int most,
                           TopShared& sh, Emit emit) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    const unsigned long long below = (1ull << lane) - 1;
    const bool listed = nchunk > top;
    // Every wave finds the same threshold `lo` over the chunk maxima:
    // count(>= lo) >= top, and as near to top as the slack, unless maxima tie.
    int lo = kLowest, spare = 0x7fffffff;  // spare: chunks equal to lo that are taken
    if (listed) {
        int hi = most + 1, above = 0, named = nchunk;  // count(>= hi) = above < top
        auto bisect = [&](auto count) {
            while (hi - (long long)lo > 1 && named > top + kSlack) {
                const int m = mid_of(lo, hi);
                const int cnt = count(m);
                if (cnt >= top) {
                    lo = m;
                    named = cnt;
                } else {
                    hi = m;
                    above = cnt;
                }
            }
        };
        if (nchunk <= kRegMax * QLM_WAVE) {
            int o[kRegMax];
#pragma unroll
            for (int j = 0; j < kRegMax; ++j) {
                o[j] = INT32_MIN;
                if (j * QLM_WAVE < nchunk && j * QLM_WAVE + lane < nchunk)
                    o[j] = mx[j * QLM_WAVE + lane];
            }
            bisect([&](int m) {
                int cnt = 0;
#pragma unroll
                for (int j = 0; j < kRegMax; ++j)
                    if (j * QLM_WAVE < nchunk) cnt += (int)__popcll(__ballot(o[j] >= m));
                return cnt;
            });
        } else {
            bisect([&](int m) {
                int cnt = 0;
                for (int c = lane; c < nchunk + lane; c += QLM_WAVE)
                    cnt += (int)__popcll(__ballot(c < nchunk && mx[min(c, nchunk - 1)] >= m));
                return cnt;
            });
        }
        if (named > top + kSlack) spare = top - above;
    }
    // The chunks, in order, into LDS (wave 0).
    if (threadIdx.x == 0) sh.ncand = 0;
    if (listed && wave == 0) {
        int at = 0, left = spare;
        for (int c0 = 0; c0 < nchunk; c0 += QLM_WAVE) {
            const int c = c0 + lane;
            const int o = mx[min(c, nchunk - 1)];
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
    // The chunks' logits, chunk `wave + j kWaves` of the list in v[j], all
    // requested before the first is used; what lies past the row is below all.
    int o[CPW][4], at[CPW];
    {
        f32x4u v[CPW];
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
            const int s = wave + j * kWaves;
            if (s < nsel) {
                const int c = listed ? __builtin_amdgcn_readfirstlane(sh.sel[s]) : s;
                at[j] = c * kChunk + 4 * lane;
                v[j] = load_chunk(row, n, c);
            }
        }
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * kWaves < nsel)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    o[j][k] = at[j] + k < n ? order_of(v[j][k]) : INT32_MIN;
    }
    auto count_from = [&](int from) {
        int cnt = 0;
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * kWaves < nsel)
#pragma unroll
                for (int k = 0; k < 4; ++k) cnt += (int)__popcll(__ballot(o[j][k] >= from));
        return block_count(cnt, sh.red);
    };
    auto gather = [&](int from) {
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * kWaves < nsel)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = o[j][k] >= from;
                    const unsigned long long b = __ballot(in);
                    if (b == 0) continue;
                    int base = 0;
                    if (lane == 0) base = atomicAdd(&sh.ncand, (int)__popcll(b));
                    base = __builtin_amdgcn_readfirstlane(base) + (int)__popcll(b & below);
                    if (in && base < kCand) {
                        sh.cand_o[base] = o[j][k];
                        sh.cand_i[base] = at[j] + k;
                    }
                }
    };
    int from = lo, cnt = count_from(lo);
    bool tied = false;
    if (cnt > kCand) {
        // bisect over the logits: count(>= from) >= top, <= kCand
        int hi = most + 1;
        while (hi - (long long)from > 1 && cnt > kCand) {
            const int m = mid_of(from, hi);
            const int k = count_from(m);
            if (k >= top) {
                from = m;
                cnt = k;
            } else {
                hi = m;
            }
        }
        tied = cnt > kCand;
    }
    gather(tied ? from + 1 : from);  // tied: fewer than `top` lie above
    if (tied) {
        // those equal to it follow in the order of their ids: places by the
        // counts of the chunks before, then of the lanes before
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * kWaves < nsel) {
                int c = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) c += (int)__popcll(__ballot(o[j][k] == from));
                if (lane == 0) sh.same[wave + j * kWaves] = c;
            }
        __syncthreads();
        const int over = sh.ncand;
        __syncthreads();
        int before = 0, s0 = 0;
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * kWaves < nsel) {
                for (; s0 < wave + j * kWaves; ++s0) before += sh.same[s0];
                if (over + before >= top) continue;
                unsigned long long b[4];
                int place = over + before;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    b[k] = __ballot(o[j][k] == from);
                    place += (int)__popcll(b[k] & below);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (o[j][k] == from) {
                        if (place < top) {
                            sh.cand_o[place] = from;
                            sh.cand_i[place] = at[j] + k;
                        }
                        ++place;
                    }
            }
        cnt = top;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < cnt; i += kThreads) {
        const int oi = sh.cand_o[i], id = sh.cand_i[i];
        int rank = 0;
        for (int j = 0; j < cnt; ++j) {
            const int oj = sh.cand_o[j];
            rank += oj > oi || (oj == oi && sh.cand_i[j] < id);
        }
        if (rank < top) emit(rank, id, row[id]);
    }
}

// What is wanted of a row whose (M, z, u) is p; `mx` as select_top's.
template <int CPW>
__device__ __forceinline__ void finish_row(const LpArgs& a, int row, Part p, const int* mx,
                                           TopShared& sh) {
    const float* lr = a.logits + (size_t)row * a.ldl;
    const int most = order_of(p.m);
    // no distribution: every logit masked, a NaN, or +inf among them
    if (!(p.z > 0.0f)) p.z = NAN;
    const float lz = logf(p.z);
    if (a.entropy && threadIdx.x == 0) a.entropy[row] = lz - p.u / p.z;
    for (int j = threadIdx.x; j < a.n_ids; j += kThreads) {
        const int id = a.ids[(size_t)row * a.n_ids + j];
        // an id outside the row is not read
        a.id_lp[(size_t)row * a.n_ids + j] = id >= 0 && id < a.n ? (lr[id] - p.m) - lz : NAN;
    }
    if constexpr (CPW > 0)
        select_top<CPW>(lr, a.n, a.nchunk, a.top, mx, most, sh, [&](int rank, int id, float v) {
            a.top_ids[(size_t)row * a.top + rank] = id;
            a.top_lp[(size_t)row * a.top + rank] = (v - p.m) - lz;
        });
}

// CPW 0: no alternatives. WHOLE: a workgroup a row, finished at once.
template <int CPW, bool WHOLE>
__global__ __launch_bounds__(kThreads) void k_logprob(LpArgs a) {
    extern __shared__ int mx[];
    __shared__ Part parts[kWaves];
    __shared__ TopShared sh;
    const int row = WHOLE ? blockIdx.x : blockIdx.x / a.slices;
    const int slice = WHOLE ? 0 : blockIdx.x - row * a.slices;
    const float* lr = a.logits + (size_t)row * a.ldl;
    const int per = (a.nchunk + a.slices - 1) / a.slices;
    const int c0 = slice * per, c1 = min(a.nchunk, c0 + per);
    int* maxima = a.maxima + (size_t)row * a.nchunk;
    const Part p = stream_row(lr, a.n, c0, c1, parts, CPW > 0, [&](int c, int o) {
        if constexpr (WHOLE)
            mx[c] = o;
        else
            maxima[c] = o;
    });
    if constexpr (WHOLE)
        finish_row<CPW>(a, row, p, mx, sh);
    else if (threadIdx.x == 0)
        a.part[(size_t)row * a.slices + slice] = p;
}

template <int CPW>
__global__ __launch_bounds__(kThreads) void k_logprob_finish(LpArgs a) {
    extern __shared__ int mx[];
    __shared__ TopShared sh;
    const int row = blockIdx.x, lane = threadIdx.x & (QLM_WAVE - 1);
    if (CPW > 0)
        for (int c = threadIdx.x; c < a.nchunk; c += kThreads)
            mx[c] = a.maxima[(size_t)row * a.nchunk + c];
    // the slices joined over the lanes, alike in every wave
    const Part* parts = a.part + (size_t)row * a.slices;
    Part p{-INFINITY, 0.0f, 0.0f};
    for (int s = lane; s < a.slices; s += QLM_WAVE) p = join(p, parts[s]);
#pragma unroll
    for (int m = QLM_WAVE / 2; m >= 1; m >>= 1)
        p = join(p, Part{__shfl_down(p.m, m, QLM_WAVE), __shfl_down(p.z, m, QLM_WAVE),
                         __shfl_down(p.u, m, QLM_WAVE)});
    p.m = __shfl(p.m, 0, QLM_WAVE);
    p.z = __shfl(p.z, 0, QLM_WAVE);
    p.u = __shfl(p.u, 0, QLM_WAVE);
    __syncthreads();
    finish_row<CPW>(a, row, p, mx, sh);
}

// Whether rows are finished by the workgroups that read them. Many
// alternatives take registers that would leave too few of them on a CU.
bool whole(int slices, int top) { return slices == 1 && top + kSlack <= 8 * kWaves; }

template <int CPW>
void launch(const LpArgs& a, hipStream_t st) {
    const size_t lds = CPW > 0 ? (size_t)a.nchunk * sizeof(int) : 0;
    if constexpr (CPW <= 8)
        if (whole(a.slices, a.top)) {
            hipLaunchKernelGGL((k_logprob<CPW, true>), dim3(a.rows), dim3(kThreads), lds, st, a);
            return;
        }
    hipLaunchKernelGGL((k_logprob<CPW, false>), dim3((unsigned)(a.slices * a.rows)),
                       dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL((k_logprob_finish<CPW>), dim3(a.rows), dim3(kThreads), lds, st, a);
}

int chunks_of(int n) { return (n + kChunk - 1) / kChunk; }

// Workgroups a row: enough in all to fill the GPU, each with work for every
// wave's loads in flight.
int slices_of(int rows, int n) {
    const int most = (chunks_of(n) + kWaves * kUnroll - 1) / (kWaves * kUnroll);
    const int want = rows >= 1024 ? 1 : 2048 / rows;
    return want < most ? want : most;
}

size_t round16(size_t b) { return (b + 15) / 16 * 16; }

}  // namespace

extern "C" size_t qlm_token_logprobs_workspace_bytes(int rows, int n, int top) {
    if (rows <= 0 || n <= 0 || n > kMaxVocab || top < 0) return 0;
    const int slices = slices_of(rows, n);
    if (whole(slices, top)) return 16;
    return round16((size_t)rows * slices * sizeof(Part)) +
           (top ? (size_t)rows * chunks_of(n) * sizeof(int) : 0);
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
    LpArgs a{};
    a.logits = logits;
    a.ldl = ldl;
    a.n = n;
    a.rows = rows;
    a.slices = slices_of(rows, n);
    a.nchunk = chunks_of(n);
    a.ids = ids;
    a.n_ids = n_ids;
    a.id_lp = id_logprobs;
    a.entropy = entropy;
    a.top = top;
    a.top_ids = top_ids;
    a.top_lp = top_logprobs;
    a.part = static_cast<Part*>(work);
    a.maxima = reinterpret_cast<int*>(static_cast<char*>(work) +
                                      round16((size_t)rows * a.slices * sizeof(Part)));
    hipStream_t st = as_stream(stream);
    // chunks a wave holds: top + kSlack of them over kWaves
    if (top == 0)
        launch<0>(a, st);
    else if (top + kSlack <= 4 * kWaves)
        launch<4>(a, st);
    else if (top + kSlack <= 8 * kWaves)
        launch<8>(a, st);
    else
        launch<(kMaxTop + kSlack) / kWaves>(a, st);
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_logprobs() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(k_logprob<0, true>));
}
