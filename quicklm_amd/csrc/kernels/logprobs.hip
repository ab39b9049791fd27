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

#include <type_traits>

#include "common.hpp"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 256;   // of a workgroup that reads a row or a slice
constexpr int kWaves = kThreads / QLM_WAVE;
constexpr int kFinishWaves = 8;  // of a workgroup that finishes a sliced row
constexpr int kMostWaves = 16;   // of a workgroup that reads one of few short rows
constexpr int kChunk = 4 * QLM_WAVE;  // logits of a chunk: a vector of four a lane
// Chunks a wave keeps in flight: many where one workgroup reads a long row
// (2047 x 151936 211 us with 8, 221 with 4), few where slices are many.
constexpr int kLongUnroll = 8, kShortUnroll = 4, kSliceUnroll = 2;
constexpr int kMaxTop = QLM_TOKEN_LOGPROBS_MAX_TOP;
constexpr int kSlack = 8;             // chunks beyond k that a threshold may name
constexpr int kCand = 512;            // logits that are ranked by counting
constexpr int kMaxVocab = 1 << 21;    // chunk maxima of a row fit 32 KB of LDS
constexpr int kMaxRows = 1 << 22;     // a launch's threads fit 32 bits
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

// A lane's four logits of chunk c (-inf past the row's end). c is uniform: a
// branch by lane would wait for the load inside it. STREAM: not kept in the
// caches, which read 2047 rows of 151936 in 213 us instead of 235.
template <bool STREAM = false>
__device__ __forceinline__ f32x4u load_chunk(const float* row, int n, int c) {
    const int i = c * kChunk + 4 * (int)(threadIdx.x & (QLM_WAVE - 1));
    if ((c + 1) * kChunk <= n) {
        const f32x4u* p = reinterpret_cast<const f32x4u*>(row + i);
        return STREAM ? __builtin_nontemporal_load(p) : *p;
    }
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
__device__ __forceinline__ float value_of(int o) {
    return __int_as_float(o < 0 ? o ^ 0x7fffffff : o);
}
// A place to cut the orders lo .. hi, lo < cut < hi, where hi - lo > 1: the
// middle of the values and the middle of the orders in turn. Values are cut in
// a few steps where they lie near each other; the orders end any other case.
__device__ __forceinline__ int cut_of(int lo, int hi, int step) {
    const int mid = (lo & hi) + ((lo ^ hi) >> 1);
    if (step & 1) return mid;
    const float v = 0.5f * value_of(lo) + 0.5f * value_of(hi);
    const int o = order_of(v);
    return v == v && o > lo && o < hi ? o : mid;
}

// The workgroup's share of a row: chunks c0 .. c1 - 1, a part each of the NW
// waves. keep(c, order of chunk c's maximum), by one lane.
template <int NW, int U, typename Keep>
__device__ __forceinline__ void stream_row(const float* lr, int n, int c0, int c1, Part* parts,
                                           bool want_max, Keep keep) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    Part p{-INFINITY, 0.0f, 0.0f};
    for (int c = c0 + wave; c < c1; c += NW * U) {
        f32x4u v[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (c + j * NW < c1) v[j] = load_chunk<true>(lr, n, c + j * NW);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int cj = c + j * NW;
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
}

// `count` parts joined over the lanes of a wave, in one order; for every lane.
__device__ __forceinline__ Part join_parts(const Part* parts, int count) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    Part p{-INFINITY, 0.0f, 0.0f};
    for (int s = lane; s < count; s += QLM_WAVE) p = s < QLM_WAVE ? parts[s] : join(p, parts[s]);
    for (int m = QLM_WAVE / 2; m >= 1; m >>= 1)
        if (m < count)
            p = join(p, Part{__shfl_down(p.m, m, QLM_WAVE), __shfl_down(p.z, m, QLM_WAVE),
                             __shfl_down(p.u, m, QLM_WAVE)});
    return Part{__shfl(p.m, 0, QLM_WAVE), __shfl(p.z, 0, QLM_WAVE), __shfl(p.u, 0, QLM_WAVE)};
}

struct TopShared {
    float m, lz;  // the row's largest logit and log z
    int red[kMostWaves];
    int nsel, lo;  // chunks named, and their threshold
    int sel[kMaxTop + kSlack];
    int same[kMaxTop + kSlack];
    long long cand[kCand];  // order of the logit, then what is left of 2^32 - 1 by the id
};

// Sum, minimum and maximum of an int over the wave, for every lane.
template <typename Op>
__device__ __forceinline__ int wave_reduce(int v, Op op) {
    auto dpp = [](int x, auto ctrl) {
        return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xf, 0xf, false);
    };
    v = op(v, dpp(v, std::integral_constant<int, kDppXor1>{}));
    v = op(v, dpp(v, std::integral_constant<int, kDppXor2>{}));
    v = op(v, dpp(v, std::integral_constant<int, kDppHalfMirror>{}));
    v = op(v, dpp(v, std::integral_constant<int, kDppMirror>{}));
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op((int)s[0], (int)s[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane(op((int)t[0], (int)t[1]));
}
__device__ __forceinline__ int wave_sum_i(int v) {
    return wave_reduce(v, [](int a, int b) { return a + b; });
}

// The threshold over a row's chunk maxima and the chunks that reach it, in
// order, by one wave. at(c): order of chunk c's maximum.
template <typename At>
__device__ __forceinline__ void name_chunks(int nchunk, int top, At at, TopShared& sh) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const unsigned long long below = (1ull << lane) - 1;
    // count(>= lo) >= top, as near to top as the slack, unless maxima tie
    int lo, hi, above = 0, named = nchunk;  // count(>= hi) = above < top
    auto bisect = [&](int least, int most, auto count) {
        lo = wave_reduce(least, [](int a, int b) { return min(a, b); });
        hi = wave_reduce(most, [](int a, int b) { return max(a, b); }) + 1;
        // first whether all but a few are equal (a masked row's chunks)
        for (int m = lo + 1, step = 0; hi - (long long)lo > 1 && named > top + kSlack;
             m = cut_of(lo, hi, step++)) {
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
    int listed = 0, left = 0;
    auto list = [&](int c, int o) {
        const bool over = c < nchunk && o > lo, same = c < nchunk && o == lo;
        const unsigned long long bs = __ballot(same);
        const bool take = over || (same && (int)__popcll(bs & below) < left);
        const unsigned long long bt = __ballot(take);
        if (take) sh.sel[listed + (int)__popcll(bt & below)] = c;
        listed += (int)__popcll(bt);
        left -= min(left, (int)__popcll(bs));
    };
    if (nchunk <= kRegMax * QLM_WAVE) {  // the maxima in registers
        int o[kRegMax], least = INT32_MAX, most = INT32_MIN;
#pragma unroll
        for (int j = 0; j < kRegMax; ++j) {
            o[j] = INT32_MIN;
            if (j * QLM_WAVE + lane < nchunk) o[j] = at(j * QLM_WAVE + lane);
        }
#pragma unroll
        for (int j = 0; j < kRegMax; ++j) {
            most = max(most, o[j]);
            if (j * QLM_WAVE + lane < nchunk) least = min(least, o[j]);
        }
        bisect(least, most, [&](int m) {
            int cnt = 0;
#pragma unroll
            for (int j = 0; j < kRegMax; ++j)
                if (j * QLM_WAVE < nchunk) cnt += o[j] >= m;
            return wave_sum_i(cnt);
        });
        left = named > top + kSlack ? top - above : INT32_MAX;
#pragma unroll
        for (int j = 0; j < kRegMax; ++j)
            if (j * QLM_WAVE < nchunk) list(j * QLM_WAVE + lane, o[j]);
    } else {
        int least = INT32_MAX, most = INT32_MIN;
        for (int c = lane; c < nchunk; c += QLM_WAVE) {
            const int o = at(c);
            least = min(least, o);
            most = max(most, o);
        }
        bisect(least, most, [&](int m) {
            int cnt = 0;
            for (int c = lane; c < nchunk; c += QLM_WAVE) cnt += at(c) >= m;
            return wave_sum_i(cnt);
        });
        left = named > top + kSlack ? top - above : INT32_MAX;
        for (int c0 = 0; c0 < nchunk; c0 += QLM_WAVE)
            list(c0 + lane, at(min(c0 + lane, nchunk - 1)));
    }
    if (lane == 0) {
        sh.nsel = listed;
        sh.lo = lo;
    }
}

// The first `top` tokens of a row by (logit, then lower id), the chunks that
// hold them named in `sh` (or all, where there are no more than `top`), `most`
// the order of its largest logit. CPW: chunks a wave can hold, NW CPW >= top +
// kSlack. Called by the whole workgroup. emit(rank, id, order of the logit).
template <int CPW, int NW, typename Emit>
__device__ __forceinline__ void select_top(const float* row, int n, int nchunk, int top, int most,
                                           TopShared& sh, Emit emit) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    const unsigned long long below = (1ull << lane) - 1;
    const bool listed = nchunk > top;
    const int nsel = listed ? sh.nsel : nchunk;
    // The chunks' logits, chunk `wave + j NW` of the list in o[j], all
    // requested before the first is used; what lies past the row is below all.
    int o[CPW][4], at[CPW];
    {
        f32x4u v[CPW];
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
            const int s = wave + j * NW;
            if (s < nsel) {
                const int c = listed ? __builtin_amdgcn_readfirstlane(sh.sel[s]) : s;
                at[j] = c * kChunk;
                v[j] = load_chunk(row, n, c);
            }
        }
#pragma unroll
        for (int j = 0; j < CPW; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[j][k] = INT32_MIN;
                if (wave + j * NW < nsel && at[j] + 4 * lane + k < n)
                    o[j][k] = order_of(v[j][k]);
            }
    }
    // a count over the workgroup, its own share left in `mine`
    auto total = [&](int c) {
        c = wave_sum_i(c);
        __syncthreads();
        if (lane == 0) sh.red[wave] = c;
        __syncthreads();
        int t = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) t += sh.red[w];
        return t;
    };
    // how many logits reach `from`
    auto count_from = [&](int from) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * NW < nsel)
#pragma unroll
                for (int k = 0; k < 4; ++k) c += o[j][k] >= from;
        return total(c);
    };
    int from = listed ? sh.lo : kLowest, cnt = count_from(from);
    bool tied = false;
    // (ranking many more than `top` costs more than cutting them: 1271 x 5675
    // with 20 alternatives 35 us where any 512 were ranked)
    if (cnt > max(128, 3 * top)) {
        // Logits equal to `from` may be many (masked ones): fewer than `top`
        // above it leave only those, in order. Otherwise bisect: first over
        // the threads' largest logits (at least as many logits reach what
        // `top` of them reach, and hardly more), then, where that was not
        // enough, over the logits: count(>= from) >= top, <= kCand.
        int k = count_from(from + 1);
        if (k >= top) {
            from += 1;
            cnt = k;
            int mine = INT32_MIN;
#pragma unroll
            for (int j = 0; j < CPW; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) mine = max(mine, o[j][i]);
            int hi = most + 1, reach = total(mine >= from);
            if (reach >= top) {
                // from what every thread that has logits reaches
                const int least = wave_reduce(mine >= from ? mine : INT32_MAX,
                                              [](int a, int b) { return min(a, b); });
                __syncthreads();
                if (lane == 0) sh.red[wave] = least;
                __syncthreads();
                from = sh.red[0];
#pragma unroll
                for (int w = 1; w < NW; ++w) from = min(from, sh.red[w]);
                for (int step = 0; hi - (long long)from > 1 && reach > 2 * top; ++step) {
                    const int m = cut_of(from, hi, step);
                    k = total(mine >= m);
                    if (k >= top) {
                        from = m;
                        reach = k;
                    } else {
                        hi = m;
                    }
                }
                cnt = count_from(from);
                hi = most + 1;
            }
            for (int step = 0; hi - (long long)from > 1 && cnt > kCand; ++step) {
                const int m = cut_of(from, hi, step);
                k = count_from(m);
                if (k >= top) {
                    from = m;
                    cnt = k;
                } else {
                    hi = m;
                }
            }
        }
        tied = cnt > kCand;
        cnt = count_from(tied ? from + 1 : from);  // the waves' shares again
    }
    // candidates, this wave's behind those of the waves before it
    int place = 0;
    for (int w = 0; w < wave; ++w) place += sh.red[w];
    auto take = [&](bool in, int order, int id, int p) {
        if (in) sh.cand[p] = ((long long)order << 32) | (unsigned)(0x7fffffff - id);
    };
    {
        const int least = tied ? from + 1 : from;
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * NW < nsel)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = o[j][k] >= least;
                    const unsigned long long b = __ballot(in);
                    if (b == 0) continue;
                    take(in, o[j][k], at[j] + 4 * lane + k, place + (int)__popcll(b & below));
                    place += (int)__popcll(b);
                }
    }
    if (tied) {
        // those equal to `from` follow in the order of their ids: places by
        // the counts of the chunks before, then of the lanes before
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * NW < nsel) {
                int c = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) c += o[j][k] == from;
                c = wave_sum_i(c);
                if (lane == 0) sh.same[wave + j * NW] = c;
            }
        __syncthreads();
        int before = cnt, s0 = 0;
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * NW < nsel) {
                for (; s0 < wave + j * NW && before < top; ++s0) before += sh.same[s0];
                if (before >= top) continue;
                int p = before;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    p += (int)__popcll(__ballot(o[j][k] == from) & below);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = o[j][k] == from;
                    take(in && p < top, from, at[j] + 4 * lane + k, p);
                    p += in;
                }
            }
        cnt = top;
    }
    __syncthreads();
    // ranks: four lanes a candidate, each against a quarter of the others
    for (int i0 = 0; i0 < cnt; i0 += NW * QLM_WAVE / 4) {
        const int i = i0 + (int)threadIdx.x / 4;
        const long long key = sh.cand[min(i, cnt - 1)];
        int rank = 0;
#pragma unroll 8
        for (int j = threadIdx.x & 3; j < cnt; j += 4) rank += sh.cand[j] > key;
        rank += __shfl_xor(rank, 1, QLM_WAVE);
        rank += __shfl_xor(rank, 2, QLM_WAVE);
        if ((threadIdx.x & 3) == 0 && i < cnt && rank < top)
            emit(rank, 0x7fffffff - (int)(key & 0x7fffffff), (int)(key >> 32));
    }
}

// What is wanted of a row. The last wave joins the `count` parts and does
// what needs nothing but sums while the first names the chunks; at(c): order of
// chunk c's maximum.
template <int CPW, int NW, typename At>
__device__ __forceinline__ void finish_row(const LpArgs& a, int row, const Part* parts, int count,
                                           TopShared& sh, At at) {
    const float* lr = a.logits + (size_t)row * a.ldl;
    const int wave = threadIdx.x / QLM_WAVE, lane = threadIdx.x & (QLM_WAVE - 1);
    if (wave == NW - 1) {
        const Part p = join_parts(parts, count);
        // no distribution: every logit masked, a NaN, or +inf among them
        const float z = p.z > 0.0f ? p.z : NAN;
        const float lz = logf(z);
        if (lane == 0) {
            sh.m = p.m;
            sh.lz = lz;
            if (a.entropy) a.entropy[row] = lz - p.u / z;
        }
        for (int j = lane; j < a.n_ids; j += QLM_WAVE) {
            const int id = a.ids[(size_t)row * a.n_ids + j];
            // an id outside the row is not read
            a.id_lp[(size_t)row * a.n_ids + j] =
                id >= 0 && id < a.n ? (lr[id] - p.m) - lz : NAN;
        }
    }
    if constexpr (CPW > 0) {
        if (wave == 0 && a.nchunk > a.top) name_chunks(a.nchunk, a.top, at, sh);
        __syncthreads();
        const float m = sh.m, lz = sh.lz;
        select_top<CPW, NW>(lr, a.n, a.nchunk, a.top, order_of(m), sh,
                            [&](int rank, int id, int order) {
                                a.top_ids[(size_t)row * a.top + rank] = id;
                                a.top_lp[(size_t)row * a.top + rank] = (value_of(order) - m) - lz;
                            });
    }
}

// CPW 0: no alternatives. WHOLE: a workgroup a row, finished at once.
template <int CPW, int NW, bool WHOLE>
__global__ __launch_bounds__(NW* QLM_WAVE) void k_logprob(LpArgs a) {
    extern __shared__ int mx[];
    __shared__ Part parts[NW];
    __shared__ TopShared sh;
    const int row = WHOLE ? blockIdx.x : blockIdx.x / a.slices;
    const int slice = WHOLE ? 0 : blockIdx.x - row * a.slices;
    const float* lr = a.logits + (size_t)row * a.ldl;
    const int per = (a.nchunk + a.slices - 1) / a.slices;
    const int c0 = slice * per, c1 = min(a.nchunk, c0 + per);
    int* maxima = a.maxima + (size_t)row * a.nchunk;
    constexpr int U = !WHOLE ? kSliceUnroll : NW == kMostWaves ? kShortUnroll : kLongUnroll;
    stream_row<NW, U>(lr, a.n, c0, c1, parts, CPW > 0, [&](int c, int o) {
        if constexpr (WHOLE)
            mx[c] = o;
        else
            maxima[c] = o;
    });
    if constexpr (WHOLE) {
        finish_row<CPW, NW>(a, row, parts, NW, sh, [&](int c) { return mx[c]; });
    } else if (threadIdx.x < QLM_WAVE) {
        const Part p = join_parts(parts, NW);
        if (threadIdx.x == 0) a.part[(size_t)row * a.slices + slice] = p;
    }
}

template <int CPW>
__global__ __launch_bounds__(kFinishWaves* QLM_WAVE) void k_logprob_finish(LpArgs a) {
    __shared__ TopShared sh;
    const int row = blockIdx.x;
    const int* maxima = a.maxima + (size_t)row * a.nchunk;
    finish_row<CPW, kFinishWaves>(a, row, a.part + (size_t)row * a.slices, a.slices, sh,
                                  [&](int c) { return maxima[c]; });
}

template <int CPW, int NW>
void launch_whole(const LpArgs& a, hipStream_t st) {
    const size_t lds = CPW > 0 ? (size_t)a.nchunk * sizeof(int) : 0;
    hipLaunchKernelGGL((k_logprob<CPW, NW, true>), dim3(a.rows), dim3(NW * QLM_WAVE), lds, st, a);
}

template <int CPW>
void launch_sliced(const LpArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_logprob<CPW, kWaves, false>), dim3((unsigned)(a.slices * a.rows)),
                       dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL((k_logprob_finish<CPW>), dim3(a.rows), dim3(kFinishWaves * QLM_WAVE), 0, st,
                       a);
}

int chunks_of(int n) { return (n + kChunk - 1) / kChunk; }

// Waves of the workgroup that reads a whole row, 0: rows are sliced. Few short
// rows need no second launch (38 x 6839 11 us sliced, 9 whole); many rows fill
// the GPU with small workgroups. The sums' order goes by this and slices_of alone.
int whole_waves(int rows, int n) {
    if (rows >= 768 || chunks_of(n) <= 4 * kWaves) return kWaves;
    return rows <= 256 && chunks_of(n) <= 4 * kMostWaves ? kMostWaves : 0;
}

// Workgroups a row otherwise: enough in all to fill the GPU, each with work for
// every wave's loads in flight.
int slices_of(int rows, int n) {
    if (whole_waves(rows, n)) return 1;
    const int most = (chunks_of(n) + kWaves * kSliceUnroll - 1) / (kWaves * kSliceUnroll);
    const int want = 2048 / rows;
    return want < most ? want : most;
}

// Whether rows are finished by the workgroups that read them: with few waves
// many alternatives take registers that would leave too few of them on a CU.
bool finished(int waves, int top) {
    return waves == kMostWaves || (waves == kWaves && top + kSlack <= 8 * kWaves);
}

size_t round16(size_t b) { return (b + 15) / 16 * 16; }

}  // namespace

extern "C" size_t qlm_token_logprobs_workspace_bytes(int rows, int n, int top) {
    if (rows <= 0 || n <= 0 || n > kMaxVocab || top < 0) return 0;
    if (finished(whole_waves(rows, n), top)) return 16;
    const int slices = slices_of(rows, n);
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
    // chunks a wave holds: top + kSlack of them over the waves
    constexpr int kFinish = (kMaxTop + kSlack + kFinishWaves - 1) / kFinishWaves;
    constexpr int kShort = (kMaxTop + kSlack + kMostWaves - 1) / kMostWaves;
    const int waves = whole_waves(rows, n);
    if (!finished(waves, top))
        top ? launch_sliced<kFinish>(a, st) : launch_sliced<0>(a, st);
    else if (waves == kMostWaves)
        top ? launch_whole<kShort, kMostWaves>(a, st) : launch_whole<0, kMostWaves>(a, st);
    else if (top == 0)
        launch_whole<0, kWaves>(a, st);
    else if (top + kSlack <= 4 * kWaves)
        launch_whole<4, kWaves>(a, st);
    else
        launch_whole<8, kWaves>(a, st);
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_logprobs() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(k_logprob<0, kWaves, true>));
}
