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
// (histograms over the floats' bits, the maxima in one wave's registers) names
// about k chunks of 1 KB, which are read again (1 % of a 152 K row for
// k = 5); their logits that reach the threshold, little more than k, are
// ranked by counting. Where too many reach it (few chunks, equal or masked
// logits) the threshold is bisected over the logits held, and logits equal to
// it are taken in order. With few rows all of this is a chain of short steps
// of one workgroup, where every instruction shows: a bisection step over the
// chunk maxima takes 0.3 us of one wave, and of 16 waves with a barrier 0.4.
// One workgroup a row does all of it (k_logprob<.., true>) where the rows fill
// the GPU; otherwise slices leave (M, z, u) and their maxima to
// k_logprob_finish. Many rows are bound by the one read of the logits: 2047 x
// 151936 with 5 alternatives 205 us, 6.06 TB/s. Few are bound by that chain and
// two launches: 1 x 151936 with 20 alternatives 8.1 us (10.9 with bisections
// for both thresholds), 37 x 32003 with 64, masked, 11.9 (16.1).

#include <type_traits>

#include "common.hpp"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 256;   // of a workgroup that reads a row or a slice
constexpr int kWaves = kThreads / QLM_WAVE;
constexpr int kFinishWaves = 16;  // of a workgroup that finishes a sliced row
constexpr int kMostWaves = 16;   // of a workgroup that reads one of few short rows
constexpr int kChunk = 4 * QLM_WAVE;  // logits of a chunk: a vector of four a lane
// Chunks a wave keeps in flight: many where one workgroup reads a long row
// (2047 x 151936 211 us with 8, 221 with 4), few where slices are many.
constexpr int kLongUnroll = 8, kShortUnroll = 4, kSliceUnroll = 2;
constexpr int kMaxTop = QLM_TOKEN_LOGPROBS_MAX_TOP;
constexpr int kSlack = 8;             // chunks beyond k that a threshold may name
constexpr int kCand = 512;            // logits that are ranked by counting
constexpr int kMaxVocab = 1 << 21;    // chunk maxima of a row fit 32 KB of LDS
constexpr int kMaxRows = 1 << 21;     // a launch's threads fit 32 bits
constexpr int kRegMax = 16;           // chunk maxima a lane holds in registers
constexpr int kBuckets = 256;         // of a histogram of the chunk maxima
constexpr int kSums = 160;            // over the workgroup: at most 2 x 66 steps and 10
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
                // The product of d with log2 e is rounded, as log2 e itself is, so a
                // term is off by 2 |d| roundings; weighted by the terms themselves
                // that is a few in all (2047 x 151936: results off by 1.3e-7;
                // torch's sums of its exp by 0.6e-7).
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
    float m, lz;   // the row's largest logit and log z
    int nsel, lo;  // chunks named, and their threshold
    int sums[kSums];  // each sum over the workgroup has its own, zero at the start
    int wave[kMostWaves];
    int sel[kMaxTop + kSlack];
    int same[kMaxTop + kSlack];
    long long cand[kCand];  // order of the logit, then what is left of 2^31 - 1 by the id
};

// Sums of the waves' counts, for everyone; the next of them each time.
struct Sums {
    TopShared& sh;
    int used = 0;
    // this wave's place among the counts
    __device__ __forceinline__ int add(int c) {
        int place = 0;
        if ((threadIdx.x & (QLM_WAVE - 1)) == 0) place = atomicAdd(&sh.sums[used], c);
        return __builtin_amdgcn_readfirstlane(place);
    }
    __device__ __forceinline__ int total() {
        __syncthreads();
        return __builtin_amdgcn_readfirstlane(sh.sums[used++]);
    }
    __device__ __forceinline__ int operator()(int c) {
        if (c && (threadIdx.x & (QLM_WAVE - 1)) == 0) atomicAdd(&sh.sums[used], c);
        return total();
    }
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

// Lanes of the mask before this one.
__device__ __forceinline__ int before_me(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31
    return v;
}

// The threshold over a row's chunk maxima and the chunks that reach it, in
// order, by one wave. at(c): order of chunk c's maximum, held in R registers a
// lane, or (R 0) read each time.
template <int R, typename At>
__device__ __forceinline__ void name_chunks_r(int nchunk, int top, At at, TopShared& sh) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    int o[R ? R : 1];
#pragma unroll
    for (int j = 0; j < R; ++j) o[j] = at(min(j * QLM_WAVE + lane, nchunk - 1));
    // f(c, order) for every 64 chunks, c this lane's; past the last INT32_MIN
    auto each = [&](auto f) {
        if constexpr (R > 0) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if (j * QLM_WAVE >= nchunk) break;
                const int c = j * QLM_WAVE + lane;
                f(c, c < nchunk ? o[j] : INT32_MIN);
            }
        } else {
            for (int c = lane; c - lane < nchunk; c += QLM_WAVE)
                f(c, c < nchunk ? at(c) : INT32_MIN);
        }
    };
    int least = INT32_MAX, most = INT32_MIN;
    each([&](int c, int v) {
        most = max(most, v);
        least = c < nchunk ? min(least, v) : least;
    });
    // count(>= lo) = named >= top, as near to top as the slack, unless maxima
    // tie; count(>= hi) = above < top
    int lo = wave_reduce(least, [](int x, int y) { return min(x, y); });
    int hi = wave_reduce(most, [](int x, int y) { return max(x, y); }) + 1;
    int above = 0, named = nchunk;
    int* hist = reinterpret_cast<int*>(sh.cand);
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    while (named > top + kSlack && (unsigned)hi - (unsigned)lo > 1) {
        // lo .. hi - 1 in buckets of 2^shift orders, the highest first
        const int shift = max(0, 24 - __builtin_clz((unsigned)hi - (unsigned)lo - 1));
        *reinterpret_cast<i32x4*>(hist + 4 * lane) = i32x4{0, 0, 0, 0};
        each([&](int, int v) {
            if (v >= lo && v < hi)
                atomicAdd(&hist[kBuckets - 1 - (((unsigned)v - (unsigned)lo) >> shift)], 1);
        });
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const i32x4 h = *reinterpret_cast<const i32x4*>(hist + 4 * lane);
        const int s = (h.x + h.y) + (h.z + h.w), upto = wave_scan(s);
        // the bucket that completes `top`
        const int l = __ffsll(__ballot(above + upto >= top)) - 1;
        int b = kBuckets - 1 - 4 * l, got = above + __builtin_amdgcn_readlane(upto - s, l);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int next = got + __builtin_amdgcn_readlane(h[k], l);
            named = next;
            if (next >= top) break;
            got = next;
            --b;
        }
        above = got;
        const unsigned first = (unsigned)lo + ((unsigned)b << shift);
        if ((unsigned)hi - first > 1u << shift) hi = (int)(first + (1u << shift));
        lo = (int)first;
    }
    // None of those equal to lo is left out, or all but the first that complete
    // `top`. A chunk of the lowest order alone holds nothing else: one is enough
    // (a shorter one is the row's last).
    const bool all = named <= top + kSlack;
    int listed = 0, left = lo == kLowest ? 1 : top - above;
    each([&](int c, int v) {
        bool take = v >= lo;
        if (!all) {
            const unsigned long long same = __ballot(v == lo);
            take = v > lo || (v == lo && before_me(same) < left);
            left -= min(left, (int)__popcll(same));
        }
        const unsigned long long m = __ballot(take);
        if (take) sh.sel[listed + before_me(m)] = c;
        listed += (int)__popcll(m);
    });
    if (lane == 0) {
        sh.nsel = listed;
        sh.lo = lo;
    }
}
template <typename At>
__device__ __forceinline__ void name_chunks(int nchunk, int top, At at, TopShared& sh) {
    if (nchunk <= 2 * QLM_WAVE)
        name_chunks_r<2>(nchunk, top, at, sh);
    else if (nchunk <= kRegMax * QLM_WAVE)
        name_chunks_r<kRegMax>(nchunk, top, at, sh);
    else
        name_chunks_r<0>(nchunk, top, at, sh);
}

// The first `top` tokens of a row by (logit, then lower id), the chunks that
// hold them named in `sh` (or all, where there are no more than `top`). CPW:
// chunks a wave can hold, NW CPW >= top + kSlack. Called by the whole
// workgroup. emit(rank, id, order of the logit).
template <int CPW, int NW, typename Emit>
__device__ __forceinline__ void select_top(const float* row, int n, int nchunk, int top,
                                           TopShared& sh, Sums& sum, Emit emit) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    const bool listed = nchunk > top;
    const int nsel = listed ? __builtin_amdgcn_readfirstlane(sh.nsel) : nchunk;
    const int lo = listed ? __builtin_amdgcn_readfirstlane(sh.lo) : kLowest;
    // Chunk `wave + j NW` of the list (number j of the lanes' `mine`) in v[j],
    // all requested before the first is used. At the row's end a lane's four
    // overlap those of the lane before: what is not this lane's is masked.
    const int s = min(wave + min(lane, CPW - 1) * NW, nsel - 1);
    const int mine = listed ? sh.sel[s] : s;
    auto chunk = [&](int j) { return __builtin_amdgcn_readlane(mine, j); };
    auto first_of = [&](int c) { return max(min(c * kChunk + 4 * lane, n - 4), 0); };
    f32x4u v[CPW];
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        if (wave + j * NW >= nsel) break;
        const float* p = row + first_of(chunk(j));
        if (n >= 4)
            v[j] = *reinterpret_cast<const f32x4u*>(p);
        else
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][k] = p[min(k, n - 1)];
    }
    auto put = [&](int order, int id, int p) {
        sh.cand[p] = ((long long)order << 32) | (unsigned)(0x7fffffff - id);
    };
    // the waves' places for their candidates, the lanes' from a count of each
    auto places = [&](int c) {
        int p = sum.add(wave_sum_i(c));
#pragma unroll
        for (int bit = 1; bit <= 4 * CPW; bit *= 2) p += bit * before_me(__ballot(c & bit));
        return p;
    };
    int cnt = kCand + 1;
    // Ranking many more than `top` costs more than cutting them: 1271 x 5675
    // with 20 alternatives 35 us where any 512 were ranked.
    const int enough = max(128, 3 * top);
    // The threshold says much where chunks were left out; a NaN and what is
    // masked are below it.
    if (lo > kLowest && nchunk > top + kSlack) {
        const float from = value_of(lo);
        // a lane has one candidate or none, hardly ever more: the last of them
        // before number `end` of its 4 CPW logits, and how many there are
        auto last = [&](int end, float& what, int& which) {
            int c = 0;
#pragma unroll
            for (int j = 0; j < CPW; ++j) {
                if (wave + j * NW >= nsel) break;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = v[j][k] >= from && 4 * j + k < end;
                    c += in;
                    what = in ? v[j][k] : what;
                    which = in ? 4 * j + k : which;
                }
            }
            return c;
        };
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * NW < nsel && (chunk(j) + 1) * kChunk > n) {
                const int skip = chunk(j) * kChunk + 4 * lane - first_of(chunk(j));
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < skip) v[j][k] = -INFINITY;
            }
        float what = 0.0f;
        int which = 0, c = last(4 * CPW, what, which), p = places(c);
        while (__ballot(c > 0)) {
            const int id = first_of(__shfl(mine, which >> 2, QLM_WAVE)) + (which & 3);
            if (c > 0 && p < kCand) put(order_of(what), id, p);
            p += 1;
            c -= 1;
            if (__ballot(c > 0)) last(which, what, which);
        }
        cnt = sum.total();
    }
    if (cnt > enough) {
        int o[CPW][4], first[CPW];  // what is not there is below all
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
#pragma unroll
            for (int k = 0; k < 4; ++k) o[j][k] = INT32_MIN;
            if (wave + j * NW < nsel) {
                first[j] = first_of(chunk(j));
                const int skip = chunk(j) * kChunk + 4 * lane - first[j];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k >= skip && k < n) o[j][k] = order_of(v[j][k]);
            }
        }
        auto count_of = [&](auto in) {
            int c = 0;
#pragma unroll
            for (int j = 0; j < CPW; ++j)
                if (wave + j * NW < nsel)
#pragma unroll
                    for (int k = 0; k < 4; ++k) c += in(o[j][k]);
            return c;
        };
        auto count_from = [&](int from) {
            return sum(wave_sum_i(count_of([&](int x) { return x >= from; })));
        };
        int from = lo;
        cnt = count_from(from);
        const int past = order_of(sh.m) + 1;  // the row's largest logit
        bool tied = false;
        if (cnt > enough) {
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
                auto reached = [&](int m) { return sum((int)__popcll(__ballot(mine >= m))); };
                int hi = past, reach = reached(from);
                if (reach >= top) {
                    // from what every thread that has logits reaches
                    const int least = wave_reduce(mine >= from ? mine : INT32_MAX,
                                                  [](int x, int y) { return min(x, y); });
                    if (lane == 0) sh.wave[wave] = least;
                    __syncthreads();
                    from = sh.wave[0];
#pragma unroll
                    for (int w = 1; w < NW; ++w) from = min(from, sh.wave[w]);
                    for (int step = 0; hi - (long long)from > 1 && reach > 2 * top; ++step) {
                        const int m = cut_of(from, hi, step);
                        k = reached(m);
                        if (k >= top) {
                            from = m;
                            reach = k;
                        } else {
                            hi = m;
                        }
                    }
                    cnt = count_from(from);
                    hi = past;
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
        }
        const int least = tied ? from + 1 : from;
        int p = places(count_of([&](int x) { return x >= least; }));
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            if (wave + j * NW < nsel)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (o[j][k] >= least) put(o[j][k], first[j] + k, p++);
        cnt = sum.total();
        if (tied) {
            // those equal to `from` follow in the order of their ids: places by
            // the counts of the chunks before, then of the lanes before
#pragma unroll
            for (int j = 0; j < CPW; ++j)
                if (wave + j * NW < nsel) {
                    int c = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) c += (int)__popcll(__ballot(o[j][k] == from));
                    if (lane == 0) sh.same[wave + j * NW] = c;
                }
            __syncthreads();
            int before = cnt, s0 = 0;
#pragma unroll
            for (int j = 0; j < CPW; ++j)
                if (wave + j * NW < nsel) {
                    for (; s0 < wave + j * NW && before < top; ++s0) before += sh.same[s0];
                    if (before >= top) continue;
                    int q = before;
#pragma unroll
                    for (int k = 0; k < 4; ++k) q += before_me(__ballot(o[j][k] == from));
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool in = o[j][k] == from;
                        if (in && q < top) put(from, first[j] + k, q);
                        q += in;
                    }
                }
            cnt = top;
            __syncthreads();
        }
    }
    // ranks: eight lanes a candidate, each against an eighth of the others
    constexpr int S = 8;
    for (int i0 = 0; i0 < cnt; i0 += NW * QLM_WAVE / S) {
        const int i = i0 + (int)threadIdx.x / S;
        const long long key = sh.cand[min(i, cnt - 1)];
        int rank = 0;
#pragma unroll 4
        for (int j = threadIdx.x % S; j < cnt; j += S) rank += sh.cand[j] > key;
#pragma unroll
        for (int m = 1; m < S; m *= 2) rank += __shfl_xor(rank, m, QLM_WAVE);
        if (threadIdx.x % S == 0 && i < cnt && rank < top)
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
    if constexpr (CPW > 0)
        for (int i = threadIdx.x; i < kSums; i += NW * QLM_WAVE) sh.sums[i] = 0;
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
        Sums sum{sh};
        select_top<CPW, NW>(lr, a.n, a.nchunk, a.top, sh, sum, [&](int rank, int id, int order) {
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
    hipLaunchKernelGGL((k_logprob<(CPW > 0), kWaves, false>), dim3((unsigned)(a.slices * a.rows)),
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
// With 64 alternatives, finished by a second launch and by the reading one: 2047
// x 151936 251 us and 315, 3000 x 32000 132 and 157; rows short enough that the
// second launch counts are the other way round (2047 x 5000 74 and 63).
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
    const int waves = whole_waves(rows, n), held = top ? top + kSlack : 0;
    static_assert(kFinishWaves == kMostWaves, "one number of chunks a wave");
    constexpr int kAll = (kMaxTop + kSlack + kMostWaves - 1) / kMostWaves;
    const int per = (held + kMostWaves - 1) / kMostWaves;
    if (!finished(waves, top)) {
        per == 0   ? launch_sliced<0>(a, st)
        : per == 1 ? launch_sliced<1>(a, st)
        : per == 2 ? launch_sliced<2>(a, st)
                   : launch_sliced<kAll>(a, st);
    } else if (waves == kMostWaves) {
        per == 0   ? launch_whole<0, kMostWaves>(a, st)
        : per == 1 ? launch_whole<1, kMostWaves>(a, st)
        : per == 2 ? launch_whole<2, kMostWaves>(a, st)
                   : launch_whole<kAll, kMostWaves>(a, st);
    } else {
        held == 0            ? launch_whole<0, kWaves>(a, st)
        : held <= 4 * kWaves ? launch_whole<4, kWaves>(a, st)
                             : launch_whole<8, kWaves>(a, st);
    }
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_logprobs() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(k_logprob<0, kWaves, true>));
}
