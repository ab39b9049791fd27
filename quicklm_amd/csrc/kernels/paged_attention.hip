// Attention of ragged rows (single tokens, trees of drafted tokens, prompts)
// over a paged KV cache on the bf16 matrix cores (qlm_paged_attention).
//
// A row of a unit is a (token, query head) pair: the G = n_q / n_kv heads of a
// kv head share its keys, so a unit is MT such pairs of one sequence and kv head
// and reads every key and value once. Keys go through in blocks of 32 with a
// running maximum and sum (exponentials to the base 2, the scale folded into
// the queries):
//   S^T = K Q^T: A = 16 keys, B = the 16 rows of a tile; lane (qd, n) = (l / 16,
//     l % 16) then holds row n's scores of keys 4 qd + i of each 16-key half;
//   O^T += V^T P^T: the k-slots of lane group qd are those eight keys, so the
//     probabilities are the B operand in the registers that computed them, and
//     V^T comes out of row-major LDS through the transposing LDS read (4 keys
//     of 16 columns a lane group).
// fp32 operands are split into two bf16 terms, x = h + l to 2^-17 of x: queries
// and probabilities take two products each, with an fp32 cache three (h h, h l,
// l h; what is left out is below 2^-16). Up to 8 rows need one product
// where others need two: rows 0..7 of the tile hold the h terms, rows 8..15 the
// l terms, and the two halves are added.
//
// Keys and values go straight from the pages to LDS. A 16-key group lies in one
// page and is read through a buffer descriptor that ends where the group's
// slots do, so that slots behind the last key arrive as zeros, whatever lies
// there, and a page number that is out of range reads nothing. 16-byte piece c of
// a row sits at piece c ^ (key % 16), which spreads the 16 rows that an LDS
// access touches over all banks.
//
// Lengths are known on the device alone. A launch has room for `target` + units
// work items a kv head; each workgroup reads the lengths, forms the chunk that
// cuts all sequences' keys into about `target` items and finds its own. A unit of
// more than one chunk leaves records [m, l, O] that k_pa_join merges; the others
// write their outputs.

#include <algorithm>

#include "paged.hpp"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct PaArgs {
    const float* q;
    const float* gate;  // NULL: none
    float* out;
    float* rec;  // records of HD + 4 floats
    int2* desc;  // [rows, n_kv]: a row's first record (of the kv head's first query head), chunks
    long long ldq, ldg, ldo;
    int gate_stride, n_q, lg;  // G = 1 << lg
    int target, items, rec_rows, slots;
    float qscale;  // log2(e) / sqrt(hd)
    qlm_row_batch bt;
    qlm_kv_pages pg;
};

// ---- which work a workgroup does ----

struct Item {
    SeqRows sq;
    int b, tile, chunk;  // chunk: which
    int len;             // keys of a chunk
    int rec;             // the unit's first record block
    bool split;          // the sequence's units may have several chunks
};

__device__ __forceinline__ int tiles_of(int n, int lg, int mt) {
    return (int)((((long long)n << lg) + mt - 1) / mt);
}

// new rows that any row can see
__device__ __forceinline__ int seen_rows(const PaArgs& a, const SeqRows& s) {
    return a.bt.parent ? min(s.n, QLM_TREE_MAX) : s.n;
}

// Item `want` of a kv head, counted over the sequences: the longest prompts'
// last tiles, which see the most keys, first. Every lane gets it.
constexpr int kMinChunk = 128;  // keys of a chunk at least
template <int MT>
__device__ __forceinline__ bool find_item(const PaArgs& a, int want, Item& it) {
    const int lane = threadIdx.x & (QLM_WAVE - 1), B = a.bt.B;
    double cost = 0.0;
    SeqRows s{};
    for (int i = 0; i < B; i += QLM_WAVE) {
        s = seq_rows(a.bt, min(i + lane, B - 1));
        if (i + lane >= B) s.n = 0;
        if (s.n > 0)
            cost += (double)tiles_of(s.n, a.lg, MT) * min(s.ctx + seen_rows(a, s), a.slots);
    }
#pragma unroll
    for (int d = 1; d < QLM_WAVE; d <<= 1) cost += __shfl_xor(cost, d);
    const double share = ceil(cost / (double)a.target / 32.0) * 32.0;
    it.len = (int)fmin(fmax(share, (double)kMinChunk), (double)(1 << 30));
    int before = 0, rec = 0;
    for (int i = 0; i < B; i += QLM_WAVE) {
        if (B > QLM_WAVE) {
            s = seq_rows(a.bt, min(i + lane, B - 1));
            if (i + lane >= B) s.n = 0;
        }
        int items = 0, recs = 0;
        if (s.n > 0) {
            const int keys = min(s.ctx + seen_rows(a, s), a.slots);
            const int nch = (keys - 1) / it.len + 1;
            items = tiles_of(s.n, a.lg, MT) * nch;
            recs = nch > 1 ? items : 0;
        }
        int ic = items, rc = recs;  // inclusive sums
#pragma unroll
        for (int d = 1; d < QLM_WAVE; d <<= 1) {
            const int x = __shfl_up(ic, d), y = __shfl_up(rc, d);
            if (lane >= d) {
                ic += x;
                rc += y;
            }
        }
        const unsigned long long at = __ballot(before + ic > want);
        if (at) {
            const int w = __ffsll((long long)at) - 1;
            auto of = [&](int x) { return __builtin_amdgcn_readlane(x, w); };
            it.b = i + w;
            it.sq = SeqRows{of(s.first), of(s.n), of(s.ctx)};
            it.len = __builtin_amdgcn_readfirstlane(it.len);
            const int mine = want - before - of(ic - items);
            const int tiles = tiles_of(it.sq.n, a.lg, MT), nch = of(items) / tiles;
            it.chunk = mine % nch;
            it.tile = tiles - 1 - mine / nch;
            it.split = nch > 1;
            it.rec = rec + of(rc - recs) + mine - it.chunk;
            return true;
        }
        before += __builtin_amdgcn_readlane(ic, QLM_WAVE - 1);
        rec += __builtin_amdgcn_readlane(rc, QLM_WAVE - 1);
    }
    return false;
}

// Workgroups go to the 8 XCDs in turn; those of a kv head, which share its
// keys, to as few of them as the heads leave it.
__device__ __forceinline__ void head_and_item(int id, int n_kv, int& g, int& item) {
    if (n_kv <= 8 && (n_kv & (n_kv - 1)) == 0) {
        const int per = 8 / n_kv, x = id & 7;
        g = x / per;
        item = (id >> 3) * per + x % per;
    } else {
        g = id % n_kv;
        item = id / n_kv;
    }
}

// ---- moving keys and values ----

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const char* p, unsigned bytes) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0,
                                             (int)__builtin_amdgcn_readfirstlane(bytes),
                                             0x00027000);
}

__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, char* to, int lane_off,
                                            int uniform_off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)to, 16,
                                             lane_off, uniform_off, 0, 0);
}

// A 16-key group: its page and how many of its slots are there.
struct Group {
    int page, valid;
};

// Group at `slot` (a multiple of 16, uniform) of keys that end at `end`.
__device__ __forceinline__ Group group_at(const PaArgs& a, int b, int slot, int end, int lgp) {
    const int i = slot >> lgp;
    const bool in = slot < end && i < a.pg.ld_table;
    // a scalar load: of the constant address space
    const auto* table = reinterpret_cast<const __attribute__((address_space(4))) int*>(
        reinterpret_cast<uintptr_t>(a.pg.table));
    const int p = table[(size_t)b * a.pg.ld_table + (in ? i : 0)];
    Group g;
    g.valid = in && (unsigned)p < (unsigned)a.pg.n_pages ? min(end - slot, 16) : 0;
    g.page = g.valid > 0 ? p : 0;
    return g;
}

// The layouts of a 16-key group in LDS. bf16: rows of HD, pieces swizzled.
// fp32: rows as they are, split into two such planes afterwards.
template <int HD, bool F32>
struct Lay {
    static constexpr int ROW = HD * 2;        // bytes of a plane's row
    static constexpr int GRP = 16 * ROW;      // of a plane's group
    static constexpr int RAW = F32 ? 2 * GRP : GRP;  // of a group as it is loaded
    static constexpr int LOADS = RAW / 1024;  // a wave's loads of a group
    // the lane's source offset of load j
    __device__ static __forceinline__ int src(int j) {
        const int lane = threadIdx.x & (QLM_WAVE - 1);
        if constexpr (F32) return j * 1024 + lane * 16;
        constexpr int PPR = ROW / 16;  // pieces of a row
        const int row = (j * QLM_WAVE + lane) / PPR, piece = lane % PPR;
        return row * ROW + ((piece ^ row) * 16);
    }
};

template <int HD, bool F32>
__device__ __forceinline__ void fetch_group(const PaArgs& a, const void* pool, const Group& gr,
                                            int g, int slot, char* to) {
    using L = Lay<HD, F32>;
    constexpr int SIZE = F32 ? 4 : 2;
    const size_t at = (((size_t)gr.page * a.pg.n_kv + g) * a.pg.page_size +
                       (slot & (a.pg.page_size - 1))) * (HD * SIZE);
    const __amdgpu_buffer_rsrc_t r =
        make_rsrc(reinterpret_cast<const char*>(pool) + at, (unsigned)gr.valid * (HD * SIZE));
#pragma unroll
    for (int j = 0; j < L::LOADS; ++j) load_to_lds(r, to + j * 1024, L::src(j), 0);
}

__device__ __forceinline__ unsigned pk_bf16(float x, float y) {
    const f32x2 v = {x, y};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}

// eight floats as two bf16 terms each
__device__ __forceinline__ void split8(const float (&x)[8], u32x4& h, u32x4& l) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned w = pk_bf16(x[2 * i], x[2 * i + 1]);
        h[i] = w;
        l[i] = pk_bf16(x[2 * i] - __uint_as_float(w << 16),
                       x[2 * i + 1] - __uint_as_float(w & 0xffff0000u));
    }
}

// A raw fp32 group (or part p of `parts` of it) into its two planes.
template <int HD>
__device__ __forceinline__ void split_group(const char* raw, char* hi, char* lo, int part,
                                            int parts) {
    constexpr int ROW = HD * 2, PPR = ROW / 16, N = 16 * PPR / QLM_WAVE;
    const int lane = threadIdx.x & (QLM_WAVE - 1);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (parts > 1 && j % parts != part) continue;
        const int at = j * QLM_WAVE + lane, row = at / PPR, piece = at % PPR;
        const f32x4 x0 = *reinterpret_cast<const f32x4*>(raw + at * 32);
        const f32x4 x1 = *reinterpret_cast<const f32x4*>(raw + at * 32 + 16);
        const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        u32x4 h, l;
        split8(x, h, l);
        const int to = row * ROW + ((piece ^ row) * 16);
        *reinterpret_cast<u32x4*>(hi + to) = h;
        *reinterpret_cast<u32x4*>(lo + to) = l;
    }
}

// ---- a wave's rows ----

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// over the four lane groups of a column
__device__ __forceinline__ float cols_max(float v) { return xor32_max(xor16_max(v)); }
__device__ __forceinline__ float cols_sum(float v) { return xor32_add(xor16_add(v)); }

// v(l) + v(l ^ 8) of each 16 lanes
__device__ __forceinline__ float fold8(float v) { return v + dpp_mov<0x128>(v); }  // row_ror:8

// RT tiles of 16 rows; PACK: one tile of 8 rows, h and l terms side by side.
template <int HD, int RT, bool PACK>
struct Rows {
    static constexpr int KS = HD / 32, CB = HD / 16, QT = PACK ? 1 : 2;
    u32x4 q[RT][QT][KS];
    f32x4 acc[RT][CB];
    float m[RT], l[RT];
    int lim[RT];  // slots below this one are seen; -1: a row outside the tree
    unsigned long long line[RT];  // new rows seen beside those
};

// Query rows r0 + 16 t + n of the unit (r: its token and head) and what they see.
template <int HD, int RT, bool PACK>
__device__ __forceinline__ void load_rows(const PaArgs& a, const Item& it, int g, int r0,
                                          Rows<HD, RT, PACK>& R) {
    using T = Rows<HD, RT, PACK>;
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15, qd = lane >> 4;
    const int total = it.sq.n << a.lg;
    unsigned long long mine = 0;
    if (a.bt.parent) mine = tree_line(tree_parent(a.bt, it.sq, lane));
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = r0 + 16 * t + (PACK ? n & 7 : n);
        const int rc = min(r, total - 1), tok = rc >> a.lg, h = rc & ((1 << a.lg) - 1);
        const float* qr = a.q + (size_t)(it.sq.first + tok) * a.ldq +
                          ((size_t)(g << a.lg) + h) * HD;
        R.m[t] = -INFINITY;
        R.l[t] = 0.0f;
        R.lim[t] = it.sq.ctx + tok + 1;
        R.line[t] = 0;
        if (a.bt.parent) {
            const int at = min(tok, QLM_TREE_MAX - 1);
            const unsigned long long ln = (unsigned long long)__shfl((unsigned)(mine >> 32), at)
                                              << 32 | __shfl((unsigned)mine, at);
            R.line[t] = tok < QLM_TREE_MAX ? ln : 0;
            R.lim[t] = R.line[t] ? it.sq.ctx : -1;
        }
        f32x4u x[T::KS][2];
#pragma unroll
        for (int s = 0; s < T::KS; ++s) {
            x[s][0] = *reinterpret_cast<const f32x4u*>(qr + 32 * s + 8 * qd);
            x[s][1] = *reinterpret_cast<const f32x4u*>(qr + 32 * s + 8 * qd + 4);
        }
#pragma unroll
        for (int s = 0; s < T::KS; ++s) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = x[s][i / 4][i % 4] * a.qscale;
            u32x4 hi, lo;
            split8(v, hi, lo);
            if constexpr (PACK) {
                R.q[t][0][s] = n < 8 ? hi : lo;
            } else {
                R.q[t][0][s] = hi;
                R.q[t][1][s] = lo;
            }
        }
#pragma unroll
        for (int c = 0; c < T::CB; ++c) R.acc[t][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// A block of 32 keys from slot k0 on; kp, vp: its K and V planes (of an fp32
// cache the h planes, the l planes `lo` bytes behind). `all`: every row sees
// every key of it.
template <int HD, int RT, bool PACK, bool F32>
__device__ __forceinline__ void block32(Rows<HD, RT, PACK>& R, const char* kp, const char* vp,
                                        int lo, int k0, int ctx, int valid0, int valid1, bool all) {
    using T = Rows<HD, RT, PACK>;
    constexpr int ROW = HD * 2, GRP = 16 * ROW;
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15, qd = lane >> 4;
    f32x4 s[2][RT];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < RT; ++t) s[h][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < T::KS; ++k) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = h * GRP + n * ROW + (((4 * k + qd) ^ n) * 16);
            const u32x4 kh = *reinterpret_cast<const u32x4*>(kp + at);
            u32x4 kl;
            if constexpr (F32) kl = *reinterpret_cast<const u32x4*>(kp + lo + at);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                if constexpr (F32) s[h][t] = mfma(kl, R.q[t][0][k], s[h][t]);
                if constexpr (!PACK) s[h][t] = mfma(kh, R.q[t][1][k], s[h][t]);
                s[h][t] = mfma(kh, R.q[t][0][k], s[h][t]);
            }
        }
    }
    u32x4 ph[RT], pl[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = s[j / 4][t][j % 4];
            if constexpr (PACK) x[j] = fold8(x[j]);
        }
        if (!all) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int in = 4 * qd + j % 4, slot = k0 + 16 * (j / 4) + in, row = slot - ctx;
                bool sees = slot < R.lim[t];
                if (row >= 0 && row < QLM_TREE_MAX) sees |= (R.line[t] >> row) & 1ull;
                sees &= in < (j < 4 ? valid0 : valid1);
                x[j] = sees ? x[j] : -INFINITY;
            }
        }
        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                          fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        top = fmaxf(cols_max(top), R.m[t]);
        const float ref = top == -INFINITY ? 0.0f : top;
        if (__ballot(top > R.m[t])) {  // a row's maximum has risen
            const float f = __builtin_amdgcn_exp2f(R.m[t] - ref);  // 0 the first time
            R.l[t] *= f;
#pragma unroll
            for (int c = 0; c < T::CB; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) R.acc[t][c][i] *= f;
            R.m[t] = top;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(x[j] - ref);
        R.l[t] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        split8(x, ph[t], pl[t]);
        if constexpr (PACK) ph[t] = n < 8 ? ph[t] : pl[t];
    }
    // V^T: lane l of a group reads 4 columns of key 4 qd + (l % 16) / 4
    const int key = 4 * qd + (n >> 2);
#pragma unroll
    for (int c = 0; c < T::CB; ++c) {
        const int at = key * ROW + (((2 * c + ((n >> 1) & 1)) ^ key) * 16) + (n & 1) * 8;
        auto tr = [&](const char* p) {
            return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                 (__attribute__((address_space(3))) s16x4*)p));
        };
        const u32x2 v0 = tr(vp + at), v1 = tr(vp + GRP + at);
        const u32x4 vh = {v0.x, v0.y, v1.x, v1.y};
        u32x4 vl;
        if constexpr (F32) {
            const u32x2 w0 = tr(vp + lo + at), w1 = tr(vp + lo + GRP + at);
            vl = u32x4{w0.x, w0.y, w1.x, w1.y};
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            if constexpr (F32) R.acc[t][c] = mfma(vl, ph[t], R.acc[t][c]);
            if constexpr (!PACK) R.acc[t][c] = mfma(vh, pl[t], R.acc[t][c]);
            R.acc[t][c] = mfma(vh, ph[t], R.acc[t][c]);
        }
    }
}

// ---- outputs ----

// Head h of row i of a sequence in fp32, key after key, by a whole wave: for
// results that did not come out finite. What a row does not see is not
// touched here, so that only its own keys and values can make it NaN.
template <int HD, typename KV>
__device__ void row_in_fp32(const PaArgs& a, int b, const SeqRows& sq, int i, int h,
                            float (&o)[HD / QLM_WAVE]) {
    constexpr int E = HD / QLM_WAVE;
    const int lane = threadIdx.x & (QLM_WAVE - 1), g = h >> a.lg;
    unsigned long long line = ~0ull;
    if (a.bt.parent) {
        const unsigned long long mine = tree_line(tree_parent(a.bt, sq, lane));
        const int at = min(i, QLM_TREE_MAX - 1);
        line = (unsigned long long)__shfl((unsigned)(mine >> 32), at) << 32 |
               __shfl((unsigned)mine, at);
        if (i >= QLM_TREE_MAX) line = 0;
    }
    float q[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        q[j] = a.q[(size_t)(sq.first + i) * a.ldq + (size_t)h * HD + lane + 64 * j] * a.qscale;
        o[j] = 0.0f;
    }
    bool any = false;
    const int end = line ? min(sq.ctx + (a.bt.parent ? seen_rows(a, sq) : i + 1), a.slots) : 0;
    for (int s = 0; s < end; ++s) {
        if (a.bt.parent && s >= sq.ctx && !(line >> (s - sq.ctx) & 1ull)) continue;
        const int page = page_of(a.pg, b, s);
        if (page < 0) continue;
        any = true;
        const size_t at = slot_at(a.pg, page, g, s) + lane;
        float x = 0.0f, v[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            float k;
            if constexpr (sizeof(KV) == 4) {
                k = reinterpret_cast<const float*>(a.pg.k)[at + 64 * j];
                v[j] = reinterpret_cast<const float*>(a.pg.v)[at + 64 * j];
            } else {
                k = bf16_to_f32(reinterpret_cast<const uint16_t*>(a.pg.k)[at + 64 * j]);
                v[j] = bf16_to_f32(reinterpret_cast<const uint16_t*>(a.pg.v)[at + 64 * j]);
            }
            x = fmaf(q[j], k, x);
        }
        x = wave_sum(x);
        const float top = fmaxf(m, x), ref = top == -INFINITY ? 0.0f : top;
        const float f = exp2f(m - ref), p = exp2f(x - ref);
        l = fmaf(l, f, p);
#pragma unroll
        for (int j = 0; j < E; ++j)
            // a key of no weight leaves no trace of its value
            o[j] = p == 0.0f ? o[j] * f : fmaf(p, v[j], o[j] * f);
        m = top;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = any ? o[j] / l : 0.0f;
}

// A row's outputs, E of them a lane (element lane + 64 j): checked, gated, stored.
template <int HD, typename KV>
__device__ __forceinline__ void put_row(const PaArgs& a, int b, const SeqRows& sq, int i, int h,
                                        float (&o)[HD / QLM_WAVE], float l) {
    constexpr int E = HD / QLM_WAVE;
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    bool fine = l > 0.0f && l < INFINITY;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        o[j] /= l;
        fine &= fabsf(o[j]) < INFINITY;
    }
    if (__ballot(!fine)) row_in_fp32<HD, KV>(a, b, sq, i, h, o);
    const size_t r = (size_t)(sq.first + i);
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int e = lane + 64 * j;
        if (a.gate) o[j] *= sigmoid_f(a.gate[r * a.ldg + (size_t)h * a.gate_stride + e]);
        a.out[r * a.ldo + (size_t)h * HD + e] = o[j];
    }
}

// Keys that a unit's rows can see end here; its last token is `last`.
__device__ __forceinline__ int keys_end(const PaArgs& a, const SeqRows& sq, int last) {
    const int n = a.bt.parent ? seen_rows(a, sq) : last + 1;
    return min(sq.ctx + n, a.slots);
}

// Where the unit's rows leave their results: descriptors for k_pa_join.
template <int MT>
__device__ __forceinline__ void put_desc(const PaArgs& a, const Item& it, int g, int nch) {
    const int total = it.sq.n << a.lg, r0 = it.tile * MT;
    const int t0 = r0 >> a.lg, t1 = (min(r0 + MT, total) - 1) >> a.lg;
    for (int t = t0 + (int)threadIdx.x; t <= t1; t += blockDim.x) {
        const int base = (it.rec * a.pg.n_kv + g) * MT + (t << a.lg) - r0;
        a.desc[(size_t)(it.sq.first + t) * a.pg.n_kv + g] = make_int2(base, nch);
    }
}

// ---- up to 16 rows a unit: every wave streams blocks of its own ----
// NW waves take the chunk's 32-key blocks in turn, each through a ring in LDS of
// its own, and meet at the end: nothing waits for another wave's loads.
template <int HD, bool F32>
struct FewShape {
    static constexpr int BLK = 2 * 2 * Lay<HD, F32>::RAW;  // a block's bytes: K, V, two groups
    static constexpr int NW = 65536 * 2 / (2 * BLK);       // 128 KB of LDS: two blocks a wave
};

template <int HD, bool F32, bool PACK>
__global__ __launch_bounds__((FewShape<HD, F32>::NW * QLM_WAVE)) void k_pa_few(PaArgs a) {
    using L = Lay<HD, F32>;
    using S = FewShape<HD, F32>;
    using KV = typename std::conditional<F32, float, uint16_t>::type;
    constexpr int MT = PACK ? 8 : 16, NW = S::NW, GRP = L::GRP, RAW = L::RAW;
    constexpr int LOADS = 4 * L::LOADS;  // a block's
    constexpr int OST = HD + 4;
    static_assert(NW * 16 * OST * 4 + NW * 16 * 8 <= NW * 2 * S::BLK, "the join fits the rings");
    __shared__ __attribute__((aligned(1024))) char smem[NW * 2 * S::BLK];
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15, qd = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    int g, want;
    head_and_item(blockIdx.x, a.pg.n_kv, g, want);
    Item it;
    if (want >= a.items || !find_item<MT>(a, want, it)) return;
    const int total = it.sq.n << a.lg, r0 = it.tile * MT;
    const int end = keys_end(a, it.sq, (min(r0 + MT, total) - 1) >> a.lg);
    const int nch = (end - 1) / it.len + 1;
    if (it.chunk >= nch) return;
    const int b = it.b, k0 = it.chunk * it.len, k1 = min(k0 + it.len, end);
    const int lgp = 31 - __clz(a.pg.page_size);
    const int blocks = (k1 - k0 + 31) / 32, mine = (blocks - wave + NW - 1) / NW;
    char* ring = smem + wave * 2 * S::BLK;
    auto slot_of = [&](int j) { return k0 + 32 * (wave + j * NW); };
    auto groups = [&](int j, Group (&gr)[2]) {
        gr[0] = group_at(a, b, slot_of(j), k1, lgp);
        gr[1] = group_at(a, b, slot_of(j) + 16, k1, lgp);
    };
    // a block in LDS: K groups, V groups
    auto fetch = [&](int j, const Group (&gr)[2]) {
        char* to = ring + (F32 ? 0 : j & 1) * S::BLK;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            fetch_group<HD, F32>(a, a.pg.k, gr[h], g, slot_of(j) + 16 * h, to + h * RAW);
            fetch_group<HD, F32>(a, a.pg.v, gr[h], g, slot_of(j) + 16 * h, to + (2 + h) * RAW);
        }
    };
    constexpr int D = F32 ? 1 : 2;  // blocks in flight
    Group gr[3][2];                 // of blocks j, j + 1 and j + 2
#pragma unroll
    for (int j = 0; j < 3; ++j) groups(j, gr[j]);
    Rows<HD, 1, PACK> R;
    load_rows<HD, 1, PACK>(a, it, g, r0, R);
    // (the queries' loads are waited for before any of the ring's goes out)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < D; ++j)
        if (j < mine) fetch(j, gr[j]);
#pragma unroll 1
    for (int j = 0; j < mine; ++j) {
        if (!F32 && j + 1 < mine)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const int s0 = slot_of(j);
        const bool all = s0 + 32 <= it.sq.ctx && gr[0][0].valid == 16 && gr[0][1].valid == 16;
        char* at = ring + (F32 ? 0 : j & 1) * S::BLK;
        if constexpr (F32) {
            // planes: K h, K l, V h, V l
            char* pl = ring + S::BLK;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                split_group<HD>(at + h * RAW, pl + h * GRP, pl + (2 + h) * GRP, 0, 1);
                split_group<HD>(at + (2 + h) * RAW, pl + (4 + h) * GRP, pl + (6 + h) * GRP, 0, 1);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (j + 1 < mine) fetch(j + 1, gr[1]);
            block32<HD, 1, PACK, F32>(R, pl, pl + 4 * GRP, 2 * GRP, s0, it.sq.ctx, gr[0][0].valid,
                                      gr[0][1].valid, all);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        } else {
            block32<HD, 1, PACK, F32>(R, at, at + 2 * RAW, 0, s0, it.sq.ctx, gr[0][0].valid,
                                      gr[0][1].valid, all);
            // the block is read: its place takes the next but one
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (j + 2 < mine) fetch(j + 2, gr[2]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            gr[0][h] = gr[1][h];
            gr[1][h] = gr[2][h];
        }
        groups(j + 3, gr[2]);
    }
    // ---- the waves' sums meet ----
    __syncthreads();
    float* po = reinterpret_cast<float*>(smem);         // [NW][16][OST]
    float* pm = po + NW * 16 * OST;                     // [NW][16] maxima, then sums
    float* ps = pm + NW * 16;
    const float lsum = cols_sum(R.l[0]);
    if (qd == 0) {
        pm[wave * 16 + n] = R.m[0];
        ps[wave * 16 + n] = lsum;
    }
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) {
        f32x4 o = R.acc[0][c];
        if constexpr (PACK) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fold8(o[i]);
        }
        *reinterpret_cast<f32x4*>(po + (wave * 16 + n) * OST + 16 * c + 4 * qd) = o;
    }
    __syncthreads();
    if (it.chunk == 0 && a.desc) put_desc<MT>(a, it, g, nch);
    const int rows = min(MT, total - r0);
    for (int r = wave; r < rows; r += NW) {
        float m = -INFINITY, l = 0.0f, o[HD / 64] = {};
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, pm[w * 16 + r]);
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(pm[w * 16 + r] - ref);
            l = fmaf(ps[w * 16 + r], f, l);
#pragma unroll
            for (int e = 0; e < HD / 64; ++e)
                o[e] = fmaf(po[(w * 16 + r) * OST + lane + 64 * e], f, o[e]);
        }
        // (blocks that every row sees go unmasked: a row outside the tree too)
        if (__shfl(R.lim[0], r) < 0) l = 0.0f;
        const int tok = (r0 + r) >> a.lg, h = (g << a.lg) + ((r0 + r) & ((1 << a.lg) - 1));
        if (nch == 1) {
            put_row<HD, KV>(a, b, it.sq, tok, h, o, l);
        } else {
            const int at = ((it.rec + it.chunk) * a.pg.n_kv + g) * MT + r;
            if (at < a.rec_rows) {
                float* rec = a.rec + (size_t)at * (HD + 4);
                if (lane == 0) {
                    rec[0] = m;
                    rec[1] = l;
                }
#pragma unroll
                for (int e = 0; e < HD / 64; ++e) rec[4 + lane + 64 * e] = o[e];
            }
        }
    }
}

// ---- more rows: four waves share each block of keys ----
template <int HD, bool F32>
struct TileShape {
    static constexpr int KB = HD == 128 && !F32 ? 64 : 32;  // keys of a block
    static constexpr int BLK = KB / 16 * 2 * Lay<HD, F32>::RAW;
    static constexpr int OST = HD + 4;  // floats of an output row on its way out
    static constexpr int LDS = std::max(F32 ? BLK + KB / 16 * 4 * Lay<HD, F32>::GRP : 2 * BLK,
                                        4 * 16 * OST * 4);
};

template <int HD, bool F32, int RT>
__global__ __launch_bounds__(256, HD == 128 ? 2 : 1) void k_pa_tile(PaArgs a) {
    using L = Lay<HD, F32>;
    using S = TileShape<HD, F32>;
    using KV = typename std::conditional<F32, float, uint16_t>::type;
    constexpr int NW = 4, MT = 16 * RT * NW, KB = S::KB, NG = KB / 16, GRP = L::GRP, RAW = L::RAW;
    constexpr int OST = S::OST;
    __shared__ __attribute__((aligned(1024))) char smem[S::LDS];
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15, qd = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    int g, want;
    head_and_item(blockIdx.x, a.pg.n_kv, g, want);
    Item it;
    if (want >= a.items || !find_item<MT>(a, want, it)) return;
    const int total = it.sq.n << a.lg, r0 = it.tile * MT;
    const int end = keys_end(a, it.sq, (min(r0 + MT, total) - 1) >> a.lg);
    const int nch = (end - 1) / it.len + 1;
    if (it.chunk >= nch) return;
    const int b = it.b, k0 = it.chunk * it.len, k1 = min(k0 + it.len, end);
    const int lgp = 31 - __clz(a.pg.page_size);
    const int blocks = (k1 - k0 + KB - 1) / KB;
    // units (a group's K or V) u = wave, wave + 4, ... are this wave's to fetch
    auto groups = [&](int j, Group (&gr)[NG]) {
#pragma unroll
        for (int i = 0; i < NG; ++i) gr[i] = group_at(a, b, k0 + j * KB + 16 * i, k1, lgp);
    };
    auto fetch = [&](int j, const Group (&gr)[NG]) {
        char* to = smem + (F32 ? 0 : j & 1) * S::BLK;
#pragma unroll
        for (int u = 0; u < 2 * NG; ++u) {
            if (u % NW != wave) continue;
            fetch_group<HD, F32>(a, u < NG ? a.pg.k : a.pg.v, gr[u % NG], g,
                                 k0 + j * KB + 16 * (u % NG), to + u * RAW);
        }
    };
    Group gr[2][NG];
    groups(0, gr[0]);
    groups(1, gr[1]);
    Rows<HD, RT, false> R;
    const int w0 = r0 + 16 * RT * wave;  // this wave's first row
    load_rows<HD, RT, false>(a, it, g, w0, R);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    fetch(0, gr[0]);
    // what all of this wave's rows see without a mask, and all they can see
    const int wave_end = min(w0 < total ? keys_end(a, it.sq, (min(w0 + 16 * RT, total) - 1) >> a.lg) : 0, k1);
    const int free_end = a.bt.parent ? it.sq.ctx : it.sq.ctx + (w0 >> a.lg) + 1;
#pragma unroll 1
    for (int j = 0; j < blocks; ++j) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // the block is there, and every wave is done with the last one
        char* at = smem + (F32 ? 0 : j & 1) * S::BLK;
        if constexpr (F32) {
            char* pl = smem + S::BLK;  // planes: K h, K l, V h, V l
#pragma unroll
            for (int u = 0; u < 2 * NG; ++u) {
                if (u % NW != wave) continue;
                char* to = pl + (u < NG ? u : u + NG) * GRP;
                split_group<HD>(at + u * RAW, to, to + NG * GRP, 0, 1);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __syncthreads();
        }
        if (j + 1 < blocks) fetch(j + 1, gr[1]);
#pragma unroll
        for (int h = 0; h < NG / 2; ++h) {
            const int s0 = k0 + j * KB + 32 * h;
            if (s0 >= wave_end) break;
            const int va = gr[0][2 * h].valid, vb = gr[0][2 * h + 1].valid;
            const bool all = s0 + 32 <= free_end && va == 16 && vb == 16;
            const char* kp = F32 ? smem + S::BLK + 2 * h * GRP : at + 2 * h * RAW;
            const char* vp = F32 ? kp + 2 * NG * GRP : kp + NG * RAW;
            block32<HD, RT, false, F32>(R, kp, vp, NG * GRP, s0, it.sq.ctx, va, vb, all);
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) gr[0][i] = gr[1][i];
        groups(j + 2, gr[1]);
    }
    if (it.chunk == 0 && a.desc) put_desc<MT>(a, it, g, nch);
    // a tile at a time through LDS, a row a time out of it
    __syncthreads();
    float* po = reinterpret_cast<float*>(smem) + wave * 16 * OST;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float lsum = cols_sum(R.l[t]);
#pragma unroll
        for (int c = 0; c < HD / 16; ++c)
            *reinterpret_cast<f32x4*>(po + n * OST + 16 * c + 4 * qd) = R.acc[t][c];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int rows = min(16, total - w0 - 16 * t);
        for (int i = 0; i < rows; ++i) {
            const int r = w0 + 16 * t + i;
            const float m = __shfl(R.m[t], i);
            const float l = __shfl(R.lim[t], i) < 0 ? 0.0f : __shfl(lsum, i);
            float o[HD / 64];
#pragma unroll
            for (int e = 0; e < HD / 64; ++e) o[e] = po[i * OST + lane + 64 * e];
            if (nch == 1) {
                put_row<HD, KV>(a, b, it.sq, r >> a.lg, (g << a.lg) + (r & ((1 << a.lg) - 1)), o,
                                l);
            } else {
                const int to = ((it.rec + it.chunk) * a.pg.n_kv + g) * MT + r - r0;
                if (to < a.rec_rows) {
                    float* rec = a.rec + (size_t)to * (HD + 4);
                    if (lane == 0) {
                        rec[0] = m;
                        rec[1] = l;
                    }
#pragma unroll
                    for (int e = 0; e < HD / 64; ++e) rec[4 + lane + 64 * e] = o[e];
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- the chunks' records of a row and head, merged: a workgroup a row and head ----
template <int HD, typename KV>
__global__ __launch_bounds__(256) void k_pa_join(PaArgs a, int mt) {
    constexpr int E = HD / QLM_WAVE, NW = 4;
    __shared__ float pm[NW], pl[NW], po[NW][HD];
    const int row = blockIdx.x, h = blockIdx.y, g = h >> a.lg, lane = threadIdx.x & 63;
    const int wave = threadIdx.x / QLM_WAVE;
    const int2 d = a.desc[(size_t)row * a.pg.n_kv + g];
    const int b = seq_of_row(a.bt, row);
    if (b < 0) return;
    const SeqRows sq = seq_rows(a.bt, b);
    const int i = row - sq.first, nch = d.y;
    if (i < 0 || i >= sq.n || nch <= 1) return;
    const long long stride = (long long)a.pg.n_kv * mt;
    const long long base = (long long)d.x + (h & ((1 << a.lg) - 1));
    if (d.x < 0 || base + (nch - 1) * stride >= a.rec_rows) return;
    float m = -INFINITY, l = 0.0f, o[E] = {};
    // four records a wave in flight
    for (int c0 = wave; c0 < nch; c0 += 4 * NW) {
        float rm[4], rl[4], ro[4][E];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = min(c0 + u * NW, nch - 1);
            const float* rec = a.rec + (size_t)(base + c * stride) * (HD + 4);
            rm[u] = rec[0];
            rl[u] = rec[1];
#pragma unroll
            for (int e = 0; e < E; ++e) ro[u][e] = rec[4 + lane + 64 * e];
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < 4; ++u) top = fmaxf(top, rm[u]);
        const float ref = top == -INFINITY ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(m - ref);
        l *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (c0 + u * NW >= nch) break;
            const float w = __builtin_amdgcn_exp2f(rm[u] - ref);
            l = fmaf(rl[u], w, l);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(ro[u][e], w, o[e]);
        }
        m = top;
    }
    if (lane == 0) {
        pm[wave] = m;
        pl[wave] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) po[wave][lane + 64 * e] = o[e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, pm[w]);
    const float ref = m == -INFINITY ? 0.0f : m;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(pm[w] - ref);
        l = fmaf(pl[w], f, l);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(po[w][lane + 64 * e], f, o[e]);
    }
    put_row<HD, KV>(a, b, sq, i, h, o, l);
}

// ---- the host's part ----

struct PaPlan {
    int mt;              // rows of a unit: 8, 16 (k_pa_few), 64 or 128 (k_pa_tile)
    int target;          // items a kv head to cut the keys into
    int items;           // at most
    int rec_rows;        // records
    bool join;           // some unit may have several chunks
    size_t desc_at, bytes;
};

PaPlan plan_of(int rows, int B, int G, int n_kv, int hd, long long slots) {
    PaPlan p{};
    // about the rows of a sequence
    const long long per = ((long long)rows * G + B - 1) / B;
    p.mt = per <= 8 ? 8 : per <= 16 ? 16 : per <= 64 ? 64 : 128;
    const int wanted = p.mt <= 16 ? 512 : 512;
    p.target = std::max(1, wanted / n_kv);
    const long long units = ((long long)rows * G) / p.mt + B;
    p.items = (int)(units + p.target);
    p.join = slots > kMinChunk;
    if (p.join) p.rec_rows = 2 * p.target * n_kv * p.mt;
    const size_t rec = (size_t)p.rec_rows * (hd + 4) * sizeof(float);
    p.desc_at = rec;
    p.bytes = p.join ? rec + (size_t)rows * n_kv * sizeof(int2) : 0;
    return p;
}

bool pa_shape(int rows, int B, int n_q, int n_kv, int hd, long long slots) {
    if (rows <= 0 || B <= 0 || n_q <= 0 || n_kv <= 0 || slots <= 0) return false;
    if (rows > kMaxBatchRows || B > 65535 || n_kv > 1024 || slots > 1LL << 30) return false;
    if ((hd != 128 && hd != 256) || n_q % n_kv != 0) return false;
    const int G = n_q / n_kv;
    return G == 1 || G == 2 || G == 4 || G == 8;
}

// Workgroups of a launch: whole groups of 8, one an XCD, where the heads are
// dealt out that way.
long long groups_of(int items, int n_kv) {
    if (n_kv > 8 || (n_kv & (n_kv - 1)) != 0) return (long long)items * n_kv;
    const int per = 8 / n_kv;
    return ((long long)items + per - 1) / per * 8;
}

template <int HD, bool F32>
int launch_attention(const PaArgs& a, const PaPlan& p, hipStream_t st) {
    using KV = typename std::conditional<F32, float, uint16_t>::type;
    const dim3 grid((unsigned)groups_of(p.items, a.pg.n_kv));
    if (p.mt == 8)
        hipLaunchKernelGGL((k_pa_few<HD, F32, true>), grid, dim3(FewShape<HD, F32>::NW * QLM_WAVE),
                           0, st, a);
    else if (p.mt == 16)
        hipLaunchKernelGGL((k_pa_few<HD, F32, false>), grid, dim3(FewShape<HD, F32>::NW * QLM_WAVE),
                           0, st, a);
    else if (p.mt == 64)
        hipLaunchKernelGGL((k_pa_tile<HD, F32, 1>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_pa_tile<HD, F32, 2>), grid, dim3(256), 0, st, a);
    const int rc = qlm_launch_status();
    if (rc != QLM_OK || !p.join) return rc;
    hipLaunchKernelGGL((k_pa_join<HD, KV>), dim3(a.bt.rows, a.n_q), dim3(256), 0, st, a, p.mt);
    return qlm_launch_status();
}

}  // namespace

extern "C" size_t qlm_paged_attention_workspace_bytes(int rows, int B, int n_q, int n_kv, int hd,
                                                      long long slots) {
    if (!pa_shape(rows, B, n_q, n_kv, hd, slots)) return 0;
    return plan_of(rows, B, n_q / n_kv, n_kv, hd, slots).bytes;
}

extern "C" int qlm_paged_attention(const float* q, int ldq, const qlm_row_batch* batch,
                                   const qlm_kv_pages* pages, const float* gate, int ldg,
                                   int gate_stride, float* out, int ldo, int n_q, void* work,
                                   size_t work_bytes, void* stream) {
    int rc = check_row_batch(batch);
    if (rc == QLM_OK) rc = check_kv_pages(pages);
    if (rc != QLM_OK) return rc;
    if (!q || !out || q == out || n_q <= 0) return QLM_ERR_ARG;
    const int hd = pages->hd, n_kv = pages->n_kv;
    const long long slots = (long long)pages->ld_table * pages->page_size;
    if (!pa_shape(batch->rows, batch->B, n_q, n_kv, hd, slots)) return QLM_ERR_SHAPE;
    if (ldq < n_q * hd || ldo < n_q * hd) return QLM_ERR_SHAPE;
    if (gate && (gate_stride < hd || ldg < (n_q - 1) * gate_stride + hd)) return QLM_ERR_SHAPE;
    const int G = n_q / n_kv;
    const PaPlan p = plan_of(batch->rows, batch->B, G, n_kv, hd, slots);
    if (groups_of(p.items, n_kv) >= 1LL << 24) return QLM_ERR_SHAPE;  // a launch's threads fit 32 bits
    if (p.bytes > 0 && (!work || work_bytes < p.bytes)) return QLM_ERR_ARG;
    if ((uintptr_t)work & 15u) return QLM_ERR_SHAPE;
    PaArgs a{};
    a.q = q;
    a.gate = gate;
    a.out = out;
    a.rec = p.join ? reinterpret_cast<float*>(work) : nullptr;
    a.desc = p.join ? reinterpret_cast<int2*>(reinterpret_cast<char*>(work) + p.desc_at) : nullptr;
    a.ldq = ldq;
    a.ldg = ldg;
    a.ldo = ldo;
    a.gate_stride = gate_stride;
    a.n_q = n_q;
    while ((1 << a.lg) < G) ++a.lg;
    a.target = p.target;
    a.items = p.items;
    a.rec_rows = p.rec_rows;
    a.slots = (int)slots;
    a.qscale = 1.44269504088896341f / sqrtf((float)hd);
    a.bt = *batch;
    a.pg = *pages;
    hipStream_t st = as_stream(stream);
    if (hd == 128)
        return pages->dtype == 0 ? launch_attention<128, true>(a, p, st)
                                 : launch_attention<128, false>(a, p, st);
    return pages->dtype == 0 ? launch_attention<256, true>(a, p, st)
                             : launch_attention<256, false>(a, p, st);
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_paged_attention() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>((k_pa_join<128, float>)));
}
