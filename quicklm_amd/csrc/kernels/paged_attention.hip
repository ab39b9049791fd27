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
// With a bf16 cache queries and probabilities, fp32, are split into three bf16
// terms, x = h + m + l (24 bits: exact), a product each, so that nothing is lost
// but in the fp32 sums; two terms, two thirds of the products, left 5e-6 of the
// result, five times what fp32 arithmetic does. Up to 8 rows take two products:
// rows 0..7 of the tile hold the h terms and rows 8..15 the m terms, then the l
// terms and zeros, and the halves are added. An fp32 cache's keys and values are
// split likewise: six products of terms (the three others are below 2^-25 of the
// whole), which the rows of a tile of 64 share the splitting for; the fp32 matrix
// cores (16x16x4), a sixteenth of the rate, took 503 us where this takes 326 (2048
// rows after 2048, 16 / 4 heads of 128) and 977 where this takes 626 (16 / 2 of
// 256), and with the splitting in every wave 482 and 908. Up to 16 rows a unit
// stay on them, bound by the cache's bytes all the same.
//
// Keys and values go straight from the pages to LDS. A 16-key group lies in one
// page and is read through a buffer descriptor that ends where the group's
// slots do, so that slots behind the last key arrive as zeros, whatever lies
// there, and a page number that is out of range reads nothing. 16-byte piece c of
// a row sits at piece c ^ (key % 16), which spreads the 16 rows that an LDS
// access touches over all banks.
//
// Lengths are known on the device alone. Each workgroup reads them, forms the
// chunk length that cuts all sequences' keys into about `target` items a kv head,
// and finds its own; a launch has room for as many as there can be. A unit of
// more than one chunk leaves records [m, l, O] that k_pa_join merges; the others
// write their outputs.
//
// Measured with 16 / 4 heads of 128, bf16, calls one after the other: 64 single
// tokens after 256 to 8192 slots 107 us, HBM (5.2 TB/s; 5.1 when something else has
// been read in between, 6.1 for 64 after 32768, 4.3 GB); 2048 rows after 2048 148 us,
// matrix cores (1050 TFLOP/s of bf16 products, half of their cycles in the key
// loop); 8 trees of 64 nodes after 4032 62, 74 with the keys out of HBM, of which 13
// are the start and the join; one token after 600 11 us, latency.

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
    int target, least, alone;  // items to cut a kv head's keys into; keys of an item, at
                               // least; of a batch's longest sequence that is not cut
    int items, rec_rows, slots;
    float qscale;  // log2(e) / sqrt(hd)
    qlm_row_batch bt;
    qlm_kv_pages pg;
};

// a value that is the same in all lanes, in a scalar register
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ---- which work a workgroup does ----

struct Item {
    SeqRows sq;
    int b, tile, chunk;  // chunk: which
    int len;             // keys of a chunk
    int rec;             // the unit's first record block
};

__device__ __forceinline__ int tiles_of(int n, int lg, int mt) {
    return (int)((((long long)n << lg) + mt - 1) / mt);
}

// new rows that any row can see
__device__ __forceinline__ int seen_rows(const PaArgs& a, const SeqRows& s) {
    return a.bt.parent ? min(s.n, QLM_TREE_MAX) : s.n;
}

// Sums over the lanes up to each (DPP: shifts within rows of 16, then the rows'
// last lanes to the rows behind).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return v;
}

// Sequences that are all about as long are cut so that every CU has one item: 64
// single tokens after 4096 slots 99 us (16 / 4 heads of 128, bf16), in twice as
// many 104; one after 32768 26 and 36. Where the longest is well above the mean
// one item a CU leaves most of them waiting for it: half as many items again, 64
// after 256 to 8192 slots 108 us, 121 without, 120 with twice as many; 16 after up to
// 30000 110 and 135, 8 51 and 62 (128 after up to 4000, where the rounds of items
// come out otherwise, 121 and 116). All equally long and cut like that: 64 after
// 4096 104 for 99, one after 32768 33 for 26.
constexpr float kUneven = 2.0f / 3.0f;

// Item `want` of a kv head, counted over the sequences: the longest prompts'
// last tiles, which see the most keys, first. Every lane gets it. Sums that
// only say how long a chunk is are in fp32, the same in every wave.
template <int MT>
__device__ __forceinline__ bool find_item(const PaArgs& a, int want, Item& it) {
    const int lane = threadIdx.x & (QLM_WAVE - 1), B = a.bt.B;
    float cost = 0.0f, longest = 0.0f, units = 0.0f;
    SeqRows s{};
    for (int i = 0; i < B; i += QLM_WAVE) {
        s = seq_rows(a.bt, min(i + lane, B - 1));
        if (i + lane >= B) s.n = 0;
        if (s.n > 0) {
            const float keys = (float)min(s.ctx + seen_rows(a, s), a.slots);
            const float tiles = (float)tiles_of(s.n, a.lg, MT);
            cost += tiles * keys;
            units += tiles;
            longest = fmaxf(longest, keys);
        }
    }
    cost = wave_sum(cost);
    longest = wave_max(longest);
    float share = cost / (float)a.target;
    if (MT <= 16 && longest * wave_sum(units) > 1.5f * cost) share *= kUneven;
    // (no context is longer than 2^30: what `target` has no room for stays uncut)
    int len = uni(min((int)fminf(share, (float)(1 << 30)) / 32 * 32 + 32, 1 << 30));
    len = uni(max(len, longest <= (float)a.alone ? a.alone : a.least));
    int before = 0, rec = 0;
    for (int i = 0; i < B; i += QLM_WAVE) {
        if (B > QLM_WAVE) {
            s = seq_rows(a.bt, min(i + lane, B - 1));
            if (i + lane >= B) s.n = 0;
        }
        int items = 0, recs = 0, keys = 0;
        if (s.n > 0) {
            keys = min(s.ctx + seen_rows(a, s), a.slots);
            const int nch = (keys - 1) / len + 1;
            items = tiles_of(s.n, a.lg, MT) * nch;
            recs = nch > 1 ? items : 0;
        }
        const int ic = wave_scan(items), rc = wave_scan(recs);
        const unsigned long long at = __ballot(before + ic > want);
        if (at) {
            const int w = __ffsll((long long)at) - 1;
            auto of = [&](int x) { return __builtin_amdgcn_readlane(x, w); };
            it.b = i + w;
            it.sq = SeqRows{of(s.first), of(s.n), of(s.ctx)};
            const int mine = want - before - of(ic - items);
            const int tiles = tiles_of(it.sq.n, a.lg, MT), nch = of(items) / tiles;
            it.len = ((of(keys) + nch - 1) / nch + 31) / 32 * 32;  // all about as long
            it.chunk = mine % nch;
            it.tile = tiles - 1 - mine / nch;
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
    const int p = uniform_load(a.pg.table, (size_t)b * a.pg.ld_table + (in ? i : 0));
    Group g;
    g.valid = uni(in && (unsigned)p < (unsigned)a.pg.n_pages ? min(end - slot, 16) : 0);
    g.page = uni(g.valid > 0 ? p : 0);
    return g;
}

// A 16-key group in LDS: rows as they are in the page, 16-byte pieces swizzled.
template <int HD, bool F32>
struct Lay {
    static constexpr int ROW = HD * (F32 ? 4 : 2);  // bytes of a row
    static constexpr int GRP = 16 * ROW;
    static constexpr int LOADS = GRP / 1024;  // a wave's loads of a group
    // the lane's source offset of load j
    __device__ static __forceinline__ int src(int j) {
        const int lane = threadIdx.x & (QLM_WAVE - 1);
        constexpr int PPR = ROW / 16;  // pieces of a row
        const int row = (j * QLM_WAVE + lane) / PPR, piece = (j * QLM_WAVE + lane) % PPR;
        return row * ROW + ((piece ^ row) * 16);
    }
};

// A head's group in a pool, ending where its slots do.
template <int HD, bool F32>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t group_rsrc(const PaArgs& a, const void* pool,
                                                             const Group& gr, int g, int slot) {
    constexpr int SIZE = F32 ? 4 : 2;
    const size_t at = (((size_t)gr.page * a.pg.n_kv + g) * a.pg.page_size +
                       (slot & (a.pg.page_size - 1))) * (HD * SIZE);
    return make_rsrc(reinterpret_cast<const char*>(pool) + at, (unsigned)gr.valid * (HD * SIZE));
}

// Loads J0 .. J0 + N - 1 of a group.
template <int HD, bool F32, int N = Lay<HD, F32>::LOADS>
__device__ __forceinline__ void fetch_group(const PaArgs& a, const void* pool, const Group& gr,
                                            int g, int slot, char* to, int j0 = 0) {
    using L = Lay<HD, F32>;
    const __amdgpu_buffer_rsrc_t r = group_rsrc<HD, F32>(a, pool, gr, g, slot);
#pragma unroll
    for (int j = 0; j < N; ++j) load_to_lds(r, to + (j0 + j) * 1024, L::src(j0 + j), 0);
}

// LDS by its own 32-bit addresses
__device__ __forceinline__ uint32_t lds_at(const char* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
template <typename T>
__device__ __forceinline__ T lds_read(uint32_t at) {
    return *(__attribute__((address_space(3))) const T*)(uintptr_t)at;
}
template <typename T>
__device__ __forceinline__ void lds_write(uint32_t at, T v) {
    *(__attribute__((address_space(3))) T*)(uintptr_t)at = v;
}

// N floats (four, eight) as three bf16 terms each (24 bits: exact). What a term
// leaves is x - h, exact: one product with -1 and its sum with x (v_dot2_f32_bf16)
// instead of widening h and subtracting it.
template <int N, typename V>
__device__ __forceinline__ void split_terms(const float (&x)[N], V (&term)[3]) {
    // (-1, 0) and (0, -1); in registers, since the compiler writes the second as the
    // inline constant -1.0, which the instruction does not read as that pair
    unsigned c0 = 0x0000bf80u, c1 = 0xbf800000u;
    asm("" : "+v"(c0), "+v"(c1));
    const bf16x2 first = __builtin_bit_cast(bf16x2, c0), second = __builtin_bit_cast(bf16x2, c1);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        f32x2 v = {x[2 * i], x[2 * i + 1]};
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const bf16x2 w = __builtin_convertvector(v, bf16x2);
            term[k][i] = __builtin_bit_cast(unsigned, w);
            v.x = __builtin_amdgcn_fdot2_f32_bf16(w, first, v.x, false);
            v.y = __builtin_amdgcn_fdot2_f32_bf16(w, second, v.y, false);
        }
    }
}

// ---- a wave's rows ----

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// over the four lane groups of a column
__device__ __forceinline__ float cols_max(float v) { return xor32_max(xor16_max(v)); }
__device__ __forceinline__ float cols_sum(float v) { return xor32_add(xor16_add(v)); }

// v(l) + v(l ^ 8) of each 16 lanes
__device__ __forceinline__ float fold8(float v) { return v + dpp_mov<0x128>(v); }  // row_ror:8

// How products are formed: of a bf16 cache; of an fp32 cache on the fp32 matrix
// cores; of an fp32 cache whose keys and values lie in LDS as three bf16 terms.
enum Math { kBf16, kF32, kSplit };

// Split keys (or values) of a block, 4096 elements: planes of their h, m and l terms.
constexpr int kPlane = 4096 * 2;

// Keys go through in parts of NH 16-key halves; a lane has XN scores of a row.
template <bool F32>
struct Part {
    static constexpr int NH = F32 ? 1 : 2, XN = 4 * NH, KEYS = 16 * NH;
};

// RT tiles of 16 rows; PACK: one tile of 8 rows (bf16: h and m terms side by side,
// then l terms and zeros).
// A row's scores come out of the products relative to a reference `m` (the
// accumulators begin at -m): the largest score of the row's first part, and of
// a later one where a score passes it by more than kRise. So exponentials go
// up to 2^kRise, sums over 2^30 keys stay in range, and what is lost below 2^-126
// is less than that part of the row's largest; no part needs a maximum over
// the lanes, and the sums are hardly ever scaled. A part that moves a reference
// is begun again (the loops below): with the scaling inside of the loop's body
// its registers were copied every time, a third of its vector instructions.
constexpr float kRise = 60.0f;
constexpr int kAnyScore = (int)0x80000000;
template <int HD, int RT, bool PACK, Math M>
struct Rows {
    static constexpr int KS = HD / 32, CB = HD / 16, QT = PACK ? 2 : 3;
    u32x4 q[M == kF32 ? 1 : RT][M == kF32 ? 1 : QT][M == kF32 ? 1 : KS];
    // lane (qd, n): elements 16 s + 4 qd .. + 3
    f32x4 qf[M == kF32 ? RT : 1][M == kF32 ? HD / 16 : 1];
    f32x4 acc[RT][CB];
    f32x4 from[RT];       // four times -m
    float m[RT], l[RT];   // m -inf: no score yet
    int high[RT];         // bits of the relative score that moves it: kRise, at first any
    int lim[RT];  // slots below this one are seen; -1: a row outside the tree
    unsigned long long line[RT];  // new rows seen beside those
    unsigned long long unseen;    // new rows that no row sees, the same in all lanes
};

// Query rows r0 + 16 t + n of the unit (r: its token and head): requested here.
// (bf16 cores: elements 32 s + 8 qd .. + 7; fp32: 16 s + 4 qd .. + 3.)
template <int HD, int RT>
struct Queries {
    f32x4u x[RT][HD / 16];
};
template <int HD, int RT, bool PACK, Math M>
__device__ __forceinline__ void request_rows(const PaArgs& a, const Item& it, int g, int r0,
                                             Queries<HD, RT>& Q) {
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15, qd = lane >> 4;
    const int total = it.sq.n << a.lg;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int rc = min(r0 + 16 * t + (PACK ? n & 7 : n), total - 1);
        const float* qr = a.q + (size_t)(it.sq.first + (rc >> a.lg)) * a.ldq +
                          ((size_t)(g << a.lg) + (rc & ((1 << a.lg) - 1))) * HD;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
            const int e = M == kF32 ? 16 * s + 4 * qd : 32 * (s / 2) + 8 * qd + 4 * (s % 2);
            Q.x[t][s] = *reinterpret_cast<const f32x4u*>(qr + e);
        }
    }
}

// What the rows see, and their queries' terms. parent: of the sequence's row `lane`,
// requested ahead of the keys (loads come back in order).
template <int HD, int RT, bool PACK, Math M>
__device__ __forceinline__ void take_rows(const PaArgs& a, const Item& it, int r0, int parent,
                                          const Queries<HD, RT>& Q, Rows<HD, RT, PACK, M>& R) {
    using T = Rows<HD, RT, PACK, M>;
    const int n = threadIdx.x & 15;
    const int total = it.sq.n << a.lg;
    unsigned long long mine = 0;
    R.unseen = 0;
    if (a.bt.parent) {
        mine = tree_line(parent);
        R.unseen = __ballot((int)(threadIdx.x & (QLM_WAVE - 1)) < it.sq.n && mine == 0);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int tok = min(r0 + 16 * t + (PACK ? n & 7 : n), total - 1) >> a.lg;
        R.m[t] = -INFINITY;
        R.l[t] = 0.0f;
        R.from[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        R.high[t] = kAnyScore;
        R.lim[t] = it.sq.ctx + tok + 1;
        R.line[t] = 0;
        if (a.bt.parent) {
            const int at = min(tok, QLM_TREE_MAX - 1);
            const unsigned long long ln = (unsigned long long)__shfl((unsigned)(mine >> 32), at)
                                              << 32 | __shfl((unsigned)mine, at);
            R.line[t] = tok < QLM_TREE_MAX ? ln : 0;
            R.lim[t] = R.line[t] ? it.sq.ctx : -1;
        }
        if constexpr (M == kF32) {
#pragma unroll
            for (int s = 0; s < HD / 16; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) R.qf[t][s][i] = Q.x[t][s][i] * a.qscale;
        } else {
#pragma unroll
            for (int s = 0; s < T::KS; ++s) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = Q.x[t][2 * s + i / 4][i % 4] * a.qscale;
                u32x4 term[3];
                split_terms(v, term);
                if constexpr (PACK) {
                    R.q[t][0][s] = n < 8 ? term[0] : term[1];
                    R.q[t][1][s] = n < 8 ? term[2] : u32x4{0u, 0u, 0u, 0u};
                } else {
#pragma unroll
                    for (int k = 0; k < 3; ++k) R.q[t][k][s] = term[k];
                }
            }
        }
#pragma unroll
        for (int c = 0; c < T::CB; ++c) R.acc[t][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// Keeps the compiler from holding what it derives from x over the loop: with heads
// of 256 the addresses of every piece, 24 registers, drove queries into scratch.
template <int HD>
__device__ __forceinline__ void fresh(uint32_t& x) {
    if constexpr (HD > 128) asm volatile("" : "+v"(x));
}

// Zeros over the values of new rows that no row sees, of the part from slot k0 on
// at vp. A padding row's slot is never written, and a probability of 0 times a NaN
// that happens to lie there would be one. Waves that share the part all write
// these zeros, each before it reads them.
template <int HD, Math M>
__device__ __forceinline__ void clear_unseen(unsigned long long unseen, const char* vp, int k0,
                                             int ctx) {
    using L = Lay<HD, M == kF32>;
    constexpr int KEYS = Part<M != kBf16>::KEYS;
    const int r0 = k0 - ctx;  // the part's first slot as a new row
    if (unseen == 0 || r0 <= -KEYS || r0 >= QLM_TREE_MAX) return;
    unsigned left = (unsigned)(r0 < 0 ? unseen << -r0 : unseen >> r0);
    left &= 0xffffffffu >> (32 - KEYS);
    uint32_t at = lds_at(vp) + (threadIdx.x & (QLM_WAVE - 1)) * 4, zero = 0u;
    asm volatile("" : "+v"(at), "+v"(zero));  // (not held over the loop either)
    for (; left; left &= left - 1) {
        const uint32_t row = at + (__ffs((int)left) - 1) * L::ROW;
#pragma unroll
        for (int p = 0; p < (M == kSplit ? 3 : 1); ++p)
#pragma unroll
            for (int e = 0; e < L::ROW; e += 4 * QLM_WAVE)
                lds_write(row + p * kPlane + e, zero);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// Scores of a part of the keys, from slot k0 on, relative to the references, of
// keys that a row does not see -inf: x[t][4 h + i] of key 16 h + 4 qd + i. kp, vp:
// its K and V groups in LDS. `all`: every row sees every key of it. False: none of its
// slots is there.
template <int HD, int RT, bool PACK, Math M>
__device__ __forceinline__ bool scores(const Rows<HD, RT, PACK, M>& R, const char* kp,
                                       const char* vp, int k0, int ctx, int valid0, int valid1,
                                       bool all, float (&x)[RT][Part<M != kBf16>::XN]) {
    using T = Rows<HD, RT, PACK, M>;
    using L = Lay<HD, M == kF32>;
    constexpr int NH = Part<M != kBf16>::NH, XN = Part<M != kBf16>::XN;
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15, qd = lane >> 4;
    f32x4 s[NH][RT];
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int t = 0; t < RT; ++t) s[h][t] = R.from[t];
    // piece (4 k + qd) ^ n of row n: the bits of k come in by an exclusive or
    uint32_t ka = lds_at(kp) + n * L::ROW + ((qd ^ n) * 16);
    if constexpr (M == kSplit) {
        fresh<HD>(ka);
        // of the nine products of terms the last three are below 2^-25; two sums,
        // whose products take turns
        f32x4 other[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) other[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < T::KS; k += 2) {
            u32x4 kt[2][3];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    kt[e][p] = lds_read<u32x4>((ka ^ (64u * (k + e))) + p * kPlane);
#pragma unroll
            for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                for (int p = 0; p <= sum; ++p)
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        s[0][t] = mfma(kt[0][sum - p], R.q[t][p][k], s[0][t]);
                        other[t] = mfma(kt[1][sum - p], R.q[t][p][k + 1], other[t]);
                    }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) s[0][t] += other[t];
    } else {
        constexpr int KN = L::ROW / 64;         // pieces of a row a lane
        constexpr int KC = KN < 4 ? KN : 4;     // read at once
#pragma unroll
        for (int k0s = 0; k0s < KN; k0s += KC) {
            u32x4 kf[KC][NH];
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int h = 0; h < NH; ++h)
                    kf[k][h] = lds_read<u32x4>((ka ^ (64u * (k0s + k))) + h * L::GRP);
            __builtin_amdgcn_sched_barrier(0);
            // (a sum's terms apart from each other: each waits for the one before)
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                if constexpr (M == kF32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int t = 0; t < RT; ++t)
                            s[0][t] = mfma(__uint_as_float(kf[k][0][i]), R.qf[t][k0s + k][i],
                                           s[0][t]);
                } else {
#pragma unroll
                    for (int p = T::QT - 1; p >= 0; --p)
#pragma unroll
                        for (int h = 0; h < NH; ++h)
#pragma unroll
                            for (int t = 0; t < RT; ++t)
                                s[h][t] = mfma(kf[k][h], R.q[t][p][k0s + k], s[h][t]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < XN; ++j) {
            x[t][j] = s[j / 4][t][j % 4];
            if constexpr (PACK && M == kBf16) x[t][j] = fold8(x[t][j]);
        }
    if (all) return true;
    asm volatile("");  // (a branch, not selections that every part would compute)
    if ((valid0 | valid1) == 0) return false;
    clear_unseen<HD, M>(R.unseen, vp, k0, ctx);
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < XN; ++j) {
            const int in = 4 * qd + j % 4, slot = k0 + 16 * (j / 4) + in, row = slot - ctx;
            bool sees = slot < R.lim[t];
            if (row >= 0 && row < QLM_TREE_MAX) sees |= (R.line[t] >> row) & 1ull;
            sees &= in < (j < 4 ? valid0 : valid1);
            x[t][j] = sees ? x[t][j] : -INFINITY;
        }
    return true;
}

// Whether some score is too far above its row's reference.
template <int HD, int RT, bool PACK, Math M>
__device__ __forceinline__ bool too_high(const Rows<HD, RT, PACK, M>& R,
                                         const float (&x)[RT][Part<M != kBf16>::XN]) {
    bool high = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        // as integers, in whose order positive floats are: no canonical forms
        int top = __float_as_int(x[t][0]);
#pragma unroll
        for (int j = 1; j < Part<M != kBf16>::XN; ++j) top = max(top, __float_as_int(x[t][j]));
        high |= top > R.high[t];
    }
    return __ballot(high) != 0;
}

// Moves the references to the part's largest scores where those are higher.
template <int HD, int RT, bool PACK, Math M>
__device__ __forceinline__ void raise(Rows<HD, RT, PACK, M>& R,
                                      const float (&x)[RT][Part<M != kBf16>::XN]) {
    using T = Rows<HD, RT, PACK, M>;
    const int n = threadIdx.x & 15;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float top = x[t][0];
#pragma unroll
        for (int j = 1; j < Part<M != kBf16>::XN; ++j) top = fmaxf(top, x[t][j]);
        top = cols_max(top);
        const bool first = R.m[t] == -INFINITY;
        const bool moves = top > (first ? -INFINITY : 0.0f);
        const float by = moves ? top : 0.0f;
        const float f = first ? 0.0f : __builtin_amdgcn_exp2f(-by);
        R.m[t] = moves ? (first ? 0.0f : R.m[t]) + by : R.m[t];
        R.l[t] *= f;
#pragma unroll
        for (int c = 0; c < T::CB; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) R.acc[t][c][i] *= f;
        // (a packed tile's two halves are added: one of them begins at 0)
        const float from = moves && !(PACK && M == kBf16 && n >= 8) ? -R.m[t] : R.from[t][0];
        R.from[t] = f32x4{from, from, from, from};
        // a row that has seen nothing in the part waits for its first score
        R.high[t] = R.m[t] == -INFINITY ? kAnyScore : __float_as_int(kRise);
    }
}

// The part's probabilities into the rows' sums; vp: its V groups in LDS.
template <int HD, int RT, bool PACK, Math M>
__device__ __forceinline__ void accumulate(Rows<HD, RT, PACK, M>& R,
                                           float (&x)[RT][Part<M != kBf16>::XN], const char* vp) {
    using T = Rows<HD, RT, PACK, M>;
    using L = Lay<HD, M == kF32>;
    constexpr int XN = Part<M != kBf16>::XN;
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15, qd = lane >> 4;
    auto exponentials = [&](int t) {
#pragma unroll
        for (int j = 0; j < XN; ++j) x[t][j] = __builtin_amdgcn_exp2f(x[t][j]);
        float sum = (x[t][0] + x[t][1]) + (x[t][2] + x[t][3]);
        if constexpr (XN == 8) sum += (x[t][4] + x[t][5]) + (x[t][6] + x[t][7]);
        R.l[t] += sum;
    };
    if constexpr (M == kF32) {
        // step i: keys 4 qd + i; lane (qd, n) reads element 16 c + n of its key, in
        // piece (4 c + n / 4) ^ key: 64 banks once
        uint32_t va[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            va[i] = lds_at(vp) + (4 * qd + i) * L::ROW + (((n >> 2) ^ (4 * qd + i)) * 16) +
                    (n & 3) * 4;
        constexpr int VC = 8;
        float v[4][VC];
        auto read_some = [&](int c0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < VC; ++c) v[i][c] = lds_read<float>(va[i] ^ (64u * (c0 + c)));
        };
        read_some(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < RT; ++t) exponentials(t);
#pragma unroll
        for (int c0 = 0; c0 < T::CB; c0 += VC) {
            if (c0) read_some(c0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int t = 0; t < RT; ++t)
                        R.acc[t][c0 + c] = mfma(v[i][c], x[t][i], R.acc[t][c0 + c]);
        }
    } else {
        // V^T: lane l of a group reads 4 columns of key 4 qd + (l % 16) / 4
        const int key = 4 * qd + (n >> 2);
        uint32_t va =
            lds_at(vp) + key * L::ROW + ((((n >> 1) & 1) ^ key) * 16) + (n & 1) * 8;
        auto tr = [&](uint32_t at) {
            return __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (__attribute__((address_space(3))) s16x4*)(uintptr_t)at));
        };
        if constexpr (M == kSplit) {
            // the eight k-slots of a lane group are its four keys twice, so that a
            // product of 32 slots takes two pairs of terms: (h, m) with the
            // probabilities' (h, h) and (m, m), (l, h) with (h, l)
            constexpr int VC = 4;
            fresh<HD>(va);
            u32x2 v[3][VC];
            auto read_some = [&](int c0) {
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        v[p][c] = tr((va ^ (32u * (c0 + c))) + p * kPlane);
            };
            read_some(0);
            __builtin_amdgcn_sched_barrier(0);
            u32x4 p[RT][3];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                exponentials(t);
                u32x2 w[3];
                split_terms(x[t], w);
                p[t][0] = u32x4{w[0].x, w[0].y, w[0].x, w[0].y};
                p[t][1] = u32x4{w[1].x, w[1].y, w[1].x, w[1].y};
                p[t][2] = u32x4{w[0].x, w[0].y, w[2].x, w[2].y};
            }
#pragma unroll
            for (int c0 = 0; c0 < T::CB; c0 += VC) {
                if (c0) read_some(c0);
#pragma unroll
                for (int k = 2; k >= 0; --k)
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        const u32x2 a = v[k == 2 ? 2 : 0][c], b = v[k == 2 ? 0 : 1][c];
#pragma unroll
                        for (int t = 0; t < RT; ++t)
                            R.acc[t][c0 + c] =
                                mfma(u32x4{a.x, a.y, b.x, b.y}, p[t][k], R.acc[t][c0 + c]);
                    }
            }
            return;
        }
        constexpr int VC = 4;  // column blocks read at once, the first before the exponentials
        u32x4 v[VC];
        auto read_some = [&](int c0) {  // piece (2 c + ..) ^ key of row `key`
#pragma unroll
            for (int c = 0; c < VC; ++c) {
                const uint32_t at = va ^ (32u * (c0 + c));
                const u32x2 v0 = tr(at), v1 = tr(at + L::GRP);
                v[c] = u32x4{v0.x, v0.y, v1.x, v1.y};
            }
        };
        read_some(0);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 p[RT][3];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            exponentials(t);
            split_terms(x[t], p[t]);
            if constexpr (PACK) {
                p[t][0] = n < 8 ? p[t][0] : p[t][1];
                p[t][1] = n < 8 ? p[t][2] : u32x4{0u, 0u, 0u, 0u};
            }
        }
#pragma unroll
        for (int c0 = 0; c0 < T::CB; c0 += VC) {
            if (c0) read_some(c0);
#pragma unroll
            for (int k = T::QT - 1; k >= 0; --k)
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int t = 0; t < RT; ++t)
                        R.acc[t][c0 + c] = mfma(v[c], p[t][k], R.acc[t][c0 + c]);
        }
    }
}

// ---- outputs ----

// Head h of row i of a sequence in fp32, key after key, by a whole wave: for
// results that did not come out finite. What a row does not see is not
// touched here, so that only its own keys and values can make it NaN. About half a
// microsecond a key, a wave's rows in turn: one token after 4000 slots 2.7 ms, 8 trees
// of 64 after 4032 5.8, a prompt of 2048 rows after 2048 42.
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
    const int size = a.pg.page_size;
    // 64 pages' numbers at a time: those that are not there cost nothing else
    for (int p0 = 0; p0 * (long long)size < end; p0 += QLM_WAVE) {
        const int mine = page_of(a.pg, b, (p0 + lane) * size);
        for (unsigned long long left = __ballot(mine >= 0); left; left &= left - 1) {
            const int w = __ffsll((long long)left) - 1, s0 = (p0 + w) * size;
            const int page = __builtin_amdgcn_readlane(mine, w);
            for (int s = s0; s < min(s0 + size, end); ++s) {
                if (a.bt.parent && s >= sq.ctx && !(line >> (s - sq.ctx) & 1ull)) continue;
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
        }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = any ? o[j] / l : 0.0f;
}

// The gate of a row and head, requested ahead of its use (element lane + 64 j).
template <int HD>
__device__ __forceinline__ void load_gate(const PaArgs& a, const SeqRows& sq, int i, int h,
                                          float (&g)[HD / QLM_WAVE]) {
    if (!a.gate) return;
    const float* p = a.gate + (size_t)(sq.first + i) * a.ldg + (size_t)h * a.gate_stride +
                     (threadIdx.x & (QLM_WAVE - 1));
#pragma unroll
    for (int j = 0; j < HD / QLM_WAVE; ++j) g[j] = p[64 * j];
}

// A row's outputs, E of them a lane (element lane + 64 j): checked, gated, stored.
// l < 0: a row outside the tree.
template <int HD, typename KV>
__device__ __forceinline__ void put_row(const PaArgs& a, int b, const SeqRows& sq, int i, int h,
                                        float (&o)[HD / QLM_WAVE], float l,
                                        const float (&g)[HD / QLM_WAVE]) {
    constexpr int E = HD / QLM_WAVE;
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const bool dead = l < 0.0f;
    bool fine = l > 0.0f && l < INFINITY;
    const float inv = 1.0f / l;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        o[j] *= inv;
        fine &= fabsf(o[j]) < INFINITY;
    }
    if (__ballot(!fine && !dead)) row_in_fp32<HD, KV>(a, b, sq, i, h, o);
    float* to = a.out + (size_t)(sq.first + i) * a.ldo + (size_t)h * HD + lane;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        if (a.gate) o[j] *= sigmoid_f(g[j]);
        to[64 * j] = dead ? 0.0f : o[j];
    }
}

// Keys that a unit's rows can see end here; its last token is `last`.
__device__ __forceinline__ int keys_end(const PaArgs& a, const SeqRows& sq, int last) {
    const int n = a.bt.parent ? seen_rows(a, sq) : last + 1;
    return min(sq.ctx + n, a.slots);
}

// A row's record of a chunk.
template <int HD>
__device__ __forceinline__ void put_record(const PaArgs& a, int at, float m, float l,
                                           const float (&o)[HD / QLM_WAVE]) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    if (at >= a.rec_rows) return;
    float* rec = a.rec + (size_t)at * (HD + 4);
    if (lane == 0) {
        rec[0] = m;
        rec[1] = l;
    }
#pragma unroll
    for (int e = 0; e < HD / QLM_WAVE; ++e) rec[4 + lane + 64 * e] = o[e];
}

// A tile's rows as they lie in the accumulators: lane (qd, n) has row n's elements
// 16 c + 4 qd .. + 3. `r`: the lane's row of the unit; l < 0: outside the tree.
template <int HD>
__device__ __forceinline__ void put_records(const PaArgs& a, int at, bool real, float m, float l,
                                            const f32x4 (&acc)[HD / 16]) {
    const int qd = (threadIdx.x & (QLM_WAVE - 1)) >> 4;
    if (!real || at >= a.rec_rows) return;
    float* rec = a.rec + (size_t)at * (HD + 4);
    if (qd == 0) {
        rec[0] = m;
        rec[1] = l;
    }
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) *reinterpret_cast<f32x4*>(rec + 4 + 16 * c + 4 * qd) = acc[c];
}
template <int HD, typename KV>
__device__ __forceinline__ void put_tile(const PaArgs& a, int b, const SeqRows& sq, int g, int r,
                                         int total, float l, f32x4 (&acc)[HD / 16]) {
    constexpr int CB = HD / 16;
    const int lane = threadIdx.x & (QLM_WAVE - 1), qd = lane >> 4;
    const bool real = r < total, dead = l < 0.0f;
    const int rc = min(r, total - 1), tok = rc >> a.lg, h = (g << a.lg) + (rc & ((1 << a.lg) - 1));
    const size_t row = (size_t)(sq.first + tok);
    f32x4u gate[CB];
    if (a.gate) {
        const float* p = a.gate + row * a.ldg + (size_t)h * a.gate_stride + 4 * qd;
#pragma unroll
        for (int c = 0; c < CB; ++c) gate[c] = *reinterpret_cast<const f32x4u*>(p + 16 * c);
    }
    const float inv = 1.0f / l;
    bool fine = l > 0.0f && l < INFINITY;
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[c][i] *= inv;
            fine &= fabsf(acc[c][i]) < INFINITY;
        }
    unsigned long long bad = __ballot(real && !dead && !fine);
    bad |= bad >> 32;
    bad = (bad | bad >> 16) & 0xffffull;
    float* to = a.out + row * a.ldo + (size_t)h * HD + 4 * qd;
    if (real && !(bad >> (lane & 15) & 1ull)) {
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            f32x4u o = acc[c];
            if (a.gate) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] *= sigmoid_f(gate[c][i]);
            }
            if (dead) o = f32x4u{0.0f, 0.0f, 0.0f, 0.0f};
            *reinterpret_cast<f32x4u*>(to + 16 * c) = o;
        }
    }
    for (; bad; bad &= bad - 1) {  // a row at a time, the whole wave
        const int from = __ffsll((long long)bad) - 1;
        const int i = __builtin_amdgcn_readlane(tok, from), hh = __builtin_amdgcn_readlane(h, from);
        float o[HD / QLM_WAVE] = {}, gr[HD / QLM_WAVE] = {};
        load_gate<HD>(a, sq, i, hh, gr);
        put_row<HD, KV>(a, b, sq, i, hh, o, 0.0f, gr);
    }
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
    static constexpr int BLK = 2 * Part<F32>::NH * Lay<HD, F32>::GRP;  // a part's K and V
    static constexpr int NW = 128 * 1024 / (2 * BLK);  // 128 KB of LDS: two parts a wave
};

template <int HD, bool F32, bool PACK>
__global__ __launch_bounds__((FewShape<HD, F32>::NW * QLM_WAVE)) void k_pa_few(PaArgs a) {
    using L = Lay<HD, F32>;
    using S = FewShape<HD, F32>;
    using KV = typename std::conditional<F32, float, uint16_t>::type;
    using P = Part<F32>;
    constexpr Math M = F32 ? kF32 : kBf16;
    constexpr int MT = PACK ? 8 : 16, NW = S::NW, NH = P::NH, GRP = L::GRP;
    constexpr int LOADS = 2 * NH * L::LOADS;  // a block's
    constexpr int OST = HD + 4;
    static_assert(NW * 16 * OST * 4 + NW * 16 * 8 <= NW * 2 * S::BLK, "the join fits the rings");
    __shared__ __attribute__((aligned(1024))) char smem[NW * 2 * S::BLK];
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15, qd = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    int g, want;
    head_and_item(blockIdx.x, a.pg.n_kv, g, want);
    Item it;
    if (want >= a.items || !find_item<MT>(a, want, it)) return;
    it.sq = SeqRows{uni(it.sq.first), uni(it.sq.n), uni(it.sq.ctx)};
    const int total = uni(it.sq.n << a.lg), r0 = uni(it.tile * MT);
    const int end = uni(keys_end(a, it.sq, (min(r0 + MT, total) - 1) >> a.lg));
    const int nch = uni((end - 1) / it.len + 1);
    if (it.chunk >= nch) return;
    const int b = uni(it.b), k0 = uni(it.chunk * it.len), k1 = uni(min(k0 + it.len, end));
    const int lgp = uni(31 - __clz(a.pg.page_size));
    const int blocks = uni((k1 - k0 + P::KEYS - 1) / P::KEYS);
    const int mine = uni((blocks - wave + NW - 1) / NW);
    char* ring = smem + wave * 2 * S::BLK;
    auto slot_of = [&](int j) { return k0 + P::KEYS * (wave + j * NW); };
    auto groups = [&](int j, Group (&gr)[NH]) {
#pragma unroll
        for (int h = 0; h < NH; ++h) gr[h] = group_at(a, b, slot_of(j) + 16 * h, k1, lgp);
    };
    // a block in LDS: K groups, V groups
    auto fetch = [&](int j, const Group (&gr)[NH]) {
        char* to = ring + (j & 1) * S::BLK;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            fetch_group<HD, F32>(a, a.pg.k, gr[h], g, slot_of(j) + 16 * h, to + h * GRP);
            fetch_group<HD, F32>(a, a.pg.v, gr[h], g, slot_of(j) + 16 * h, to + (NH + h) * GRP);
        }
    };
    const int parent = a.bt.parent ? tree_parent(a.bt, it.sq, lane) : 0;
    Group gr[3][NH];  // of blocks j, j + 1 and j + 2
#pragma unroll
    for (int j = 0; j < 3; ++j) groups(j, gr[j]);
    // queries first: what is waited for first
    Queries<HD, 1> Q;
    request_rows<HD, 1, PACK, M>(a, it, g, r0, Q);
    __builtin_amdgcn_sched_barrier(0);
    if (mine > 0) fetch(0, gr[0]);
    if (mine > 1) fetch(1, gr[1]);
    __builtin_amdgcn_sched_barrier(0);
    Rows<HD, 1, PACK, M> R;
    take_rows<HD, 1, PACK, M>(a, it, r0, parent, Q, R);
    int staged = -1, raised = -1;  // the block that is there, and the last one begun again
    float x[1][P::XN];
    for (int j = 0;;) {
        bool move = false;
#pragma unroll 1
        for (; j < mine; ++j) {
            const int s0 = slot_of(j);
            const char* at = ring + (j & 1) * S::BLK;
            if (staged != j) {
                staged = j;
                if (j + 1 < mine)
                    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
                else
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            const int va = gr[0][0].valid, vb = gr[0][NH - 1].valid;
            const bool all = s0 + P::KEYS <= it.sq.ctx && va == 16 && vb == 16;
            if (scores<HD, 1, PACK, M>(R, at, at + NH * GRP, s0, it.sq.ctx, va, vb, all, x)) {
                move = raised != j && too_high(R, x);
                if (move) break;
                accumulate<HD, 1, PACK, M>(R, x, at + NH * GRP);
            }
            // the block is read: its place takes the next but one
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (j + 2 < mine) fetch(j + 2, gr[2]);
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                gr[0][h] = gr[1][h];
                gr[1][h] = gr[2][h];
            }
            groups(j + 3, gr[2]);
        }
        if (!move) break;
        raise(R, x);
        raised = j;  // once a block: a score that is not finite stays too high
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
        if constexpr (PACK && !F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fold8(o[i]);
        }
        *reinterpret_cast<f32x4*>(po + (wave * 16 + n) * OST + 16 * c + 4 * qd) = o;
    }
    __syncthreads();
    if (it.chunk == 0 && a.desc) put_desc<MT>(a, it, g, nch);
    const int rows = min(MT, total - r0);
    for (int r = wave; r < rows; r += NW) {
        const int tok = (r0 + r) >> a.lg, h = (g << a.lg) + ((r0 + r) & ((1 << a.lg) - 1));
        float m = -INFINITY, l = 0.0f, o[HD / 64] = {}, gate[HD / 64] = {};
        if (nch == 1) load_gate<HD>(a, it.sq, tok, h, gate);
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
        if (__shfl(R.lim[0], r) < 0) l = -1.0f;
        if (nch == 1)
            put_row<HD, KV>(a, b, it.sq, tok, h, o, l, gate);
        else
            put_record<HD>(a, ((it.rec + it.chunk) * a.pg.n_kv + g) * MT + r, m, l, o);
    }
}

// ---- more rows: four waves share each block of keys ----
// WK such fours take the blocks in turn, each through LDS of its own, so that
// every SIMD has two waves whose products and exponentials take turns; they
// meet at the end.
template <int HD, bool F32>
struct TileShape {
    static constexpr int WK = 2;
    static constexpr int KB = 64 * 128 / HD / (F32 ? 2 : 1);  // keys of a block: 16 KB of each pool
    static constexpr int GRP = Lay<HD, false>::GRP;  // a group in LDS, or of a plane
    static constexpr int POOL = F32 ? 3 * kPlane : KB / 16 * GRP;
    static_assert(!F32 || KB / 16 * GRP == kPlane, "a block's planes");
    // of a four: two blocks, or one in three terms
    static constexpr int LDS = F32 ? 2 * POOL : 4 * POOL;
};

template <int HD, bool F32>
__global__ __launch_bounds__(512, 2) void k_pa_tile(PaArgs a) {
    using L = Lay<HD, F32>;
    using S = TileShape<HD, F32>;
    using P = Part<F32>;
    constexpr Math M = F32 ? kSplit : kBf16;
    using KV = typename std::conditional<F32, float, uint16_t>::type;
    // (two tiles a wave, 128 rows a workgroup: half the LDS reads, but out of
    // registers and fewer workgroups: 2048 rows after 2048 166 us, one tile 150)
    constexpr int RT = 1, NW = 4, WK = S::WK, MT = 16 * RT * NW, KB = S::KB, NG = KB / 16;
    constexpr int GRP = S::GRP, NH = P::NH;
    constexpr int PART = RT * (HD / 16) * 1024 + RT * 512;  // a wave's sums on their way to join
    static_assert(NW * PART <= WK * S::LDS, "the sums fit");
    __shared__ __attribute__((aligned(1024))) char smem[WK * S::LDS];
    __shared__ int there[WK][2][NG];  // slots of a block's groups that are there
    const int lane = threadIdx.x & (QLM_WAVE - 1), n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE % NW);
    const int four = __builtin_amdgcn_readfirstlane(threadIdx.x / (QLM_WAVE * NW));
    int g, want;
    head_and_item(blockIdx.x, a.pg.n_kv, g, want);
    Item it;
    if (want >= a.items || !find_item<MT>(a, want, it)) return;
    it.sq = SeqRows{uni(it.sq.first), uni(it.sq.n), uni(it.sq.ctx)};
    const int total = uni(it.sq.n << a.lg), r0 = uni(it.tile * MT);
    const int end = uni(keys_end(a, it.sq, (min(r0 + MT, total) - 1) >> a.lg));
    const int nch = uni((end - 1) / it.len + 1);
    if (it.chunk >= nch) return;
    const int b = uni(it.b), k0 = uni(it.chunk * it.len), k1 = uni(min(k0 + it.len, end));
    const int lgp = uni(31 - __clz(a.pg.page_size));
    // this four's blocks four, four + WK, ..: as many steps as the first four has
    const int blocks = uni(((k1 - k0 + KB - 1) / KB + WK - 1) / WK);
    auto slot_of = [&](int j) { return k0 + (j * WK + four) * KB; };
    char* const lds = smem + four * S::LDS;
    // a wave fetches a quarter of a block: loads of K and of V of one group
    constexpr int SHARE = NW / NG;          // waves of a group
    constexpr int LPW = L::LOADS / SHARE;  // a wave's loads of either
    static_assert(NW % NG == 0 && L::LOADS % SHARE == 0, "whole loads a wave");
    const int own = wave % NG, j0 = wave / NG * LPW;
    auto group = [&](int j) { return group_at(a, b, slot_of(j) + 16 * own, k1, lgp); };
    // bf16: to LDS, two blocks in turn. fp32: to registers; when the block before is
    // done with, each wave splits what it has loaded, for all four.
    u32x4 staged_x[F32 ? 2 : 1][F32 ? LPW : 1];
    auto fetch = [&](int j, const Group& gr) {
        if constexpr (F32) {
#pragma unroll
            for (int pool = 0; pool < 2; ++pool) {
                const __amdgpu_buffer_rsrc_t r = group_rsrc<HD, F32>(
                    a, pool ? a.pg.v : a.pg.k, gr, g, slot_of(j) + 16 * own);
#pragma unroll
                for (int i = 0; i < LPW; ++i)
                    staged_x[pool][i] = __builtin_bit_cast(
                        u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                   r, ((j0 + i) * QLM_WAVE + lane) * 16, 0, 0));
            }
        } else {
            char* to = lds + (j & 1) * 2 * S::POOL + own * GRP;
            fetch_group<HD, F32, LPW>(a, a.pg.k, gr, g, slot_of(j) + 16 * own, to, j0);
            fetch_group<HD, F32, LPW>(a, a.pg.v, gr, g, slot_of(j) + 16 * own, to + S::POOL, j0);
        }
        if (lane == 0) there[four][j & 1][own] = gr.valid;
    };
    auto split_staged = [&]() {
#pragma unroll
        for (int pool = 0; pool < 2; ++pool)
#pragma unroll
            for (int i = 0; i < LPW; ++i) {
                const int at = (j0 + i) * QLM_WAVE + lane, row = at / (HD / 4), e4 = at % (HD / 4);
                float x4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x4[e] = __uint_as_float(staged_x[pool][i][e]);
                u32x2 w[3];
                split_terms(x4, w);
                char* to = lds + pool * S::POOL + own * GRP + row * (HD * 2) +
                           (((e4 >> 1) ^ row) * 16) + (e4 & 1) * 8;
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<u32x2*>(to + p * kPlane) = w[p];
            }
    };
    const int parent = a.bt.parent ? tree_parent(a.bt, it.sq, lane) : 0;
    Group gr[2] = {group(0), group(1)};
    const int w0 = uni(r0 + 16 * RT * wave);  // this wave's first row
    Queries<HD, RT> Q;
    request_rows<HD, RT, false, M>(a, it, g, w0, Q);
    __builtin_amdgcn_sched_barrier(0);
    fetch(0, gr[0]);
    __builtin_amdgcn_sched_barrier(0);
    Rows<HD, RT, false, M> R;
    take_rows<HD, RT, false, M>(a, it, w0, parent, Q, R);
    // what all of this wave's rows see without a mask, and all they can see
    const int wave_end = uni(
        w0 < total ? min(keys_end(a, it.sq, (min(w0 + 16 * RT, total) - 1) >> a.lg), k1) : 0);
    const int free_end = uni(a.bt.parent ? it.sq.ctx : it.sq.ctx + (w0 >> a.lg) + 1);
    constexpr int SUB = KB / P::KEYS;  // parts of a block
    int staged = -1, raised = -1, valid[NG];
    float x[RT][P::XN];
    for (int i = 0;;) {
        bool move = false;
#pragma unroll 1
        for (; i < blocks * SUB; ++i) {
            const int j = i / SUB, h = i % SUB, s0 = slot_of(j) + P::KEYS * h;
            if (staged != j) {
                staged = j;
                if constexpr (F32) {
                    __syncthreads();  // every wave is done with the last block
                    split_staged();
                    __syncthreads();
                } else {
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    __syncthreads();  // the block is there, and every wave is done with the last
                }
#pragma unroll
                for (int k = 0; k < NG; ++k) valid[k] = uni(there[four][j & 1][k]);
                if (j + 1 < blocks) fetch(j + 1, gr[1]);
                gr[1] = group(j + 2);
            }
            if (s0 >= wave_end) continue;
            int va = valid[0], vb = valid[NH - 1];
#pragma unroll
            for (int k = 1; k < SUB; ++k)
                if (h == k) {
                    va = valid[k * NH];
                    vb = valid[k * NH + NH - 1];
                }
            const bool all = s0 + P::KEYS <= free_end && va == 16 && vb == 16;
            const char* kp = lds + (F32 ? 0 : (j & 1) * 2 * S::POOL) + h * NH * GRP;
            if (scores<HD, RT, false, M>(R, kp, kp + S::POOL, s0, it.sq.ctx, va, vb, all, x)) {
                move = raised != i && too_high(R, x);
                if (move) break;
                accumulate<HD, RT, false, M>(R, x, kp + S::POOL);
            }
        }
        if (!move) break;
        raise(R, x);
        raised = i;  // once a part: a score that is not finite stays too high
    }
    if (it.chunk == 0 && a.desc) put_desc<MT>(a, it, g, nch);
    __syncthreads();
    {
        // the second four's sums to the wave of the first that has the same rows
        char* const to = smem + wave * PART;
        float* const st = reinterpret_cast<float*>(to + RT * (HD / 16) * 1024);
        if (four) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
#pragma unroll
                for (int c = 0; c < HD / 16; ++c)
                    *reinterpret_cast<f32x4*>(to + (t * (HD / 16) + c) * 1024 + lane * 16) =
                        R.acc[t][c];
                st[t * 128 + lane] = R.m[t];
                st[t * 128 + 64 + lane] = R.l[t];
            }
        }
        __syncthreads();
        if (four) return;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float m1 = st[t * 128 + lane], l1 = st[t * 128 + 64 + lane];
            const float m = fmaxf(R.m[t], m1), ref = m == -INFINITY ? 0.0f : m;
            const float f0 = __builtin_amdgcn_exp2f(R.m[t] - ref);
            const float f1 = __builtin_amdgcn_exp2f(m1 - ref);
            R.m[t] = m;
            R.l[t] = R.l[t] * f0 + l1 * f1;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
                const f32x4 o = *reinterpret_cast<const f32x4*>(to + (t * (HD / 16) + c) * 1024 +
                                                               lane * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) R.acc[t][c][i] = R.acc[t][c][i] * f0 + o[i] * f1;
            }
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float l = R.lim[t] < 0 ? -1.0f : cols_sum(R.l[t]);
        const int r = w0 + 16 * t + n;
        if (nch == 1)
            put_tile<HD, KV>(a, b, it.sq, g, r, total, l, R.acc[t]);
        else
            put_records<HD>(a, ((it.rec + it.chunk) * a.pg.n_kv + g) * MT + r - r0, r < total, R.m[t],
                            l, R.acc[t]);
    }
}

// ---- the chunks' records, merged: a row and head a task ----
// WPT waves take a task's records in turn, kJoinFlight of them in flight each,
// and meet in LDS. Few tasks (tokens) have many records: four waves a task.
// Many (trees, prompts) have few or one: a wave a task, which looks `per` tasks'
// descriptors up at once, since most rows of a prompt have nothing to merge.
constexpr int kJoinThreads = 256, kJoinFlight = 8;

template <int HD, typename KV, int WPT>
__global__ __launch_bounds__(kJoinThreads) void k_pa_join(PaArgs a, int mt, int per) {
    constexpr int E = HD / QLM_WAVE, NW = kJoinThreads / QLM_WAVE;
    __shared__ float pm[NW], pl[NW], po[NW][HD];
    const int lane = threadIdx.x & 63, G = 1 << a.lg, tasks = a.bt.rows * a.n_q;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    const int first = (blockIdx.x * (NW / WPT) + wave / WPT) * per;
    int2 d = make_int2(0, 0);
    if (lane < per && first + lane < tasks) {
        const int row = (first + lane) / a.n_q, h = first + lane - row * a.n_q;
        d = a.desc[(size_t)row * a.pg.n_kv + (h >> a.lg)];
        d.x += h & (G - 1);
    }
    const long long stride = (long long)a.pg.n_kv * mt;
    // (a row of no sequence has no descriptor: whatever lies there)
    unsigned long long todo =
        __ballot(d.y > 1 && d.x >= 0 && d.x + (d.y - 1) * stride < a.rec_rows);
    for (; todo; todo &= todo - 1) {  // WPT > 1: one task, the same in all its waves
        const int k = __ffsll((long long)todo) - 1;
        const int nch = __builtin_amdgcn_readlane(d.y, k);
        const int task = first + k, row = task / a.n_q, h = task - row * a.n_q;
        const int b = seq_of_row(a.bt, row);
        if (b < 0) continue;
        const SeqRows sq = seq_rows(a.bt, b);
        const int i = row - sq.first;
        if (i < 0 || i >= sq.n) continue;
        float gate[E] = {};
        load_gate<HD>(a, sq, i, h, gate);
        const float* rec = a.rec + (size_t)__builtin_amdgcn_readlane(d.x, k) * (HD + 4);
        const size_t step = (size_t)stride * (HD + 4);
        float m = -INFINITY, l = 0.0f, o[E] = {};
        for (int c0 = wave % WPT; c0 < nch; c0 += kJoinFlight * WPT) {
            float rm[kJoinFlight], rl[kJoinFlight], ro[kJoinFlight][E];
#pragma unroll
            for (int u = 0; u < kJoinFlight; ++u) {
                const float* r = rec + (size_t)min(c0 + u * WPT, nch - 1) * step;
                rm[u] = r[0];
                rl[u] = r[1];
#pragma unroll
                for (int e = 0; e < E; ++e) ro[u][e] = r[4 + lane + 64 * e];
            }
            if (rl[0] < 0.0f) {  // a row outside the tree, in every chunk
                m = -INFINITY;
                l = -1.0f;
                break;
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < kJoinFlight; ++u) top = fmaxf(top, rm[u]);
            const float ref = top == -INFINITY ? 0.0f : top;
            const float f = __builtin_amdgcn_exp2f(m - ref);
            l *= f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= f;
#pragma unroll
            for (int u = 0; u < kJoinFlight; ++u) {
                if (c0 + u * WPT >= nch) break;
                const float w = __builtin_amdgcn_exp2f(rm[u] - ref);
                l = fmaf(rl[u], w, l);
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = fmaf(ro[u][e], w, o[e]);
            }
            m = top;
        }
        if constexpr (WPT > 1) {
            if (lane == 0) {
                pm[wave] = m;
                pl[wave] = l;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) po[wave][lane + 64 * e] = o[e];
            __syncthreads();
            if (wave) return;
#pragma unroll
            for (int w = 0; w < WPT; ++w) m = fmaxf(m, pm[w]);
            const float ref = m == -INFINITY ? 0.0f : m;
            const bool dead = l < 0.0f;
            l = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < WPT; ++w) {
                const float f = __builtin_amdgcn_exp2f(pm[w] - ref);
                l = fmaf(pl[w], f, l);
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = fmaf(po[w][lane + 64 * e], f, o[e]);
            }
            if (dead) l = -1.0f;
        }
        put_row<HD, KV>(a, b, sq, i, h, o, l, gate);
    }
}

// ---- the host's part ----

struct PaPlan {
    int mt;              // rows of a unit: 8, 16 (k_pa_few) or 64 (k_pa_tile)
    int target;          // items a kv head to cut the keys into
    int least, alone;    // keys of an item, at least; of a sequence that is not cut
    int items;           // at most
    int rec_rows;        // records
    bool join;           // some unit may have several chunks
    size_t desc_at, bytes;
};

PaPlan plan_of(int rows, int B, int G, int n_kv, int hd, long long slots) {
    PaPlan p{};
    // about the rows of a sequence
    const long long per = ((long long)rows * G + B - 1) / B;
    p.mt = per <= 8 ? 8 : per <= 16 ? 16 : 64;
    p.target = std::max(1, 256 / n_kv);  // a CU holds one workgroup
    const long long units = ((long long)rows * G) / p.mt + B;
    const long long most = p.mt <= 16 ? p.target + p.target / 2 + 1 : p.target;  // items but those
    // Cutting costs the join's launch. Single tokens, whole up to 1024 slots and up to
    // 512: one after 1000 14.8 and 13.4 us, 16 15.5 and 14.9, but 64 26.0 and 29.3 (up
    // to 256: 64 after 500 20.7 for 17.3; up to 2048: one after 2000 22.0 for 13.4).
    // Pieces of 256 slots at least, 512 and 128: one after 1500 13.4, 15.0 and 13.1,
    // after 16000 18.7, 17.1 and 19.4. Tiles have work enough in 128: 5 trees of 33 in
    // fp32 35, with 256 44, with 512 65; the bf16 cases within 2 of each other.
    p.alone = p.mt <= 16 ? 1024 : 128;
    p.least = p.mt <= 16 ? 256 : 128;
    p.join = slots > p.alone;
    // (8: what fp32 sums may be off by)
    p.items = (int)std::min(units + most + 8, units * (p.join ? (slots - 1) / p.least + 1 : 1));
    if (p.join) p.rec_rows = (int)(2 * most + 16) * n_kv * p.mt;
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
    const dim3 few(FewShape<HD, F32>::NW * QLM_WAVE), tile(512);
    if (p.mt == 8)
        hipLaunchKernelGGL((k_pa_few<HD, F32, true>), grid, few, 0, st, a);
    else if (p.mt == 16)
        hipLaunchKernelGGL((k_pa_few<HD, F32, false>), grid, few, 0, st, a);
    else
        hipLaunchKernelGGL((k_pa_tile<HD, F32>), grid, tile, 0, st, a);
    const int rc = qlm_launch_status();
    if (rc != QLM_OK || !p.join) return rc;
    // The join: one token after 4000, 16 tasks of 16 records, 14.0 us with four waves a
    // task, 16.8 with one; 4 trees of 64, 4096 tasks, 36.8 and 29.9 (2 of them, 2048,
    // 23.4 and 20.9). Many tasks in 8192 waves: 2048 rows after 2048 148.6, a task a wave
    // 151.3; 8192 tasks a wave each 62.8, four a wave 65.1.
    const int tasks = a.bt.rows * a.n_q;
    if (tasks <= 2048) {
        hipLaunchKernelGGL((k_pa_join<HD, KV, 4>), dim3(tasks), dim3(kJoinThreads), 0, st, a, p.mt,
                           1);
    } else {
        const int per = std::min((tasks + 8191) / 8192, QLM_WAVE);
        hipLaunchKernelGGL((k_pa_join<HD, KV, 1>), dim3((tasks + 4 * per - 1) / (4 * per)),
                           dim3(kJoinThreads), 0, st, a, p.mt, per);
    }
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
    if (gate && (gate_stride < hd || ldg < (long long)(n_q - 1) * gate_stride + hd))
        return QLM_ERR_SHAPE;
    const int G = n_q / n_kv;
    const PaPlan p = plan_of(batch->rows, batch->B, G, n_kv, hd, slots);
    if (groups_of(p.items, n_kv) >= 1LL << 23) return QLM_ERR_SHAPE;  // a launch's threads fit 32 bits
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
    a.least = p.least;
    a.alone = p.alone;
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
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>((k_pa_join<128, float, 1>)));
}
