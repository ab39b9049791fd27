// Ragged rows, trees of drafted tokens and the paged KV cache (qlm_row_batch,
// qlm_kv_pages): what their kernels share. The arrays are device memory that no
// host check has seen, so every index that comes out of them is bounded here
// before it addresses anything.
#pragma once

#include "common.hpp"

// A sequence of the batch, as the kernels see it.
struct SeqRows {
    int first;  // its first row
    int n;      // its rows
    int ctx;    // positions before them
};

__device__ __forceinline__ SeqRows seq_rows(const qlm_row_batch& bt, int b) {
    const int s = min(max(bt.row_start[b], 0), bt.rows);
    const int e = min(max(bt.row_start[b + 1], 0), bt.rows);
    return SeqRows{s, max(e - s, 0), min(max(bt.ctx_len[b], 0), 1 << 30)};
}

// The sequence of row r: the last b < B with row_start[b] <= r, or -1 for a row
// that no sequence owns. The whole wave takes part. start0: row_start[min(lane, B)].
__device__ __forceinline__ int seq_of_row(const qlm_row_batch& bt, int r, int start0) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    int count = 0;  // entries of row_start[0..B] that are <= r
    for (int i = 0; i <= bt.B; i += QLM_WAVE) {
        const int e = i ? bt.row_start[min(i + lane, bt.B)] : start0;
        const int c = __popcll(__ballot(i + lane <= bt.B && max(e, 0) <= r));
        count += c;
        if (c < QLM_WAVE) break;
    }
    return count > 0 && count <= bt.B ? count - 1 : -1;
}

__device__ __forceinline__ int seq_of_row(const qlm_row_batch& bt, int r) {
    return seq_of_row(bt, r, bt.row_start[min((int)(threadIdx.x & (QLM_WAVE - 1)), bt.B)]);
}

// p[i], i the same in all lanes, through the scalar cache: memory that the launch
// does not write.
__device__ __forceinline__ int uniform_load(const int* p, size_t i) {
    const auto* q = reinterpret_cast<const __attribute__((address_space(4))) int*>(
        reinterpret_cast<uintptr_t>(p));
    return q[i];
}

// The tree over a sequence's first QLM_TREE_MAX rows, one row a lane: the line
// of row `lane` as a set of rows (0 for a row outside the tree). The whole wave
// takes part. Each round doubles the length of line that a lane has followed.
static_assert(QLM_TREE_MAX == QLM_WAVE, "a lane a row");
__device__ __forceinline__ unsigned long long tree_line(int parent) {
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const unsigned long long roots = __ballot(parent == -1);
    int up = parent >= 0 && parent < lane ? parent : -1;
    unsigned long long line = 1ull << lane;
    while (__ballot(up >= 0)) {
        const int from = up >= 0 ? up : lane;
        const unsigned lo = __shfl((unsigned)line, from), hi = __shfl((unsigned)(line >> 32), from);
        const int next = __shfl(up, from);
        line |= (unsigned long long)hi << 32 | lo;
        up = up >= 0 ? next : -1;
    }
    return line & roots ? line : 0ull;
}

// The parent that row `i` (a lane's) of a sequence has in the tree; -2: none.
__device__ __forceinline__ int tree_parent(const qlm_row_batch& bt, const SeqRows& s, int i) {
    if (i >= s.n || i >= QLM_TREE_MAX) return -2;
    return bt.parent ? bt.parent[s.first + i] : i - 1;
}

// The page of a sequence's slot, or -1 where there is none.
__device__ __forceinline__ int page_of(const qlm_kv_pages& pg, int b, int slot) {
    const int i = slot / pg.page_size;
    if (slot < 0 || i >= pg.ld_table) return -1;
    const int p = pg.table[(size_t)b * pg.ld_table + i];
    return (unsigned)p < (unsigned)pg.n_pages ? p : -1;
}

// Where slot `slot` of page `page` begins for head g, in elements of a pool.
__device__ __forceinline__ size_t slot_at(const qlm_kv_pages& pg, int page, int g, int slot) {
    return (((size_t)page * pg.n_kv + g) * pg.page_size + (slot & (pg.page_size - 1))) * pg.hd;
}

constexpr int kMaxBatchRows = 1 << 21;

// Checks that every entry point of this family makes.
static inline int check_row_batch(const qlm_row_batch* b) {
    if (!b || !b->row_start || !b->ctx_len || b->B <= 0 || b->rows <= 0) return QLM_ERR_ARG;
    if (b->B > 65535 || b->rows > kMaxBatchRows) return QLM_ERR_SHAPE;
    return QLM_OK;
}

static inline int check_kv_pages(const qlm_kv_pages* p) {
    if (!p || !p->k || !p->v || !p->table || p->n_pages <= 0 || p->n_kv <= 0 || p->ld_table <= 0)
        return QLM_ERR_ARG;
    if (p->dtype != 0 && p->dtype != 1) return QLM_ERR_ARG;
    if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)) != 0)
        return QLM_ERR_SHAPE;
    if (p->hd != 128 && p->hd != 256) return QLM_ERR_SHAPE;
    if (p->n_kv > 1024 || (long long)p->ld_table * p->page_size > 1LL << 30)
        return QLM_ERR_SHAPE;
    if (((uintptr_t)p->k | (uintptr_t)p->v) & 15u) return QLM_ERR_SHAPE;
    return QLM_OK;
}
