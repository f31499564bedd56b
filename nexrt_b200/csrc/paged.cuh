// A key-value cache in pages: pool [pages][kv heads][slots of a page][head dim] for K and for V, and a table that names the
// pages of every sequence.  The index arithmetic that the kernels share, as host and device functions: the host forms are what
// the CPU tests run (nexrt_paged_slot, nexrt_paged_split).
#pragma once

#include "common.cuh"

namespace nexrt {

struct PageTable {
    const int* table;    // [rows][width]: page of positions [page * j, page * (j + 1)) of a row, -1: none
    int64_t stride;      // ints between two rows
    int rows, width;
    int page;            // slots of a page
    int pages;           // pages of the pool
};

// Entry `j` of a row as the table has it, -1 outside the table.
__host__ __device__ __forceinline__ int page_entry(const PageTable& t, int row, int j) {
    return row < 0 || row >= t.rows || j < 0 || j >= t.width ? -1 : t.table[row * t.stride + j];
}

// The same, -1 also where it names no page of the pool.
__host__ __device__ __forceinline__ int page_at(const PageTable& t, int row, int j) {
    const int p = page_entry(t, row, j);
    return p >= 0 && p < t.pages ? p : -1;
}

// Pages that `len` positions take.
__host__ __device__ __forceinline__ int pages_of(int len, int page) { return len <= 0 ? 0 : (len - 1) / page + 1; }

// ---- the split of a batch's keys over the CTAs of the attention kernel ------------------------------------------------
// Work is counted in chunks of kChunk keys of one item (sequence, kv head, head group), and each item with keys counts kItemCost
// chunks more, in front of its own: what it costs to begin and to end one (a ragged batch takes 168 us without, 134 / 111 / 97 / 98 / 107
// with 1 / 2 / 3 / 4 / 5).  Of the `total` in the order sequence, head, chunk CTA
// c of n takes [total c / n, total (c + 1) / n), so all CTAs have the same work whatever the lengths.
constexpr int kChunk = 64;
constexpr int kItemCost = 3;

// Keys [lo, hi) that the query behind the last of `len` keys sees; `room` keys have a place in the table, and a longer row ends with them.
__host__ __device__ __forceinline__ void key_span(int len, int64_t room, int window, int& lo, int& hi) {
    hi = len < 0 ? 0 : (len > room ? static_cast<int>(room) : len);
    lo = window > 0 && hi > window ? hi - window : 0;
}
__host__ __device__ __forceinline__ int chunks_of(int lo, int hi) { return hi <= lo ? 0 : (hi - 1) / kChunk - lo / kChunk + 1; }
__host__ __device__ __forceinline__ int cost_of(int chunks) { return chunks ? chunks + kItemCost : 0; }

// a / b of numbers that are not negative: 32 bits where they fit (a 64-bit division takes about 100 instructions on the GPU).
__host__ __device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
__host__ __device__ __forceinline__ int64_t range_begin(int64_t total, int c, int n) { return quotient(total * c, n); }
// The CTA whose range holds unit x: the largest c with total c / n <= x.
__host__ __device__ __forceinline__ int owner_of(int64_t x, int64_t total, int n) { return static_cast<int>(quotient(n * (x + 1) - 1, total)); }
// CTAs that get work: at most `grid`, no more than there are units.  (With little work a chunk each is best, although that cuts every item:
// 18 chunks of 256 dims take 9.2 us in 18 CTAs, 4 us more in 5.)
__host__ __device__ __forceinline__ int active_ctas(int64_t total, int grid) { return total < grid ? (total > 0 ? static_cast<int>(total) : 1) : grid; }
// Chunks [c0, c1) of an item (its units begin at item0) that lie in [x, x_end).
__host__ __device__ __forceinline__ void item_part(int64_t item0, int chunks, int64_t x, int64_t x_end, int& c0, int& c1) {
    const int64_t real = item0 + kItemCost, from = x - real, to = x_end - real;
    c0 = from < 0 ? 0 : static_cast<int>(from);
    c1 = to < 0 ? 0 : (to < chunks ? static_cast<int>(to) : chunks);
}

// ---- asynchronous copies of 16 bytes into shared memory -------------------------------------------------------------------
#ifdef __CUDACC__
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
#endif

}  // namespace nexrt
