// Pages of a shared key-value cache: rows of a table are continued, forked and freed, the pages they share are counted, a
// begun page that is about to be written is copied, live pages are moved to the front of the pool.
//
// Everything is planned on the device, so that a beam-search step needs no word from the host and can be captured: a grid
// copies and counts the table (integer atomics: the order does not show), one CTA plans (what is ordered - which row copies,
// which page is free next - is a prefix sum over rows or pages), a grid moves the bytes.  Free pages are those that no row of
// the table names; the lowest go first, to the rows in their order.
//
// Bound by the bytes of the copied pages; for a table without copies by the launches and the plan's few round trips.  Measured: 360
// pages of 15 layers (708 MB both ways) compacted in 124 us, 0.88 of copy rate; eight beams of 8191 keys forked in 9.6 us, 128 of up to
// 20000 in 15, 4096 of 300 in 51.
#include "api.h"
#include "paged.cuh"

namespace nexrt {

constexpr int kPlanThreads = 1024;
constexpr int kPlanRows = 4096;         // rows whose plan one CTA holds in shared memory
constexpr int kPagesPerThread = 8;
// Rows up to which each searches the others for holders of its begun page; of more they are counted page by page (forks of 300 positions, eight
// rows a prompt, searched and counted: 8 rows 7.4 and 7.5 us, 32 rows 9.2 and 9.3, 64 rows 9.0 and 8.9, 96 rows 9.5 and 9.3, 256 rows 13.4 and
// 11.5, 4096 rows 548 and 51: the line may lie anywhere up to 64).
constexpr int kSearchRows = 32;
// Entries of a table that the planning CTA counts itself (8 rows of 130 entries: a fork 14.4 -> 9.6 us on the device; a CTA takes
// about 1 us a thousand entries, a launch and a memset 5 us).
constexpr int kSmallTable = 4096;

// Sum of `v` over the threads before this one; `total` gets the sum over all.  red: 33 ints.
__device__ __forceinline__ int block_prefix(int v, int* red, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += n;
    }
    __syncthreads();
    if (lane == 31) red[warp] = s;
    __syncthreads();
    if (warp == 0) {
        int w = lane < static_cast<int>(blockDim.x >> 5) ? red[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += n;
        }
        red[lane] = w;
    }
    __syncthreads();
    total = red[31];
    return s - v + (warp ? red[warp - 1] : 0);
}

__device__ __forceinline__ void latch(int* status, Status code) {
    if (status) atomicCAS(status, 0, static_cast<int>(code));
}

// Positions of old row p that a new row takes over: what has a place in the table.
__device__ __forceinline__ int kept_len(const PageTable& t, const int* lens, int p) {
    if (p < 0 || p >= t.rows) return 0;
    const int64_t room = static_cast<int64_t>(t.width) * t.page;
    const int n = lens[p];
    return n < 0 ? 0 : (n > room ? static_cast<int>(room) : n);
}

// new table[r] = old table[parents[r]] (-1 behind its last page), refs[page] += rows that name it; columns [j0, width) by steps of `step`.
__device__ __forceinline__ void go_on(const PageTable& t, const int* lens, const int* parents, int* out, int64_t out_stride, int* refs, int r, int j0, int step, int* status) {
    const int p = parents ? parents[r] : r;
    if (j0 == 0 && (p >= t.rows || (p >= 0 && lens[p] > static_cast<int64_t>(t.width) * t.page))) latch(status, kStatusBadPage);
    const int used = pages_of(kept_len(t, lens, p), t.page);
    for (int j = j0; j < t.width; j += step) {
        int page = -1;
        if (j < used) {
            page = page_at(t, p, j);
            if (page < 0) latch(status, kStatusBadPage);
            else atomicAdd(refs + page, 1);
        }
        if (out) out[r * out_stride + j] = page;
    }
}

// A table of more than kSmallTable entries; refs comes in as zero.
__global__ void __launch_bounds__(256) fork_rows_kernel(PageTable t, const int* lens, const int* parents, int* out, int64_t out_stride, int* refs, int n,
                                                        int* status) {
    pdl_launch_dependents();
    pdl_wait();
    for (int r = blockIdx.y; r < n; r += gridDim.y) go_on(t, lens, parents, out, out_stride, refs, r, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x, status);
}

// The same by the CTA that plans: a launch and a memset less where there is little to count.
__device__ __forceinline__ void count_here(const PageTable& t, const int* lens, const int* parents, int* out, int64_t out_stride, int* refs, int n, int* status) {
    for (int p = threadIdx.x; p < t.pages; p += blockDim.x) refs[p] = 0;
    __syncthreads();
    const int warps = blockDim.x >> 5, cols = t.width > 0 ? t.width : 1;
    // a row a warp, whose parent and length are then found once; of more rows an entry a thread (8 rows of 130 entries 9.6 us, by entries
    // 11.3; 512 rows of 8 entries 29 and 17)
    if (n <= warps) {
        if (threadIdx.x >> 5 < n) go_on(t, lens, parents, out, out_stride, refs, threadIdx.x >> 5, threadIdx.x & 31, 32, status);
    } else {
        for (int e = threadIdx.x; e < n * cols; e += blockDim.x) go_on(t, lens, parents, out, out_stride, refs, e / cols, e % cols, cols, status);
    }
    __syncthreads();
}

struct ForkPlan {
    PageTable t;                // the old table
    const int *lens, *parents, *grow;
    int* table;                 // the new one, as fork_rows_kernel left it
    int64_t table_stride;
    int *lens_out, *refs;
    int* copies;                // [n][3]: source page, target page, positions to copy
    int* n_copies;
    int* free_list;             // [pages] scratch
    int *writers, *first;       // [pages] scratch: rows that go on writing in a begun page, the lowest of them
    int* status;
    int* grown;                 // may be null: the row where it got its positions, else -1
    int n, grow_all, pages;
    int count;                  // the table has not been copied and counted yet
};

// One CTA.  A row with g more positions needs pages for them, and, if it goes on writing in a begun page that other rows hold
// too, a copy of that page.  Where all holders of the page go on writing, the first of them keeps it.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const ForkPlan a) {
    extern __shared__ int plan_smem[];
    int* const last = plan_smem;             // [n] begun page that the row writes in, -1: none
    int* const fresh = last + a.n;           // [n] pages that the row takes; bit 30: the first of them is a copy
    __shared__ int red[33];
    pdl_launch_dependents();
    pdl_wait();
    if (a.count) count_here(a.t, a.lens, a.parents, a.table, a.table_stride, a.refs, a.n, a.status);
    constexpr int kCopy = 1 << 30;
    for (int r = threadIdx.x; r < a.n; r += blockDim.x) {
        const int p = a.parents[r], len = kept_len(a.t, a.lens, p);
        const bool alive = p >= 0 && p < a.t.rows;
        int g = alive ? (a.grow ? a.grow[r] : a.grow_all) : 0;
        if (g < 0) g = 0;
        const int used = pages_of(len, a.t.page);
        int want = 0, open = -1;
        if (g > 0) {
            const int64_t room = static_cast<int64_t>(a.t.width) * a.t.page;
            if (static_cast<int64_t>(len) + g > (room < INT32_MAX ? room : INT32_MAX)) {
                latch(a.status, kStatusNoPages);
                g = 0;
            } else if (len % a.t.page) {
                open = a.table[r * a.table_stride + used - 1];
                if (open < 0) g = 0;         // the page is missing (latched before): nowhere to write
            }
            if (g > 0) want = pages_of(len + g, a.t.page) - used;
        }
        last[r] = open;
        fresh[r] = want;
        a.lens_out[r] = len + g;
        if (a.grown) a.grown[r] = g > 0 ? r : -1;
    }
    __syncthreads();
    const bool many = a.n > kSearchRows;
    if (many) {
        for (int r = threadIdx.x; r < a.n; r += blockDim.x)
            if (const int page = last[r]; page >= 0) {
                a.writers[page] = 0;
                a.first[page] = a.n;
            }
        __syncthreads();
        for (int r = threadIdx.x; r < a.n; r += blockDim.x)
            if (const int page = last[r]; page >= 0) {
                atomicAdd(a.writers + page, 1);
                atomicMin(a.first + page, r);
            }
        __syncthreads();
    }
    for (int r = threadIdx.x; r < a.n; r += blockDim.x) {
        const int page = last[r];
        if (page < 0) continue;
        const int held = a.refs[page];
        if (held <= 1) continue;
        int same = 0, first = 1;
        if (many) {
            same = a.writers[page];
            first = a.first[page] == r;
        } else {
            for (int i = 0; i < a.n; ++i)
                if (last[i] == page) {
                    ++same;
                    if (i < r) first = 0;
                }
        }
        if (!(same == held && first)) fresh[r] += 1 + kCopy;     // only this thread reads or writes this entry
    }
    __syncthreads();

    // pages wanted by all rows, and the lowest free ones of the pool
    int need = 0;
    for (int r0 = 0; r0 < a.n; r0 += blockDim.x) {
        const int r = r0 + threadIdx.x;
        int total;
        block_prefix(r < a.n ? fresh[r] & (kCopy - 1) : 0, red, total);
        need += total;
    }
    int found = 0;
    for (int p0 = 0; p0 < a.pages && found < need; p0 += blockDim.x * kPagesPerThread) {
        const int base = p0 + threadIdx.x * kPagesPerThread;
        int mask = 0;
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i)
            if (base + i < a.pages && a.refs[base + i] == 0) mask |= 1 << i;
        int total;
        int at = found + block_prefix(__popc(mask), red, total);
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i)
            if (mask >> i & 1) a.free_list[at++] = base + i;
        found += total;
    }
    __syncthreads();

    int before = 0, copied = 0;
    for (int r0 = 0; r0 < a.n; r0 += blockDim.x) {
        const int r = r0 + threadIdx.x;
        const int f = r < a.n ? fresh[r] : 0, k = f & (kCopy - 1);
        int total;
        const int at = before + block_prefix(k, red, total);
        before += total;
        const int p = k > 0 ? a.parents[r] : -1, len = kept_len(a.t, a.lens, p);
        int src = 0, dst = 0, fill = 0;
        if (k > 0 && at + k > found) {
            latch(a.status, kStatusNoPages);                     // the pool is full: the row keeps what it has and does not grow
            a.lens_out[r] = len;
            if (a.grown) a.grown[r] = -1;
        } else if (k > 0) {
            int* row = a.table + r * a.table_stride;
            int used = pages_of(len, a.t.page), i = 0;
            if (f & kCopy) {
                src = last[r];
                dst = a.free_list[at];
                fill = len % a.t.page;
                row[used - 1] = dst;
                a.refs[dst] = 1;
                atomicSub(a.refs + src, 1);
                i = 1;
            }
            for (; i < k; ++i) {
                const int page = a.free_list[at + i];
                row[used++] = page;
                a.refs[page] = 1;
            }
        }
        // only what is copied is listed
        const int place = copied + block_prefix(fill > 0, red, total);
        copied += total;
        if (fill > 0) {
            a.copies[3 * place] = src;
            a.copies[3 * place + 1] = dst;
            a.copies[3 * place + 2] = fill;
        }
    }
    if (threadIdx.x == 0) *a.n_copies = copied;
}

struct CompactPlan {
    PageTable t;
    const int* lens;
    int* refs;                  // [pages] rows that name a page
    int *refs_out, *remap;      // of the moved pages; new place of a page, -1: free
    int* copies;                // [pages][3]
    int* n_copies;
    int* live;
    int* holes;                 // [pages] scratch
    int pages;
    int count;                  // the table has not been counted yet
    int* status;
};

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactPlan a) {
    __shared__ int red[33];
    pdl_launch_dependents();
    pdl_wait();
    if (a.count) count_here(a.t, a.lens, nullptr, nullptr, 0, a.refs, a.t.rows, a.status);
    constexpr int kStep = kPlanThreads * kPagesPerThread;
    int live = 0;
    for (int p0 = 0; p0 < a.pages; p0 += kStep) {
        const int base = p0 + threadIdx.x * kPagesPerThread;
        int c = 0, total;
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) c += base + i < a.pages && a.refs[base + i] > 0;
        block_prefix(c, red, total);
        live += total;
    }
    // holes in front of `live`, in order; what stays keeps its count
    int holes = 0;
    for (int p0 = 0; p0 < live; p0 += kStep) {
        const int base = p0 + threadIdx.x * kPagesPerThread;
        int mask = 0, total;
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) {
            const int p = base + i;
            if (p >= live) break;
            const int n = a.refs[p];
            if (n > 0) {
                a.remap[p] = p;
                a.refs_out[p] = n;
            } else {
                a.remap[p] = -1;
                mask |= 1 << i;
            }
        }
        int at = holes + block_prefix(__popc(mask), red, total);
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i)
            if (mask >> i & 1) a.holes[at++] = base + i;
        holes += total;
    }
    __syncthreads();
    // pages behind `live` move into them, in order
    int moved = 0;
    for (int p0 = live / kPagesPerThread * kPagesPerThread; p0 < a.pages; p0 += kStep) {
        const int base = p0 + threadIdx.x * kPagesPerThread;
        int mask = 0, total;
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) {
            const int p = base + i;
            if (p < live || p >= a.pages) continue;
            a.refs_out[p] = 0;
            if (a.refs[p] > 0) mask |= 1 << i;
            else a.remap[p] = -1;
        }
        int at = moved + block_prefix(__popc(mask), red, total);
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i)
            if (mask >> i & 1) {
                const int to = a.holes[at], p = base + i;
                a.remap[p] = to;
                a.refs_out[to] = a.refs[p];
                a.copies[3 * at] = p;
                a.copies[3 * at + 1] = to;
                a.copies[3 * at + 2] = -1;                       // the whole page
                ++at;
            }
        moved += total;
    }
    if (threadIdx.x == 0) {
        *a.n_copies = moved;
        *a.live = live;
    }
}

// Checks a caller's list of copies: pages that do not exist, a target that is also a source, a target given twice (the last one counts).
// One CTA marks sources and targets page by page, so that a list costs its length (1000 copies of 128 bytes 56 us where each copy looked
// through the others).
__global__ void __launch_bounds__(kPlanThreads) copy_list_kernel(const int* src, const int* dst, int n, int pages, int* copies, int* source, int* writer, int* status) {
    pdl_launch_dependents();
    pdl_wait();
    auto counts = [&](int s, int d) { return s >= 0 && d >= 0 && s != d; };
    for (int i = threadIdx.x; i < n; i += blockDim.x)
        for (const int p : {src[i], dst[i]})
            if (p >= 0 && p < pages) source[p] = writer[p] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = src[i], d = dst[i];
        if (!counts(s, d)) continue;
        if (s < pages) source[s] = i;
        if (d < pages) atomicMax(writer + d, i);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = src[i], d = dst[i];
        int fill = -1;
        if (!counts(s, d)) {
            fill = 0;                                                // left out
        } else if (s >= pages || d >= pages) {
            latch(status, kStatusBadPage);
            fill = 0;
        } else if (source[d] >= 0 || writer[d] > i) {
            latch(status, kStatusPageConflict);
            fill = 0;
        }
        copies[3 * i] = s;
        copies[3 * i + 1] = d;
        copies[3 * i + 2] = fill;
    }
}

struct PageMove {
    char* pool;                 // [planes][pages][heads][slots][dim]
    const int* copies;          // [n][3] source, target, positions (-1: the page, 0: nothing)
    const int* n_copies;        // null: n
    int n, planes, heads;
    int64_t plane_bytes, page_bytes, head_bytes, slot_bytes;
    // the table of a compaction, renamed by the same launch
    PageTable t;
    const int *lens, *remap;
    int* table_out;
    int64_t table_stride;
};

constexpr int kMoveThreads = 256;
constexpr int kMoveLoads = 4;                         // 16-byte loads of a thread in flight (with eight a compaction gains nothing, small copies lose)
constexpr int kMovePiece = kMoveThreads * 16 * kMoveLoads;

__global__ void __launch_bounds__(kMoveThreads, 6) page_move_kernel(const PageMove a) {
    pdl_launch_dependents();
    pdl_wait();
    const int n = a.n_copies ? *a.n_copies : a.n;
    if (a.table_out) {
        for (int r = blockIdx.x; r < a.t.rows; r += gridDim.x) {
            const int used = pages_of(kept_len(a.t, a.lens, r), a.t.page);
            for (int j = threadIdx.x; j < a.t.width; j += blockDim.x) {
                const int p = j < used ? page_at(a.t, r, j) : -1;
                a.table_out[r * a.table_stride + j] = p < 0 ? -1 : a.remap[p];
            }
        }
    }
    // a piece never crosses a head, so that copies of a begun page move its written positions only
    const int per_head = static_cast<int>((a.head_bytes + kMovePiece - 1) / kMovePiece);
    const int64_t units = static_cast<int64_t>(n) * a.planes * a.heads * per_head;
    struct Unit {
        const char* src;
        int64_t step, bytes;        // from source to target; of this piece, 0: nothing
    };
    auto unit = [&](int64_t u) -> Unit {
        if (u >= units) return {nullptr, 0, 0};
        const int64_t run = quotient(u, per_head), page = quotient(run, a.heads), i = quotient(page, a.planes);
        const int piece = static_cast<int>(u - run * per_head), head = static_cast<int>(run - page * a.heads), plane = static_cast<int>(page - i * a.planes);
        const int from = a.copies[3 * i], to = a.copies[3 * i + 1], fill = a.copies[3 * i + 2];
        const int64_t begin = static_cast<int64_t>(piece) * kMovePiece, bytes = fill < 0 ? a.head_bytes : fill * a.slot_bytes;
        return {a.pool + plane * a.plane_bytes + from * a.page_bytes + head * a.head_bytes + begin, static_cast<int64_t>(to - from) * a.page_bytes, bytes - begin};
    };
    // the next piece is looked up while this one's loads are on their way
    Unit now = unit(blockIdx.x);
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        uint4 v[kMoveLoads];
#pragma unroll
        for (int k = 0; k < kMoveLoads; ++k) {
            const int o = (k * kMoveThreads + threadIdx.x) * 16;
            if (o < now.bytes) v[k] = *reinterpret_cast<const uint4*>(now.src + o);
        }
        const Unit next = unit(u + gridDim.x);
#pragma unroll
        for (int k = 0; k < kMoveLoads; ++k) {
            const int o = (k * kMoveThreads + threadIdx.x) * 16;
            if (o < now.bytes) *reinterpret_cast<uint4*>(const_cast<char*>(now.src) + now.step + o) = v[k];
        }
        now = next;
    }
}

// whole: every copy is of a whole page, whose heads then are one run.
static int move_launch(PageMove& a, const NexrtPagesArgs& x, bool whole, cudaStream_t st) {
    a.pool = static_cast<char*>(x.pool);
    a.planes = x.planes; a.heads = whole ? 1 : x.heads;
    a.slot_bytes = x.slot_bytes; a.head_bytes = static_cast<int64_t>(x.slots) * x.slot_bytes * (whole ? x.heads : 1);
    a.page_bytes = a.head_bytes * a.heads; a.plane_bytes = a.page_bytes * x.pages;
    const int64_t units = static_cast<int64_t>(a.n) * a.planes * a.heads * ((a.head_bytes + kMovePiece - 1) / kMovePiece);
    const int64_t most = 16ll * sm_count();
    int64_t grid = units < most ? units : most;
    if (a.table_out && grid < a.t.rows) grid = a.t.rows < most ? a.t.rows : most;
    return grid > 0 ? launch(page_move_kernel, dim3(static_cast<unsigned>(grid)), dim3(kMoveThreads), 0, st, a) : 0;
}

static bool pool_ok(const NexrtPagesArgs& x) {
    return x.size == sizeof(x) && x.planes >= 0 && x.pages >= 0 && x.heads >= 1 && x.slots >= 1 && x.slot_bytes >= 16 && x.slot_bytes % 16 == 0 &&
           (reinterpret_cast<uintptr_t>(x.pool) & 15) == 0 && x.rows >= 0 && x.width >= 0;
}

static bool counts_here(const NexrtPagesArgs& x, int n) { return static_cast<int64_t>(n) * x.width <= kSmallTable && x.pages <= 16 * kSmallTable; }

// Counts the pages that rows name, and writes the rows that go on, where the planning CTA does not.
static int rows_launch(const NexrtPagesArgs& x, const PageTable& t, const int* parents, int* out, int* refs, int n, cudaStream_t st) {
    if (counts_here(x, n) && n > 0) return 0;
    if (x.pages > 0)
        if (const cudaError_t e = cudaMemsetAsync(refs, 0, sizeof(int) * static_cast<size_t>(x.pages), st); e != cudaSuccess) return static_cast<int>(e);
    if (n == 0 || x.width == 0) return 0;
    const int cols = (x.width + 255) / 256;
    return launch(fork_rows_kernel, dim3(cols < 64 ? cols : 64, n < 65535 ? n : 65535), dim3(256), 0, st, t, static_cast<const int*>(x.lens), parents, out, x.out_row, refs, n,
                  static_cast<int*>(x.status));
}

}  // namespace nexrt

using namespace nexrt;

extern "C" int nexrt_page_fork(const NexrtPagesArgs* x, void* stream) {
    if (!pool_ok(*x) || x->rows_out < 0 || x->rows_out > kPlanRows) return cudaErrorInvalidValue;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const PageTable t = {static_cast<const int*>(x->table), x->table_row, x->rows, x->width, x->slots, x->pages};
    if (const int e = rows_launch(*x, t, static_cast<const int*>(x->parents), static_cast<int*>(x->table_out), static_cast<int*>(x->refs), x->rows_out, st)) return e;
    if (x->rows_out == 0) return 0;
    ForkPlan p = {};
    p.t = t; p.lens = static_cast<const int*>(x->lens); p.parents = static_cast<const int*>(x->parents); p.grow = static_cast<const int*>(x->grow);
    p.table = static_cast<int*>(x->table_out); p.table_stride = x->out_row; p.lens_out = static_cast<int*>(x->lens_out); p.refs = static_cast<int*>(x->refs);
    p.free_list = static_cast<int*>(x->scratch); p.copies = p.free_list + x->pages; p.n_copies = p.copies + 3 * x->rows_out;
    p.writers = p.n_copies + 1; p.first = p.writers + x->pages;
    p.status = static_cast<int*>(x->status); p.grown = static_cast<int*>(x->grown); p.n = x->rows_out; p.grow_all = x->grow_all; p.pages = x->pages; p.count = counts_here(*x, x->rows_out);
    // up to a row a warp few threads plan sooner, barriers are what it waits for: 8 rows 9.8 us, by 1024 threads 10.6 (24 rows 10.0 and 9.1)
    const bool few = x->rows_out <= 8 && x->pages <= 8 * kSmallTable;
    if (const int e = launch(fork_plan_kernel, dim3(1), dim3(few ? 256 : kPlanThreads), sizeof(int) * 2 * x->rows_out, st, p)) return e;
    PageMove m = {};
    m.copies = p.copies; m.n_copies = p.n_copies; m.n = x->rows_out;
    return move_launch(m, *x, false, st);
}

extern "C" int nexrt_page_compact(const NexrtPagesArgs* x, void* stream) {
    if (!pool_ok(*x)) return cudaErrorInvalidValue;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int* refs = static_cast<int*>(x->scratch);
    const PageTable t = {static_cast<const int*>(x->table), x->table_row, x->rows, x->width, x->slots, x->pages};
    if (const int e = rows_launch(*x, t, nullptr, nullptr, refs, x->rows, st)) return e;
    const int64_t pages = x->pages;
    CompactPlan p = {};
    p.refs = refs; p.refs_out = static_cast<int*>(x->refs); p.remap = static_cast<int*>(x->remap);
    p.holes = refs + pages; p.copies = refs + 2 * pages; p.n_copies = refs + 5 * pages;
    p.live = static_cast<int*>(x->live); p.pages = x->pages;
    p.t = t; p.lens = static_cast<const int*>(x->lens); p.count = x->rows > 0 && counts_here(*x, x->rows); p.status = static_cast<int*>(x->status);
    if (const int e = launch(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p)) return e;
    PageMove m = {};
    m.copies = p.copies; m.n_copies = p.n_copies; m.n = x->pages;
    m.t = t; m.lens = static_cast<const int*>(x->lens); m.remap = p.remap; m.table_out = static_cast<int*>(x->table_out); m.table_stride = x->out_row;
    return move_launch(m, *x, true, st);
}

extern "C" int nexrt_page_copy(const NexrtPagesArgs* x, void* stream) {
    if (!pool_ok(*x)) return cudaErrorInvalidValue;
    const int n = x->rows;
    if (n == 0) return 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int* copies = static_cast<int*>(x->scratch);
    int* source = copies + static_cast<int64_t>(3) * n;
    if (const int e = launch(copy_list_kernel, dim3(1), dim3(n < kPlanThreads ? (n + 31) / 32 * 32 : kPlanThreads), 0, st, static_cast<const int*>(x->table),
                             static_cast<const int*>(x->lens), n, x->pages, copies, source, source + x->pages, static_cast<int*>(x->status)))
        return e;
    PageMove m = {};
    m.copies = copies; m.n = n;
    return move_launch(m, *x, true, st);
}
