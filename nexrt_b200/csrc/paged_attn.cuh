// Attention of one new token of every sequence over a key-value cache in pages.
//
//   s_j = scale q.k_j;  s_j = cap tanh(s_j / cap);  s_j -= slope (len - 1 - j);   j in [max(0, len - window), len)
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   lse = m + log sum_j exp(s_j - m)
//
// Bound by the bytes of K and V: with 16 query heads on a key head there are eight multiply-adds a byte.  So the design is for the
// stream.  The keys of the whole batch are cut into equal ranges, one per resident CTA, whatever the sequences' lengths; a CTA
// walks its range item by item (sequence, key head, up to 16 query heads).  A warp has a ring of 16-key half tiles (K, V, K, V ...)
// of its own in shared memory, filled row by row through the page table, so it waits for no other warp, and pages of any size, also
// ones that end inside a tile, cost the same.  From 192 dims up a row is one bulk copy (cp.async.bulk: one instruction for the 16
// rows of a half tile; 200K keys of 256 dims 76 us, by 16-byte cp.async 92); shorter rows go by cp.async (a ragged batch of 128 dims
// 97 us, by bulk copies of 256 bytes 145).  Rows are padded by 16 bytes: ldmatrix and the copies meet no bank twice.
//
// Products are mma.sync m16n8k16: a tensor-memory product wants 64 rows at least, here are 16 at most.  Scores have the query rows on
// the M side, values are transposed (dims on M, rows on N), so that the score fragments are the value product's operands without a
// shuffle.  P enters as a 16-bit pair hi + lo: one 16-bit P would add an error as large as the result's own rounding.  Maximum, sum
// and accumulators are 32 bits.
//
// fp16 has no numbers between 0 and 2^-24: beside a key that outweighs all others by 17 nats their weights would vanish from the
// numerator, and where that key's value is near zero they are the result.  So there exp(s_j - m) is formed against a reference of the
// row that goes down as well as up, the same in numerator and sum, and the largest weight of a tile lies between 2^6 and 2^15; weights of the
// same tile below 2^-13, which the pair does not hold to 2^-12, go through the value product once more against a lower reference.  32-bit sums
// hold the maximum 60 binary orders above the reference.  It costs 2 % under sustained load with 128 dims (ragged batch
// 98.8 -> 101.1 us), 3 % with 64 (64 sequences of 2000 keys 37.3 -> 38.3), 12 % where a steep bias moves the reference in every tile (the
// ragged batch with cap and bias 80 -> 90).
//
// An item that lies in one CTA's range is written at once; of one that is cut, each CTA leaves its part (at most two parts a
// CTA) and a second kernel joins them in the order of the keys: results do not depend on timing (they do, in the last bits, on where the
// batch's lengths cut an item).
//
// Measured: 200K keys, 2 key heads of 256, 32 query heads: 75 us, 5.4 TB/s of keys and values, 0.84 of copy rate (the rings alone fill in
// 64); 48 sequences of 0 to 16384 keys, 8 heads of 128, fp16: 93 us, 0.86; 16 sequences of up to
// 4097 keys, 8 heads of 64, capped and biased: 16 us; one sequence of 1100 keys: 9.2 us, two launches and their chains.
#pragma once

#include <type_traits>

#include "api.h"
#include "paged.cuh"

namespace nexrt {

constexpr int kPaWarps = 4;
constexpr int kPaThreads = kPaWarps * 32;
constexpr int kPaRows = 16;                 // query rows of an item
constexpr int kTile = 16;                   // keys of a warp's tile
constexpr uint32_t kNoRow = 0xffffffffu;
static_assert(kChunk == kPaWarps * kTile, "a chunk is one tile a warp");

struct PagedAttnArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;                              // may be null
    int64_t q_b, q_h, o_b, o_h, head_s, lse_b;
    uint32_t page_s, slot_s;                 // of a pool, in units of 16 bytes: a row's place is 32 bits wide
    PageTable table;
    const int* lens;
    const float* slopes;                     // may be null
    float *ws_o, *ws_ml;                     // parts: [2 grid][16][dim], [2 grid][16][2]
    int4* cuts;                              // [min(grid, items)] of a cut item: sequence, first head, first CTA, parts; parts 0: none
    int by_item;                             // cuts of items, not of CTAs
    int* status;
    int seqs, kv_heads, group, head_groups, window, grid;
    float scale, softcap;
};

// CTAs on an SM, and half tiles of a warp's ring: what registers and shared memory hold.  (64 dims: three CTAs take 0.8 of the time of
// two; 128 dims: two with rings of four 94.9, three 99.9, two with rings of six 96.4.)
constexpr int resident_ctas(int dim) { return dim == 64 ? 3 : 2; }
template <int D> constexpr int ring_depth() { return D == 256 ? 3 : (D == 64 ? 6 : 4); }
template <int D> constexpr int half_bytes() { return kTile * (D * 2 + 16); }
template <int D> constexpr size_t ring_bytes() { return static_cast<size_t>(kPaWarps) * ring_depth<D>() * half_bytes<D>(); }
template <int D> constexpr size_t merge_bytes() { return sizeof(float) * kPaWarps * kPaRows * (D + 4); }
template <int D> constexpr size_t paged_smem() { return (ring_bytes<D>() > merge_bytes<D>() ? ring_bytes<D>() : merge_bytes<D>()) + D / 16 * 512; }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The larger of two; NaN if one is: a score that is not a number is to show in the output, not to vanish in a maximum.
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
// (x, y) as a pair of 16-bit values and the pair of what that leaves
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo, __half) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// fp16: a row's largest score of a tile lies kRefLeast to kRefMost binary orders above the reference, kRefPlace where it is set, and no
// reference lies more than kRefSpan below the highest so far.
constexpr float kRefLeast = 6.f, kRefMost = 15.f;
constexpr int kRefPlace = 11, kRefSpan = 45;
// A weight that fp16 holds too coarsely, and one that is too small to matter, in binary orders above the reference.
constexpr float kLow = -13.f, kNothing = -70.f;
// The logarithm of l 2^ref.  (fp16: l may be 2^70, and its logarithm's last bits would be as large as those of a far larger result.)
template <typename T> __device__ __forceinline__ float log_of(float ref, float l) {
    if (l == 0.f) return -INFINITY;
    int e = 0;
    if constexpr (std::is_same<T, __half>::value) l = frexpf(l, &e);
    return ((ref + static_cast<float>(e)) + log2f(l)) * 0.6931471805599453f;
}

// ---- where a CTA's range lies ------------------------------------------------------------------------------------------
// Chunks of one item of sequence b, and what all its items count.
__device__ __forceinline__ int seq_chunks(const PagedAttnArgs& a, int b) {
    int lo, hi;
    key_span(a.lens[b], static_cast<int64_t>(a.table.width) * a.table.page, a.window, lo, hi);
    return chunks_of(lo, hi);
}
__device__ __forceinline__ int64_t seq_cost(const PagedAttnArgs& a, int items, int b) { return static_cast<int64_t>(cost_of(seq_chunks(a, b))) * items; }

// Sum over the CTA's threads of `v`, and the sum over the threads before this one.  Every thread calls it.  red: 32 words.
__device__ __forceinline__ int64_t scan_add(int64_t v, int64_t* red, int64_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 31) red[warp] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int i = 0; i < n; ++i) {
        if (i < warp) before += red[i];
        total += red[i];
    }
    return before + s - v;
}

struct Place {
    int seq;            // sequence
    int64_t first;      // units in front of it
};

// Units of the whole batch; with up to as many sequences as threads `cost` and `at` are those of this thread's sequence and of the ones in front.
__device__ __forceinline__ int64_t total_cost(const PagedAttnArgs& a, int items, int64_t* red, int64_t& cost, int64_t& at) {
    cost = at = 0;
    if (a.seqs == 1) {
        if (threadIdx.x == 0) cost = seq_cost(a, items, 0);
        return seq_cost(a, items, 0);
    }
    int64_t total;
    for (int b = threadIdx.x; b < a.seqs; b += blockDim.x) cost += seq_cost(a, items, b);
    at = scan_add(cost, red, total);
    return total;
}

// The sequence that holds unit x (x < total).  place: shared.
__device__ __forceinline__ Place find_seq(const PagedAttnArgs& a, int items, int64_t x, int64_t cost, int64_t at, int64_t* red, Place* place) {
    if (a.seqs == 1) return {0, 0};
    if (a.seqs <= static_cast<int>(blockDim.x)) {
        if (x >= at && x < at + cost) *place = {static_cast<int>(threadIdx.x), at};
    } else {
        int64_t before = 0;
        for (int b0 = 0; b0 < a.seqs; b0 += blockDim.x) {
            const int b = b0 + threadIdx.x;
            const int64_t n = b < a.seqs ? seq_cost(a, items, b) : 0;
            int64_t total;
            const int64_t first = before + scan_add(n, red, total);
            if (x >= first && x < first + n) *place = {b, first};
            before += total;
            if (x < before) break;
        }
    }
    __syncthreads();
    return *place;
}

// A ring place's copies have arrived.  Bounded: a wait that runs out latches kStatusPipeTimeout, and those behind it are short; the
// result is not to be used then, but every copy has been waited for when the kernel ends.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t phase, bool& late, int* status) {
    bool ok = false;
    for (int i = late ? 1 << 10 : 1 << 20; i > 0 && !ok; --i) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(phase) : "memory");
        ok = done != 0;
    }
    if (!ok) {
        late = true;
        if (status) atomicCAS(status, 0, static_cast<int>(kStatusPipeTimeout));
    }
}

template <typename T, int D, int NTR, bool MODS>
__global__ void __launch_bounds__(kPaThreads, resident_ctas(D)) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int KS = D / 16, R = ring_depth<D>(), PITCH = D * 2 + 16, HALF = half_bytes<D>(), CPR = D / 8;
    extern __shared__ __align__(128) unsigned char pa_smem[];
    uint4* const qf = reinterpret_cast<uint4*>(pa_smem);                           // query fragments, 512 bytes a k step
    unsigned char* const ring = pa_smem + KS * 512;
    __shared__ int64_t red[32];
    __shared__ Place place;
    __shared__ float part_m[kPaWarps][kPaRows], part_l[kPaWarps][kPaRows];
    __shared__ uint64_t bars[kPaWarps][R];
    constexpr bool kHalf = std::is_same<T, __half>::value;
    __shared__ float low_s[kHalf ? kPaWarps : 1][kHalf ? NTR * 4 : 1][32];         // weights that wait for a lower reference
    constexpr bool kBulk = D >= 192;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t bar0 = static_cast<uint32_t>(__cvta_generic_to_shared(&bars[warp][0]));
    if (kBulk) {
        if (lane < R) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + lane * 8) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
    }
    pdl_launch_dependents();
    pdl_wait();
    const int items = a.kv_heads * a.head_groups;
    const int64_t room = static_cast<int64_t>(a.table.width) * a.table.page;

    int64_t my_cost, my_at;
    const int64_t total = total_cost(a, items, red, my_cost, my_at);
    const int n = active_ctas(total, gridDim.x);
    int64_t x = 0, x_end = 0, first = 0;
    int b = 0;
    if (total > 0 && static_cast<int>(blockIdx.x) < n) {
        x = range_begin(total, blockIdx.x, n);
        x_end = range_begin(total, blockIdx.x + 1, n);
        const Place start = find_seq(a, items, x, my_cost, my_at, red, &place);
        b = start.seq;
        first = start.first;
    }

    const uint32_t my_ring = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + warp * R * HALF;
    // ldmatrix row of this lane: keys on the rows, V's read transposed
    const uint32_t k_lane = ((lane & 7) + ((lane >> 4) << 3)) * PITCH + ((lane >> 3) & 1) * 16;
    int to = 0, use = 0;                                               // places of the ring: of the next half that is fed, and used
    uint32_t phases = 0;                                               // bit: phase of a place's barrier
    bool late = false;
    int4 cut = make_int4(0, 0, 0, 0);                                  // the item that this CTA begins and another one ends

    while (x < x_end) {
        int lo, hi;
        key_span(a.lens[b], room, a.window, lo, hi);
        const int per = chunks_of(lo, hi), cost = cost_of(per);
        if (x >= first + static_cast<int64_t>(cost) * items) {       // also sequences without keys
            first += static_cast<int64_t>(cost) * items;
            ++b;
            continue;
        }
        const int item = static_cast<int>(quotient(x - first, cost));
        const int64_t item0 = first + static_cast<int64_t>(item) * cost;
        int c0, c1;
        item_part(item0, per, x, x_end, c0, c1);
        x = item0 + cost;
        if (c1 <= c0) continue;                                       // the range ends in front of the item's first chunk
        const int kvh = item / a.head_groups, h0 = kvh * a.group + item % a.head_groups * kPaRows;
        const int rows = min(kPaRows, (kvh + 1) * a.group - h0);
        const int key0 = (lo / kChunk + c0) * kChunk + warp * kTile;  // first key of this warp's tile of chunk c0
        const int tiles = c1 - c0;
        const char* const kbase = static_cast<const char*>(a.k) + kvh * a.head_s * 2;
        const char* const vbase = static_cast<const char*>(a.v) + kvh * a.head_s * 2;

        // ---- page lookups one tile ahead of the copies: lane l (mod 16) finds the row of key l of the tile, in units of 16 bytes
        auto find = [&](int tile) -> uint32_t {
            const int p = key0 + tile * kChunk + (lane & 15);
            if (tile >= tiles || p < lo || p >= hi) return kNoRow;
            const int j = static_cast<int>(static_cast<uint32_t>(p) / static_cast<uint32_t>(a.table.page)), page = page_at(a.table, b, j);
            if (page < 0) {
                if (a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
                return kNoRow;
            }
            return static_cast<uint32_t>(page) * a.page_s + static_cast<uint32_t>(p - j * a.table.page) * a.slot_s;
        };
        // the first tiles' lookups side by side.  at: rows of the tile that is being copied, next: of the one behind it; newest: which
        // of its keys are there
        constexpr int Q = R / 2;
        uint32_t at = kNoRow, newest = 0, ahead[Q + 1];
#pragma unroll
        for (int i = 0; i <= Q; ++i) ahead[i] = find(i);
        auto copy = [&](int half) {
            if (half < 2 * tiles) {
                const char* const base = (half & 1) ? vbase : kbase;
                const uint32_t ring_to = my_ring + to * HALF;
                if (kBulk) {
                    const uint32_t bar = bar0 + to * 8;
                    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(__popc(newest) * D * 2) : "memory");
                    if ((half & 1) && newest != 0xffffu) {             // values of absent keys meet a P of zero: they have to be numbers
                        for (int i = lane; i < kTile * CPR; i += 32)
                            if (!(newest >> (i / CPR) & 1)) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring_to + i / CPR * PITCH + i % CPR * 16), "r"(0) : "memory");
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    __syncwarp();
                    if (lane < kTile && at != kNoRow)
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                     ::"r"(ring_to + lane * PITCH), "l"(base + static_cast<uint64_t>(at) * 16), "r"(D * 2), "r"(bar) : "memory");
                } else {
#pragma unroll
                    for (int i = 0; i < kTile * CPR / 32; ++i) {
                        const int r = i * (32 / CPR) + lane / CPR, c = lane % CPR;
                        const uint32_t row = __shfl_sync(0xffffffffu, at, r);
                        cp16(ring_to + r * PITCH + c * 16, base + c * 16 + (row == kNoRow ? 0ull : static_cast<uint64_t>(row) * 16), row != kNoRow);
                    }
                }
                to = to + 1 == R ? 0 : to + 1;
            }
            if (!kBulk) cp_commit();
        };
        // halves 0 .. R-2 are on their way before the first is used.  masks: which keys are there, 16 bits a tile, of the tile in use and
        // of the R / 2 - 1 behind it
        uint64_t masks = 0;
#pragma unroll
        for (int i = 0; i < R - 1; ++i) {
            if (i % 2 == 0) {
                at = ahead[i / 2];
                newest = __ballot_sync(0xffffffffu, at != kNoRow) & 0xffffu;
                masks |= static_cast<uint64_t>(newest) << (i * 8);
            }
            copy(i);
        }
        uint32_t next = ahead[Q];
        int fed = R - 1;
        auto feed = [&]() {
            if (!(fed & 1)) {
                at = next;
                next = find(fed / 2 + 1);
                newest = __ballot_sync(0xffffffffu, at != kNoRow) & 0xffffu;
            }
            copy(fed++);
        };
        auto arrived = [&]() {
            if (kBulk) bar_wait(bar0 + use * 8, phases >> use & 1, late, a.status);
            else cp_wait<R - 2>();
            __syncwarp();
        };
        auto used = [&]() {
            phases ^= 1u << use;
            use = use + 1 == R ? 0 : use + 1;
        };

        // ---- query fragments
        {
            const T* q = static_cast<const T*>(a.q) + b * a.q_b;
            const bool pairs = ((reinterpret_cast<uintptr_t>(q) >> 1 | a.q_h) & 1) == 0;
#pragma unroll
            for (int i0 = 0; i0 < KS * 32; i0 += kPaThreads) {
                const int i = i0 + threadIdx.x, ks = i >> 5, l = i & 31, gr = l >> 2, d = ks * 16 + (l & 3) * 2;
                uint32_t f[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int r = gr + (u & 1) * 8, dd = d + (u >> 1) * 8;
                    f[u] = 0;
                    if (r < rows && ks < KS) {
                        const T* s = q + (h0 + r) * a.q_h + dd;
                        if (pairs) f[u] = *reinterpret_cast<const uint32_t*>(s);
                        else f[u] = reinterpret_cast<const unsigned short*>(s)[0] | static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(s)[1]) << 16;
                    }
                }
                if (ks < KS) qf[i] = make_uint4(f[0], f[1], f[2], f[3]);
            }
        }
        __syncthreads();

        float o[KS][NTR][4];
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int r = 0; r < NTR; ++r) o[j][r][0] = o[j][r][1] = o[j][r][2] = o[j][r][3] = 0.f;
        float mx[NTR], highest[NTR], sum[NTR], slope[NTR];             // mx: what weights are formed against: the maximum so far, of fp16 the reference
#pragma unroll
        for (int r = 0; r < NTR; ++r) {
            mx[r] = highest[r] = -INFINITY;
            sum[r] = 0.f;
            slope[r] = MODS && a.slopes && g + 8 * r < rows ? a.slopes[h0 + g + 8 * r] * 1.4426950408889634f : 0.f;
        }
        const float scale2 = a.scale * 1.4426950408889634f, to_cap = a.scale / a.softcap, cap2 = a.softcap * 1.4426950408889634f;
        // with few registers' worth of queries they stay there
        constexpr bool kHold = KS * NTR <= 16;
        uint32_t qr[kHold ? KS : 1][4];
        if (kHold) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint4 q4 = qf[ks * 32 + lane];
                qr[ks][0] = q4.x; qr[ks][1] = NTR == 1 ? 0u : q4.y; qr[ks][2] = q4.z; qr[ks][3] = NTR == 1 ? 0u : q4.w;
            }
        }

        for (int i = 0; i < tiles; ++i) {
            const uint32_t have = static_cast<uint32_t>(masks) & 0xffffu;
            // ---- scores
            arrived();
            feed();
            float s[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
            const uint32_t kt = my_ring + use * HALF + k_lane;
            used();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t kf[4];
                ldsm4(kf, kt + ks * 32);
                if (!kHold) {
                    const uint4 q4 = qf[ks * 32 + lane];
                    qr[0][0] = q4.x; qr[0][1] = q4.y; qr[0][2] = q4.z; qr[0][3] = q4.w;
                }
                mma16816(s[0], qr[kHold ? ks : 0], kf[0], kf[1], T());
                mma16816(s[1], qr[kHold ? ks : 0], kf[2], kf[3], T());
            }
            // ---- mask and running softmax: row g + 8 r has its 16 scores in the four lanes of a g
            uint32_t ph[NTR][2], pl[NTR][2];
            float corr[NTR];
            int again = 0;                                             // bit r: rows g + 8 r have weights that wait
            const float dist = static_cast<float>(hi - 1 - (key0 + i * kChunk) - 2 * t);   // of the lane's first key (exact up to 2^24)
#pragma unroll
            for (int r = 0; r < NTR; ++r) {
                float v[4] = {s[0][2 * r], s[0][2 * r + 1], s[1][2 * r], s[1][2 * r + 1]};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int key = (u >> 1) * 8 + 2 * t + (u & 1);
                    if (MODS) {
                        const float y = a.softcap > 0.f ? cap2 * tanhf(v[u] * to_cap) : v[u] * scale2;
                        v[u] = y - slope[r] * (dist - static_cast<float>((u >> 1) * 8 + (u & 1)));
                    } else {
                        v[u] *= scale2;
                    }
                    if (!(have >> key & 1)) v[u] = -INFINITY;
                }
                auto row_max = [&](float m) {
                    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    return max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
                };
                corr[r] = 1.f;
                if constexpr (kHalf) {
                    // as a rule the references of all rows g + 8 r stay and no weight has to wait: that is looked up beside the exponentials
                    float p[4];
                    bool low = false;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        p[u] = v[u] - mx[r];
                        low |= p[u] < kLow && p[u] > kNothing;
                    }
                    const float m = max_nan(max_nan(p[0], p[1]), max_nan(p[2], p[3]));
                    const uint32_t above = __ballot_sync(0xffffffffu, !(m <= kRefMost) || low), there = __ballot_sync(0xffffffffu, m >= kRefLeast), pairs = there | there >> 1;
#pragma unroll
                    for (int u = 0; u < 4; ++u) p[u] = exp2_ftz(p[u]);
                    if (above != 0 || ((pairs | pairs >> 2) & 0x11111111u) != 0x11111111u) {
                        // (a whole number, so that differences of references are exact; a row without a key in this tile keeps its own)
                        const float top = row_max(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])));
                        const bool fits = top <= mx[r] + kRefMost && (top >= mx[r] + kRefLeast || top == -INFINITY);
                        const float ref = fits ? mx[r] : rintf(max_nan(top - kRefPlace, highest[r] - kRefSpan)), shift = ref == -INFINITY ? 0.f : ref;
                        highest[r] = max_nan(highest[r], ref);
                        if (mx[r] != ref) corr[r] = exp2_ftz(mx[r] - shift);
                        mx[r] = ref;
                        low = false;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            p[u] = v[u] - shift;
                            low |= p[u] < kLow && p[u] > kNothing;
                        }
                        const bool waits = __any_sync(0xffffffffu, low);
                        if (waits) again |= 1 << r;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const bool late = p[u] < kLow && p[u] > kNothing;
                            p[u] = exp2_ftz(p[u]);
                            v[u] = late ? 0.f : p[u];
                            if (waits) low_s[warp][r * 4 + u][lane] = late ? p[u] : 0.f;
                        }
                        sum[r] = fmaf(sum[r], corr[r], (p[0] + p[1]) + (p[2] + p[3]));
                    } else {
                        sum[r] += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
                        for (int u = 0; u < 4; ++u) v[u] = p[u];
                    }
                } else {
                    const float m = max_nan(row_max(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3]))), mx[r]), shift = m == -INFINITY ? 0.f : m;
                    if (mx[r] != m) corr[r] = exp2_ftz(mx[r] - shift);
                    mx[r] = m;
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] = exp2_ftz(v[u] - shift);
                    sum[r] = fmaf(sum[r], corr[r], (v[0] + v[1]) + (v[2] + v[3]));
                }
                split2(v[0], v[1], ph[r][0], pl[r][0], T());
                split2(v[2], v[3], ph[r][1], pl[r][1], T());
            }
            // the accumulators of this lane are of rows 2t and 2t + 1 (mod 8): their factors are with lanes 8t and 8t + 4
            auto rescale = [&]() {
#pragma unroll
                for (int r = 0; r < NTR; ++r) {
                    if (__any_sync(0xffffffffu, corr[r] != 1.f)) {
                        const float f0 = __shfl_sync(0xffffffffu, corr[r], 8 * t), f1 = __shfl_sync(0xffffffffu, corr[r], 8 * t + 4);
#pragma unroll
                        for (int j = 0; j < KS; ++j) {
                            o[j][r][0] *= f0;
                            o[j][r][1] *= f1;
                            o[j][r][2] *= f0;
                            o[j][r][3] *= f1;
                        }
                    }
                }
            };
            rescale();
            // ---- values
            arrived();
            feed();
            const uint32_t vt = my_ring + use * HALF + k_lane;
            used();
            auto add_values = [&]() {
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    uint32_t vf[4];
                    ldsm4t(vf, vt + j * 32);
#pragma unroll
                    for (int r = 0; r < NTR; ++r) {
                        mma16816(o[j][r], vf, ph[r][0], ph[r][1], T());
                        mma16816(o[j][r], vf, pl[r][0], pl[r][1], T());
                    }
                }
            };
            add_values();
            // ---- the weights that wait, the largest of a row brought to 2^11 (a lane reads back what it wrote).  What is too low even then is less than
            // 2^-43 of the tile's largest weight, and off by less than 2^-54 of it.
            if constexpr (kHalf) {
                if (again) {
#pragma unroll
                    for (int r = 0; r < NTR; ++r) {
                        corr[r] = 1.f;
                        ph[r][0] = ph[r][1] = pl[r][0] = pl[r][1] = 0u;
                        if (!(again >> r & 1)) continue;
                        float v[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) v[u] = low_s[warp][r * 4 + u][lane];
                        float m = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                        int down = 0;
                        if (m > 0.f) down = max(0, min(kRefPlace + 127 - static_cast<int>(__float_as_uint(m) >> 23), static_cast<int>(mx[r] - highest[r]) + kRefSpan));
                        corr[r] = __uint_as_float(static_cast<uint32_t>(127 + down) << 23);
                        mx[r] -= static_cast<float>(down);
                        sum[r] *= corr[r];
                        split2(v[0] * corr[r], v[1] * corr[r], ph[r][0], pl[r][0], T());
                        split2(v[2] * corr[r], v[3] * corr[r], ph[r][1], pl[r][1], T());
                    }
                    rescale();
                    add_values();
                }
            }
            masks = masks >> 16 | static_cast<uint64_t>(newest) << (16 * (R / 2 - 1));
        }
        if (!kBulk) cp_wait<0>();

        // ---- join the warps: rings are free from here on
#pragma unroll
        for (int r = 0; r < NTR; ++r) {
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
            if (t == 0) {
                part_m[warp][g + 8 * r] = mx[r];
                part_l[warp][g + 8 * r] = sum[r];
            }
        }
        __syncthreads();
        float* const merge = reinterpret_cast<float*>(ring);           // [warp][row][D + 4]
#pragma unroll
        for (int r = 0; r < NTR; ++r) {
            float f[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = 2 * t + u + 8 * r;
                float m = part_m[0][row];
#pragma unroll
                for (int w = 1; w < kPaWarps; ++w) m = max_nan(m, part_m[w][row]);
                f[u] = m == -INFINITY ? 0.f : exp2f(part_m[warp][row] - m);
            }
            float* const row0 = merge + (warp * kPaRows + 2 * t + 8 * r) * (D + 4);
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                row0[j * 16 + g] = o[j][r][0] * f[0];
                row0[D + 4 + j * 16 + g] = o[j][r][1] * f[1];
                row0[j * 16 + 8 + g] = o[j][r][2] * f[0];
                row0[D + 4 + j * 16 + 8 + g] = o[j][r][3] * f[1];
            }
        }
        __syncthreads();
        const bool whole = c0 == 0 && c1 == per;
        // a part whose item began in front of this range is the CTA's first, else its last
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (c0 == 0);
        for (int i = threadIdx.x; i < rows * (D / 4); i += kPaThreads) {
            const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) {
                const float4 p = *reinterpret_cast<const float4*>(merge + (w * kPaRows + row) * (D + 4) + d);
                y.x += p.x; y.y += p.y; y.z += p.z; y.w += p.w;
                m = max_nan(m, part_m[w][row]);
            }
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) l += m == -INFINITY ? 0.f : part_l[w][row] * exp2f(part_m[w][row] - m);
            if (whole) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                T* out = static_cast<T*>(a.out) + b * a.o_b + (h0 + row) * a.o_h + d;
                out[0] = static_cast<T>(y.x * inv); out[1] = static_cast<T>(y.y * inv); out[2] = static_cast<T>(y.z * inv); out[3] = static_cast<T>(y.w * inv);
                if (a.lse && d == 0) a.lse[b * a.lse_b + h0 + row] = log_of<T>(m, l);
            } else {
                *reinterpret_cast<float4*>(a.ws_o + (slot * kPaRows + row) * D + d) = y;
                if (d == 0) {
                    a.ws_ml[(slot * kPaRows + row) * 2] = m;
                    a.ws_ml[(slot * kPaRows + row) * 2 + 1] = l;
                }
            }
        }
        if (c0 == 0) {
            const int parts = whole ? 0 : owner_of(item0 + cost - 1, total, n) - static_cast<int>(blockIdx.x) + 1;
            cut = make_int4(b, h0, blockIdx.x, parts);
            if (a.by_item && threadIdx.x == 0) a.cuts[b * items + item] = cut;
        }
        // the next item's copies go where these values lay
        if (kBulk) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }

    if (!a.by_item && threadIdx.x == 0) a.cuts[blockIdx.x] = cut;

    // ---- sequences without keys: zeros, and an lse of -infinity
    for (int s = blockIdx.x; s < a.seqs; s += gridDim.x) {
        if (a.lens[s] > room && threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
        if (seq_chunks(a, s)) continue;
        const int heads = a.kv_heads * a.group;
        for (int i = threadIdx.x; i < heads * D; i += kPaThreads) static_cast<T*>(a.out)[s * a.o_b + i / D * a.o_h + i % D] = static_cast<T>(0.f);
        if (a.lse)
            for (int i = threadIdx.x; i < heads; i += kPaThreads) a.lse[s * a.lse_b + i] = -INFINITY;
        if (a.by_item)
            for (int i = threadIdx.x; i < items; i += kPaThreads) a.cuts[s * items + i] = make_int4(0, 0, 0, 0);
    }
}

// One CTA per (cut, row): joins the parts of an item that was cut.  The parts' maxima and sums first, then their accumulators with
// D / 4 lanes of four dims side by side and the parts shared out over the groups of lanes.
constexpr int kMaxCtas = 1024;

template <typename T, int D, int kJoinThreads>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int LANES = D / 4, GROUPS = kJoinThreads / LANES;
    __shared__ float weight[kMaxCtas], top_s[kJoinThreads / 32], sum_s[kJoinThreads / 32];
    __shared__ float4 acc_s[GROUPS][LANES];
    pdl_launch_dependents();
    pdl_wait();
    const int4 cut = a.cuts[blockIdx.x];
    const int b = cut.x, row = blockIdx.y, h = cut.y + row, cta0 = cut.z, parts = cut.w;
    if (parts == 0 || h >= (cut.y / a.group + 1) * a.group) return;
    // part p: row of the scratch.  Where an item begins it is its CTA's second part, elsewhere the first
    auto slot_of = [&](int p) { return (2 * static_cast<int64_t>(cta0 + p) + (p == 0)) * kPaRows + row; };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = threadIdx.x % LANES, grp = threadIdx.x / LANES;
    // the first parts' accumulators are on their way while the weights are made
    constexpr int kEarly = 4;
    float4 early[kEarly];
#pragma unroll
    for (int i = 0; i < kEarly; ++i) {
        early[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (grp < GROUPS && grp + i * GROUPS < parts) early[i] = *reinterpret_cast<const float4*>(a.ws_o + slot_of(grp + i * GROUPS) * D + d * 4);
    }
    float m = -INFINITY, l = 0.f;
    for (int p = threadIdx.x; p < parts; p += kJoinThreads) {
        weight[p] = a.ws_ml[slot_of(p) * 2];
        m = max_nan(m, weight[p]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) top_s[warp] = m;
    __syncthreads();
    m = top_s[0];
#pragma unroll
    for (int i = 1; i < kJoinThreads / 32; ++i) m = max_nan(m, top_s[i]);
    const float shift = m == -INFINITY ? 0.f : m;
    for (int p = threadIdx.x; p < parts; p += kJoinThreads) {
        const float w = exp2f(weight[p] - shift);
        weight[p] = w;
        l = fmaf(a.ws_ml[slot_of(p) * 2 + 1], w, l);
    }
    l = warp_sum(l);
    if (lane == 0) sum_s[warp] = l;
    __syncthreads();
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp < GROUPS) {
        auto add = [&](const float4& v, int p) {
            const float w = weight[p];
            y.x = fmaf(v.x, w, y.x); y.y = fmaf(v.y, w, y.y); y.z = fmaf(v.z, w, y.z); y.w = fmaf(v.w, w, y.w);
        };
#pragma unroll
        for (int i = 0; i < kEarly; ++i)
            if (grp + i * GROUPS < parts) add(early[i], grp + i * GROUPS);
#pragma unroll 4
        for (int p = grp + kEarly * GROUPS; p < parts; p += GROUPS) add(*reinterpret_cast<const float4*>(a.ws_o + slot_of(p) * D + d * 4), p);
        acc_s[grp][d] = y;
    }
    __syncthreads();
    if (grp != 0) return;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) l += sum_s[i];
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
        const float4 v = acc_s[i][d];
        y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = static_cast<T*>(a.out) + b * a.o_b + h * a.o_h + d * 4;
    out[0] = static_cast<T>(y.x * inv); out[1] = static_cast<T>(y.y * inv); out[2] = static_cast<T>(y.z * inv); out[3] = static_cast<T>(y.w * inv);
    if (a.lse && d == 0) a.lse[b * a.lse_b + h] = log_of<T>(m, l);
}

template <typename T, int D> static int paged_launch(const PagedAttnArgs& a, bool join, cudaStream_t st) {
    const bool mods = a.softcap > 0.f || a.slopes != nullptr;
    const dim3 grid(a.grid), block(kPaThreads);
    const size_t smem = paged_smem<D>();
    int e;
    if (a.group <= 8) e = mods ? launch(paged_attn_kernel<T, D, 1, true>, grid, block, smem, st, a) : launch(paged_attn_kernel<T, D, 1, false>, grid, block, smem, st, a);
    else e = mods ? launch(paged_attn_kernel<T, D, 2, true>, grid, block, smem, st, a) : launch(paged_attn_kernel<T, D, 2, false>, grid, block, smem, st, a);
    if (e || !join) return e;
    const int rows = a.group < kPaRows ? a.group : kPaRows, items = a.seqs * a.kv_heads * a.head_groups;
    // items cut into dozens of parts are few and want many threads (200K keys in 148 parts: 75.5 us, with 256 threads 80.3), items cut once
    // or twice are many and want many CTAs (a ragged batch 91.9, with 1024 threads where it may 95.0; 1100 keys 9.2 and 10.0).  Between them the
    // line is a matter of a microsecond, and it depends on the dims (4 heads on one, 256 and 1024 threads: 9 sequences of 4000 keys, 33 parts each,
    // of 128 dims 10.6 and 11.6 us, of 256 dims 15.7 and 15.5; 2 of 4000, 66 parts, 9.3 and 8.9, 11.7 and 10.9)
    if (a.by_item && a.grid >= 32 * items) return launch(paged_join_kernel<T, D, 1024>, dim3(items, rows), dim3(1024), 0, st, a);
    return launch(paged_join_kernel<T, D, 256>, dim3(a.by_item ? items : a.grid, rows), dim3(256), 0, st, a);
}

template <typename T> int paged_dispatch(const PagedAttnArgs& a, int dim, bool join, cudaStream_t st) {
    switch (dim) {
        case 64: return paged_launch<T, 64>(a, join, st);
        case 128: return paged_launch<T, 128>(a, join, st);
        case 192: return paged_launch<T, 192>(a, join, st);
        case 256: return paged_launch<T, 256>(a, join, st);
        default: return static_cast<int>(cudaErrorInvalidValue);
    }
}

}  // namespace nexrt
