// Attention of one new token of every sequence over a key-value cache in pages.
//
//   s_j = scale q.k_j;  s_j = cap tanh(s_j / cap);  s_j -= slope (len - 1 - j);   j in [max(0, len - window), len)
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   lse = m + log sum_j exp(s_j - m)
//
// Bound by the bytes of K and V: with at most 16 query heads on a key head there are at most 32 multiply-adds a byte.  So the
// design is for the stream.  The keys of the whole batch are cut into equal ranges, one per resident CTA (two on an SM), whatever
// the sequences' lengths; a CTA walks its range item by item (sequence, key head, up to 16 query heads).  A warp has a ring of
// 16-key half tiles (K, V, K, V ...) of its own in shared memory, filled by 16-byte cp.async row by row through the page table, so
// it waits for nobody, and pages of any size, also ones that end inside a tile, cost the same.  Rows are padded by 16 bytes:
// ldmatrix and the copies meet no bank twice.  Products are mma.sync m16n8k16 - a tensor-memory product wants 128 rows, and here
// are 16 at most: scores with the query rows on the M side, values transposed (dims on M, rows on N), so that the score
// fragments are the value product's operands without a shuffle.  P enters as a 16-bit pair hi + lo: one 16-bit P would add an
// error as large as the result's own rounding.  Maximum, sum and accumulators are 32 bits.
//
// An item that lies in one CTA's range is written at once; of one that is cut, each CTA leaves its part (at most two parts a
// CTA) and a second kernel joins them in the order of the keys, so results do not depend on timing.
#include "api.h"
#include "paged.cuh"

namespace nexrt {

constexpr int kPaWarps = 4;
constexpr int kPaThreads = kPaWarps * 32;
constexpr int kPaRows = 16;                 // query rows of an item
constexpr int kTile = 16;                   // keys of a warp's tile
static_assert(kChunk == kPaWarps * kTile, "a chunk is one tile a warp");

struct PagedAttnArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;                              // may be null
    int64_t q_b, q_h, o_b, o_h, page_s, head_s, slot_s, lse_b;
    PageTable table;
    const int* lens;
    const float* slopes;                     // may be null
    float *ws_o, *ws_ml;                     // parts: [2 grid][16][dim], [2 grid][16][2]
    int* status;
    int seqs, kv_heads, group, head_groups, window, grid;
    float scale, softcap;
};

template <int D> constexpr int ring_depth() { return D == 256 ? 3 : (D == 192 ? 4 : (D == 128 ? 6 : 8)); }
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

// ---- where a CTA's range lies ------------------------------------------------------------------------------------------
// Chunks of one item of sequence b.
__device__ __forceinline__ int seq_chunks(const PagedAttnArgs& a, int b) {
    int lo, hi;
    key_span(a.lens[b], static_cast<int64_t>(a.table.width) * a.table.page, a.window, lo, hi);
    return chunks_of(lo, hi);
}

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
    int seq;            // sequence, or seqs when there is none
    int64_t first;      // chunks in front of the sequence
};

__device__ __forceinline__ int64_t total_chunks(const PagedAttnArgs& a, int items, int64_t* red) {
    int64_t mine = 0, total;
    for (int b = threadIdx.x; b < a.seqs; b += blockDim.x) mine += static_cast<int64_t>(seq_chunks(a, b)) * items;
    scan_add(mine, red, total);
    return total;
}

// The sequence that holds chunk x (x < total).  place: shared.
__device__ __forceinline__ Place find_seq(const PagedAttnArgs& a, int items, int64_t x, int64_t* red, Place* place) {
    int64_t before = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        const int64_t n = b < a.seqs ? static_cast<int64_t>(seq_chunks(a, b)) * items : 0;
        int64_t total;
        const int64_t at = before + scan_add(n, red, total);
        if (x >= at && x < at + n) *place = {b, at};
        before += total;
        if (x < before) break;
    }
    __syncthreads();
    return *place;
}

template <typename T, int D, int NTR, bool MODS>
__global__ void __launch_bounds__(kPaThreads, 2) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int KS = D / 16, R = ring_depth<D>(), PITCH = D * 2 + 16, HALF = half_bytes<D>(), CPR = D / 8;
    extern __shared__ __align__(128) unsigned char pa_smem[];
    uint4* const qf = reinterpret_cast<uint4*>(pa_smem);                           // query fragments, 512 bytes a k step
    unsigned char* const ring = pa_smem + KS * 512;
    __shared__ int64_t red[32];
    __shared__ Place place;
    __shared__ float part_m[kPaWarps][kPaRows], part_l[kPaWarps][kPaRows];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int items = a.kv_heads * a.head_groups;
    const int64_t room = static_cast<int64_t>(a.table.width) * a.table.page;

    // sequences without keys: zeros, and an lse of -infinity
    for (int b = blockIdx.x; b < a.seqs; b += gridDim.x) {
        if (a.lens[b] > room && threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
        if (seq_chunks(a, b)) continue;
        const int heads = a.kv_heads * a.group;
        for (int i = threadIdx.x; i < heads * D; i += kPaThreads) static_cast<T*>(a.out)[b * a.o_b + i / D * a.o_h + i % D] = static_cast<T>(0.f);
        if (a.lse)
            for (int i = threadIdx.x; i < heads; i += kPaThreads) a.lse[b * a.lse_b + i] = -INFINITY;
    }

    const int64_t total = total_chunks(a, items, red);
    const int n = active_ctas(total, gridDim.x);
    if (total == 0 || static_cast<int>(blockIdx.x) >= n) return;
    int64_t x = range_begin(total, blockIdx.x, n);
    const int64_t x_end = range_begin(total, blockIdx.x + 1, n);
    const Place start = find_seq(a, items, x, red, &place);
    int b = start.seq;
    int64_t first = start.first;
    const int64_t range0 = x;

    const uint32_t my_ring = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + warp * R * HALF;
    // ldmatrix rows of this lane.  K: keys on the rows; V: keys on the rows, read transposed
    const uint32_t k_lane = ((lane & 7) + ((lane >> 4) << 3)) * PITCH + ((lane >> 3) & 1) * 16;
    const uint32_t v_lane = ((lane & 7) + ((lane >> 4) << 3)) * PITCH + ((lane >> 3) & 1) * 16;

    while (x < x_end) {
        int lo, hi;
        key_span(a.lens[b], room, a.window, lo, hi);
        const int per = chunks_of(lo, hi);
        if (x >= first + static_cast<int64_t>(per) * items) {        // also sequences without keys
            first += static_cast<int64_t>(per) * items;
            ++b;
            continue;
        }
        const int item = static_cast<int>((x - first) / per);
        const int64_t item0 = first + static_cast<int64_t>(item) * per;
        const int c0 = static_cast<int>(x - item0);
        const int c1 = item0 + per < x_end ? per : static_cast<int>(x_end - item0);
        const int kvh = item / a.head_groups, h0 = kvh * a.group + item % a.head_groups * kPaRows;
        const int rows = min(kPaRows, (kvh + 1) * a.group - h0);
        const int key0 = (lo / kChunk + c0) * kChunk + warp * kTile;  // first key of this warp's tile of chunk c0
        const int tiles = c1 - c0;
        const T* const kbase = static_cast<const T*>(a.k) + kvh * a.head_s;
        const T* const vbase = static_cast<const T*>(a.v) + kvh * a.head_s;

        // ---- page lookups one tile ahead of the copies: lane l (mod 16) finds the row of key l of the tile, -1 outside
        auto find = [&](int tile) -> int64_t {
            const int p = key0 + tile * kChunk + (lane & 15);
            if (tile >= tiles || p < lo || p >= hi) return -1;
            const int j = p / a.table.page, page = page_at(a.table, b, j);
            if (page < 0) {
                if (a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
                return -1;
            }
            return static_cast<int64_t>(page) * a.page_s + static_cast<int64_t>(p - j * a.table.page) * a.slot_s;
        };
        auto issue = [&](int half, int64_t at) {
            if (half < 2 * tiles) {
                const T* base = (half & 1) ? vbase : kbase;
                const uint32_t dst = my_ring + half % R * HALF;
#pragma unroll
                for (int i = 0; i < kTile * CPR / 32; ++i) {
                    const int idx = i * 32 + lane, r = idx / CPR, c = idx - r * CPR;
                    const int64_t off = __shfl_sync(0xffffffffu, at, r);
                    cp16(dst + r * PITCH + c * 16, base + (off < 0 ? 0 : off + c * 8), off >= 0);
                }
            }
            cp_commit();
        };
        // halves 0 .. R-2 are in flight before the first is used; `at`: rows of the tile that is being copied
        int64_t at = find(0), next = find(1);
        auto feed = [&](int half) {
            if (half > 0 && !(half & 1)) {
                at = next;
                next = find(half / 2 + 1);
            }
            issue(half, at);
        };
#pragma unroll
        for (int i = 0; i < R - 1; ++i) feed(i);

        // ---- query fragments
        {
            const T* q = static_cast<const T*>(a.q) + b * a.q_b;
            for (int i = threadIdx.x; i < KS * 32; i += kPaThreads) {
                const int ks = i >> 5, l = i & 31, gr = l >> 2, d = ks * 16 + (l & 3) * 2;
                uint32_t f[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int r = gr + (u & 1) * 8, dd = d + (u >> 1) * 8;
                    f[u] = 0;
                    if (r < rows) {
                        const unsigned short* s = reinterpret_cast<const unsigned short*>(q + (h0 + r) * a.q_h + dd);
                        f[u] = s[0] | static_cast<uint32_t>(s[1]) << 16;
                    }
                }
                qf[i] = make_uint4(f[0], f[1], f[2], f[3]);
            }
        }
        __syncthreads();

        float o[KS][NTR][4];
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int r = 0; r < NTR; ++r) o[j][r][0] = o[j][r][1] = o[j][r][2] = o[j][r][3] = 0.f;
        float mx[NTR], sum[NTR], slope[NTR];
#pragma unroll
        for (int r = 0; r < NTR; ++r) {
            mx[r] = -INFINITY;
            sum[r] = 0.f;
            slope[r] = MODS && a.slopes && g + 8 * r < rows ? a.slopes[h0 + g + 8 * r] * 1.4426950408889634f : 0.f;
        }
        const float scale2 = a.scale * 1.4426950408889634f;

        int64_t here = find(0);                                        // rows of the tile in use: which of its keys are there
        for (int i = 0; i < tiles; ++i) {
            const unsigned int have = __ballot_sync(0xffffffffu, here >= 0);
            here = find(i + 1);
            // ---- scores
            cp_wait<R - 2>();
            __syncwarp();
            feed(2 * i + R - 1);
            float s[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
            const uint32_t kt = my_ring + (2 * i) % R * HALF + k_lane;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t kf[4];
                ldsm4(kf, kt + ks * 32);
                const uint4 q4 = qf[ks * 32 + lane];
                const uint32_t qa[4] = {q4.x, q4.y, q4.z, q4.w};
                mma16816(s[0], qa, kf[0], kf[1], T());
                mma16816(s[1], qa, kf[2], kf[3], T());
            }
            // ---- mask and running softmax: row g + 8 r has its 16 scores in the four lanes of a g
            uint32_t ph[NTR][2], pl[NTR][2];
            float corr[NTR];
            const int tile0 = key0 + i * kChunk;
#pragma unroll
            for (int r = 0; r < NTR; ++r) {
                float v[4] = {s[0][2 * r], s[0][2 * r + 1], s[1][2 * r], s[1][2 * r + 1]};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int key = (u >> 1) * 8 + 2 * t + (u & 1);
                    if (MODS) {
                        float y = v[u] * a.scale;
                        if (a.softcap > 0.f) y = a.softcap * tanhf(y / a.softcap);
                        v[u] = y * 1.4426950408889634f - slope[r] * static_cast<float>(hi - 1 - tile0 - key);
                    } else {
                        v[u] *= scale2;
                    }
                    if (!(have >> key & 1)) v[u] = -INFINITY;
                }
                float m = max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3]));
                m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
                m = max_nan(m, mx[r]);
                const float shift = m == -INFINITY ? 0.f : m;
                corr[r] = mx[r] == m ? 1.f : exp2f(mx[r] - shift);
                mx[r] = m;
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = exp2f(v[u] - shift);
                sum[r] = fmaf(sum[r], corr[r], (v[0] + v[1]) + (v[2] + v[3]));
                split2(v[0], v[1], ph[r][0], pl[r][0], T());
                split2(v[2], v[3], ph[r][1], pl[r][1], T());
            }
            // the accumulators of this lane are of rows 2t and 2t + 1 (mod 8): their factors are with lanes 8t and 8t + 4
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
            // ---- values
            cp_wait<R - 2>();
            __syncwarp();
            feed(2 * i + R);
            const uint32_t vt = my_ring + (2 * i + 1) % R * HALF + v_lane;
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
        }
        cp_wait<0>();

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
        // a part that began in front of this range is the CTA's first, else its last
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (item0 < range0 ? 0 : 1);
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
                if (a.lse && d == 0) a.lse[b * a.lse_b + h0 + row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
            } else {
                *reinterpret_cast<float4*>(a.ws_o + (slot * kPaRows + row) * D + d) = y;
                if (d == 0) {
                    a.ws_ml[(slot * kPaRows + row) * 2] = m;
                    a.ws_ml[(slot * kPaRows + row) * 2 + 1] = l;
                }
            }
        }
        __syncthreads();
        x = item0 + c1;
    }
}

// One CTA per (sequence, query head): joins the parts of an item that was cut.  Threads: D / 4 lanes of four dims, in 1024 / D * 4 groups of parts.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int LANES = D / 4, GROUPS = 256 / LANES;
    __shared__ int64_t red[32];
    __shared__ float4 acc_s[GROUPS][LANES];
    __shared__ float ml_s[GROUPS][2];
    pdl_launch_dependents();
    pdl_wait();
    const int heads = a.kv_heads * a.group, b = blockIdx.x / heads, h = blockIdx.x - b * heads;
    const int items = a.kv_heads * a.head_groups;
    const int per = seq_chunks(a, b);
    if (per == 0) return;
    // chunks in front of sequence b, and of all
    int64_t mine = 0, before = 0, total;
    for (int i = threadIdx.x; i < a.seqs; i += blockDim.x) {
        const int64_t c = static_cast<int64_t>(seq_chunks(a, i)) * items;
        mine += c;
        if (i < b) before += c;
    }
    scan_add(mine, red, total);
    int64_t first;
    scan_add(before, red, first);
    const int n = active_ctas(total, a.grid);
    const int kvh = h / a.group, in_group = h - kvh * a.group, item = kvh * a.head_groups + in_group / kPaRows, row = in_group % kPaRows;
    const int64_t item0 = first + static_cast<int64_t>(item) * per;
    const int cta0 = owner_of(item0, total, n), cta1 = owner_of(item0 + per - 1, total, n);
    if (cta0 == cta1) return;                                           // one CTA wrote it
    const int d = threadIdx.x % LANES, grp = threadIdx.x / LANES;
    float m = -INFINITY, l = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp < GROUPS) {
        for (int c = cta0 + grp; c <= cta1; c += GROUPS) {
            const int64_t slot = (2 * static_cast<int64_t>(c) + (c == cta0)) * kPaRows + row;
            const float pm = a.ws_ml[slot * 2], pl = a.ws_ml[slot * 2 + 1];
            const float4 p = *reinterpret_cast<const float4*>(a.ws_o + slot * D + d * 4);
            const float mn = max_nan(m, pm);
            if (mn == -INFINITY) continue;
            const float f0 = exp2f(m - mn), f1 = exp2f(pm - mn);
            l = l * f0 + pl * f1;
            y.x = y.x * f0 + p.x * f1; y.y = y.y * f0 + p.y * f1; y.z = y.z * f0 + p.z * f1; y.w = y.w * f0 + p.w * f1;
            m = mn;
        }
        acc_s[grp][d] = y;
        if (d == 0) {
            ml_s[grp][0] = m;
            ml_s[grp][1] = l;
        }
    }
    __syncthreads();
    if (grp != 0) return;
    float top = -INFINITY;
    for (int i = 0; i < GROUPS; ++i) top = max_nan(top, ml_s[i][0]);
    l = 0.f;
    y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (top != -INFINITY) {
        for (int i = 0; i < GROUPS; ++i) {
            const float f = exp2f(ml_s[i][0] - top);
            const float4 p = acc_s[i][d];
            l += ml_s[i][1] * f;
            y.x += p.x * f; y.y += p.y * f; y.z += p.z * f; y.w += p.w * f;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = static_cast<T*>(a.out) + b * a.o_b + h * a.o_h + d * 4;
    out[0] = static_cast<T>(y.x * inv); out[1] = static_cast<T>(y.y * inv); out[2] = static_cast<T>(y.z * inv); out[3] = static_cast<T>(y.w * inv);
    if (a.lse && d == 0) a.lse[b * a.lse_b + h] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
}

template <typename T, int D> static int paged_launch(const PagedAttnArgs& a, bool join, cudaStream_t st) {
    const bool mods = a.softcap > 0.f || a.slopes != nullptr;
    const dim3 grid(a.grid), block(kPaThreads);
    const size_t smem = paged_smem<D>();
    int e;
    if (a.group <= 8) e = mods ? launch(paged_attn_kernel<T, D, 1, true>, grid, block, smem, st, a) : launch(paged_attn_kernel<T, D, 1, false>, grid, block, smem, st, a);
    else e = mods ? launch(paged_attn_kernel<T, D, 2, true>, grid, block, smem, st, a) : launch(paged_attn_kernel<T, D, 2, false>, grid, block, smem, st, a);
    if (e || !join) return e;
    return launch(paged_join_kernel<T, D>, dim3(a.seqs * a.kv_heads * a.group), dim3(256), 0, st, a);
}

template <typename T> static int paged_dispatch(const PagedAttnArgs& a, int dim, bool join, cudaStream_t st) {
    switch (dim) {
        case 64: return paged_launch<T, 64>(a, join, st);
        case 128: return paged_launch<T, 128>(a, join, st);
        case 192: return paged_launch<T, 192>(a, join, st);
        case 256: return paged_launch<T, 256>(a, join, st);
        default: return static_cast<int>(cudaErrorInvalidValue);
    }
}

}  // namespace nexrt

using namespace nexrt;

// CTAs of a call (its parts take 2 * that many * 16 * (dim + 2) floats of scratch).
extern "C" int nexrt_paged_ctas(int seqs, int q_heads, int kv_heads, int width, int page, int window) {
    if (seqs < 1 || kv_heads < 1 || q_heads < kv_heads) return 1;
    const int64_t room = static_cast<int64_t>(width) * page;
    const int64_t keys = window > 0 && window < room ? window + kChunk : room;
    const int64_t most = (keys / kChunk + 1) * seqs * kv_heads * ((q_heads / kv_heads + kPaRows - 1) / kPaRows);
    const int64_t resident = 2ll * sm_count();
    return static_cast<int>(most < resident ? most : resident);
}

// type: 0 bf16, 1 fp16.  strides: q (sequence, head), out, pools (page, head, slot), table row, lse row - in elements.
extern "C" int nexrt_paged_attn(const void* q, const void* k_pages, const void* v_pages, const void* table, const void* lens, const void* slopes, void* out, void* lse,
                                void* scratch, void* status, const int64_t* strides, int seqs, int q_heads, int kv_heads, int dim, int width, int page, int pages,
                                int window, int type, float scale, float softcap, int ctas, void* stream) {
    if (seqs < 0 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || width < 0 || page < 1 || pages < 0 || window < 0 || ctas < 1 || !(softcap >= 0.f))
        return cudaErrorInvalidValue;
    if (seqs == 0) return 0;
    PagedAttnArgs a = {};
    a.q = q; a.k = k_pages; a.v = v_pages; a.out = out; a.lse = static_cast<float*>(lse);
    a.q_b = strides[0]; a.q_h = strides[1]; a.o_b = strides[2]; a.o_h = strides[3];
    a.page_s = strides[4]; a.head_s = strides[5]; a.slot_s = strides[6]; a.lse_b = strides[8];
    if (((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) || a.page_s % 8 || a.head_s % 8 || a.slot_s % 8) return cudaErrorInvalidValue;
    a.table = {static_cast<const int*>(table), strides[7], seqs, width, page, pages};
    a.lens = static_cast<const int*>(lens); a.slopes = static_cast<const float*>(slopes);
    a.ws_o = static_cast<float*>(scratch); a.ws_ml = a.ws_o + static_cast<int64_t>(2) * ctas * kPaRows * dim;
    a.status = static_cast<int*>(status);
    a.seqs = seqs; a.kv_heads = kv_heads; a.group = q_heads / kv_heads; a.head_groups = (a.group + kPaRows - 1) / kPaRows;
    a.window = window; a.grid = ctas; a.scale = scale; a.softcap = softcap;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // with room for one chunk an item is never cut
    const bool join = static_cast<int64_t>(width) * page > kChunk;
    return type == 0 ? paged_dispatch<__nv_bfloat16>(a, dim, join, st) : (type == 1 ? paged_dispatch<__half>(a, dim, join, st) : static_cast<int>(cudaErrorInvalidValue));
}

// Host forms of the index arithmetic above, for tests without a GPU.
extern "C" int64_t nexrt_paged_slot(const int* table, int64_t stride, int rows, int width, int page, int pages, int row, int pos) {
    return page_slot({table, stride, rows, width, page, pages}, row, pos);
}
// out [parts][5]: CTA, sequence, item, first chunk, chunks - the walk of every CTA; returns the number of parts (at most `most` are written).
extern "C" int nexrt_paged_split(const int* lens, int seqs, int items, int64_t room, int window, int grid, int64_t* out, int most) {
    int64_t total = 0;
    auto chunks = [&](int b) {
        int lo, hi;
        key_span(lens[b], room, window, lo, hi);
        return static_cast<int64_t>(chunks_of(lo, hi));
    };
    for (int b = 0; b < seqs; ++b) total += chunks(b) * items;
    const int n = active_ctas(total, grid);
    int parts = 0;
    for (int c = 0; total > 0 && c < n; ++c) {
        int64_t x = range_begin(total, c, n), first = 0;
        const int64_t end = range_begin(total, c + 1, n);
        int b = 0;
        while (x < end) {
            const int64_t per = chunks(b);
            if (x >= first + per * items) {
                first += per * items;
                ++b;
                continue;
            }
            const int64_t item = (x - first) / per, item0 = first + item * per, stop = item0 + per < end ? item0 + per : end;
            if (parts < most) {
                int64_t* o = out + static_cast<int64_t>(parts) * 5;
                o[0] = c; o[1] = b; o[2] = item; o[3] = x - item0; o[4] = stop - x;
            }
            ++parts;
            x = stop;
        }
    }
    return parts;
}
