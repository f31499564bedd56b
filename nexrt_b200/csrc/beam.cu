// One step of a beam search: for every request the k best of beams x vocabulary, and the reordering of what belongs to a beam.
//
//   total(beam, token) = score(beam) + logit(beam, token) - log sum exp of the beam's logits
//
// in 64 bits, so that beams whose totals are near each other keep their order; equal totals go to the lower beam, then to the
// larger logit, then to the lower token.  A finished beam has one candidate, its end token at its own score.
//
// Within a beam the order of the totals is that of the logits, so one pass over a slice of a row gives everything that is
// needed of it: its maximum, its sum of exp and its k largest logits (values stay in registers, 16 a thread).  The k largest:
// the k-th largest of 64 group maxima bounds them from below, the few values at or above it are ranked by counting.  A second
// kernel, one CTA a request, joins the slices.  Bound by the logits' bytes; for one request by the two launches.
#include "api.h"
#include "common.cuh"

namespace nexrt {

using u64 = unsigned long long;

constexpr int kBeamMaxK = 64;
constexpr int kSliceThreads = 512;
constexpr int kPerThread = 16;
constexpr int kSliceValues = kSliceThreads * kPerThread;
constexpr int kBeamGroups = 64;             // of 8 lanes
constexpr int kBeamKeep = 1024;             // values that are ranked by counting; more (ties) take the search below
constexpr int kJoinThreads = 1024;
constexpr int kBeamMaxWidth = 256;          // beams of a request
constexpr int kBeamMaxVocab = 1 << 24;      // (beam, logit, token) in one 64-bit word

__device__ __forceinline__ unsigned int ord32(float f) {
    const unsigned int b = __float_as_uint(f + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unord32(unsigned int o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }
__device__ __forceinline__ u64 ord64(double d) {
    const u64 b = static_cast<u64>(__double_as_longlong(d + 0.0));
    return (b >> 63) ? ~b : (b | (1ull << 63));
}
__device__ __forceinline__ double unord64(u64 o) { return __longlong_as_double(static_cast<long long>((o >> 63) ? (o & ~(1ull << 63)) : ~o)); }

struct BeamArgs {
    const void* logits;
    const float* scores;
    const unsigned char* finished;      // may be null
    int64_t l_b, l_w, s_b, s_w, f_b, f_w;
    int batch, beams, vocab, k, eos, slices;
    u64* keys;                          // [batch * beams][slices][k]: logit in order, ~token; 0: none
    double* sums;                       // [batch * beams][slices] sum of exp(logit - maximum)
    float* tops;                        // [batch * beams][slices] maximum
    float* scores_out;
    int *rows_out, *tokens_out, *status;
};

// A beam with no candidates of its own vocabulary: finished, or with a score that nothing can follow.
__device__ __forceinline__ bool beam_is_closed(const BeamArgs& a, int b, int w) {
    if (a.finished && a.finished[b * a.f_b + w * a.f_w]) return true;
    const float s = a.scores[b * a.s_b + w * a.s_w];
    return !(s > -INFINITY) || s == INFINITY;
}

// sum of an int over the CTA, for all threads; red: 32 ints
__device__ __forceinline__ int cta_sum(int v, int* red) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int n = blockDim.x >> 5, lane = threadIdx.x & 31;
    return __reduce_add_sync(0xffffffffu, lane < n ? red[lane] : 0);
}

template <typename T>
__global__ void __launch_bounds__(kSliceThreads) beam_slice_kernel(const BeamArgs a) {
    constexpr int VEC = 16 / sizeof(T), NV = kPerThread / VEC;
    __shared__ float group_top[kBeamGroups];
    __shared__ double warp_sum_s[kSliceThreads / 32];
    __shared__ u64 keep[kBeamKeep];
    __shared__ float bound_s, top_s;
    __shared__ int count_s, red[32];
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, slice = blockIdx.x, b = row / a.beams, w = row - b * a.beams;
    if (beam_is_closed(a, b, w)) return;
    const T* base = static_cast<const T*>(a.logits) + b * a.l_b + w * a.l_w;
    // the row in 16-byte pieces: piece c holds values [c VEC - off, (c + 1) VEC - off)
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(base) / sizeof(T) % VEC);
    const int pieces = (a.vocab + off + VEC - 1) / VEC;
    const int lo = static_cast<int>(static_cast<int64_t>(pieces) * slice / a.slices), hi = static_cast<int>(static_cast<int64_t>(pieces) * (slice + 1) / a.slices);
    float x[kPerThread];
    unsigned int have = 0;              // bit per value: inside the row
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = lo + j * kSliceThreads + threadIdx.x, at = c * VEC - off;
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[j * VEC + i] = -INFINITY;
        if (c >= hi) continue;
        if (at >= 0 && at + VEC <= a.vocab) {
            const uint4 v = ld_stream16(base + at);
            const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[j * VEC + i] = static_cast<float>(t[i]);
            have |= ((1u << VEC) - 1u) << (j * VEC);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (at + i >= 0 && at + i < a.vocab) {
                    x[j * VEC + i] = static_cast<float>(base[at + i]);
                    have |= 1u << (j * VEC + i);
                }
        }
    }
    auto token_of = [&](int i) { return (lo + i / VEC * kSliceThreads + static_cast<int>(threadIdx.x)) * VEC - off + i % VEC; };
    auto key_of = [&](int i) -> u64 {
        if (!(have >> i & 1) || x[i] != x[i]) return 0;
        return (static_cast<u64>(ord32(x[i])) << 32) | static_cast<unsigned int>(~token_of(i));
    };

    // ---- maxima of 64 groups, the k-th largest of them, the slice's maximum
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float top = x[0];
#pragma unroll
    for (int i = 1; i < kPerThread; ++i) top = fmaxf(top, x[i]);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((lane & 7) == 0) group_top[threadIdx.x >> 3] = top;
    if (threadIdx.x == 0) count_s = 0;
    __syncthreads();
    if (threadIdx.x < kBeamGroups) {
        const float mine = group_top[threadIdx.x];
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < kBeamGroups; ++i) {
            const float g = group_top[i];
            rank += g > mine || (g == mine && i < static_cast<int>(threadIdx.x));
        }
        if (rank == 0) top_s = mine;
        if (rank == a.k - 1) bound_s = mine;
    }
    __syncthreads();
    const float bound = bound_s, m = top_s, shift = m == -INFINITY ? 0.f : m;

    // ---- sum of exp, in 64 bits from 16 values on; the values that can be among the k largest
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        if (have >> i & 1) {
            part += exp2f((x[i] - shift) * 1.4426950408889634f);
            if (x[i] >= bound) {
                const int at = atomicAdd(&count_s, 1);
                if (at < kBeamKeep) keep[at] = key_of(i);
            }
        }
    }
    double sum = part;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum_s[warp] = sum;
    __syncthreads();
    const int64_t at = static_cast<int64_t>(row) * a.slices + slice;
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < kSliceThreads / 32; ++i) t += warp_sum_s[i];
        a.sums[at] = t;
        a.tops[at] = m;
    }
    u64* out = a.keys + at * a.k;
    const int count = count_s;
    if (count <= kBeamKeep) {
        for (int i = threadIdx.x; i < count; i += kSliceThreads) {
            const u64 mine = keep[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += keep[j] > mine;
            if (rank < a.k) out[rank] = mine;
        }
        for (int i = count + threadIdx.x; i < a.k; i += kSliceThreads) out[i] = 0;
        return;
    }
    // many equal values: the k-th largest key bit by bit (keys differ, so exactly k are at or above it)
    u64 edge = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const u64 next = edge | (1ull << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) n += key_of(i) >= next;
        if (cta_sum(n, red) >= a.k) edge = next;
    }
    __syncthreads();
    if (threadIdx.x == 0) count_s = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const u64 key = key_of(i);
        if (key != 0 && key >= edge) out[atomicAdd(&count_s, 1)] = key;
    }
    __syncthreads();
    for (int i = count_s + threadIdx.x; i < a.k; i += kSliceThreads) out[i] = 0;
}

__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(const BeamArgs a) {
    __shared__ double lse[kBeamMaxWidth];           // of a live beam
    __shared__ int kind[kBeamMaxWidth];             // 0 live, 1 finished, 2 closed without a candidate above -infinity
    __shared__ u64 group_top[kJoinThreads / 8], keep[kBeamKeep], keep_tie[kBeamKeep];
    __shared__ u64 bound_s;
    __shared__ int count_s, red[32];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.beams, S = a.slices, k = a.k;
    for (int w = warp; w < W; w += kJoinThreads / 32) {
        int what = 0;
        double value = 0.0;
        if (a.finished && a.finished[b * a.f_b + w * a.f_w]) {
            what = 1;
            if (!(a.scores[b * a.s_b + w * a.s_w] < INFINITY)) what = 2;
        } else if (beam_is_closed(a, b, w)) {
            what = 2;
        } else {
            const int64_t at = (static_cast<int64_t>(b) * W + w) * S;
            float m = -INFINITY;
            for (int s = lane; s < S; s += 32) m = fmaxf(m, a.tops[at + s]);
            m = warp_max(m);
            double sum = 0.0;
            for (int s = lane; s < S; s += 32) {
                const float ms = a.tops[at + s];
                const double part = a.sums[at + s];
                sum += ms == m ? part : part * exp(static_cast<double>(ms) - static_cast<double>(m));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (m == -INFINITY && sum == 0.0) {
                value = 0.0;                         // nothing is allowed: every candidate is at -infinity
            } else if (sum > 0.0 && sum < INFINITY && m < INFINITY) {
                value = static_cast<double>(m) + log(sum);
            } else {
                what = 2;                            // a logit is NaN or +infinity
                if (lane == 0 && a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusNonFinite));
            }
        }
        if (what == 2 && lane == 0 && a.status) {
            const float s = a.scores[b * a.s_b + w * a.s_w];
            if (s != s || s == INFINITY) atomicCAS(a.status, 0, static_cast<int>(kStatusNonFinite));
        }
        if (lane == 0) {
            lse[w] = value;
            kind[w] = what;
        }
    }
    if (threadIdx.x == 0) count_s = 0;
    __syncthreads();

    // candidate n of the request: its total in order (0: none), and the word that orders equal totals
    const int per = S * k, total_n = W * per;
    auto candidate = [&](int n, u64& tie) -> u64 {
        const int w = n / per, i = n - w * per;
        const u64 beam = static_cast<u64>(kBeamMaxWidth - 1 - w) << 56;
        const double score = a.scores[b * a.s_b + w * a.s_w];
        if (kind[w] == 0) {
            const u64 key = a.keys[(static_cast<int64_t>(b) * W + w) * per + i];
            if (key == 0) return 0;
            const unsigned int logit = static_cast<unsigned int>(key >> 32), token = ~static_cast<unsigned int>(key);
            tie = beam | (static_cast<u64>(logit) << 24) | (kBeamMaxVocab - 1 - token);
            return ord64(score + (static_cast<double>(unord32(logit)) - lse[w]));
        }
        // a closed beam: its end token, if it is finished, and the vocabulary at -infinity
        int token = i - (kind[w] == 1);
        if (kind[w] == 1 && token >= a.eos) ++token;
        if (kind[w] == 1 && i == 0) token = a.eos;
        else if (i >= k || token >= a.vocab) return 0;
        tie = beam | (kBeamMaxVocab - 1 - token);
        return ord64(kind[w] == 1 && i == 0 ? score : -INFINITY);
    };

    u64 top = 0, tie = 0;
    for (int n = threadIdx.x; n < total_n; n += kJoinThreads) {
        const u64 key = candidate(n, tie);
        top = key > top ? key : top;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, top, o);
        top = other > top ? other : top;
    }
    if ((lane & 7) == 0) group_top[threadIdx.x >> 3] = top;
    __syncthreads();
    if (threadIdx.x < kJoinThreads / 8) {
        const u64 mine = group_top[threadIdx.x];
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < kJoinThreads / 8; ++i) {
            const u64 g = group_top[i];
            rank += g > mine || (g == mine && i < static_cast<int>(threadIdx.x));
        }
        if (rank == k - 1) bound_s = mine;
    }
    __syncthreads();
    const u64 bound = bound_s;
    for (int n = threadIdx.x; n < total_n; n += kJoinThreads) {
        const u64 key = candidate(n, tie);
        if (key != 0 && key >= bound) {
            const int at = atomicAdd(&count_s, 1);
            if (at < kBeamKeep) {
                keep[at] = key;
                keep_tie[at] = tie;
            }
        }
    }
    __syncthreads();
    int count = count_s;
    if (count > kBeamKeep) {
        // the k-th largest total bit by bit, then the last of its equals that is still among the k
        u64 edge = 0, edge_tie = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const u64 next = edge | (1ull << bit);
            int n = 0;
            for (int i = threadIdx.x; i < total_n; i += kJoinThreads) n += candidate(i, tie) >= next;
            if (cta_sum(n, red) >= k) edge = next;
        }
        int above = 0;
        for (int i = threadIdx.x; i < total_n; i += kJoinThreads) above += candidate(i, tie) > edge;
        above = cta_sum(above, red);
        for (int bit = 63; bit >= 0; --bit) {
            const u64 next = edge_tie | (1ull << bit);
            int n = 0;
            for (int i = threadIdx.x; i < total_n; i += kJoinThreads) n += candidate(i, tie) == edge && tie >= next;
            if (above + cta_sum(n, red) >= k) edge_tie = next;
        }
        __syncthreads();
        if (threadIdx.x == 0) count_s = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < total_n; i += kJoinThreads) {
            const u64 key = candidate(i, tie);
            if (key != 0 && (key > edge || (key == edge && tie >= edge_tie))) {
                const int at = atomicAdd(&count_s, 1);
                if (at < kBeamKeep) {
                    keep[at] = key;
                    keep_tie[at] = tie;
                }
            }
        }
        __syncthreads();
        count = count_s;
    }
    for (int i = threadIdx.x; i < count; i += kJoinThreads) {
        const u64 mine = keep[i], mine_tie = keep_tie[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += keep[j] > mine || (keep[j] == mine && keep_tie[j] > mine_tie);
        if (rank < k) {
            const int64_t o = static_cast<int64_t>(b) * k + rank;
            a.scores_out[o] = static_cast<float>(unord64(mine));
            a.rows_out[o] = b * W + kBeamMaxWidth - 1 - static_cast<int>(mine_tie >> 56);
            a.tokens_out[o] = kBeamMaxVocab - 1 - static_cast<int>(mine_tie & (kBeamMaxVocab - 1));
        }
    }
}

constexpr int kReorderTensors = 16;
constexpr int kReorderThreads = 256;
constexpr int kReorderPiece = kReorderThreads * 64;     // bytes that a CTA moves at a time

struct ReorderArgs {
    const char* in[kReorderTensors];
    char* out[kReorderTensors];
    int64_t in_stride[kReorderTensors], out_stride[kReorderTensors], bytes[kReorderTensors];
    int64_t first[kReorderTensors + 1];      // pieces in front of a tensor's
    int width[kReorderTensors];              // 16, 4 or 1 bytes a access
    const int* rows;
    int64_t r_0, r_1;
    int cols, n, n_in, tensors;
    int* status;
};

template <typename V> __device__ __forceinline__ void copy_piece(const char* src, char* dst, int64_t begin, int64_t bytes) {
    constexpr int kSteps = 4;
    const int64_t end = begin + kReorderPiece < bytes ? begin + kReorderPiece : bytes;
    for (int64_t o0 = begin + threadIdx.x * sizeof(V); o0 < end; o0 += kSteps * kReorderThreads * sizeof(V)) {
        V v[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int64_t o = o0 + i * kReorderThreads * static_cast<int64_t>(sizeof(V));
            if (o < end) v[i] = *reinterpret_cast<const V*>(src + o);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int64_t o = o0 + i * kReorderThreads * static_cast<int64_t>(sizeof(V));
            if (o < end) *reinterpret_cast<V*>(dst + o) = v[i];
        }
    }
}

// out[i] = in[rows[i]] for several tensors.  The rows of one piece run side by side, so a row that several take is read from
// memory once.
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const __grid_constant__ ReorderArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t units = a.first[a.tensors] * a.n;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int i = static_cast<int>(u % a.n);
        const int64_t p = u / a.n;
        int t = 0;
        while (p >= a.first[t + 1]) ++t;
        const int row = a.rows[i / a.cols * a.r_0 + i % a.cols * a.r_1];
        if (row < 0 || row >= a.n_in) {
            if (threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
            continue;
        }
        const char* src = a.in[t] + row * a.in_stride[t];
        char* dst = a.out[t] + i * a.out_stride[t];
        const int64_t begin = (p - a.first[t]) * kReorderPiece;
        if (a.width[t] == 16) copy_piece<uint4>(src, dst, begin, a.bytes[t]);
        else if (a.width[t] == 4) copy_piece<uint32_t>(src, dst, begin, a.bytes[t]);
        else copy_piece<uint8_t>(src, dst, begin, a.bytes[t]);
    }
}

static int beam_slices(int vocab) { return (vocab + 8 + kSliceValues - 1) / kSliceValues; }

}  // namespace nexrt

using namespace nexrt;

// Slices of a row: a call's scratch is batch * beams * slices * (k + 2) words of 8 bytes.
extern "C" int nexrt_beam_slices(int vocab) { return beam_slices(vocab); }

// type: 0 bf16, 1 fp16, 2 fp32; strides: logits (request, beam), scores, finished, in elements.
extern "C" int nexrt_beam_select(const void* logits, const void* scores, const void* finished, const int64_t* strides, void* scores_out, void* rows_out, void* tokens_out,
                                 void* scratch, void* status, int batch, int beams, int vocab, int k, int eos, int type, void* stream) {
    if (batch < 0 || beams < 1 || beams > kBeamMaxWidth || vocab < 1 || vocab > kBeamMaxVocab || k < 1 || k > kBeamMaxK || static_cast<int64_t>(beams) * vocab < k ||
        (finished != nullptr && (eos < 0 || eos >= vocab)) || static_cast<int64_t>(batch) * beams > 65535)
        return cudaErrorInvalidValue;
    if (batch == 0) return 0;
    BeamArgs a = {};
    a.logits = logits; a.scores = static_cast<const float*>(scores); a.finished = static_cast<const unsigned char*>(finished);
    a.l_b = strides[0]; a.l_w = strides[1]; a.s_b = strides[2]; a.s_w = strides[3]; a.f_b = strides[4]; a.f_w = strides[5];
    a.batch = batch; a.beams = beams; a.vocab = vocab; a.k = k; a.eos = eos; a.slices = beam_slices(vocab);
    const int64_t parts = static_cast<int64_t>(batch) * beams * a.slices;
    a.keys = static_cast<u64*>(scratch);
    a.sums = reinterpret_cast<double*>(a.keys + parts * k);
    a.tops = reinterpret_cast<float*>(a.sums + parts);
    a.scores_out = static_cast<float*>(scores_out); a.rows_out = static_cast<int*>(rows_out); a.tokens_out = static_cast<int*>(tokens_out);
    a.status = static_cast<int*>(status);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(a.slices, batch * beams);
    int e = cudaErrorInvalidValue;
    if (type == 0) e = launch(beam_slice_kernel<__nv_bfloat16>, grid, dim3(kSliceThreads), 0, st, a);
    else if (type == 1) e = launch(beam_slice_kernel<__half>, grid, dim3(kSliceThreads), 0, st, a);
    else if (type == 2) e = launch(beam_slice_kernel<float>, grid, dim3(kSliceThreads), 0, st, a);
    if (e) return e;
    return launch(beam_join_kernel, dim3(batch), dim3(kJoinThreads), 0, st, a);
}

// in, out, meta: arrays of `tensors` (at most 16) pointers and of 3 int64 each (row stride of in, of out, bytes of a row).
extern "C" int nexrt_reorder_rows(const void* const* in, void* const* out, const int64_t* meta, int tensors, const void* rows, int64_t r_0, int64_t r_1, int cols, int n,
                                  int n_in, void* status, void* stream) {
    if (tensors < 0 || tensors > kReorderTensors || n < 0 || cols < 1 || n_in < 0) return cudaErrorInvalidValue;
    ReorderArgs a = {};
    for (int t = 0; t < tensors; ++t) {
        a.in[t] = static_cast<const char*>(in[t]);
        a.out[t] = static_cast<char*>(out[t]);
        a.in_stride[t] = meta[3 * t]; a.out_stride[t] = meta[3 * t + 1]; a.bytes[t] = meta[3 * t + 2];
        if (a.bytes[t] < 0) return cudaErrorInvalidValue;
        const uint64_t all = reinterpret_cast<uintptr_t>(in[t]) | reinterpret_cast<uintptr_t>(out[t]) | static_cast<uint64_t>(a.in_stride[t]) |
                             static_cast<uint64_t>(a.out_stride[t]) | static_cast<uint64_t>(a.bytes[t]);
        a.width[t] = all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : 1);
        a.first[t + 1] = a.first[t] + (a.bytes[t] + kReorderPiece - 1) / kReorderPiece;
    }
    a.rows = static_cast<const int*>(rows); a.r_0 = r_0; a.r_1 = r_1; a.cols = cols; a.n = n; a.n_in = n_in; a.tensors = tensors;
    a.status = static_cast<int*>(status);
    const int64_t units = a.first[tensors] * n, most = 8ll * sm_count();
    if (units == 0) return 0;
    return launch(reorder_kernel, dim3(static_cast<unsigned>(units < most ? units : most)), dim3(kReorderThreads), 0, static_cast<cudaStream_t>(stream), a);
}
