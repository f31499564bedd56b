// One step of a beam search: for every request the k best of beams x vocabulary, and the reordering of what belongs to a beam.
//
//   total(beam, token) = score(beam) + logit(beam, token) - log sum exp of the beam's logits
//
// in 64 bits; equal totals go to the lower beam, then to the larger logit, then to the lower token.  A finished beam has one candidate, its
// end token at its own score.  What is not 64 bits are the exponentials and the sums of 16 or 32 of them: a row's logarithm is off by
// 1e-7 as a rule, at worst by a few 1e-6 (where values 16 below the maximum make up the sum: each is off by up to 2.5 units of 2^-24 of its
// distance), and beams whose totals are nearer than that may change places.  Beams that hold the same numbers tie to the
// last bit: which values meet in a partial sum goes by their tokens, never by the address of the row.
//
// Within a beam the order of the totals is that of the logits, so one pass over a slice of a row gives everything that is
// needed of it: its maximum, its sum of exp and its k largest logits.  A CTA walks its slice in steps of 16 KB, 64 bytes a thread in
// registers as they came, the next step's loads in flight.  The k largest: the k-th largest of 64 or 128 maxima of the first step bounds
// them from below; the few values of that step at or above it, and of the later ones above it (an equal one comes behind k with lower
// tokens), are collected and at the end ranked by counting.  Equal values in masses, as masked vocabularies have them, are taken in the
// order of their tokens, k of them at most; what still does not fit is selected digit by digit.  A second kernel, one CTA a request, joins
// the slices.  Bound by the logits' bytes, and for one request by the two launches.  Measured: 117 live rows of 248320 bf16 logits
// (58 MB) 29 us, about 16 instructions a value, 128 rows with all but ten values masked 28; four rows of fp32 11 us.
#include <type_traits>

#include "api.h"
#include "common.cuh"

namespace nexrt {

using u64 = unsigned long long;

constexpr int kBeamMaxK = 64;
constexpr int kSliceThreads = 256;
constexpr int kPieces = 4;                  // 16-byte pieces of a thread and step
constexpr int kStepBytes = kSliceThreads * kPieces * 16;
constexpr int kBeamGroups = 128;            // at most
constexpr int kBeamKeep = 1024;             // values that are ranked by counting; more (ties) take the search below
constexpr int kJoinThreads = 512;
constexpr int kJoinHold = 4;               // candidates of a thread that it keeps in registers
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
    const bool done = a.finished && a.finished[b * a.f_b + w * a.f_w];
    const float s = a.scores[b * a.s_b + w * a.s_w];
    return done || !(s > -INFINITY) || s == INFINITY;
}

// The threshold of the k largest of n keys, a digit of eight bits at a time; 0 is no key.  Taken are keys above `edge`, and of those equal to
// it `ties` (-1: all; equal keys are told apart by the caller).  hist: 258 ints.
template <typename Key> __device__ __forceinline__ u64 largest_edge(Key key_of, int n, int k, int* hist, int& ties) {
    u64 edge = 0;
    ties = -1;
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 258; i += blockDim.x) hist[i] = 0;
        __syncthreads();
        for (int i0 = 0; i0 < n; i0 += blockDim.x) {
            const int i = i0 + threadIdx.x;
            const u64 key = i < n ? key_of(i) : 0;
            const int digit = key != 0 && (shift == 56 || key >> (shift + 8) == edge >> (shift + 8)) ? static_cast<int>(key >> shift & 255) : -1;
            int same;
            __match_all_sync(0xffffffffu, digit, &same);           // (equal keys in masses: one addition a warp)
            if (digit >= 0 && (!same || (threadIdx.x & 31) == 0)) atomicAdd(hist + digit, same ? 32 : 1);
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            int above = 0;
#pragma unroll 8
            for (int i = threadIdx.x + 1; i < 256; ++i) above += hist[i];
            if (above < k && above + hist[threadIdx.x] >= k) {
                hist[256] = static_cast<int>(threadIdx.x) + 1;
                hist[257] = above;
            }
        }
        __syncthreads();
        if (hist[256] == 0) return 0;                              // fewer than k
        const int digit = hist[256] - 1;
        edge |= static_cast<u64>(digit) << shift;
        k -= hist[257];
        if (hist[digit] == k) return edge;
    }
    ties = k;
    return edge;
}

// 16 bytes of a row as they came; `top` takes maxNum over two or four such pieces' words without unpacking 16-bit types.
template <typename T> struct Piece {
    static constexpr int kValues = 16 / sizeof(T);
    uint32_t w[4];
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
    }
    static __device__ __forceinline__ uint4 nothing() {          // -infinity throughout
        constexpr uint32_t low = sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __nv_bfloat16>::value ? 0xff80ff80u : 0xfc00fc00u);
        return make_uint4(low, low, low, low);
    }
    // value(i) of an i that is not known when this is compiled
    __device__ __forceinline__ float value_at(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(i & 2 ? (i & 1 ? w[3] : w[2]) : (i & 1 ? w[1] : w[0]));
        } else {
            const uint32_t u = i & 4 ? (i & 2 ? w[3] : w[2]) : (i & 2 ? w[1] : w[0]);
            if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
            else return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? u >> 16 : u)));
        }
    }
    // Bit i: value i >= bound, a value of the same type (16-bit types are compared two at a time).
    __device__ __forceinline__ uint32_t at_least(float bound) const {
        uint32_t bits = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) bits |= static_cast<uint32_t>(value(i) >= bound) << i;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t m;
                if constexpr (std::is_same<T, __nv_bfloat16>::value) m = __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), __float2bfloat162_rn(bound));
                else m = __hge2_mask(*reinterpret_cast<const __half2*>(&w[i]), __float2half2_rn(bound));
                bits |= ((m & 1u) | (m >> 15 & 2u)) << (2 * i);
            }
        }
        return bits;
    }
    // The smallest value of the type above v (NaN above infinity: nothing is at least that).
    static __device__ __forceinline__ float above(float v) {
        auto up = [](unsigned int bits, unsigned int sign) { return bits & sign ? (bits == sign ? 1u : bits - 1u) : bits + 1u; };
        if constexpr (sizeof(T) == 4) return __uint_as_float(up(__float_as_uint(v), 0x80000000u));
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(up(__float_as_uint(v) >> 16, 0x8000u) << 16);
        else return __half2float(__ushort_as_half(static_cast<unsigned short>(up(__half_as_ushort(__float2half_rn(v)), 0x8000u))));
    }
    __device__ __forceinline__ float top() const {
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(value(0), value(1)), fmaxf(value(2), value(3)));
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
            const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
            return fmaxf(f.x, f.y);
        } else {
            const __half2* h = reinterpret_cast<const __half2*>(w);
            const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
            return fmaxf(f.x, f.y);
        }
    }
};

// The word at value `at` of a row where it may reach over an end of it, -infinity outside.
template <typename T> __device__ __forceinline__ uint32_t edge_word(const T* base, int at, int vocab) {
    if constexpr (sizeof(T) == 4) {
        return at >= 0 && at < vocab ? reinterpret_cast<const uint32_t*>(base)[at] : 0xff800000u;
    } else {
        const uint32_t low = std::is_same<T, __nv_bfloat16>::value ? 0xff80u : 0xfc00u;
        const unsigned short* p = reinterpret_cast<const unsigned short*>(base);
        return (at >= 0 && at < vocab ? p[at] : low) | (at + 1 >= 0 && at + 1 < vocab ? p[at + 1] : low) << 16;
    }
}
// Four of them.  Out of line: a row has two such pieces at most.
template <typename T> __device__ __noinline__ uint4 edge_piece(const T* base, int at, int vocab) {
    constexpr int PER = 4 / sizeof(T);
    return make_uint4(edge_word(base, at, vocab), edge_word(base, at + PER, vocab), edge_word(base, at + 2 * PER, vocab), edge_word(base, at + 3 * PER, vocab));
}
__device__ __forceinline__ uint32_t ld_word(const void* p) {     // (a line serves several such loads: it may stay in L1)
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// ALIGNED: every row starts on a 16-byte boundary and is read 16 bytes at a time.  Else by words, so that a thread has the same values wherever its
// row starts (128 rows of 248320 or 248321 values: bf16 31.3 and 35.3 us, fp32 39.4 and 41.7).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kSliceThreads, 4) beam_slice_kernel(const BeamArgs a) {
    constexpr int VEC = Piece<T>::kValues, NV = kPieces, kWarps = kSliceThreads / 32, PER = 4 / sizeof(T);
    constexpr int WORDS = ALIGNED || PER == 1 ? 4 : 5;                 // of a piece: one of 16-bit values that starts in the middle of a word touches five
    __shared__ float group_top[kBeamGroups], warp_top[kWarps];
    __shared__ double warp_part[kWarps];
    __shared__ u64 keep[kBeamKeep];
    __shared__ unsigned int bound_s;
    __shared__ float equal_s;
    __shared__ int count_s, tied_s, red[32];
    static_assert(sizeof(keep) >= 258 * sizeof(int), "the digits' counts lie where the candidates did");
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, slice = blockIdx.x, b = row / a.beams, w = row - b * a.beams;
    const bool closed = beam_is_closed(a, b, w);        // looked at when the first loads are on their way
    const T* base = static_cast<const T*>(a.logits) + b * a.l_b + w * a.l_w;
    // the row in pieces of 16 bytes: piece c holds values [c VEC, (c + 1) VEC)
    const int pieces = (a.vocab + VEC - 1) / VEC;
    const int odd = WORDS == 5 ? static_cast<int>(reinterpret_cast<uintptr_t>(base) >> 1 & 1) : 0;     // the row starts in the middle of a word
    // a slice is whole steps: only a row's last one is ragged
    const int steps = (pieces + kSliceThreads * NV - 1) / (kSliceThreads * NV);
    const unsigned int slices = a.slices;                              // (no more than there are steps, at most 4096: 32 bits will do)
    const int lo = static_cast<int>(static_cast<unsigned int>(steps * slice) / slices) * kSliceThreads * NV;
    const int hi = min(pieces, static_cast<int>(static_cast<unsigned int>(steps * (slice + 1)) / slices) * kSliceThreads * NV);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t at_slice = static_cast<int64_t>(row) * a.slices + slice;
    u64* out = a.keys + at_slice * a.k;
    if (threadIdx.x == 0) count_s = tied_s = 0;

    // the thread's maximum and its sum of exp below it, in 64 bits from 32 values on
    float top = -INFINITY, bound = 0.f;
    double sum = 0.0;
    bool over = false;                  // more candidates than there is room for
    uint32_t ahead[NV][WORDS];          // the next step's pieces are on their way while a step is worked on
    auto load = [&](uint32_t (&to)[WORDS], const T* from) {
        if constexpr (ALIGNED) {
            const uint4 v = ld_stream16(from);
            to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) to[i] = ld_word(from + i * PER);
        }
    };
    auto fetch = [&](int p0) {
        if (p0 >= odd && (p0 + kSliceThreads * NV) * VEC + (WORDS - 4) * PER - odd <= a.vocab) {
            const T* from = base + (static_cast<int64_t>(p0 + threadIdx.x) * VEC - odd);
#pragma unroll
            for (int j = 0; j < NV; ++j) load(ahead[j], from + j * kSliceThreads * VEC);
            return;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = (p0 + j * kSliceThreads + static_cast<int>(threadIdx.x)) * VEC - odd;
            if (at >= 0 && at + WORDS * PER <= a.vocab) {
                load(ahead[j], base + at);
            } else {
                const uint4 v = at + odd < a.vocab ? edge_piece(base, at, a.vocab) : Piece<T>::nothing();
                ahead[j][0] = v.x; ahead[j][1] = v.y; ahead[j][2] = v.z; ahead[j][3] = v.w;
                if constexpr (WORDS == 5) ahead[j][4] = edge_word(base, at + 4 * PER, a.vocab);
            }
        }
    };
    fetch(lo);
    if (closed) return;
    int step = 0;
    for (int p0 = lo; p0 < hi; p0 += kSliceThreads * NV, ++step) {
        Piece<T> x[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (WORDS == 5) x[j].w[i] = __funnelshift_r(ahead[j][i], ahead[j][i + 1], odd * 16);
                else x[j].w[i] = ahead[j][i];
            }
        if (p0 + kSliceThreads * NV < hi) fetch(p0 + kSliceThreads * NV);
        float piece_top[NV], new_top = top;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            piece_top[j] = x[j].top();
            new_top = fmaxf(new_top, piece_top[j]);
        }
        const float shift = new_top == -INFINITY ? 0.f : new_top;
        const float2 minus = make_float2(-shift, -shift), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
        float2 part = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const float2 e = mul2(add2(make_float2(x[j].value(i), x[j].value(i + 1)), minus), log2e);
                part = add2(part, make_float2(exp2_ftz(e.x), exp2_ftz(e.y)));
            }
        sum = fma(sum, static_cast<double>(exp2_ftz((top - shift) * 1.4426950408889634f)), static_cast<double>(part.x + part.y));
        top = new_top;
        if (p0 == lo) {
            // the k-th largest maximum of 64 groups of lanes (of 128 for many beams) bounds the k-th largest value of the slice from below
            const int wide = a.k > 16 ? 1 : 2, lanes = 1 << wide, groups = kSliceThreads >> wide, part = threadIdx.x & (lanes - 1);
            float group = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            if (lanes == 4) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, 2));
            if (part == 0) group_top[threadIdx.x >> wide] = group;
            if (threadIdx.x == 0) bound_s = 0xffffffffu;
            __syncthreads();
            int above = 0;
            float least = group;
#pragma unroll 16
            for (int i = part; i < groups; i += lanes) {
                above += group_top[i] > group;
                least = fminf(least, group_top[i]);
            }
            above += __shfl_xor_sync(0xffffffffu, above, 1);
            least = fminf(least, __shfl_xor_sync(0xffffffffu, least, 1));
            if (lanes == 4) {
                above += __shfl_xor_sync(0xffffffffu, above, 2);
                least = fminf(least, __shfl_xor_sync(0xffffffffu, least, 2));
            }
            if (part == 0 && above < a.k) {
                atomicMin(&bound_s, ord32(group));
                if (group == least) {                    // even the smallest reaches the bound: values equal to it in masses, a masked slice
                    tied_s = 1;
                    equal_s = group;
                }
            }
            __syncthreads();
            bound = unord32(bound_s);
            if (tied_s) bound = Piece<T>::above(bound);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (piece_top[j] >= bound) {
                const int first = (p0 + j * kSliceThreads + static_cast<int>(threadIdx.x)) * VEC;
#pragma unroll 1
                for (uint32_t there = x[j].at_least(bound); there; there &= there - 1) {
                    const int i = __ffs(there) - 1, token = first + i;
                    if (token >= a.vocab) continue;
                    const float v = x[j].value_at(i);
                    const int to = atomicAdd(&count_s, 1);
                    if (to < kBeamKeep) keep[to] = (static_cast<u64>(ord32(v)) << 32) | static_cast<unsigned int>(~token);
                }
            }
        // what equals the bound comes behind the k of the first step, whose tokens are lower
        if (p0 == lo && !tied_s) bound = Piece<T>::above(bound);
        if ((step & 3) == 3 && p0 + kSliceThreads * NV < hi) {
            // half full: only the k largest so far go on, and what follows has to reach the last of them
            __syncthreads();
            const int count = count_s;
            if (count > kBeamKeep) {
                over = true;
            } else if (count > kBeamKeep / 2) {
                u64 mine[kBeamKeep / kSliceThreads];
                int rank[kBeamKeep / kSliceThreads];
#pragma unroll
                for (int i = 0; i < kBeamKeep / kSliceThreads; ++i) {
                    const int n = i * kSliceThreads + threadIdx.x;
                    mine[i] = n < count ? keep[n] : 0;
                    rank[i] = n < count ? 0 : a.k;
                }
                for (int j = 0; j < count; ++j) {
                    const u64 other = keep[j];
#pragma unroll
                    for (int i = 0; i < kBeamKeep / kSliceThreads; ++i) rank[i] += other > mine[i];
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kBeamKeep / kSliceThreads; ++i) {
                    if (rank[i] < a.k) keep[rank[i]] = mine[i];
                    if (rank[i] == a.k - 1) bound_s = static_cast<unsigned int>(mine[i] >> 32);
                }
                if (threadIdx.x == 0) count_s = a.k;
                __syncthreads();
                bound = Piece<T>::above(unord32(bound_s));
            }
            __syncthreads();
        }
    }

    // ---- the CTA's maximum and sum
    float all = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    if (top != all && top > -INFINITY) sum *= exp2_ftz((top - all) * 1.4426950408889634f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
        warp_top[warp] = all;
        warp_part[warp] = sum;
    }
    __syncthreads();
    if (threadIdx.x == kSliceThreads - 1) {
        float m = warp_top[0];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) m = fmaxf(m, warp_top[i]);
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) t += warp_top[i] == m || warp_top[i] == -INFINITY ? warp_part[i] : warp_part[i] * exp2_ftz((warp_top[i] - m) * 1.4426950408889634f);
        a.sums[at_slice] = t;
        a.tops[at_slice] = m;
    }
    const int first = lo * VEC, last = min(hi * VEC, a.vocab);
    if (tied_s) {
        // of the first step's values equal to its bound the k lowest tokens
        const float equal = equal_s;
        const int end = min(last, (lo + kSliceThreads * NV) * VEC);
        for (int t0 = first, taken = 0; t0 < end && taken < a.k; t0 += kSliceThreads) {
            const int token = t0 + threadIdx.x;
            const bool here = token < end && static_cast<float>(base[token]) == equal;
            const unsigned int mask = __ballot_sync(0xffffffffu, here);
            if (lane == 0) red[warp] = __popc(mask);
            __syncthreads();
            int place = taken + __popc(mask & ((1u << lane) - 1u));
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                if (i < warp) place += red[i];
                taken += red[i];
            }
            if (here && place < a.k) {
                const int to = atomicAdd(&count_s, 1);
                if (to < kBeamKeep) keep[to] = (static_cast<u64>(ord32(equal)) << 32) | static_cast<unsigned int>(~token);
            }
            __syncthreads();
        }
    }
    const int count = count_s;
    if (!over && count <= kBeamKeep) {
        for (int i = threadIdx.x; i < count; i += kSliceThreads) {
            const u64 mine = keep[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += keep[j] > mine;
            if (rank < a.k) out[rank] = mine;
        }
        for (int i = count + threadIdx.x; i < a.k; i += kSliceThreads) out[i] = 0;
        return;
    }
    // more than there is room for (keys differ, so exactly k are at or above the edge); the slice is read again for each digit
    auto key_at = [&](int token) -> u64 {
        const float v = static_cast<float>(base[token]);
        return v != v ? 0 : (static_cast<u64>(ord32(v)) << 32) | static_cast<unsigned int>(~token);
    };
    int ties;
    const u64 edge = largest_edge([&](int i) { return key_at(first + i); }, last - first, a.k, reinterpret_cast<int*>(keep), ties);
    if (threadIdx.x == 0) count_s = 0;
    __syncthreads();
    for (int i = first + threadIdx.x; i < last; i += kSliceThreads) {
        const u64 key = key_at(i);
        if (key != 0 && key >= edge) out[atomicAdd(&count_s, 1)] = key;
    }
    __syncthreads();
    for (int i = count_s + threadIdx.x; i < a.k; i += kSliceThreads) out[i] = 0;
}

template <typename T> static int slice_launch(const BeamArgs& a, bool aligned, cudaStream_t st) {
    const dim3 grid(a.slices, a.batch * a.beams), block(kSliceThreads);
    return aligned ? launch(beam_slice_kernel<T, true>, grid, block, 0, st, a) : launch(beam_slice_kernel<T, false>, grid, block, 0, st, a);
}

__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(const BeamArgs a) {
    __shared__ double lse[kBeamMaxWidth];           // of a live beam
    __shared__ float score_s[kBeamMaxWidth];
    __shared__ int kind[kBeamMaxWidth];             // 0 live, 1 finished, 2 closed without a candidate above -infinity
    __shared__ u64 group_top[kJoinThreads / 4], group_tie[kJoinThreads / 4], keep[kBeamKeep], keep_tie[kBeamKeep];
    __shared__ u64 bound_s, bound_tie_s;
    __shared__ int count_s;
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.beams, S = a.slices, k = a.k;
    const int per = S * k, total_n = W * per;
    const u64* const keys = a.keys + static_cast<int64_t>(b) * total_n;
    // Candidate `i` of this thread.  Lists of 64 would put all their first ones with the same threads, and too many would reach the bound that
    // the groups below give (8 beams of 61 slices, k = 64: 2.2 ms); turned round by round, every group has some of the largest.
    auto index = [&](int i) { return i * kJoinThreads + static_cast<int>((threadIdx.x + i * 199u) % kJoinThreads); };
    const int rounds = (total_n + kJoinThreads - 1) / kJoinThreads;
    // the first candidates are on their way while the beams' sums are made (what belongs to a closed beam was not written and is not used)
    u64 raw[kJoinHold];
#pragma unroll
    for (int i = 0; i < kJoinHold; ++i) {
        const int n = index(i);
        raw[i] = n < total_n ? keys[n] : 0;
    }
    for (int w = warp; w < W; w += kJoinThreads / 32) {
        const int64_t at = (static_cast<int64_t>(b) * W + w) * S;
        const float score = a.scores[b * a.s_b + w * a.s_w];
        const bool done = a.finished && a.finished[b * a.f_b + w * a.f_w];
        float ms = lane < S ? a.tops[at + lane] : -INFINITY;
        double part = lane < S ? a.sums[at + lane] : 0.0;
        int what = 0;
        double value = 0.0;
        if (done || !(score > -INFINITY && score < INFINITY)) {
            what = done && score < INFINITY ? 1 : 2;
            if (lane == 0 && a.status && (score != score || score == INFINITY)) atomicCAS(a.status, 0, static_cast<int>(kStatusNonFinite));
        } else {
            float m = ms;
            for (int s = lane + 32; s < S; s += 32) m = fmaxf(m, a.tops[at + s]);
            m = warp_max(m);
            double sum = 0.0;
            for (int s = lane; s < S; s += 32) {
                if (s != lane) {
                    ms = a.tops[at + s];
                    part = a.sums[at + s];
                }
                sum += ms == m ? part : part * static_cast<double>(exp2_ftz((ms - m) * 1.4426950408889634f));
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
        if (lane == 0) {
            lse[w] = value;
            score_s[w] = score;
            kind[w] = what;
        }
    }
    if (threadIdx.x == 0) count_s = 0;
    __syncthreads();

    // candidate n of the request: its total in order (0: none), and the word that orders equal totals
    auto candidate = [&](int n, u64 key, u64& tie) -> u64 {
        const int w = n / per, i = n - w * per;
        const u64 beam = static_cast<u64>(kBeamMaxWidth - 1 - w) << 56;
        const double score = score_s[w];
        if (kind[w] == 0) {
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
    auto reload = [&](int n, u64& tie) { return candidate(n, keys[n], tie); };

    u64 held[kJoinHold], held_tie[kJoinHold], top = 0, top_tie = 0, tie = 0;
    auto larger = [](u64 x, u64 x_tie, u64 y, u64 y_tie) { return x > y || (x == y && x_tie > y_tie); };
    auto raise = [&](u64 key, u64 key_tie) {
        if (larger(key, key_tie, top, top_tie)) {
            top = key;
            top_tie = key_tie;
        }
    };
#pragma unroll
    for (int i = 0; i < kJoinHold; ++i) {
        const int n = index(i);
        held_tie[i] = 0;
        held[i] = n < total_n ? candidate(n, raw[i], held_tie[i]) : 0;
        if (held[i]) raise(held[i], held_tie[i]);
    }
    for (int i = kJoinHold; i < rounds; ++i) {
        const int n = index(i);
        if (const u64 key = n < total_n ? reload(n, tie) : 0) raise(key, tie);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, top, o), other_tie = __shfl_xor_sync(0xffffffffu, top_tie, o);
        raise(other, other_tie);
    }
    if ((lane & 3) == 0) {
        group_top[threadIdx.x >> 2] = top;
        group_tie[threadIdx.x >> 2] = top_tie;
    }
    if (threadIdx.x == 0) bound_s = bound_tie_s = 0;
    __syncthreads();
    {
        // the k-th largest of the groups' maxima, which all differ where there is one: four threads a group
        int above = 0, same = 0;
#pragma unroll 8
        for (int i = threadIdx.x & 3; i < kJoinThreads / 4; i += 4) {
            above += group_top[i] > top;
            same += group_top[i] == top;
        }
        if (same > ((threadIdx.x >> 2 & 3) == (threadIdx.x & 3)))        // others than the group itself
            for (int i = threadIdx.x & 3; i < kJoinThreads / 4; i += 4) above += group_top[i] == top && group_tie[i] > top_tie;
        above += __shfl_xor_sync(0xffffffffu, above, 1);
        above += __shfl_xor_sync(0xffffffffu, above, 2);
        if ((lane & 3) == 0 && above == k - 1 && top != 0) {
            bound_s = top;
            bound_tie_s = top_tie;
        }
    }
    __syncthreads();
    const u64 bound = bound_s, bound_tie = bound_tie_s;
    auto collect = [&](u64 key, u64 key_tie) {
        if (key != 0 && !larger(bound, bound_tie, key, key_tie)) {
            const int at = atomicAdd(&count_s, 1);
            if (at < kBeamKeep) {
                keep[at] = key;
                keep_tie[at] = key_tie;
            }
        }
    };
#pragma unroll
    for (int i = 0; i < kJoinHold; ++i) collect(held[i], held_tie[i]);
    for (int i = kJoinHold; i < rounds; ++i) {
        const int n = index(i);
        if (const u64 key = n < total_n ? reload(n, tie) : 0) collect(key, tie);
    }
    __syncthreads();
    int count = count_s;
    if (count > kBeamKeep) {
        // the k-th largest total, then the last of its equals that is still among the k
        int ties, none;
        u64 edge_tie = 0;
        const u64 edge = largest_edge([&](int n) { return reload(n, tie); }, total_n, k, reinterpret_cast<int*>(keep), ties);
        if (ties >= 0)
            edge_tie = largest_edge([&](int n) { const u64 key = reload(n, tie); return key == edge ? tie : 0; }, total_n, ties, reinterpret_cast<int*>(keep), none);
        __syncthreads();
        if (threadIdx.x == 0) count_s = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < total_n; i += kJoinThreads) {
            const u64 key = reload(i, tie);
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
    int cols, n, n_in, tensors, clear;
    int* status;
};

template <typename V> __device__ __forceinline__ void clear_piece(char* dst, int64_t begin, int64_t bytes) {
    const int64_t end = begin + kReorderPiece < bytes ? begin + kReorderPiece : bytes;
    for (int64_t o = begin + threadIdx.x * sizeof(V); o < end; o += kReorderThreads * sizeof(V)) *reinterpret_cast<V*>(dst + o) = V{};
}
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
        char* dst = a.out[t] + i * a.out_stride[t];
        const int64_t begin = (p - a.first[t]) * kReorderPiece;
        if (row < 0 || row >= a.n_in) {
            if (threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
            if (a.clear) {
                if (a.width[t] == 16) clear_piece<uint4>(dst, begin, a.bytes[t]);
                else if (a.width[t] == 4) clear_piece<uint32_t>(dst, begin, a.bytes[t]);
                else clear_piece<uint8_t>(dst, begin, a.bytes[t]);
            }
            continue;
        }
        const char* src = a.in[t] + row * a.in_stride[t];
        if (a.width[t] == 16) copy_piece<uint4>(src, dst, begin, a.bytes[t]);
        else if (a.width[t] == 4) copy_piece<uint32_t>(src, dst, begin, a.bytes[t]);
        else copy_piece<uint8_t>(src, dst, begin, a.bytes[t]);
    }
}

// Slices of a row: no more than there are steps, and together about two waves of CTAs (four on an SM at a time).  A CTA's first step
// finds its bound, which costs as much as the step; those behind it are cheap.  One CTA joins a request's k of every slice: with large k
// and many beams no more of them than it reads in a few microseconds (8 beams of 248320, k = 64: 61 slices 80 us, 16 slices 39).
constexpr int kJoinMost = 8192;
static int beam_slices(int rows, int beams, int vocab, int k, int type) {
    const int64_t bytes = static_cast<int64_t>(vocab) * (type == 2 ? 4 : 2);
    const int most = static_cast<int>((bytes + kStepBytes - 1) / kStepBytes), wave = 8 * sm_count() / (rows > 0 ? rows : 1), join = kJoinMost / (beams * k);
    const int share = wave < join ? wave : join;
    return share < 1 ? 1 : (share < most ? share : most);
}

}  // namespace nexrt

using namespace nexrt;

// Slices of a row: a call's scratch is batch * beams * slices * (k + 2) words of 8 bytes.
extern "C" int nexrt_beam_slices(int rows, int beams, int vocab, int k, int type) { return beams < 1 || k < 1 ? 1 : beam_slices(rows, beams, vocab, k, type); }

extern "C" int nexrt_beam_select(const NexrtBeamArgs* x, void* stream) {
    if (x->size != sizeof(*x) || x->batch < 0 || x->beams < 1 || x->beams > kBeamMaxWidth || x->vocab < 1 || x->vocab > kBeamMaxVocab || x->k < 1 || x->k > kBeamMaxK ||
        static_cast<int64_t>(x->beams) * x->vocab < x->k || (x->finished != nullptr && (x->eos < 0 || x->eos >= x->vocab)) ||
        static_cast<int64_t>(x->batch) * x->beams > 65535 || x->type < 0 || x->type > 2 || x->slices != beam_slices(x->batch * x->beams, x->beams, x->vocab, x->k, x->type))
        return cudaErrorInvalidValue;
    if (x->batch == 0) return 0;
    BeamArgs a = {};
    a.logits = x->logits; a.scores = static_cast<const float*>(x->scores); a.finished = static_cast<const unsigned char*>(x->finished);
    a.l_b = x->logits_request; a.l_w = x->logits_beam; a.s_b = x->scores_request; a.s_w = x->scores_beam; a.f_b = x->finished_request; a.f_w = x->finished_beam;
    a.batch = x->batch; a.beams = x->beams; a.vocab = x->vocab; a.k = x->k; a.eos = x->eos; a.slices = x->slices;
    const int64_t parts = static_cast<int64_t>(x->batch) * x->beams * x->slices;
    a.keys = static_cast<u64*>(x->scratch);
    a.sums = reinterpret_cast<double*>(a.keys + parts * x->k);
    a.tops = reinterpret_cast<float*>(a.sums + parts);
    a.scores_out = static_cast<float*>(x->scores_out); a.rows_out = static_cast<int*>(x->rows_out); a.tokens_out = static_cast<int*>(x->tokens_out);
    a.status = static_cast<int*>(x->status);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t size = x->type == 2 ? 4 : 2, strides = (x->batch > 1 ? x->logits_request : 0) | (x->beams > 1 ? x->logits_beam : 0);
    const bool aligned = ((reinterpret_cast<uintptr_t>(x->logits) | static_cast<uintptr_t>(strides * size)) & 15) == 0;
    const int e = x->type == 0 ? slice_launch<__nv_bfloat16>(a, aligned, st) : (x->type == 1 ? slice_launch<__half>(a, aligned, st) : slice_launch<float>(a, aligned, st));
    if (e) return e;
    return launch(beam_join_kernel, dim3(a.batch), dim3(kJoinThreads), 0, st, a);
}

extern "C" int nexrt_reorder_rows(const NexrtReorderArgs* x, void* stream) {
    if (x->size != sizeof(*x) || x->tensors < 0 || x->tensors > kReorderTensors || x->n < 0 || x->cols < 1 || x->n_in < 0) return cudaErrorInvalidValue;
    ReorderArgs a = {};
    for (int t = 0; t < x->tensors; ++t) {
        a.in[t] = static_cast<const char*>(x->in[t]);
        a.out[t] = static_cast<char*>(x->out[t]);
        a.in_stride[t] = x->in_row[t]; a.out_stride[t] = x->out_row[t]; a.bytes[t] = x->bytes[t];
        if (a.bytes[t] < 0) return cudaErrorInvalidValue;
        const uint64_t all = reinterpret_cast<uintptr_t>(x->in[t]) | reinterpret_cast<uintptr_t>(x->out[t]) | static_cast<uint64_t>(x->in_row[t]) |
                             static_cast<uint64_t>(x->out_row[t]) | static_cast<uint64_t>(x->bytes[t]);
        a.width[t] = all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : 1);
        a.first[t + 1] = a.first[t] + (a.bytes[t] + kReorderPiece - 1) / kReorderPiece;
    }
    a.rows = static_cast<const int*>(x->rows); a.r_0 = x->rows_0; a.r_1 = x->rows_1; a.cols = x->cols; a.n = x->n; a.n_in = x->n_in; a.tensors = x->tensors; a.clear = x->clear;
    a.status = static_cast<int*>(x->status);
    const int64_t units = a.first[x->tensors] * x->n, most = 8ll * sm_count();
    if (units == 0) return 0;
    return launch(reorder_kernel, dim3(static_cast<unsigned>(units < most ? units : most)), dim3(kReorderThreads), 0, static_cast<cudaStream_t>(stream), a);
}
