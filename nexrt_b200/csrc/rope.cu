// Rotary positions: rows of q and k heads are normalised (optionally) and rotated, k and v stored into the pages of their
// sequences, in one pass over the projection's output.
//
// Pair i of a head at position p turns by p * inv_freq[i]:  (a, b) -> scale * (a cos - b sin, b cos + a sin), with the pair at
// dims (i, i + rotary / 2), or (2 i, 2 i + 1) where the layout is interleaved; dims from `rotary` on pass through.  The angle is
// taken in turns in 64 bits and reduced before it is rounded to 32: at position 262144 a 32-bit product is 0.016 rad off, and
// sinpi / cospi of a reduced turn need no range reduction of their own.
//
// Bound by the bytes (each value read and written once), with the instructions close behind.  The heads of all tokens are cut into
// equal runs, one per resident warp, so the last wave is as full as the first; a warp keeps four steps of loads in flight over
// the tokens' borders and makes a token's sines itself, so no warp waits for another.  The factors of a token - sines times the
// norm's multipliers - stay in registers for all its heads.  A head lies over 4, 8 or 16 lanes, 16 values a lane: its sum of
// squares is two to four shuffles for several heads at once; sums and products go two values an instruction.
//
// Measured: 4099 tokens of 36 heads of 256 (151 MB) 34 us, 0.69 of copy rate: 130 instructions a head keep the schedulers half busy, with
// four warps each to hide their latencies (six CTAs an SM have to spill: 37 us).  Eight tokens of six heads: 4.1 us, the chain from
// the position to the stores.
#include "api.h"
#include "paged.cuh"

namespace nexrt {

struct RopeArgs {
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;        // q_out: [tokens][heads][dim]; k_out and v_out are the pools
    int64_t q_t, k_t, v_t, qo_t;        // strides in elements: of a token,
    int q_h, k_h, v_h, qo_h;            // of a head (32 bits: one multiply-add an address)
    int64_t page_s, slot_s;             // of the pools
    int head_s;
    const int *positions, *rows;
    PageTable table;
    const float *inv_freq, *q_norm, *k_norm;
    int* status;
    int tokens, q_heads, kv_heads, dim, rotary, interleaved, paged, vec;
    float scale, eps;
};

__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight values of a head as they lie in memory: four words of 16-bit pairs, or eight of 32 bits.
template <typename T> struct Eight {
    static constexpr int kWords = sizeof(T) == 4 ? 8 : 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* p, bool vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const unsigned short*>(p)[2 * i] | static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(p)[2 * i + 1]) << 16;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void values(float2 (&x)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) x[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
            else x[i] = unpack2(w[i], T());
        }
    }
};

template <typename T> __device__ __forceinline__ void store8(T* p, const float2 (&f)[4], bool vec) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(p)[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
            reinterpret_cast<float4*>(p)[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
        } else {
            *reinterpret_cast<uint4*>(p) = make_uint4(pack2(f[0].x, f[0].y, T()), pack2(f[1].x, f[1].y, T()), pack2(f[2].x, f[2].y, T()), pack2(f[3].x, f[3].y, T()));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[2 * i] = static_cast<T>(f[i].x);
            p[2 * i + 1] = static_cast<T>(f[i].y);
        }
    }
}

constexpr int kRopeThreads = 128;
constexpr int kRopeResident = 4;        // CTAs on an SM
constexpr int kRopeWarps = kRopeThreads / 32;

// How a value meets the other one of its pair: (2 i, 2 i + 1) are in one lane; the rotated dims lie in the first halves of the lanes'
// values, a shuffle apart; they are the two halves of a lane's values; anything else goes through shared memory, and so do tensors that
// cannot be read 16 bytes at a time.  (4096 tokens of 32 heads of 192, all dims turned: across 25.2 us, through shared memory 55.6.)
enum RopeLayout { kPairsInLane, kPairsByShuffle, kPairsAcross, kPairsByLine };

// LPH lanes hold a head, 16 values each: 4 for dims up to 64, 8 up to 128, 16 up to 256.  Values 8 sub .. and LPH * 8 + 8 sub .. are lane
// sub's, so that a warp reads whole lines; where pairs lie across, 8 sub .. and dim / 2 + 8 sub .. of the lanes below dim / 16.
template <typename TI, typename TO, int LPH, int LAYOUT>
__global__ void __launch_bounds__(kRopeThreads, kRopeResident) rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int kHeads = 32 / LPH;                     // heads that a warp turns at once
    constexpr int kAhead = 4;                            // steps of which so many are in flight
    constexpr bool kVec = LAYOUT != kPairsByLine;
    constexpr int kWide = sizeof(TI) == 4 ? 2 : 1;       // 16-byte pieces of eight values
    __shared__ float2 turns_s[kRopeWarps][128];          // (cos, sin) of a warp's token's pairs
    __shared__ float line[LAYOUT == kPairsByLine ? kRopeWarps : 1][LAYOUT == kPairsByLine ? 512 : 1];
    __shared__ uint4 ring_s[kVec ? kRopeWarps : 1][kVec ? kAhead : 1][2 * kWide][32];   // a lane reads back what it copied itself
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LPH;
    const int e0 = sub * 8, half = a.rotary / 2, gap = LAYOUT == kPairsAcross ? half : LPH * 8;    // gap: from a lane's first eight values to its second
    const bool vec = kVec || a.vec;                      // 16-byte stores
    const int heads = a.q_heads + 2 * a.kv_heads, qk = a.q_heads + a.kv_heads, steps = (heads + kHeads - 1) / kHeads;
    float2* const turn = turns_s[warp];

    // ---- this warp's steps, of all tokens' (kHeads heads of one token each)
    const int64_t total = static_cast<int64_t>(a.tokens) * steps;
    const int n = gridDim.x * kRopeWarps, w_id = blockIdx.x * kRopeWarps + warp;
    const int64_t begin = range_begin(total, w_id, n);
    int left = static_cast<int>(range_begin(total, w_id + 1, n) - begin), ahead = left;
    if (left == 0) return;
    int t = static_cast<int>(quotient(begin, steps)), i = static_cast<int>(begin - static_cast<int64_t>(t) * steps);

    uint4 (*const ring)[2 * kWide][32] = ring_s[kVec ? warp : 0];
    int ft = t, fi = i;                                  // the step that is fetched next
    auto source = [&](int64_t t_, int h) -> const TI* {
        if (h < a.q_heads) return static_cast<const TI*>(a.q) + t_ * a.q_t + static_cast<int64_t>(h) * a.q_h + e0;
        if (h < qk) return static_cast<const TI*>(a.k) + t_ * a.k_t + static_cast<int64_t>(h - a.q_heads) * a.k_h + e0;
        return static_cast<const TI*>(a.v) + t_ * a.v_t + static_cast<int64_t>(h - qk) * a.v_h + e0;
    };
    // steps whose heads are all of q, the most there are, need no choice: a pointer runs along
    const int q_steps = a.q_heads / kHeads;
    const int64_t q_step = static_cast<int64_t>(kHeads) * a.q_h, out_step = static_cast<int64_t>(kHeads) * a.qo_h;
    const TI* q_from = static_cast<const TI*>(a.q) + ft * a.q_t + static_cast<int64_t>(fi * kHeads + lane / LPH) * a.q_h + e0;
    const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(&ring_s[kVec ? warp : 0][0][0][lane]));
    const bool in0 = e0 < (LAYOUT == kPairsAcross ? half : a.dim), in1 = in0 && e0 + gap < a.dim;
    const int far = in1 ? gap : 0;
    auto fetch = [&](int at) {
        const int h = fi * kHeads + lane / LPH;
        if (ahead > 0 && h < heads) {
            const TI* src = fi < q_steps ? q_from : source(ft, h);
            if (!in0) src -= e0;                         // (a lane without dims copies nothing, from a valid place)
            const uint32_t dst = ring_at + at * (2 * kWide * 512);
#pragma unroll
            for (int j = 0; j < kWide; ++j) {
                cp16(dst + j * 512, src + (in0 ? j * 4 : 0), in0);
                cp16(dst + (kWide + j) * 512, src + far + (in1 ? j * 4 : 0), in1);
            }
        }
        cp_commit();
        --ahead;
        q_from += q_step;
        if (++fi == steps) {
            fi = 0;
            ++ft;
            q_from = static_cast<const TI*>(a.q) + ft * a.q_t + static_cast<int64_t>(lane / LPH) * a.q_h + e0;
        }
    };
    if (kVec) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) fetch(u);
    }

    // ---- a token: its angles, and the entry of the table that its k and v need; the next one's position and row are on their way
    TO* q_to = nullptr;                                  // head lane / LPH of the token's q
    int pos = 0, row = -1, entry = -1, next_pos = a.positions[t], next_row = a.paged ? a.rows[t] : -1;
    auto begin_token = [&]() {
        q_to = static_cast<TO*>(a.q_out) + t * a.qo_t + static_cast<int64_t>(lane / LPH) * a.qo_h + e0;
        pos = next_pos;
        row = next_row;
        if (t + 1 < a.tokens) {
            next_pos = a.positions[t + 1];
            if (a.paged) next_row = a.rows[t + 1];
        }
        entry = pos < 0 ? -1 : page_entry(a.table, row, pos / a.table.page);     // (checked where it is used: the load is not waited for here)
        __syncwarp();
        for (int p = lane; p < half; p += 32) {
            double turns = static_cast<double>(pos) * static_cast<double>(a.inv_freq[p]) * 0.15915494309189533577;
            turns -= rint(turns);
            float s, c;
            sincospif(2.f * static_cast<float>(turns), &s, &c);
            turn[p] = make_float2(c * a.scale, s * a.scale);
        }
        __syncwarp();
    };

    // ---- value i of the lane becomes r (x cw + other sw): cos and sin, and the norm's multipliers of both
    float2 cw[2][4], sw[2][4];
    int kind = -1;                                       // whose they are: 0 q, 1 k
    const bool pairs_in_lane = LAYOUT == kPairsInLane || (LAYOUT == kPairsByLine && a.interleaved);
    auto factors = [&](const float* w) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float cs_[8], sn[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = e0 + c * gap + i;
                cs_[i] = w != nullptr && e < a.dim ? w[e] : 1.f;
                sn[i] = 0.f;
                if (e < a.rotary) {
                    const bool second = pairs_in_lane ? (i & 1) : e >= half;
                    const int pair = pairs_in_lane ? e >> 1 : (second ? e - half : e);
                    const int other = pairs_in_lane ? e ^ 1 : (second ? e - half : e + half);
                    const float2 cs = turn[pair];
                    cs_[i] *= cs.x;
                    sn[i] = (second ? cs.y : -cs.y) * (w != nullptr ? w[other] : 1.f);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                cw[c][i] = make_float2(cs_[2 * i], cs_[2 * i + 1]);
                sw[c][i] = make_float2(sn[2 * i], sn[2 * i + 1]);
            }
        }
    };
    const bool turned = e0 < a.rotary;
    const int from = !turned ? lane : (e0 < half ? lane + half / 8 : lane - half / 8);
    const float inv_dim = 1.f / static_cast<float>(a.dim);

    begin_token();
    for (int at = 0; left > 0; --left, at = at + 1 == kAhead ? 0 : at + 1) {
        if (i == steps) {
            i = 0;
            ++t;
            kind = -1;
            begin_token();
        }
        const bool all_q = i < q_steps;                  // the same for all lanes
        const int h = i++ * kHeads + lane / LPH;
        Eight<TI> raw[2];
        if (kVec) {
            cp_wait<kAhead - 1>();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int j = 0; j < kWide; ++j) {
                    const uint4 v = ring[at][c * kWide + j][lane];
                    raw[c].w[4 * j] = v.x; raw[c].w[4 * j + 1] = v.y; raw[c].w[4 * j + 2] = v.z; raw[c].w[4 * j + 3] = v.w;
                }
        } else {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (h < heads && e0 + c * gap < a.dim) raw[c].load(source(t, h) + c * gap, a.vec);
                else raw[c].clear();
            }
        }
        float2 x[2][4];
        raw[0].values(x[0]);
        raw[1].values(x[1]);
        float2 other[4];                             // of the first eight, by shuffle
        if (LAYOUT == kPairsByShuffle) {
            Eight<TI> o;
#pragma unroll
            for (int i = 0; i < Eight<TI>::kWords; ++i) {
                o.w[i] = __shfl_sync(0xffffffffu, raw[0].w[i], from);
                o.w[i] = turned ? o.w[i] : 0u;       // a value that does not turn meets a zero: no 0 * infinity
            }
            o.values(other);
        }
        float* const mine = line[LAYOUT == kPairsByLine ? warp : 0] + (lane - sub) * 16;
        if (LAYOUT == kPairsByLine) {
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(mine + e0 + c * gap + 2 * i) = x[c][i];
            __syncwarp();
        }
        float r = 1.f;
        if (a.q_norm != nullptr || a.k_norm != nullptr) {
            float2 sq = mul2(x[0][0], x[0][0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) sq = fma2(x[0][i], x[0][i], sq);
#pragma unroll
            for (int i = 0; i < 4; ++i) sq = fma2(x[1][i], x[1][i], sq);
            float ss = sq.x + sq.y;
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if ((all_q || h < a.q_heads ? a.q_norm : a.k_norm) != nullptr) r = rsqrtf(fmaf(ss, inv_dim, a.eps));
        }
        if (kVec) {
            __syncwarp();
            fetch(at);                               // into the place that was just read
        }
        if (!all_q && h >= heads) continue;
        if (all_q || h < qk) {
            if (kind != (all_q || h < a.q_heads ? 0 : 1)) {
                kind = all_q || h < a.q_heads ? 0 : 1;
                factors(kind ? a.k_norm : a.q_norm);
            }
            const float2 rr = make_float2(r, r);
            if (LAYOUT == kPairsByShuffle) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[0][i] = mul2(rr, fma2(other[i], sw[0][i], mul2(x[0][i], cw[0][i])));
                    x[1][i] = mul2(rr, mul2(x[1][i], cw[1][i]));
                }
            } else if (LAYOUT == kPairsAcross) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 y = x[0][i], z = x[1][i];
                    x[0][i] = mul2(rr, fma2(z, sw[0][i], mul2(y, cw[0][i])));
                    x[1][i] = mul2(rr, fma2(y, sw[1][i], mul2(z, cw[1][i])));
                }
            } else {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = e0 + c * gap + 2 * i;
                        float2 o = make_float2(0.f, 0.f);
                        if (pairs_in_lane) {
                            if (e < a.rotary) o = make_float2(x[c][i].y, x[c][i].x);
                        } else {
                            if (e < a.rotary) o.x = mine[e < half ? e + half : e - half];
                            if (e + 1 < a.rotary) o.y = mine[e + 1 < half ? e + 1 + half : e + 1 - half];
                        }
                        x[c][i] = mul2(rr, fma2(o, sw[c][i], mul2(x[c][i], cw[c][i])));
                    }
            }
        }
        TO* dst;
        if (all_q || h < a.q_heads) {
            dst = q_to + (i - 1) * out_step;
        } else {
            if (row < 0) continue;                   // padding: nothing is stored for it
            if (entry < 0 || entry >= a.table.pages) {
                if (a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
                continue;
            }
            dst = static_cast<TO*>(h < qk ? a.k_out : a.v_out) + entry * a.page_s + static_cast<int64_t>(pos % a.table.page) * a.slot_s +
                  static_cast<int64_t>(h < qk ? h - a.q_heads : h - qk) * a.head_s + e0;
        }
        if (in0) store8(dst, x[0], vec);
        if (in1) store8(dst + gap, x[1], vec);
    }
}

template <typename TI, typename TO, int LPH> static int rope_layout(const RopeArgs& a, cudaStream_t st) {
    constexpr int kHeads = 32 / LPH;
    const int64_t steps = static_cast<int64_t>(a.tokens) * ((a.q_heads + 2 * a.kv_heads + kHeads - 1) / kHeads), most = static_cast<int64_t>(kRopeResident) * sm_count();
    const int64_t ctas = (steps + kRopeWarps - 1) / kRopeWarps;
    const dim3 grid(static_cast<unsigned>(ctas < most ? ctas : most)), block(kRopeThreads);
    if (!a.vec) return launch(rope_kernel<TI, TO, LPH, kPairsByLine>, grid, block, 0, st, a);
    if (a.interleaved) return launch(rope_kernel<TI, TO, LPH, kPairsInLane>, grid, block, 0, st, a);
    if (a.rotary % 16 == 0 && a.rotary <= LPH * 8) return launch(rope_kernel<TI, TO, LPH, kPairsByShuffle>, grid, block, 0, st, a);
    if (a.rotary == a.dim && a.dim % 16 == 0) return launch(rope_kernel<TI, TO, LPH, kPairsAcross>, grid, block, 0, st, a);
    return launch(rope_kernel<TI, TO, LPH, kPairsByLine>, grid, block, 0, st, a);
}

template <typename TI, typename TO> static int rope_launch(const RopeArgs& a, cudaStream_t st) {
    if (a.dim <= 64) return rope_layout<TI, TO, 4>(a, st);
    if (a.dim <= 128) return rope_layout<TI, TO, 8>(a, st);
    return rope_layout<TI, TO, 16>(a, st);
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace nexrt

using namespace nexrt;

extern "C" int nexrt_rope_append(const NexrtRopeArgs* x, void* stream) {
    if (x->size != sizeof(*x)) return cudaErrorInvalidValue;
    const bool paged = x->rows != nullptr;      // (a table without entries has no address)
    if (x->tokens < 0 || x->q_heads < 0 || x->kv_heads < 0 || x->dim < 8 || x->dim > 256 || x->dim % 8 || x->rotary < 0 || x->rotary > x->dim || x->rotary % 2) return cudaErrorInvalidValue;
    if (paged ? (x->slots < 1 || x->width < 0 || x->pages < 0 || x->table_rows < 0) : x->kv_heads != 0) return cudaErrorInvalidValue;
    if (x->tokens == 0 || x->q_heads + x->kv_heads == 0) return 0;
    const int64_t head_strides[5] = {x->q_head, x->k_head, x->v_head, x->out_head, x->head};
    for (const int64_t h : head_strides)
        if (h < 0 || h > INT32_MAX) return cudaErrorInvalidValue;
    RopeArgs a = {};
    a.q = x->q; a.k = x->k; a.v = x->v; a.q_out = x->q_out; a.k_out = x->k_pages; a.v_out = x->v_pages;
    a.q_t = x->q_token; a.k_t = x->k_token; a.v_t = x->v_token; a.qo_t = x->out_token; a.page_s = x->page; a.slot_s = x->slot;
    a.q_h = static_cast<int>(x->q_head); a.k_h = static_cast<int>(x->k_head); a.v_h = static_cast<int>(x->v_head);
    a.qo_h = static_cast<int>(x->out_head); a.head_s = static_cast<int>(x->head);
    a.positions = static_cast<const int*>(x->positions); a.rows = static_cast<const int*>(x->rows);
    a.table = {static_cast<const int*>(x->table), x->table_row, x->table_rows, x->width, paged ? x->slots : 1, x->pages};
    a.inv_freq = static_cast<const float*>(x->inv_freq); a.q_norm = static_cast<const float*>(x->q_norm); a.k_norm = static_cast<const float*>(x->k_norm);
    a.status = static_cast<int*>(x->status);
    a.tokens = x->tokens; a.q_heads = x->q_heads; a.kv_heads = x->kv_heads; a.dim = x->dim; a.rotary = x->rotary; a.interleaved = x->interleaved;
    a.paged = paged; a.scale = x->scale; a.eps = x->eps;
    // 16-byte accesses where every head starts on such a boundary on both sides
    const int64_t strides = x->q_token | x->q_head | x->k_token | x->k_head | x->v_token | x->v_head | x->out_token | x->out_head | x->page | x->head | x->slot;
    a.vec = aligned16(x->q) && aligned16(x->k) && aligned16(x->v) && aligned16(x->q_out) && aligned16(x->k_pages) && aligned16(x->v_pages) && strides % 8 == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (x->in_type * 3 + x->out_type) {
        case 0: return rope_launch<__nv_bfloat16, __nv_bfloat16>(a, st);
        case 4: return rope_launch<__half, __half>(a, st);
        case 6: return rope_launch<float, __nv_bfloat16>(a, st);
        case 7: return rope_launch<float, __half>(a, st);
        case 8: return rope_launch<float, float>(a, st);
        default: return cudaErrorInvalidValue;
    }
}
