// Rotary positions: rows of q and k heads are normalised (optionally) and rotated, k and v stored into the pages of their
// sequences, in one pass over the projection's output.
//
// Pair i of a head at position p turns by p * inv_freq[i]:  (a, b) -> scale * (a cos - b sin, b cos + a sin), with the pair at
// dims (i, i + rotary / 2), or (2 i, 2 i + 1) where the layout is interleaved; dims from `rotary` on pass through.  The angle is
// taken in turns in 64 bits and reduced before it is rounded to 32: at position 262144 a 32-bit product is 0.016 rad off, and
// sinpi / cospi of a reduced turn need no range reduction of their own.
//
// Bound by the bytes (each value read and written once).  A CTA takes one token: its sines serve all its heads, and lie in the
// registers of the lanes that need them, multiplied with the norm's multipliers.  A head lies over 8, 16 or 32 lanes, eight
// values a lane: its sum of squares is three to five shuffles, and a value meets the other one of its pair in its own lane
// (interleaved), by a shuffle of the raw words, or, where half the rotated dims are no multiple of eight, in shared memory.
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

// Two 32-bit values in one register pair: one instruction does for both what the names say.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

constexpr int kRopeThreads = 128;
constexpr int kRopeWarps = kRopeThreads / 32;

// How a value meets the other one of its pair.
enum RopeLayout { kPairsInLane, kPairsByShuffle, kPairsByLine };

// LPH lanes hold a head (8 values each): 8 for dims up to 64, 16 up to 128, 32 up to 256.
template <typename TI, typename TO, int LPH, int LAYOUT>
__global__ void __launch_bounds__(kRopeThreads, sizeof(TI) == 4 ? 6 : 7) rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int kHeads = 32 / LPH;                     // heads that a warp turns at once
    constexpr int kAhead = sizeof(TI) == 4 ? 2 : 4;      // of which so many are in flight
    __shared__ float2 turn[128];                         // (cos, sin) of the token's pairs
    __shared__ int64_t slot_s;                           // where the token's slot lies in the pools, -1: nowhere
    __shared__ float line[LAYOUT == kPairsByLine ? kRopeWarps : 1][256];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LPH;
    const int e0 = sub * 8, half = a.rotary / 2;
    const bool in_dim = e0 < a.dim;
    const int heads = a.q_heads + 2 * a.kv_heads, qk = a.q_heads + a.kv_heads;
    const int64_t t = blockIdx.x;
    const TI* const q = static_cast<const TI*>(a.q) + t * a.q_t + e0;
    const TI* const k = static_cast<const TI*>(a.k) + t * a.k_t + e0;
    const TI* const v = static_cast<const TI*>(a.v) + t * a.v_t + e0;
    TO* const q_out = static_cast<TO*>(a.q_out) + t * a.qo_t + e0;

    // ---- a warp's heads lie side by side, so that few warps meet more than one kind; the first loads do not wait for the angles
    const int per_warp = ((heads + kHeads - 1) / kHeads + kRopeWarps - 1) / kRopeWarps * kHeads;
    const int end = min(heads, (warp + 1) * per_warp), first = warp * per_warp + lane / LPH;
    Eight<TI> raw[kAhead];
    auto fetch = [&](int h, Eight<TI>& r) {
        if (!in_dim || h >= end) {
            r.clear();
            return;
        }
        r.load(h < a.q_heads ? q + static_cast<int64_t>(h) * a.q_h
                             : (h < qk ? k + static_cast<int64_t>(h - a.q_heads) * a.k_h : v + static_cast<int64_t>(h - qk) * a.v_h), a.vec);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(first + i * kHeads, raw[i]);

    const int pos = a.positions[t];
    if (a.paged && threadIdx.x == kRopeThreads - 1) {
        int64_t at = -1;
        const int row = a.rows[t];
        if (row >= 0) {                                  // a negative row is padding: nothing is stored for it
            const int j = pos / a.table.page, page = pos < 0 ? -1 : page_at(a.table, row, j);
            if (page >= 0) at = page * a.page_s + (pos - j * a.table.page) * a.slot_s;
            else if (a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
        }
        slot_s = at;
    }
    for (int i = threadIdx.x; i < half; i += kRopeThreads) {
        double turns = static_cast<double>(pos) * static_cast<double>(a.inv_freq[i]) * 0.15915494309189533577;
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * static_cast<float>(turns), &s, &c);
        turn[i] = make_float2(c * a.scale, s * a.scale);
    }
    __syncthreads();
    const int64_t slot = a.paged ? slot_s : -1;
    TO* const k_out = static_cast<TO*>(a.k_out) + slot + e0;
    TO* const v_out = static_cast<TO*>(a.v_out) + slot + e0;

    // ---- value i of the lane becomes r (x cw + other sw): cos and sin, and the norm's multipliers of both
    float2 cw[4], sw[4];
    int kind = -1;                                       // whose they are: 0 q, 1 k
    auto factors = [&](const float* w) {
        float c[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = e0 + i;
            c[i] = w != nullptr ? w[e] : 1.f;
            s[i] = 0.f;
            if (e < a.rotary) {
                const bool second = LAYOUT == kPairsInLane ? (i & 1) : e >= half;
                const int pair = LAYOUT == kPairsInLane ? e >> 1 : (second ? e - half : e);
                const int other = LAYOUT == kPairsInLane ? e ^ 1 : (second ? e - half : e + half);
                const float2 cs = turn[pair];
                c[i] *= cs.x;
                s[i] = (second ? cs.y : -cs.y) * (w != nullptr ? w[other] : 1.f);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cw[i] = make_float2(c[2 * i], c[2 * i + 1]);
            sw[i] = make_float2(s[2 * i], s[2 * i + 1]);
        }
    };
    const bool turned = e0 < a.rotary;
    const int from = !turned ? lane : (e0 < half ? lane + half / 8 : lane - half / 8);
    const float inv_dim = 1.f / static_cast<float>(a.dim);

    for (int h0 = first; h0 - lane / LPH < end; h0 += kAhead * kHeads) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int h = h0 + u * kHeads;
            if (h - lane / LPH >= end) break;            // the same for all lanes of the warp
            // (a value that does not turn meets a zero: no 0 * infinity)
            float2 x[4], other[4];
            raw[u].values(x);
            if (LAYOUT == kPairsByShuffle) {
                Eight<TI> o;
#pragma unroll
                for (int i = 0; i < Eight<TI>::kWords; ++i) {
                    o.w[i] = __shfl_sync(0xffffffffu, raw[u].w[i], from);
                    o.w[i] = turned ? o.w[i] : 0u;
                }
                o.values(other);
            } else if (LAYOUT == kPairsInLane) {
#pragma unroll
                for (int i = 0; i < 4; ++i) other[i] = e0 + 2 * i < a.rotary ? make_float2(x[i].y, x[i].x) : make_float2(0.f, 0.f);
            } else {
                float* const mine = line[warp] + (lane - sub) * 8;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(mine + e0 + 2 * i) = x[i];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = e0 + 2 * i;
                    other[i].x = e < a.rotary ? mine[e < half ? e + half : e - half] : 0.f;
                    other[i].y = e + 1 < a.rotary ? mine[e + 1 < half ? e + 1 + half : e + 1 - half] : 0.f;
                }
            }
            float r = 1.f;
            if (a.q_norm != nullptr || a.k_norm != nullptr) {
                float2 sq = mul2(x[0], x[0]);
#pragma unroll
                for (int i = 1; i < 4; ++i) sq = fma2(x[i], x[i], sq);
                float ss = sq.x + sq.y;
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if ((h < a.q_heads ? a.q_norm : a.k_norm) != nullptr) r = rsqrtf(fmaf(ss, inv_dim, a.eps));
            }
            fetch(h + kAhead * kHeads, raw[u]);
            if (!in_dim || h >= end) continue;
            if (h < qk) {
                if (kind != (h < a.q_heads ? 0 : 1)) {
                    kind = h < a.q_heads ? 0 : 1;
                    factors(kind ? a.k_norm : a.q_norm);
                }
                const float2 rr = make_float2(r, r);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = mul2(rr, fma2(other[i], sw[i], mul2(x[i], cw[i])));
            }
            if (h < a.q_heads) store8(q_out + static_cast<int64_t>(h) * a.qo_h, x, a.vec);
            else if (slot >= 0) store8((h < qk ? k_out : v_out) + static_cast<int64_t>(h < qk ? h - a.q_heads : h - qk) * a.head_s, x, a.vec);
        }
    }
}

template <typename TI, typename TO, int LPH> static int rope_layout(const RopeArgs& a, cudaStream_t st) {
    const dim3 grid(a.tokens), block(kRopeThreads);
    if (a.interleaved) return launch(rope_kernel<TI, TO, LPH, kPairsInLane>, grid, block, 0, st, a);
    if (a.rotary % 16 == 0) return launch(rope_kernel<TI, TO, LPH, kPairsByShuffle>, grid, block, 0, st, a);   // both values of a pair at the same place of their lanes
    return launch(rope_kernel<TI, TO, LPH, kPairsByLine>, grid, block, 0, st, a);
}

template <typename TI, typename TO> static int rope_launch(const RopeArgs& a, cudaStream_t st) {
    if (a.dim <= 64) return rope_layout<TI, TO, 8>(a, st);
    if (a.dim <= 128) return rope_layout<TI, TO, 16>(a, st);
    return rope_layout<TI, TO, 32>(a, st);
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace nexrt

using namespace nexrt;

// in_type, out_type: 0 bf16, 1 fp16, 2 fp32.  table == NULL: q alone, kv_heads is 0.
extern "C" int nexrt_rope_append(const void* q, const void* k, const void* v, const void* positions, const void* rows, void* q_out, void* k_out, void* v_out,
                                 const void* table, const void* inv_freq, const void* q_norm, const void* k_norm, void* status, const int64_t* strides,
                                 int tokens, int q_heads, int kv_heads, int dim, int rotary, int interleaved, int table_rows, int width, int page, int pages,
                                 int in_type, int out_type, float scale, float eps, void* stream) {
    if (tokens < 0 || q_heads < 0 || kv_heads < 0 || dim < 8 || dim > 256 || dim % 8 || rotary < 0 || rotary > dim || rotary % 2) return cudaErrorInvalidValue;
    if (table != nullptr ? (page < 1 || width < 0 || pages < 0 || table_rows < 0) : kv_heads != 0) return cudaErrorInvalidValue;
    if (tokens == 0 || q_heads + kv_heads == 0) return 0;
    RopeArgs a = {};
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.k_out = k_out; a.v_out = v_out;
    for (const int i : {1, 3, 5, 7, 9})
        if (strides[i] < 0 || strides[i] > INT32_MAX) return cudaErrorInvalidValue;
    a.q_t = strides[0]; a.k_t = strides[2]; a.v_t = strides[4]; a.qo_t = strides[6]; a.page_s = strides[8]; a.slot_s = strides[10];
    a.q_h = static_cast<int>(strides[1]); a.k_h = static_cast<int>(strides[3]); a.v_h = static_cast<int>(strides[5]);
    a.qo_h = static_cast<int>(strides[7]); a.head_s = static_cast<int>(strides[9]);
    a.positions = static_cast<const int*>(positions); a.rows = static_cast<const int*>(rows);
    a.table = {static_cast<const int*>(table), strides[11], table_rows, width, page, pages};
    a.inv_freq = static_cast<const float*>(inv_freq); a.q_norm = static_cast<const float*>(q_norm); a.k_norm = static_cast<const float*>(k_norm);
    a.status = static_cast<int*>(status);
    a.tokens = tokens; a.q_heads = q_heads; a.kv_heads = kv_heads; a.dim = dim; a.rotary = rotary; a.interleaved = interleaved;
    a.paged = table != nullptr; a.scale = scale; a.eps = eps;
    // 16-byte accesses where every head starts on such a boundary on both sides
    bool vec = aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(k_out) && aligned16(v_out);
    for (int i = 0; i < 11; ++i) vec = vec && strides[i] % 8 == 0;
    a.vec = vec;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (in_type * 3 + out_type) {
        case 0: return rope_launch<__nv_bfloat16, __nv_bfloat16>(a, st);
        case 4: return rope_launch<__half, __half>(a, st);
        case 6: return rope_launch<float, __nv_bfloat16>(a, st);
        case 7: return rope_launch<float, __half>(a, st);
        case 8: return rope_launch<float, float>(a, st);
        default: return cudaErrorInvalidValue;
    }
}
