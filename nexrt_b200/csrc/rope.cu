// Rotary positions: rows of q and k heads are normalised (optionally) and rotated, k and v stored into the pages of their
// sequences, in one pass over the projection's output.
//
// Pair i of a head at position p turns by p * inv_freq[i]:  (a, b) -> scale * (a cos - b sin, b cos + a sin), with the pair at
// dims (i, i + rotary / 2), or (2 i, 2 i + 1) where the layout is interleaved; dims from `rotary` on pass through.  The angle is
// taken in turns in 64 bits and reduced before it is rounded to 32: at position 262144 a 32-bit product is 0.016 rad off, and
// sinpi / cospi of a reduced turn need no range reduction of their own.
//
// Bound by the bytes (each value read and written once).  A token's sines serve all its heads, so a CTA takes whole tokens; a
// head lies over 8, 16 or 32 lanes, eight values a lane, so its sum of squares is three to five shuffles and its pairs meet in
// shared memory without a barrier of the CTA.
#include "api.h"
#include "paged.cuh"

namespace nexrt {

struct RopeArgs {
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;        // q_out, k_out: [tokens][heads][dim]; with pages k_out and v_out are the pools
    int64_t q_t, q_h, k_t, k_h, v_t, v_h, qo_t, qo_h;   // strides in elements
    int64_t page_s, head_s, slot_s;     // strides of the pools
    const int *positions, *rows;
    PageTable table;
    const float *inv_freq, *q_norm, *k_norm;
    int* status;
    int tokens, q_heads, kv_heads, dim, rotary, interleaved, paged, vec;
    float scale, eps;
};

template <typename T> __device__ __forceinline__ float rope_load1(const T* p) { return static_cast<float>(*p); }
template <typename T> __device__ __forceinline__ void rope_store1(T* p, float v) { *p = static_cast<T>(v); }

__device__ __forceinline__ void unpack8(const uint4& w, float* f, __nv_bfloat16) { unpack8_bf16(w, f); }
__device__ __forceinline__ void unpack8(const uint4& w, float* f, __half) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        f[2 * i] = a.x;
        f[2 * i + 1] = a.y;
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T> __device__ __forceinline__ void load8(const T* p, float* f, bool vec) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        } else {
            unpack8(*reinterpret_cast<const uint4*>(p), f, T());
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = rope_load1(p + i);
    }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* f, bool vec) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>(p) = make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) rope_store1(p + i, f[i]);
    }
}

constexpr int kRopeThreads = 256;

// LPH lanes hold a head (8 values each): 8 for dims up to 64, 16 up to 128, 32 up to 256.
template <typename TI, typename TO, int LPH>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a) {
    constexpr int kHeads = 32 / LPH;                     // heads that a warp turns at once
    __shared__ float2 turn[128];                         // (cos, sin) of the token's pairs
    __shared__ float line[kRopeThreads / 32][256];       // a warp's heads in 32 bits
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int e0 = (lane % LPH) * 8, half = a.rotary / 2;
    const bool in_dim = e0 < a.dim;
    float* const mine = line[warp] + (lane / LPH) * LPH * 8;
    const int heads = a.q_heads + a.kv_heads + (a.v != nullptr ? a.kv_heads : 0);

    for (int t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const int pos = a.positions[t];
        __syncthreads();
        for (int i = threadIdx.x; i < half; i += kRopeThreads) {
            double turns = static_cast<double>(pos) * static_cast<double>(a.inv_freq[i]) * 0.15915494309189533577;
            turns -= rint(turns);
            float s, c;
            sincospif(2.f * static_cast<float>(turns), &s, &c);
            turn[i] = make_float2(c * a.scale, s * a.scale);
        }
        int64_t slot = -1;
        if (a.paged) {
            const int row = a.rows[t];
            if (row >= 0) {                              // a negative row is padding: nothing is stored for it
                slot = page_slot(a.table, row, pos);
                if (slot < 0 && threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, static_cast<int>(kStatusBadPage));
            }
        }
        const int64_t slot_at = slot < 0 ? 0 : slot / a.table.page * a.page_s + slot % a.table.page * a.slot_s;
        __syncthreads();

        for (int h0 = warp * kHeads; h0 < heads; h0 += kRopeThreads / 32 * kHeads) {
            const int h = h0 + lane / LPH;
            const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads, is_v = !is_q && !is_k && h < heads;
            const int hk = is_k ? h - a.q_heads : h - a.q_heads - a.kv_heads;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
            if (in_dim && h < heads) {
                const TI* src = is_q ? static_cast<const TI*>(a.q) + t * a.q_t + h * a.q_h
                                     : (is_k ? static_cast<const TI*>(a.k) + t * a.k_t + hk * a.k_h : static_cast<const TI*>(a.v) + t * a.v_t + hk * a.v_h);
                load8(src + e0, x, a.vec);
            }
            const float* w = is_q ? a.q_norm : (is_k ? a.k_norm : nullptr);
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (w != nullptr && in_dim) {
                const float r = rsqrtf(ss / static_cast<float>(a.dim) + a.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= r * w[e0 + i];
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) mine[e0 + i] = x[i];
            __syncwarp();
            if ((is_q || is_k) && e0 < a.rotary) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = e0 + i;
                    if (e < a.rotary) {
                        const bool second = a.interleaved ? (e & 1) : e >= half;
                        const int pair = a.interleaved ? e >> 1 : (second ? e - half : e);
                        const int other = a.interleaved ? e ^ 1 : (second ? e - half : e + half);
                        const float2 cs = turn[pair];
                        const float y = mine[other];
                        x[i] = second ? fmaf(x[i], cs.x, y * cs.y) : fmaf(x[i], cs.x, -(y * cs.y));
                    }
                }
            }
            if (!in_dim || h >= heads) continue;
            if (is_q) {
                store8(static_cast<TO*>(a.q_out) + t * a.qo_t + h * a.qo_h + e0, x, a.vec);
            } else if (!a.paged) {
                store8(static_cast<TO*>(a.k_out) + (static_cast<int64_t>(t) * a.kv_heads + hk) * a.dim + e0, x, a.vec);
            } else if (slot >= 0) {
                store8(static_cast<TO*>(is_v ? a.v_out : a.k_out) + slot_at + hk * a.head_s + e0, x, a.vec);
            }
        }
    }
}

template <typename TI, typename TO> static int rope_launch(const RopeArgs& a, cudaStream_t st) {
    const int grid = a.tokens < 8 * sm_count() ? a.tokens : 8 * sm_count();
    if (a.dim <= 64) return launch(rope_kernel<TI, TO, 8>, dim3(grid), dim3(kRopeThreads), 0, st, a);
    if (a.dim <= 128) return launch(rope_kernel<TI, TO, 16>, dim3(grid), dim3(kRopeThreads), 0, st, a);
    return launch(rope_kernel<TI, TO, 32>, dim3(grid), dim3(kRopeThreads), 0, st, a);
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace nexrt

using namespace nexrt;

// in_type, out_type: 0 bf16, 1 fp16, 2 fp32.  table == NULL: no pages, k goes to k_out (may be NULL with k == NULL, kv_heads 0).
extern "C" int nexrt_rope_append(const void* q, const void* k, const void* v, const void* positions, const void* rows, void* q_out, void* k_out, void* v_out,
                                 const void* table, const void* inv_freq, const void* q_norm, const void* k_norm, void* status, const int64_t* strides,
                                 int tokens, int q_heads, int kv_heads, int dim, int rotary, int interleaved, int table_rows, int width, int page, int pages,
                                 int in_type, int out_type, float scale, float eps, void* stream) {
    if (tokens < 0 || q_heads < 0 || kv_heads < 0 || dim < 8 || dim > 256 || dim % 8 || rotary < 0 || rotary > dim || rotary % 2) return cudaErrorInvalidValue;
    if (table != nullptr && (page < 1 || width < 0 || pages < 0 || table_rows < 0)) return cudaErrorInvalidValue;
    if (tokens == 0 || q_heads + kv_heads == 0) return 0;
    RopeArgs a = {};
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.k_out = k_out; a.v_out = v_out;
    a.q_t = strides[0]; a.q_h = strides[1]; a.k_t = strides[2]; a.k_h = strides[3]; a.v_t = strides[4]; a.v_h = strides[5];
    a.qo_t = strides[6]; a.qo_h = strides[7]; a.page_s = strides[8]; a.head_s = strides[9]; a.slot_s = strides[10];
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
