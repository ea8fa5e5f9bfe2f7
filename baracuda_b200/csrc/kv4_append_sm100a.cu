// Norms of queries and keys per head, the rotation by position, and the 4-bit cache's writer and reader.
//   y = x * (1 / sqrt(mean(x^2) + eps)) * weight                    (per head; skipped without a weight)
//   (a, b) -> (a * cos - b * sin, b * cos + a * sin)                (channel pairs; angle by the position on the pair's axis)
//   out = bf16(...)                                                 (one rounding, queries and dense keys)
//   s = f16((max - min) / 15), m = f16(min), c = clamp(rint((x - m) / s), 0, 15)    (per 64 channels of the bf16 keys and values)
// Every step is one IEEE rounding in f32, in this order, except the mean square: it is summed in 64 bits and rounded once, so
// its bits do not depend on the order of the sum and a key next to the border of two codes gets the same code from this kernel,
// from the two-call sequence and from any other evaluation.
// Bound: bytes (each element read and written once).  A head is D / 8 lanes of 8 channels, held as two quads that contain
// whole rotation pairs, so nothing is exchanged between lanes but the sums and the groups' extrema.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/baracuda_kernels_q.h"
#include "kv4_format.cuh"

namespace bq {

namespace {

__device__ int g_kv4_append_device_status = 0;

constexpr int NR_THREADS = 128;

struct NormRopeParams {
    NormRopeDesc g;
    uint8_t axis[128];  // of each rotation pair
};

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ void unpack4(uint2 raw, float* x) {
    const __nv_bfloat162 lo = *reinterpret_cast<const __nv_bfloat162*>(&raw.x);
    const __nv_bfloat162 hi = *reinterpret_cast<const __nv_bfloat162*>(&raw.y);
    x[0] = __low2float(lo);
    x[1] = __high2float(lo);
    x[2] = __low2float(hi);
    x[3] = __high2float(hi);
}
__device__ __forceinline__ uint2 pack4(const float* x) {
    __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
    return make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
}

// Code of x in a group of minimum m and scale s (both as the cache holds them).
__device__ __forceinline__ uint32_t code_of(float x, float m, float s) {
    if (!(s > 0.0f)) return 0u;  // one value only (or no number: the scale then says so)
    return static_cast<uint32_t>(fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x, m), s)), 0.0f), 15.0f));
}

enum : int { HEAD_Q = 0, HEAD_K = 1, HEAD_V = 2, HEAD_NONE = 3 };

template <int D, int IT>
__global__ void __launch_bounds__(NR_THREADS) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
    constexpr int LPH = D / 8;     // lanes of a head
    constexpr int HPW = 32 / LPH;  // heads of a warp
    constexpr int G = D / KV4_GROUP;
    const NormRopeDesc& g = p.g;
    const int lane = threadIdx.x & 31;
    const int sub = lane / LPH, l = lane % LPH;
    const int heads = g.heads_q + g.heads_kv * (g.to_cache ? 2 : 1);
    const int jobs = (heads + HPW * IT - 1) / (HPW * IT);  // of one token
    const int64_t warp = static_cast<int64_t>(blockIdx.x) * (NR_THREADS / 32) + (threadIdx.x >> 5);
    const int64_t token = warp / jobs;
    if (token >= g.tokens) return;
    const int first = static_cast<int>(warp % jobs) * HPW * IT + sub;

    // channels of this lane: rotation lanes hold 4 pairs, the others 8 channels in a row; values hold channels d and d + 8
    const int rot_lanes = g.rot_dim / 8;
    const bool turns = l < rot_lanes;
    const int qk0 = (turns && !g.interleaved) ? 4 * l : 8 * l;
    const int qk1 = (turns && !g.interleaved) ? g.rot_dim / 2 + 4 * l : 8 * l + 4;
    const int v0 = 16 * (l >> 1) + 4 * (l & 1);

    // all loads first: IT heads in flight per lane
    uint2 raw[IT][2];
    int kind[IT], head[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        int h = first + i * HPW;
        kind[i] = h >= heads ? HEAD_NONE : h < g.heads_q ? HEAD_Q : h < g.heads_q + g.heads_kv ? HEAD_K : HEAD_V;
        h -= kind[i] == HEAD_Q ? 0 : kind[i] == HEAD_K ? g.heads_q : g.heads_q + g.heads_kv;
        head[i] = h;
        raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
        if (kind[i] != HEAD_NONE) {
            const __nv_bfloat16* x = kind[i] == HEAD_Q   ? static_cast<const __nv_bfloat16*>(g.q) + token * g.ldq
                                     : kind[i] == HEAD_K ? static_cast<const __nv_bfloat16*>(g.k) + token * g.ldk
                                                         : static_cast<const __nv_bfloat16*>(g.v) + token * g.ldv;
            x += static_cast<int64_t>(h) * D;
            raw[i][0] = *reinterpret_cast<const uint2*>(x + (kind[i] == HEAD_V ? v0 : qk0));
            raw[i][1] = *reinterpret_cast<const uint2*>(x + (kind[i] == HEAD_V ? v0 + 8 : qk1));
        }
    }
    float c[4], s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = 1.0f, s[e] = 0.0f;
    if (turns) {
        const int half = g.rot_dim / 2;
        if (g.axes == 1) {
            int pos = g.positions[token];
            if (pos < 0 || pos >= g.max_pos) {
                atomicCAS(&g_kv4_append_device_status, 0, 401);
                pos = pos < 0 ? 0 : g.max_pos - 1;
            }
            const float* row = g.cos_sin + static_cast<int64_t>(pos) * g.rot_dim + 4 * l;
            const float4 cv = __ldg(reinterpret_cast<const float4*>(row));
            const float4 sv = __ldg(reinterpret_cast<const float4*>(row + half));
            c[0] = cv.x, c[1] = cv.y, c[2] = cv.z, c[3] = cv.w;
            s[0] = sv.x, s[1] = sv.y, s[2] = sv.z, s[3] = sv.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                int pos = g.positions[p.axis[4 * l + e] * g.pos_stride + token];
                if (pos < 0 || pos >= g.max_pos) {
                    atomicCAS(&g_kv4_append_device_status, 0, 401);
                    pos = pos < 0 ? 0 : g.max_pos - 1;
                }
                const float* row = g.cos_sin + static_cast<int64_t>(pos) * g.rot_dim + 4 * l + e;
                c[e] = __ldg(row);
                s[e] = __ldg(row + half);
            }
        }
    }
    // where the cache takes this token
    uint8_t* tile = nullptr;
    int at = 0;
    int64_t head_stride = 0;
    if (g.to_cache) {
        const int64_t slot = g.slots[token];
        if (slot >= 0) {
            const int64_t page = slot / g.cache.page_size;
            const int off = static_cast<int>(slot - page * g.cache.page_size);
            head_stride = static_cast<int64_t>(g.cache.page_size / KV4_TILE) * kv4_tile_bytes(D);
            if (page < g.cache.num_pages) {
                tile = g.cache.base + page * g.cache.page_stride + (off / KV4_TILE) * kv4_tile_bytes(D);
                at = off % KV4_TILE;
            } else {
                atomicCAS(&g_kv4_append_device_status, 0, 402);
            }
        }
    }

#pragma unroll
    for (int i = 0; i < IT; ++i) {
        float x[8];
        unpack4(raw[i][0], x);
        unpack4(raw[i][1], x + 4);
        const float* w = kind[i] == HEAD_Q ? g.q_weight : kind[i] == HEAD_K ? g.k_weight : nullptr;
        double ss = 0.0;
        if (g.q_weight != nullptr || g.k_weight != nullptr) {
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fma(static_cast<double>(x[e]), static_cast<double>(x[e]), ss);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
        if (w != nullptr) {
            const float mean = static_cast<float>(ss * (1.0 / D));
            const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, g.eps)));
            const float4 w0 = __ldg(reinterpret_cast<const float4*>(w + qk0)), w1 = __ldg(reinterpret_cast<const float4*>(w + qk1));
            const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], r), ww[e]);
        }
        if (turns && kind[i] <= HEAD_K) {
            if (g.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = x[2 * e], b = x[2 * e + 1];
                    x[2 * e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
                    x[2 * e + 1] = __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = x[e], b = x[4 + e];
                    x[e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
                    x[4 + e] = __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
                }
            }
        }
        const uint2 o0 = pack4(x), o1 = pack4(x + 4);
        const bool cached = g.to_cache && (kind[i] == HEAD_K || kind[i] == HEAD_V);
        if (kind[i] == HEAD_Q || (kind[i] == HEAD_K && !g.to_cache)) {
            __nv_bfloat16* out = kind[i] == HEAD_Q ? static_cast<__nv_bfloat16*>(g.q_out) + token * g.ldqo
                                                   : static_cast<__nv_bfloat16*>(g.k_out) + token * g.ldko;
            out += static_cast<int64_t>(head[i]) * D;
            *reinterpret_cast<uint2*>(out + qk0) = o0;
            *reinterpret_cast<uint2*>(out + qk1) = o1;
        }
        if (!__any_sync(0xffffffffu, cached && tile != nullptr)) continue;
        // the groups' extrema over the bf16 values, then codes; all lanes of the warp take part in the exchange
        unpack4(o0, x);
        unpack4(o1, x + 4);
        const int d0 = kind[i] == HEAD_V ? v0 : qk0, d1 = kind[i] == HEAD_V ? v0 + 8 : qk1;
        float lo0 = min_nan(min_nan(x[0], x[1]), min_nan(x[2], x[3])), hi0 = max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3]));
        float lo1 = min_nan(min_nan(x[4], x[5]), min_nan(x[6], x[7])), hi1 = max_nan(max_nan(x[4], x[5]), max_nan(x[6], x[7]));
        float sc[G], mn[G];
#pragma unroll
        for (int q = 0; q < G; ++q) {
            const bool in0 = (d0 >> 6) == q, in1 = (d1 >> 6) == q;
            float lo = min_nan(in0 ? lo0 : INFINITY, in1 ? lo1 : INFINITY), hi = max_nan(in0 ? hi0 : -INFINITY, in1 ? hi1 : -INFINITY);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) {
                lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            sc[q] = __half2float(__float2half_rn(min_nan(__fdiv_rn(__fsub_rn(hi, lo), 15.0f), KV4_F16_MAX)));
            mn[q] = __fadd_rn(__half2float(__float2half_rn(max_nan(min_nan(lo, KV4_F16_MAX), -KV4_F16_MAX))), 0.0f);  // no -0: one form of a zero
        }
        if (!cached || tile == nullptr) continue;
        uint8_t* to = tile + head[i] * head_stride;
        float s0 = sc[0], m0 = mn[0], s1 = sc[0], m1 = mn[0];
#pragma unroll
        for (int q = 1; q < G; ++q) {
            if ((d0 >> 6) == q) s0 = sc[q], m0 = mn[q];
            if ((d1 >> 6) == q) s1 = sc[q], m1 = mn[q];
        }
        uint32_t code[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) code[e] = code_of(x[e], m0, s0), code[4 + e] = code_of(x[4 + e], m1, s1);
        if (kind[i] == HEAD_K) {
            *reinterpret_cast<uint16_t*>(to + kv4_key_byte<D>(at, d0)) =
                static_cast<uint16_t>(code[0] | (code[1] << 4) | (code[2] << 8) | (code[3] << 12));
            *reinterpret_cast<uint16_t*>(to + kv4_key_byte<D>(at, d1)) =
                static_cast<uint16_t>(code[4] | (code[5] << 4) | (code[6] << 8) | (code[7] << 12));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) to[kv4_value_byte<D>(at, v0 + e)] = static_cast<uint8_t>(code[e] | (code[4 + e] << 4));
        }
#pragma unroll
        for (int q = 0; q < G; ++q) {
            if (l == q) {
                const __half2 pair = __floats2half2_rn(sc[q], mn[q]);
                *reinterpret_cast<__half2*>(to + kv4_pair_offset(D, kind[i] == HEAD_V) + (at * G + q) * 4) = pair;
            }
        }
    }
}

template <int D>
int32_t launch_norm_rope_d(const NormRopeParams& p, cudaStream_t stream) {
    constexpr int HPW = 256 / D;
    const int heads = p.g.heads_q + p.g.heads_kv * (p.g.to_cache ? 2 : 1);
    auto go = [&](auto kern, int it) {
        const int64_t jobs = (heads + HPW * it - 1) / (HPW * it);
        const int64_t blocks = (jobs * p.g.tokens + NR_THREADS / 32 - 1) / (NR_THREADS / 32);
        if (blocks > 0x7fffffff) return static_cast<int32_t>(BQ_STATUS_UNSUPPORTED);
        kern<<<static_cast<unsigned>(blocks), NR_THREADS, 0, stream>>>(p);
        return static_cast<int32_t>(cudaPeekAtLastError() == cudaSuccess ? BQ_STATUS_OK : BQ_STATUS_LAUNCH_FAILURE);
    };
    // few tokens: one head per lane group, as many warps as there are; many: four, for bytes in flight and one look at the angles
    if (static_cast<int64_t>(heads) * p.g.tokens < 16384) return go(norm_rope_kernel<D, 1>, 1);
    return go(norm_rope_kernel<D, 4>, 4);
}

// One lane of the reader holds 8 channels of one token and head: keys 8 in a row (one word), values r = 0..7 of one nibble
// column (8 bytes, which the neighbouring lane reads as well).
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4ReadDesc g) {
    constexpr int LPH = D / 8;
    constexpr int G = D / KV4_GROUP;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int l = static_cast<int>(id % LPH);
    const int64_t row = id / LPH;
    const int h = static_cast<int>(row % g.cache.heads_kv);
    const int64_t token = row / g.cache.heads_kv;
    if (token >= g.tokens) return;
    const int64_t slot = g.slots[token];
    if (slot < 0) return;
    const int64_t page = slot / g.cache.page_size;
    if (page >= g.cache.num_pages) {
        atomicCAS(&g_kv4_append_device_status, 0, 402);
        return;
    }
    const int off = static_cast<int>(slot - page * g.cache.page_size), t = off % KV4_TILE;
    const uint8_t* tile = g.cache.base + page * g.cache.page_stride +
                          (static_cast<int64_t>(h) * (g.cache.page_size / KV4_TILE) + off / KV4_TILE) * kv4_tile_bytes(D);
    const int d = 8 * l;
    auto pair_of = [&](int values) {
        return __half22float2(*reinterpret_cast<const __half2*>(tile + kv4_pair_offset(D, values) + (t * G + (d >> 6)) * 4));
    };
    auto store = [&](void* base, int64_t ld, const float* x) {
        const uint2 a = pack4(x), b = pack4(x + 4);
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + token * ld + static_cast<int64_t>(h) * D + d) =
            make_uint4(a.x, a.y, b.x, b.y);
    };
    float x[8];
    {
        const float2 sm = pair_of(0);
        const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + kv4_key_byte<D>(t, d));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(__fmul_rn(sm.x, static_cast<float>((word >> (4 * e)) & 15u)), sm.y);
        store(g.k, g.ldk, x);
    }
    {
        const float2 sm = pair_of(1);
        const int shift = (d & 8) ? 4 : 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t byte = tile[kv4_value_byte<D>(t, (d & ~15) + e)];
            x[e] = __fadd_rn(__fmul_rn(sm.x, static_cast<float>((byte >> shift) & 15u)), sm.y);
        }
        store(g.v, g.ldv, x);
    }
}

}  // namespace

int32_t launch_qk_norm_rope(const NormRopeDesc& g, cudaStream_t stream) {
    NormRopeParams p;
    p.g = g;
    for (int i = 0; i < 128; ++i) p.axis[i] = (g.axis_of_pair != nullptr && i < g.rot_dim / 2) ? g.axis_of_pair[i] : 0;
    p.g.axis_of_pair = nullptr;
    switch (g.head_dim) {
        case 64: return launch_norm_rope_d<64>(p, stream);
        case 128: return launch_norm_rope_d<128>(p, stream);
        case 256: return launch_norm_rope_d<256>(p, stream);
        default: return BQ_STATUS_UNSUPPORTED;
    }
}

int32_t launch_kv4_read(const Kv4ReadDesc& g, cudaStream_t stream) {
    const int64_t threads = static_cast<int64_t>(g.tokens) * g.cache.heads_kv * (g.cache.head_dim / 8);
    const int64_t blocks = (threads + 255) / 256;
    if (blocks > 0x7fffffff) return BQ_STATUS_UNSUPPORTED;
    switch (g.cache.head_dim) {
        case 64: kv4_read_kernel<64><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(g); break;
        case 128: kv4_read_kernel<128><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(g); break;
        case 256: kv4_read_kernel<256><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(g); break;
        default: return BQ_STATUS_UNSUPPORTED;
    }
    return cudaPeekAtLastError() == cudaSuccess ? BQ_STATUS_OK : BQ_STATUS_LAUNCH_FAILURE;
}

int32_t read_and_clear_kv4_append_device_status() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_kv4_append_device_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) {
        int zero = 0;
        (void)cudaMemcpyToSymbol(g_kv4_append_device_status, &zero, sizeof(int));
    }
    return v;
}

}  // namespace bq
