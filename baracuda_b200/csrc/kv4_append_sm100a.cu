// Norms of queries and keys per head, the rotation by position, and the 4-bit cache's writer and reader.
//   y = x * (1 / sqrt(mean(x^2) + eps)) * weight                    (per head; skipped without a weight)
//   (a, b) -> (a * cos - b * sin, b * cos + a * sin)                (channel pairs; angle by the position on the pair's axis)
//   out = bf16(...)                                                 (one rounding, queries and dense keys)
//   s = f16((max - min) / 15), m = f16(min), c = clamp(rint((x - m) / s), 0, 15)    (per 64 channels of the bf16 keys and values)
// Every step is one IEEE rounding in f32, in this order, except the mean square: it is summed as pairs of f32 numbers (about 44
// bits) and rounded once, so its bits do not depend on the order of the sum and a key next to the border of two codes gets the
// same code from this kernel, from the two-call sequence and from any other evaluation.
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

constexpr int NR_THREADS = 256;

struct NormRopeParams {
    NormRopeDesc g;
    int jobs_q, jobs_kv;  // warps of one token: its queries, then its keys, then (to the cache) its values
    uint8_t axis[128];    // of each rotation pair
};

// Two f32 numbers in one register pair; each operation rounds each of them once.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 both(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 each(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// The sum of two rounded products: scalar additions, since the assembler joins a packed product and a packed sum into one
// operation with one rounding.
__device__ __forceinline__ f32x2 add_products(f32x2 a, f32x2 b) {
    const float2 x = each(a), y = each(b);
    return both(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
}
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) { return fma2(b, 0xbf800000bf800000ull, a); }
// a + b = sum + err exactly (Knuth's two-sum); `low` collects the errors.
__device__ __forceinline__ f32x2 two_sum2(f32x2 a, f32x2 b, f32x2& low) {
    const f32x2 s = add2(a, b), t = sub2(s, a);
    low = add2(low, add2(sub2(a, sub2(s, t)), sub2(b, t)));
    return s;
}
__device__ __forceinline__ float two_sum(float a, float b, float& low) {
    const float s = __fadd_rn(a, b), t = __fsub_rn(s, a);
    low = __fadd_rn(low, __fadd_rn(__fsub_rn(a, __fsub_rn(s, t)), __fsub_rn(b, t)));
    return s;
}

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
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// bf16 pair -> f32 pair and back
__device__ __forceinline__ f32x2 unpack2(uint32_t raw) { return both(__uint_as_float(raw << 16), __uint_as_float(raw & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack2(f32x2 v) {
    const float2 f = each(v);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint2 pack4(const float* x) {
    return make_uint2(pack2(both(x[0], x[1])), pack2(both(x[2], x[3])));
}

// Codes of a quad of bf16 channels, one byte each: c = clamp(rint((x - m) / s), 0, 15), the quotient rounded once.
// For scales and minima that were not cut (`plain`) the quotient comes from the reciprocal: with q near (x - m) / s the
// remainder r = (x - m) - q s is exact, and q + r / s, off by less than 2^-46 of itself before its one rounding, rounds as the
// quotient does: s has 11 significant bits, so a quotient of 24 bits by s is at least 2^-36 away from where the rounding changes.
__device__ __forceinline__ uint32_t codes4(uint2 x, float m, float s, float inv, bool plain) {
    const f32x2 a = sub2(unpack2(x.x), both(m, m)), b = sub2(unpack2(x.y), both(m, m));
    f32x2 qa, qb;
    if (plain) {
        const f32x2 i2 = both(inv, inv), n2 = both(-s, -s);
        qa = mul2(a, i2), qb = mul2(b, i2);
        qa = fma2(fma2(qa, n2, a), i2, qa);
        qb = fma2(fma2(qb, n2, b), i2, qb);
    } else {
        const float2 fa = each(a), fb = each(b);
        const bool none = !(s > 0.0f);  // one value only, or no number (the scale then says so)
        qa = both(none ? 0.0f : __fdiv_rn(fa.x, s), none ? 0.0f : __fdiv_rn(fa.y, s));
        qb = both(none ? 0.0f : __fdiv_rn(fb.x, s), none ? 0.0f : __fdiv_rn(fb.y, s));
    }
    const float2 fa = each(qa), fb = each(qb);
    // 1.5 * 2^23 + q: the integer nearest to q, ties to even, in the low bits
    const f32x2 magic = both(12582912.0f, 12582912.0f);
    const float2 ca = each(add2(both(fminf(fmaxf(fa.x, 0.0f), 15.0f), fminf(fmaxf(fa.y, 0.0f), 15.0f)), magic));
    const float2 cb = each(add2(both(fminf(fmaxf(fb.x, 0.0f), 15.0f), fminf(fmaxf(fb.y, 0.0f), 15.0f)), magic));
    const uint32_t lo = __byte_perm(__float_as_uint(ca.x), __float_as_uint(ca.y), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(cb.x), __float_as_uint(cb.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}

enum : int { HEAD_Q = 0, HEAD_K = 1, HEAD_V = 2 };

// 1 / rms of IT heads per lane group from the lanes' squares.  The 8 squares of a lane are exact (16 bits each); they are added
// with two-sums, so that sum and error together hold about 44 bits whatever the order.  With IT = 4 the lanes trade heads on
// the way: after two exchanges each lane goes on with one head, and one division and square root serve four.
template <int LPH, int IT>
__device__ __forceinline__ void inverse_rms(const uint2 (&raw)[IT][2], float eps, int l, float (&r)[IT]) {
    float s[IT], e[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const f32x2 a = unpack2(raw[i][0].x), b = unpack2(raw[i][0].y), c = unpack2(raw[i][1].x), d = unpack2(raw[i][1].y);
        f32x2 low = 0ull;
        const f32x2 ab = two_sum2(mul2(a, a), mul2(b, b), low), cd = two_sum2(mul2(c, c), mul2(d, d), low);
        const float2 t = each(two_sum2(ab, cd, low)), lo = each(low);
        e[i] = __fadd_rn(lo.x, lo.y);
        s[i] = two_sum(t.x, t.y, e[i]);
    }
    float sum = s[0], err = e[0];
    int o = LPH / 2;
    if constexpr (IT == 4) {
        const bool up = (l & o) != 0;  // keeps heads 2 and 3
        f32x2 err2 = both(up ? e[2] : e[0], up ? e[3] : e[1]);
        const f32x2 mine = both(up ? s[2] : s[0], up ? s[3] : s[1]);
        const f32x2 theirs = both(__shfl_xor_sync(0xffffffffu, up ? s[0] : s[2], o), __shfl_xor_sync(0xffffffffu, up ? s[1] : s[3], o));
        err2 = add2(err2, both(__shfl_xor_sync(0xffffffffu, up ? e[0] : e[2], o), __shfl_xor_sync(0xffffffffu, up ? e[1] : e[3], o)));
        const float2 two = each(two_sum2(mine, theirs, err2)), terr = each(err2);
        o >>= 1;
        const bool odd = (l & o) != 0;  // keeps the second of its two
        err = __fadd_rn(odd ? terr.y : terr.x, __shfl_xor_sync(0xffffffffu, odd ? terr.x : terr.y, o));
        sum = two_sum(odd ? two.y : two.x, __shfl_xor_sync(0xffffffffu, odd ? two.x : two.y, o), err);
        o >>= 1;
    }
#pragma unroll
    for (int x = IT == 4 ? LPH / 8 : LPH / 2; x > 0; x >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, sum, x), other_err = __shfl_xor_sync(0xffffffffu, err, x);
        err = __fadd_rn(err, other_err);
        sum = two_sum(sum, other, err);
    }
    const float mean = __fadd_rn(sum, err) * (1.0f / (8 * LPH));
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, eps)));
    if constexpr (IT == 4) {
#pragma unroll
        for (int i = 0; i < IT; ++i) r[i] = __shfl_sync(0xffffffffu, inv, (i >> 1) * (LPH / 2) + (i & 1) * (LPH / 4), LPH);
    } else {
        r[0] = inv;
    }
}

template <int D, int IT>
__global__ void __launch_bounds__(NR_THREADS) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
    constexpr int LPH = D / 8;     // lanes of a head
    constexpr int HPW = 32 / LPH;  // heads of a warp
    constexpr int G = D / KV4_GROUP;
    const NormRopeDesc& g = p.g;
    const int lane = threadIdx.x & 31;
    const int sub = lane / LPH, l = lane % LPH;
    const int jobs = p.jobs_q + p.jobs_kv * (g.to_cache ? 2 : 1);
    const int64_t warp = static_cast<int64_t>(blockIdx.x) * (NR_THREADS / 32) + (threadIdx.x >> 5);
    const int64_t token = warp / jobs;
    if (token >= g.tokens) return;
    int job = static_cast<int>(warp - token * jobs);
    const int kind = job < p.jobs_q ? HEAD_Q : job < p.jobs_q + p.jobs_kv ? HEAD_K : HEAD_V;  // of the whole warp
    job -= kind == HEAD_Q ? 0 : kind == HEAD_K ? p.jobs_q : p.jobs_q + p.jobs_kv;
    const int first = job * HPW * IT + sub;
    const int heads = kind == HEAD_Q ? g.heads_q : g.heads_kv;

    // channels of this lane, two quads: rotation lanes hold 4 pairs, the others 8 channels in a row; values hold d and d + 8
    const bool turns = kind != HEAD_V && l < g.rot_dim / 8;
    int d0 = 8 * l, d1 = 8 * l + 4;
    if (turns && !g.interleaved) d0 = 4 * l, d1 = g.rot_dim / 2 + 4 * l;
    if (kind == HEAD_V) d0 = 16 * (l >> 1) + 4 * (l & 1), d1 = d0 + 8;

    // all loads first: IT heads in flight per lane
    const __nv_bfloat16* from = kind == HEAD_Q   ? static_cast<const __nv_bfloat16*>(g.q) + token * g.ldq
                                : kind == HEAD_K ? static_cast<const __nv_bfloat16*>(g.k) + token * g.ldk
                                                 : static_cast<const __nv_bfloat16*>(g.v) + token * g.ldv;
    uint2 raw[IT][2];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int h = first + i * HPW;
        raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
        if (h < heads) {
            raw[i][0] = *reinterpret_cast<const uint2*>(from + static_cast<int64_t>(h) * D + d0);
            raw[i][1] = *reinterpret_cast<const uint2*>(from + static_cast<int64_t>(h) * D + d1);
        }
    }
    if (kind != HEAD_V) {
        f32x2 c[2], s[2], ns[2];  // of this lane's 4 pairs
        c[0] = c[1] = both(1.0f, 1.0f);
        s[0] = s[1] = ns[0] = ns[1] = 0ull;
        if (turns) {
            const int half = g.rot_dim / 2;
            float4 cv, sv;
            if (g.axes == 1) {
                int pos = g.positions[token];
                if (pos < 0 || pos >= g.max_pos) {
                    atomicCAS(&g_kv4_append_device_status, 0, 401);
                    pos = pos < 0 ? 0 : g.max_pos - 1;
                }
                const float* row = g.cos_sin + static_cast<int64_t>(pos) * g.rot_dim + 4 * l;
                cv = __ldg(reinterpret_cast<const float4*>(row));
                sv = __ldg(reinterpret_cast<const float4*>(row + half));
            } else {
                float t[2][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    int pos = g.positions[p.axis[4 * l + e] * g.pos_stride + token];
                    if (pos < 0 || pos >= g.max_pos) {
                        atomicCAS(&g_kv4_append_device_status, 0, 401);
                        pos = pos < 0 ? 0 : g.max_pos - 1;
                    }
                    const float* row = g.cos_sin + static_cast<int64_t>(pos) * g.rot_dim + 4 * l + e;
                    t[0][e] = __ldg(row);
                    t[1][e] = __ldg(row + half);
                }
                cv = make_float4(t[0][0], t[0][1], t[0][2], t[0][3]);
                sv = make_float4(t[1][0], t[1][1], t[1][2], t[1][3]);
            }
            c[0] = both(cv.x, cv.y), c[1] = both(cv.z, cv.w);
            s[0] = both(sv.x, sv.y), s[1] = both(sv.z, sv.w);
            ns[0] = both(-sv.x, -sv.y), ns[1] = both(-sv.z, -sv.w);
        }
        const float* weight = kind == HEAD_Q ? g.q_weight : g.k_weight;
        float r[IT];
        f32x2 w[4];
        if (weight != nullptr) {
            const float4 w0 = __ldg(reinterpret_cast<const float4*>(weight + d0)), w1 = __ldg(reinterpret_cast<const float4*>(weight + d1));
            w[0] = both(w0.x, w0.y), w[1] = both(w0.z, w0.w), w[2] = both(w1.x, w1.y), w[3] = both(w1.z, w1.w);
            inverse_rms<LPH, IT>(raw, g.eps, l, r);
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            f32x2 x[4] = {unpack2(raw[i][0].x), unpack2(raw[i][0].y), unpack2(raw[i][1].x), unpack2(raw[i][1].y)};
            if (weight != nullptr) {
                const f32x2 r2 = both(r[i], r[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = mul2(mul2(x[e], r2), w[e]);
            }
            if (turns) {
                if (g.interleaved) {  // neighbours: gather the pairs' first and second channels, and back
                    const float2 x0 = each(x[0]), x1 = each(x[1]), x2 = each(x[2]), x3 = each(x[3]);
                    const f32x2 a0 = both(x0.x, x1.x), b0 = both(x0.y, x1.y), a1 = both(x2.x, x3.x), b1 = both(x2.y, x3.y);
                    const float2 p0 = each(add_products(mul2(a0, c[0]), mul2(b0, ns[0]))), q0 = each(add_products(mul2(b0, c[0]), mul2(a0, s[0])));
                    const float2 p1 = each(add_products(mul2(a1, c[1]), mul2(b1, ns[1]))), q1 = each(add_products(mul2(b1, c[1]), mul2(a1, s[1])));
                    x[0] = both(p0.x, q0.x), x[1] = both(p0.y, q0.y), x[2] = both(p1.x, q1.x), x[3] = both(p1.y, q1.y);
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const f32x2 a = x[e], b = x[2 + e];
                        x[e] = add_products(mul2(a, c[e]), mul2(b, ns[e]));
                        x[2 + e] = add_products(mul2(b, c[e]), mul2(a, s[e]));
                    }
                }
            }
            raw[i][0] = make_uint2(pack2(x[0]), pack2(x[1]));
            raw[i][1] = make_uint2(pack2(x[2]), pack2(x[3]));
        }
        if (kind == HEAD_Q || !g.to_cache) {
            __nv_bfloat16* out = kind == HEAD_Q ? static_cast<__nv_bfloat16*>(g.q_out) + token * g.ldqo
                                                : static_cast<__nv_bfloat16*>(g.k_out) + token * g.ldko;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int h = first + i * HPW;
                if (h < heads) {
                    *reinterpret_cast<uint2*>(out + static_cast<int64_t>(h) * D + d0) = raw[i][0];
                    *reinterpret_cast<uint2*>(out + static_cast<int64_t>(h) * D + d1) = raw[i][1];
                }
            }
            return;
        }
    }

    // keys and values into the cache
    const int64_t slot = g.slots[token];
    if (slot < 0) return;
    const int64_t page = slot / g.cache.page_size;
    const int off = static_cast<int>(slot - page * g.cache.page_size);
    if (page >= g.cache.num_pages) {
        atomicCAS(&g_kv4_append_device_status, 0, 402);
        return;
    }
    uint8_t* tile = g.cache.base + page * g.cache.page_stride + (off / KV4_TILE) * kv4_tile_bytes(D);
    const int64_t head_stride = static_cast<int64_t>(g.cache.page_size / KV4_TILE) * kv4_tile_bytes(D);
    const int at = off % KV4_TILE;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int h = first + i * HPW;
        if (job * HPW * IT + i * HPW >= heads) break;  // of the whole warp
        // the groups' extrema over the bf16 values as (max, -min), one exchange for both
        uint32_t ext[G];
        const uint32_t hi0 = max_bf16x2(raw[i][0].x, raw[i][0].y), hi1 = max_bf16x2(raw[i][1].x, raw[i][1].y);
        const uint32_t lo0 = max_bf16x2(raw[i][0].x ^ 0x80008000u, raw[i][0].y ^ 0x80008000u);
        const uint32_t lo1 = max_bf16x2(raw[i][1].x ^ 0x80008000u, raw[i][1].y ^ 0x80008000u);
        const uint32_t e0 = max_bf16x2(__byte_perm(hi0, lo0, 0x5410), __byte_perm(hi0, lo0, 0x7632));
        const uint32_t e1 = max_bf16x2(__byte_perm(hi1, lo1, 0x5410), __byte_perm(hi1, lo1, 0x7632));
        float sc[G], mn[G];
#pragma unroll
        for (int q = 0; q < G; ++q) {
            ext[q] = max_bf16x2((d0 >> 6) == q ? e0 : 0xff80ff80u, (d1 >> 6) == q ? e1 : 0xff80ff80u);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ext[q] = max_bf16x2(ext[q], __shfl_xor_sync(0xffffffffu, ext[q], o));
            const float hi = __uint_as_float(ext[q] << 16), lo = -__uint_as_float(ext[q] & 0xffff0000u);
            sc[q] = __half2float(__float2half_rn(min_nan(__fdiv_rn(__fsub_rn(hi, lo), 15.0f), KV4_F16_MAX)));
            mn[q] = __fadd_rn(__half2float(__float2half_rn(max_nan(min_nan(lo, KV4_F16_MAX), -KV4_F16_MAX))), 0.0f);  // no -0: one form of a zero
        }
        float s0 = sc[0], m0 = mn[0], s1 = sc[0], m1 = mn[0];
#pragma unroll
        for (int q = 1; q < G; ++q) {
            if ((d0 >> 6) == q) s0 = sc[q], m0 = mn[q];
            if ((d1 >> 6) == q) s1 = sc[q], m1 = mn[q];
        }
        const bool plain0 = s0 > 0.0f && s0 < KV4_F16_MAX && fabsf(m0) < KV4_F16_MAX, plain1 = s1 > 0.0f && s1 < KV4_F16_MAX && fabsf(m1) < KV4_F16_MAX;
        const bool plain = __all_sync(0xffffffffu, (plain0 && plain1) || h >= heads);
        const uint32_t k0 = codes4(raw[i][0], m0, s0, __fdiv_rn(1.0f, s0), plain), k1 = codes4(raw[i][1], m1, s1, __fdiv_rn(1.0f, s1), plain);
        if (h >= heads) continue;
        uint8_t* to = tile + h * head_stride;
        if (kind == HEAD_K) {  // bytes 0, 1 and 2, 3 of each quad share a byte
            const uint32_t b0 = k0 | (k0 >> 4), b1 = k1 | (k1 >> 4);
            *reinterpret_cast<uint16_t*>(to + kv4_key_byte<D>(at, d0)) = static_cast<uint16_t>(__byte_perm(b0, 0u, 0x4420));
            *reinterpret_cast<uint16_t*>(to + kv4_key_byte<D>(at, d1)) = static_cast<uint16_t>(__byte_perm(b1, 0u, 0x4420));
        } else {  // channels d and d + 8 share a byte
            const uint32_t bytes = k0 | (k1 << 4);
            uint8_t* v = to + kv4_value_byte<D>(at, d0);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[64 * e] = static_cast<uint8_t>(bytes >> (8 * e));
        }
#pragma unroll
        for (int q = 0; q < G; ++q) {
            if (l == q) {
                const __half2 pair = __floats2half2_rn(sc[q], mn[q]);
                *reinterpret_cast<__half2*>(to + kv4_pair_offset(D, kind == HEAD_V) + (at * G + q) * 4) = pair;
            }
        }
    }
}

template <int D>
int32_t launch_norm_rope_d(NormRopeParams& p, cudaStream_t stream) {
    constexpr int HPW = 256 / D;
    auto go = [&](auto kern, int it) {
        p.jobs_q = (p.g.heads_q + HPW * it - 1) / (HPW * it);
        p.jobs_kv = (p.g.heads_kv + HPW * it - 1) / (HPW * it);
        const int64_t jobs = p.jobs_q + p.jobs_kv * (p.g.to_cache ? 2 : 1);
        const int64_t blocks = (jobs * p.g.tokens + NR_THREADS / 32 - 1) / (NR_THREADS / 32);
        if (blocks > 0x7fffffff) return static_cast<int32_t>(BQ_STATUS_UNSUPPORTED);
        kern<<<static_cast<unsigned>(blocks), NR_THREADS, 0, stream>>>(p);
        return static_cast<int32_t>(cudaPeekAtLastError() == cudaSuccess ? BQ_STATUS_OK : BQ_STATUS_LAUNCH_FAILURE);
    };
    // few tokens: one head per lane group, as many warps as there are; many: four, for bytes in flight and one look at the angles
    const int64_t heads = p.g.heads_q + static_cast<int64_t>(p.g.heads_kv) * (p.g.to_cache ? 2 : 1);
    if (heads * p.g.tokens < 16384) return go(norm_rope_kernel<D, 1>, 1);
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
    NormRopeParams p = {};
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
