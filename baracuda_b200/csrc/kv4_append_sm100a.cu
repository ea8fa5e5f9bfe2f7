// Norms of queries and keys per head, the rotation by position, and the 4-bit cache's writer and reader.
//   y = x * (1 / sqrt(mean(x^2) + eps)) * weight                    (per head; skipped without a weight)
//   (a, b) -> (a * cos - b * sin, b * cos + a * sin)                (channel pairs; angle by the position on the pair's axis)
//   out = bf16(...)                                                 (one rounding, queries and dense keys)
//   s = f16((max - min) / 15), m = f16(min), c = clamp(rint((x - m) / s), 0, 15)    (per 64 channels of the bf16 keys and values;
//   max and min cut to +-32768)
// Of keys and values every step is one IEEE rounding in f32, in this order, and the mean square of a key is summed as pairs of f32
// numbers (about 44 bits) and rounded once: its bits do not depend on the order of the sum, and a key next to the border of two
// codes gets the same code from this kernel, from the two-call sequence and from any other evaluation.  Queries meet no such border:
// their mean square is an f32 sum, its root's inverse comes at once, and the rotation's products and sums are fused.
// Bound: bytes (each element read and written once), once the instructions per head are few: a head is D / 16 lanes of 16
// channels, which contain whole rotation pairs, so nothing is exchanged between lanes but the sums and the groups' extrema; a
// warp takes twice 512 / D heads of one token, whose sums share their exchanges, division and square root.
//
// Measured (B200): 4097 tokens of 28 + 4 heads of 128, three axes, dense output: 25.8 us (2.7 TB/s; a plain copy takes 12, this
// structure without norm and rotation 15); 8191 tokens of 64 + 8 + 8 heads into the cache: 99 us, and 11 to read them back; 5 tokens:
// 2.9 us; 8191 tokens of 8 + 8 heads into the cache as they are: 26.8 us (1.6 TB/s, the values leave by single bytes).  Half of the
// issue slots are used: what is left is the chain position -> angles -> product within a warp, the ramp at both ends, and spills: the
// two-head form is held to 64 registers for four resident blocks and loads 210 to 470 bytes a thread back (88 registers, none
// spilled, for one head).  With 8 heads a warp in fragment order, sums of squares from mma.sync and a loop over blocks of heads, the
// same cases took 29.6 and 131 us: its angles and weights need twice the registers.
// Reading 65536 tokens of 8 heads: 56 us, 6.0 TB/s, of one sequence or of several that begin at the same place of a tile; of eight
// that do not: 138 us, since all but the first are read token by token.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/baracuda_kernels_q.h"
#include "kv4_format.cuh"

namespace bq {

namespace {

__device__ int g_kv4_append_device_status = 0;

constexpr int NR_THREADS = 256;
constexpr int NR_IT = 2;          // heads of a lane group where there are many tokens
constexpr int NR_MIN_BLOCKS = 4;  // resident blocks then: 115 us for 8191 tokens of 64 + 8 + 8 heads with the read-back, 122 with 3, 135 with 4 heads and 2 blocks

struct NormRopeParams {
    NormRopeDesc g;
    uint32_t jobs_q, jobs_kv, jobs;  // warps of one token: its queries, then its keys, then (to the cache) its values; all
    uint64_t axis[2][3];             // axis of each rotation pair: bit b of pair i at bit i % 64 of axis[i / 64][b]
};

// The sum of two rounded products: scalar additions, since the assembler joins a packed product and a packed sum into one
// operation with one rounding.
__device__ __forceinline__ f32x2 add_products(f32x2 a, f32x2 b) {
    const float2 x = each(a), y = each(b);
    return both(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
}
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
// For groups within the cut, of more than one value (`plain`), the quotient comes from the reciprocal: with q near (x - m) / s the
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

// The 16 channels of a lane: quads q[0], q[2] from one place on and q[1], q[3] from another.
struct Lane16 {
    uint2 q[4];
};

// A lane's sum of squares; EXACT with the part that an f32 does not hold in `err`.
template <bool EXACT>
__device__ __forceinline__ float squares(const Lane16& x, float& err) {
    if constexpr (EXACT) {  // squares of bf16 are exact
        f32x2 low = 0ull, part[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x2 a = unpack2(x.q[i].x), b = unpack2(x.q[i].y);
            part[i] = two_sum2(mul2(a, a), mul2(b, b), low);
        }
        const float2 t = each(two_sum2(two_sum2(part[0], part[1], low), two_sum2(part[2], part[3], low), low)), lo = each(low);
        err = __fadd_rn(lo.x, lo.y);
        return two_sum(t.x, t.y, err);
    } else {
        f32x2 a = 0ull, b = 0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x2 u = unpack2(x.q[i].x), v = unpack2(x.q[i].y);
            a = fma2(u, u, a);
            b = fma2(v, v, b);
        }
        const float2 t = each(add2(a, b));
        return t.x + t.y;
    }
}

// 1 / rms of IT heads per lane group, one or two.  With two the lanes trade halves first: each goes on with one head, so the other
// exchanges and the root serve both.  EXACT (keys): division and square root rounded, as the definition says; queries
// take the reciprocal root at once.
template <int LPH, int IT, bool EXACT>
__device__ __forceinline__ void inverse_rms(const Lane16 (&x)[IT], float eps, int l, float (&r)[IT]) {
    static_assert(IT == 1 || IT == 2, "heads trade one exchange");
    float s[IT], e[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) e[i] = 0.0f, s[i] = squares<EXACT>(x[i], e[i]);
    auto join = [&](float& sum, float& err, float other, float other_err) {
        if constexpr (EXACT) {
            err = __fadd_rn(err, other_err);
            sum = two_sum(sum, other, err);
        } else {
            sum += other;
        }
    };
    auto trade = [&](float v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); };
    int left = IT;
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) {
        if (left > 1) {  // keep one half of the heads
            left /= 2;
            const bool up = (l & o) != 0;
#pragma unroll
            for (int i = 0; i < left; ++i) {
                const float give = up ? s[i] : s[left + i], give_err = up ? e[i] : e[left + i];
                if (up) s[i] = s[left + i], e[i] = e[left + i];
                join(s[i], e[i], trade(give, o), EXACT ? trade(give_err, o) : 0.0f);
            }
        } else {
            join(s[0], e[0], trade(s[0], o), EXACT ? trade(e[0], o) : 0.0f);
        }
    }
    float inv;
    if constexpr (EXACT) {
        // a sum beyond f32 is infinite, and what the two-sums make of it is no number
        const float sum = __fadd_rn(s[0], s[0] < INFINITY ? e[0] : 0.0f);
        inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(sum * (1.0f / (16 * LPH)), eps)));
    } else {
        inv = rsqrtf(fmaf(s[0], 1.0f / (16 * LPH), eps));
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        r[i] = IT == 1 ? inv : __shfl_sync(0xffffffffu, inv, i * (LPH / 2), LPH);
    }
}

// Angles of 4 rotation pairs.
struct Turn {
    f32x2 c[2], s[2];
};
__device__ __forceinline__ f32x2 minus(f32x2 v) { return v ^ 0x8000000080000000ull; }

// Two quads as rotation pairs: of quad a's channels with quad b's, or of neighbours within each (4 pairs in either case).
// EXACT (keys): products and sums rounded one by one; queries join them.
template <bool EXACT>
__device__ __forceinline__ void turn_halves(f32x2 (&a)[2], f32x2 (&b)[2], const Turn& t) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const f32x2 u = a[e], v = b[e];
        if constexpr (EXACT) {
            a[e] = add_products(mul2(u, t.c[e]), minus(mul2(v, t.s[e])));
            b[e] = add_products(mul2(v, t.c[e]), mul2(u, t.s[e]));
        } else {
            a[e] = fma2(u, t.c[e], minus(mul2(v, t.s[e])));
            b[e] = fma2(v, t.c[e], mul2(u, t.s[e]));
        }
    }
}
template <bool EXACT>
__device__ __forceinline__ void turn_neighbours(f32x2 (&a)[2], f32x2 (&b)[2], const Turn& t) {
    const float2 a0 = each(a[0]), a1 = each(a[1]), b0 = each(b[0]), b1 = each(b[1]);
    f32x2 u[2] = {both(a0.x, a1.x), both(b0.x, b1.x)}, v[2] = {both(a0.y, a1.y), both(b0.y, b1.y)};
    turn_halves<EXACT>(u, v, t);
    const float2 u0 = each(u[0]), v0 = each(v[0]), u1 = each(u[1]), v1 = each(v[1]);
    a[0] = both(u0.x, v0.x), a[1] = both(u0.y, v0.y);
    b[0] = both(u1.x, v1.x), b[1] = both(u1.y, v1.y);
}

// Norm and rotation of IT heads in place.
template <int LPH, int IT, bool EXACT>
__device__ __forceinline__ void norm_and_turn(Lane16 (&x)[IT], const float* weight, const f32x2 (&w)[4][2], float eps, int l, bool interleaved,
                                              bool turns, bool turns_second, const Turn (&t)[2]) {
    float r[IT];
    if (weight != nullptr) inverse_rms<LPH, IT, EXACT>(x, eps, l, r);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        f32x2 y[4][2];
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q][0] = unpack2(x[i].q[q].x), y[q][1] = unpack2(x[i].q[q].y);
        if (weight != nullptr) {
            const f32x2 r2 = both(r[i], r[i]);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 2; ++e) y[q][e] = mul2(mul2(y[q][e], r2), w[q][e]);
        }
        if (interleaved) {  // pairs 8 l .. lie in quads 0 and 2, 8 l + 4 .. in 1 and 3
            if (turns) turn_neighbours<EXACT>(y[0], y[2], t[0]);
            if (turns_second) turn_neighbours<EXACT>(y[1], y[3], t[1]);
        } else {
            if (turns) turn_halves<EXACT>(y[0], y[1], t[0]);
            if (turns_second) turn_halves<EXACT>(y[2], y[3], t[1]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) x[i].q[q] = make_uint2(pack2(y[q][0]), pack2(y[q][1]));
    }
}

// WIDE: 16-byte accesses, no lane mixes rotated and other channels.
template <int D, int IT, bool WIDE>
__global__ void __launch_bounds__(NR_THREADS, IT == 1 ? 1 : NR_MIN_BLOCKS) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
    constexpr int LPH = D / 16;    // lanes of a head
    constexpr int HPW = 32 / LPH;  // heads of a warp at a time
    constexpr int G = D / KV4_GROUP;
    const NormRopeDesc& g = p.g;
    const int lane = threadIdx.x & 31;
    const int sub = lane / LPH, l = lane % LPH;
    const uint32_t warp = blockIdx.x * (NR_THREADS / 32) + (threadIdx.x >> 5);
    const uint32_t token = warp / p.jobs;
    if (token >= static_cast<uint32_t>(g.tokens)) return;
    uint32_t job = warp - token * p.jobs;
    const int kind = job < p.jobs_q ? HEAD_Q : job < p.jobs_q + p.jobs_kv ? HEAD_K : HEAD_V;  // of the whole warp
    job -= kind == HEAD_Q ? 0 : kind == HEAD_K ? p.jobs_q : p.jobs_q + p.jobs_kv;
    const int begin = static_cast<int>(job) * HPW * IT, first = begin + sub;
    const int heads = kind == HEAD_Q ? g.heads_q : g.heads_kv;

    // where this lane's quads lie: rotated halves hold pairs 8 l .. 8 l + 7, everything else 16 channels in a row
    const int half = g.rot_dim / 2;
    const bool turns = kind != HEAD_V && 8 * l < half, turns_second = WIDE ? turns : kind != HEAD_V && 8 * l + 4 < half;  // first, last 4 pairs
    int d[4] = {16 * l, 16 * l + 8, 16 * l + 4, 16 * l + 12};
    if (turns && !g.interleaved) {
        d[0] = 8 * l, d[1] = half + 8 * l;
        d[2] = turns_second ? d[0] + 4 : g.rot_dim, d[3] = turns_second ? d[1] + 4 : g.rot_dim + 4;
    }

    // all loads first: IT heads in flight per lane (the last head again where there is none)
    const __nv_bfloat16* from = static_cast<const __nv_bfloat16*>(kind == HEAD_Q ? g.q : kind == HEAD_K ? g.k : g.v) +
                                static_cast<int64_t>(token) * (kind == HEAD_Q ? g.ldq : kind == HEAD_K ? g.ldk : g.ldv);
    Lane16 x[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const __nv_bfloat16* at = from + min(first + i * HPW, heads - 1) * D;
        if constexpr (WIDE) {
            const uint4 a = *reinterpret_cast<const uint4*>(at + d[0]), b = *reinterpret_cast<const uint4*>(at + d[1]);
            x[i].q[0] = make_uint2(a.x, a.y), x[i].q[2] = make_uint2(a.z, a.w);
            x[i].q[1] = make_uint2(b.x, b.y), x[i].q[3] = make_uint2(b.z, b.w);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) x[i].q[q] = *reinterpret_cast<const uint2*>(at + d[q]);
        }
    }
    if (kind != HEAD_V) {
        Turn t[2] = {};
        if (turns) {
            // the axes of this lane's 8 pairs, 8 bits for each bit of the axis
            uint32_t ax[3] = {0u, 0u, 0u};
            if (g.axes > 1) {
#pragma unroll
                for (int bit = 0; bit < 3; ++bit) ax[bit] = static_cast<uint32_t>((l < 8 ? p.axis[0][bit] : p.axis[1][bit]) >> ((8 * l) & 63)) & 255u;
            }
            auto row_of = [&](int e) {
                const uint32_t axis = ((ax[0] >> e) & 1u) | (((ax[1] >> e) & 1u) << 1) | (((ax[2] >> e) & 1u) << 2);
                int pos = g.positions[axis * g.pos_stride + token];
                if (pos < 0 || pos >= g.max_pos) {
                    atomicCAS(&g_kv4_append_device_status, 0, 401);
                    pos = pos < 0 ? 0 : g.max_pos - 1;
                }
                return g.cos_sin + static_cast<int64_t>(pos) * g.rot_dim + 8 * l;
            };
            const bool same = ((ax[0] + 1u) & 254u) == 0u && ((ax[1] + 1u) & 254u) == 0u && ((ax[2] + 1u) & 254u) == 0u;  // each 0 or 255
            if (same && turns_second) {  // the rule with sections: 8 pairs in a row lie on one axis
                const float* row = row_of(0);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float4 cv = __ldg(reinterpret_cast<const float4*>(row + 4 * n)), sv = __ldg(reinterpret_cast<const float4*>(row + half + 4 * n));
                    t[n].c[0] = both(cv.x, cv.y), t[n].c[1] = both(cv.z, cv.w);
                    t[n].s[0] = both(sv.x, sv.y), t[n].s[1] = both(sv.z, sv.w);
                }
            } else {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    if (n == 1 && !turns_second) break;
                    float v[2][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float* row = row_of(4 * n + e) + 4 * n + e;
                        v[0][e] = __ldg(row);
                        v[1][e] = __ldg(row + half);
                    }
                    t[n].c[0] = both(v[0][0], v[0][1]), t[n].c[1] = both(v[0][2], v[0][3]);
                    t[n].s[0] = both(v[1][0], v[1][1]), t[n].s[1] = both(v[1][2], v[1][3]);
                }
            }
        }
        const float* weight = kind == HEAD_Q ? g.q_weight : g.k_weight;
        f32x2 w[4][2];
        if (weight != nullptr) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(weight + d[q]));
                w[q][0] = both(v.x, v.y), w[q][1] = both(v.z, v.w);
            }
        }
        if (kind == HEAD_Q) {
            norm_and_turn<LPH, IT, false>(x, weight, w, g.eps, l, g.interleaved != 0, turns, turns_second, t);
        } else {
            norm_and_turn<LPH, IT, true>(x, weight, w, g.eps, l, g.interleaved != 0, turns, turns_second, t);
        }
        if (kind == HEAD_Q || !g.to_cache) {
            __nv_bfloat16* out = kind == HEAD_Q ? static_cast<__nv_bfloat16*>(g.q_out) + static_cast<int64_t>(token) * g.ldqo
                                                : static_cast<__nv_bfloat16*>(g.k_out) + static_cast<int64_t>(token) * g.ldko;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int h = first + i * HPW;
                if (h >= heads) return;
                __nv_bfloat16* at = out + h * D;
                if constexpr (WIDE) {
                    *reinterpret_cast<uint4*>(at + d[0]) = make_uint4(x[i].q[0].x, x[i].q[0].y, x[i].q[2].x, x[i].q[2].y);
                    *reinterpret_cast<uint4*>(at + d[1]) = make_uint4(x[i].q[1].x, x[i].q[1].y, x[i].q[3].x, x[i].q[3].y);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) *reinterpret_cast<uint2*>(at + d[q]) = x[i].q[q];
                }
            }
            return;
        }
    }

    // keys and values into the cache
    const int64_t slot = g.slots[token];
    if (slot < 0) return;
    if (slot >= static_cast<int64_t>(g.cache.num_pages) * g.cache.page_size) {
        atomicCAS(&g_kv4_append_device_status, 0, 402);
        return;
    }
    int64_t page;
    if (slot >> 32 == 0) {
        page = static_cast<uint32_t>(slot) / static_cast<uint32_t>(g.cache.page_size);
    } else {
        page = slot / g.cache.page_size;
    }
    const int off = static_cast<int>(slot - page * g.cache.page_size);
    uint8_t* tile = g.cache.base + page * g.cache.page_stride + (off / KV4_TILE) * kv4_tile_bytes(D);
    const int64_t head_stride = static_cast<int64_t>(g.cache.page_size / KV4_TILE) * kv4_tile_bytes(D);
    const int at = off % KV4_TILE;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int h = first + i * HPW;
        if (begin + i * HPW >= heads) break;  // of the whole warp
        // the groups' extrema over the bf16 values as (max, -min), one exchange for both
        uint32_t ext[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t hi = max_bf16x2(x[i].q[q].x, x[i].q[q].y), lo = max_bf16x2(x[i].q[q].x ^ 0x80008000u, x[i].q[q].y ^ 0x80008000u);
            ext[q] = max_bf16x2(__byte_perm(hi, lo, 0x5410), __byte_perm(hi, lo, 0x7632));
        }
        float sc[G], mn[G], rc[G];
        bool plain = true;
#pragma unroll
        for (int n = 0; n < G; ++n) {
            uint32_t m = 0xff80ff80u;  // minus infinity
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if ((d[q] >> 6) == n) m = max_bf16x2(m, ext[q]);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) m = max_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float hi = max_nan(min_nan(__uint_as_float(m << 16), KV4_CUT), -KV4_CUT);
            const float lo = max_nan(min_nan(-__uint_as_float(m & 0xffff0000u), KV4_CUT), -KV4_CUT);
            sc[n] = __half2float(__float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f)));
            mn[n] = __fadd_rn(__half2float(__float2half_rn(lo)), 0.0f);  // no -0: one form of a zero
            rc[n] = __fdiv_rn(1.0f, sc[n]);
            plain = plain && sc[n] > 0.0f && hi < KV4_CUT && lo > -KV4_CUT;
        }
        plain = __all_sync(0xffffffffu, plain || h >= heads);
        if (h >= heads) continue;
        uint32_t code[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float s = sc[0], m = mn[0], rec = rc[0];
#pragma unroll
            for (int n = 1; n < G; ++n)
                if ((d[q] >> 6) == n) s = sc[n], m = mn[n], rec = rc[n];
            code[q] = codes4(x[i].q[q], m, s, rec, plain);
        }
        uint8_t* to = tile + h * head_stride;
        if (kind == HEAD_K) {  // neighbouring channels share a byte; bytes 0 and 2 of each word below
            uint32_t b[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) b[q] = code[q] | (code[q] >> 4);
            if constexpr (WIDE) {  // 8 channels in a row, 4 bytes
                *reinterpret_cast<uint32_t*>(to + kv4_key_byte<D>(at, d[0])) = __byte_perm(b[0], b[2], 0x6420);
                *reinterpret_cast<uint32_t*>(to + kv4_key_byte<D>(at, d[1])) = __byte_perm(b[1], b[3], 0x6420);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<uint16_t*>(to + kv4_key_byte<D>(at, d[q])) = static_cast<uint16_t>(__byte_perm(b[q], 0u, 0x4420));
            }
        } else {  // channels d and d + 8 share a byte
            uint8_t* v = to + kv4_value_byte<D>(at, d[0]);
            const uint32_t lo = code[0] | (code[1] << 4), hi = code[2] | (code[3] << 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[64 * e] = static_cast<uint8_t>(lo >> (8 * e));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[64 * (4 + e)] = static_cast<uint8_t>(hi >> (8 * e));
        }
#pragma unroll
        for (int n = 0; n < G; ++n) {
            if (l == n) {
                const __half2 pair = __floats2half2_rn(sc[n], mn[n]);
                *reinterpret_cast<__half2*>(to + kv4_pair_offset(D, kind == HEAD_V) + (at * G + n) * 4) = pair;
            }
        }
    }
}

template <int D>
int32_t launch_norm_rope_d(NormRopeParams& p, cudaStream_t stream) {
    constexpr int HPW = 512 / D;
    const NormRopeDesc& g = p.g;
    auto go = [&](auto kern, int it) {
        p.jobs_q = (g.heads_q + HPW * it - 1) / (HPW * it);
        p.jobs_kv = (g.heads_kv + HPW * it - 1) / (HPW * it);
        p.jobs = p.jobs_q + p.jobs_kv * (g.to_cache ? 2 : 1);
        const int64_t blocks = (static_cast<int64_t>(p.jobs) * g.tokens + NR_THREADS / 32 - 1) / (NR_THREADS / 32);
        if (blocks * (NR_THREADS / 32) > 0xffffffffll) return static_cast<int32_t>(BQ_STATUS_UNSUPPORTED);  // counted in 32 bits
        kern<<<static_cast<unsigned>(blocks), NR_THREADS, 0, stream>>>(p);
        return static_cast<int32_t>(cudaPeekAtLastError() == cudaSuccess ? BQ_STATUS_OK : BQ_STATUS_LAUNCH_FAILURE);
    };
    auto aligned = [](const void* ptr, int64_t ld) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && ld % 8 == 0; };
    const bool wide = g.rot_dim % 16 == 0 && aligned(g.q, g.ldq) && aligned(g.k, g.ldk) && aligned(g.q_out, g.ldqo) &&
                      (g.to_cache ? aligned(g.v, g.ldv) : aligned(g.k_out, g.ldko));
    // few tokens: one head per lane group, as many warps as there are; many: several, for bytes in flight and one look at the angles
    const int64_t heads = g.heads_q + static_cast<int64_t>(g.heads_kv) * (g.to_cache ? 2 : 1);
    if (heads * g.tokens < 16384) return wide ? go(norm_rope_kernel<D, 1, true>, 1) : go(norm_rope_kernel<D, 1, false>, 1);
    return wide ? go(norm_rope_kernel<D, NR_IT, true>, NR_IT) : go(norm_rope_kernel<D, NR_IT, false>, NR_IT);
}

// 8 codes as f32 pairs in the order of the nibbles: each code becomes the low byte of 2^23 + c, from which 2^23 is taken.
__device__ __forceinline__ void codes_f32(uint32_t even, uint32_t odd, f32x2 (&out)[4]) {
    const f32x2 back = both(-8388608.0f, -8388608.0f);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        out[e] = add2(both(__uint_as_float(__byte_perm(even, 0x4b000000u, 0x7440 + e)), __uint_as_float(__byte_perm(odd, 0x4b000000u, 0x7440 + e))), back);
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

constexpr int RD_WARPS = 4;

// A warp reads one tile of one head: the tokens of the call whose slots are that tile's, in a row, as they are for a sequence's
// tokens.  Lanes hold what a 16-byte read gives them: of the keys 16 channels of a token (twice per group), of the values 2 channels
// of 4 tokens per word, which 8 x 8 transposes turn into pairs of channels of one token.  Rows are put together in shared memory and
// leave whole.  Tokens whose slots are not a tile's are read one by one, 8 channels per lane.
template <int D>
__global__ void __launch_bounds__(RD_WARPS * 32) kv4_read_kernel(const __grid_constant__ Kv4ReadDesc g) {
    constexpr int G = D / KV4_GROUP, W = D >= 128 ? 2 : 1, PITCH = 2 * D + 16;  // bytes of a staged row: 4 banks on from the one before
    __shared__ __align__(16) uint8_t staged[RD_WARPS][KV4_TILE * PITCH];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * RD_WARPS + warp;
    const int64_t chunk = id / g.cache.heads_kv;
    const int h = static_cast<int>(id - chunk * g.cache.heads_kv);
    // chunks are cut where the first token's tile ends, and every 16 tokens from there
    const int64_t slot0 = g.slots[0];
    const int64_t token0 = chunk * KV4_TILE - (slot0 > 0 ? slot0 & (KV4_TILE - 1) : 0);
    if (token0 >= g.tokens) return;
    const int64_t limit = static_cast<int64_t>(g.cache.num_pages) * g.cache.page_size;
    const int t = lane & (KV4_TILE - 1);
    const bool asked = token0 + t >= 0 && token0 + t < g.tokens;
    const int64_t slot = asked ? g.slots[token0 + t] : -1;
    const uint32_t asked_mask = __ballot_sync(0xffffffffu, asked);
    const int64_t tile_slot = __shfl_sync(0xffffffffu, slot - t, __ffs(asked_mask) - 1);
    const bool whole = __all_sync(0xffffffffu, !asked || (slot - t == tile_slot && slot >= 0 && slot < limit && (tile_slot & (KV4_TILE - 1)) == 0));
    auto tile_at = [&](int64_t s) {
        const int64_t page = s >> 32 == 0 ? static_cast<uint32_t>(s) / static_cast<uint32_t>(g.cache.page_size) : s / g.cache.page_size;
        const int off = static_cast<int>(s - page * g.cache.page_size);
        return g.cache.base + page * g.cache.page_stride + (static_cast<int64_t>(h) * (g.cache.page_size / KV4_TILE) + off / KV4_TILE) * kv4_tile_bytes(D);
    };
    if (whole) {
        const uint8_t* tile = tile_at(tile_slot);
        uint8_t* mine = staged[warp];
        uint32_t kw[2][2 * G], kp[2][G], vw[4 * G], vp[4][G];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if constexpr (W == 2) {
#pragma unroll
                for (int q = 0; q < G / 2; ++q) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(tile + q * 1024 + e * 512 + lane * 16));
                    kw[e][4 * q] = v.x, kw[e][4 * q + 1] = v.y, kw[e][4 * q + 2] = v.z, kw[e][4 * q + 3] = v.w;
                }
            } else {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(tile + e * 256 + lane * 8));
                kw[e][0] = v.x, kw[e][1] = v.y;
            }
#pragma unroll
            for (int q = 0; q < G; ++q) kp[e][q] = __ldg(reinterpret_cast<const uint32_t*>(tile + kv4_pair_offset(D, 0)) + (r + 8 * e) * G + q);
        }
#pragma unroll
        for (int q = 0; q < G; ++q) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(tile + 8 * D + q * 512 + lane * 16));
            vw[4 * q] = v.x, vw[4 * q + 1] = v.y, vw[4 * q + 2] = v.z, vw[4 * q + 3] = v.w;
#pragma unroll
            for (int e = 0; e < 4; ++e)  // tokens 2 c, 8 + 2 c, 2 c + 1, 9 + 2 c, as the bytes of a word
                vp[e][q] = __ldg(reinterpret_cast<const uint32_t*>(tile + kv4_pair_offset(D, 1)) + (2 * c + (e >> 1) + 8 * (e & 1)) * G + q);
        }
        auto pair = [](uint32_t v, f32x2& s, f32x2& m) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
            s = both(f.x, f.x), m = both(f.y, f.y);
        };
        auto leave = [&](void* base, int64_t ld) {
            __syncwarp();
            constexpr int CHUNKS = D / 8;  // of 16 bytes in a row
#pragma unroll
            for (int y = 0; y < KV4_TILE * CHUNKS / 32; ++y) {
                const int row = (y * 32 + lane) / CHUNKS, at = lane % CHUNKS;
                if ((asked_mask >> row) & 1u)
                    *(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + (token0 + row) * ld + static_cast<int64_t>(h) * D) + at) =
                        *reinterpret_cast<const uint4*>(mine + row * PITCH + at * 16);
            }
            __syncwarp();
        };
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int q = 0; q < G; ++q) {
                f32x2 s, m;
                pair(kp[e][q], s, m);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t word = W == 2 ? kw[e][q / 2 * 4 + (q & 1) * 2 + u] : kw[e][u];
                    f32x2 x[4];
                    codes_f32(word & 0x0f0f0f0fu, (word >> 4) & 0x0f0f0f0fu, x);  // byte b: channels 2 b and 2 b + 1
                    uint32_t o[4];
#pragma unroll
                    for (int b = 0; b < 4; ++b) o[b] = pack2(fma2(s, x[b], m));
                    *reinterpret_cast<uint4*>(mine + (r + 8 * e) * PITCH + 2 * (64 * q + 16 * c + 8 * u)) = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
        leave(g.k, g.ldk);
#pragma unroll
        for (int q = 0; q < G; ++q) {
            // pairs of tokens: (2 c, 2 c + 1) are bytes 0 and 2 of a word, (8 + 2 c, 9 + 2 c) bytes 1 and 3
            f32x2 s[2], m[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&vp[e][q])), b = __half22float2(*reinterpret_cast<const __half2*>(&vp[2 + e][q]));
                s[e] = both(a.x, b.x), m[e] = both(a.y, b.y);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const uint32_t four = (vw[4 * q + j] >> (4 * n)) & 0x0f0f0f0fu;
                    const f32x2 back = both(-8388608.0f, -8388608.0f);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const f32x2 x = add2(both(__uint_as_float(__byte_perm(four, 0x4b000000u, 0x7440 + e)), __uint_as_float(__byte_perm(four, 0x4b000000u, 0x7442 + e))), back);
                        const uint32_t turned = movmatrix_trans(pack2(fma2(s[e], x, m[e])));  // token 8 e + r, channels 2 c, 2 c + 1 of eight
                        *reinterpret_cast<uint32_t*>(mine + (8 * e + r) * PITCH + 2 * (64 * q + 16 * j + 8 * n + 2 * c)) = turned;
                    }
                }
        }
        leave(g.v, g.ldv);
        return;
    }
    for (uint32_t left = asked_mask & 0xffffu; left != 0u; left &= left - 1u) {
        const int row = __ffs(left) - 1;
        const int64_t s = __shfl_sync(0xffffffffu, slot, row);
        if (s < 0) continue;
        if (s >= limit) {
            atomicCAS(&g_kv4_append_device_status, 0, 402);
            continue;
        }
        const uint8_t* tile = tile_at(s);
        const int tok = static_cast<int>(s & (KV4_TILE - 1));
        if (lane < D / 8) {
            const int d = 8 * lane;
            auto pair_of = [&](int values) {
                return __half22float2(*reinterpret_cast<const __half2*>(tile + kv4_pair_offset(D, values) + (tok * G + (d >> 6)) * 4));
            };
            auto store = [&](void* base, int64_t ld, const float* x) {
                const uint2 a = pack4(x), b = pack4(x + 4);
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + (token0 + row) * ld + static_cast<int64_t>(h) * D + d) = make_uint4(a.x, a.y, b.x, b.y);
            };
            float x[8];
            float2 sm = pair_of(0);
            const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + kv4_key_byte<D>(tok, d));
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(__fmul_rn(sm.x, static_cast<float>((word >> (4 * e)) & 15u)), sm.y);
            store(g.k, g.ldk, x);
            sm = pair_of(1);
            const int shift = (d & 8) ? 4 : 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t byte = tile[kv4_value_byte<D>(tok, (d & ~15) + e)];
                x[e] = __fadd_rn(__fmul_rn(sm.x, static_cast<float>((byte >> shift) & 15u)), sm.y);
            }
            store(g.v, g.ldv, x);
        }
    }
}

}  // namespace

int32_t launch_qk_norm_rope(const NormRopeDesc& g, cudaStream_t stream) {
    NormRopeParams p = {};
    p.g = g;
    for (int i = 0; g.axis_of_pair != nullptr && i < g.rot_dim / 2; ++i)
        for (int bit = 0; bit < 3; ++bit) p.axis[i / 64][bit] |= static_cast<uint64_t>((g.axis_of_pair[i] >> bit) & 1) << (i % 64);
    p.g.axis_of_pair = nullptr;
    switch (g.head_dim) {
        case 64: return launch_norm_rope_d<64>(p, stream);
        case 128: return launch_norm_rope_d<128>(p, stream);
        case 256: return launch_norm_rope_d<256>(p, stream);
        default: return BQ_STATUS_UNSUPPORTED;
    }
}

int32_t launch_kv4_read(const Kv4ReadDesc& g, cudaStream_t stream) {
    const int64_t warps = (static_cast<int64_t>(g.tokens) + 2 * KV4_TILE - 2) / KV4_TILE * g.cache.heads_kv;  // the first tile may begin anywhere
    const int64_t blocks = (warps + RD_WARPS - 1) / RD_WARPS;
    if (blocks > 0x7fffffff) return BQ_STATUS_UNSUPPORTED;
    switch (g.cache.head_dim) {
        case 64: kv4_read_kernel<64><<<static_cast<unsigned>(blocks), RD_WARPS * 32, 0, stream>>>(g); break;
        case 128: kv4_read_kernel<128><<<static_cast<unsigned>(blocks), RD_WARPS * 32, 0, stream>>>(g); break;
        case 256: kv4_read_kernel<256><<<static_cast<unsigned>(blocks), RD_WARPS * 32, 0, stream>>>(g); break;
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
