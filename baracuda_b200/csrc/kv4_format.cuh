// The 4-bit cache's storage and the launch descriptors of the kernels that fill and read it.
//
// A page holds `page_size` tokens (a multiple of 16) of every kv head: [heads_kv][page_size / 16] tiles of 18 * D bytes.
// Each group of 64 channels of one token and head is 64 codes c = 0..15 with an f16 scale s and an f16 minimum m; the value
// is s * c + m.  A tile (16 tokens of one head) is laid out so that a warp's 16-byte shared-memory reads, lane after lane, ARE
// the fragments of mma.m16n8k16, with no permutation in between:
//   keys    8 D bytes: row t, chunk c, group-in-chunk gw, half u, byte b, nibble n hold channel 64 g + 16 c + 8 u + 2 b + n at
//           byte (((h * 16 + t) * 4 + c) * W + gw) * 8 + 4 u + b, W = min(2, D / 64), h = g / W, gw = g % W
//   values  8 D bytes: channel 64 h + 16 j + 8 n + r of token 8 e + 2 c + o is nibble n of byte
//           h * 512 + (r * 4 + c) * 16 + 4 j + 2 o + e  (one 32-bit word: 4 tokens x 2 channels, a whole A fragment)
//   (s, m)  of the keys [16][D / 64], then of the values
// Both nibble orders leave token- or channel-pairs 16 bits apart, so `word & 0x000f000f` is already a pair of f16 numbers
// (subnormals, code * 2^-24) and `word & 0x00f000f0` one of code * 2^-20: the matrix instructions take them as they are.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "launch.h"

namespace bq {

constexpr int KV4_GROUP = 64;  // channels that share a scale and a minimum
constexpr int KV4_TILE = 16;   // tokens of a tile
constexpr float KV4_CUT = 32768.0f;  // channels beyond are cut: every value of the cache is then a finite f16 number

__host__ __device__ constexpr int kv4_tile_bytes(int d) { return 18 * d; }
__host__ __device__ constexpr int kv4_pair_offset(int d, int values) { return 16 * d + values * d; }

// Offset of the keys' byte that holds channels d and d + 1 (d even) of token t.
template <int D>
__device__ __forceinline__ int kv4_key_byte(int t, int d) {
    constexpr int W = D >= 128 ? 2 : 1;
    const int g = d >> 6;
    return ((((g / W) * 16 + t) * 4 + ((d & 63) >> 4)) * W + g % W) * 8 + ((d & 15) >> 1);
}
// Offset, within a tile, of the values' byte that holds channels d and d + 8 (d % 16 < 8) of token t.
template <int D>
__device__ __forceinline__ int kv4_value_byte(int t, int d) {
    return 8 * D + (d >> 6) * 512 + ((d & 7) * 4 + ((t & 7) >> 1)) * 16 + ((d & 63) >> 4) * 4 + (t & 1) * 2 + (t >> 3);
}

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
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) { return fma2(b, 0xbf800000bf800000ull, a); }

struct Kv4Cache {
    uint8_t* base;
    int64_t page_stride;  // bytes, a multiple of 16
    int32_t num_pages;
    int32_t page_size;
    int32_t heads_kv;
    int32_t head_dim;
};

struct NormRopeDesc {
    int32_t tokens, heads_q, heads_kv, head_dim;
    const void* q;
    int64_t ldq;
    const void* k;
    int64_t ldk;
    const void* v;  // cache only
    int64_t ldv;
    const float* q_weight;  // null: no norm
    const float* k_weight;
    float eps;
    const float* cos_sin;  // [max_pos][rot_dim]: cosines of the pairs, then sines; null when rot_dim is 0
    int32_t rot_dim, max_pos, interleaved;
    const int32_t* positions;  // [axes][pos_stride]
    int64_t pos_stride;
    int32_t axes;
    const uint8_t* axis_of_pair;  // host, rot_dim / 2 entries; null: axis 0
    void* q_out;
    int64_t ldqo;
    void* k_out;  // dense keys, or null when the cache takes them
    int64_t ldko;
    int32_t to_cache;
    Kv4Cache cache;
    const int64_t* slots;
};
int32_t launch_qk_norm_rope(const NormRopeDesc& g, cudaStream_t stream);

struct Kv4ReadDesc {
    int32_t tokens;
    Kv4Cache cache;
    const int64_t* slots;
    void* k;
    int64_t ldk;
    void* v;
    int64_t ldv;
};
int32_t launch_kv4_read(const Kv4ReadDesc& g, cudaStream_t stream);
int32_t read_and_clear_kv4_append_device_status();

struct Kv4AttentionDesc {
    int32_t batch, total_q, max_q, max_kv, heads_q;
    const void* q;
    int64_t ldq;
    const int32_t* cu_q;
    Kv4Cache cache;
    const int32_t* page_table;
    int64_t ld_table;
    const int32_t* kv_lens;
    float scale;
    int32_t causal, window;
    void* out;
    int64_t ldo;
    float* lse;  // [total_q][heads_q], or null
    void* workspace;
    size_t workspace_bytes;
};
int32_t launch_kv4_attention(const Kv4AttentionDesc& g, cudaStream_t stream);
size_t kv4_attention_workspace_bytes(int32_t batch, int32_t max_q, int32_t max_kv, int32_t heads_q, int32_t heads_kv,
                                     int32_t head_dim);
// Whether the launch's block count fits a grid.
bool kv4_attention_fits(int32_t batch, int32_t max_q, int32_t max_kv, int32_t heads_q, int32_t heads_kv, int32_t head_dim);
int32_t read_and_clear_kv4_attention_device_status();
int32_t set_kv4_wait_selftest(int64_t limit_cycles);

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

}  // namespace bq
