// What the two attention kernels over the 4-bit cache share: the launch's parameters, a sequence's lengths, small arithmetic.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kv4_format.cuh"
#include "ptx_sm100a.cuh"

namespace bq {

constexpr float KV4_NO_REF = -3.0e38f;                    // the softmax's reference before the first key: below every score
constexpr float KV4_FAR = 1048576.0f;                     // scores (log2) up to here have steps of 2^-3 at most
constexpr long long KV4_WAIT_LIMIT = 2000000000LL;        // cycles: about a second

struct AttnParams {
    const __nv_bfloat16* q;
    int64_t ldq;
    const int32_t* cu_q;
    Kv4Cache cache;
    const int32_t* table;
    int64_t ld_table;
    const int32_t* kv_lens;
    __nv_bfloat16* out;
    int64_t ldo;
    float* lse;
    float scale_log2;  // scale * log2(e)
    int32_t causal, back;  // keys that a row sees before its last one: the window less 1, 2^31 - 2 without a window
    int32_t batch, total_q, max_q, max_kv, heads_q, group;
    int32_t row_tiles, splits, tile_rows;  // blocks of query rows of a kv head, slices of the keys, rows of a block
    int32_t ctas;                          // of the launch
    float* part_o;   // [tile][split][rows][D]
    float2* part_ml; // [tile][split][rows]
    int2* shares;    // null, or of each block of rows: place of its first part, CTA of its last; part_o is then [CTA][2][rows][D]
    int32_t stall;         // 1: barriers that nothing completes (the self-test of the waits)
    long long wait_limit;  // of every wait, in cycles
};

// How many parts a block of rows has by its entry in `shares`; 0 for an entry that no CTA of the launch can have written: one that
// gave up a wait leaves those of its later blocks as they were, and the workspace may hold anything.
__device__ __forceinline__ int parts_of_share(int2 share, int ctas) {
    if (share.x < 0 || share.x >= 2 * ctas || share.y < share.x / 2 || share.y >= ctas) return 0;
    return share.y - share.x / 2 + 1;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A sequence as this launch sees it: query rows [row0, row0 + n), len keys.  Lengths beyond what the caller announced are cut
// (and reported), so that no read or write leaves the buffers.
struct Sequence {
    int row0, n, len;
};
__device__ __forceinline__ Sequence sequence_of(const AttnParams& p, int b, int* status) {
    Sequence s;
    int end = p.cu_q[b + 1];
    s.row0 = p.cu_q[b];
    s.len = p.kv_lens[b];
    if (s.row0 < 0 || end > p.total_q || end - s.row0 > p.max_q || s.len > p.max_kv) atomicCAS(status, 0, 403);
    s.row0 = max(s.row0, 0);
    end = min(end, p.total_q);
    s.n = max(0, min(end - s.row0, p.max_q));
    s.len = max(0, min(s.len, p.max_kv));
    return s;
}

// The first key that a row sees whose last one is `last` (negative: before the first).  Nothing here leaves 32 bits, whatever the window.
__device__ __forceinline__ int first_seen(const AttnParams& p, int last) { return max(last, p.back) - p.back; }

// Shape of a launch: which kernel, its blocks and slices.
struct AttnShape {
    int tensor;     // 1: kv4_prompt_sm100a.cu, 0: kv4_attention_sm100a.cu
    int tile_rows;  // 8 or 16; 128 or 256
    int row_tiles, splits;
    int64_t tiles, ctas;
    bool joined;    // a second kernel adds parts of blocks
};
int32_t launch_kv4_prompt(const AttnParams& p, const AttnShape& s, cudaStream_t stream);
int32_t read_and_clear_kv4_prompt_device_status();

}  // namespace bq
