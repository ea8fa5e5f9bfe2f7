// Attention of a few query rows per sequence over the 4-bit cache (kv4_format.cuh).
//   out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j]) v[j],  j over the keys that row i sees; lse = log sum_j exp(...)
//
// Bound: the cache's bytes (144 per token and kv head at D = 128), which every other term hides behind as long as a token
// costs few instructions.  So codes are never turned into numbers: both products run on mma.m16n8k16 with the codes as the A
// operand in the form in which they lie in memory (f16 subnormals, one AND per pair; one shift per word), 16 tokens x 8 query
// rows at a time, and scales and minima enter outside, per group g of 64 channels:
//   q . k[t]  = sum_g s[t, g] * (q_g . c[t, g]) + sum_g m[t, g] * sum(q_g)      (S^T = C Q^T; the minima's part is one more product,
//                                                                               of m and the sums as two f16 numbers each)
//   sum_t p[t] v[t] = sum_t (p[t] s[t, g]) c[t, g] + sum_t p[t] m[t, g]         (O^T = C^T W, W = p * s in f16; again one more)
// The query rows are brought to f16 by a power of two of their own (bf16 has 8 bits of precision, f16 11: exact unless 2^-38
// of the row's largest), products and sums are f32.  p and W are rounded to f16, 2^-11 each.  The softmax is the one-pass form
// with a running reference, kept so that p lies at most at 2^cap, and cap so that W fits f16 whatever the scales: with the
// largest p near 2^11, weights keep full precision down to 2^-25 of it.  The reference moves only when a p would exceed 2^cap,
// so the common step has one vote instead of a reduction.
//
// Work: as many CTAs of 4 warps as are resident at once share the launch's work equally, whatever the lengths of its sequences:
// each takes a run of blocks of 8 or 16 query rows of a kv head, the first and the last perhaps in part.  Each warp streams its
// own 64-token steps (32 where D is 256) through two shared-memory stages filled by bulk copies (one lane per 16-token tile
// issues the copy, the pages of the next 32 tiles are looked up at once), so the main loop has no CTA-wide synchronisation.
// Warps are joined in shared memory, parts of a block through the workspace by a second kernel (in the order of the keys: the
// result does not depend on timing).
//
// Measured (B200), 32 query and 8 kv heads of 128 unless said: one sequence of 129 tokens 7 us; 64 ragged ones up to 4001 tokens
// (179 MB) 49.9 us; 2 x 131071 tokens with 64 query heads 65.7 us, 4.6 TB/s over all; from 64 x 2048 to 64 x 8192 tokens a call grows
// by 6.4 TB/s, from 2 x 131071 to 2 x 262143 by 6.5, and about 20 us do not depend on the number of keys; 16 x 5 drafted tokens over up
// to 6001 with 40 heads 50.4 us: 25 rows of a kv head are two blocks of 16, whose products and softmax are the bound.  Blocks of 24 rows
// spilled more and took 41 us against 41 (24 rows, 16 x 6000) and 60 against 54 (48 rows); D = 128 spills 60 (8 rows, 168 registers) and
// 80 bytes (16 rows, 255) of loads as it is.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>

#include <type_traits>

#include "../../include/baracuda_kernels_q.h"
#include "kv4_attention.cuh"

namespace bq {

namespace {

__device__ int g_kv4_attention_device_status = 0;

constexpr int AT_WARPS = 4;
constexpr int AT_BLOCK_UNITS = 2;  // look-ups, queries and join of a block take the time of about two units
constexpr int AT_STAGES = 2;  // the parts of a CTA alternate between them: not another number
// Rows of a kv head up to which codes go to mma.sync as they are: 16 sequences x 6000 tokens take 54 us with 48 rows (tcgen05 kernel 53),
// 42 with 32 (52) and 97 with 96 (54); with D = 256, 84 us with 32 rows (96) and 122 with 48 (96)
constexpr int AT_MOST_ROWS = 48, AT_MOST_ROWS_256 = 32;
constexpr float SLACK = 4.0f;  // a new reference leaves this many powers of two before the next
constexpr int AT_ASSUMED_SMS = 148;  // the workspace's size must not depend on the device that asks
thread_local long long t_wait_selftest = 0;  // 0, or the limit of waits whose barriers are not to be completed

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <int D, int NT>
struct AttnCfg {
    static constexpr int TILES = D == 256 ? 2 : 4;           // of 16 tokens, of a warp's step
    static constexpr int STEP = TILES * KV4_TILE;
    static constexpr int RESIDENT = NT == 2 || D == 256 ? 2 : D == 128 ? 3 : 4;  // CTAs of an SM (registers, shared memory)
};
template <int D, int NT>
struct AttnSmem {
    static constexpr int AT_TILES = AttnCfg<D, NT>::TILES;
    static constexpr int STAGE = AT_TILES * kv4_tile_bytes(D);
    static constexpr int RING = AT_WARPS * AT_STAGES * STAGE;  // [stage][warp]: the join takes the place of one stage
    static constexpr int PITCH = D + 4;  // of a row in the join: a warp's stores go to all banks
    static constexpr int JOIN = AT_WARPS * 8 * NT * (PITCH + 2) * 4;
    static_assert(JOIN <= AT_WARPS * STAGE, "the join fits one stage");
    static constexpr int BARS = RING;
    static constexpr int VALID = BARS + AT_WARPS * AT_STAGES * 8;
    static constexpr int SCAN = VALID + AT_WARPS * AT_STAGES * 4;  // sums of the warps, then what the scan found
    static constexpr int TOTAL = SCAN + (AT_WARPS + 4) * 8;
};

// What a sequence asks for: blocks of rows, the warp steps from the first row's first key to the last row's last, units of a block
// (AT_BLOCK_UNITS of them for what a block costs apart from its keys: they come first, without keys).
struct Extent {
    Sequence sq;
    int blocks, step0, steps, units;
};
template <int STEP, int ROWS>
__device__ __forceinline__ Extent extent_of(const AttnParams& p, int b) {
    Extent x;
    x.sq = sequence_of(p, b, &g_kv4_attention_device_status);
    x.blocks = (x.sq.n * p.group + ROWS - 1) / ROWS;
    const int first = x.sq.len - x.sq.n;
    const int hi = max(0, p.causal ? min(x.sq.len, first + x.sq.n) : x.sq.len), lo = first_seen(p, first);
    x.step0 = lo / STEP;
    x.steps = max(0, (hi + STEP - 1) / STEP - x.step0);
    x.units = AT_BLOCK_UNITS + max(1, (x.steps + AT_WARPS - 1) / AT_WARPS);  // rows without keys are to be written too
    return x;
}

template <int D, int NT>
__global__ void __launch_bounds__(AT_WARPS * 32, AttnCfg<D, NT>::RESIDENT) kv4_attention_kernel(const __grid_constant__ AttnParams p) {
    using L = AttnSmem<D, NT>;
    constexpr int G = D / KV4_GROUP;
    constexpr int W = D >= 128 ? 2 : 1;       // groups of a 16-byte chunk of keys
    constexpr int TILE = kv4_tile_bytes(D);
    constexpr int ROWS = 8 * NT;
    constexpr int MT = D / 16;                // 16-channel blocks of the output
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;

    constexpr int AT_TILES = AttnCfg<D, NT>::TILES, AT_STEP = AttnCfg<D, NT>::STEP;

    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS) + warp * AT_STAGES;
    volatile uint32_t* valid = reinterpret_cast<volatile uint32_t*>(smem + L::VALID) + warp * AT_STAGES;
    uint8_t* ring = smem + warp * L::STAGE;  // stages AT_WARPS * STAGE apart
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < AT_STAGES; ++s) mbar_init(&bars[s], 1 + p.stall);
        fence_barrier_init();
    }
    __syncwarp();

    // This CTA's share: of the launch's units (256 tokens of one block of rows and kv head; 128 where D is 256), numbered over
    // sequences, kv heads, blocks of rows and tokens, an equal part in a row.  Its ends may lie inside a block: the parts of such a
    // block are joined by the second kernel.
    auto units_of = [&](int b_) -> int64_t {
        if (b_ >= p.batch) return 0;
        const Extent x = extent_of<AT_STEP, ROWS>(p, b_);
        return static_cast<int64_t>(x.blocks) * p.cache.heads_kv * x.units;
    };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may take its place early; it waits for the end
    int64_t total = 0, before = 0;  // units of the launch; of the sequences before b
    int b = 0;
    if (p.batch <= 32) {  // each warp for itself
        const int64_t own = units_of(lane);
        int64_t sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        total = __shfl_sync(0xffffffffu, sum, 31);
        const int64_t ctas_ = min(static_cast<int64_t>(gridDim.x), total);
        b = __popc(__ballot_sync(0xffffffffu, sum <= blockIdx.x * total / max(ctas_, int64_t{1})));  // sequences that end at or before this CTA's first unit
        before = __shfl_sync(0xffffffffu, sum - own, b & 31);
    } else {
        int64_t* scan = reinterpret_cast<int64_t*>(smem + L::SCAN);  // [AT_WARPS] sums, then sequence and the units before it
        const int64_t mine0 = units_of(threadIdx.x);                 // of the first 128 sequences, often all
        total = mine0;
        for (int x = threadIdx.x + AT_WARPS * 32; x < p.batch; x += AT_WARPS * 32) total += units_of(x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lane == 0) scan[warp] = total;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < AT_WARPS; ++w) total += scan[w];
        const int64_t first = blockIdx.x * total / max(min(static_cast<int64_t>(gridDim.x), total), int64_t{1});
        if (first < total) {
            for (int x0 = 0;; x0 += AT_WARPS * 32) {
                int64_t sum = x0 == 0 ? mine0 : units_of(x0 + threadIdx.x);
                const int64_t own = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += y;
                }
                __syncthreads();
                if (lane == 31) scan[warp] = sum;
                __syncthreads();
                int64_t chunk = 0;
#pragma unroll
                for (int w = 0; w < AT_WARPS; ++w) {
                    if (w < warp) sum += scan[w];
                    chunk += scan[w];
                }
                if (before + sum - own <= first && first < before + sum) scan[AT_WARPS] = x0 + threadIdx.x, scan[AT_WARPS + 1] = before + sum - own;
                if (first < before + chunk) break;
                before += chunk;
            }
            __syncthreads();
            b = static_cast<int>(scan[AT_WARPS]);
            before = scan[AT_WARPS + 1];
        }
    }
    const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);  // none without a unit: parts are counted by CTAs
    if (blockIdx.x >= ctas) return;
    int64_t unit = blockIdx.x * total / ctas;
    const int64_t unit_end = (blockIdx.x + 1) * total / ctas;
    Extent xt = extent_of<AT_STEP, ROWS>(p, b);
    uint32_t phases = 0;  // bit s: the phase that stage s is waited for next; every part begins with stage 0
    bool at_start = true;

    // a block of rows, or the part of one that falls to this CTA
    struct Part {
        int b, hk, rt, unit0, unit1, units;  // units with keys: [unit0, unit1) of `units`
        int64_t begin;                       // number of the block's first unit
        Sequence sq;
        int step0, my_begin, my_end, hi_all, mine;
    };
    // the next part of this CTA from `unit` on that has keys (or is a block without any); false at the end
    auto next_part = [&](Part& t) {
        while (unit < unit_end) {
            while (unit >= before + static_cast<int64_t>(xt.blocks) * p.cache.heads_kv * xt.units) {
                before += static_cast<int64_t>(xt.blocks) * p.cache.heads_kv * xt.units;
                xt = extent_of<AT_STEP, ROWS>(p, ++b);
            }
            const int64_t in_seq = unit - before;
            const int block = static_cast<int>(in_seq / xt.units), at = static_cast<int>(in_seq - static_cast<int64_t>(block) * xt.units);
            const int to = static_cast<int>(min(static_cast<int64_t>(xt.units), at + (unit_end - unit)));
            t.begin = unit - at;
            unit += to - at;
            t.units = xt.units - AT_BLOCK_UNITS;
            t.unit0 = max(0, at - AT_BLOCK_UNITS), t.unit1 = max(0, to - AT_BLOCK_UNITS);
            if (t.unit0 == t.unit1) continue;
            t.b = b, t.hk = block / xt.blocks, t.rt = block - t.hk * xt.blocks;
            t.sq = xt.sq;
            const int last_row = min(ROWS, t.sq.n * p.group - t.rt * ROWS) - 1 + t.rt * ROWS;
            t.hi_all = max(0, p.causal ? min(t.sq.len, t.sq.len - t.sq.n + last_row / p.group + 1) : t.sq.len);
            t.step0 = xt.step0, t.my_begin = t.unit0 * AT_WARPS, t.my_end = min(t.unit1 * AT_WARPS, xt.steps);
            t.mine = t.my_end - t.my_begin > warp ? (t.my_end - t.my_begin - warp + AT_WARPS - 1) / AT_WARPS : 0;  // steps of this warp
            return true;
        }
        return false;
    };
    // lane i knows where the i-th of the warp's next 32 tiles lies (-1: nowhere); the first lanes fetch the tiles of a step
    const int tiles_per_page = p.cache.page_size / KV4_TILE;
    int64_t ahead = -1;
    constexpr int LOOK = 32 / AT_TILES;
    auto look_up = [&](const Part& t, int k) {  // of this warp's steps k .. k + LOOK - 1
        const int step = t.my_begin + warp + (k + lane / AT_TILES) * AT_WARPS;
        const int tile = (t.step0 + step) * AT_TILES + lane % AT_TILES;
        ahead = -1;
        // a step's first tiles may lie before the first key that the sequence's rows see: they need not be anywhere
        if (step < t.my_end && tile * KV4_TILE < t.hi_all && (tile + 1) * KV4_TILE > first_seen(p, t.sq.len - t.sq.n)) {
            const int at = tile / tiles_per_page, page = p.table[static_cast<int64_t>(t.b) * p.ld_table + at];
            if (page >= 0 && page < p.cache.num_pages) {
                ahead = static_cast<int64_t>(page) * p.cache.page_stride + (static_cast<int64_t>(t.hk) * tiles_per_page + tile - at * tiles_per_page) * TILE;
            } else {
                atomicCAS(&g_kv4_attention_device_status, 0, 404);
            }
        }
    };
    auto fetch = [&](const Part& t, int k, int to_stage) {  // the warp's k-th step
        if (k % LOOK == 0) look_up(t, k);
        const int64_t where = __shfl_sync(0xffffffffu, ahead, k % LOOK * AT_TILES + (lane & (AT_TILES - 1)));
        const uint32_t have = __ballot_sync(0xffffffffu, where >= 0) & ((1u << AT_TILES) - 1u);
        if (lane == 0) {
            valid[to_stage] = have;
            mbar_arrive_expect_tx(&bars[to_stage], __popc(have) * TILE);
        }
        __syncwarp();
        if (lane < AT_TILES && where >= 0) bulk_load_1d(ring + to_stage * (AT_WARPS * L::STAGE) + lane * TILE, p.cache.base + where, TILE, &bars[to_stage]);
    };

    Part now;
    if (!next_part(now)) return;
    if (now.mine > 0) fetch(now, 0, 0);
    for (;;) {
    const Sequence sq = now.sq;
    const int hk = now.hk, rt = now.rt, step0 = now.step0, my_begin = now.my_begin, mine = now.mine;
    const int rows = min(ROWS, sq.n * p.group - rt * ROWS);  // row = query index * group + head in group
    const int past = sq.len - sq.n;                          // the last key that query row i sees is past + i when causal
    if (mine > 1) fetch(now, 1, 1);  // the first step is on its way
    int stage = 0;

    // the query rows as B fragments: lane (r, c) holds, of row r of each 8-row block, channels 64 g + 16 c .. + 15
    uint32_t qf[NT][G][8];
    uint32_t qsum[NT];    // the sum over group c, as two f16 numbers, for the minima's product
    float qscale[NT][2];  // of this lane's score columns 2 c, 2 c + 1
    int row_hi[NT][2], row_lo[NT][2];     // keys [lo, hi) that those rows see
    int hi_min = 0x7fffffff, lo_max = 0;  // over the rows that exist: steps inside need no mask
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = rt * ROWS + nt * 8 + r;
        const bool there = nt * 8 + r < rows;
        float x[G][16];
        float top = 0.0f, sums[G];
        const __nv_bfloat16* src = p.q + static_cast<int64_t>(sq.row0 + (there ? row / p.group : 0)) * p.ldq +
                                   static_cast<int64_t>(hk * p.group + (there ? row % p.group : 0)) * D + 16 * c;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
            if (there) {
                raw[0] = *reinterpret_cast<const uint4*>(src + 64 * g);
                raw[1] = *reinterpret_cast<const uint4*>(src + 64 * g + 8);
            }
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(raw);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[g][2 * e] = __low2float(h[e]);
                x[g][2 * e + 1] = __high2float(h[e]);
                top = fmaxf(top, fmaxf(fabsf(x[g][2 * e]), fabsf(x[g][2 * e + 1])));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14;  // 2^-ex brings the largest into [2^14, 2^15)
        ex = top == 0.0f || top == INFINITY ? 0 : max(-100, ex);  // at most 113
        const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23), up = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            sums[g] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[g] += fmaf(x[g][2 * e], down, x[g][2 * e + 1] * down);
            sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
            sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
#pragma unroll
            for (int u = 0; u < 2; ++u) {  // nibbles n and n + 4 of a word are a pair; odd nibbles come as 16 times the code
                const float* w = &x[g][8 * u];
                const float odd = down * 0.0625f;
                qf[nt][g][4 * u] = pack_half2(w[0] * down, w[4] * down);
                qf[nt][g][4 * u + 1] = pack_half2(w[1] * odd, w[5] * odd);
                qf[nt][g][4 * u + 2] = pack_half2(w[2] * down, w[6] * down);
                qf[nt][g][4 * u + 3] = pack_half2(w[3] * odd, w[7] * odd);
            }
        }
        {
            float mine_sum = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) mine_sum = c == g ? sums[g] : mine_sum;
            mine_sum *= 0.0078125f;  // 64 * 2^15 at most: 2^-7 brings it into f16
            const float high = __half2float(__float2half_rn(mine_sum));
            qsum[nt] = pack_half2(high, mine_sum - high);
        }
        const int i = row / p.group;
        const int hi = !there ? 0 : p.causal ? max(0, min(sq.len, past + i + 1)) : sq.len;
        const int lo = first_seen(p, past + i);
        if (there) hi_min = min(hi_min, hi), lo_max = max(lo_max, lo);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int from = (2 * c + e) * 4;  // a lane that holds row 2 c + e
            // finite for queries of any size: a score is then too, if it fits f32
            qscale[nt][e] = fmaxf(fminf(__shfl_sync(0xffffffffu, up, from) * (16777216.0f * p.scale_log2), FLT_MAX), -FLT_MAX);
            row_hi[nt][e] = __shfl_sync(0xffffffffu, hi, from);
            row_lo[nt][e] = __shfl_sync(0xffffffffu, lo, from);
        }
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        hi_min = min(hi_min, __shfl_xor_sync(0xffffffffu, hi_min, o));
        lo_max = max(lo_max, __shfl_xor_sync(0xffffffffu, lo_max, o));
    }

    float acc[NT][MT][4], low[NT][4];  // O^T of the codes, and of the minima (row r: group r % G)
    float l[NT][2], ref[NT][2];
    bool fresh[NT][2];  // no key seen yet: any reference will do
    float cap = 15.0f, s_cap = 1.0f;  // p <= 2^cap keeps p and p * s within f16 for s <= s_cap
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) low[nt][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][j][e] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) l[nt][e] = 0.0f, ref[nt][e] = 0.0f, fresh[nt][e] = true;
    }

    // x = log2 p of the tiles of a step.  EDGE: some row does not see some key, or a tile is missing.
    auto weights = [&](auto edge, const uint8_t* base, int token0, uint32_t have, auto& x, float (&top)[NT][2], uint32_t& s_top) {
        constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
        for (int t = 0; t < AT_TILES; ++t) {
            const uint8_t* tile = base + t * TILE;
            float s[G][NT][4], m[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    m[nt][e] = 0.0f;
#pragma unroll
                    for (int g = 0; g < G; ++g) s[g][nt][e] = 0.0f;
                }
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(tile + kv4_pair_offset(D, 0));
            const uint32_t* vp = reinterpret_cast<const uint32_t*>(tile + kv4_pair_offset(D, 1));
            {  // the minima, against the sums (zero for c >= G)
                const int g = c < G ? c : 0;
                const uint32_t a0 = __byte_perm(kp[r * G + g], 0u, 0x3232), a1 = __byte_perm(kp[(r + 8) * G + g], 0u, 0x3232);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16(m[nt], a0, a1, 0u, 0u, c < G ? qsum[nt] : 0u, 0u);
                // every token and group lies in some lane
                uint32_t v0 = vp[r * G + g], v1 = vp[(r + 8) * G + g];
                if constexpr (EDGE) {
                    const int j = token0 + t * KV4_TILE + r;
                    if (j >= sq.len || ((have >> t) & 1u) == 0u) v0 = 0u;
                    if (j + 8 >= sq.len || ((have >> t) & 1u) == 0u) v1 = 0u;
                }
                s_top = max_f16x2(s_top, max_f16x2(v0, v1));
            }
#pragma unroll
            for (int h = 0; h < G / W; ++h) {
                uint32_t wa[2 * W], wb[2 * W];
                if constexpr (W == 2) {
                    const uint4 a = *reinterpret_cast<const uint4*>(tile + h * 1024 + lane * 16);
                    const uint4 bb = *reinterpret_cast<const uint4*>(tile + h * 1024 + 512 + lane * 16);
                    wa[0] = a.x, wa[1] = a.y, wa[2] = a.z, wa[3] = a.w;
                    wb[0] = bb.x, wb[1] = bb.y, wb[2] = bb.z, wb[3] = bb.w;
                } else {
                    const uint2 a = *reinterpret_cast<const uint2*>(tile + lane * 8);
                    const uint2 bb = *reinterpret_cast<const uint2*>(tile + 256 + lane * 8);
                    wa[0] = a.x, wa[1] = a.y;
                    wb[0] = bb.x, wb[1] = bb.y;
                }
#pragma unroll
                for (int y = 0; y < 2 * W; ++y) {
                    const int g = h * W + y / 2, u = y % 2;
                    const uint32_t a8 = wa[y] >> 8, b8 = wb[y] >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_f16(s[g][nt], wa[y] & 0x000f000fu, wb[y] & 0x000f000fu, wa[y] & 0x00f000f0u, wb[y] & 0x00f000f0u,
                                qf[nt][g][4 * u], qf[nt][g][4 * u + 1]);
                        mma_f16(s[g][nt], a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u,
                                qf[nt][g][4 * u + 2], qf[nt][g][4 * u + 3]);
                    }
                }
            }
            float sk[2][G];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int g = 0; g < G; ++g) sk[e][g] = __low2float(*reinterpret_cast<const __half2*>(kp + (r + 8 * e) * G + g));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float dot = m[nt][e] * 7.62939453125e-06f;  // 2^-17: in units of 2^-24, as the codes are
#pragma unroll
                    for (int g = 0; g < G; ++g) dot = fmaf(sk[e >> 1][g], s[g][nt][e], dot);
                    x[t][nt][e] = fmaf(dot, qscale[nt][e & 1], -ref[nt][e & 1]);
                }
            }
            if constexpr (EDGE) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int j = token0 + t * KV4_TILE + r + 8 * e;
                    const bool dead = j >= sq.len || ((have >> t) & 1u) == 0u;  // nothing there, whatever the bytes say
                    uint32_t ones = 0u;  // a value that is no number: rows that see the key become none either
#pragma unroll
                    for (int g = 0; g < G; ++g) ones |= (vp[(r + 8 * e) * G + g] & 0x7c007c00u) + 0x04000400u;
                    const bool bad = (ones & 0x80008000u) != 0u;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            float& v = x[t][nt][2 * e + y];
                            v = dead || j >= row_hi[nt][y] || j < row_lo[nt][y] ? -INFINITY : bad ? NAN : v;
                        }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                top[nt][0] = fmaxf(fmaxf(top[nt][0], x[t][nt][0]), x[t][nt][2]);
                top[nt][1] = fmaxf(fmaxf(top[nt][1], x[t][nt][1]), x[t][nt][3]);
            }
        }
    };
    auto values = [&](auto edge, const uint8_t* base, int token0, uint32_t have, const auto& x) {
        constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
        for (int t = 0; t < AT_TILES; ++t) {
            const uint8_t* tile = base + t * TILE;
            // (s, m) of the tokens 2 c, 2 c + 1 and 8 + 2 c, 9 + 2 c, as pairs of tokens
            uint32_t sv[2][G], mv[2][G];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t v[2 * G];
                const uint8_t* at = tile + kv4_pair_offset(D, 1) + (2 * c + 8 * e) * G * 4;
                if constexpr (G == 1) {
                    const uint2 y = *reinterpret_cast<const uint2*>(at);
                    v[0] = y.x, v[1] = y.y;
                } else {
#pragma unroll
                    for (int q = 0; q < G / 2; ++q) {
                        const uint4 y = *reinterpret_cast<const uint4*>(at + 16 * q);
                        v[4 * q] = y.x, v[4 * q + 1] = y.y, v[4 * q + 2] = y.z, v[4 * q + 3] = y.w;
                    }
                }
                if constexpr (EDGE) {  // zeros for what is not there or no number
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t ones = 0u;
#pragma unroll
                        for (int g = 0; g < G; ++g) ones |= (v[G * q + g] & 0x7c007c00u) + 0x04000400u;
                        const bool gone = token0 + t * KV4_TILE + 2 * c + 8 * e + q >= sq.len || ((have >> t) & 1u) == 0u || (ones & 0x80008000u) != 0u;
#pragma unroll
                        for (int g = 0; g < G; ++g) v[G * q + g] = gone ? 0u : v[G * q + g];
                    }
                }
#pragma unroll
                for (int g = 0; g < G; ++g) sv[e][g] = __byte_perm(v[g], v[G + g], 0x5410), mv[e][g] = __byte_perm(v[g], v[G + g], 0x7632);
            }
            uint32_t m0 = mv[0][0], m1 = mv[1][0];  // row r of the minima's product is group r % G
#pragma unroll
            for (int g = 1; g < G; ++g) m0 = (r & (G - 1)) == g ? mv[0][g] : m0, m1 = (r & (G - 1)) == g ? mv[1][g] : m1;
            uint32_t wf[NT][G][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float pr[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    pr[e] = ex2(x[t][nt][e]);
                    l[nt][e & 1] += pr[e];
                }
                const uint32_t b0 = movmatrix_trans(pack_half2(pr[0], pr[1])), b1 = movmatrix_trans(pack_half2(pr[2], pr[3]));
                mma_f16(low[nt], m0, 0u, m1, 0u, b0, b1);
#pragma unroll
                for (int g = 0; g < G; ++g) wf[nt][g][0] = mul_f16x2(b0, sv[0][g]), wf[nt][g][1] = mul_f16x2(b1, sv[1][g]);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint4 v = *reinterpret_cast<const uint4*>(tile + 8 * D + g * 512 + lane * 16);
                const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w0 = words[j], w8 = words[j] >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_f16(acc[nt][4 * g + j], w0 & 0x000f000fu, w0 & 0x00f000f0u, w8 & 0x000f000fu, w8 & 0x00f000f0u,
                                wf[nt][g][0], wf[nt][g][1]);
                }
            }
        }
    };

    int k = 0;
    bool gave_up = false;
    for (; k < mine; ++k) {
        const uint32_t parity = (phases >> stage) & 1u;
        if (!mbar_try_wait(&bars[stage], parity)) {
            const long long t0 = clock64();
            while (!mbar_try_wait(&bars[stage], parity)) {
                if (clock64() - t0 > p.wait_limit) {
                    gave_up = true;
                    break;
                }
            }
        }
        gave_up = __any_sync(0xffffffffu, gave_up);
        if (gave_up) break;
        const uint32_t have = valid[stage];
        const uint8_t* base = ring + stage * (AT_WARPS * L::STAGE);
        const int token0 = (step0 + my_begin + warp + k * AT_WARPS) * AT_STEP;
        const bool edge = token0 + AT_STEP > hi_min || token0 < lo_max || have != (1u << AT_TILES) - 1u;

        float x[AT_TILES][NT][4], top[NT][2];
        uint32_t s_top = 0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
        if (edge) {
            weights(std::true_type{}, base, token0, have, x, top, s_top);
        } else {
            weights(std::false_type{}, base, token0, have, x, top, s_top);
        }
        float largest = __low2float(*reinterpret_cast<const __half2*>(&s_top));
        bool grow = largest > s_cap;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) grow = grow || fresh[nt][0] || fresh[nt][1] || top[nt][0] > cap || top[nt][1] > cap;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) top[nt][e] = fmaxf(top[nt][e], __shfl_xor_sync(0xffffffffu, top[nt][e], o));
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
            if (largest > s_cap && largest < INFINITY) {  // the scale's power of two comes off the cap
                const int ex = static_cast<int>(__float_as_uint(largest) >> 23) - 126;
                cap = static_cast<float>(15 - ex);
                s_cap = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float fix[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool move = top[nt][e] > cap || (fresh[nt][e] && top[nt][e] > -INFINITY);
                    // where a step of f32 is no small number of powers of two, the largest itself is the reference
                    const float by = !move ? 0.0f : fabsf(ref[nt][e] + top[nt][e]) > KV4_FAR ? top[nt][e] : top[nt][e] - (cap - SLACK);
                    fix[e] = fresh[nt][e] ? 1.0f : ex2(-by);  // nothing to rescale before the first key
                    fresh[nt][e] = fresh[nt][e] && !move;
                    ref[nt][e] += by;
                    l[nt][e] *= fix[e];
#pragma unroll
                    for (int t = 0; t < AT_TILES; ++t) x[t][nt][e] -= by, x[t][nt][2 + e] -= by;
                }
                low[nt][0] *= fix[0], low[nt][1] *= fix[1];
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    acc[nt][j][0] *= fix[0], acc[nt][j][2] *= fix[0];
                    acc[nt][j][1] *= fix[1], acc[nt][j][3] *= fix[1];
                }
            }
        }
        if (edge) {
            values(std::true_type{}, base, token0, have, x);
        } else {
            values(std::false_type{}, base, token0, have, x);
        }
        __syncwarp();
        if (k + AT_STAGES < mine) fetch(now, k + AT_STAGES, stage);
        phases ^= 1u << stage;
        stage ^= 1;
    }
    if (gave_up) {
        if (lane == 0) atomicCAS(&g_kv4_attention_device_status, 0, 411);
        // copies of this warp may still be in flight into its ring: wait for them, again within a limit
        const long long t0 = clock64();
        for (int s = 0; s < AT_STAGES; ++s) {
            if (k + s >= mine) break;
            while (!mbar_try_wait(&bars[stage], (phases >> stage) & 1u) && clock64() - t0 < p.wait_limit) {
            }
            phases ^= 1u << stage;
            stage ^= 1;
        }
    }

    // join the lanes, then the warps
    float z[NT][2][G];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], o);
#pragma unroll
            for (int g = 0; g < G; ++g) z[nt][e][g] = __shfl_sync(0xffffffffu, low[nt][e], g * 4 + c);
        }
    // the next part's first step goes to stage 0, the join to the place of stage 1
    Part then;
    const bool more = next_part(then);
    fence_proxy_async_smem();
    __syncthreads();  // every warp has left its ring
    if (more && then.mine > 0 && !gave_up) fetch(then, 0, 0);
    float* join = reinterpret_cast<float*>(smem + AT_WARPS * L::STAGE);  // [warp][row][PITCH], then [warp][row] (ref, l)
    float2* join_ml = reinterpret_cast<float2*>(join + AT_WARPS * ROWS * L::PITCH);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float* row = join + (warp * ROWS + nt * 8 + 2 * c + e) * L::PITCH;
#pragma unroll
            for (int j = 0; j < MT; ++j) {  // codes were 2^-24 and 2^-20
                row[16 * j + r] = fmaf(acc[nt][j][e], 16777216.0f, z[nt][e][j / 4]);
                row[16 * j + 8 + r] = fmaf(acc[nt][j][2 + e], 1048576.0f, z[nt][e][j / 4]);
            }
            if (r == 0) join_ml[warp * ROWS + nt * 8 + 2 * c + e] = make_float2(fresh[nt][e] ? KV4_NO_REF : ref[nt][e], l[nt][e]);
        }
    __syncthreads();
    const bool whole = now.unit0 == 0 && now.unit1 == now.units;
    for (int at = threadIdx.x; at < rows * (D / 4); at += AT_WARPS * 32) {
        const int row = at / (D / 4), d = at % (D / 4) * 4;
        float m = KV4_NO_REF;
#pragma unroll
        for (int w = 0; w < AT_WARPS; ++w) m = fmaxf(m, join_ml[w * ROWS + row].x);
        float sum = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < AT_WARPS; ++w) {
            const float2 ml = join_ml[w * ROWS + row];
            const float f = ex2(ml.x - m);
            const float4 x = *reinterpret_cast<const float4*>(join + (w * ROWS + row) * L::PITCH + d);
            sum = fmaf(ml.y, f, sum);
            o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
        }
        if (whole) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int gr = rt * ROWS + row;
            const int64_t q_row = sq.row0 + gr / p.group;
            const int head = hk * p.group + gr % p.group;
            const __nv_bfloat162 a = __floats2bfloat162_rn(o.x * inv, o.y * inv), bb = __floats2bfloat162_rn(o.z * inv, o.w * inv);
            *reinterpret_cast<uint2*>(p.out + q_row * p.ldo + static_cast<int64_t>(head) * D + d) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&bb));
            if (p.lse != nullptr && d == 0) p.lse[q_row * p.heads_q + head] = sum == 0.0f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
        } else {
            const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (at_start ? 0 : 1)) * ROWS + row;
            *reinterpret_cast<float4*>(p.part_o + slot * D + d) = o;
            if (d == 0) p.part_ml[slot] = make_float2(m, sum);
        }
    }
    // the CTA with a block's first unit says who has the others (parts of a CTA's first block are in its first place, of its last
    // in its second)
    if (now.unit0 == 0 && threadIdx.x == 0 && p.shares != nullptr) {
        const int64_t tile_id = (static_cast<int64_t>(now.b) * p.cache.heads_kv + hk) * p.row_tiles + rt;
        const int64_t last = ((now.begin + AT_BLOCK_UNITS + now.units) * ctas - 1) / total;  // the CTA of the block's last unit
        p.shares[tile_id] = make_int2(2 * blockIdx.x + (at_start ? 0 : 1), static_cast<int>(last));
    }
    // a warp that gave up has no copy in flight; the others may have one, which its own barrier waits for at the end
    if (__syncthreads_or(gave_up)) {
        if (more && then.mine > 0 && !gave_up) {
            const long long t0 = clock64();
            while (!mbar_try_wait(&bars[0], phases & 1u) && clock64() - t0 < p.wait_limit) {
            }
        }
        return;
    }
    if (!more) return;
    at_start = false;
    now = then;
    fence_proxy_async_smem();  // the join's place is read; copies may follow
    __syncthreads();
    }
}

// Adds the parts of one block of rows, in the order of the keys.  One warp per row; launched to start while the kernel before it ends.
template <int D>
__global__ void __launch_bounds__(128) kv4_attention_join_kernel(const __grid_constant__ AttnParams p) {
    const int rows_of_tile = p.tile_rows;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int row = static_cast<int>(id % rows_of_tile);
    const int64_t tile_id = id / rows_of_tile;
    int rest = static_cast<int>(tile_id / p.row_tiles);
    const int rt = static_cast<int>(tile_id % p.row_tiles);
    const int hk = rest % p.cache.heads_kv, b = rest / p.cache.heads_kv;
    if (b >= p.batch) return;
    const Sequence sq = sequence_of(p, b, &g_kv4_attention_device_status);
    const int gr = rt * rows_of_tile + row;
    if (gr >= sq.n * p.group) return;
    // where the block's parts are: in slices of its own, or in the places of the CTAs that shared it
    int parts = p.splits;
    int64_t first = tile_id * p.splits, second = first + 1, stride = 1;
    if (p.shares != nullptr) {
        const int2 share = p.shares[tile_id];
        parts = parts_of_share(share, p.ctas);
        if (parts == 0) atomicCAS(&g_kv4_attention_device_status, 0, 411);
        if (parts <= 1) return;
        first = share.x, second = share.x / 2 * 2 + 2, stride = 2;
    }
    auto place = [&](int s) { return (s == 0 ? first : second + (s - 1) * stride) * rows_of_tile + row; };
    float m = KV4_NO_REF;
    for (int s = lane; s < parts; s += 32) m = fmaxf(m, p.part_ml[place(s)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    constexpr int PER = D / 32;
    float sum = 0.0f, acc[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = 0.0f;
    for (int s0 = 0; s0 < parts; s0 += 32) {  // lane i weighs slice s0 + i
        float f = 0.0f;
        if (s0 + lane < parts) {
            const float2 ml = p.part_ml[place(s0 + lane)];
            f = ex2(ml.x - m);
            sum = fmaf(ml.y, f, sum);
        }
        const int n = min(32, parts - s0);
        for (int s1 = 0; s1 < n; s1 += 8) {  // eight slices in flight
            float2 x[8][PER / 2];
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int e = 0; e < PER / 2; ++e)
                    x[s][e] = s1 + s < n ? *reinterpret_cast<const float2*>(p.part_o + place(s0 + s1 + s) * D + lane * PER + 2 * e) : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const float w = __shfl_sync(0xffffffffu, f, (s1 + s) & 31);
#pragma unroll
                for (int e = 0; e < PER / 2; ++e) {
                    if (s1 + s < n) acc[2 * e] = fmaf(x[s][e].x, w, acc[2 * e]), acc[2 * e + 1] = fmaf(x[s][e].y, w, acc[2 * e + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t q_row = sq.row0 + gr / p.group;
    const int head = hk * p.group + gr % p.group;
    __nv_bfloat16* out = p.out + q_row * p.ldo + static_cast<int64_t>(head) * D + lane * PER;
#pragma unroll
    for (int e = 0; e < PER; e += 2) *reinterpret_cast<__nv_bfloat162*>(out + e) = __floats2bfloat162_rn(acc[e] * inv, acc[e + 1] * inv);
    if (p.lse != nullptr && lane == 0) p.lse[q_row * p.heads_q + head] = sum == 0.0f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
}

// Which kernel and how the work is cut.  A few rows of a kv head meet the codes as they are, 8 or 16 rows at a time (8 where D is 256:
// its accumulators take the registers), on as many CTAs as are resident at once; beyond, keys and values are brought to f16 in
// shared memory for tcgen05 blocks of 128 rows, or two of them from 129 rows on (D <= 128), in slices where there are few blocks.
AttnShape shape_of(int64_t batch, int64_t max_q, int64_t max_kv, int64_t heads_q, int64_t heads_kv, int64_t head_dim) {
    AttnShape s;
    const int64_t rows = max_q * (heads_q / heads_kv);
    s.tensor = rows > (head_dim <= 128 ? AT_MOST_ROWS : AT_MOST_ROWS_256);
    s.tile_rows = s.tensor ? (rows > 128 && head_dim <= 128 ? 256 : 128) : (rows > 8 && head_dim <= 128 ? 16 : 8);
    s.row_tiles = static_cast<int>((rows + s.tile_rows - 1) / s.tile_rows);
    s.tiles = batch * heads_kv * s.row_tiles;
    s.splits = 1;
    s.ctas = s.tiles;
    if (s.tensor) {  // one block per SM; a slice has at least 512 keys
        const int64_t want = AT_ASSUMED_SMS / (s.tiles > 0 ? s.tiles : 1), most = max_kv / 512;
        s.splits = static_cast<int>(want < most ? want : most);
        if (s.splits < 1) s.splits = 1;
        s.ctas = s.tiles * s.splits;
        s.joined = s.splits > 1;
    } else {
        const int resident = s.tile_rows == 16 || head_dim == 256 ? 2 : head_dim == 128 ? 3 : 4;
        const int64_t unit = head_dim == 256 ? 32 * AT_WARPS : 64 * AT_WARPS, units = s.tiles * (max_kv > unit ? (max_kv + unit - 1) / unit : 1);
        s.ctas = units < AT_ASSUMED_SMS * resident ? units : AT_ASSUMED_SMS * resident;
        s.joined = max_kv > unit;  // else no block has two parts
    }
    return s;
}

size_t parts_of(const AttnShape& s) { return static_cast<size_t>(s.tensor ? s.ctas : 2 * s.ctas) * s.tile_rows; }

template <int D, int NT>
int32_t launch_rows(const AttnParams& p, const AttnShape& s, cudaStream_t stream) {
    auto kern = kv4_attention_kernel<D, NT>;
    using L = AttnSmem<D, NT>;
    if (L::TOTAL > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL) != cudaSuccess) {
        (void)cudaGetLastError();
        return BQ_STATUS_LAUNCH_FAILURE;
    }
    kern<<<static_cast<unsigned>(s.ctas), AT_WARPS * 32, L::TOTAL, stream>>>(p);
    return cudaPeekAtLastError() == cudaSuccess ? BQ_STATUS_OK : BQ_STATUS_LAUNCH_FAILURE;
}

template <int D>
int32_t launch_d(const AttnParams& p, const AttnShape& s, cudaStream_t stream) {
    int32_t st;
    if (s.tensor) {
        st = launch_kv4_prompt(p, s, stream);
    } else if constexpr (D <= 128) {
        st = s.tile_rows == 16 ? launch_rows<D, 2>(p, s, stream) : launch_rows<D, 1>(p, s, stream);
    } else {
        st = launch_rows<D, 1>(p, s, stream);
    }
    if (st != BQ_STATUS_OK || !s.joined) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((s.tiles * s.tile_rows + 3) / 4), 1, 1);
    cfg.blockDim = dim3(128, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kv4_attention_join_kernel<D>, p) != cudaSuccess) {
        (void)cudaGetLastError();
        return BQ_STATUS_LAUNCH_FAILURE;
    }
    return BQ_STATUS_OK;
}

}  // namespace

bool kv4_attention_fits(int32_t batch, int32_t max_q, int32_t max_kv, int32_t heads_q, int32_t heads_kv, int32_t head_dim) {
    if (batch == 0 || max_q == 0) return true;
    const AttnShape s = shape_of(batch, max_q, max_kv, heads_q, heads_kv, head_dim);
    return s.tiles * s.tile_rows <= 0x7fffffff && s.ctas <= 0x7fffffff;
}

size_t kv4_attention_workspace_bytes(int32_t batch, int32_t max_q, int32_t max_kv, int32_t heads_q, int32_t heads_kv,
                                     int32_t head_dim) {
    const AttnShape s = shape_of(batch, max_q, max_kv, heads_q, heads_kv, head_dim);
    if (!s.joined) return 0;
    return parts_of(s) * (head_dim + 2) * 4 + (s.tensor ? 0 : static_cast<size_t>(s.tiles) * sizeof(int2));
}

int32_t launch_kv4_attention(const Kv4AttentionDesc& g, cudaStream_t stream) {
    const AttnShape s = shape_of(g.batch, g.max_q, g.max_kv, g.heads_q, g.cache.heads_kv, g.cache.head_dim);
    AttnParams p;
    p.q = static_cast<const __nv_bfloat16*>(g.q);
    p.ldq = g.ldq;
    p.cu_q = g.cu_q;
    p.cache = g.cache;
    p.table = g.page_table;
    p.ld_table = g.ld_table;
    p.kv_lens = g.kv_lens;
    p.out = static_cast<__nv_bfloat16*>(g.out);
    p.ldo = g.ldo;
    p.lse = g.lse;
    p.scale_log2 = static_cast<float>(static_cast<double>(g.scale) * 1.4426950408889634);
    p.causal = g.causal;
    p.back = (g.window > 0 ? g.window : 0x7fffffff) - 1;
    p.batch = g.batch;
    p.total_q = g.total_q;
    p.max_q = g.max_q;
    p.max_kv = g.max_kv;
    p.heads_q = g.heads_q;
    p.group = g.heads_q / g.cache.heads_kv;
    p.row_tiles = s.row_tiles;
    p.splits = s.splits;
    p.tile_rows = s.tile_rows;
    p.ctas = static_cast<int32_t>(s.ctas);
    p.stall = t_wait_selftest != 0;
    p.wait_limit = p.stall ? t_wait_selftest : KV4_WAIT_LIMIT;
    p.part_o = static_cast<float*>(g.workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + parts_of(s) * g.cache.head_dim);
    p.shares = s.tensor || !s.joined ? nullptr : reinterpret_cast<int2*>(p.part_ml + parts_of(s));
    switch (g.cache.head_dim) {
        case 64: return launch_d<64>(p, s, stream);
        case 128: return launch_d<128>(p, s, stream);
        case 256: return launch_d<256>(p, s, stream);
        default: return BQ_STATUS_UNSUPPORTED;
    }
}

int32_t set_kv4_wait_selftest(int64_t limit_cycles) {
    // long enough for every copy in flight to arrive meanwhile, a sixth of a second at most
    if (limit_cycles != 0 && (limit_cycles < (1LL << 20) || limit_cycles > (1LL << 28))) return BQ_STATUS_INVALID_PROBLEM;
    t_wait_selftest = limit_cycles;
    return BQ_STATUS_OK;
}

int32_t read_and_clear_kv4_attention_device_status() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_kv4_attention_device_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) {
        int zero = 0;
        (void)cudaMemcpyToSymbol(g_kv4_attention_device_status, &zero, sizeof(int));
    }
    const int prompt = read_and_clear_kv4_prompt_device_status();
    return v != 0 ? v : prompt;
}

}  // namespace bq
