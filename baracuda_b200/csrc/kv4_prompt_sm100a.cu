// Attention of many query rows (prompts, chunks of them, batches of drafted tokens) over the 4-bit cache: the formulas of
// kv4_attention_sm100a.cu on tcgen05.
//
// A CTA takes 128 or 256 rows (query index x head of the kv head's group) of one sequence and kv head and walks the keys in
// steps of KT.  Keys and values become f16 in shared memory once per step, for all rows:
//   k'[t] = f16(s * c + m), one fused operation per pair; the keys' channels keep the order in which the masks leave them
//   (0 4 1 5 2 6 3 7 of each 8), which the queries are given too: a product does not mind.
//   v' likewise, but stored by channel with the tokens in a row, as the masks leave pairs of tokens: both products have
//   operands whose contraction index is contiguous, in the 128-byte swizzle.
// S = Q K'^T (f16 x f16 -> f32 in TMEM), one softmax thread per row reads S, writes P (f16) over it in TMEM, O += P V' with P as
// the operand from TMEM; Q too lies in TMEM where that has room, which spares shared memory 128 x D x 2 bytes a step.  Queries
// are brought to f16 by a power of two per row (exact unless 2^-38 of the row's largest).
// Roundings to 16 bits: k', v' and P, 2^-11 each, and the output.
// The softmax reads S once: a row's reference moves only when a score exceeds it by 2^SLACK, and only then S is read again and O
// rescaled (TMEM -> registers -> TMEM).  Steps that a mask or a NaN touches read S twice, first for the maximum.
//
// Two row blocks (256 rows, D <= 128): while one block's softmax runs, the tensor core works on the other.  One row block
// (128 rows; D = 256, or few rows): S is double-buffered instead, the next step's S is computed under this step's softmax.
// Warps: 4 softmax warps per row block, 8 (D = 256: 16) bring keys and values to f16, one issues the MMAs.
// Every mbarrier wait is bounded (status 412..416).
//
// Measured (B200): 4096 rows x 32 heads on 8, D = 128, causal: 175 us, 0.78 PFLOP/s of the products that the mask leaves.  The tensor
// core is busy 38 % of the time: the chain S -> P -> O of a row block takes 4400 clocks a step, 2150 of them the softmax of two
// warps per quarter of an SM, which share its issue slots with the feeding warps.  2048 rows x 16 heads on 2, D = 256, window
// 4096: 293 us; there the steps wait for the feeding warps (issue slots 62 % busy; 16 of them: 315 -> 294 us), and the blocks of equal
// length leave the last wave of three a third full.  A sequence of one row among prompts is walked by one CTA per kv head, 18 ns a key:
// the launcher goes by the longest sequence's rows.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>

#include "../../include/baracuda_kernels_q.h"
#include "kv4_attention.cuh"

namespace bq {

namespace {

__device__ int g_kv4_prompt_device_status = 0;

constexpr float PR_SLACK = 7.0f;  // p <= 2^(SLACK + LIFT) stays within f16
// of 8 pairs of exponentials one comes from the polynomial: prompts of 4096 tokens took 190.3 us with none, 186.2 with 1 of 8, 188.4
// with 1 of 4, 204 with 1 of 2
constexpr int PR_POLY_MASK = 14, PR_POLY_AT = 2;
constexpr float PR_LIFT = 8.0f;   // f16's range below the reference: 2^-22 in full precision

template <int D, int NQ>
struct PromptCfg {
    static constexpr int KT = D == 256 ? 64 : 128;  // keys of a step
    static constexpr int SOFTMAX_WARPS = 4 * NQ;
    static constexpr int FEED_WARPS = D == 256 ? 16 : 8;
    static constexpr int SHARES = FEED_WARPS / (KT / KV4_TILE);  // of a tile of 16 keys: whole tiles, or a group of its channels each
    static constexpr int MMA_WARP = SOFTMAX_WARPS + FEED_WARPS;
    static constexpr int THREADS = (MMA_WARP + 1) * 32;
    // 17 or 21 warps leave 96 or 80 registers a thread at launch, and, the feeding warps hand some of theirs to the softmax warps
    static constexpr bool SPLIT_REGS = NQ == 2 || D == 256;
    static constexpr int LAUNCH_REGS = D == 256 ? 80 : 96, SOFTMAX_REGS = 128, FEED_REGS = 64;
    static_assert(!SPLIT_REGS || SOFTMAX_WARPS * SOFTMAX_REGS + FEED_WARPS * FEED_REGS + LAUNCH_REGS <= (MMA_WARP + 1) * LAUNCH_REGS,
                  "the shares come out of what the block was launched with");
    static constexpr int Q_BYTES = NQ * 128 * D * 2;
    static constexpr int K_BYTES = KT * D * 2;  // V the same
    static constexpr int K_OFF = Q_BYTES;
    static constexpr int V_OFF = K_OFF + 2 * K_BYTES;
    static constexpr int BAR_OFF = V_OFF + 2 * K_BYTES;
    static constexpr int FLAG_OFF = BAR_OFF + 192;           // [2][dead, nan][FEED_WARPS] halfwords
    static constexpr int FAR_OFF = FLAG_OFF + 2 * 2 * FEED_WARPS * 2;       // [row] f32
    static constexpr int TOTAL = FAR_OFF + NQ * 128 * 4 + 1024;             // + alignment slack
    static constexpr uint32_t S_COL = NQ * D;                // TMEM columns: O of each block, then two S
    static constexpr uint32_t Q_COL = S_COL + 2 * KT;        // then the queries, where there is room for them
    static constexpr bool Q_TMEM = Q_COL + NQ * D / 2 <= 512;
};

struct PromptBars {
    uint64_t kfull[2], vfull[2], kfree[2], vfree[2], sfull[2], pready[2], pvdone[2], qfull, done;
    uint32_t tmem_slot;
    uint32_t abort_word;
};
static_assert(sizeof(PromptBars) <= 192, "fits");

__device__ __forceinline__ void give_up(volatile uint32_t* abort_word, int code) {
    *abort_word = 1u;
    atomicCAS(&g_kv4_prompt_device_status, 0, code);
}

// kind::f16, f16 operands, f32 accumulator, both K-major; A from shared memory or from TMEM.
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x64(uint32_t taddr, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 bytes to shared memory, zeros where there are none.
__device__ __forceinline__ void cp_async16(void* to, const void* from, bool have) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(have ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));  // (a & mask) | bits
    return r;
}
__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }

// 2^x of a pair on the FMA units, x at most 16: n = rint(x), 2^(x - n) by the polynomial of degree 4 that is nearest in relative
// error on [-1/2, 1/2] (Remez exchange; 2.7e-6 with its f32 roundings), n added to the exponent.  Below 2^-125, and of a NaN, the
// result is no more than that.  The special function unit takes 8 clocks for a warp's results, 2048 for 256 rows x 128 keys, so some
// are computed here.
__device__ __forceinline__ float2 ex2_pair(float2 x) {
    const f32x2 magic = both(12582912.0f, 12582912.0f), back = both(-12582912.0f, -12582912.0f);  // 1.5 * 2^23
    const f32x2 v = both(fmaxf(x.x, -125.0f), fmaxf(x.y, -125.0f));
    const f32x2 t = add2(v, magic);
    const f32x2 f = sub2(v, add2(t, back));
    f32x2 p = both(0.009570102207362652f, 0.009570102207362652f);
    p = fma2(p, f, both(0.05591785907745361f, 0.05591785907745361f));
    p = fma2(p, f, both(0.240247443318367f, 0.240247443318367f));
    p = fma2(p, f, both(0.6931217908859253f, 0.6931217908859253f));
    p = fma2(p, f, both(0.9999992847442627f, 0.9999992847442627f));
    const float2 r = each(p), n = each(t);
    return make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(n.x) << 23)), __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(n.y) << 23)));
}

// The 8 codes of a word as 4 pairs of f16 values s * c + m: pairs (0, 4), (1, 5), (2, 6), (3, 7), where nibbles 0, 2, 4, 6 take
// (s, m) of `even` and 1, 3, 5, 7 the same (keys: one scale; values: nibble parity is a channel, the pair two tokens, and the
// shifted half two further tokens, hence four parameters).
__device__ __forceinline__ void expand(uint32_t w, __half2 s_lo, __half2 m_lo, __half2 s_hi, __half2 m_hi, uint32_t (&out)[4]) {
    const uint32_t w8 = w >> 8;
    const __half2 k1024 = as_h2(0xe400e400u), k16 = as_h2(0x2c002c00u), k64 = as_h2(0xd400d400u);  // -1024, 1 / 16, -64
    // 1024 + c and 1024 + 16 c as f16, then c, both exact
    const __half2 c0 = __hadd2(as_h2(lop_and_or(w, 0x000f000fu, 0x64006400u)), k1024);
    const __half2 c1 = __hfma2(as_h2(lop_and_or(w, 0x00f000f0u, 0x64006400u)), k16, k64);
    const __half2 c2 = __hadd2(as_h2(lop_and_or(w8, 0x000f000fu, 0x64006400u)), k1024);
    const __half2 c3 = __hfma2(as_h2(lop_and_or(w8, 0x00f000f0u, 0x64006400u)), k16, k64);
    out[0] = h2(__hfma2(c0, s_lo, m_lo));
    out[1] = h2(__hfma2(c1, s_lo, m_lo));
    out[2] = h2(__hfma2(c2, s_hi, m_hi));
    out[3] = h2(__hfma2(c3, s_hi, m_hi));
}

// Bits of the 32 keys from `key` on that lie in [lo, hi).
__device__ __forceinline__ uint32_t seen_keys(int key, int lo, int hi) {
    const int from = max(lo - key, 0), to = min(hi - key, 32);
    if (to <= 0 || from >= 32) return 0u;
    return (to == 32 ? 0xffffffffu : (1u << to) - 1u) & (0xffffffffu << from);
}

// What a feeding warp's lane holds of a step: codes and (s, m) pairs of the keys r and r + 8, of the values of 2 c, 2 c + 1,
// 8 + 2 c, 9 + 2 c (GW groups of channels).
template <int GW>
struct FeedRegs {
    uint32_t key[2][2 * GW] = {}, key_pair[2][GW] = {};
    uint32_t value[4 * GW] = {}, value_pair[4][GW] = {};
    bool have = false;  // the values' tile
};

template <int D, int NQ>
__global__ void __launch_bounds__(PromptCfg<D, NQ>::THREADS, 1) kv4_prompt_kernel(const __grid_constant__ AttnParams p) {
    using C = PromptCfg<D, NQ>;
    constexpr int KT = C::KT;
    constexpr int G = D / KV4_GROUP;
    constexpr int W = D >= 128 ? 2 : 1;
    constexpr int TILE = kv4_tile_bytes(D);
    constexpr int ROWS = 128 * NQ;
    extern __shared__ uint8_t pr_smem_raw[];
    uint8_t* smem = pr_smem_raw + ((1024u - (smem_u32(pr_smem_raw) & 1023u)) & 1023u);
    PromptBars* bar = reinterpret_cast<PromptBars*>(smem + C::BAR_OFF);
    volatile uint32_t* abort_word = &bar->abort_word;
    constexpr int FLAGS = 2 * C::FEED_WARPS;
    uint16_t* flags = reinterpret_cast<uint16_t*>(smem + C::FLAG_OFF);  // [stage][dead, nan][feeding warp], a bit per key
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // blocks of late rows see the most keys: they go first
    int id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int pairs = p.batch * p.cache.heads_kv;
    const int rt = p.row_tiles - 1 - id / pairs;
    id %= pairs;
    const int hk = id % p.cache.heads_kv, b = id / p.cache.heads_kv;
    const int64_t tile_id = (static_cast<int64_t>(b) * p.cache.heads_kv + hk) * p.row_tiles + rt;
    const Sequence sq = sequence_of(p, b, &g_kv4_prompt_device_status);
    const int all_rows = sq.n * p.group;
    const int rows = min(ROWS, all_rows - rt * ROWS);
    if (rows <= 0) return;
    const int past = sq.len - sq.n;
    const int i_first = rt * ROWS / p.group, i_last = (rt * ROWS + rows - 1) / p.group;
    const int hi_all = max(0, p.causal ? min(sq.len, past + i_last + 1) : sq.len);
    const int lo_all = first_seen(p, past + i_first);
    const int step0 = lo_all / KT, steps = max(0, (hi_all + KT - 1) / KT - step0);
    const int per = (steps + p.splits - 1) / p.splits;
    const int begin = step0 + min(split * per, steps);
    const int n = max(0, min(per, steps - split * per));

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bar->kfull[s], C::FEED_WARPS);
            mbar_init(&bar->vfull[s], C::FEED_WARPS + p.stall);
            mbar_init(&bar->kfree[s], 1);
            mbar_init(&bar->vfree[s], 1);
            mbar_init(&bar->sfull[s], 1);
            mbar_init(&bar->pready[s], 4);
            mbar_init(&bar->pvdone[s], 1);
        }
        mbar_init(&bar->qfull, C::SOFTMAX_WARPS);
        mbar_init(&bar->done, 1);
        bar->abort_word = 0u;
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    if (warp == C::MMA_WARP) {
        tmem_alloc(&bar->tmem_slot, 512);
        tmem_relinquish_alloc_permit();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = bar->tmem_slot;

    if (warp < C::SOFTMAX_WARPS) {
        if constexpr (C::SPLIT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
        // ---------------------------------------------------------------- softmax: one thread per row
        const int t = warp >> 2;                         // row block
        const int in_block = threadIdx.x & 127;
        const int row = rt * ROWS + t * 128 + in_block;  // of the sequence and kv head
        const bool there = row < all_rows;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 TMEM lanes
        const int i = row / p.group;
        const int hi = !there ? 0 : p.causal ? max(0, min(sq.len, past + i + 1)) : sq.len;
        const int lo = first_seen(p, past + i);
        // this warp's 32 query rows: D / 8 lanes copy one to shared memory, all copies in flight; then each thread brings its row
        // to f16 by a power of two, to TMEM or back to its place
        const int64_t q_row = sq.row0 + (there ? i : 0);
        const int head = hk * p.group + (there ? row % p.group : 0);
        constexpr int LPR = D / 8, RPI = 32 / LPR;  // lanes of a row, rows of a copy
        uint8_t* q_smem = smem + t * 128 * D * 2;
        auto chunk = [&](int at, int w) { return q_smem + (w >> 3) * (128 * 128) + at * 128 + (((w & 7) ^ (at & 7)) << 4); };
#pragma unroll 8
        for (int y = 0; y < LPR; ++y) {
            const int from = y * RPI + lane / LPR;  // of the warp's 32
            const int rr = __shfl_sync(0xffffffffu, static_cast<int>(q_row), from), hh = __shfl_sync(0xffffffffu, head, from);
            const bool have = __shfl_sync(0xffffffffu, static_cast<int>(there), from) != 0;
            cp_async16(chunk((warp & 3) * 32 + from, lane % LPR), have ? p.q + rr * p.ldq + static_cast<int64_t>(hh) * D + lane % LPR * 8 : p.q, have);
        }
        cp_async_wait_all();
        __syncwarp();
        uint32_t top2 = 0u;  // of |x|, the even and the odd channels
#pragma unroll 8
        for (int w = 0; w < LPR; ++w) {
            const uint4 v = *reinterpret_cast<const uint4*>(chunk(in_block, w));
            top2 = max_bf16x2(top2, max_bf16x2(max_bf16x2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), max_bf16x2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
        }
        const uint32_t top = max(top2 & 0xffffu, top2 >> 16);
        const int ex = top == 0u || top >= 0x7f80u ? 0 : max(-100, static_cast<int>(top >> 7) - 127 - 14);  // at most 113
        const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23) * (p.scale_log2 < 0.0f ? -1.0f : 1.0f);
#pragma unroll 1
        for (int x = 0; x < D / 64; ++x) {
            uint32_t h[32];
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const uint4 u = *reinterpret_cast<const uint4*>(chunk(in_block, 8 * x + w));
                const uint32_t v[4] = {u.x, u.y, u.z, u.w};
                float f[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[2 * e] = __uint_as_float(v[e] << 16) * down, f[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u) * down;
#pragma unroll
                for (int e = 0; e < 4; ++e) h[4 * w + e] = pack_half2(f[e], f[e + 4]);
                if constexpr (!C::Q_TMEM)
                    *reinterpret_cast<uint4*>(chunk(in_block, 8 * x + w)) = make_uint4(h[4 * w], h[4 * w + 1], h[4 * w + 2], h[4 * w + 3]);
            }
            if constexpr (C::Q_TMEM) tmem_st_32x32b_x32(tmem + lanes + C::Q_COL + t * (D / 2) + 32 * x, h);
        }
        if constexpr (C::Q_TMEM) {
            tmem_st_wait();
            tc_fence_before_sync();
        } else {
            fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->qfull);
        const float factor = fminf(fmaxf(__uint_as_float(static_cast<uint32_t>(127 + ex) << 23) * fabsf(p.scale_log2), 1.0e-37f), FLT_MAX);

        // rows of this block that exist see at least [lo_max, hi_min)
        const int last_there = min(all_rows, rt * ROWS + t * 128 + 128) - 1;  // may lie before the block's first row
        const int first_i = (rt * ROWS + t * 128) / p.group, last_i = last_there / p.group;
        const int hi_min = p.causal ? min(sq.len, past + first_i + 1) : sq.len;
        const int lo_max = first_seen(p, past + last_i);
        const uint32_t o_tmem = tmem + lanes + t * D;
        // The product of step j with the values completes a phase of its score slot's barrier.  A warp of the block may be a whole step
        // ahead of another (one row block: S(j + 1) is there before P(j) is), never two: S(j) is issued after the product of step j
        // less the number of slots, so a slot's barrier is at most in the phase that is waited for, and its parity tells.
        auto pv_slot = [&](int j) { return NQ == 2 ? t : j & 1; };
        auto pv_parity = [](int j) { return static_cast<uint32_t>(NQ == 2 ? j : j >> 1) & 1u; };
        // A reference beyond KV4_FAR lies in shared memory, with KV4_NO_REF in its place: such a row takes the path that reads S twice in
        // every step, where its scores are brought down to that size, so that one operation is exact enough for them (the keys that this
        // brings near the first are those whose scores the roundings of their operands could have exchanged).
        float* far_ref = reinterpret_cast<float*>(smem + C::FAR_OFF) + t * 128 + in_block;
        *far_ref = KV4_NO_REF;
        float ref = KV4_NO_REF, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            const int slot = NQ == 2 ? t : j & 1;
            const uint32_t slot_parity = (NQ == 2 ? j : j >> 1) & 1;
            const uint32_t s_tmem = tmem + lanes + C::S_COL + slot * KT;
            if (!mbar_wait_bounded(&bar->vfull[j & 1], (j >> 1) & 1, abort_word, p.wait_limit) ||
                !mbar_wait_bounded(&bar->sfull[slot], slot_parity, abort_word, p.wait_limit)) {
                give_up(abort_word, 412);
                ok = false;
            }
            if (!__all_sync(0xffffffffu, ok)) break;
            ok = true;
            tc_fence_after_sync();
            const int key0 = (begin + j) * KT;
            // keys that hold nothing (no page) and keys whose values are NaN, one bit each
            const uint32_t* gone = reinterpret_cast<const uint32_t*>(flags + (j & 1) * FLAGS);
            const uint32_t* nans = gone + FLAGS / 4;
            uint32_t any = 0u;
#pragma unroll
            for (int x = 0; x < FLAGS / 8; ++x) {
                const uint4 f = reinterpret_cast<const uint4*>(gone)[x];
                any |= f.x | f.y | f.z | f.w;
            }
            auto bits_of = [](const uint32_t* w, int x) {  // of keys 32 x .. 32 x + 31
                if constexpr (C::SHARES == 1) {
                    return w[x];
                } else {
                    static_assert(C::SHARES == 4, "two words a tile");
                    const uint32_t a = w[4 * x] | w[4 * x + 1], b = w[4 * x + 2] | w[4 * x + 3];
                    return ((a | (a >> 16)) & 0xffffu) | ((b | (b << 16)) & 0xffff0000u);
                }
            };
            const bool edge = key0 + KT > hi_min || key0 < lo_max || any != 0u;
            const f32x2 factor2 = both(factor, factor);
            float mx = -INFINITY;
            bool done = false;
            if (!edge) {
                // the common step in one reading: P with the reference as it is, and the maximum that tells whether it holds; P goes
                // over S only then
                const f32x2 base2 = both(PR_LIFT - ref, PR_LIFT - ref);
                f32x2 sum[2] = {0ull, 0ull}, nan2 = 0ull;  // nan2: 0, or NaN for a NaN among the polynomial's scores; the row's sum takes it over
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                uint32_t pk[KT / 32][16];
                constexpr int CH = D == 256 ? 32 : 64;
#pragma unroll
                for (int x = 0; x < KT / CH; ++x) {
                    uint32_t v[CH];
                    if constexpr (CH == 64) {
                        tmem_ld_32x32b_x64(s_tmem + CH * x, v);
                    } else {
                        tmem_ld_32x32b_x32(s_tmem + CH * x, v);
                    }
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < CH; e += 2) {
                        const float s0 = __uint_as_float(v[e]), s1 = __uint_as_float(v[e + 1]);
                        m4[(e >> 1) & 3] = fmaxf(fmaxf(m4[(e >> 1) & 3], s0), s1);
                        const float2 w = each(fma2(both(s0, s1), factor2, base2));
                        const float2 pr = (e & PR_POLY_MASK) == PR_POLY_AT ? ex2_pair(w) : make_float2(ex2(w.x), ex2(w.y));
                        sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], both(pr.x, pr.y));
                        if ((e & PR_POLY_MASK) == PR_POLY_AT) nan2 = fma2(both(s0, s1), 0ull, nan2);  // the polynomial makes a number of a NaN
                        pk[CH / 32 * x + (e >> 5)][(e & 31) / 2] = pack_half2(pr.x, pr.y);
                    }
                }
                mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * factor;
                if (!__any_sync(0xffffffffu, mx > ref + PR_SLACK)) {
                    done = true;
#pragma unroll
                    for (int x = 0; x < KT / 32; ++x) tmem_st_32x32b_x16(s_tmem + 16 * x, pk[x]);
                    const float2 total = each(add2(add2(sum[0], sum[1]), nan2));
                    l += total.x + total.y;
                }
            } else {
#pragma unroll 1
                for (int x = 0; x < KT / 32; ++x) {
                    uint32_t s[32];
                    tmem_ld_32x32b_x32(s_tmem + 32 * x, s);
                    tmem_ld_wait();
                    const uint32_t seen = seen_keys(key0 + 32 * x, lo, hi) & ~bits_of(gone, x);
#pragma unroll
                    for (int e = 0; e < 32; ++e) mx = fmaxf(mx, ((seen >> e) & 1u) ? __uint_as_float(s[e]) : -INFINITY);
                }
                mx *= factor;
            }
            if (!done) {
                float shrink = 1.0f, slow_ref = ref;
                if (__any_sync(0xffffffffu, mx > ref + PR_SLACK)) {
                    float fix = 1.0f;
                    if (mx > ref + PR_SLACK) {
                        const float from = ref > KV4_NO_REF ? ref : *far_ref, to = fmaxf(from, mx);
                        const bool far = fabsf(to) > KV4_FAR;
                        if (far) *far_ref = to, shrink = KV4_FAR / fabsf(to);
                        ref = far ? KV4_NO_REF : to;
                        slow_ref = to * shrink;
                        fix = ex2((from - to) * shrink);
                    }
                    l *= fix;
                    if (j > 0) {
                        if (!mbar_wait_bounded(&bar->pvdone[pv_slot(j - 1)], pv_parity(j - 1), abort_word, p.wait_limit)) {
                            give_up(abort_word, 413);
                            ok = false;
                        }
                        if (!__all_sync(0xffffffffu, ok)) break;
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int x = 0; x < D / 32; ++x) {
                            uint32_t s[32];
                            tmem_ld_32x32b_x32(o_tmem + 32 * x, s);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * fix);
                            tmem_st_32x32b_x32(o_tmem + 32 * x, s);
                        }
                        tmem_st_wait();
                    }
                }
                const f32x2 slow2 = both(factor * shrink, factor * shrink), base2 = both(PR_LIFT - slow_ref, PR_LIFT - slow_ref);
                f32x2 sum[2] = {0ull, 0ull};
#pragma unroll 1
                for (int x = 0; x < KT / 32; ++x) {
                    uint32_t s[32];
                    tmem_ld_32x32b_x32(s_tmem + 32 * x, s);
                    tmem_ld_wait();
                    const uint32_t seen = seen_keys(key0 + 32 * x, lo, hi) & ~bits_of(gone, x), bad = bits_of(nans, x);
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float2 v = each(fma2(both(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), slow2, base2));
                        v.x = ((seen >> e) & 1u) == 0u ? -INFINITY : ((bad >> e) & 1u) ? NAN : v.x;
                        v.y = ((seen >> (e + 1)) & 1u) == 0u ? -INFINITY : ((bad >> (e + 1)) & 1u) ? NAN : v.y;
                        const float p0 = ex2(v.x), p1 = ex2(v.y);
                        sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], both(p0, p1));
                        pk[e / 2] = pack_half2(p0, p1);
                    }
                    tmem_st_32x32b_x16(s_tmem + 16 * x, pk);  // over columns that have been read
                }
                const float2 total = each(add2(sum[0], sum[1]));
                l += total.x + total.y;
            }
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->pready[slot]);
        }
        // ---------------------------------------------------------------- output
        if (n > 0 && ok && *abort_word == 0u) {
            if (!mbar_wait_bounded(&bar->pvdone[pv_slot(n - 1)], pv_parity(n - 1), abort_word, p.wait_limit)) {
                give_up(abort_word, 414);
                ok = false;
            }
            tc_fence_after_sync();
        }
        ok = __all_sync(0xffffffffu, ok && *abort_word == 0u);
        if (ok) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t part = (tile_id * p.splits + split) * ROWS + t * 128 + in_block;
            // the queries are no longer needed (of any warp: the last MMA is over, or, where there was none, the block's warps have
            // written theirs): their place takes this warp's output rows (bf16, or half of an f32 row at a time), and whole rows
            // leave from there
            if (n == 0) named_bar_sync(1 + t, 128);
            constexpr int CHUNKS = D / 8;  // of 16 bytes in a row
            auto place = [&](int r_, int w) { return q_smem + ((warp & 3) * 32 + r_) * (D * 2) + ((w ^ (r_ & 7)) << 4); };
            const bool direct = p.splits == 1;
#pragma unroll 1
            for (int half = 0; half < (direct ? 1 : 2); ++half) {
#pragma unroll 1
                for (int x = direct ? 0 : half * (D / 64); x < (direct ? D / 32 : (half + 1) * (D / 64)); ++x) {
                    uint32_t o[32];
                    if (n > 0) {
                        tmem_ld_32x32b_x32(o_tmem + 32 * x, o);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0u;
                    }
                    if (direct) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint32_t v[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(o[e + 2 * y]) * inv, __uint_as_float(o[e + 2 * y + 1]) * inv);
                                v[y] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                            *reinterpret_cast<uint4*>(place(lane, 4 * x + e / 8)) = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<uint4*>(place(lane, 8 * (x - half * (D / 64)) + e / 4)) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
                __syncwarp();
#pragma unroll 4
                for (int y = 0; y < CHUNKS; ++y) {  // 32 chunks at a time
                    const int from = (y * 32 + lane) / CHUNKS, w = lane % CHUNKS;
                    const int rr = __shfl_sync(0xffffffffu, static_cast<int>(q_row), from), hh = __shfl_sync(0xffffffffu, head, from);
                    const bool have = __shfl_sync(0xffffffffu, static_cast<int>(there), from) != 0;
                    const uint4 v = *reinterpret_cast<const uint4*>(place(from, w));
                    if (have && direct) {
                        *(reinterpret_cast<uint4*>(p.out + rr * p.ldo + static_cast<int64_t>(hh) * D) + w) = v;
                    } else if (have) {
                        *(reinterpret_cast<uint4*>(p.part_o + (part - lane + from) * D + half * (D / 2)) + w) = v;
                    }
                }
                __syncwarp();
            }
            if (there) {
                const float m = l == 0.0f ? KV4_NO_REF : (ref > KV4_NO_REF ? ref : *far_ref) - PR_LIFT;
                if (p.splits > 1) {
                    p.part_ml[part] = make_float2(m, l);
                } else if (p.lse != nullptr) {
                    p.lse[q_row * p.heads_q + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
                }
            }
        }
    } else if (warp < C::MMA_WARP) {
        if constexpr (C::SPLIT_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::FEED_REGS));
        // ---------------------------------------------------------------- keys and values to f16
        // a warp's share of a step: one tile of 16 keys, or half of its channels (groups g0 .. g0 + GW - 1)
        constexpr int STEP_TILES = KT / KV4_TILE, GW = G / C::SHARES;
        const int feeder = warp - C::SOFTMAX_WARPS, in_step = feeder / C::SHARES, g0 = feeder % C::SHARES * GW;
        const int r = lane >> 2, c = lane & 3;
        const int32_t* table = p.table + static_cast<int64_t>(b) * p.ld_table;
        const int tiles_per_page = p.cache.page_size / KV4_TILE;
        const uint8_t* head_base = p.cache.base + static_cast<int64_t>(hk) * tiles_per_page * TILE;
        // lane i looks up where this warp's tile lies in the i-th of the next 32 steps
        int64_t ahead = -1;
        auto look_up = [&](int j) {
            const int tile = (begin + j + lane) * STEP_TILES + in_step;
            ahead = -1;
            // a step's first tiles may lie before the first key that a row sees: they need not be anywhere
            if (j + lane < n && tile * KV4_TILE < hi_all && (tile + 1) * KV4_TILE > lo_all) {
                const int at = tile / tiles_per_page, page = table[at];
                if (page >= 0 && page < p.cache.num_pages) {
                    ahead = static_cast<int64_t>(page) * p.cache.page_stride + (tile - at * tiles_per_page) * TILE;
                } else {
                    atomicCAS(&g_kv4_prompt_device_status, 0, 404);
                }
            }
        };
        FeedRegs<GW> h;
        auto place_of = [&](int j) -> const uint8_t* {
            const int64_t where = __shfl_sync(0xffffffffu, ahead, j & 31);
            return where < 0 ? nullptr : head_base + where;
        };
        auto load_keys = [&](int j) {
            if ((j & 31) == 0) look_up(j);
            const uint8_t* at = place_of(j);
            if (at == nullptr) return;  // whatever is in the registers: these keys are masked
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if constexpr (W == 2 && GW == 1) {
                    const uint2 v = *reinterpret_cast<const uint2*>(at + (g0 >> 1) * 1024 + e * 512 + lane * 16 + (g0 & 1) * 8);
                    h.key[e][0] = v.x, h.key[e][1] = v.y;
                    h.key_pair[e][0] = *reinterpret_cast<const uint32_t*>(at + kv4_pair_offset(D, 0) + ((r + 8 * e) * G + g0) * 4);
                } else if constexpr (W == 2) {
#pragma unroll
                    for (int x = 0; x < GW / 2; ++x) {
                        const uint4 v = *reinterpret_cast<const uint4*>(at + (g0 / 2 + x) * 1024 + e * 512 + lane * 16);
                        h.key[e][4 * x] = v.x, h.key[e][4 * x + 1] = v.y, h.key[e][4 * x + 2] = v.z, h.key[e][4 * x + 3] = v.w;
                    }
                    const uint2 v = *reinterpret_cast<const uint2*>(at + kv4_pair_offset(D, 0) + ((r + 8 * e) * G + g0) * 4);
                    h.key_pair[e][0] = v.x, h.key_pair[e][1] = v.y;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(at + e * 256 + lane * 8);
                    h.key[e][0] = v.x, h.key[e][1] = v.y;
                    h.key_pair[e][0] = *reinterpret_cast<const uint32_t*>(at + kv4_pair_offset(D, 0) + (r + 8 * e) * 4);
                }
            }
        };
        auto load_values = [&](int j) {
            const uint8_t* at = place_of(j);
            h.have = at != nullptr;
            if (!h.have) return;  // as above: zeroed below
#pragma unroll
            for (int g = 0; g < GW; ++g) {
                const uint4 v = *reinterpret_cast<const uint4*>(at + 8 * D + (g0 + g) * 512 + lane * 16);
                h.value[4 * g] = v.x, h.value[4 * g + 1] = v.y, h.value[4 * g + 2] = v.z, h.value[4 * g + 3] = v.w;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint8_t* pair = at + kv4_pair_offset(D, 1) + ((2 * c + (e & 1) + 8 * (e >> 1)) * G + g0) * 4;
                if constexpr (GW == 2) {
                    const uint2 v = *reinterpret_cast<const uint2*>(pair);
                    h.value_pair[e][0] = v.x, h.value_pair[e][1] = v.y;
                } else {
                    h.value_pair[e][0] = *reinterpret_cast<const uint32_t*>(pair);
                }
            }
        };
        auto convert_keys = [&](uint8_t* k_smem) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint8_t* row = k_smem + (in_step * KV4_TILE + r + 8 * e) * 128;
#pragma unroll
                for (int g = 0; g < GW; ++g) {
                    const __half2 sm = as_h2(h.key_pair[e][g]), s2 = __low2half2(sm), m2 = __high2half2(sm);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t o[4];
                        expand(h.key[e][2 * g + u], s2, m2, s2, m2, o);
                        *reinterpret_cast<uint4*>(row + (g0 + g) * (KT * 128) + (((2 * c + u) ^ r) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
        };
        auto convert_values = [&](uint8_t* v_smem, int j, int stage) {
            const int key0 = (begin + j) * KT + in_step * KV4_TILE;
            // values of keys that are not there, and NaN values, are zeroed: a zero weight times NaN would reach every row
            uint32_t top = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int g = 0; g < GW; ++g) top |= (h.value_pair[e][g] & 0x7c007c00u) + 0x04000400u;  // sign bits: an exponent of ones
            uint32_t nan_bits = 0u;
            if (__any_sync(0xffffffffu, (top & 0x80008000u) != 0u || key0 + KV4_TILE > sq.len || !h.have)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int tok = 2 * c + (e & 1) + 8 * (e >> 1);
                    uint32_t ones = 0u;
#pragma unroll
                    for (int g = 0; g < GW; ++g) ones |= (h.value_pair[e][g] & 0x7c007c00u) + 0x04000400u;
                    const bool beyond = key0 + tok >= sq.len || !h.have, nan = (ones & 0x80008000u) != 0u;
                    if (beyond || nan) {
#pragma unroll
                        for (int g = 0; g < GW; ++g) h.value_pair[e][g] = 0u;
                    }
                    if (nan && !beyond) nan_bits |= 1u << tok;
                }
                nan_bits |= __shfl_xor_sync(0xffffffffu, nan_bits, 1);
                nan_bits |= __shfl_xor_sync(0xffffffffu, nan_bits, 2);
            }
            if (lane == 0) {
                flags[stage * FLAGS + feeder] = h.have || key0 >= hi_all ? 0u : 0xffffu;
                flags[stage * FLAGS + C::FEED_WARPS + feeder] = static_cast<uint16_t>(nan_bits);
            }
            uint8_t* row = v_smem + (in_step >> 2) * (D * 128) + r * 128 + 4 * c;
            const int at0 = ((2 * (in_step & 3)) ^ r) << 4, at1 = ((2 * (in_step & 3) + 1) ^ r) << 4;
#pragma unroll
            for (int g = 0; g < GW; ++g) {
                const __half2 t0 = as_h2(h.value_pair[0][g]), t1 = as_h2(h.value_pair[1][g]), t2 = as_h2(h.value_pair[2][g]), t3 = as_h2(h.value_pair[3][g]);
                const __half2 s_lo = __lows2half2(t0, t1), m_lo = __highs2half2(t0, t1), s_hi = __lows2half2(t2, t3), m_hi = __highs2half2(t2, t3);
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    uint32_t o[4];  // (channel r, tokens 2 c ..), (r + 8, 2 c ..), (r, 8 + 2 c ..), (r + 8, 8 + 2 c ..)
                    expand(h.value[4 * g + jj], s_lo, m_lo, s_hi, m_hi, o);
                    uint8_t* to = row + (64 * (g0 + g) + 16 * jj) * 128;
                    *reinterpret_cast<uint32_t*>(to + at0) = o[0];
                    *reinterpret_cast<uint32_t*>(to + 8 * 128 + at0) = o[1];
                    *reinterpret_cast<uint32_t*>(to + at1) = o[2];
                    *reinterpret_cast<uint32_t*>(to + 8 * 128 + at1) = o[3];
                }
            }
        };
        // the next step's keys are on their way under this step's values, and the other way round; a step further ahead, in
        // registers, was slower (16 warps of D = 256 with two steps each: 294 -> 310 us)
        auto step = [&](int j) -> bool {
            const int stage = j & 1;
            bool ok = true;
            if (j >= 2 && !mbar_wait_bounded(&bar->kfree[stage], ((j >> 1) - 1) & 1, abort_word, p.wait_limit)) {
                give_up(abort_word, 415);
                ok = false;
            }
            if (!__all_sync(0xffffffffu, ok)) return false;
            convert_keys(smem + C::K_OFF + stage * C::K_BYTES);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->kfull[stage]);
            // the look-up of the next 32 steps must not replace what earlier steps' values still go by: they are loaded already
            if (j + 1 < n) load_keys(j + 1);
            if (j >= 2 && !mbar_wait_bounded(&bar->vfree[stage], ((j >> 1) - 1) & 1, abort_word, p.wait_limit)) {
                give_up(abort_word, 415);
                ok = false;
            }
            if (!__all_sync(0xffffffffu, ok)) return false;
            convert_values(smem + C::V_OFF + stage * C::K_BYTES, j, stage);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->vfull[stage]);
            if (j + 1 < n) load_values(j + 1);
            return true;
        };
        if (n > 0) load_keys(0), load_values(0);
        for (int j = 0; j < n && step(j); ++j) {
        }
    } else {
        // ---------------------------------------------------------------- MMA issue: the warp walks the steps, one lane issues
        constexpr uint32_t IDESC_S = idesc_f16(128, KT), IDESC_O = idesc_f16(128, D);
        const bool leader = elect_one() != 0u;
        [[maybe_unused]] const uint64_t q_desc = umma_desc_kmajor_sw128(smem_u32(smem));
        const uint64_t k_desc = umma_desc_kmajor_sw128(smem_u32(smem) + C::K_OFF), v_desc = umma_desc_kmajor_sw128(smem_u32(smem) + C::V_OFF);
        bool ok = true;
        auto wait = [&](uint64_t* what, uint32_t parity) {
            if (ok && !mbar_wait_bounded(what, parity, abort_word, p.wait_limit)) {
                give_up(abort_word, 416);
                ok = false;
            }
            ok = __all_sync(0xffffffffu, ok);
            return ok;
        };
        // descriptors count addresses in 16 bytes: a 16-deep slice is 32 bytes on within a 128-byte block of 64
        auto scores = [&](int t, int j, int slot) {
            const uint64_t k = k_desc + (j & 1) * (C::K_BYTES / 16);
            const uint32_t to = tmem + C::S_COL + slot * KT;
            if (leader) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint64_t keys = k + ((ks >> 2) * (KT * 128 / 16) + (ks & 3) * 2);
                    if constexpr (C::Q_TMEM) {
                        umma_f16_ts(to, tmem + C::Q_COL + t * (D / 2) + ks * 8, keys, IDESC_S, ks > 0);
                    } else {
                        umma_f16_ss(to, q_desc + (t * (128 * D * 2 / 16) + (ks >> 2) * (128 * 128 / 16) + (ks & 3) * 2), keys, IDESC_S, ks > 0);
                    }
                }
                umma_commit(&bar->sfull[slot]);
            }
            __syncwarp();
        };
        auto output = [&](int t, int j, int slot) {
            const uint64_t v = v_desc + (j & 1) * (C::K_BYTES / 16);
            const uint32_t to = tmem + t * D, from = tmem + C::S_COL + slot * KT;
            const uint32_t more = j > 0;
            if (leader) {
#pragma unroll
                for (int ks = 0; ks < KT / 16; ++ks)
                    umma_f16_ts(to, from + ks * 8, v + ((ks >> 2) * (D * 128 / 16) + (ks & 3) * 2), IDESC_O, ks > 0 ? 1u : more);
                umma_commit(&bar->pvdone[slot]);
                if (t == NQ - 1) umma_commit(&bar->vfree[j & 1]);
            }
            __syncwarp();
        };
        auto commit = [&](uint64_t* what) {
            if (leader) umma_commit(what);
            __syncwarp();
        };
        if (n > 0 && wait(&bar->qfull, 0)) {
            // A score tile may overwrite the P of an earlier step: MMAs of one thread run in the order of their issue.
            constexpr int ahead = NQ == 2 ? 1 : 2;
            for (int j = 0; j < ahead && j < n && wait(&bar->kfull[j & 1], 0); ++j) {
                tc_fence_after_sync();
                for (int t = 0; t < NQ; ++t) scores(t, j, NQ == 2 ? t : j & 1);
                commit(&bar->kfree[j & 1]);
            }
            for (int j = 0; ok && j < n; ++j) {
                const int next = j + ahead;
                if (!wait(&bar->vfull[j & 1], (j >> 1) & 1)) break;
#pragma unroll
                for (int t = 0; t < NQ; ++t) {
                    const int slot = NQ == 2 ? t : j & 1;
                    if (!wait(&bar->pready[slot], (NQ == 2 ? j : j >> 1) & 1)) break;
                    tc_fence_after_sync();
                    output(t, j, slot);
                    if (next < n) {
                        if (t == 0 && !wait(&bar->kfull[next & 1], (next >> 1) & 1)) break;
                        tc_fence_after_sync();
                        scores(t, next, slot);
                        if (t == NQ - 1) commit(&bar->kfree[next & 1]);
                    }
                }
            }
            // nothing of this thread's may be in flight when the TMEM is given back
            commit(&bar->done);
            const long long t0 = clock64();
            while (!mbar_try_wait(&bar->done, 0u) && clock64() - t0 < p.wait_limit) {
            }
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == C::MMA_WARP) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

template <int D, int NQ>
int32_t launch_prompt(const AttnParams& p, const AttnShape& s, cudaStream_t stream) {
    auto kern = kv4_prompt_kernel<D, NQ>;
    constexpr int bytes = PromptCfg<D, NQ>::TOTAL;
    static_assert(bytes <= 232448, "shared memory of an SM");
    if constexpr (PromptCfg<D, NQ>::SPLIT_REGS) {
        // the warps' shares of the registers are sums over what a launch gets: never start a build that gets another number
        static const bool as_assumed = [kern] {
            cudaFuncAttributes a;
            return cudaFuncGetAttributes(&a, kern) == cudaSuccess && a.numRegs == PromptCfg<D, NQ>::LAUNCH_REGS;
        }();
        if (!as_assumed) return BQ_STATUS_LAUNCH_FAILURE;
    }
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        (void)cudaGetLastError();
        return BQ_STATUS_LAUNCH_FAILURE;
    }
    kern<<<static_cast<unsigned>(s.tiles * s.splits), PromptCfg<D, NQ>::THREADS, bytes, stream>>>(p);
    return cudaPeekAtLastError() == cudaSuccess ? BQ_STATUS_OK : BQ_STATUS_LAUNCH_FAILURE;
}

}  // namespace

int32_t launch_kv4_prompt(const AttnParams& p, const AttnShape& s, cudaStream_t stream) {
    switch (p.cache.head_dim) {
        case 64: return s.tile_rows == 256 ? launch_prompt<64, 2>(p, s, stream) : launch_prompt<64, 1>(p, s, stream);
        case 128: return s.tile_rows == 256 ? launch_prompt<128, 2>(p, s, stream) : launch_prompt<128, 1>(p, s, stream);
        case 256: return launch_prompt<256, 1>(p, s, stream);
        default: return BQ_STATUS_UNSUPPORTED;
    }
}

int32_t read_and_clear_kv4_prompt_device_status() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_kv4_prompt_device_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) {
        int zero = 0;
        (void)cudaMemcpyToSymbol(g_kv4_prompt_device_status, &zero, sizeof(int));
    }
    return v;
}

}  // namespace bq
