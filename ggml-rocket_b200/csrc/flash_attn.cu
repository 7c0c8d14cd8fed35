// FLASH_ATTN_EXT prefill on sm_100a (the reference's ggml_backend_rocket_flash_attn,
// ggml-rocket.cpp:5444-5691, without its gathers, host softmax or range fallback).
//
// Three kernels:
//   q_pack     Q F32 [D, T, H] (strided) -> Q16 [H][T][D] fp16 holding scale*q, with a per-row
//              power-of-two divisor for rows whose scaled values leave fp16's range; the
//              divisor is multiplied back into that row's scores.
//   mask_flags per (token block, 128-key block) of the F16 mask: all -inf (skipped), all zero
//              (no mask loads), or mixed. Causal prefill skips ~half the key blocks.
//   fa_kernel  one CTA per (group of GP query heads that share a KV head, TQ tokens) = 128 query
//              rows. Per key block: S = Q.K^T by tcgen05 into one of two TMEM buffers; 256
//              softmax threads (two per row, 64 keys each, the row max exchanged through shared
//              memory) read S from TMEM once, keep the online max / sum in fp32 (log2 units),
//              write P (fp16) to shared memory; O += P.V by tcgen05 accumulates in TMEM for the
//              whole key range, rescaled in place only when a row max grows by more than 2^8.
//              K and V tiles arrive by TMA straight from the op's strided cache views, two
//              stages deep.
// Further down: the same over a Q4_0 cache and several streams (b200_flash_attn_kvq's larger calls).
#include <algorithm>
#include <cstdint>
#include <cstring>

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "ggml-b200-kernels.h"
#include "internal.h"
#include "ptx.cuh"

namespace b200 {

constexpr int FA_ROWS = 128;      // query rows per CTA (tcgen05 M)
constexpr int FA_KB = 128;        // keys per block (tcgen05 N of Q.K^T, K of P.V)
constexpr int FA_SPLIT = 2;                          // softmax threads per query row
constexpr int FA_SOFTMAX_WARPS = 4 * FA_SPLIT;
constexpr int FA_THREADS = 64 + 32 * FA_SOFTMAX_WARPS;   // warp 0 TMA, warp 1 MMA, then softmax
constexpr float FA_RESCALE_LOG2 = 8.0f;   // rescale O only when the row max grows by more than 2^8
enum : uint8_t { MF_MIXED = 0, MF_ZERO = 1, MF_MASKED = 2 };

// How the query tiles are shared out: CTAs below `whole` take a tile and all its keys; behind them come
// `cut` CTAs a tile, with `per` key blocks each.
struct FaUnits {
    int whole, cut, per;
};

struct FaArgs {
    const float* qscale;       // [H*T] per-row divisor (1 unless out of fp16 range); EXT: [S*H*T], times the scale
    const uint16_t* mask;      // F16 mask or nullptr
    int64_t m_stride;          // mask row stride, elements
    bool mask_vec;             // rows 16-byte aligned: 16-byte loads
    const uint8_t* flags;      // [n_tb][n_kvb]
    float* dst;                // [T][H][DV]
    int T, H, KV, HK, GP, TQ, n_hg, n_tb, n_kvb;
    int S;                     // EXT: streams
    const __half* q16;         // EXT: [S][H][T][D], an f32 q's low halves behind them
    float softcap;
    int* err;
    // the extended form only (several streams, parts of the keys, f16 results; q16 not scaled)
    int64_t m_stream;          // mask stride of a stream, elements
    float scale;
    FaUnits units;
    int dst_f16;
    float* part;               // [unit - whole][rows of a unit][DV] outputs not divided by their sums
    float* stat;               // {max in log2 units, sum, mask value it is relative to} of each of their rows
};

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// cap * tanh(s / cap) within 2^-20 of its value: tanh x = 1 - 2 / (1 + e^2x), whose terms cancel where x is
// small, and there the Taylor series to x^13. The library's tanhf is a call a score at least (inlined into the
// unrolled loop it makes code that the instruction cache does not hold): 2048 tokens x 16384 keys take 4050 us
// with it, 2320 so.
__device__ __forceinline__ float capped(float s, float cap, float inv_cap) {
    const float x = s * inv_cap, x2 = x * x;
    float y = fmaf(x2, 21844.0f / 6081075.0f, -1382.0f / 155925.0f);
    y = fmaf(x2, y, 62.0f / 2835.0f);
    y = fmaf(x2, y, -17.0f / 315.0f);
    y = fmaf(x2, y, 2.0f / 15.0f);
    y = fmaf(x2, y, -1.0f / 3.0f);
    y = fmaf(x2 * x, y, x);
    const float t = ex2_approx(x * 2.885390082f);                    // e^2x
    const float wide = fmaf(-2.0f, __fdividef(1.0f, 1.0f + t), 1.0f);
    return cap * (fabsf(x) < 0.5f ? y : wide);
}

// Shared-memory descriptor of an MN-major operand in 128-byte-swizzled rows: 64 MN elements per
// 128-byte row, rows (K) 128 B apart, 8-row groups 1024 B apart, 64-element MN groups `lbo` apart.
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

__host__ __device__ constexpr uint32_t idesc_f16_f32_bmn(int M, int N) {
    return idesc_f16_f32(M, N) | (1u << 16);   // B operand MN-major
}

// 32 mask values (fp16 bits) of one row starting at key k0; keys at or past KV read as 0
// (the score of such a key is forced to -inf separately).
__device__ __forceinline__ void load_mask32(const uint16_t* mrow, int k0, int KV, bool vec, uint4 (&mv)[4]) {
    if (vec && k0 + 32 <= KV) {
        const uint4* mp = reinterpret_cast<const uint4*>(mrow + k0);
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) mv[q4] = __ldg(mp + q4);
    } else {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            const uint32_t lo = (k0 + e < KV) ? (uint32_t)__ldg(mrow + k0 + e) : 0u;
            const uint32_t hi = (k0 + e + 1 < KV) ? (uint32_t)__ldg(mrow + k0 + e + 1) : 0u;
            w[e >> 1] = lo | (hi << 16);
        }
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) mv[q4] = make_uint4(w[4 * q4], w[4 * q4 + 1], w[4 * q4 + 2], w[4 * q4 + 3]);
    }
}

// ---------------------------------------------------------------------------------------------
// Set-up pass, one launch: CTAs [0, q_ctas) pack Q, one warp per (h, t) row; the rest classify
// the mask, one CTA per (token block, key block). Launched programmatically; the attention
// kernel that follows starts its prologue while this pass drains.
// ---------------------------------------------------------------------------------------------
template <int D>
__device__ __forceinline__ void fa_q_pack_row(const float* __restrict__ q, int64_t q_nb1, int64_t q_nb2, int T,
                                              int H, float scale, __half* __restrict__ q16,
                                              float* __restrict__ qscale, int row, int lane) {
    if (row >= H * T) return;
    const int h = row / T, t = row % T;
    const float* src = reinterpret_cast<const float*>(reinterpret_cast<const char*>(q) + (int64_t)t * q_nb1 +
                                                      (int64_t)h * q_nb2);
    constexpr int PER = D / 32;
    float x[PER];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        x[i] = scale * __ldg(src + lane * PER + i);
        amax = fmaxf(amax, fabsf(x[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float div = 1.0f, inv = 1.0f;
    if (amax > 65504.0f && amax <= 3.0e38f) {
        int e;
        frexpf(amax / 65504.0f, &e);        // amax / 2^e <= 65504
        div = ldexpf(1.0f, e);
        inv = ldexpf(1.0f, -e);
    }
    __half* dst = q16 + ((int64_t)h * T + t) * D + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 2) {
        const uint32_t w = pack_half2(x[i] * inv, x[i + 1] * inv);
        *reinterpret_cast<uint32_t*>(dst + i) = w;
    }
    if (lane == 0) qscale[row] = div;
}

// 256 threads: thread (token row trow of every 32, 16-key segment key_seg) of one 128-key block.
// With 16-byte aligned mask rows a segment is two 16-byte loads.
__device__ __forceinline__ void fa_mask_block(const uint16_t* __restrict__ mask, int64_t m_stride, bool vec, int T,
                                              int KV, int TQ, int tb, int j, int n_kvb, uint8_t* __restrict__ flags) {
    const int key_seg = threadIdx.x & 7;          // 16 keys each
    const int trow = threadIdx.x >> 3;            // 32 token rows per pass
    const int key0 = j * FA_KB + key_seg * 16;
    const bool full_seg = key0 + 16 <= KV;
    bool all_masked = true, all_zero = key0 < KV && full_seg;
    for (int tr = trow; tr < TQ; tr += 32) {
        const int t = tb * TQ + tr;
        if (t >= T) continue;
        const uint16_t* mrow = mask + (int64_t)t * m_stride + key0;
        if (vec && full_seg) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(mrow));
            const uint4 b = __ldg(reinterpret_cast<const uint4*>(mrow) + 1);
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (w[i] != 0xFC00FC00u) all_masked = false;         // two -inf
                if ((w[i] & 0x7FFF7FFFu) != 0) all_zero = false;     // two +-0
            }
        } else {
            for (int i = 0; i < 16; i++) {
                if (key0 + i >= KV) break;
                const uint16_t v = __ldg(mrow + i);
                if (v != 0xFC00u) all_masked = false;
                if ((v & 0x7FFFu) != 0) all_zero = false;
            }
        }
    }
    const int am = __syncthreads_and(all_masked ? 1 : 0);
    const int az = __syncthreads_and(all_zero ? 1 : 0);
    if (threadIdx.x == 0) flags[(int64_t)tb * n_kvb + j] = am ? MF_MASKED : (az ? MF_ZERO : MF_MIXED);
}

template <int D>
__global__ void __launch_bounds__(256) fa_prep_kernel(const float* __restrict__ q, int64_t q_nb1, int64_t q_nb2,
                                                      int T, int H, float scale, __half* __restrict__ q16,
                                                      float* __restrict__ qscale, int q_ctas,
                                                      const uint16_t* __restrict__ mask, int64_t m_stride,
                                                      bool mask_vec, int KV, int TQ, int n_kvb, int n_tb,
                                                      uint8_t* __restrict__ flags) {
    grid_dep_wait();          // q and the mask may be the previous kernel's output
    grid_dep_launch();
    if ((int)blockIdx.x < q_ctas) {
        fa_q_pack_row<D>(q, q_nb1, q_nb2, T, H, scale, q16, qscale, (int)(blockIdx.x * 8 + (threadIdx.x >> 5)),
                         (int)(threadIdx.x & 31));
        return;
    }
    const int mi = (int)blockIdx.x - q_ctas;
    if (!mask) {              // no mask: every block is all zero (one CTA writes them)
        if (mi == 0)
            for (int i = threadIdx.x; i < n_tb * n_kvb; i += blockDim.x) flags[i] = MF_ZERO;
        return;
    }
    fa_mask_block(mask, m_stride, mask_vec, T, KV, TQ, mi / n_kvb, mi % n_kvb, n_kvb, flags);
}

// A P row segment of N 32-bit columns (2N fp16 keys) into TMEM.
template <int N>
__device__ __forceinline__ void tmem_st_p(uint32_t taddr, const uint32_t (&w)[N]) {
    if constexpr (N == 64) {
        tmem_st32(taddr, reinterpret_cast<const uint32_t(&)[32]>(w[0]));
        tmem_st32(taddr + 32u, reinterpret_cast<const uint32_t(&)[32]>(w[32]));
    } else if constexpr (N == 32) {
        tmem_st32(taddr, w);
    } else {
        static_assert(N == 16, "P segments are 16, 32 or 64 columns");
        tmem_st16(taddr, w);
    }
}

// ---------------------------------------------------------------------------------------------
// The attention kernel.
// ---------------------------------------------------------------------------------------------
template <int D, int DV, bool EXT = false>
struct FaCfg {
    static constexpr int Q_BYTES = FA_ROWS * D * 2;
    static constexpr int K_BYTES = FA_KB * D * 2;
    static constexpr int V_BYTES = FA_KB * DV * 2;
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_K = EXT ? 0 : OFF_Q + Q_BYTES;   // EXT keeps Q in TMEM
    static constexpr int OFF_V = OFF_K + 2 * K_BYTES;
    // EXT: one ring of tiles in the order the products take them, high and low halves of K and V alike
    static constexpr int RING = EXT ? (D == 128 ? 6 : 10) : 0;
    // exchange between the FA_SPLIT threads of a row: maxima [2][SPLIT][128] f32 and their
    // sequence numbers (same shape, int), then sums [SPLIT][128] + sequence numbers
    static constexpr int XCH_MAX = 2 * FA_SPLIT * 128 * 4;
    static constexpr int XCH_SUM = FA_SPLIT * 128 * 4;
    static constexpr int OFF_XCH = EXT ? OFF_K + RING * K_BYTES : OFF_V + 2 * V_BYTES;
    static constexpr int OFF_REF = OFF_XCH + 2 * XCH_MAX + 2 * XCH_SUM;   // EXT: mask references, like the maxima
    static constexpr int OFF_BAR = OFF_REF + (EXT ? XCH_MAX : 0);
    static constexpr int SMEM = OFF_BAR + 256 + 1024;
    // TMEM columns: S0 [0,128) | S1 [128,256) | O [256, 256+DV) | P0 [384,448) | P1 [448,512)
    // (P is fp16, two keys per 32-bit column, read by the P.V MMA as its A operand)
    static constexpr uint32_t TMEM_COLS = 512;
    static constexpr uint32_t P_TMEM0 = 384;
    // EXT: Q's high halves [384, 384+D/2), its low ones [448, 448+D/2). P takes the place of the scores it is
    // made of: keys 64 pt .. 64 pt + 63 as columns 64 pt (high halves) and 64 pt + 32 (low halves) of S's 128.
    static constexpr uint32_t Q_TMEM0 = 384, Q_LO = 64, P_LO = 32;
    static constexpr uint32_t IDESC_S = idesc_f16_f32(FA_ROWS, FA_KB);
    static constexpr uint32_t IDESC_O = idesc_f16_f32_bmn(FA_ROWS, DV);
};

// A CTA's tile (numbered stream by stream, heavier token blocks first) and its range of key blocks.
struct FaUnit {
    int tile, first, end, slot;     // slot: of its part, -1 for a whole tile
};
__device__ __forceinline__ FaUnit fa_unit(const FaUnits& u, int n_kvb) {
    const int b = (int)blockIdx.x;
    if (b < u.whole) return {b, 0, n_kvb, -1};
    const int i = b - u.whole, piece = i % u.cut;
    return {u.whole + i / u.cut, min(n_kvb, piece * u.per), min(n_kvb, (piece + 1) * u.per), i};
}

// EXT: several streams (heads of q16 and of K / V numbered stream by stream), tiles whose keys CTAs share,
// scores scaled after the product, a key whose mask is -inf left out whatever its score, and every operand to
// 22 bits as two fp16 halves: K and V (a 4-bit code times an 11-bit scale is no fp16 number), the softmax
// weights P and, where it is f32 (QLO), q. S = Q_hi K_hi + Q_lo K_hi + Q_hi K_lo, O likewise of P and V: the
// products of two low halves are below 2^-22. Operands rounded to fp16 took an fp16 result's error from 2.1e-4,
// its own rounding, to 4.4e-4, and with P alone rounded to 2.9e-4. Q and P lie in TMEM, which leaves shared
// memory's bandwidth and its room to the ring of tiles; P takes the columns of the scores it is made of, so the
// next scores but one wait for its product. The products are issued from a converged warp: by one lane of a
// divergent one, each took its operands to uniform registers first, and the tensor core waited for the issue.
// 2048 tokens x 16384 keys, 32 heads over 8: 917 us for f16 q, 1061 for f32 (1066, 1163 in a long run, at the power
// cap), the products alone 785 and 942 at the measured rate; 626 with every operand rounded to fp16.
template <int D, int DV, bool EXT, bool QLO>
__global__ void __launch_bounds__(FA_THREADS, 1)
fa_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
          const __grid_constant__ CUtensorMap tmV, const FaArgs args) {
    using C = FaCfg<D, DV, EXT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    const uint32_t bar = sb + C::OFF_BAR;
    const uint32_t q_full = bar;
    auto k_full = [&](int s) { return bar + 8u * (1 + s); };
    auto k_empty = [&](int s) { return bar + 8u * (3 + s); };
    auto v_full = [&](int s) { return bar + 8u * (5 + s); };
    auto v_empty = [&](int s) { return bar + 8u * (7 + s); };
    // EXT: a ring's barriers in the place of K's and V's
    constexpr int X = EXT ? 2 * C::RING - 8 : 0;
    auto full = [&](int slot) { return bar + 8u * (1 + slot); };
    auto empty = [&](int slot) { return bar + 8u * (1 + C::RING + slot); };
    auto s_full = [&](int s) { return bar + 8u * (X + 9 + s); };
    auto s_empty = [&](int s) { return bar + 8u * (X + 11 + s); };
    // P of blocks b, b+2, ... written (per parity: a softmax warp may run one block ahead of
    // another, never two, because P buffer b is reused only after the P.V two blocks back)
    auto p_full = [&](int b) { return bar + 8u * (X + 17 + b); };
    auto pv_done = [&](int b) { return bar + 8u * (X + 14 + b); };   // P.V of blocks b, b+2, ... completed
    const uint32_t drain = bar + 8u * (X + 16);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + 8 * (X + 19));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_BAR + 8 * (X + 19) + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // heavier (later) token blocks first
    const int per_stream = EXT ? args.n_tb * args.n_hg : 0;
    const FaUnit un = EXT ? fa_unit(args.units, args.n_kvb) : FaUnit{(int)blockIdx.x, 0, args.n_kvb, -1};
    const int str = EXT ? un.tile / per_stream : 0, tile = EXT ? un.tile % per_stream : un.tile;
    const int tb = args.n_tb - 1 - tile / args.n_hg;
    const int hg = tile % args.n_hg;
    const int G = args.H / args.HK;
    const int hk = (hg * args.GP) / G;
    const uint8_t* flags = args.flags + ((int64_t)str * args.n_tb + tb) * args.n_kvb;
    const int j_first = un.first, j_end = un.end;

    if (threadIdx.x == 0) {
        mbar_init(q_full, EXT ? FA_SOFTMAX_WARPS : 1);
        if constexpr (EXT) {
            for (int n = 0; n < 2 * C::RING; n++) mbar_init(full(n), 1);
        } else {
            for (int s = 0; s < 2; s++) {
                mbar_init(k_full(s), 1);
                mbar_init(k_empty(s), 1);
                mbar_init(v_full(s), 1);
                mbar_init(v_empty(s), 1);
            }
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(s_full(s), 1);
            mbar_init(s_empty(s), FA_SOFTMAX_WARPS);
        }
        mbar_init(p_full(0), FA_SOFTMAX_WARPS);
        mbar_init(p_full(1), FA_SOFTMAX_WARPS);
        mbar_init(pv_done(0), 1);
        mbar_init(pv_done(1), 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        if constexpr (!EXT) tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
        tmem_relinquish();
    }
    {
        int* seqs = reinterpret_cast<int*>(smem + C::OFF_XCH + C::XCH_MAX);
        for (int k = threadIdx.x; k < 2 * FA_SPLIT * 128; k += FA_THREADS) seqs[k] = 0;
        int* seql = reinterpret_cast<int*>(smem + C::OFF_XCH + 2 * C::XCH_MAX + C::XCH_SUM);
        for (int k = threadIdx.x; k < FA_SPLIT * 128; k += FA_THREADS) seql[k] = 0;
    }
    tc_fence_before();
    cta_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // The prologue above overlapped the set-up pass (programmatic launch): Q16, its row divisors
    // and the mask flags are that pass's output, so wait for it before the first read.
    grid_dep_wait();
    grid_dep_launch();

    if (warp == 0) {
        if (lane == 0) {
            if constexpr (!EXT) {
                mbar_arrive_expect_tx(q_full, C::Q_BYTES);
                for (int c = 0; c < D / 64; c++)
                    tma_load_3d(sb + C::OFF_Q + c * (FA_ROWS * 128), &tmQ, q_full, c * 64, tb * args.TQ,
                                str * args.H + hg * args.GP);
            }
            if constexpr (EXT) {
                // tiles in the order of the products: K of a block, then V of the one before
                int n = 0, prev = -1;
                bool ok = true;
                auto push = [&](const CUtensorMap* map, int j) {
                    for (int half = 0; half < 2 && ok; half++) {
                        const int slot = n % C::RING;
                        ok = mbar_wait(empty(slot), ((uint32_t)(n / C::RING) & 1u) ^ 1u, args.err, ERR_WAIT_PRODUCER, abort_flag);
                        if (!ok) break;
                        mbar_arrive_expect_tx(full(slot), C::K_BYTES);
                        for (int c = 0; c < D / 64; c++)
                            tma_load_3d(sb + C::OFF_K + slot * C::K_BYTES + c * (FA_KB * 128), map, full(slot), c * 64, j * FA_KB,
                                        (half * args.S + str) * args.HK + hk);
                        n++;
                    }
                };
                for (int j = j_first; j < j_end && ok; j++) {
                    if (flags[j] == MF_MASKED) continue;
                    push(&tmK, j);
                    if (prev >= 0) push(&tmV, prev);
                    prev = j;
                }
                if (prev >= 0) push(&tmV, prev);
                if (!ok) {   // let every copy already issued land before the CTA exits
                    bool drained = true;
                    for (int i = max(0, n - C::RING); i < n; i++) drained &= mbar_drain(full(i % C::RING), (uint32_t)(i / C::RING) & 1u);
                    if (!drained) atomicCAS(args.err, 0, ERR_WAIT_DRAIN);
                }
            } else {
                int i = 0;
                bool ok = true;
                int k_issued[2] = {-1, -1}, v_issued[2] = {-1, -1};
                for (int j = j_first; j < j_end && ok; j++) {
                    if (flags[j] == MF_MASKED) continue;
                    const int s = i & 1;
                    const uint32_t ph = (uint32_t)(i >> 1) & 1u;
                    if (!mbar_wait(k_empty(s), ph ^ 1u, args.err, ERR_WAIT_PRODUCER, abort_flag)) { ok = false; break; }
                    k_issued[s] = (int)ph;
                    mbar_arrive_expect_tx(k_full(s), C::K_BYTES);
                    for (int c = 0; c < D / 64; c++)
                        tma_load_3d(sb + C::OFF_K + s * C::K_BYTES + c * (FA_KB * 128), &tmK, k_full(s), c * 64, j * FA_KB, str * args.HK + hk);
                    if (!mbar_wait(v_empty(s), ph ^ 1u, args.err, ERR_WAIT_PRODUCER, abort_flag)) { ok = false; break; }
                    v_issued[s] = (int)ph;
                    mbar_arrive_expect_tx(v_full(s), C::V_BYTES);
                    for (int c = 0; c < DV / 64; c++)
                        tma_load_3d(sb + C::OFF_V + s * C::V_BYTES + c * (FA_KB * 128), &tmV, v_full(s), c * 64, j * FA_KB, str * args.HK + hk);
                    i++;
                }
                if (!ok) {   // let every copy already issued land before the CTA exits
                    bool drained = mbar_drain(q_full, 0);
                    for (int s = 0; s < 2; s++) {
                        if (k_issued[s] >= 0) drained &= mbar_drain(k_full(s), (uint32_t)k_issued[s]);
                        if (v_issued[s] >= 0) drained &= mbar_drain(v_full(s), (uint32_t)v_issued[s]);
                    }
                    if (!drained) atomicCAS(args.err, 0, ERR_WAIT_DRAIN);
                }
            }
        }
    } else if (EXT && warp == 1) {
        // The whole warp walks the blocks and one lane issues: addresses and descriptors stay in uniform registers.
        const bool lead = elect_one();
        auto wait = [&](uint32_t b, uint32_t parity) {
            return __all_sync(0xffffffffu, mbar_wait(b, parity, args.err, ERR_WAIT_MMA, abort_flag));
        };
        int n_active = 0, slot = 0;                      // slot: the ring's next tile
        uint32_t turn = 0;
        // the two tiles of K or V: the high half takes A's high and (lo) low halves, the low one A's high ones
        auto product = [&](uint32_t d, uint32_t a, bool v, bool lo, uint32_t first, uint32_t done) {
            for (int half = 0; half < 2; half++) {
                if (!wait(full(slot), turn)) return false;
                tc_fence_after();
                const uint32_t tile = sb + C::OFF_K + slot * C::K_BYTES;
                const uint64_t desc = v ? sdesc_mn_sw128(tile, FA_KB * 128) : sdesc_k_sw128(tile);
                if (lead) {
                    for (int part = 0; part < (half == 0 && lo ? 2 : 1); part++) {
                        const uint32_t later = half == 0 && part == 0 ? first : 1u;
                        if (v) {
#pragma unroll
                            for (int ks = 0; ks < FA_KB / 16; ks++)
                                mma_f16_ts(d, a + C::P_LO * part + 8u * (ks & 3) + 64u * (ks >> 2),
                                           desc + (uint64_t)(ks * 2048 / 16), C::IDESC_O, ks > 0 ? 1u : later);
                        } else {
#pragma unroll
                            for (int ks = 0; ks < D / 16; ks++)
                                mma_f16_ts(d, a + C::Q_LO * part + 8u * ks,
                                           desc + (uint64_t)(((ks >> 2) * (FA_KB * 128) + (ks & 3) * 32) / 16), C::IDESC_S,
                                           ks > 0 ? 1u : later);
                        }
                    }
                    mma_commit(empty(slot));
                    if (half == 1) mma_commit(done);
                }
                __syncwarp();
                if (++slot == C::RING) slot = 0, turn ^= 1u;
            }
            return true;
        };
        auto issue_pv = [&](int i) {
            return wait(p_full(i & 1), (uint32_t)(i >> 1) & 1u) &&
                   product(tmem + 256, tmem + (uint32_t)(i & 1) * FA_KB, true, true, i > 0 ? 1u : 0u, pv_done(i & 1));
        };
        bool ok = wait(q_full, 0);
        tc_fence_after();
        for (int j = j_first; j < j_end && ok; j++) {
            if (flags[j] == MF_MASKED) continue;
            const int i = n_active, s = i & 1;
            // the buffer held P of block i - 2 last
            ok = (i < 2 || wait(pv_done(s), ((uint32_t)(i >> 1) & 1u) ^ 1u)) &&
                 product(tmem + (uint32_t)(s * FA_KB), tmem + C::Q_TMEM0, false, QLO, 0u, s_full(s));
            if (!ok) break;
            n_active++;
            if (i > 0) ok = issue_pv(i - 1);
        }
        if (ok && n_active > 0) issue_pv(n_active - 1);
        if (lead) mma_commit(drain);
        __syncwarp();
        if (!__all_sync(0xffffffffu, mbar_drain(drain, 0)) && lead) atomicCAS(args.err, 0, ERR_WAIT_DRAIN);
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = mbar_wait(q_full, 0, args.err, ERR_WAIT_MMA, abort_flag);
            tc_fence_after();
            int n_active = 0;
            auto issue_pv = [&](int i) -> bool {
                const int s = i & 1;
                const uint32_t ph = (uint32_t)(i >> 1) & 1u;
                if (!mbar_wait(p_full(i & 1), (uint32_t)(i >> 1) & 1u, args.err, ERR_WAIT_MMA, abort_flag)) return false;
                if (!mbar_wait(v_full(s), ph, args.err, ERR_WAIT_MMA, abort_flag)) return false;
                tc_fence_after();
                const uint32_t vb = sb + C::OFF_V + s * C::V_BYTES;
                const uint32_t p_tmem = tmem + C::P_TMEM0 + (uint32_t)(64 * (i & 1));
#pragma unroll
                for (int ks = 0; ks < FA_KB / 16; ks++) {
                    const uint64_t bdesc = sdesc_mn_sw128(vb + ks * 2048, FA_KB * 128);
                    mma_f16_ts(tmem + 256, p_tmem + 8u * ks, bdesc, C::IDESC_O, (i > 0 || ks > 0) ? 1u : 0u);
                }
                mma_commit(pv_done(i & 1));
                mma_commit(v_empty(s));
                return true;
            };
            for (int j = j_first; j < j_end && ok; j++) {
                if (flags[j] == MF_MASKED) continue;
                const int i = n_active;
                const int s = i & 1;
                const uint32_t ph = (uint32_t)(i >> 1) & 1u;
                if (!mbar_wait(k_full(s), ph, args.err, ERR_WAIT_MMA, abort_flag)) { ok = false; break; }
                if (!mbar_wait(s_empty(s), ph ^ 1u, args.err, ERR_WAIT_MMA, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t kb = sb + C::OFF_K + s * C::K_BYTES;
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++) {
                    const uint64_t a = sdesc_k_sw128(sb + C::OFF_Q + (ks >> 2) * (FA_ROWS * 128) + (ks & 3) * 32);
                    const uint64_t bdesc = sdesc_k_sw128(kb + (ks >> 2) * (FA_KB * 128) + (ks & 3) * 32);
                    mma_f16(tmem + (uint32_t)(s * FA_KB), a, bdesc, C::IDESC_S, ks > 0 ? 1u : 0u);
                }
                mma_commit(s_full(s));
                mma_commit(k_empty(s));
                n_active++;
                if (i > 0 && !issue_pv(i - 1)) { ok = false; break; }
            }
            if (ok && n_active > 0) issue_pv(n_active - 1);
            mma_commit(drain);
            if (!mbar_drain(drain, 0)) atomicCAS(args.err, 0, ERR_WAIT_DRAIN);
        }
    } else {
        // ---------------- softmax / output: FA_SPLIT threads per query row ----------------
        // Warps w, w+4, ... share TMEM lane quarter (w & 3); thread (row r, part pt) owns keys
        // [KPT*pt, KPT*(pt+1)) of every block and O columns [OPT*pt, OPT*(pt+1)). Scores are kept
        // in log2 units. O accumulates in TMEM across blocks (P.V MMAs with accumulate); it is
        // rescaled only when a row's max grows by more than 2^FA_RESCALE_LOG2 over the max the
        // exponentials were taken against (so P <= 2^8 and nothing overflows).
        constexpr int KPT = FA_KB / FA_SPLIT;            // keys per thread per block
        constexpr int OPT = DV / FA_SPLIT;               // O columns per thread
        const int quad = warp & 3;
        const int pt = (warp - 2) >> 2;
        const int r = quad * 32 + lane;
        const int g = r / args.TQ, tq = r % args.TQ;
        const int h = hg * args.GP + g;
        const int t = tb * args.TQ + tq;
        const bool row_valid = t < args.T;
        const float qs = row_valid ? __ldg(args.qscale + ((int64_t)str * args.H + h) * args.T + t) : 1.0f;
        const uint16_t* mrow = (args.mask && row_valid) ? args.mask + (EXT ? str * args.m_stream : 0) + (int64_t)t * args.m_stride
                                                        : nullptr;
        const float LOG2E = 1.4426950408889634f;
        const float c2 = qs * LOG2E;                     // raw score -> log2 units
        const float softcap = args.softcap;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const uint32_t o_tmem = tmem + lane_base + 256u + (uint32_t)(pt * OPT);
        volatile float* xv = reinterpret_cast<volatile float*>(smem + C::OFF_XCH);
        volatile int* xs = reinterpret_cast<volatile int*>(smem + C::OFF_XCH + C::XCH_MAX);
        volatile float* xl = reinterpret_cast<volatile float*>(smem + C::OFF_XCH + 2 * C::XCH_MAX);
        volatile int* xls = reinterpret_cast<volatile int*>(smem + C::OFF_XCH + 2 * C::XCH_MAX + C::XCH_SUM);
        // this thread's keys of a block are P columns [KPT/2*pt, KPT/2*(pt+1)) of the P buffer
        const uint32_t p_lane = tmem + lane_base + C::P_TMEM0 + (uint32_t)(pt * (KPT / 2));
        // A wait may give up in some lanes of a warp alone; votes, tcgen05.ld and .st take all of them, so the
        // warp goes on, or leaves, together.
        auto together = [](bool got) { return __all_sync(0xffffffffu, got) != 0; };
        auto wait = [&](uint32_t b, uint32_t parity) {
            return together(mbar_wait(b, parity, args.err, ERR_WAIT_EPILOGUE, abort_flag));
        };
        // wait until the P.V MMA of block k has completed (pv_done[k & 1], completion k >> 1)
        auto wait_pv = [&](int k) { return wait(pv_done(k & 1), (uint32_t)(k >> 1) & 1u); };
        // Publish a value to the other threads of this row and wait for theirs: a bounded spin on
        // sequence numbers in shared memory (the threads are in different warps). vals[k] gets
        // part k's value.
        auto exchange = [&](volatile float* v, volatile int* sq, float mine, int seq, float (&vals)[FA_SPLIT]) -> bool {
            v[pt * 128 + r] = mine;
            __threadfence_block();
            sq[pt * 128 + r] = seq;
            const uint64_t t0 = globaltimer();
            uint32_t n = 0;
#pragma unroll
            for (int k = 0; k < FA_SPLIT; k++) {
                while (sq[k * 128 + r] != seq) {
                    if ((++n & 255u) == 0) {
                        if (*abort_flag) return false;
                        if (globaltimer() - t0 > B200_WAIT_LIMIT_NS) {
                            atomicCAS(args.err, 0, ERR_WAIT_EPILOGUE);
                            *abort_flag = 1;
                            return false;
                        }
                    }
                }
            }
            __threadfence_block();
#pragma unroll
            for (int k = 0; k < FA_SPLIT; k++) vals[k] = v[k * 128 + r];
            return true;
        };
        if constexpr (EXT) {                             // Q's row, this thread's half of it, to TMEM
#pragma unroll
            for (int part = 0; part < (QLO ? 2 : 1); part++) {
                const uint4* src = reinterpret_cast<const uint4*>(
                    args.q16 + ((((int64_t)part * args.S + str) * args.H + h) * args.T + (row_valid ? t : 0)) * D + pt * (D / 2));
                uint32_t w[D / 4];
#pragma unroll
                for (int n = 0; n < D / 16; n++) {
                    const uint4 v = row_valid ? src[n] : make_uint4(0, 0, 0, 0);
                    w[4 * n] = v.x, w[4 * n + 1] = v.y, w[4 * n + 2] = v.z, w[4 * n + 3] = v.w;
                }
                tmem_st_p<D / 4>(tmem + lane_base + C::Q_TMEM0 + C::Q_LO * part + (uint32_t)(pt * (D / 4)), w);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        float m = -INFINITY;                             // running max (log2 units)
        float mref = 0.0f;                               // EXT: of a score less this mask value
        volatile float* xr = reinterpret_cast<volatile float*>(smem + C::OFF_REF);
        float l = 0.0f;                                  // this thread's partial row sum
        int i = 0;
        bool ok = true;
        for (int j = j_first; j < j_end && ok; j++) {
            const uint8_t fl = flags[j];
            if (fl == MF_MASKED) continue;
            const bool use_mask = (fl == MF_MIXED) && (mrow != nullptr);
            const bool general = use_mask || softcap != 0.0f || (j + 1) * FA_KB > args.KV || (EXT && !(args.scale >= 0.0f));
            const int s = i & 1;
            const uint32_t ph = (uint32_t)(i >> 1) & 1u;
            if (!wait(s_full(s), ph)) { ok = false; break; }
            tc_fence_after();
            float x[KPT];
#pragma unroll
            for (int c0 = 0; c0 < KPT; c0 += 32) {
                uint32_t rv[32];
                tmem_ld32(tmem + lane_base + (uint32_t)(s * FA_KB + pt * KPT + c0), rv);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; e++) x[c0 + e] = __uint_as_float(rv[e]);
            }
            if constexpr (!EXT) {
                // S is in registers: the buffer may take the next Q.K^T
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_empty(s));
            }
            const int k0 = j * FA_KB + pt * KPT;
            float bmax = -INFINITY;
            float ref = 0.0f;                            // EXT: the largest mask value of this thread's keys
            if (EXT && use_mask) {
                ref = -INFINITY;
#pragma unroll
                for (int c0 = 0; c0 < KPT; c0 += 32) {
                    uint4 mv[4];
                    load_mask32(mrow, k0 + c0, args.KV, args.mask_vec, mv);
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const uint32_t w = (&mv[e >> 2].x)[e & 3];
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
                        if (k0 + c0 + 2 * e < args.KV) ref = fmaxf(ref, f.x);
                        if (k0 + c0 + 2 * e + 1 < args.KV) ref = fmaxf(ref, f.y);
                    }
                }
                ref = fabsf(ref) <= 65504.0f ? ref : 0.0f;   // all masked (or an infinite mask): nothing to gain
            }
            if (!general) {
#pragma unroll
                for (int e = 0; e < KPT; e++) bmax = fmaxf(bmax, x[e]);
                bmax *= c2;
            } else {
#pragma unroll
                for (int c0 = 0; c0 < KPT; c0 += 32) {
                    uint4 mv[4];
                    if (use_mask) load_mask32(mrow, k0 + c0, args.KV, args.mask_vec, mv);
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        float sv = x[c0 + e] * qs;
                        if (softcap != 0.0f) sv = EXT ? capped(sv, softcap, 1.0f / softcap) : softcap * tanhf(sv / softcap);
                        sv *= LOG2E;
                        if (use_mask) {
                            const uint32_t mw = (&mv[e >> 3].x)[(e & 7) >> 1];
                            const uint16_t mb = (uint16_t)((e & 1) ? (mw >> 16) : (mw & 0xFFFFu));
                            sv = fmaf(__half2float(__ushort_as_half(mb)) - ref, LOG2E, sv);
                            if (mb == 0xFC00u) sv = -INFINITY;   // whatever its score is
                        }
                        if (k0 + c0 + e >= args.KV) sv = -INFINITY;
                        x[c0 + e] = sv;
                        bmax = fmaxf(bmax, sv);
                    }
                }
            }
            // the row max over all parts (double-buffered by block parity)
            float maxes[FA_SPLIT];
            if (EXT && use_mask) xr[(i & 1) * (FA_SPLIT * 128) + pt * 128 + r] = ref;   // published with the maximum
            if (!together(exchange(xv + (i & 1) * (FA_SPLIT * 128), xs + (i & 1) * (FA_SPLIT * 128), bmax, i + 1, maxes))) {
                ok = false;
                break;
            }
            float m_new, alpha, mu;
            if constexpr (EXT) {
                // The row's maximum as a pair (value, mask reference). Pairs are compared, and scores taken against
                // the running one, through differences, which are exact for mask values also where a score plus its
                // mask is not (fp16's lowest value on every key).
                float b_ref = 0.0f;
                bmax = maxes[0];
                if (use_mask) b_ref = xr[(i & 1) * (FA_SPLIT * 128) + r];
#pragma unroll
                for (int k = 1; k < FA_SPLIT; k++) {
                    const float k_ref = use_mask ? xr[(i & 1) * (FA_SPLIT * 128) + k * 128 + r] : 0.0f;
                    if ((maxes[k] - bmax) + (k_ref - b_ref) * LOG2E > 0.0f) bmax = maxes[k], b_ref = k_ref;
                }
                const bool grow = (bmax - m) + (b_ref - mref) * LOG2E > FA_RESCALE_LOG2;
                m_new = grow ? bmax : m;
                alpha = (grow && m != -INFINITY) ? ex2_approx((m - m_new) + (mref - b_ref) * LOG2E) : 1.0f;
                mref = grow ? b_ref : mref;
                mu = (m_new == -INFINITY) ? 0.0f : m_new - (ref - mref) * LOG2E;
            } else {
#pragma unroll
                for (int k = 0; k < FA_SPLIT; k++) bmax = fmaxf(bmax, maxes[k]);
                const bool grow = bmax > m + FA_RESCALE_LOG2;
                m_new = grow ? bmax : m;
                alpha = (grow && m != -INFINITY) ? ex2_approx(m - m_new) : 1.0f;
                mu = (m_new == -INFINITY) ? 0.0f : m_new;
            }
            // O is rescaled in place only after the previous block's P.V has landed in it
            if (i > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                if (!wait_pv(i - 1)) { ok = false; break; }
                tc_fence_after();
                {
#pragma unroll
                    for (int c0 = 0; c0 < OPT; c0 += 16) {
                        uint32_t ov[16];
                        tmem_ld16(o_tmem + (uint32_t)c0, ov);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; e++) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                        tmem_st16(o_tmem + (uint32_t)c0, ov);
                    }
                    tmem_st_wait();
                }
            }
            l *= alpha;
            m = m_new;
            if constexpr (EXT) {
                uint32_t ph[KPT / 2], pl[KPT / 2];
#pragma unroll
                for (int e = 0; e < KPT; e += 2) {
                    const float p0 = ex2_approx(general ? x[e] - mu : fmaf(x[e], c2, -mu));
                    const float p1 = ex2_approx(general ? x[e + 1] - mu : fmaf(x[e + 1], c2, -mu));
                    l += p0 + p1;
                    ph[e >> 1] = pack_half2(p0, p1);
                    const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&ph[e >> 1]));
                    pl[e >> 1] = pack_half2(p0 - hi.x, p1 - hi.y);
                }
                const uint32_t p_at = tmem + lane_base + (uint32_t)(s * FA_KB + pt * KPT);
                tmem_st_p<KPT / 2>(p_at, ph);
                tmem_st_p<KPT / 2>(p_at + C::P_LO, pl);
            } else {
                uint32_t pw[KPT / 2];
                if (!general) {
#pragma unroll
                    for (int e = 0; e < KPT; e += 2) {
                        const float p0 = ex2_approx(fmaf(x[e], c2, -mu));
                        const float p1 = ex2_approx(fmaf(x[e + 1], c2, -mu));
                        l += p0 + p1;
                        pw[e >> 1] = pack_half2(p0, p1);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < KPT; e += 2) {
                        const float p0 = ex2_approx(x[e] - mu);
                        const float p1 = ex2_approx(x[e + 1] - mu);
                        l += p0 + p1;
                        pw[e >> 1] = pack_half2(p0, p1);
                    }
                }
                // P buffer (i & 1) is free once the P.V of block i-2 has completed
                if (i >= 2) {
                    if (!wait_pv(i - 2)) { ok = false; break; }
                    tc_fence_after();
                }
                tmem_st_p<KPT / 2>(p_lane + (uint32_t)(64 * (i & 1)), pw);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(i & 1));
            i++;
        }
        bool have_o = false;
        if (ok && i > 0) {
            have_o = wait_pv(i - 1);
            tc_fence_after();
        }
        // row sum over all parts, added in part order so every thread of the row agrees
        float sums[FA_SPLIT];
        if (ok && !together(exchange(xl, xls, l, 1, sums))) ok = false;
        float l_tot = 0.0f;
#pragma unroll
        for (int k = 0; k < FA_SPLIT; k++) l_tot += sums[k];
        if constexpr (EXT) {
            if (ok) {                                    // tcgen05.ld is a whole warp's: rows past T load too
                const bool whole = un.slot < 0;
                const int64_t at = whole ? ((int64_t)str * args.T + t) * args.H + h : (int64_t)un.slot * FA_ROWS + r;
                const float inv = whole ? 1.0f / l_tot : 1.0f;
                if (!whole && pt == 0) {
                    args.stat[3 * at] = m;
                    args.stat[3 * at + 1] = l_tot;
                    args.stat[3 * at + 2] = mref;
                }
#pragma unroll
                for (int c0 = 0; c0 < OPT; c0 += 16) {
                    uint32_t ov[16];
                    if (have_o) {
                        tmem_ld16(o_tmem + (uint32_t)c0, ov);
                        tmem_ld_wait();
                    }
                    float y[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) y[e] = have_o && l_tot != 0.0f ? __uint_as_float(ov[e]) * inv : 0.0f;
                    if (whole && !row_valid) {
                    } else if (whole && args.dst_f16) {
                        uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<__half*>(args.dst) + at * DV + pt * OPT + c0);
                        out[0] = make_uint4(pack_half2(y[0], y[1]), pack_half2(y[2], y[3]), pack_half2(y[4], y[5]), pack_half2(y[6], y[7]));
                        out[1] = make_uint4(pack_half2(y[8], y[9]), pack_half2(y[10], y[11]), pack_half2(y[12], y[13]), pack_half2(y[14], y[15]));
                    } else {
                        float* out = (whole ? args.dst : args.part) + at * DV + pt * OPT + c0;
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            *reinterpret_cast<float4*>(out + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
                    }
                }
            }
        } else if (ok && have_o) {
            const float inv = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
            float* out = args.dst + ((int64_t)t * args.H + h) * DV + pt * OPT;
#pragma unroll
            for (int c0 = 0; c0 < OPT; c0 += 16) {
                uint32_t ov[16];
                tmem_ld16(o_tmem + (uint32_t)c0, ov);
                tmem_ld_wait();
                if (row_valid) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<float4*>(out + c0 + e) =
                            make_float4(__uint_as_float(ov[e]) * inv, __uint_as_float(ov[e + 1]) * inv,
                                        __uint_as_float(ov[e + 2]) * inv, __uint_as_float(ov[e + 3]) * inv);
                }
            }
        } else if (ok && row_valid) {
            // no key block survived the mask: the row is all zeros
            float* out = args.dst + ((int64_t)t * args.H + h) * DV + pt * OPT;
            for (int c = 0; c < OPT; c += 4) *reinterpret_cast<float4*>(out + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }

    tc_fence_before();
    cta_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

// Joins the parts of the tiles that several CTAs shared: W warps per row of such a tile take its parts in turn.
template <int D, int W>
__global__ void __launch_bounds__(256) fa_join_kernel(const FaArgs args, int n_rows) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float sums[8][D + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int id = (int)(blockIdx.x * (8 / W) + warp / W), w = warp % W;
    const int cut_tile = id / FA_ROWS, r = id % FA_ROWS;
    const int gt = args.units.whole + cut_tile, per_stream = args.n_tb * args.n_hg;
    const int str = gt / per_stream, tile = gt % per_stream;
    const int tb = args.n_tb - 1 - tile / args.n_hg;
    const int t = tb * args.TQ + r % args.TQ, h = tile % args.n_hg * args.GP + r / args.TQ;
    const bool in = id < n_rows && t < args.T;
    const int cut = args.units.cut;
    const int64_t first = (int64_t)cut_tile * cut * FA_ROWS + r;   // of part k: + k * FA_ROWS
    constexpr int PER = D / 32;
    float acc[PER] = {}, l_all = 0.0f;
    if (in) {
        // maxima are compared as maximum plus mask reference; their differences are formed apart, where they are exact
        constexpr float LOG2E = 1.4426950408889634f;
        float top = -INFINITY, m_best = 0.0f, r_best = 0.0f;
        for (int k = lane; k < cut; k += 32) {
            const float* st = args.stat + 3 * (first + (int64_t)k * FA_ROWS);
            const float v = st[0] + st[2] * LOG2E;
            if (st[1] != 0.0f && v > top) top = v, m_best = st[0], r_best = st[2];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float v = __shfl_xor_sync(0xffffffffu, top, o), mo = __shfl_xor_sync(0xffffffffu, m_best, o);
            const float ro = __shfl_xor_sync(0xffffffffu, r_best, o);
            if (v > top || (v == top && mo > m_best)) top = v, m_best = mo, r_best = ro;   // the same pair on every lane
        }
#pragma unroll 4
        for (int k = w; k < cut; k += W) {
            const int64_t at = first + (int64_t)k * FA_ROWS;
            const float l = args.stat[3 * at + 1];
            // l is 0 where no key is seen
            const float f = l == 0.0f ? 0.0f : ex2_approx((args.stat[3 * at] - m_best) + (args.stat[3 * at + 2] - r_best) * LOG2E);
            l_all = fmaf(l, f, l_all);
            const float* p = args.part + at * D + lane * PER;
#pragma unroll
            for (int e = 0; e < PER; e++) acc[e] = fmaf(p[e], f, acc[e]);
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int e = 0; e < PER; e++) sums[warp][lane * PER + e] = acc[e];
        if (lane == 0) sums[warp][D] = l_all;
        __syncthreads();
        if (w != 0) return;
        for (int o = 1; o < W; o++) {
#pragma unroll
            for (int e = 0; e < PER; e++) acc[e] += sums[warp + o][lane * PER + e];
            l_all += sums[warp + o][D];
        }
        l_all = __shfl_sync(0xffffffffu, l_all, 0);
    }
    if (!in) return;
    const int64_t at = (((int64_t)str * args.T + t) * args.H + h) * D + lane * PER;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const float y = l_all == 0.0f ? 0.0f : acc[e] / l_all;
        if (args.dst_f16) reinterpret_cast<__half*>(args.dst)[at + e] = __float2half_rn(y);
        else args.dst[at + e] = y;
    }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------

static bool make_tmap_3d_f16(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t nb1,
                             uint64_t nb2, uint32_t b0, uint32_t b1, uint32_t b2);

struct FaLayout {
    int GP, TQ, n_hg, n_tb, n_kvb;
    size_t q16_off, qs_off, flags_off, total;
};

static FaLayout fa_layout(int D, int T, int H, int KV, int HK) {
    FaLayout L{};
    const int G = H / HK;
    int gp = 1;
    while (gp * 2 <= 16 && G % (gp * 2) == 0) gp *= 2;
    L.GP = gp;
    L.TQ = FA_ROWS / gp;
    L.n_hg = H / gp;
    L.n_tb = (T + L.TQ - 1) / L.TQ;
    L.n_kvb = (KV + FA_KB - 1) / FA_KB;
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    L.q16_off = 0;
    L.qs_off = al((size_t)H * T * D * 2);
    L.flags_off = L.qs_off + al((size_t)H * T * 4);
    L.total = L.flags_off + al((size_t)L.n_tb * L.n_kvb);
    return L;
}

template <int D, int DV, bool EXT = false, bool QLO = false>
static cudaError_t launch_fa(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const FaArgs& a,
                             dim3 grid, cudaStream_t st) {
    using C = FaCfg<D, DV, EXT>;
    static bool set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !set[dev]) {
        cudaError_t e = cudaFuncSetAttribute(fa_kernel<D, DV, EXT, QLO>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        set[dev] = true;
    }
    return launch_pdl(fa_kernel<D, DV, EXT, QLO>, grid, dim3(FA_THREADS), C::SMEM, st, tq, tk, tv, a);
}

int flash_attn_impl(const float* q, int64_t q_nb1, int64_t q_nb2, const void* k, int64_t k_nb1, int64_t k_nb2,
                    const void* v, int64_t v_nb1, int64_t v_nb2, const void* mask, int64_t m_nb1, float* dst, int D,
                    int DV, int T, int H, int KV, int HK, float scale, float max_bias, float softcap, void* workspace,
                    size_t ws_bytes, int* dev_err, cudaStream_t st) {
    if (!q || !k || !v || !dst || !dev_err || T <= 0 || H <= 0 || KV <= 0 || HK <= 0) return B200_E_INVALID;
    if (H % HK != 0 || max_bias != 0.0f) return B200_E_UNSUPPORTED;
    if (!((D == 64 || D == 128) && (DV == 64 || DV == 128))) return B200_E_UNSUPPORTED;
    if ((k_nb1 | k_nb2 | v_nb1 | v_nb2) % 16 != 0) return B200_E_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(dst)) & 15u)
        return B200_E_UNSUPPORTED;
    if (mask && ((m_nb1 % 2) != 0 || (reinterpret_cast<uintptr_t>(mask) & 1u))) return B200_E_UNSUPPORTED;
    const FaLayout L = fa_layout(D, T, H, KV, HK);
    if (!workspace || ws_bytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return B200_E_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    __half* q16 = reinterpret_cast<__half*>(ws + L.q16_off);
    float* qs = reinterpret_cast<float*>(ws + L.qs_off);
    uint8_t* flags = reinterpret_cast<uint8_t*>(ws + L.flags_off);

    {
        const int q_ctas = (H * T + 7) / 8;
        const int m_ctas = mask ? L.n_tb * L.n_kvb : 1;
        const bool mvec = mask && (m_nb1 % 16) == 0 && (reinterpret_cast<uintptr_t>(mask) & 15u) == 0;
        const dim3 grid((unsigned)(q_ctas + m_ctas)), block(256);
        const uint16_t* m16 = static_cast<const uint16_t*>(mask);
        const cudaError_t e = D == 64
            ? launch_pdl(fa_prep_kernel<64>, grid, block, 0, st, q, q_nb1, q_nb2, T, H, scale, q16, qs, q_ctas, m16,
                         (int64_t)(m_nb1 / 2), mvec, KV, L.TQ, L.n_kvb, L.n_tb, flags)
            : launch_pdl(fa_prep_kernel<128>, grid, block, 0, st, q, q_nb1, q_nb2, T, H, scale, q16, qs, q_ctas, m16,
                         (int64_t)(m_nb1 / 2), mvec, KV, L.TQ, L.n_kvb, L.n_tb, flags);
        if (e != cudaSuccess) return B200_E_CUDA;
    }

    CUtensorMap tq, tk, tv;
    if (!make_tmap_3d_f16(&tq, q16, D, T, H, (uint64_t)D * 2, (uint64_t)T * D * 2, 64, L.TQ, L.GP)) return B200_E_CUDA;
    if (!make_tmap_3d_f16(&tk, k, D, KV, HK, k_nb1, k_nb2, 64, FA_KB, 1)) return B200_E_CUDA;
    if (!make_tmap_3d_f16(&tv, v, DV, KV, HK, v_nb1, v_nb2, 64, FA_KB, 1)) return B200_E_CUDA;
    FaArgs a{};
    a.qscale = qs;
    a.mask = static_cast<const uint16_t*>(mask);
    a.m_stride = m_nb1 / 2;
    a.mask_vec = mask && (m_nb1 % 16) == 0 && (reinterpret_cast<uintptr_t>(mask) & 15u) == 0;
    a.flags = flags;
    a.dst = dst;
    a.T = T;
    a.H = H;
    a.KV = KV;
    a.HK = HK;
    a.GP = L.GP;
    a.TQ = L.TQ;
    a.n_hg = L.n_hg;
    a.n_tb = L.n_tb;
    a.n_kvb = L.n_kvb;
    a.softcap = softcap;
    a.err = dev_err;
    const dim3 grid((unsigned)(L.n_hg * L.n_tb));
    cudaError_t e;
    if (D == 128 && DV == 128) e = launch_fa<128, 128>(tq, tk, tv, a, grid, st);
    else if (D == 64 && DV == 64) e = launch_fa<64, 64>(tq, tk, tv, a, grid, st);
    else if (D == 128 && DV == 64) e = launch_fa<128, 64>(tq, tk, tv, a, grid, st);
    else e = launch_fa<64, 128>(tq, tk, tv, a, grid, st);
    return e == cudaSuccess ? B200_OK : B200_E_CUDA;
}

// ---- the kernels over several streams, from a Q4_0 cache brought to fp16 tiles (b200_flash_attn_kvq) ----

// Set-up pass of one launch: CTAs [0, q_ctas) bring q to fp16 (one warp a row; f32 rows as two halves, times a
// power of two that brings them near 1; not scaled, so that f16 values stay exact), the next m_ctas classify the mask,
// the rest bring the cache to pairs of fp16 tiles: four lanes a block of 32 values, each eight of them. Bound by
// HBM and L2: 16384 keys, 8 KV heads of 128, 2048 tokens of 32 heads, 57 us for 19 MB of cache, 67 MB of mask
// and 17 MB of q read and 151 MB written (4.5 TB/s); making the tiles costs the call once what every query tile would else pay.
struct FaQuantPrep {
    const char* q;
    int64_t q_t, q_h, q_s;
    int q_f16;
    __half* q16;                 // [1, f32: 2 halves][S][H][T][D]
    float* qscale;               // per row: the scale times the divisor
    const uint16_t* mask;
    int64_t m_stride, m_stream;
    int mask_vec;
    uint8_t* flags;
    const uint8_t* k;
    int64_t k_r, k_h, k_s;
    const uint8_t* v;
    int64_t v_r, v_h, v_s;
    __half* k16;                 // [2: rounded values, what rounding left][S][HK][KV][D]
    __half* v16;
    int T, H, KV, HK, S, TQ, n_kvb, n_tb, q_ctas, m_ctas, m_grid;
    float scale;
};

// The eight values of bytes b of a Q4_0 block: code * d as fp16 and what that rounding leaves, exact in fp16
// again (four bits times eleven); low nibbles, high nibbles.
__device__ __forceinline__ void q4_0_values(uint32_t b, uint32_t d2, uint2 (&lo)[2], uint2 (&hi)[2]) {
    const __half2 c1032 = __half2half2(__ushort_as_half(0x6408)), c72 = __half2half2(__ushort_as_half(0x5480));
    const __half2 d = *reinterpret_cast<const __half2*>(&d2);
    const uint32_t u = b >> 8;
    const uint32_t w[4] = {(b & 0x000f000fu) | 0x64006400u, (u & 0x000f000fu) | 0x64006400u,
                           (b & 0x00f000f0u) | 0x54005400u, (u & 0x00f000f0u) | 0x54005400u};
    uint32_t x[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&w[i]), i < 2 ? c1032 : c72);
        const __half2 h = __hmul2(c, d), l = __hfma2(c, d, __hneg2(h));
        x[i] = *reinterpret_cast<const uint32_t*>(&h);
        r[i] = *reinterpret_cast<const uint32_t*>(&l);
    }
    lo[0] = make_uint2(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[0], x[1], 0x7632));
    hi[0] = make_uint2(__byte_perm(x[2], x[3], 0x5410), __byte_perm(x[2], x[3], 0x7632));
    lo[1] = make_uint2(__byte_perm(r[0], r[1], 0x5410), __byte_perm(r[0], r[1], 0x7632));
    hi[1] = make_uint2(__byte_perm(r[2], r[3], 0x5410), __byte_perm(r[2], r[3], 0x7632));
}

template <int D>
__global__ void __launch_bounds__(256) fa_quant_prep_kernel(const FaQuantPrep a) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    if ((int)blockIdx.x < a.q_ctas) {
        const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);   // (stream, head, token)
        if (row >= (int64_t)a.S * a.H * a.T) return;
        const int t = (int)(row % a.T), h = (int)(row / a.T % a.H), s = (int)(row / a.T / a.H);
        const char* src = a.q + s * a.q_s + h * a.q_h + t * a.q_t;
        constexpr int PER = D / 32;
        float x[PER], amax = 0.0f;
        if (a.q_f16) {
            uint16_t w[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) w[i] = reinterpret_cast<const uint16_t*>(src)[lane * PER + i];
#pragma unroll
            for (int i = 0; i < PER; i++) x[i] = __half2float(__ushort_as_half(w[i]));
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) x[i] = reinterpret_cast<const float*>(src)[lane * PER + i];
        }
#pragma unroll
        for (int i = 0; i < PER; i++) amax = fmaxf(amax, fabsf(x[i]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        // f32 rows are brought near 1 as well, so that their halves keep fp16's full precision
        int e = 0;
        if (!a.q_f16 && amax > 0.0f && amax <= 3.402823466e38f) frexpf(amax, &e);
        e = max(-126, e);
#pragma unroll
        for (int i = 0; i < PER; i += 2) {
            const float x0 = ldexpf(x[i], -e), x1 = ldexpf(x[i + 1], -e);
            const uint32_t hi = pack_half2(x0, x1);
            const float2 h2 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            uint32_t* dst = reinterpret_cast<uint32_t*>(a.q16 + row * D + lane * PER + i);
            *dst = hi;
            if (!a.q_f16) dst[(int64_t)a.S * a.H * a.T * D / 2] = pack_half2(x0 - h2.x, x1 - h2.y);
        }
        if (lane == 0) a.qscale[row] = ldexpf(a.scale, e);   // the scale within: 2^128 alone would be no f32 number
        return;
    }
    const int mi = (int)blockIdx.x - a.q_ctas;
    if (mi < a.m_grid) {
        if (!a.mask) {
            for (int i = threadIdx.x; i < a.S * a.n_tb * a.n_kvb; i += blockDim.x) a.flags[i] = MF_ZERO;
            return;
        }
        for (int i = mi; i < a.m_ctas; i += a.m_grid) {
            const int j = i % a.n_kvb, tb = i / a.n_kvb % a.n_tb, s = i / a.n_kvb / a.n_tb;
            fa_mask_block(a.mask + s * a.m_stream, a.m_stride, a.mask_vec != 0, a.T, a.KV, a.TQ, tb, j, a.n_kvb,
                          a.flags + (int64_t)s * a.n_tb * a.n_kvb);
        }
        return;
    }
    // A key whose value scales are no finite numbers gets zeros for them and NaN keys: rows that see it
    // become NaN through their scores, rows that do not stay clear of it (0 * NaN is NaN).
    constexpr int NB = D / 32, LANES = 4 * NB;           // lanes of a key's row
    const int64_t rows = (int64_t)a.S * a.HK * a.KV;
    const int64_t first = ((int64_t)(mi - a.m_grid) * 256 + threadIdx.x) / LANES;
    const int64_t step = (int64_t)(gridDim.x - a.q_ctas - a.m_grid) * 256 / LANES;
    const int c = (int)(threadIdx.x % LANES), b = c >> 2, p = c & 3;
    for (int64_t r0 = first - (threadIdx.x & 31) / LANES; r0 < rows; r0 += step) {   // warp-uniform bound
        const int64_t r = r0 + (threadIdx.x & 31) / LANES;
        const bool in = r < rows;
        const int64_t key = in ? r % a.KV : 0, sh = in ? r / a.KV : 0;
        const int64_t hk = sh % a.HK, s = sh / a.HK;
        const uint16_t* kb = reinterpret_cast<const uint16_t*>(a.k + s * a.k_s + hk * a.k_h + key * a.k_r + 18 * b);
        const uint16_t* vb = reinterpret_cast<const uint16_t*>(a.v + s * a.v_s + hk * a.v_h + key * a.v_r + 18 * b);
        uint32_t dk = __ldg(kb), dv = __ldg(vb);
        const uint32_t kw = __ldg(kb + 1 + 2 * p) | ((uint32_t)__ldg(kb + 2 + 2 * p) << 16);
        const uint32_t vw = __ldg(vb + 1 + 2 * p) | ((uint32_t)__ldg(vb + 2 + 2 * p) << 16);
        // codes of -8 may still take a large scale past fp16's range: such values count as no numbers too
        const float worst = fabsf(__half2float(__ushort_as_half((unsigned short)dv))) * 8.0f;
        const uint32_t votes = __ballot_sync(0xffffffffu, !(worst <= 65504.0f));
        if ((votes >> ((threadIdx.x & 31) / LANES * LANES)) & (LANES == 32 ? 0xffffffffu : (1u << LANES) - 1u))
            dk = 0x7e00u, dv = 0u;
        if (!in) continue;
        uint2 lo[2], hi[2];
        q4_0_values(kw, dk | (dk << 16), lo, hi);
        const int64_t at = r * D + 32 * b + 4 * p;
#pragma unroll
        for (int n = 0; n < 2; n++) {
            *reinterpret_cast<uint2*>(a.k16 + n * rows * D + at) = lo[n];
            *reinterpret_cast<uint2*>(a.k16 + n * rows * D + at + 16) = hi[n];
        }
        q4_0_values(vw, dv | (dv << 16), lo, hi);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            *reinterpret_cast<uint2*>(a.v16 + n * rows * D + at) = lo[n];
            *reinterpret_cast<uint2*>(a.v16 + n * rows * D + at + 16) = hi[n];
        }
    }
}

struct FaQuantLayout {
    FaLayout L;
    int cut_tiles;              // tiles whose keys CTAs share
    FaUnits units;
    size_t q16_off, qs_off, flags_off, k_off, v_off, part_off, stat_off, total;
};

static FaQuantLayout fa_quant_layout(int64_t D, int64_t T, int64_t H, int64_t KV, int64_t HK, int64_t S) {
    FaQuantLayout Q{};
    Q.L = fa_layout((int)D, (int)T, (int)H, (int)KV, (int)HK);
    // Whole tiles for as many full waves as there are; the tiles left over are cut into pieces of at least
    // four key blocks, so that their waves take the least time. In key blocks: the pieces' waves, then about
    // four for the join's launch and one for every 5.6 MB of parts it writes and reads.
    const int64_t tiles = S * Q.L.n_hg * Q.L.n_tb, sms = device_sm_count();
    const int64_t left = tiles % sms, part = D * 8 * FA_ROWS;
    int cut = 1;
    double best = left ? (double)Q.L.n_kvb : 0.0;
    for (int64_t k = 2; left && k <= 64 && Q.L.n_kvb >= 4 * k; k++) {
        const double cost = (double)((left * k + sms - 1) / sms * ((Q.L.n_kvb + k - 1) / k)) + 4.0 + (double)(left * k * part) / 5.6e6;
        if (cost < best) best = cost, cut = (int)k;
    }
    Q.cut_tiles = cut > 1 ? (int)left : 0;
    Q.units.whole = (int)(tiles - Q.cut_tiles);
    Q.units.per = (Q.L.n_kvb + cut - 1) / cut;
    Q.units.cut = cut;
    const int64_t rows = (int64_t)Q.cut_tiles * cut * FA_ROWS;
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += al(n); return o; };
    Q.q16_off = take((size_t)(S * H * T * D) * 4);
    Q.qs_off = take((size_t)(S * H * T) * 4);
    Q.flags_off = take((size_t)S * Q.L.n_tb * Q.L.n_kvb);
    Q.k_off = take((size_t)(S * HK * KV * D) * 4);
    Q.v_off = take((size_t)(S * HK * KV * D) * 4);
    Q.part_off = take((size_t)(rows * D) * 4);
    Q.stat_off = take((size_t)rows * 12);
    Q.total = at;
    return Q;
}

int64_t fa_quant_tiles(int64_t T, int64_t H, int64_t HK) {
    const FaLayout L = fa_layout(64, (int)T, (int)H, 1, (int)HK);
    return (int64_t)L.n_hg * L.n_tb;
}

size_t fa_quant_workspace(int64_t D, int64_t T, int64_t H, int64_t KV, int64_t HK, int64_t S) {
    return fa_quant_layout(D, T, H, KV, HK, S).total;
}

cudaError_t fa_quant_run(const FaQuantArgs& q, char* ws, cudaStream_t st) {
    const FaQuantLayout Q = fa_quant_layout(q.D, q.T, q.H, q.KV, q.HK, q.S);
    const FaLayout& L = Q.L;
    FaQuantPrep p{};
    p.q = q.q, p.q_t = q.q_t, p.q_h = q.q_h, p.q_s = q.q_s, p.q_f16 = q.q_f16;
    p.q16 = reinterpret_cast<__half*>(ws + Q.q16_off);
    p.qscale = reinterpret_cast<float*>(ws + Q.qs_off);
    p.mask = reinterpret_cast<const uint16_t*>(q.mask);
    p.m_stride = q.m_t / 2, p.m_stream = q.m_s / 2, p.mask_vec = q.m_vec;
    p.flags = reinterpret_cast<uint8_t*>(ws + Q.flags_off);
    p.k = reinterpret_cast<const uint8_t*>(q.k), p.k_r = q.k_r, p.k_h = q.k_h, p.k_s = q.k_s;
    p.v = reinterpret_cast<const uint8_t*>(q.v), p.v_r = q.v_r, p.v_h = q.v_h, p.v_s = q.v_s;
    p.k16 = reinterpret_cast<__half*>(ws + Q.k_off);
    p.v16 = reinterpret_cast<__half*>(ws + Q.v_off);
    p.T = q.T, p.H = q.H, p.KV = q.KV, p.HK = q.HK, p.S = q.S, p.scale = q.scale;
    p.TQ = L.TQ, p.n_kvb = L.n_kvb, p.n_tb = L.n_tb;
    const int sms = device_sm_count();
    p.q_ctas = (int)(((int64_t)q.S * q.H * q.T + 7) / 8);
    p.m_ctas = q.mask ? q.S * L.n_tb * L.n_kvb : 1;
    p.m_grid = std::min(p.m_ctas, sms * 16);
    const int64_t lanes = (int64_t)q.S * q.HK * q.KV * (q.D / 8);
    const int c_grid = (int)std::max<int64_t>(1, std::min<int64_t>((lanes + 255) / 256, (int64_t)sms * 16));
    const dim3 grid((unsigned)(p.q_ctas + p.m_grid + c_grid)), block(256);
    cudaError_t e = q.D == 64 ? launch_pdl(fa_quant_prep_kernel<64>, grid, block, 0, st, p)
                              : launch_pdl(fa_quant_prep_kernel<128>, grid, block, 0, st, p);
    if (e != cudaSuccess) return e;
    const uint64_t D = (uint64_t)q.D, row = D * 2;
    CUtensorMap tk, tv;
    if (!make_tmap_3d_f16(&tk, p.k16, D, q.KV, 2 * (uint64_t)q.S * q.HK, row, (uint64_t)q.KV * row, 64, FA_KB, 1) ||
        !make_tmap_3d_f16(&tv, p.v16, D, q.KV, 2 * (uint64_t)q.S * q.HK, row, (uint64_t)q.KV * row, 64, FA_KB, 1))
        return cudaErrorInvalidValue;
    FaArgs a{};
    a.qscale = p.qscale, a.q16 = p.q16;
    a.mask = p.mask;
    a.m_stride = p.m_stride, a.m_stream = p.m_stream, a.mask_vec = q.m_vec != 0;
    a.flags = p.flags;
    a.dst = static_cast<float*>(q.dst);
    a.S = q.S, a.T = q.T, a.H = q.H, a.KV = q.KV, a.HK = q.HK, a.GP = L.GP, a.TQ = L.TQ, a.n_hg = L.n_hg, a.n_tb = L.n_tb, a.n_kvb = L.n_kvb;
    a.softcap = q.softcap, a.scale = q.scale, a.dst_f16 = q.dst_f16;
    a.units = Q.units;
    a.part = reinterpret_cast<float*>(ws + Q.part_off);
    a.stat = reinterpret_cast<float*>(ws + Q.stat_off);
    a.err = q.err;
    const dim3 fgrid((unsigned)(Q.units.whole + Q.cut_tiles * Q.units.cut));
    // no map of Q, whose rows the softmax threads bring to TMEM: K's stands in its place, unused
    if (q.q_f16) e = q.D == 64 ? launch_fa<64, 64, true, false>(tk, tk, tv, a, fgrid, st) : launch_fa<128, 128, true, false>(tk, tk, tv, a, fgrid, st);
    else e = q.D == 64 ? launch_fa<64, 64, true, true>(tk, tk, tv, a, fgrid, st) : launch_fa<128, 128, true, true>(tk, tk, tv, a, fgrid, st);
    if (e != cudaSuccess || Q.cut_tiles == 0) return e;
    const int rows = Q.cut_tiles * FA_ROWS;
    auto join = [&](auto kernel, int warps) {
        return launch_pdl(kernel, dim3((unsigned)((rows * warps + 7) / 8)), dim3(256), 0, st, a, rows);
    };
    if (Q.units.cut <= 4) return q.D == 64 ? join(fa_join_kernel<64, 1>, 1) : join(fa_join_kernel<128, 1>, 1);
    return q.D == 64 ? join(fa_join_kernel<64, 4>, 4) : join(fa_join_kernel<128, 4>, 4);
}

}  // namespace b200

// The 3-D fp16 tensor map [d2][d1][d0] with byte strides nb1, nb2 and a 128-byte-swizzled box.
namespace b200 {
using EncodeTiledFn3 = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static bool make_tmap_3d_f16(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t nb1,
                             uint64_t nb2, uint32_t b0, uint32_t b1, uint32_t b2) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qr;
    static EncodeTiledFn3 fn = nullptr;
    if (!fn) {
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) != cudaSuccess ||
            qr != cudaDriverEntryPointSuccess)
            return false;
        fn = reinterpret_cast<EncodeTiledFn3>(p);
    }
    cuuint64_t dims[3] = {d0, d1, d2};
    cuuint64_t strides[2] = {nb1, nb2};
    cuuint32_t box[3] = {b0, b1, b2};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
}  // namespace b200

namespace b200 {

// ---- a quantized KV cache (Q8_0 / Q4_0) as the fp16 tiles the kernel reads ----------------------
// One thread per 32-value block of a [HK][KV][D] view (rows nb1 bytes apart, heads nb2): ggml's
// dequantize_row_q8_0 / _q4_0 (y = q * d, resp. (nibble - 8) * d, in f32), then fp16 (nearest
// even), written contiguous [HK][KV][D]. Blocks are 2-byte aligned only: byte loads.
// keys (the fp16 keys of these values, k_dim a key; or null): a block with values that are no finite fp16 numbers is
// written as zeros and its key's first value as a NaN, so that rows that see the key still become NaN, through their
// scores, and rows whose mask hides it stay clear of it (in the product of weights and values 0 * NaN is NaN).
template <int TYPE>
__global__ void kv_to_f16_kernel(const uint8_t* __restrict__ src, int64_t D, int64_t KV, int64_t HK, int64_t nb1,
                                 int64_t nb2, __half* __restrict__ dst, __half* __restrict__ keys, int64_t k_dim) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t per_row = D / 32, total = HK * KV * per_row;
    constexpr int BYTES = TYPE == 8 ? 34 : 18;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t c = i % per_row, r = (i / per_row) % KV, h = i / (per_row * KV);
        const uint8_t* b = src + h * nb2 + r * nb1 + c * BYTES;
        const float d = __half2float(__ushort_as_half((unsigned short)(b[0] | (b[1] << 8))));
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            float v0, v1;
            if constexpr (TYPE == 8) {
                v0 = __fmul_rn((float)(int8_t)b[2 + e], d);
                v1 = __fmul_rn((float)(int8_t)b[3 + e], d);
            } else {   // Q4_0: element j < 16 is the low nibble of byte j, j >= 16 the high nibble of byte j - 16
                const int j0 = e, j1 = e + 1;
                const int q0 = j0 < 16 ? (b[2 + j0] & 0x0f) : (b[2 + j0 - 16] >> 4);
                const int q1 = j1 < 16 ? (b[2 + j1] & 0x0f) : (b[2 + j1 - 16] >> 4);
                v0 = __fmul_rn((float)(q0 - 8), d);
                v1 = __fmul_rn((float)(q1 - 8), d);
            }
            w[e / 2] = (uint32_t)__half_as_ushort(__float2half_rn(v0)) |
                       ((uint32_t)__half_as_ushort(__float2half_rn(v1)) << 16);
        }
        if (keys) {
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 16; e++) bad |= (w[e] & 0x7c00u) == 0x7c00u || (w[e] & 0x7c000000u) == 0x7c000000u;
            if (bad) {
                keys[(h * KV + r) * k_dim] = __ushort_as_half((unsigned short)0x7e00);
#pragma unroll
                for (int e = 0; e < 16; e++) w[e] = 0u;
            }
        }
        uint4* o = reinterpret_cast<uint4*>(dst + (h * KV + r) * D + 32 * c);
#pragma unroll
        for (int q = 0; q < 4; q++) o[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    }
}

int kv_to_f16_impl(int type, const void* src, int64_t D, int64_t KV, int64_t HK, int64_t nb1, int64_t nb2, void* dst,
                   void* keys, int64_t k_dim, cudaStream_t st) {
    if (!src || !dst || D <= 0 || KV <= 0 || HK <= 0 || nb1 <= 0 || nb2 <= 0) return B200_E_INVALID;
    if ((type != 8 && type != 2) || D % 32 != 0 || (reinterpret_cast<uintptr_t>(dst) & 15u) != 0)
        return B200_E_UNSUPPORTED;
    const int64_t total = HK * KV * (D / 32);
    const int threads = 256;
    const int64_t want = (total + threads - 1) / threads;
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(want, (int64_t)device_sm_count() * 16));
    auto go = [&](auto kernel) {
        return launch_pdl(kernel, dim3(grid), dim3(threads), 0, st, static_cast<const uint8_t*>(src), D, KV, HK, nb1, nb2,
                          static_cast<__half*>(dst), static_cast<__half*>(keys), k_dim);
    };
    const cudaError_t e = type == 8 ? go(kv_to_f16_kernel<8>) : go(kv_to_f16_kernel<2>);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? B200_OK : B200_E_CUDA;
}

}  // namespace b200

extern "C" {

int b200_kv_to_f16(int type, const void* src, int64_t D, int64_t KV, int64_t HK, int64_t nb1, int64_t nb2, void* dst,
                   void* stream) {
    return b200::kv_to_f16_impl(type, src, D, KV, HK, nb1, nb2, dst, nullptr, 0, static_cast<cudaStream_t>(stream));
}

size_t b200_flash_attn_workspace_size(int D, int DV, int T, int H, int KV, int HK) {
    (void)DV;
    if (T <= 0 || H <= 0 || KV <= 0 || HK <= 0 || H % HK) return 0;
    return b200::fa_layout(D, T, H, KV, HK).total;
}

int b200_flash_attn_ext(const float* q, int64_t q_nb1, int64_t q_nb2, const void* k, int64_t k_nb1, int64_t k_nb2,
                        const void* v, int64_t v_nb1, int64_t v_nb2, const void* mask, int64_t m_nb1, float* dst,
                        int D, int DV, int T, int H, int KV, int HK, float scale, float max_bias, float softcap,
                        void* workspace, size_t workspace_bytes, int* dev_err, void* stream) {
    return b200::flash_attn_impl(q, q_nb1, q_nb2, k, k_nb1, k_nb2, v, v_nb1, v_nb2, mask, m_nb1, dst, D, DV, T, H, KV,
                                 HK, scale, max_bias, softcap, workspace, workspace_bytes, dev_err,
                                 static_cast<cudaStream_t>(stream));
}

}  // extern "C"
