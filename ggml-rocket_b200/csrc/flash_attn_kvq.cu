// FLASH_ATTN_EXT over a Q4_0 KV cache, read as it is stored (the reference's attention handler takes
// F16 K / V only, ggml-rocket.cpp:7654-7700, and leaves a quantised cache to its host):
//
//     dst[s, t, h] = sum_j softmax_j(scale q[s, t, h] . k[s, j, hk] (capped) + mask[s, t, j]) v[s, j, hk]
//
// with hk = h / (H / HK). A key whose mask is -inf is not read into the result, whatever its bytes
// hold; a row whose keys are all masked is zero.
//
// The row kernels. A warp holds 8 of the T * (H / HK) query rows that share a KV head and takes 32 keys at
// a time, with its own running maximum, sum and output:
//
//   S = Q K^T     mma.sync m16n8k16, 8 keys a tile. Rows 0-7 of the A operand are the query rows'
//                 fp16 high halves, rows 8-15 their low halves (q = hi + lo to 2^-22, scaled by a power
//                 of two into fp16's range), so both come out of one MMA. B holds the 4-bit codes as
//                 exact integers in fp16; the block scales multiply the fp32 sums of each 32 values.
//   O^T = V^T P^T the codes are the A operand (16 head dimensions x 16 keys), P times the value
//                 scales the B operand, straight from the score fragments' layout.
//
// P * scale is brought into fp16's range by a power of two per 32 keys (their largest value scale) and
// split into a high and a low half as well, for an fp16 result too: P rounded to fp16 alone takes its error
// from 2.1e-4, its own rounding, to as much as 3e-4. Sums, maxima and outputs are fp32 throughout; the output
// sums of 32 keys are added to the running ones by an fp32 FMA.
//
// Scores are in log2 units, taken relative to the largest mask value of the row in the CTA's range,
// whose difference to a key's mask is exact in fp32 also when every mask value is fp16's lowest.
//
// A CTA takes one stream, one range of keys and 8 rows of each of the KV heads whose cache rows make 144
// bytes (two heads of 128, four of 64): one thread brings tiles of 144 bytes x 32 or 64 keys by TMA (a
// head's 72 or 36 bytes are no multiple of 16), four warps take a head and 32 keys each. Rows
// 144 bytes apart fall into different banks for every fragment load. Tiles whose keys are masked for all
// the rows are never fetched: the CTA reads its mask range first. Caches TMA cannot address (heads not
// side by side, bases or strides off 16 bytes, a number of heads that does not divide) take the same
// arithmetic with cp.async copies of 8 (4) bytes, of which an SM moves about one a cycle (32 streams x 16384
// keys: 498 us so, 175 by TMA when that came). One KV head of 128 or two of 64 go that way: 32 streams, 38 us with
// one head of 128 (29 a head with two).
//
// With few rows the keys are split over CTAs, whose parts are joined through the shared memory of a cluster
// or by a second kernel. Calls with more rows go to the tcgen05 kernel of flash_attn.cu (see by_rows below).
//
// Bound by the issue of instructions, not by HBM: about 30 a key and KV head (decoding the codes, their
// fragments, the softmax). 64 streams of 16000 to 32000 keys, 8 KV heads of 128: 616 us, 2.9 TB/s of cache, 0.44
// of the measured copy bandwidth, 64 % of the issue slots; 32 streams of 8192 to 16384 keys 181 us (2.5 TB/s; 166
// with softmax weights of fp16, which an fp16 result showed). Some 15 % of that is SMs done before the others.
// A single stream: 16384 keys 17.6 us, 512 keys 7.6 us, of which some 4 are launch, mask and q; where the other ten
// of the long one go has not been taken apart (three tiles a CTA, a join in the cluster, a join of 11 parts).
#include <algorithm>
#include <cmath>
#include <cstdint>

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "ggml-b200-kernels.h"
#include "internal.h"
#include "ptx.cuh"

namespace b200 {

namespace {

constexpr int KR_ROWS = 8;             // query rows per CTA
constexpr int KR_WARPS = 4;
constexpr int KR_THREADS = 32 * KR_WARPS;
constexpr int KR_KEYS = 32;            // a warp takes at a time
constexpr int KR_BOX = 144;            // bytes of a key's row in a TMA tile
constexpr int KR_MAX_TILES = 1024;     // tiles of a CTA's range (its list of live tiles)
constexpr int KR_MAX_CLUSTER = 8;       // CTAs that join their parts through each other's shared memory
constexpr int KR_DEAD = 0x8000;         // of a list entry: a masked tile that was fetched all the same
constexpr int64_t KR_WAVES = 6;
constexpr int64_t KR_MIN_SPLIT = 2048;   // keys of a part, where they are many
constexpr float KR_LOG2E = 1.4426950408889634f;

struct KvqArgs {
    const char* q;
    int64_t q_t, q_h, q_s;             // byte strides of q: token, head, stream
    int q_f16, q_vec;                  // q_vec: four values a load
    const char* k;
    int64_t k_r, k_h, k_s;             // byte strides of k: key, head, stream
    const char* v;
    int64_t v_r, v_h, v_s;
    const char* mask;                  // f16 or nullptr
    int64_t m_t, m_s;                  // byte strides: token, stream
    int m_vec;                         // rows 16-byte aligned
    void* dst;                         // [S][T][H][D]
    int dst_f16;
    float* part;                       // [S][T][H][splits / cluster][D] outputs, then 3 floats a part
    float* stat;                       // {max (log2 units, relative), sum, mask reference}
    int T, H, KV, HK, G, S;
    int splits, tiles_per_split;       // CTAs that share a row's keys, and their ranges
    int cluster;                       // CTAs of a cluster
    float scale, softcap;
    int* err;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? BYTES : 0;   // bytes behind n are zero-filled
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with no sum to add to.
__device__ __forceinline__ void mma_16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// The eight 4-bit codes of a word as fp16 pairs of code - 8, exact: nibbles n0, n4 | n1, n5 | n2, n6 |
// n3, n7 (n0 the lowest). A nibble in the low mantissa bits of 1024 (0x6400) reads 1024 + u, one four
// bits up in 64 (0x5400) reads 64 + u.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t (&o)[4]) {
    const __half2 c1032 = __half2half2(__ushort_as_half(0x6408));   // 1032
    const __half2 c72 = __half2half2(__ushort_as_half(0x5480));     // 72
    const uint32_t u = w >> 8;
    const uint32_t a = (w & 0x000f000fu) | 0x64006400u, b = (w & 0x00f000f0u) | 0x54005400u;
    const uint32_t c = (u & 0x000f000fu) | 0x64006400u, d = (u & 0x00f000f0u) | 0x54005400u;
    __half2 h;
    h = __hsub2(*reinterpret_cast<const __half2*>(&a), c1032), o[0] = *reinterpret_cast<uint32_t*>(&h);
    h = __hsub2(*reinterpret_cast<const __half2*>(&b), c72), o[1] = *reinterpret_cast<uint32_t*>(&h);
    h = __hsub2(*reinterpret_cast<const __half2*>(&c), c1032), o[2] = *reinterpret_cast<uint32_t*>(&h);
    h = __hsub2(*reinterpret_cast<const __half2*>(&d), c72), o[3] = *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t ld32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ uint32_t ld16(const uint8_t* p) { return *reinterpret_cast<const uint16_t*>(p); }
// two 2-byte words as the halves of one
__device__ __forceinline__ uint32_t ld16x2(const uint8_t* lo, const uint8_t* hi) {
    return __byte_perm(ld16(lo), ld16(hi), 0x5410);
}
__device__ __forceinline__ float2 h2f(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    }
}


// HPB: KV heads a CTA takes; 1 with cp.async copies, 256 / D with TMA.
template <int D, int MT, int HPB>
struct KrCfg {
    static constexpr bool TMA = HPB > 1;
    static constexpr int NB = D / 32;                      // blocks of a head's row
    static constexpr int CH = D / 16;                      // bytes of a cp.async: nine make a head's row
    static constexpr int PARTS = KR_WARPS / HPB;           // warps that share a head
    static constexpr int TK = KR_KEYS * PARTS;             // keys of a CTA's tile
    static constexpr int THREADS = KR_THREADS, WARPS = KR_WARPS;
    static constexpr int PITCH = TMA ? KR_BOX : D == 128 ? 80 : 40;   // of a row in shared memory: the eight
                                                           // rows a fragment load touches fall into different banks
    static constexpr int HALF = (TMA ? TK : KR_KEYS) * PITCH;
    static constexpr int STAGE = 2 * HALF;                 // K rows, then V rows; of the CTA, or of a warp
    static constexpr int STAGES = TMA ? 3 * 18432 / STAGE : 3;
    static constexpr int RING = STAGES * STAGE * (TMA ? 1 : KR_WARPS);
    static constexpr int SCL = KR_KEYS * NB * 2;           // the scales of 32 keys (fp16), K then V
    static constexpr int OFF_SCL = RING;
    static constexpr int OFF_MSK = OFF_SCL + KR_WARPS * 2 * SCL;
    static constexpr int OFF_Q = OFF_MSK + KR_WARPS * MT * KR_KEYS * 4;
    static constexpr int OFF_BACK = OFF_Q + HPB * 2 * NB * 512;
    static constexpr int OFF_REF = OFF_BACK + HPB * KR_ROWS * 4;
    static constexpr int OFF_BAR = OFF_REF + (WARPS + 1) * KR_ROWS * 4;
    static constexpr int OFF_LIST = OFF_BAR + 16 * STAGES + 16;
    static constexpr int SMEM = OFF_LIST + KR_MAX_TILES * 2;
    static constexpr int OUT = (KR_ROWS * D + 2 * KR_ROWS) * 4;   // a warp's result, in the ring's place
    static constexpr int OFF_CTA = KR_WARPS * OUT;             // the CTA's: [head][row][D], then {max, sum} of each
    static_assert(OFF_CTA + HPB * KR_ROWS * (D + 2) * 4 <= RING && OFF_CTA % 16 == 0 && OFF_BAR % 8 == 0 && OFF_Q % 16 == 0 && HALF % 128 == 0);
};

// MT: the most tokens a CTA's rows come from (1 or 8). QLO: q is f32 (an f16 q has no low half). Leaving the codes' offsets in the MMA and starting its sums
// from minus the offset times sum(q), sum(P) saves the fp16 subtractions but measured slower (562 against
// 554 us over 64 streams x 32000 keys): they use a pipe that is idle.
template <int D, int MT, bool QLO, int HPB>
__global__ void __launch_bounds__(KrCfg<D, MT, HPB>::THREADS, 3)
kvq_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const KvqArgs a) {
    using C = KrCfg<D, MT, HPB>;
    extern __shared__ __align__(128) uint8_t sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int packs = a.HK / HPB;
    const int crank = (int)(blockIdx.x % a.cluster);     // the CTA's rank in its cluster
    const int split = blockIdx.x, pack = blockIdx.y % packs, rt = blockIdx.y / packs, str = blockIdx.z;
    const int rows_all = a.T * a.G, row0 = rt * KR_ROWS;
    const int rows = min(KR_ROWS, rows_all - row0);
    const int t_first = row0 / a.G, n_tok = MT == 1 ? 1 : (row0 + rows - 1) / a.G - t_first + 1;
    const int n_tiles = (a.KV + C::TK - 1) / C::TK;
    const int tile0 = split * a.tiles_per_split, tile1 = min(n_tiles, tile0 + a.tiles_per_split);
    const int range = max(0, tile1 - tile0);
    uint16_t* list = reinterpret_cast<uint16_t*>(sm + C::OFF_LIST);          // tiles from tile0; KR_DEAD: masked
    float* refs = reinterpret_cast<float*>(sm + C::OFF_REF);               // [warp][8], then per row
    float* backs = reinterpret_cast<float*>(sm + C::OFF_BACK);             // [head][row]
    uint4* q_frag = reinterpret_cast<uint4*>(sm + C::OFF_Q);               // [head][k-step][lane]
    const uint32_t bar = smem_u32(sm) + C::OFF_BAR;
    auto full = [&](int st) { return bar + 16u * st; };
    auto empty = [&](int st) { return bar + 16u * st + 8u; };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::OFF_BAR + 16 * C::STAGES);
    int* n_live = reinterpret_cast<int*>(sm + C::OFF_BAR + 16 * C::STAGES + 4);
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        if constexpr (C::TMA) {
            for (int st = 0; st < C::STAGES; st++) {
                mbar_init(full(st), 1);
                mbar_init(empty(st), KR_WARPS);
            }
            fence_barrier_init();
            tma_prefetch_desc(&tm_k);
            tma_prefetch_desc(&tm_v);
        }
    }
    grid_dep_wait();
    grid_dep_launch();

    // TMA: one thread brings tiles into the CTA's stages
    int sent = 0;
    auto send = [&](int tile, int st) {
        const uint32_t d = smem_u32(sm) + st * C::STAGE;
        mbar_arrive_expect_tx(full(st), C::STAGE);
        tma_load_3d(d, &tm_k, full(st), pack * KR_BOX, tile * C::TK, str);
        tma_load_3d(d + C::HALF, &tm_v, full(st), pack * KR_BOX, tile * C::TK, str);
        sent++;
    };
    // The first tiles are under way before the mask says whether they are live (one that is not is waited for
    // and passed over): a range of few tiles is all latency.
    const int early = C::TMA ? min(range, C::STAGES - 1) : 0;
    if (C::TMA && threadIdx.x == 0)
        for (int i = 0; i < early; i++) send(tile0 + i, i);

    // ---- q (warp i: head i of the CTA): high and low halves of the row, times a power of two that brings
    // its maximum to 2^10, in shared memory for every warp of the head, a k-step at a time ----
    uint4 q_raw[2 * C::NB];                              // values 16 i + 4 t4 .. + 3 of row g, as they are stored
#pragma unroll
    for (int i = 0; i < 2 * C::NB; i++) q_raw[i] = make_uint4(0, 0, 0, 0);
    if (warp < HPB && g < rows) {
        const int t = (row0 + g) / a.G, h = (pack * HPB + warp) * a.G + row0 + g - t * a.G;
        const char* qp = a.q + (int64_t)str * a.q_s + (int64_t)t * a.q_t + (int64_t)h * a.q_h;
        if (a.q_vec && a.q_f16) {
#pragma unroll
            for (int i = 0; i < 2 * C::NB; i++) {
                const uint2 v = *reinterpret_cast<const uint2*>(qp + 2 * (16 * i + 4 * t4));
                q_raw[i].x = v.x, q_raw[i].y = v.y;
            }
        } else if (a.q_vec) {
#pragma unroll
            for (int i = 0; i < 2 * C::NB; i++) q_raw[i] = *reinterpret_cast<const uint4*>(qp + 4 * (16 * i + 4 * t4));
        } else {
#pragma unroll
            for (int i = 0; i < 2 * C::NB; i++) {
                uint32_t w[4];
#pragma unroll
                for (int n = 0; n < 4; n++)
                    w[n] = a.q_f16 ? (uint32_t)reinterpret_cast<const uint16_t*>(qp)[16 * i + 4 * t4 + n]
                                   : reinterpret_cast<const uint32_t*>(qp)[16 * i + 4 * t4 + n];
                q_raw[i] = a.q_f16 ? make_uint4(w[0] | (w[1] << 16), w[2] | (w[3] << 16), 0, 0) : make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }

    // ---- the range's mask: live tiles and each token's largest mask value; eight keys a lane where the
    // mask's rows are 16-byte aligned ----
    const char* mbase = a.mask ? a.mask + (int64_t)str * a.m_s + (int64_t)t_first * a.m_t : nullptr;
    if (mbase) {
        float top[MT];
#pragma unroll
        for (int k = 0; k < MT; k++) top[k] = -INFINITY;
        constexpr int LT = C::TK / 8, PER = 32 / LT;     // lanes of a tile, tiles of a load
        for (int i = PER * warp; i < range; i += PER * C::WARPS) {
            const int key = (tile0 + i) * C::TK + 8 * lane;
            bool any = false;
#pragma unroll
            for (int k = 0; k < MT; k++) {
                if (k >= n_tok || i + lane / LT >= range) continue;
                const uint16_t* mp = reinterpret_cast<const uint16_t*>(mbase + k * a.m_t) + key;
                uint32_t w[4] = {0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};
                if (a.m_vec && key + 8 <= a.KV) {
                    const uint4 v = *reinterpret_cast<const uint4*>(mp);
                    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                } else {
#pragma unroll
                    for (int n = 0; n < 8; n++)
                        if (key + n < a.KV)
                            w[n >> 1] = (w[n >> 1] & (n & 1 ? 0x0000ffffu : 0xffff0000u)) | ((uint32_t)mp[n] << (16 * (n & 1)));
                }
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    any |= w[n] != 0xfc00fc00u;
                    const float2 f = h2f(w[n]);
                    top[k] = fmaxf(top[k], fmaxf(f.x, f.y));
                }
            }
            const uint32_t votes = __ballot_sync(0xffffffffu, any);
            if (lane < PER && i + lane < range) list[i + lane] = (votes >> (LT * lane)) & ((1u << LT) - 1u) ? 1 : 0;
        }
#pragma unroll
        for (int k = 0; k < MT; k++) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
            if (lane == 0) refs[warp * KR_ROWS + k] = top[k];
        }
    }
    // ---- q's halves ----
    if (warp < HPB) {
        float x[C::NB][8];
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * C::NB; i++) {
            const uint4 w = q_raw[i];
            const float2 lo = h2f(w.x), hi = h2f(w.y);
            float* d = &x[i >> 1][4 * (i & 1)];
            d[0] = a.q_f16 ? lo.x : __uint_as_float(w.x);
            d[1] = a.q_f16 ? lo.y : __uint_as_float(w.y);
            d[2] = a.q_f16 ? hi.x : __uint_as_float(w.z);
            d[3] = a.q_f16 ? hi.y : __uint_as_float(w.w);
        }
#pragma unroll
        for (int b = 0; b < C::NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[b][e]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int ex = 0;
        if (amax > 0.0f && amax <= 3.402823466e38f) frexpf(amax, &ex);
        ex = max(-126, ex - 10);                         // 2^126: the largest power whose inverse is a normal number
        const float mul = ldexpf(1.0f, -ex);
        if (t4 == 0) backs[warp * KR_ROWS + g] = ldexpf(a.scale, ex);   // what undoes it, with the scale
#pragma unroll
        for (int b = 0; b < C::NB; b++)
#pragma unroll
            for (int st = 0; st < 2; st++) {             // k-step 2b + st: values 16 st + {0, 2}, then {1, 3}
                float hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = x[b][4 * st + e] * mul;
                    hi[e] = __half2float(__float2half_rn(v));
                    lo[e] = v - hi[e];
                }
                q_frag[(warp * 2 * C::NB + 2 * b + st) * 32 + lane] =
                    make_uint4(pack_half2(hi[0], hi[2]), pack_half2(lo[0], lo[2]), pack_half2(hi[1], hi[3]),
                               pack_half2(lo[1], lo[3]));
            }
    }
    __syncthreads();
    const int my_tok = MT == 1 ? 0 : min(row0 + g, rows_all - 1) / a.G - t_first;   // of this lane's row (g)
    float* row_ref = refs + C::WARPS * KR_ROWS;          // per token, then per row
    if (mbase && threadIdx.x < MT) {
        float r = -INFINITY;
        if ((int)threadIdx.x < n_tok)
#pragma unroll
            for (int w = 0; w < C::WARPS; w++) r = fmaxf(r, refs[w * KR_ROWS + threadIdx.x]);
        row_ref[threadIdx.x] = r;
    }
    if (mbase) {
        if (warp == C::WARPS - 1) {                      // the live tiles in order, in place
            int n = 0;
            for (int i0 = 0; i0 < range; i0 += 32) {
                const int i = i0 + lane;
                const bool is = i < range && list[i] != 0, on = is || i < early;
                const uint32_t votes = __ballot_sync(0xffffffffu, on);
                if (on) list[n + __popc(votes & ((1u << lane) - 1u))] = (uint16_t)(i | (is ? 0 : KR_DEAD));
                n += __popc(votes);
                __syncwarp();
            }
            if (lane == 0) *n_live = n;
        }
    } else {
        for (int i = threadIdx.x; i < range; i += C::THREADS) list[i] = (uint16_t)i;
        if (threadIdx.x == 0) *n_live = range;
    }
    __syncthreads();
    const int live = *n_live;
    float ref_of[MT];                                    // the largest mask value, per token
#pragma unroll
    for (int k = 0; k < MT; k++) {
        const float r = mbase ? row_ref[k] : 0.0f;
        ref_of[k] = fabsf(r) <= 65504.0f ? r : 0.0f;     // all masked (or an infinite mask): nothing to gain
    }
    if (warp == 0 && t4 == 0) {
        float r = ref_of[0];
#pragma unroll
        for (int k = 1; k < MT; k++) r = my_tok == k ? ref_of[k] : r;
        refs[g] = r;                                     // the warps' maxima have been read: per row from here on
    }

    // ---- a warp's 32 keys of every live tile ----
    const int hs = warp % HPB, part = warp / HPB;        // its head of the CTA's, its keys of the tile's
    const float back = backs[hs * KR_ROWS + g], back2 = back * KR_LOG2E;
    const uint4* qs = q_frag + hs * 2 * C::NB * 32;
    uint8_t* ring = sm + (C::TMA ? 0 : warp * C::STAGES * C::STAGE);
    uint8_t* scl = sm + C::OFF_SCL + warp * 2 * C::SCL;
    float* msk = reinterpret_cast<float*>(sm + C::OFF_MSK) + warp * MT * KR_KEYS;

    const int c_row = lane / 9, c_chunk = lane - 9 * c_row;   // cp.async: lanes 0-26, three rows of nine pieces
    const char* kp = a.k + (int64_t)str * a.k_s + (int64_t)pack * a.k_h + c_row * a.k_r + c_chunk * C::CH;
    const char* vp = a.v + (int64_t)str * a.v_s + (int64_t)pack * a.v_h + c_row * a.v_r + c_chunk * C::CH;
    const uint32_t c_dst = smem_u32(ring) + c_row * C::PITCH + c_chunk * C::CH;
    auto fetch = [&](int e, int st) {                         // the warp's keys of live tile e into a stage
        if (e < live && lane < 27) {
            const int key0 = (tile0 + list[e]) * C::TK + part * KR_KEYS;
            const uint32_t d = c_dst + st * C::STAGE;
            const char* ks = kp + key0 * a.k_r;
            const char* vs = vp + key0 * a.v_r;
#pragma unroll
            for (int n = 0; n < 11; n++) {
                const int row = 3 * n + c_row;
                if (row >= KR_KEYS) break;
                const bool in = key0 + row < a.KV;       // rows behind the last key as zeros
                cp_async<C::CH>(d + 3 * n * C::PITCH, in ? ks : a.k, in);
                cp_async<C::CH>(d + 3 * n * C::PITCH + C::HALF, in ? vs : a.v, in);
                ks += 3 * a.k_r;
                vs += 3 * a.v_r;
            }
        }
        cp_async_commit();
    };
    if constexpr (C::TMA) {
        if (threadIdx.x == 0)
            while (sent < min(live, C::STAGES - 1)) send(tile0 + (list[sent] & ~KR_DEAD), sent);
    } else {
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) fetch(i, i);
    }

    float o[2 * C::NB][4];
#pragma unroll
    for (int m = 0; m < 2 * C::NB; m++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[m][e] = 0.0f;
    float run_max = -INFINITY, run_sum = 0.0f;           // of row g (the sum: this lane's keys)
    int unit = 0;                                        // o is in units of 2^unit

    // the lane's key's mask bits in live tile e, per token; 0xfc00 (-inf) where there is no such key
    auto load_mask = [&](int e, uint16_t (&m)[MT]) {
        const int key = e < live ? (tile0 + (list[e] & ~KR_DEAD)) * C::TK + part * KR_KEYS + lane : a.KV;
#pragma unroll
        for (int k = 0; k < MT; k++) {
            m[k] = key < a.KV ? 0 : 0xfc00;
            if (mbase && key < a.KV && k < n_tok) m[k] = *reinterpret_cast<const uint16_t*>(mbase + k * a.m_t + 2 * (int64_t)key);
        }
    };
    uint16_t mnext[MT];
    load_mask(0, mnext);

    int stage = 0;
    uint32_t phase = 0;
    bool gave_up = false;
    for (int e = 0; e < live; e++) {
        bool seen = false;
#pragma unroll
        for (int k = 0; k < MT; k++) {
            if (k >= n_tok) continue;
            seen |= mnext[k] != 0xfc00;
            const float m = __half2float(__ushort_as_half(mnext[k]));
            msk[k * KR_KEYS + lane] = m == -INFINITY ? m : (m - ref_of[k]) * KR_LOG2E;
        }
        load_mask(e + 1, mnext);
        const uint8_t *ks, *vs;
        if constexpr (C::TMA) {
            // the tile STAGES - 1 on, into the stage every warp has left behind
            if (threadIdx.x == 0) {
                const int prev = stage == 0 ? C::STAGES - 1 : stage - 1;
                if (e > 0 && sent < live && !gave_up &&
                    !mbar_wait(empty(prev), stage == 0 ? phase ^ 1u : phase, a.err, ERR_WAIT_PRODUCER, abort_flag))
                    gave_up = true;                      // the other waits end on the abort flag
                if (sent < live && !gave_up) send(tile0 + list[sent], prev);
            }
            __syncwarp();
            // a wait that gives up may do so for some lanes alone: the warp leaves together
            const bool got = mbar_wait(full(stage), phase, a.err, ERR_WAIT_STREAM, abort_flag);
            if (__any_sync(0xffffffffu, !got)) break;
            if (list[e] & KR_DEAD) {
                __syncwarp();
                if (lane == 0) mbar_arrive(empty(stage));
                if (++stage == C::STAGES) stage = 0, phase ^= 1u;
                continue;
            }
            ks = ring + stage * C::STAGE + part * KR_KEYS * C::PITCH + hs * (18 * C::NB);
        } else {
            cp_async_wait<C::STAGES - 2>();
            ks = ring + stage * C::STAGE;
        }
        vs = ks + C::HALF;
        __syncwarp();
        // the scales of key `lane`, apart from the codes; a key no row sees gets zeros
        uint32_t dk[C::NB / 2], dv[C::NB / 2];
        float vmax = 0.0f;
#pragma unroll
        for (int p = 0; p < C::NB / 2; p++) {
            const uint8_t* rk = ks + lane * C::PITCH + 36 * p;
            const uint8_t* rv = vs + lane * C::PITCH + 36 * p;
            dk[p] = seen ? ld16x2(rk, rk + 18) : 0u;
            dv[p] = seen ? ld16x2(rv, rv + 18) : 0u;
            const float2 f = h2f(dv[p] & 0x7fff7fffu);
            vmax = fmaxf(vmax, fmaxf(f.x, f.y));
        }
        if constexpr (C::NB == 4) {
            *reinterpret_cast<uint2*>(scl + lane * 8) = make_uint2(dk[0], dk[1]);
            *reinterpret_cast<uint2*>(scl + C::SCL + lane * 8) = make_uint2(dv[0], dv[1]);
        } else {
            *reinterpret_cast<uint32_t*>(scl + lane * 4) = dk[0];
            *reinterpret_cast<uint32_t*>(scl + C::SCL + lane * 4) = dv[0];
        }
        // the power of two that brings the tile's largest value scale to [2^10, 2^11)
        const uint32_t vbits = __reduce_max_sync(0xffffffffu, __float_as_uint(vmax));
        int vexp = (int)(vbits >> 23) - 127 - 10;
        if (vbits == 0 || vbits >= 0x7f800000u) vexp = unit;
        const float vmul = __uint_as_float((uint32_t)(127 - vexp) << 23);
        __syncwarp();

        // ---- S = Q K^T: a block of 32 values at a time, four 8-key columns side by side ----
        float s[4][2];
        uint32_t dd[4][C::NB];                           // scales of keys 8j + 2 t4 and + 1
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[j][0] = s[j][1] = 0.0f;
            load_words(scl + (8 * j + 2 * t4) * (C::NB * 2), dd[j]);
        }
#pragma unroll
        for (int b = 0; b < C::NB; b++) {
            const uint4 qa = qs[(2 * b) * 32 + lane], qb = qs[(2 * b + 1) * 32 + lane];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint8_t* kr = ks + (8 * j + g) * C::PITCH + 4 * t4 + 36 * (b >> 1);
                // a block of even number starts two bytes into a word
                const uint32_t w = (b & 1) ? ld32(kr + 20) : __byte_perm(ld32(kr), ld32(kr + 4), 0x5432);
                uint32_t f[4];
                float c[4];
                codes_f16(w, f);
                mma_16816_first(c, qa.x, qa.y, qa.z, qa.w, f[0], f[2]);
                mma_16816(c, qb.x, qb.y, qb.z, qb.w, f[1], f[3]);
                const float2 e0 = h2f(dd[j][b >> 1]), e1 = h2f(dd[j][C::NB / 2 + (b >> 1)]);
                s[j][0] = fmaf((b & 1) ? e0.y : e0.x, QLO ? c[0] + c[2] : c[0], s[j][0]);
                s[j][1] = fmaf((b & 1) ? e1.y : e1.x, QLO ? c[1] + c[3] : c[1], s[j][1]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 m = *reinterpret_cast<const float2*>(msk + my_tok * KR_KEYS + 8 * j + 2 * t4);
            if (a.softcap != 0.0f) {
                s[j][0] = a.softcap * KR_LOG2E * tanhf(s[j][0] * back / a.softcap) + m.x;
                s[j][1] = a.softcap * KR_LOG2E * tanhf(s[j][1] * back / a.softcap) + m.y;
            } else {
                s[j][0] = fmaf(s[j][0], back2, m.x);
                s[j][1] = fmaf(s[j][1], back2, m.y);
            }
            // K's scales were zeroed where no row sees the key; one that other rows see may still give no number
            if constexpr (MT > 1) {
                s[j][0] = m.x == -INFINITY ? -INFINITY : s[j][0];
                s[j][1] = m.y == -INFINITY ? -INFINITY : s[j][1];
            }
        }

        // ---- running maximum and sum ----
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++) top = fmaxf(top, fmaxf(s[j][0], s[j][1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float new_max = fmaxf(run_max, top);
        const float base = new_max == -INFINITY ? 0.0f : new_max;
        const float alpha = ex2(run_max - base);         // 0 before the first key
        run_max = new_max;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[j][0] = ex2(s[j][0] - base);
            s[j][1] = ex2(s[j][1] - base);
            sum += s[j][0] + s[j][1];
        }
        run_sum = fmaf(run_sum, alpha, sum);

        // ---- O^T = V^T P^T over the tile, a block of 32 values at a time ----
        // columns 2 t4 and 2 t4 + 1 of o are those query rows: their alpha, and the change of unit (scales
        // are fp16 numbers, so units lie in [-34, 5])
        const float f = __uint_as_float((uint32_t)(127 + unit - vexp) << 23);
        unit = vexp;
        const float al0 = __shfl_sync(0xffffffffu, alpha, 8 * t4) * f;
        const float al1 = __shfl_sync(0xffffffffu, alpha, 8 * t4 + 4) * f;
        uint32_t dw[4][C::NB];                           // value scales of keys 8j + 2 t4 and + 1
#pragma unroll
        for (int j = 0; j < 4; j++) {
            load_words(scl + C::SCL + (8 * j + 2 * t4) * (C::NB * 2), dw[j]);
            s[j][0] *= vmul, s[j][1] *= vmul;
        }
#pragma unroll
        for (int b = 0; b < C::NB; b++) {
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 x0 = h2f(dw[j][b >> 1]), x1 = h2f(dw[j][C::NB / 2 + (b >> 1)]);
                float w0 = s[j][0] * ((b & 1) ? x0.y : x0.x), w1 = s[j][1] * ((b & 1) ? x1.y : x1.x);
                if constexpr (MT > 1) {                  // a key other rows see: its scale may be no number
                    w0 = s[j][0] == 0.0f ? 0.0f : w0;
                    w1 = s[j][1] == 0.0f ? 0.0f : w1;
                }
                ph[j] = pack_half2(w0, w1);
                const float2 h = h2f(ph[j]);
                pl[j] = pack_half2(w0 - h.x, w1 - h.y);
            }
            float ot[2][4];
#pragma unroll
            for (int jj = 0; jj < 2; jj++) {
                const uint8_t* va = vs + (16 * jj + 2 * t4) * C::PITCH + 2 + 2 * g + 18 * b;
                const uint32_t y0 = ld16x2(va, va + C::PITCH), y1 = ld16x2(va + 8 * C::PITCH, va + 9 * C::PITCH);
                uint32_t f0[4], f1[4];                   // {2g, 16 + 2g, 2g + 1, 17 + 2g} of the block, key pairs
                codes_f16(y0, f0);
                codes_f16(y1, f1);
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    if (jj > 0) mma_16816(ot[m], f0[2 * m], f0[2 * m + 1], f1[2 * m], f1[2 * m + 1], ph[2 * jj], ph[2 * jj + 1]);
                    else mma_16816_first(ot[m], f0[2 * m], f0[2 * m + 1], f1[2 * m], f1[2 * m + 1], ph[0], ph[1]);
                    mma_16816(ot[m], f0[2 * m], f0[2 * m + 1], f1[2 * m], f1[2 * m + 1], pl[2 * jj], pl[2 * jj + 1]);
                }
            }
#pragma unroll
            for (int m = 0; m < 2; m++) {
                o[2 * b + m][0] = fmaf(o[2 * b + m][0], al0, ot[m][0]);
                o[2 * b + m][1] = fmaf(o[2 * b + m][1], al1, ot[m][1]);
                o[2 * b + m][2] = fmaf(o[2 * b + m][2], al0, ot[m][2]);
                o[2 * b + m][3] = fmaf(o[2 * b + m][3], al1, ot[m][3]);
            }
        }
        __syncwarp();                                    // the stage, the scales and the mask are free again
        if constexpr (C::TMA) {
            if (lane == 0) mbar_arrive(empty(stage));
        } else {
            fetch(e + C::STAGES - 1, stage == 0 ? C::STAGES - 1 : stage - 1);
        }
        if (++stage == C::STAGES) stage = 0, phase ^= 1u;
    }
    if constexpr (C::TMA) {
        // after an abort, let every copy land before the CTA reuses or leaves its memory
        if (threadIdx.x == 0 && *abort_flag) {
            bool drained = true;
            for (int i = max(0, sent - C::STAGES); i < sent; i++)
                drained &= mbar_drain(full(i % C::STAGES), (uint32_t)(i / C::STAGES) & 1u);
            if (!drained) atomicCAS(a.err, 0, ERR_WAIT_DRAIN);
        }
    } else {
        cp_async_wait<0>();
    }
    cta_sync();

    // ---- join the warps of a head ----
    float* wout = reinterpret_cast<float*>(sm + warp * C::OUT);
    run_sum += __shfl_xor_sync(0xffffffffu, run_sum, 1);
    run_sum += __shfl_xor_sync(0xffffffffu, run_sum, 2);
    const float lift = __uint_as_float((uint32_t)(127 + unit) << 23);
#pragma unroll
    for (int b = 0; b < C::NB; b++)
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const int d = 32 * b + 2 * g + m;            // MMA 2b + m: dimensions d and d + 16
            float* c = wout + 2 * t4 * D + d;
            c[0] = o[2 * b + m][0] * lift;
            c[D] = o[2 * b + m][1] * lift;
            c[16] = o[2 * b + m][2] * lift;
            c[D + 16] = o[2 * b + m][3] * lift;
        }
    if (t4 == 0) {
        wout[KR_ROWS * D + g] = run_max;
        wout[KR_ROWS * D + KR_ROWS + g] = run_sum;
    }
    cta_sync();
    // A thread takes value d of rows r0, r0 + 128 / D, ..; rows are numbered 8 head + r here, those from `rows`
    // on of each head left out.
    float* cta_out = reinterpret_cast<float*>(sm + C::OFF_CTA);
    float* cta_stat = cta_out + HPB * KR_ROWS * D;
    constexpr int SIDE = KR_THREADS / D;
    const int d = threadIdx.x % D, r0 = threadIdx.x / D;
    const int parts = a.splits / a.cluster;
    // value d of a row: the result, or one part of it
    auto emit = [&](int head, int r, float acc, float l, float m, float ref) {
        const int row = row0 + r, t = row / a.G, h = (pack * HPB + head) * a.G + row - t * a.G;
        const int64_t at = ((int64_t)str * a.T + t) * a.H + h;
        if (parts == 1) {
            const float y = l == 0.0f ? 0.0f : acc / l;
            if (a.dst_f16) static_cast<__half*>(a.dst)[at * D + d] = __float2half_rn(y);
            else static_cast<float*>(a.dst)[at * D + d] = y;
        } else {
            const int64_t p = at * parts + split / a.cluster;
            a.part[p * D + d] = acc;
            if (d == 0) {
                a.stat[3 * p] = m;
                a.stat[3 * p + 1] = l;
                a.stat[3 * p + 2] = ref;
            }
        }
    };
#pragma unroll
    for (int head = 0; head < HPB; head++) {
        const float* first = reinterpret_cast<const float*>(sm + head * C::OUT);
        constexpr int STEP = HPB * C::OUT / 4;           // to the head's next warp
#pragma unroll 4
        for (int r = r0; r < rows; r += SIDE) {
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < C::PARTS; w++) m = fmaxf(m, first[w * STEP + KR_ROWS * D + r]);
            const float base = m == -INFINITY ? 0.0f : m;
            float l = 0.0f, acc = 0.0f;
#pragma unroll
            for (int w = 0; w < C::PARTS; w++) {
                const float* p = first + w * STEP;
                const float f = ex2(p[KR_ROWS * D + r] - base);
                l = fmaf(p[KR_ROWS * D + KR_ROWS + r], f, l);
                acc = fmaf(p[r * D + d], f, acc);
            }
            if (a.cluster == 1) {
                emit(head, r, acc, l, m, refs[r]);
            } else {
                cta_out[(head * KR_ROWS + r) * D + d] = acc;
                if (d == 0) cta_stat[2 * (head * KR_ROWS + r)] = m, cta_stat[2 * (head * KR_ROWS + r) + 1] = l;
            }
        }
    }
    if (a.cluster == 1) return;
    cluster_sync();

    // ---- join the CTAs of the cluster, its rows shared out; maxima are compared as maximum plus mask
    // reference, their differences formed apart, where they are exact ----
    for (int hr = crank + r0 * a.cluster; hr < HPB * KR_ROWS; hr += SIDE * a.cluster) {
        const int r = hr % KR_ROWS;
        if (r >= rows) continue;
        float top = -INFINITY, m_best = 0.0f, r_best = 0.0f;
        float l_of[KR_MAX_CLUSTER], e_of[KR_MAX_CLUSTER], ref_at[KR_MAX_CLUSTER], x[KR_MAX_CLUSTER];
#pragma unroll
        for (int c = 0; c < KR_MAX_CLUSTER; c++) {
            l_of[c] = 0.0f, e_of[c] = ref_at[c] = x[c] = 0.0f;
            if (c >= a.cluster) continue;
            const uint32_t st = mapa_shared(smem_u32(cta_stat + 2 * hr), c);
            e_of[c] = ld_cluster_f32(st);
            l_of[c] = ld_cluster_f32(st + 4);
            ref_at[c] = ld_cluster_f32(mapa_shared(smem_u32(refs + r), c));
            x[c] = ld_cluster_f32(mapa_shared(smem_u32(cta_out + hr * D + d), c));
        }
#pragma unroll
        for (int c = 0; c < KR_MAX_CLUSTER; c++) {
            const float v = e_of[c] + ref_at[c] * KR_LOG2E;
            if (l_of[c] != 0.0f && v > top) top = v, m_best = e_of[c], r_best = ref_at[c];
        }
        float l = 0.0f, acc = 0.0f;
#pragma unroll
        for (int c = 0; c < KR_MAX_CLUSTER; c++) {
            // l is 0 where no key is seen
            const float f = l_of[c] == 0.0f ? 0.0f : ex2((e_of[c] - m_best) + (ref_at[c] - r_best) * KR_LOG2E);
            l = fmaf(l_of[c], f, l);
            acc = fmaf(x[c], f, acc);
        }
        emit(hr / KR_ROWS, r, acc, l, m_best, r_best);
    }
    cluster_sync();                                      // no CTA leaves while a peer reads its memory
}

// Joins the parts of a row: one CTA per (stream, token, head), its four warps taking the parts in turn.
// Maxima are compared as maximum plus mask reference; their differences are formed apart, where they are
// exact.
template <int D>
__global__ void __launch_bounds__(128) kvq_join_kernel(const float* __restrict__ part, const float* __restrict__ stat,
                                                       int splits, int dst_f16, void* __restrict__ dst) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float sums[4][D + 1];
    const int64_t row = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* st = stat + 3 * row * splits;
    float top = -INFINITY, m_best = 0.0f, r_best = 0.0f;
    for (int i = lane; i < splits; i += 32) {
        const float m = st[3 * i], l = st[3 * i + 1], r = st[3 * i + 2];
        const float v = m + r * KR_LOG2E;
        if (l != 0.0f && v > top) top = v, m_best = m, r_best = r;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, top, o), m = __shfl_xor_sync(0xffffffffu, m_best, o);
        const float r = __shfl_xor_sync(0xffffffffu, r_best, o);
        // equal sums of different terms: the same pair on every lane
        if (v > top || (v == top && m > m_best)) top = v, m_best = m, r_best = r;
    }
    constexpr int PER = D / 32;
    float acc[PER] = {}, l_all = 0.0f;
#pragma unroll 4
    for (int i = warp; i < splits; i += 4) {
        const float l = st[3 * i + 1];
        // a part with no visible key may hold anything but counts for nothing
        const float f = l == 0.0f ? 0.0f : ex2((st[3 * i] - m_best) + (st[3 * i + 2] - r_best) * KR_LOG2E);
        l_all = fmaf(l, f, l_all);
        const float* p = part + (row * splits + i) * D + lane * PER;
        float x[PER];
        if constexpr (PER == 4) {
            const float4 v = *reinterpret_cast<const float4*>(p);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
            const float2 v = *reinterpret_cast<const float2*>(p);
            x[0] = v.x, x[1] = v.y;
        }
#pragma unroll
        for (int k = 0; k < PER; k++) acc[k] = fmaf(x[k], f, acc[k]);
    }
#pragma unroll
    for (int k = 0; k < PER; k++) sums[warp][lane * PER + k] = acc[k];
    if (lane == 0) sums[warp][D] = l_all;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += 128) {
        const float l = (sums[0][D] + sums[1][D]) + (sums[2][D] + sums[3][D]);
        const float x = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
        const float y = l == 0.0f ? 0.0f : x / l;
        if (dst_f16) static_cast<__half*>(dst)[row * D + d] = __float2half_rn(y);
        else static_cast<float*>(dst)[row * D + d] = y;
    }
}

struct KvqPlan {
    int heads;                                   // KV heads a CTA takes (1: the cp.async kernel)
    int splits, tiles_per_split, cluster;
    size_t part_off, stat_off, total;
};

// tma: the cache's layout lets TMA address it. The workspace covers either kernel.
KvqPlan kvq_plan(int64_t D, int64_t T, int64_t H, int64_t KV, int64_t HK, int64_t S, bool tma) {
    KvqPlan p{};
    p.heads = tma && HK % (256 / D) == 0 ? (int)(256 / D) : 1;
    const int64_t tk = KR_KEYS * KR_WARPS / p.heads;
    const int64_t rows = T * (H / HK), tiles = (KV + tk - 1) / tk;
    const int64_t ctas = S * (HK / p.heads) * ((rows + KR_ROWS - 1) / KR_ROWS);
    // Three CTAs fit an SM, seven eighths of that when they come in clusters. Where it leaves a CTA no more
    // than four tiles, or where a row's keys are spread over sixteen CTAs or more, clusters join the parts
    // (one stream x 16384 keys 24.2 -> 18.1 us, x 512 keys 9.3 -> 8.4). Otherwise CTAs stand alone: clusters
    // wait for their slowest and for room in one GPC (32 streams x 16384 keys 167 us alone, 202 in clusters).
    // Then one wave when the keys are few, several where they are many, with at least KR_MIN_SPLIT keys each,
    // so that streams of unequal length even out, and up to two waves with half as many (8 streams x 16384
    // keys 57.5 -> 53.0 us, 32 x 5000 79 -> 68; for every wave it is slower: 32 x 16384 166 -> 170).
    const int64_t slots = (int64_t)device_sm_count() * 3, fit = slots * 7 / 8;
    int64_t splits = 0;
    p.cluster = 1;
    for (int c = KR_MAX_CLUSTER; c > 1; c /= 2)
        if (ctas * c <= fit && (tiles + c - 1) / c <= 4 && tiles > c / 2) {
            p.cluster = c;
            splits = c;
            break;
        }
    if (!splits && ctas * 2 * KR_MAX_CLUSTER <= fit && tiles >= 2 * KR_MAX_CLUSTER) {
        p.cluster = KR_MAX_CLUSTER;
        splits = std::min(fit / ctas, tiles) / p.cluster * p.cluster;
    }
    if (!splits) {
        splits = std::max<int64_t>(1, slots / ctas);
        splits = std::max(splits, std::min(KR_WAVES * slots / ctas, tiles * tk / KR_MIN_SPLIT));
        splits = std::max(splits, std::min(2 * slots / ctas, 2 * tiles * tk / KR_MIN_SPLIT));
        splits = std::min(splits, tiles);
    }
    splits = std::max(splits, (tiles + KR_MAX_TILES - 1) / KR_MAX_TILES);
    const int64_t per = (tiles + splits - 1) / splits;
    splits = ((tiles + per - 1) / per + p.cluster - 1) / p.cluster * p.cluster;
    p.splits = (int)splits;
    p.tiles_per_split = (int)per;
    const int64_t parts = splits / p.cluster;
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.part_off = 0;
    p.stat_off = parts > 1 ? al((size_t)(S * T * H * parts * D) * 4) : 0;
    p.total = parts > 1 ? p.stat_off + al((size_t)(S * T * H * parts) * 12) : 256;
    return p;
}

// The cache as [streams][keys][bytes of a key's heads], tiles of 144 bytes x `keys`; rows behind the last
// key read as zeros.
bool make_cache_map(CUtensorMap* map, const void* base, int64_t row_bytes, int64_t KV, int64_t S, int64_t nb_key,
                    int64_t nb_stream, int keys) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) != cudaSuccess ||
            qr != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<Encode>(p);
    }();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)row_bytes, (cuuint64_t)KV, (cuuint64_t)S};
    const cuuint64_t strides[2] = {(cuuint64_t)nb_key, (cuuint64_t)nb_stream};
    const cuuint32_t box[3] = {(cuuint32_t)KR_BOX, (cuuint32_t)keys, 1}, step[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int MT, bool QLO, int HPB>
cudaError_t launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const KvqArgs& a, dim3 grid, cudaStream_t st) {
    using C = KrCfg<D, MT, HPB>;
    static bool set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kvq_rows_kernel<D, MT, QLO, HPB>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    return launch_pdl_cluster(kvq_rows_kernel<D, MT, QLO, HPB>, grid, dim3(C::THREADS), C::SMEM, st, a.cluster, tk, tv, a);
}

template <int D, int HPB>
cudaError_t launch_kvq(const CUtensorMap& tk, const CUtensorMap& tv, const KvqArgs& a, cudaStream_t st) {
    const int64_t rows = (int64_t)a.T * a.G;
    const dim3 grid((unsigned)a.splits, (unsigned)(a.HK / HPB * ((rows + KR_ROWS - 1) / KR_ROWS)), (unsigned)a.S);
    // one token a CTA: its mask is one row, and keys it hides are hidden from all the CTA's rows
    const bool one = a.T == 1 || a.G % KR_ROWS == 0;
    cudaError_t e;
    if (one) e = a.q_f16 ? launch_rows<D, 1, false, HPB>(tk, tv, a, grid, st) : launch_rows<D, 1, true, HPB>(tk, tv, a, grid, st);
    else e = a.q_f16 ? launch_rows<D, 8, false, HPB>(tk, tv, a, grid, st) : launch_rows<D, 8, true, HPB>(tk, tv, a, grid, st);
    const int parts = a.splits / a.cluster;
    if (e != cudaSuccess || parts == 1) return e;
    return launch_pdl(kvq_join_kernel<D>, dim3((unsigned)((int64_t)a.S * a.T * a.H)), dim3(128), 0, st,
                      (const float*)a.part, (const float*)a.stat, parts, a.dst_f16, a.dst);
}

// Whether the row kernels take the call, or the tcgen05 kernel over fp16 tiles of the cache. The row kernels take
// some 15 us and 0.95 for every 8 rows of a KV head, the other the time to make the tiles and 0.6 for every query
// tile it has (128 rows, of several heads where a power of two of them shares a KV head). In us, rows / tiles, f16:
// 32 heads of 128 over 8, 16384 keys: 12 tokens 61 / 66, 16 88 / 67; 4096 keys: 12 tokens 25 / 30, 16 30 / 30, 24
// 38 / 31, four streams of them 61 / 67, 88 / 67, 118 / 67; 56 heads over 8, 4096 keys: 16 tokens 44 / 51, 24 53 /
// 51; 14 heads of 64 over 2, 4096 keys: 16 tokens 16 / 21, 32 21 / 22. The number of keys does not enter, so that
// with 1024 the tiles come too early (32 heads over 8: 16 tokens 16 / 25, 48 tokens 23 / 28, 64 31 / 28).
bool by_rows(int64_t T, int64_t H, int64_t HK) {
    const int64_t row_tiles = HK * ((T * (H / HK) + KR_ROWS - 1) / KR_ROWS);
    return 5 * row_tiles <= 25 * HK + 7 * fa_quant_tiles(T, H, HK);
}

// The sizes the grids and 32-bit counters hold.
bool kvq_sizes_ok(int64_t D, int64_t T, int64_t H, int64_t KV, int64_t HK, int64_t S) {
    if ((D != 64 && D != 128) || T <= 0 || T > 65536 || H <= 0 || H > (1 << 20) || KV <= 0 || KV > (1ll << 30) || HK <= 0 ||
        S <= 0 || S > 65535 || H % HK != 0)
        return false;
    const int64_t rows = T * (H / HK);
    if (rows > (1 << 20) || S * T * H > INT32_MAX / 4 || HK * ((rows + KR_ROWS - 1) / KR_ROWS) > 65535) return false;
    // mask blocks of the prompt path: a token at least and 128 keys each
    return by_rows(T, H, HK) || S * T * ((KV + 127) / 128) <= INT32_MAX;
}

}  // namespace

}  // namespace b200

extern "C" {

size_t b200_flash_attn_kvq_workspace_size(int64_t D, int64_t T, int64_t H, int64_t KV, int64_t HK, int64_t S) {
    using namespace b200;
    if (!kvq_sizes_ok(D, T, H, KV, HK, S)) return 0;
    if (!by_rows(T, H, HK)) return fa_quant_workspace(D, T, H, KV, HK, S);
    return std::max(kvq_plan(D, T, H, KV, HK, S, true).total, kvq_plan(D, T, H, KV, HK, S, false).total);
}

int b200_flash_attn_kvq(int kv_type, int q_type, const void* q, const int64_t qne[4], const size_t qnb[4],
                        const void* k, const int64_t kne[4], const size_t knb[4], const void* v, const int64_t vne[4],
                        const size_t vnb[4], const void* mask, const size_t mnb[4], int dst_type, void* dst,
                        float scale, float softcap, void* workspace, size_t workspace_bytes, int* dev_err,
                        void* stream) {
    using namespace b200;
    if (!q || !qne || !qnb || !k || !kne || !knb || !v || !vne || !vnb || (mask && !mnb) || !dst || !dev_err)
        return B200_E_INVALID;
    const int64_t D = qne[0], T = qne[1], H = qne[2], S = qne[3], KV = kne[1], HK = kne[2];
    for (int i = 0; i < 4; i++)
        if (qne[i] <= 0 || kne[i] <= 0 || vne[i] <= 0) return B200_E_INVALID;
    if (kne[0] != D || kne[3] != S || vne[0] != D || vne[1] != KV || vne[2] != HK || vne[3] != S || H % HK != 0)
        return B200_E_INVALID;
    if (kv_type != 2 || (q_type != 0 && q_type != 1) || (dst_type != 0 && dst_type != 1)) return B200_E_UNSUPPORTED;
    const size_t qe = q_type == 1 ? 2 : 4, unit = (size_t)D / 16;
    if (!kvq_sizes_ok(D, T, H, KV, HK, S)) return B200_E_UNSUPPORTED;
    auto off = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
    if (qnb[0] != qe || (qnb[1] | qnb[2] | qnb[3]) % qe != 0 || off(q, qe) || knb[0] != 18 || vnb[0] != 18 ||
        (knb[1] | knb[2] | knb[3] | vnb[1] | vnb[2] | vnb[3]) % unit != 0 || off(k, unit) || off(v, unit) ||
        off(dst, 16))
        return B200_E_UNSUPPORTED;
    if (mask && (mnb[0] != 2 || ((mnb[1] | mnb[3]) & 1) || off(mask, 2))) return B200_E_UNSUPPORTED;
    const size_t need = b200_flash_attn_kvq_workspace_size(D, T, H, KV, HK, S);
    if (!workspace || workspace_bytes < need || off(workspace, 256)) return B200_E_WORKSPACE;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!by_rows(T, H, HK)) {
        FaQuantArgs f{};
        f.q = static_cast<const char*>(q);
        f.q_t = (int64_t)qnb[1], f.q_h = (int64_t)qnb[2], f.q_s = (int64_t)qnb[3], f.q_f16 = q_type == 1;
        f.k = static_cast<const char*>(k), f.k_r = (int64_t)knb[1], f.k_h = (int64_t)knb[2], f.k_s = (int64_t)knb[3];
        f.v = static_cast<const char*>(v), f.v_r = (int64_t)vnb[1], f.v_h = (int64_t)vnb[2], f.v_s = (int64_t)vnb[3];
        f.mask = static_cast<const char*>(mask);
        f.m_t = mask ? (int64_t)mnb[1] : 0, f.m_s = mask ? (int64_t)mnb[3] : 0;
        f.m_vec = mask && ((mnb[1] | mnb[3]) & 15) == 0 && !off(mask, 16);
        f.dst = dst, f.dst_f16 = dst_type == 1;
        f.D = (int)D, f.T = (int)T, f.H = (int)H, f.KV = (int)KV, f.HK = (int)HK, f.S = (int)S;
        f.scale = scale, f.softcap = softcap, f.err = dev_err;
        const cudaError_t e = fa_quant_run(f, static_cast<char*>(workspace), st);
        return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? B200_OK : B200_E_CUDA;
    }
    const int64_t row = D / 32 * 18;
    // what a tensor map of the cache needs: heads side by side, 16-byte bases and strides, strides below 2^40
    auto tma_ok = [&](const void* p, const size_t* s) {
        return (int64_t)s[2] == row && ((s[1] | s[3]) & 15) == 0 && !off(p, 16) && (int64_t)s[1] >= HK * row &&
               s[1] < (1ull << 40) && s[3] < (1ull << 40) && (S == 1 || s[3] > 0);
    };
    const KvqPlan p = kvq_plan(D, T, H, KV, HK, S, tma_ok(k, knb) && tma_ok(v, vnb));
    KvqArgs a{};
    a.q = static_cast<const char*>(q);
    a.q_t = (int64_t)qnb[1], a.q_h = (int64_t)qnb[2], a.q_s = (int64_t)qnb[3];
    a.q_f16 = q_type == 1;
    a.q_vec = (qnb[1] | qnb[2] | qnb[3]) % (4 * qe) == 0 && !off(q, 4 * qe);
    a.k = static_cast<const char*>(k);
    a.k_r = (int64_t)knb[1], a.k_h = (int64_t)knb[2], a.k_s = (int64_t)knb[3];
    a.v = static_cast<const char*>(v);
    a.v_r = (int64_t)vnb[1], a.v_h = (int64_t)vnb[2], a.v_s = (int64_t)vnb[3];
    a.mask = static_cast<const char*>(mask);
    a.m_t = mask ? (int64_t)mnb[1] : 0, a.m_s = mask ? (int64_t)mnb[3] : 0;
    a.m_vec = mask && ((mnb[1] | mnb[3]) & 15) == 0 && !off(mask, 16);
    a.dst = dst;
    a.dst_f16 = dst_type == 1;
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.part_off);
    a.stat = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.stat_off);
    a.T = (int)T, a.H = (int)H, a.KV = (int)KV, a.HK = (int)HK, a.G = (int)(H / HK), a.S = (int)S;
    a.splits = p.splits, a.tiles_per_split = p.tiles_per_split, a.cluster = p.cluster;
    a.scale = scale, a.softcap = softcap;
    a.err = dev_err;
    CUtensorMap tk{}, tv{};
    if (p.heads > 1) {
        const int keys = KR_KEYS * KR_WARPS / p.heads;
        // a single stream's stride is never used but has to be one a map accepts
        const int64_t ks = S > 1 ? (int64_t)knb[3] : 16, vs = S > 1 ? (int64_t)vnb[3] : 16;
        if (!make_cache_map(&tk, k, HK * row, KV, S, (int64_t)knb[1], ks, keys) ||
            !make_cache_map(&tv, v, HK * row, KV, S, (int64_t)vnb[1], vs, keys))
            return B200_E_CUDA;
    }
    cudaError_t e;
    if (D == 64) e = p.heads > 1 ? launch_kvq<64, 4>(tk, tv, a, st) : launch_kvq<64, 1>(tk, tv, a, st);
    else e = p.heads > 1 ? launch_kvq<128, 2>(tk, tv, a, st) : launch_kvq<128, 1>(tk, tv, a, st);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? B200_OK : B200_E_CUDA;
}

}  // extern "C"
