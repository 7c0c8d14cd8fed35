// FLASH_ATTN_EXT over a Q4_0 KV cache, read as it is stored (the reference's attention handler takes
// F16 K / V only, ggml-rocket.cpp:7654-7700, and leaves a quantised cache to its host):
//
//     dst[s, t, h] = sum_j softmax_j(scale q[s, t, h] . k[s, j, hk] (capped) + mask[s, t, j]) v[s, j, hk]
//
// with hk = h / (H / HK). A key whose mask is -inf is not read into the result, whatever its bytes
// hold; a row whose keys are all masked is zero.
//
// The row kernel. A CTA takes 8 of the T * (H / HK) query rows that share a KV head, one stream and one
// range of keys; its four warps take the range's 32-key tiles in turn, each with its own ring of
// cp.async stages, running maximum, sum and output, so nothing but the end is shared between them.
// Tiles whose keys are masked for all the rows are never fetched: the CTA reads its mask range first.
//
//   S = Q K^T     mma.sync m16n8k16, 8 keys a tile. Rows 0-7 of the A operand are the query rows'
//                 fp16 high halves, rows 8-15 their low halves (q = hi + lo to 2^-22, scaled by a power
//                 of two into fp16's range), so both come out of one MMA. B holds the 4-bit codes as
//                 exact integers in fp16; the block scales multiply the fp32 sums of each 32 values.
//   O^T = V^T P^T the codes are the A operand (16 head dimensions x 16 keys), P times the value
//                 scales the B operand, straight from the score fragments' layout.
//
// P * scale is brought into fp16's range by a power of two per tile (the tile's largest value scale)
// and, for an f32 result, split into a high and a low half as well; for an fp16 result its rounding
// (2^-12) stays below the result's own. Sums, maxima and outputs are fp32 throughout; a tile's output
// sums are added to the running ones by an fp32 FMA.
//
// Scores are in log2 units, taken relative to the largest mask value of the row in the CTA's range,
// whose difference to a key's mask is exact in fp32 also when every mask value is fp16's lowest.
//
// With few rows the keys are split over CTAs and a second kernel joins the parts.
#include <algorithm>
#include <cmath>
#include <cstdint>

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
constexpr int KR_TILE = 32;            // keys per tile
constexpr int KR_STAGES = 3;
constexpr int KR_MAX_TILES = 2048;     // tiles of a CTA's range (its list of live tiles)
constexpr float KR_LOG2E = 1.4426950408889634f;

struct KvqArgs {
    const char* q;
    int64_t q_t, q_h, q_s;             // byte strides of q: token, head, stream
    int q_f16;
    const char* k;
    int64_t k_r, k_h, k_s;             // byte strides of k: key, head, stream
    const char* v;
    int64_t v_r, v_h, v_s;
    const char* mask;                  // f16 or nullptr
    int64_t m_t, m_s;                  // byte strides: token, stream
    void* dst;                         // [S][T][H][D]
    int dst_f16;
    float* part;                       // [S][HK][rows][splits][D] outputs, then 3 floats a part
    float* stat;                       // {max (log2 units, relative), sum, mask reference}
    int T, H, KV, HK, G, S;
    int splits, tiles_per_split;
    float scale, softcap;
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
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    uint16_t v;
    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(a));
    return v;
}

template <int D>
struct KrCfg {
    static constexpr int NB = D / 32;              // blocks of a head's row
    static constexpr int CH = D / 16;              // bytes of a cp.async: nine of them make a head's row
    static constexpr int PITCH = D == 128 ? 80 : 40;   // of a row in shared memory: the eight rows a fragment
                                                       // load touches fall into different banks
    static constexpr int HALF = KR_TILE * PITCH;
    static constexpr int STAGE = 2 * HALF;         // K rows, then V rows
    static constexpr int SCL = KR_TILE * NB * 2;   // a tile's scales (fp16), K then V
    static constexpr int OFF_SCL = KR_STAGES * STAGE;
    static constexpr int OFF_MSK = OFF_SCL + 2 * SCL;
    static constexpr int WARP(int mt) { return OFF_MSK + mt * KR_TILE * 4; }
    static constexpr int OUT = KR_ROWS * D * 4 + 2 * KR_ROWS * 4;
    static constexpr int OFF_LIST(int mt) { return KR_WARPS * (WARP(mt) > OUT ? WARP(mt) : OUT); }
    static constexpr int OFF_REF(int mt) { return OFF_LIST(mt) + KR_MAX_TILES * 2; }
    static constexpr int SMEM(int mt) { return OFF_REF(mt) + KR_WARPS * KR_ROWS * 4 + 16; }
};

// MT: the most tokens a CTA's rows come from (1 or 8). EXACT: f32 results (P split in two halves).
template <int D, int MT, bool EXACT>
__global__ void __launch_bounds__(KR_THREADS) kvq_rows_kernel(const KvqArgs a) {
    using C = KrCfg<D>;
    extern __shared__ __align__(16) uint8_t sm[];
    grid_dep_wait();
    grid_dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int split = blockIdx.x, hk = blockIdx.y % a.HK, rt = blockIdx.y / a.HK, str = blockIdx.z;
    const int rows_all = a.T * a.G, row0 = rt * KR_ROWS;
    const int rows = min(KR_ROWS, rows_all - row0);
    const int t_first = row0 / a.G, n_tok = MT == 1 ? 1 : (row0 + rows - 1) / a.G - t_first + 1;
    const int n_tiles = (a.KV + KR_TILE - 1) / KR_TILE;
    const int tile0 = split * a.tiles_per_split, tile1 = min(n_tiles, tile0 + a.tiles_per_split);
    uint16_t* list = reinterpret_cast<uint16_t*>(sm + C::OFF_LIST(MT));
    float* refs = reinterpret_cast<float*>(sm + C::OFF_REF(MT));           // [warp][8]
    int* n_live = reinterpret_cast<int*>(sm + C::OFF_REF(MT) + KR_WARPS * KR_ROWS * 4);

    // ---- the range's mask: live tiles and each token's largest mask value ----
    const char* mbase = a.mask ? a.mask + (int64_t)str * a.m_s + (int64_t)t_first * a.m_t : nullptr;
    float ref = 0.0f;                                    // of this lane's row (g)
    const int my_tok = MT == 1 ? 0 : min(row0 + g, rows_all - 1) / a.G - t_first;
    if (mbase) {
        float top[MT];
#pragma unroll
        for (int k = 0; k < MT; k++) top[k] = -INFINITY;
        for (int i = tile0 + warp; i < tile1; i += KR_WARPS) {
            const int key = i * KR_TILE + lane;
            bool any = false;
#pragma unroll
            for (int k = 0; k < MT; k++) {
                if (k >= n_tok || key >= a.KV) continue;
                const float m = __half2float(*reinterpret_cast<const __half*>(mbase + k * a.m_t + 2 * (int64_t)key));
                any |= !(m == -INFINITY);
                top[k] = fmaxf(top[k], m);
            }
            const bool on = __any_sync(0xffffffffu, any);
            if (lane == 0) list[i - tile0] = on ? 1 : 0;
        }
#pragma unroll
        for (int k = 0; k < MT; k++) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
            if (lane == 0) refs[warp * KR_ROWS + k] = top[k];
        }
        __syncthreads();
        ref = -INFINITY;
#pragma unroll
        for (int w = 0; w < KR_WARPS; w++) ref = fmaxf(ref, refs[w * KR_ROWS + my_tok]);
        if (!(fabsf(ref) <= 65504.0f)) ref = 0.0f;       // all masked (or an infinite mask): nothing to gain
        if (warp == 0) {                                 // the live tiles in order, in place
            int n = 0;
            for (int i0 = 0; i0 < tile1 - tile0; i0 += 32) {
                const int i = i0 + lane;
                const bool on = i < tile1 - tile0 && list[i] != 0;
                const uint32_t votes = __ballot_sync(0xffffffffu, on);
                if (on) list[n + __popc(votes & ((1u << lane) - 1u))] = (uint16_t)i;
                n += __popc(votes);
                __syncwarp();
            }
            if (lane == 0) *n_live = n;
        }
    } else {
        for (int i = threadIdx.x; i < tile1 - tile0; i += KR_THREADS) list[i] = (uint16_t)i;
        if (threadIdx.x == 0) *n_live = max(0, tile1 - tile0);
    }
    __syncthreads();
    const int live = *n_live;

    // ---- q: high and low halves of the row, times a power of two that brings its maximum to 2^10 ----
    uint32_t qa[2 * C::NB][4];
    float back = 1.0f;                                   // what undoes it, with the scale
    {
        const int r = row0 + g;
        const bool in = g < rows;
        const int t = in ? r / a.G : 0, h = hk * a.G + (in ? r - t * a.G : 0);
        const char* qp = a.q + (int64_t)str * a.q_s + (int64_t)t * a.q_t + (int64_t)h * a.q_h;
        float x[C::NB][8];
        float amax = 0.0f;
#pragma unroll
        for (int b = 0; b < C::NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = 32 * b + 16 * (e >> 2) + 4 * t4 + (e & 3);
                float v = 0.0f;
                if (in) v = a.q_f16 ? __half2float(reinterpret_cast<const __half*>(qp)[d]) : reinterpret_cast<const float*>(qp)[d];
                x[b][e] = v;
                amax = fmaxf(amax, fabsf(v));
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int ex = 0;
        if (amax > 0.0f && amax <= 3.402823466e38f) frexpf(amax, &ex);
        ex = max(-100, ex - 10);
        const float mul = ldexpf(1.0f, -ex);
        back = ldexpf(a.scale, ex);
#pragma unroll
        for (int b = 0; b < C::NB; b++)
#pragma unroll
            for (int s = 0; s < 2; s++) {                // k-step 2b + s: values 16 s + {0, 2}, then {1, 3}
                float hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = x[b][4 * s + e] * mul;
                    hi[e] = __half2float(__float2half_rn(v));
                    lo[e] = v - hi[e];
                }
                qa[2 * b + s][0] = pack_half2(hi[0], hi[2]);
                qa[2 * b + s][1] = pack_half2(lo[0], lo[2]);
                qa[2 * b + s][2] = pack_half2(hi[1], hi[3]);
                qa[2 * b + s][3] = pack_half2(lo[1], lo[3]);
            }
    }

    // ---- the warp's own stages ----
    const uint32_t wsm = smem_u32(sm) + warp * (C::WARP(MT) > C::OUT ? C::WARP(MT) : C::OUT);
    const int c_row = lane / 9, c_chunk = lane - 9 * c_row;   // lanes 0-26: three rows of nine pieces
    const char* kp = a.k + (int64_t)str * a.k_s + (int64_t)hk * a.k_h + c_chunk * C::CH;
    const char* vp = a.v + (int64_t)str * a.v_s + (int64_t)hk * a.v_h + c_chunk * C::CH;
    auto fetch = [&](int i) {                                 // the i-th live tile of this warp
        const int e = warp + i * KR_WARPS;
        if (e < live && lane < 27) {
            const int key0 = (tile0 + list[e]) * KR_TILE;
            const uint32_t d = wsm + (i % KR_STAGES) * C::STAGE + c_row * C::PITCH + c_chunk * C::CH;
#pragma unroll
            for (int n = 0; n < 11; n++) {
                const int row = 3 * n + c_row;
                if (n == 10 && row >= KR_TILE) break;
                const bool in = key0 + row < a.KV;
                const int64_t key = in ? key0 + row : a.KV - 1;
                cp_async<C::CH>(d + 3 * n * C::PITCH, kp + key * a.k_r, in);
                cp_async<C::CH>(d + 3 * n * C::PITCH + C::HALF, vp + key * a.v_r, in);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < KR_STAGES - 1; i++) fetch(i);

    float o[2 * C::NB][4];
#pragma unroll
    for (int m = 0; m < 2 * C::NB; m++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[m][e] = 0.0f;
    float run_max = -INFINITY, run_sum = 0.0f;           // of row g (the sum: this lane's keys)
    int unit = 0;                                        // o is in units of 2^unit
    const uint32_t scl = wsm + C::OFF_SCL, msk = wsm + C::OFF_MSK;

    for (int i = 0; warp + i * KR_WARPS < live; i++) {
        const int key0 = (tile0 + list[warp + i * KR_WARPS]) * KR_TILE;
        float mv[MT];                                    // key key0 + lane's mask, per token
        bool seen = key0 + lane < a.KV;
        if (mbase) {
            bool any = false;
#pragma unroll
            for (int k = 0; k < MT; k++) {
                mv[k] = -INFINITY;
                if (k < n_tok && seen)
                    mv[k] = __half2float(*reinterpret_cast<const __half*>(mbase + k * a.m_t + 2 * (int64_t)(key0 + lane)));
                any |= !(mv[k] == -INFINITY);
            }
            seen = any;
        } else {
#pragma unroll
            for (int k = 0; k < MT; k++) mv[k] = seen ? 0.0f : -INFINITY;
        }
        cp_async_wait<KR_STAGES - 2>();
        __syncwarp();
        const uint32_t ks = wsm + (i % KR_STAGES) * C::STAGE, vs = ks + C::HALF;
        // the scales of key `lane`, apart from the codes; a key no row sees gets zeros
        uint32_t dk[C::NB / 2], dv[C::NB / 2];
        float vmax = 0.0f;
#pragma unroll
        for (int p = 0; p < C::NB / 2; p++) {
            const uint32_t rk = ks + lane * C::PITCH + 36 * p, rv = vs + lane * C::PITCH + 36 * p;
            dk[p] = lds16(rk) | (lds16(rk + 18) << 16);
            dv[p] = lds16(rv) | (lds16(rv + 18) << 16);
            if (!seen) dk[p] = dv[p] = 0;
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&dv[p]));
            vmax = fmaxf(vmax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        if constexpr (C::NB == 4) {
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(scl + lane * 8), "r"(dk[0]), "r"(dk[1]) : "memory");
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(scl + C::SCL + lane * 8), "r"(dv[0]), "r"(dv[1]) : "memory");
        } else {
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(scl + lane * 4), "r"(dk[0]) : "memory");
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(scl + C::SCL + lane * 4), "r"(dv[0]) : "memory");
        }
#pragma unroll
        for (int k = 0; k < MT; k++)
            if (k < n_tok)
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(msk + (k * KR_TILE + lane) * 4), "f"(mv[k]) : "memory");
        // the power of two that brings the tile's largest value scale to at most 2^11
        const uint32_t vbits = __reduce_max_sync(0xffffffffu, __float_as_uint(vmax));
        int vexp = (int)(vbits >> 23) - 127 - 10;
        if (vbits == 0 || vbits >= 0x7f800000u) vexp = 0;
        const float vmul = __uint_as_float((uint32_t)(127 - vexp) << 23);
        __syncwarp();

        // ---- S = Q K^T ----
        float s[4][2];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float s0 = 0.0f, s1 = 0.0f;
            uint32_t dd[C::NB];                          // scales of keys 8j + 2 t4 and + 1
            const uint32_t da = scl + (8 * j + 2 * t4) * (C::NB * 2);
            if constexpr (C::NB == 4)
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(dd[0]), "=r"(dd[1]), "=r"(dd[2]), "=r"(dd[3]) : "r"(da));
            else
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(dd[0]), "=r"(dd[1]) : "r"(da));
            const uint32_t kr = ks + (8 * j + g) * C::PITCH + 4 * t4;
#pragma unroll
            for (int p = 0; p < C::NB / 2; p++) {
                const float2 e0 = __half22float2(*reinterpret_cast<const __half2*>(&dd[p]));
                const float2 e1 = __half22float2(*reinterpret_cast<const __half2*>(&dd[C::NB / 2 + p]));
                const uint32_t w0 = lds32(kr + 36 * p), w1 = lds32(kr + 36 * p + 4), w2 = lds32(kr + 36 * p + 20);
                uint32_t f[4];
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                codes_f16(__byte_perm(w0, w1, 0x5432), f);
                mma_16816(c, qa[4 * p][0], qa[4 * p][1], qa[4 * p][2], qa[4 * p][3], f[0], f[2]);
                mma_16816(c, qa[4 * p + 1][0], qa[4 * p + 1][1], qa[4 * p + 1][2], qa[4 * p + 1][3], f[1], f[3]);
                s0 = fmaf(e0.x, c[0] + c[2], s0);
                s1 = fmaf(e1.x, c[1] + c[3], s1);
                float c2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                codes_f16(w2, f);
                mma_16816(c2, qa[4 * p + 2][0], qa[4 * p + 2][1], qa[4 * p + 2][2], qa[4 * p + 2][3], f[0], f[2]);
                mma_16816(c2, qa[4 * p + 3][0], qa[4 * p + 3][1], qa[4 * p + 3][2], qa[4 * p + 3][3], f[1], f[3]);
                s0 = fmaf(e0.y, c2[0] + c2[2], s0);
                s1 = fmaf(e1.y, c2[1] + c2[3], s1);
            }
            s0 *= back, s1 *= back;
            if (a.softcap != 0.0f) {
                s0 = a.softcap * tanhf(s0 / a.softcap);
                s1 = a.softcap * tanhf(s1 / a.softcap);
            }
            float m0, m1;
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(m0), "=f"(m1) : "r"(msk + (my_tok * KR_TILE + 8 * j + 2 * t4) * 4));
            s[j][0] = m0 == -INFINITY ? -INFINITY : (s0 + (m0 - ref)) * KR_LOG2E;
            s[j][1] = m1 == -INFINITY ? -INFINITY : (s1 + (m1 - ref)) * KR_LOG2E;
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

        // ---- O^T = V^T P^T over the tile ----
        float ot[2 * C::NB][4];
#pragma unroll
        for (int m = 0; m < 2 * C::NB; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) ot[m][e] = 0.0f;
#pragma unroll
        for (int jj = 0; jj < 2; jj++) {
            uint32_t da[C::NB], db[C::NB];               // value scales of keys 16 jj + 2 t4, + 1 and those 8 on
            const uint32_t dp = scl + C::SCL + (16 * jj + 2 * t4) * (C::NB * 2);
            if constexpr (C::NB == 4) {
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(da[0]), "=r"(da[1]), "=r"(da[2]), "=r"(da[3]) : "r"(dp));
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(db[0]), "=r"(db[1]), "=r"(db[2]), "=r"(db[3]) : "r"(dp + 8 * C::NB * 2));
            } else {
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(da[0]), "=r"(da[1]) : "r"(dp));
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(db[0]), "=r"(db[1]) : "r"(dp + 8 * C::NB * 2));
            }
            float pv[4] = {s[2 * jj][0] * vmul, s[2 * jj][1] * vmul, s[2 * jj + 1][0] * vmul, s[2 * jj + 1][1] * vmul};
            const uint32_t vr = vs + (16 * jj + 2 * t4) * C::PITCH + 2 + 2 * g;
#pragma unroll
            for (int b = 0; b < C::NB; b++) {
                const int p = b >> 1;
                const float2 x0 = __half22float2(*reinterpret_cast<const __half2*>(&da[p]));
                const float2 x1 = __half22float2(*reinterpret_cast<const __half2*>(&da[C::NB / 2 + p]));
                const float2 x2 = __half22float2(*reinterpret_cast<const __half2*>(&db[p]));
                const float2 x3 = __half22float2(*reinterpret_cast<const __half2*>(&db[C::NB / 2 + p]));
                float w[4] = {pv[0] * ((b & 1) ? x0.y : x0.x), pv[1] * ((b & 1) ? x1.y : x1.x),
                              pv[2] * ((b & 1) ? x2.y : x2.x), pv[3] * ((b & 1) ? x3.y : x3.x)};
                if constexpr (MT > 1) {                  // a key other rows see: its scale may be no number
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = pv[e] == 0.0f ? 0.0f : w[e];
                }
                const uint32_t b0 = pack_half2(w[0], w[1]), b1 = pack_half2(w[2], w[3]);
                const uint32_t va = vr + 18 * b;
                const uint32_t y0 = lds16(va) | (lds16(va + C::PITCH) << 16);
                const uint32_t y1 = lds16(va + 8 * C::PITCH) | (lds16(va + 9 * C::PITCH) << 16);
                uint32_t f0[4], f1[4];                   // {2g, 16 + 2g, 2g + 1, 17 + 2g} of the block, key pairs
                codes_f16(y0, f0);
                codes_f16(y1, f1);
                mma_16816(ot[2 * b], f0[0], f0[1], f1[0], f1[1], b0, b1);
                mma_16816(ot[2 * b + 1], f0[2], f0[3], f1[2], f1[3], b0, b1);
                if constexpr (EXACT) {
                    const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&b0));
                    const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&b1));
                    const uint32_t l0 = pack_half2(w[0] - h0.x, w[1] - h0.y), l1 = pack_half2(w[2] - h1.x, w[3] - h1.y);
                    mma_16816(ot[2 * b], f0[0], f0[1], f1[0], f1[1], l0, l1);
                    mma_16816(ot[2 * b + 1], f0[2], f0[3], f1[2], f1[3], l0, l1);
                }
            }
        }
        // columns 2 t4 and 2 t4 + 1 of o are those query rows: their alpha, and the change of unit
        const float f = ldexpf(1.0f, max(-126, min(126, unit - vexp)));
        unit = vexp;
        const float al0 = __shfl_sync(0xffffffffu, alpha, 8 * t4) * f;
        const float al1 = __shfl_sync(0xffffffffu, alpha, 8 * t4 + 4) * f;
#pragma unroll
        for (int m = 0; m < 2 * C::NB; m++) {
            o[m][0] = fmaf(o[m][0], al0, ot[m][0]);
            o[m][1] = fmaf(o[m][1], al1, ot[m][1]);
            o[m][2] = fmaf(o[m][2], al0, ot[m][2]);
            o[m][3] = fmaf(o[m][3], al1, ot[m][3]);
        }
        __syncwarp();                                    // the stage and the scales are free again
        fetch(i + KR_STAGES - 1);
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- join the warps ----
    float* wout = reinterpret_cast<float*>(sm + warp * (C::WARP(MT) > C::OUT ? C::WARP(MT) : C::OUT));
    run_sum += __shfl_xor_sync(0xffffffffu, run_sum, 1);
    run_sum += __shfl_xor_sync(0xffffffffu, run_sum, 2);
    const float lift = ldexpf(1.0f, unit);
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
    float* wstat = wout + KR_ROWS * D;
    if (t4 == 0) {
        wstat[g] = run_max;
        wstat[KR_ROWS + g] = run_sum;
        if (warp == 0) refs[g] = ref;                    // per row from here on
    }
    __syncthreads();
    constexpr int WSTRIDE = (C::WARP(MT) > C::OUT ? C::WARP(MT) : C::OUT) / 4;
    const float* all = reinterpret_cast<const float*>(sm);
    for (int r = threadIdx.x / D; r < rows; r += KR_THREADS / D) {
        const int d = threadIdx.x % D;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < KR_WARPS; w++) m = fmaxf(m, all[w * WSTRIDE + KR_ROWS * D + r]);
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < KR_WARPS; w++) {
            const float* p = all + w * WSTRIDE;
            const float e = ex2(p[KR_ROWS * D + r] - base);
            l = fmaf(p[KR_ROWS * D + KR_ROWS + r], e, l);
            acc = fmaf(p[r * D + d], e, acc);
        }
        const int row = row0 + r, t = row / a.G, h = hk * a.G + row - t * a.G;
        if (a.splits == 1) {
            const float y = l == 0.0f ? 0.0f : acc / l;
            const int64_t at = (((int64_t)str * a.T + t) * a.H + h) * D + d;
            if (a.dst_f16) static_cast<__half*>(a.dst)[at] = __float2half_rn(y);
            else static_cast<float*>(a.dst)[at] = y;
        } else {
            const int64_t p = (((int64_t)str * a.T + t) * a.H + h) * a.splits + split;
            a.part[p * D + d] = acc;
            if (d == 0) {
                a.stat[3 * p] = m;
                a.stat[3 * p + 1] = l;
                a.stat[3 * p + 2] = refs[r];
            }
        }
    }
}

// Joins the parts of a row: one warp per (stream, token, head). Maxima are compared as maximum plus
// mask reference; their differences are formed apart, where they are exact.
template <int D>
__global__ void __launch_bounds__(128) kvq_join_kernel(const float* __restrict__ part, const float* __restrict__ stat,
                                                       int splits, int64_t n_rows, int dst_f16, void* __restrict__ dst) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= n_rows) return;
    const int lane = threadIdx.x & 31;
    const float* st = stat + 3 * row * splits;
    float top = -INFINITY, m_best = 0.0f, r_best = 0.0f;
    for (int i = 0; i < splits; i++) {
        const float l = st[3 * i + 1], m = st[3 * i], r = st[3 * i + 2];
        const float v = m + r * KR_LOG2E;
        if (l != 0.0f && v > top) top = v, m_best = m, r_best = r;
    }
    constexpr int PER = D / 32;
    float acc[PER] = {}, l_all = 0.0f;
    for (int i = 0; i < splits; i++) {
        const float l = st[3 * i + 1];
        if (l == 0.0f) continue;                         // no key of this part is seen
        const float e = ex2((st[3 * i] - m_best) + (st[3 * i + 2] - r_best) * KR_LOG2E);
        l_all = fmaf(l, e, l_all);
        const float* p = part + (row * splits + i) * D + lane * PER;
#pragma unroll
        for (int k = 0; k < PER; k++) acc[k] = fmaf(p[k], e, acc[k]);
    }
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const float y = l_all == 0.0f ? 0.0f : acc[k] / l_all;
        const int64_t at = row * D + lane * PER + k;
        if (dst_f16) static_cast<__half*>(dst)[at] = __float2half_rn(y);
        else static_cast<float*>(dst)[at] = y;
    }
}

struct KvqPlan {
    int splits, tiles_per_split;
    size_t part_off, stat_off, total;
};

KvqPlan kvq_plan(int64_t D, int64_t T, int64_t H, int64_t KV, int64_t HK, int64_t S) {
    KvqPlan p{};
    const int64_t rows = T * (H / HK), tiles = (KV + KR_TILE - 1) / KR_TILE;
    const int64_t ctas = S * HK * ((rows + KR_ROWS - 1) / KR_ROWS);
    const int64_t target = (int64_t)device_sm_count() * 3;   // three CTAs an SM
    int64_t splits = std::max<int64_t>(1, target / ctas);
    splits = std::min(splits, (tiles + KR_WARPS - 1) / KR_WARPS);
    splits = std::max(splits, (tiles + KR_MAX_TILES - 1) / KR_MAX_TILES);
    const int64_t per = (tiles + splits - 1) / splits;
    splits = (tiles + per - 1) / per;
    p.splits = (int)splits;
    p.tiles_per_split = (int)per;
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.part_off = 0;
    p.stat_off = splits > 1 ? al((size_t)(S * T * H * splits * D) * 4) : 0;
    p.total = splits > 1 ? p.stat_off + al((size_t)(S * T * H * splits) * 12) : 256;
    return p;
}

template <int D, int MT, bool EXACT>
cudaError_t launch_rows(const KvqArgs& a, dim3 grid, cudaStream_t st) {
    constexpr int smem = KrCfg<D>::SMEM(MT);
    static bool set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kvq_rows_kernel<D, MT, EXACT>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        set[dev] = true;
    }
    return launch_pdl(kvq_rows_kernel<D, MT, EXACT>, grid, dim3(KR_THREADS), smem, st, a);
}

template <int D>
cudaError_t launch_kvq(const KvqArgs& a, const KvqPlan& p, cudaStream_t st) {
    const int64_t rows = (int64_t)a.T * a.G;
    const dim3 grid((unsigned)p.splits, (unsigned)(a.HK * ((rows + KR_ROWS - 1) / KR_ROWS)), (unsigned)a.S);
    cudaError_t e;
    if (a.T == 1) e = a.dst_f16 ? launch_rows<D, 1, false>(a, grid, st) : launch_rows<D, 1, true>(a, grid, st);
    else e = a.dst_f16 ? launch_rows<D, 8, false>(a, grid, st) : launch_rows<D, 8, true>(a, grid, st);
    if (e != cudaSuccess || p.splits == 1) return e;
    const int64_t n = (int64_t)a.S * a.T * a.H;
    return launch_pdl(kvq_join_kernel<D>, dim3((unsigned)((n + 3) / 4)), dim3(128), 0, st, (const float*)a.part,
                      (const float*)a.stat, p.splits, n, a.dst_f16, a.dst);
}

bool kvq_dims_ok(int64_t D, int64_t T, int64_t H, int64_t KV, int64_t HK, int64_t S) {
    return (D == 64 || D == 128) && T > 0 && H > 0 && KV > 0 && HK > 0 && S > 0 && H % HK == 0;
}

}  // namespace

}  // namespace b200

extern "C" {

size_t b200_flash_attn_kvq_workspace_size(int64_t D, int64_t T, int64_t H, int64_t KV, int64_t HK, int64_t S) {
    using namespace b200;
    if (!kvq_dims_ok(D, T, H, KV, HK, S)) return 0;
    return kvq_plan(D, T, H, KV, HK, S).total;
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
    if (!kvq_dims_ok(D, T, H, KV, HK, S) || T > 65536 || S > 65535 || KV > (1ll << 30) || T * (H / HK) > (1 << 20) ||
        HK * ((T * (H / HK) + KR_ROWS - 1) / KR_ROWS) > 65535)
        return B200_E_UNSUPPORTED;
    auto off = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
    if (qnb[0] != qe || (qnb[1] | qnb[2] | qnb[3]) % qe != 0 || off(q, qe) || knb[0] != 18 || vnb[0] != 18 ||
        (knb[1] | knb[2] | knb[3] | vnb[1] | vnb[2] | vnb[3]) % unit != 0 || off(k, unit) || off(v, unit) ||
        off(dst, dst_type == 1 ? 2 : 4))
        return B200_E_UNSUPPORTED;
    if (mask && (mnb[0] != 2 || ((mnb[1] | mnb[3]) & 1) || off(mask, 2))) return B200_E_UNSUPPORTED;
    const KvqPlan p = kvq_plan(D, T, H, KV, HK, S);
    if (!workspace || workspace_bytes < p.total || off(workspace, 256)) return B200_E_WORKSPACE;
    KvqArgs a{};
    a.q = static_cast<const char*>(q);
    a.q_t = (int64_t)qnb[1], a.q_h = (int64_t)qnb[2], a.q_s = (int64_t)qnb[3];
    a.q_f16 = q_type == 1;
    a.k = static_cast<const char*>(k);
    a.k_r = (int64_t)knb[1], a.k_h = (int64_t)knb[2], a.k_s = (int64_t)knb[3];
    a.v = static_cast<const char*>(v);
    a.v_r = (int64_t)vnb[1], a.v_h = (int64_t)vnb[2], a.v_s = (int64_t)vnb[3];
    a.mask = static_cast<const char*>(mask);
    a.m_t = mask ? (int64_t)mnb[1] : 0, a.m_s = mask ? (int64_t)mnb[3] : 0;
    a.dst = dst;
    a.dst_f16 = dst_type == 1;
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.part_off);
    a.stat = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.stat_off);
    a.T = (int)T, a.H = (int)H, a.KV = (int)KV, a.HK = (int)HK, a.G = (int)(H / HK), a.S = (int)S;
    a.splits = p.splits, a.tiles_per_split = p.tiles_per_split;
    a.scale = scale, a.softcap = softcap;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = D == 64 ? launch_kvq<64>(a, p, st) : launch_kvq<128>(a, p, st);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? B200_OK : B200_E_CUDA;
}

}  // extern "C"
