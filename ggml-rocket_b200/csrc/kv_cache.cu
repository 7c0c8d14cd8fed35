// A KV cache quantised as it is written (SET_ROWS) and read back (GET_ROWS over Q4_0 / Q8_0).
//
// The reference leaves both to the host's CPU backend (its supports_op claims neither,
// ggml-rocket.cpp:7410-7772). Formats are ggml's: blocks of 32 values, an fp16 scale d, then the codes.
//   Q4_0  m = the block's value of largest size (the first of equals), d = m / -8,
//         code = min(15, trunc(x * id + 8.5)), id = 1 / d in f32 (0 when d is 0); element j < 16 is
//         the low nibble of byte j, element j + 16 its high nibble; a code c stands for (c - 8) d.
//         The product and sum are not rounded before the truncation: one FMA rounded toward zero
//         truncates to the same integer as the exact value. ggml rounds both to f32, so that about one
//         code in two million, next to a border, differs by one; the exact one is the nearer to x.
//   Q8_0  d = amax / 127, code = roundf(x * id), the product rounded to f32; it stands for code * d.
//
// Both are bound by HBM (4 bytes a value on the f32 side, 0.5625 / 1.0625 on the other; no reuse).
// Eight lanes take a block, four consecutive values each, so a warp reads or writes 512 consecutive
// bytes of f32 with one 16-byte access per lane; the block's maximum is three shuffles. Blocks are
// only 2-byte aligned, so codes and scales move as 2-byte words, which L1 and L2 join into sectors.
//
// Q8_0 rows of 1024 values: 12345 read back in 9.7 us (6.6 TB/s, as fast as a copy), 1999 written at scattered
// places in 9.9 us (1.1 TB/s: every CTA scans the indices behind its own for a later row of the same place, after
// which the work is short; more rows find their last writers in a workspace, in linear time). 512 rows written in
// 4.3 us as Q4_0, 4.0 as F16, 4096 Q4_0 rows read back in 4.6 us, a single token's in 2.5 us each: launches.
#include <algorithm>
#include <cstdint>

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "ggml-b200-kernels.h"
#include "internal.h"
#include "ptx.cuh"

namespace b200 {

namespace {

enum : int { KT_F32 = 0, KT_F16 = 1, KT_Q4_0 = 2, KT_Q8_0 = 8, KT_I32 = 26, KT_I64 = 27 };

struct Dims4 {
    int64_t ne[4];
    int64_t nb[4];   // bytes
};

Dims4 dims_of(const int64_t ne[4], const size_t nb[4]) {
    Dims4 s;
    for (int i = 0; i < 4; i++) s.ne[i] = ne[i], s.nb[i] = (int64_t)nb[i];
    return s;
}
bool dims_ok(const int64_t ne[4], const size_t nb[4]) {
    if (!ne || !nb) return false;
    for (int i = 0; i < 4; i++)
        if (ne[i] <= 0) return false;
    return true;
}

constexpr int KV_THREADS = 256;
constexpr int KV_WARPS = KV_THREADS / 32;
constexpr int KV_MAX_UNITS = 8;                        // 128-value chunks per warp
constexpr int KV_AHEAD = 4;                            // of them with their loads under way
constexpr int KV_MAX_ROWS = KV_WARPS * KV_MAX_UNITS;   // rows a CTA can touch

__device__ __forceinline__ int64_t load_index(const char* p, int is64) {
    return is64 ? *reinterpret_cast<const int64_t*>(p) : (int64_t)*reinterpret_cast<const int32_t*>(p);
}

// Four consecutive values x of a block, lanes 8b .. 8b + 7 of the warp holding the block's 32 in
// order; every lane of the warp calls. The block's bytes go to `out` (not written when null). A block
// with a NaN or an infinity is stored with a NaN scale, so that reading it back shows it.
__device__ __forceinline__ void put_q4_0(const float (&x)[4], uint8_t* out) {
    const int q = threadIdx.x & 7;
    float m = x[0];
    int at = 4 * q;
#pragma unroll
    for (int e = 1; e < 4; e++)
        if (fabsf(x[e]) > fabsf(m)) m = x[e], at = 4 * q + e;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; e++) bad |= !(fabsf(x[e]) <= 3.402823466e38f);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oat = __shfl_xor_sync(0xffffffffu, at, o);
        if (fabsf(om) > fabsf(m) || (fabsf(om) == fabsf(m) && oat < at)) m = om, at = oat;
    }
    const uint32_t votes = __ballot_sync(0xffffffffu, bad);
    bad = (votes >> (threadIdx.x & 24)) & 0xffu;
    const float d = __fdiv_rn(m, -8.0f);
    const float id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int c = bad ? 8 : min(15, max(0, __float2int_rz(__fmaf_rz(x[e], id, 8.5f))));
        w |= (uint32_t)c << (8 * e);
    }
    const uint32_t hi = __shfl_xor_sync(0xffffffffu, w, 4);   // lanes q < 4: the codes 16 elements on
    if (!out) return;
    uint16_t* o16 = reinterpret_cast<uint16_t*>(out);
    if (q < 4) {
        const uint32_t b = w | (hi << 4);
        o16[1 + 2 * q] = (uint16_t)b;
        o16[2 + 2 * q] = (uint16_t)(b >> 16);
    }
    if (q == 0) o16[0] = bad ? 0x7e00u : __half_as_ushort(__float2half_rn(d));
}

__device__ __forceinline__ void put_q8_0(const float (&x)[4], uint8_t* out) {
    const int q = threadIdx.x & 7;
    float amax = 0.0f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        amax = fmaxf(amax, fabsf(x[e]));
        bad |= !(fabsf(x[e]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const uint32_t votes = __ballot_sync(0xffffffffu, bad);
    bad = (votes >> (threadIdx.x & 24)) & 0xffu;
    const float d = __fdiv_rn(amax, 127.0f);
    const float id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        // a subnormal d can make 1 / d round the largest value past 127
        const int c = bad ? 0 : min(127, max(-127, (int)roundf(__fmul_rn(x[e], id))));
        w |= ((uint32_t)c & 0xffu) << (8 * e);
    }
    if (!out) return;
    uint16_t* o16 = reinterpret_cast<uint16_t*>(out);
    o16[1 + 2 * q] = (uint16_t)w;
    o16[2 + 2 * q] = (uint16_t)(w >> 16);
    if (q == 0) o16[0] = bad ? 0x7e00u : __half_as_ushort(__float2half_rn(d));
}

// The last source row of every destination row that a slice of the indices names, in two passes: -1 into each
// of them, then the largest row. owner: [slices of idx][destination rows].
template <bool CLEAR>
__global__ void __launch_bounds__(KV_THREADS) set_rows_owner_kernel(const char* __restrict__ idx, Dims4 si, int idx64,
                                                                   int64_t dst_rows, int* __restrict__ owner) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t n = si.ne[0], slice = blockIdx.y;
    const char* ip = idx + (slice % si.ne[1]) * si.nb[1] + (slice / si.ne[1]) * si.nb[2];
    int* own = owner + slice * dst_rows;
    for (int64_t r = (int64_t)blockIdx.x * KV_THREADS + threadIdx.x; r < n; r += (int64_t)gridDim.x * KV_THREADS) {
        const int64_t at = load_index(ip + r * si.nb[0], idx64);
        if (at < 0 || at >= dst_rows) continue;
        if constexpr (CLEAR) own[at] = -1;
        else atomicMax(own + at, (int)r);
    }
}

// Unit u of a slice: 128 values from 128 * (u % cpr) of source row u / cpr. A CTA takes 8 * upw
// consecutive units of slice blockIdx.y; its rows' indices are read once, and a row that a later row
// of the slice writes again is left to that one (the result of writing the rows in order): as `owner`
// says, or where that is null the CTA scans the indices behind its first row once for all its rows,
// which takes time by the square of their number (2.1 ms for 131072).
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(KV_THREADS) set_rows_kernel(const char* __restrict__ src, Dims4 ss,
                                                             const char* __restrict__ idx, Dims4 si, int idx64,
                                                             char* __restrict__ dst, Dims4 sd, int upw, int cpr,
                                                             const int* __restrict__ owner, int* err) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int64_t row_at[KV_MAX_ROWS + 1];
    __shared__ int live[KV_MAX_ROWS + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_rows = (int)ss.ne[1], n_units = n_rows * cpr;          // below 2^31
    const int u0 = blockIdx.x * KV_WARPS * upw;
    const int u1 = min(n_units, u0 + KV_WARPS * upw);
    const int r0 = u0 / cpr;
    const int rows = (u1 - 1) / cpr - r0 + 1;
    const int n2 = (int)ss.ne[2], slices = n2 * (int)ss.ne[3];
    for (int slice = blockIdx.y; slice < slices; slice += gridDim.y) {
        const int i2 = slices == 1 ? 0 : slice % n2, i3 = slices == 1 ? 0 : slice / n2;
        const char* ip = idx;
        const int* own = owner;
        if (slices > 1) {
            const int j1 = i2 % (int)si.ne[1], j2 = i3 % (int)si.ne[2];
            ip += j1 * si.nb[1] + j2 * si.nb[2];
            if (owner) own += (j1 + j2 * si.ne[1]) * sd.ne[1];
        }
        const char* sp = src + i2 * ss.nb[2] + i3 * ss.nb[3];
        char* dp = dst + i2 * sd.nb[2] + i3 * sd.nb[3];
        // the warp's 128 values of its units k .. k + KV_AHEAD - 1, all under way together
        auto load = [&](int k, float (&x)[KV_AHEAD][4]) {
#pragma unroll
            for (int n = 0; n < KV_AHEAD; n++) {
                const int u = u0 + (k + n) * KV_WARPS + warp;
#pragma unroll
                for (int e = 0; e < 4; e++) x[n][e] = 0.0f;
                if (k + n >= upw || u >= u1) continue;
                const int r = u / cpr;
                const int64_t e0 = 128ll * (u - r * cpr) + 4 * lane;
                const float* p = reinterpret_cast<const float*>(sp + r * ss.nb[1]) + e0;
                if constexpr (VEC) {
                    if (e0 < ss.ne[0]) {
                        const float4 v = __ldg(reinterpret_cast<const float4*>(p));
                        x[n][0] = v.x, x[n][1] = v.y, x[n][2] = v.z, x[n][3] = v.w;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (e0 + e < ss.ne[0]) x[n][e] = __ldg(p + e);
                }
            }
        };
        float x[KV_AHEAD][4];
        load(0, x);                      // under way while the indices are read
        for (int r = threadIdx.x; r < rows; r += KV_THREADS) {
            const int64_t at = load_index(ip + (int64_t)(r0 + r) * si.nb[0], idx64);
            const bool in = at >= 0 && at < sd.ne[1];
            if (!in) atomicCAS(err, 0, ERR_BAD_INDEX);
            row_at[r] = at;
            live[r] = in && (!own || own[at] == r0 + r) ? 1 : 0;
        }
        __syncthreads();
        constexpr int SCAN = 4;          // indices a thread has in flight
        for (int64_t j0 = r0 + 1 + threadIdx.x; !own && j0 < n_rows; j0 += KV_THREADS * SCAN) {
            int64_t at[SCAN];
#pragma unroll
            for (int n = 0; n < SCAN; n++) {
                const int64_t j = j0 + n * KV_THREADS;
                at[n] = j < n_rows ? load_index(ip + j * si.nb[0], idx64) : -1;
            }
#pragma unroll
            for (int n = 0; n < SCAN; n++) {
                const int before = at[n] < 0 ? 0 : (int)min((int64_t)rows, j0 + n * KV_THREADS - r0);
                for (int r = 0; r < before; r++)
                    if (row_at[r] == at[n]) live[r] = 0;
            }
        }
        __syncthreads();
        for (int k = 0; k < upw; k += KV_AHEAD) {
            if (k > 0) load(k, x);
#pragma unroll
            for (int n = 0; n < KV_AHEAD; n++) {
                const int u = u0 + (k + n) * KV_WARPS + warp;
                if (k + n >= upw || u >= u1) break;
                const int r = u / cpr;
                const int64_t e0 = 128ll * (u - r * cpr) + 4 * lane;
                const bool in = e0 < ss.ne[0];   // rows of quantised types are whole blocks of 8 lanes
                if (!live[r - r0]) continue;
                char* out = dp + row_at[r - r0] * sd.nb[1];
                if constexpr (TYPE == KT_Q4_0) {
                    put_q4_0(x[n], in ? reinterpret_cast<uint8_t*>(out) + (e0 / 32) * 18 : nullptr);
                } else if constexpr (TYPE == KT_Q8_0) {
                    put_q8_0(x[n], in ? reinterpret_cast<uint8_t*>(out) + (e0 / 32) * 34 : nullptr);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (e0 + e >= ss.ne[0]) continue;
                        if constexpr (TYPE == KT_F16) reinterpret_cast<__half*>(out)[e0 + e] = __float2half_rn(x[n][e]);
                        else reinterpret_cast<float*>(out)[e0 + e] = x[n][e];
                    }
                }
            }
        }
        __syncthreads();   // row_at / live are rewritten for the next slice
    }
}

// GET_ROWS of a quantised table: unit u is 128 values of output row u / cpr; a warp takes GET_UNITS
// consecutive ones, all their loads under way before the first is used (the index, then the block, are two
// memory latencies in a row). An index outside the table records ERR_BAD_INDEX and yields a zero row, as
// get_rows_kernel does for f32 / f16.
constexpr int GET_UNITS = 4;
template <int TYPE>
__global__ void __launch_bounds__(KV_THREADS) get_rows_q_kernel(const char* __restrict__ src, Dims4 ss,
                                                               const char* __restrict__ idx, Dims4 si,
                                                               float* __restrict__ dst, int vec_out, int cpr,
                                                               int64_t n_units, int* err) {
    grid_dep_wait();
    grid_dep_launch();
    constexpr int BYTES = TYPE == KT_Q8_0 ? 34 : 18;
    const int lane = threadIdx.x & 31, q = lane & 7;
    const bool flat = si.ne[1] == 1 && si.ne[2] == 1;      // one index row: no division by its shape
    const int64_t stride = (int64_t)gridDim.x * KV_WARPS * GET_UNITS;
    for (int64_t u0 = ((int64_t)blockIdx.x * KV_WARPS + (threadIdx.x >> 5)) * GET_UNITS; u0 < n_units; u0 += stride) {
        int64_t orow = n_units < (1ll << 31) ? (int64_t)((uint32_t)u0 / (uint32_t)cpr) : u0 / cpr;
        int c = (int)(u0 - orow * cpr);
        int64_t r[GET_UNITS], out[GET_UNITS];
        const uint16_t* b[GET_UNITS];
#pragma unroll
        for (int n = 0; n < GET_UNITS; n++) {
            const int64_t e0 = 128ll * c + 4 * lane;
            out[n] = u0 + n < n_units && e0 < ss.ne[0] ? orow * ss.ne[0] + e0 : -1;
            r[n] = -1;
            b[n] = nullptr;
            if (out[n] >= 0) {
                int64_t i10 = orow, i11 = 0, i12 = 0;
                if (!flat) {
                    i10 = orow % si.ne[0];
                    i11 = orow / si.ne[0] % si.ne[1];
                    i12 = orow / (si.ne[0] * si.ne[1]);
                }
                r[n] = __ldg(reinterpret_cast<const int32_t*>(idx + i10 * si.nb[0] + i11 * si.nb[1] + i12 * si.nb[2]));
                b[n] = reinterpret_cast<const uint16_t*>(src + i11 * ss.nb[2] + i12 * ss.nb[3] + (e0 / 32) * BYTES);
            }
            if (++c == cpr) c = 0, orow++;
        }
        uint32_t d[GET_UNITS], w[GET_UNITS];
#pragma unroll
        for (int n = 0; n < GET_UNITS; n++) {
            d[n] = w[n] = 0;
            if (out[n] < 0) continue;
            if (r[n] < 0 || r[n] >= ss.ne[1]) {
                atomicCAS(err, 0, ERR_BAD_INDEX);
                out[n] = -2 - out[n];                      // zeros, past the loads
                continue;
            }
            const uint16_t* p = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(b[n]) + r[n] * ss.nb[1]);
            const int at = TYPE == KT_Q8_0 ? 2 * q : 2 * (q & 3);
            d[n] = __ldg(p);
            w[n] = (uint32_t)__ldg(p + 1 + at) | ((uint32_t)__ldg(p + 2 + at) << 16);
        }
#pragma unroll
        for (int n = 0; n < GET_UNITS; n++) {
            if (out[n] == -1) continue;
            const bool bad = out[n] < -1;
            const float f = __half2float(__ushort_as_half((unsigned short)d[n]));
            const uint32_t x = TYPE == KT_Q8_0 || q < 4 ? w[n] : w[n] >> 4;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int code = TYPE == KT_Q8_0 ? (int)(int8_t)(x >> (8 * e)) : (int)((x >> (8 * e)) & 15u) - 8;
                v[e] = bad ? 0.0f : __fmul_rn((float)code, f);
            }
            float* o = dst + (bad ? -2 - out[n] : out[n]);
            if (vec_out) {
                *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = v[e];
            }
        }
    }
}

// The same for rows of at least GET_UNITS units: a warp takes WIDE_UNITS consecutive units of one row, so
// that the index and the row's address are worked out once and a unit costs three loads and one store.
constexpr int WIDE_UNITS = 8;
template <int TYPE>
__global__ void __launch_bounds__(KV_THREADS) get_rows_q_wide_kernel(const char* __restrict__ src, Dims4 ss,
                                                                    const char* __restrict__ idx, Dims4 si,
                                                                    float* __restrict__ dst, int vec_out, int cpr,
                                                                    int64_t n_rows, int* err) {
    grid_dep_wait();
    grid_dep_launch();
    constexpr int BYTES = TYPE == KT_Q8_0 ? 34 : 18;
    const int lane = threadIdx.x & 31, q = lane & 7;
    const int64_t orow = (int64_t)blockIdx.x * KV_WARPS + (threadIdx.x >> 5);
    if (orow >= n_rows) return;
    const int c0 = blockIdx.y * WIDE_UNITS;
    int64_t i10 = orow, i11 = 0, i12 = 0;
    if (si.ne[1] != 1 || si.ne[2] != 1) {
        i10 = orow % si.ne[0];
        i11 = orow / si.ne[0] % si.ne[1];
        i12 = orow / (si.ne[0] * si.ne[1]);
    }
    const int64_t r = __ldg(reinterpret_cast<const int32_t*>(idx + i10 * si.nb[0] + i11 * si.nb[1] + i12 * si.nb[2]));
    const bool bad = r < 0 || r >= ss.ne[1];
    if (bad && lane == 0) atomicCAS(err, 0, ERR_BAD_INDEX);
    const uint16_t* row = reinterpret_cast<const uint16_t*>(src + (bad ? 0 : r) * ss.nb[1] + i11 * ss.nb[2] + i12 * ss.nb[3]);
    const uint16_t* p = row + ((int64_t)c0 * 4 + (lane >> 3)) * (BYTES / 2);
    const int at = TYPE == KT_Q8_0 ? 1 + 2 * q : 1 + 2 * (q & 3);
    const int left = (int)min((int64_t)(WIDE_UNITS * 128), ss.ne[0] - (int64_t)c0 * 128) - 4 * lane;   // values from this lane's first
    uint32_t d[WIDE_UNITS], w[WIDE_UNITS];
#pragma unroll
    for (int n = 0; n < WIDE_UNITS; n++) {
        d[n] = w[n] = 0;
        if (128 * n < left && !bad) {
            d[n] = __ldg(p + 2 * n * BYTES);
            w[n] = (uint32_t)__ldg(p + 2 * n * BYTES + at) | ((uint32_t)__ldg(p + 2 * n * BYTES + at + 1) << 16);
        }
    }
    float* out = dst + orow * ss.ne[0] + 128ll * c0 + 4 * lane;
#pragma unroll
    for (int n = 0; n < WIDE_UNITS; n++) {
        if (128 * n >= left) break;
        const float f = __half2float(__ushort_as_half((unsigned short)d[n]));
        const uint32_t x = TYPE == KT_Q8_0 || q < 4 ? w[n] : w[n] >> 4;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int code = TYPE == KT_Q8_0 ? (int)(int8_t)(x >> (8 * e)) : (int)((x >> (8 * e)) & 15u) - 8;
            v[e] = bad ? 0.0f : __fmul_rn((float)code, f);
        }
        if (vec_out) {
            *reinterpret_cast<float4*>(out + 128 * n) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) out[128 * n + e] = v[e];
        }
    }
}

constexpr int64_t SCAN_ROWS = 131072;                  // the most rows the scan takes
constexpr int64_t OWNER_ROWS = 2048;                   // rows from which owners are quicker (1024 values: 1999 rows 10.5
                                                       // by the scan, 11.0 us, 4096 rows 20.2, 16.7; single values: 8192
                                                       // rows 24, 7.3, 524288 rows 31.8 ms, 108 us)

int launched(cudaError_t e) { return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? B200_OK : B200_E_CUDA; }

}  // namespace

// The quantised half of b200_get_rows; the caller has checked pointers, shapes and idx.
int get_rows_quant_impl(int src_type, const void* src, const int64_t sne[4], const size_t snb[4], const int32_t* idx,
                        const int64_t ine[4], const size_t inb[4], float* dst, int* dev_err, cudaStream_t st) {
    const size_t bytes = src_type == KT_Q8_0 ? 34 : 18;
    if (sne[0] % 32 != 0) return B200_E_INVALID;
    if (snb[0] != bytes || ((snb[1] | snb[2] | snb[3]) & 1) || (reinterpret_cast<uintptr_t>(src) & 1u) ||
        sne[0] > (1ll << 36))
        return B200_E_UNSUPPORTED;
    const int cpr = (int)((sne[0] + 127) / 128);
    const int64_t n_units = ine[0] * ine[1] * ine[2] * cpr;
    const int64_t n_rows = ine[0] * ine[1] * ine[2], gx = (n_rows + KV_WARPS - 1) / KV_WARPS;
    const int gy = (cpr + WIDE_UNITS - 1) / WIDE_UNITS;
    if (cpr >= GET_UNITS && gx <= INT32_MAX && gy <= 65535) {
        const int vo = (reinterpret_cast<uintptr_t>(dst) & 15u) == 0 ? 1 : 0;
        const dim3 wide((unsigned)gx, (unsigned)gy), block(KV_THREADS);
        const char* ix = reinterpret_cast<const char*>(idx);
        return launched(src_type == KT_Q8_0
                            ? launch_pdl(get_rows_q_wide_kernel<KT_Q8_0>, wide, block, 0, st, static_cast<const char*>(src),
                                         dims_of(sne, snb), ix, dims_of(ine, inb), dst, vo, cpr, n_rows, dev_err)
                            : launch_pdl(get_rows_q_wide_kernel<KT_Q4_0>, wide, block, 0, st, static_cast<const char*>(src),
                                         dims_of(sne, snb), ix, dims_of(ine, inb), dst, vo, cpr, n_rows, dev_err));
    }
    const int64_t want = (n_units + KV_WARPS * GET_UNITS - 1) / (KV_WARPS * GET_UNITS);
    const unsigned grid = (unsigned)std::min<int64_t>(want, (int64_t)device_sm_count() * 32);
    const int vec = (reinterpret_cast<uintptr_t>(dst) & 15u) == 0 ? 1 : 0;
    const char* s = static_cast<const char*>(src);
    const char* ix = reinterpret_cast<const char*>(idx);
    if (src_type == KT_Q8_0)
        return launched(launch_pdl(get_rows_q_kernel<KT_Q8_0>, dim3(grid), dim3(KV_THREADS), 0, st, s,
                                   dims_of(sne, snb), ix, dims_of(ine, inb), dst, vec, cpr, n_units, dev_err));
    return launched(launch_pdl(get_rows_q_kernel<KT_Q4_0>, dim3(grid), dim3(KV_THREADS), 0, st, s, dims_of(sne, snb),
                               ix, dims_of(ine, inb), dst, vec, cpr, n_units, dev_err));
}

}  // namespace b200

extern "C" {

size_t b200_set_rows_workspace_size(const int64_t ine[4], const int64_t dne[4]) {
    using namespace b200;
    if (!ine || !dne || ine[0] < OWNER_ROWS || ine[1] <= 0 || ine[2] <= 0 || dne[1] <= 0) return 0;
    if ((double)ine[1] * (double)ine[2] * (double)dne[1] > 1e18) return 0;
    return (size_t)(ine[1] * ine[2] * dne[1]) * 4;
}

int b200_set_rows(const float* src, const int64_t sne[4], const size_t snb[4], int idx_type, const void* idx,
                  const int64_t ine[4], const size_t inb[4], int dst_type, void* dst, const int64_t dne[4],
                  const size_t dnb[4], int* dev_err, void* stream) {
    return b200_set_rows_ws(src, sne, snb, idx_type, idx, ine, inb, dst_type, dst, dne, dnb, nullptr, 0, dev_err, stream);
}

int b200_set_rows_ws(const float* src, const int64_t sne[4], const size_t snb[4], int idx_type, const void* idx,
                     const int64_t ine[4], const size_t inb[4], int dst_type, void* dst, const int64_t dne[4],
                     const size_t dnb[4], void* workspace, size_t workspace_bytes, int* dev_err, void* stream) {
    using namespace b200;
    if (!src || !idx || !dst || !dev_err || !dims_ok(sne, snb) || !dims_ok(ine, inb) || !dims_ok(dne, dnb))
        return B200_E_INVALID;
    if (dst_type != KT_F32 && dst_type != KT_F16 && dst_type != KT_Q4_0 && dst_type != KT_Q8_0)
        return B200_E_UNSUPPORTED;
    if (idx_type != KT_I32 && idx_type != KT_I64) return B200_E_UNSUPPORTED;
    const bool quant = dst_type == KT_Q4_0 || dst_type == KT_Q8_0;
    if (dne[0] != sne[0] || dne[2] != sne[2] || dne[3] != sne[3] || ine[0] != sne[1] || sne[2] % ine[1] != 0 ||
        sne[3] % ine[2] != 0 || ine[3] != 1 || (quant && sne[0] % 32 != 0))
        return B200_E_INVALID;
    const size_t isz = idx_type == KT_I64 ? 8 : 4;
    const size_t cell = dst_type == KT_F32 ? 4 : dst_type == KT_F16 ? 2 : dst_type == KT_Q4_0 ? 18 : 34;
    const size_t unit = dst_type == KT_F32 ? 4 : 2;   // the widest store
    if (sne[0] > (1ll << 36) || sne[1] > INT32_MAX || sne[2] > INT32_MAX || sne[3] > INT32_MAX) return B200_E_UNSUPPORTED;
    // rows of dst that lie in one another would take values from several rows of src
    const size_t row = (size_t)(quant ? dne[0] / 32 : dne[0]) * cell;
    if (!rows_apart(dne, dnb, row)) return B200_E_INVALID;
    if (snb[0] != 4 || ((snb[1] | snb[2] | snb[3]) & 3) || (reinterpret_cast<uintptr_t>(src) & 3u) ||
        ((inb[0] | inb[1] | inb[2]) & (isz - 1)) || (reinterpret_cast<uintptr_t>(idx) & (isz - 1)) ||
        dnb[0] != cell || ((dnb[1] | dnb[2] | dnb[3]) & (unit - 1)) || (reinterpret_cast<uintptr_t>(dst) & (unit - 1)))
        return B200_E_UNSUPPORTED;
    const bool vec = sne[0] % 4 == 0 && ((snb[1] | snb[2] | snb[3]) & 15) == 0 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
    const int cpr = (int)((sne[0] + 127) / 128);
    const int64_t n_units = sne[1] * cpr;
    // more units a warp once every SM has its four CTAs: fewer scans of the indices, more loads in flight
    int upw = 1;
    while (upw < KV_MAX_UNITS && n_units / (KV_WARPS * upw) > (int64_t)device_sm_count() * 4) upw *= 2;
    const int64_t gx = (n_units + (int64_t)KV_WARPS * upw - 1) / ((int64_t)KV_WARPS * upw);
    if (n_units > INT32_MAX - 1024 || sne[2] * sne[3] > INT32_MAX) return B200_E_UNSUPPORTED;
    const size_t need = b200_set_rows_workspace_size(ine, dne);
    int* owner = nullptr;
    if (workspace && need > 0 && ine[1] * ine[2] <= 65535) {
        if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3u)) return B200_E_WORKSPACE;
        owner = static_cast<int*>(workspace);
    } else if (sne[1] > SCAN_ROWS) {
        return workspace ? B200_E_UNSUPPORTED : B200_E_WORKSPACE;
    }
    const dim3 grid((unsigned)gx, (unsigned)std::min<int64_t>(sne[2] * sne[3], 65535)), block(KV_THREADS);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (owner) {
        const dim3 og((unsigned)std::min<int64_t>((sne[1] + KV_THREADS - 1) / KV_THREADS, (int64_t)device_sm_count() * 16),
                      (unsigned)(ine[1] * ine[2]));
        const char* ix = static_cast<const char*>(idx);
        const int idx64 = idx_type == KT_I64 ? 1 : 0;
        int rc = launched(launch_pdl(set_rows_owner_kernel<true>, og, block, 0, st, ix, dims_of(ine, inb), idx64, dne[1], owner));
        if (rc == B200_OK)
            rc = launched(launch_pdl(set_rows_owner_kernel<false>, og, block, 0, st, ix, dims_of(ine, inb), idx64, dne[1], owner));
        if (rc != B200_OK) return rc;
    }
    auto go = [&](auto kernel) {
        return launched(launch_pdl(kernel, grid, block, 0, st, reinterpret_cast<const char*>(src), dims_of(sne, snb),
                                   static_cast<const char*>(idx), dims_of(ine, inb), idx_type == KT_I64 ? 1 : 0,
                                   static_cast<char*>(dst), dims_of(dne, dnb), upw, cpr, (const int*)owner, dev_err));
    };
    switch (dst_type) {
        case KT_Q4_0: return vec ? go(set_rows_kernel<KT_Q4_0, true>) : go(set_rows_kernel<KT_Q4_0, false>);
        case KT_Q8_0: return vec ? go(set_rows_kernel<KT_Q8_0, true>) : go(set_rows_kernel<KT_Q8_0, false>);
        case KT_F16: return vec ? go(set_rows_kernel<KT_F16, true>) : go(set_rows_kernel<KT_F16, false>);
        default: return vec ? go(set_rows_kernel<KT_F32, true>) : go(set_rows_kernel<KT_F32, false>);
    }
}

}  // extern "C"
