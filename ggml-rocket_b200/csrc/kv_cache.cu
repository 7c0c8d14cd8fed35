// A KV cache quantised as it is written (SET_ROWS) and read back (GET_ROWS over Q4_0 / Q8_0).
//
// The reference leaves both to the host's CPU backend (its supports_op claims neither,
// ggml-rocket.cpp:7410-7772). Formats are ggml's: blocks of 32 values, an fp16 scale d, then the codes.
//   Q4_0  m = the block's value of largest size (the first of equals), d = m / -8,
//         code = min(15, trunc(x * id + 8.5)), id = 1 / d in f32 (0 when d is 0); element j < 16 is
//         the low nibble of byte j, element j + 16 its high nibble; a code c stands for (c - 8) d.
//         The product and sum are not rounded before the truncation: one FMA rounded toward zero
//         truncates to the same integer as the exact value.
//   Q8_0  d = amax / 127, code = roundf(x * id), the product rounded to f32; it stands for code * d.
//
// Both are bound by HBM (4 bytes a value on the f32 side, 0.5625 / 1.0625 on the other; no reuse).
// Eight lanes take a block, four consecutive values each, so a warp reads or writes 512 consecutive
// bytes of f32 with one 16-byte access per lane; the block's maximum is three shuffles. Blocks are
// only 2-byte aligned, so codes and scales move as 2-byte words, which L1 and L2 join into sectors.
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

// Unit u of a slice: 128 values from 128 * (u % cpr) of source row u / cpr. A CTA takes 8 * upw
// consecutive units of slice blockIdx.y; its rows' indices are read once, and a row that a later row
// of the slice writes again is left to that one (the result of writing the rows in order): the CTA
// scans the indices behind its first row once for all its rows.
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(KV_THREADS) set_rows_kernel(const char* __restrict__ src, Dims4 ss,
                                                             const char* __restrict__ idx, Dims4 si, int idx64,
                                                             char* __restrict__ dst, Dims4 sd, int upw, int cpr,
                                                             int* err) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int64_t row_at[KV_MAX_ROWS + 1];
    __shared__ int live[KV_MAX_ROWS + 1];
    const int64_t n_rows = ss.ne[1], n_units = n_rows * cpr;
    const int64_t u0 = (int64_t)blockIdx.x * KV_WARPS * upw;
    const int64_t u1 = min(n_units, u0 + (int64_t)KV_WARPS * upw);
    const int64_t r0 = u0 / cpr;
    const int rows = (int)((u1 - 1) / cpr - r0) + 1;
    for (int64_t slice = blockIdx.y; slice < ss.ne[2] * ss.ne[3]; slice += gridDim.y) {
        const int64_t i2 = slice % ss.ne[2], i3 = slice / ss.ne[2];
        const char* ip = idx + (i2 % si.ne[1]) * si.nb[1] + (i3 % si.ne[2]) * si.nb[2];
        for (int r = threadIdx.x; r < rows; r += KV_THREADS) {
            const int64_t at = load_index(ip + (r0 + r) * si.nb[0], idx64);
            const bool in = at >= 0 && at < sd.ne[1];
            if (!in) atomicCAS(err, 0, ERR_BAD_INDEX);
            row_at[r] = at;
            live[r] = in ? 1 : 0;
        }
        __syncthreads();
        for (int64_t j = r0 + 1 + threadIdx.x; j < n_rows; j += KV_THREADS) {
            const int64_t at = load_index(ip + j * si.nb[0], idx64);
            const int before = (int)min((int64_t)rows, j - r0);
            for (int r = 0; r < before; r++)
                if (row_at[r] == at) live[r] = 0;
        }
        __syncthreads();
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int k = 0; k < upw; k++) {
            const int64_t u = u0 + (int64_t)k * KV_WARPS + warp;
            if (u >= u1) break;
            const int64_t r = u / cpr;
            if (!live[r - r0]) continue;
            const int64_t e0 = 128 * (u - r * cpr) + 4 * lane;
            const bool in = e0 < ss.ne[0];   // rows of quantised types are whole blocks of 8 lanes
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const char* sp = src + r * ss.nb[1] + i2 * ss.nb[2] + i3 * ss.nb[3] + e0 * 4;
            if (in) {
                if constexpr (VEC) {
                    const float4 v = __ldg(reinterpret_cast<const float4*>(sp));
                    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (e0 + e < ss.ne[0]) x[e] = __ldg(reinterpret_cast<const float*>(sp) + e);
                }
            }
            char* dp = dst + row_at[r - r0] * sd.nb[1] + i2 * sd.nb[2] + i3 * sd.nb[3];
            if constexpr (TYPE == KT_Q4_0) {
                put_q4_0(x, in ? reinterpret_cast<uint8_t*>(dp) + (e0 / 32) * 18 : nullptr);
            } else if constexpr (TYPE == KT_Q8_0) {
                put_q8_0(x, in ? reinterpret_cast<uint8_t*>(dp) + (e0 / 32) * 34 : nullptr);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (e0 + e >= ss.ne[0]) continue;
                    if constexpr (TYPE == KT_F16) reinterpret_cast<__half*>(dp)[e0 + e] = __float2half_rn(x[e]);
                    else reinterpret_cast<float*>(dp)[e0 + e] = x[e];
                }
            }
        }
        __syncthreads();   // row_at / live are rewritten for the next slice
    }
}

// GET_ROWS of a quantised table: unit u is 128 values of output row u / cpr. An index outside the
// table records ERR_BAD_INDEX and yields a zero row, as get_rows_kernel does for f32 / f16.
template <int TYPE>
__global__ void __launch_bounds__(KV_THREADS) get_rows_q_kernel(const char* __restrict__ src, Dims4 ss,
                                                               const char* __restrict__ idx, Dims4 si,
                                                               float* __restrict__ dst, int vec_out, int cpr,
                                                               int64_t n_units, int* err) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, q = lane & 7;
    const int64_t stride = (int64_t)gridDim.x * KV_WARPS;
    for (int64_t u = (int64_t)blockIdx.x * KV_WARPS + (threadIdx.x >> 5); u < n_units; u += stride) {
        const int64_t orow = u / cpr;
        const int64_t e0 = 128 * (u - orow * cpr) + 4 * lane;
        if (e0 >= ss.ne[0]) continue;
        const int64_t i10 = orow % si.ne[0], i11 = (orow / si.ne[0]) % si.ne[1], i12 = orow / (si.ne[0] * si.ne[1]);
        const int64_t r = *reinterpret_cast<const int32_t*>(idx + i10 * si.nb[0] + i11 * si.nb[1] + i12 * si.nb[2]);
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < 0 || r >= ss.ne[1]) {
            if (lane == 0) atomicCAS(err, 0, ERR_BAD_INDEX);
        } else {
            constexpr int BYTES = TYPE == KT_Q8_0 ? 34 : 18;
            const uint16_t* b = reinterpret_cast<const uint16_t*>(src + r * ss.nb[1] + i11 * ss.nb[2] + i12 * ss.nb[3] +
                                                                  (e0 / 32) * BYTES);
            const float d = __half2float(__ushort_as_half(__ldg(b)));
            const int w = TYPE == KT_Q8_0 ? 2 * q : 2 * (q & 3);
            uint32_t c = (uint32_t)__ldg(b + 1 + w) | ((uint32_t)__ldg(b + 2 + w) << 16);
            if constexpr (TYPE == KT_Q8_0) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = __fmul_rn((float)(int8_t)(c >> (8 * e)), d);
            } else {
                if (q >= 4) c >>= 4;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = __fmul_rn((float)((int)((c >> (8 * e)) & 15u) - 8), d);
            }
        }
        float* out = dst + orow * ss.ne[0] + e0;
        if (vec_out) {
            *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) out[e] = v[e];
        }
    }
}

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
    const int64_t want = (n_units + KV_WARPS - 1) / KV_WARPS;
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

int b200_set_rows(const float* src, const int64_t sne[4], const size_t snb[4], int idx_type, const void* idx,
                  const int64_t ine[4], const size_t inb[4], int dst_type, void* dst, const int64_t dne[4],
                  const size_t dnb[4], int* dev_err, void* stream) {
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
    if (snb[0] != 4 || ((snb[1] | snb[2] | snb[3]) & 3) || (reinterpret_cast<uintptr_t>(src) & 3u) ||
        ((inb[0] | inb[1] | inb[2]) & (isz - 1)) || (reinterpret_cast<uintptr_t>(idx) & (isz - 1)) ||
        dnb[0] != cell || ((dnb[1] | dnb[2] | dnb[3]) & (unit - 1)) || (reinterpret_cast<uintptr_t>(dst) & (unit - 1)) ||
        sne[0] > (1ll << 36))
        return B200_E_UNSUPPORTED;
    const bool vec = sne[0] % 4 == 0 && ((snb[1] | snb[2] | snb[3]) & 15) == 0 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
    const int cpr = (int)((sne[0] + 127) / 128);
    const int64_t n_units = sne[1] * cpr;
    // more units a warp once every SM has its CTAs, so that long calls scan their indices less often
    int upw = 1;
    while (upw < KV_MAX_UNITS && n_units / (KV_WARPS * upw) > (int64_t)device_sm_count() * 16) upw *= 2;
    const int64_t gx = (n_units + (int64_t)KV_WARPS * upw - 1) / ((int64_t)KV_WARPS * upw);
    if (gx > INT32_MAX) return B200_E_UNSUPPORTED;
    const dim3 grid((unsigned)gx, (unsigned)std::min<int64_t>(sne[2] * sne[3], 65535)), block(KV_THREADS);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto kernel) {
        return launched(launch_pdl(kernel, grid, block, 0, st, reinterpret_cast<const char*>(src), dims_of(sne, snb),
                                   static_cast<const char*>(idx), dims_of(ine, inb), idx_type == KT_I64 ? 1 : 0,
                                   static_cast<char*>(dst), dims_of(dne, dnb), upw, cpr, dev_err));
    };
    switch (dst_type) {
        case KT_Q4_0: return vec ? go(set_rows_kernel<KT_Q4_0, true>) : go(set_rows_kernel<KT_Q4_0, false>);
        case KT_Q8_0: return vec ? go(set_rows_kernel<KT_Q8_0, true>) : go(set_rows_kernel<KT_Q8_0, false>);
        case KT_F16: return vec ? go(set_rows_kernel<KT_F16, true>) : go(set_rows_kernel<KT_F16, false>);
        default: return vec ? go(set_rows_kernel<KT_F32, true>) : go(set_rows_kernel<KT_F32, false>);
    }
}

}  // extern "C"
