// ROPE with several position axes (ggml's rope modes MROPE 8, VISION 24 and IMROPE 40), which the
// reference leaves to the host's CPU backend (its supports_op claims no ROPE, ggml-rocket.cpp:7410-7772).
//
//     y[i]       = x[i] cos a_i - x[i + gap] sin a_i
//     y[i + gap] = x[i] sin a_i + x[i + gap] cos a_i       a_i = freq_scale pos[axis(i)] base^(-2 step(i) / n_dims)
//
// for i < pairs, both factors times attn_factor; what lies behind the pairs is copied. MROPE and IMROPE
// rotate n_dims values (pairs = gap = n_dims / 2, step(i) = i); VISION the whole head (pairs = gap =
// n_dims = head_dim / 2, step(i) counted from the start of i's section). Sections count pairs; sector =
// i % sum(sections). MROPE, VISION: axis = the section the sector lies in. IMROPE: axis = sector % 3
// while sector < 3 sections[axis], else 3.
//
// The angle is formed and reduced to a half turn in 64 bits: pos reaches 10^5 and more, where an f32
// angle is off by 10^-2. Bound by HBM (one read and one write of x): a CTA first issues its loads, then
// a thread per (token, pair) computes the cosine and sine into shared memory for every head of the
// token, so that the 64-bit work hides behind the loads. 4096 tokens x 32 heads x 128 f32 (134 MB): 23.5 us,
// 5.7 TB/s, 0.87 of the measured copy bandwidth (30.3 us with two items in flight and a 64-bit exp2 a pair).
// A picture's 27.5 MB take 9.0 us (3.1 TB/s: 445 CTAs, three quarters of one wave, which load together and
// store together), a few tokens 2.9 us, a launch.
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

constexpr int RM_THREADS = 256;
constexpr int RM_TABLE = 1024;      // (token, pair) entries of a CTA's cosine / sine table
constexpr int RM_MAX_TOKENS = 16;   // tokens a CTA takes at most
constexpr int RM_U = 4;             // items (16 bytes of either half) a thread has in flight

struct RopeMulti {
    const char* x;
    const int32_t* pos;
    char* dst;
    int64_t nb1, nb2, nb3;          // bytes of x's strides: head, token, batch
    int64_t tokens;
    int heads, dim, pairs, gap, tpc;   // tpc: tokens a CTA
    int s[4];
    int mode;
    double first;                   // half turns a position of pair step 0: freq_scale / pi
    double power[10];               // base^(-2 2^k / n_dims): a step's frequency is the product over its bits
    float attn_factor;
};

// Pair i's axis and its angle a token position, in half turns.
__device__ __forceinline__ double half_turns_per_position(const RopeMulti& a, int i, int* axis_out) {
    const int total = a.s[0] + a.s[1] + a.s[2] + a.s[3];
    const int sector = i % total;
    const int b1 = a.s[0], b2 = b1 + a.s[1], b3 = b2 + a.s[2];
    int axis, step = i;
    if (a.mode == 40) {
        axis = sector % 3;
        if (sector >= 3 * a.s[axis]) axis = 3;
    } else {
        axis = sector < b1 ? 0 : sector < b2 ? 1 : sector < b3 ? 2 : 3;
        if (a.mode == 24) step = sector - (axis == 0 ? 0 : axis == 1 ? b1 : axis == 2 ? b2 : b3);
    }
    *axis_out = axis;
    // ten 64-bit products at most, where a 64-bit exp2 is a chain of some sixty operations
    double f = a.first;
#pragma unroll
    for (int k = 0; k < 10; k++)
        if (step >> k & 1) f *= a.power[k];
    return f;
}

// V consecutive values of type T: 16 bytes, or one value
template <typename T, int V>
struct Pack {
    uint32_t w[V == 1 ? 1 : 4];
    __device__ __forceinline__ void load(const char* p) {
        if constexpr (V > 1) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (sizeof(T) == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ void store(char* p) const {
        if constexpr (V > 1) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        else *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    }
    __device__ __forceinline__ void get(float (&v)[V]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < V; k++) v[k] = __uint_as_float(w[k]);
        } else if constexpr (V == 1) {
            v[0] = __half2float(__ushort_as_half((unsigned short)w[0]));
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
                v[2 * k] = f.x, v[2 * k + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ void set(const float (&v)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < V; k++) w[k] = __float_as_uint(v[k]);
        } else if constexpr (V == 1) {
            w[0] = __half_as_ushort(__float2half_rn(v[0]));
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = pack_half2(v[2 * k], v[2 * k + 1]);
        }
    }
};

// V: values a vector access moves (16 bytes), or 1 where rows are not 16-byte aligned or pairs do not
// divide by it.
template <typename T, int V>
__global__ void __launch_bounds__(RM_THREADS, 4) rope_multi_kernel(const RopeMulti a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float2 table[RM_TABLE];
    const int64_t tok0 = (int64_t)blockIdx.x * a.tpc;
    const int n_tok = (int)min((int64_t)a.tpc, a.tokens - tok0);
    const int64_t i3 = blockIdx.y;
    const int ppr = a.pairs / V;                       // rotated items of a head
    const int tail = (a.dim - 2 * a.pairs) / V;        // copied items of a head
    const int per_tok = a.heads * ppr;
    const int n = n_tok * per_tok;
    const char* x = a.x + i3 * a.nb3 + tok0 * a.nb2;
    char* d = a.dst + (i3 * a.tokens + tok0) * (int64_t)a.heads * a.dim * (int64_t)sizeof(T);
    bool made = false;
    for (int base = 0; base < n; base += RM_THREADS * RM_U) {
        Pack<T, V> lo[RM_U], hi[RM_U];
#pragma unroll
        for (int u = 0; u < RM_U; u++) {
            const int it = base + u * RM_THREADS + (int)threadIdx.x;
            if (it >= n) continue;
            const int tk = it / per_tok, rest = it - tk * per_tok, h = rest / ppr, j = (rest - h * ppr) * V;
            const char* p = x + tk * a.nb2 + h * a.nb1 + j * (int64_t)sizeof(T);
            lo[u].load(p);
            hi[u].load(p + a.gap * (int64_t)sizeof(T));
        }
        if (!made) {
            int last = -1, axis = 0;
            double rate = 0.0;
            for (int e = threadIdx.x; e < n_tok * a.pairs; e += RM_THREADS) {
                const int tk = e / a.pairs, i = e - tk * a.pairs;
                if (i != last) rate = half_turns_per_position(a, i, &axis), last = i;
                const double turns = (double)__ldg(a.pos + (int64_t)axis * a.tokens + tok0 + tk) * rate;
                float sn, cs;
                sincospif((float)(turns - 2.0 * rint(0.5 * turns)), &sn, &cs);   // of a value in [-1, 1]
                table[e] = make_float2(cs * a.attn_factor, sn * a.attn_factor);
            }
            __syncthreads();
            made = true;
        }
#pragma unroll
        for (int u = 0; u < RM_U; u++) {
            const int it = base + u * RM_THREADS + (int)threadIdx.x;
            if (it >= n) continue;
            const int tk = it / per_tok, rest = it - tk * per_tok, h = rest / ppr, j = (rest - h * ppr) * V;
            float x0[V], x1[V], y0[V], y1[V];
            lo[u].get(x0);
            hi[u].get(x1);
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float2 c = table[tk * a.pairs + j + e];
                y0[e] = x0[e] * c.x - x1[e] * c.y;
                y1[e] = x0[e] * c.y + x1[e] * c.x;
            }
            lo[u].set(y0);
            hi[u].set(y1);
            char* p = d + (((int64_t)tk * a.heads + h) * a.dim + j) * (int64_t)sizeof(T);
            lo[u].store(p);
            hi[u].store(p + a.gap * (int64_t)sizeof(T));
        }
    }
    const int m = n_tok * a.heads * tail;
    for (int it = threadIdx.x; it < m; it += RM_THREADS) {
        const int tk = it / (a.heads * tail), rest = it - tk * a.heads * tail, h = rest / tail;
        const int j = 2 * a.pairs + (rest - h * tail) * V;
        Pack<T, V> y;
        y.load(x + tk * a.nb2 + h * a.nb1 + j * (int64_t)sizeof(T));
        y.store(d + (((int64_t)tk * a.heads + h) * a.dim + j) * (int64_t)sizeof(T));
    }
}

}  // namespace

}  // namespace b200

extern "C" {

int b200_rope_multi(int type, const void* x, const int64_t ne[4], const size_t nb[4], const int32_t* pos, int n_dims,
                    int mode, const int32_t sections[4], float freq_base, float freq_scale, float attn_factor,
                    void* dst, void* stream) {
    using namespace b200;
    if (!x || !ne || !nb || !pos || !sections || !dst) return B200_E_INVALID;
    for (int i = 0; i < 4; i++)
        if (ne[i] <= 0 || sections[i] < 0 || sections[i] > 65536) return B200_E_INVALID;
    if (n_dims <= 0 || n_dims % 2 != 0 || n_dims > ne[0] || !(freq_base > 0.0f) ||
        sections[0] + sections[1] + sections[2] + sections[3] <= 0)
        return B200_E_INVALID;
    if (type != 0 && type != 1) return B200_E_UNSUPPORTED;
    if (mode != 8 && mode != 24 && mode != 40) return B200_E_UNSUPPORTED;
    if (mode == 24 && 2 * (int64_t)n_dims != ne[0]) return B200_E_INVALID;
    const int64_t es = type == 1 ? 2 : 4;
    RopeMulti a{};
    const int64_t pairs = mode == 24 ? n_dims : n_dims / 2;
    if ((int64_t)nb[0] != es || (nb[1] | nb[2] | nb[3]) % es != 0 || reinterpret_cast<uintptr_t>(x) % es != 0 ||
        reinterpret_cast<uintptr_t>(dst) % es != 0 || reinterpret_cast<uintptr_t>(pos) % 4 != 0 || pairs > RM_TABLE || ne[0] > 4096 || ne[1] > 65536 ||
        ne[3] > 65535)
        return B200_E_UNSUPPORTED;
    const int vw = (int)(16 / es);
    const bool vec = pairs % vw == 0 && (ne[0] - 2 * pairs) % vw == 0 && ((nb[1] | nb[2] | nb[3]) & 15) == 0 &&
                     ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dst)) & 15u) == 0;
    a.x = static_cast<const char*>(x);
    a.pos = pos;
    a.dst = static_cast<char*>(dst);
    a.nb1 = (int64_t)nb[1], a.nb2 = (int64_t)nb[2], a.nb3 = (int64_t)nb[3];
    a.tokens = ne[2];
    a.heads = (int)ne[1], a.dim = (int)ne[0], a.pairs = (int)pairs, a.gap = (int)pairs;
    for (int i = 0; i < 4; i++) a.s[i] = sections[i];
    a.mode = mode;
    a.first = (double)freq_scale * 0.31830988618379067154;
    const double l2 = -2.0 * log2((double)freq_base) / (double)n_dims;
    for (int k = 0; k < 10; k++) a.power[k] = exp2(l2 * (double)(1 << k));
    a.attn_factor = attn_factor;
    // tokens a CTA: enough items and enough angles for its threads, as far as the table holds them
    const int64_t items = ne[1] * (pairs / (vec ? vw : 1));
    int64_t tpc = std::max<int64_t>({1, (int64_t)RM_THREADS * RM_U / items, RM_THREADS / pairs});
    tpc = std::min({tpc, (int64_t)RM_MAX_TOKENS, (int64_t)RM_TABLE / pairs, ne[2]});
    while (tpc > 1 && (ne[2] + tpc - 1) / tpc * ne[3] < device_sm_count()) tpc = (tpc + 1) / 2;
    a.tpc = (int)tpc;
    const int64_t gx = (ne[2] + tpc - 1) / tpc;
    if (gx > INT32_MAX) return B200_E_UNSUPPORTED;
    const dim3 grid((unsigned)gx, (unsigned)ne[3]), block(RM_THREADS);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = type == 1 ? (vec ? launch_pdl(rope_multi_kernel<__half, 8>, grid, block, 0, st, a)
                                           : launch_pdl(rope_multi_kernel<__half, 1>, grid, block, 0, st, a))
                                    : (vec ? launch_pdl(rope_multi_kernel<float, 4>, grid, block, 0, st, a)
                                           : launch_pdl(rope_multi_kernel<float, 1>, grid, block, 0, st, a));
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? B200_OK : B200_E_CUDA;
}

}  // extern "C"
