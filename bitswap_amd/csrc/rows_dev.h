// rows_dev.h -- device helpers of the channels-last layer kernels (linear.hip, norm_act.hip, pack8.hip): element types, 16-byte
// accesses at any alignment, activations and their slopes, the 8-bit form of a saved activation.
#ifndef BITSWAP_ROWS_DEV_H
#define BITSWAP_ROWS_DEV_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/bitswap_hip.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int esize(int dt) { return dt == BS_DT_F32 ? 4 : 2; }
constexpr int vlen(int dt) { return 16 / esize(dt); }        // elements of a 16-byte access

__device__ __forceinline__ float bits_f32(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t f32_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
// two floats -> two bfloat16 / float16 in one word, round to nearest even (one v_cvt_pk on gfx950)
__device__ __forceinline__ uint32_t pk_bf16(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ uint32_t pk_f16(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// one element
template <int DT>
__device__ __forceinline__ float load1(const char* p) {
    if (DT == BS_DT_F32) return *reinterpret_cast<const float*>(p);
    const uint16_t u = *reinterpret_cast<const uint16_t*>(p);
    if (DT == BS_DT_BF16) return bits_f32((uint32_t)u << 16);
    return (float)__builtin_bit_cast(_Float16, u);
}
template <int DT>
__device__ __forceinline__ void store1(char* p, float v) {
    if (DT == BS_DT_F32) *reinterpret_cast<float*>(p) = v;
    else if (DT == BS_DT_BF16) *reinterpret_cast<uint16_t*>(p) = (uint16_t)pk_bf16(v, 0.0f);
    else *reinterpret_cast<_Float16*>(p) = (_Float16)v;
}

// 4 / 8 / 16 bytes at an address that need not be aligned to more than an element: gfx950 takes such vector accesses as they are,
// so rows of an odd number of channels cost no more instructions than others
__device__ __forceinline__ u32x4 load16(const char* p) { u32x4 r; __builtin_memcpy(&r, p, 16); return r; }
__device__ __forceinline__ u32x2 load8(const char* p) { u32x2 r; __builtin_memcpy(&r, p, 8); return r; }
__device__ __forceinline__ uint32_t load4(const char* p) { uint32_t r; __builtin_memcpy(&r, p, 4); return r; }
__device__ __forceinline__ void store16(char* p, u32x4 v) { __builtin_memcpy(p, &v, 16); }
__device__ __forceinline__ void store8(char* p, u32x2 v) { __builtin_memcpy(p, &v, 8); }

// 16 bytes <-> the floats they hold (4 or 8)
template <int DT>
__device__ __forceinline__ void unpack16(u32x4 r, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == BS_DT_F32) {
            f[i] = bits_f32(r[i]);
        } else if (DT == BS_DT_BF16) {
            f[2 * i] = bits_f32(r[i] << 16);
            f[2 * i + 1] = bits_f32(r[i] & 0xffff0000u);
        } else {
            const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)r[i]);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        }
    }
}
template <int DT>
__device__ __forceinline__ u32x4 pack16(const float* f) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == BS_DT_F32) r[i] = f32_bits(f[i]);
        else if (DT == BS_DT_BF16) r[i] = pk_bf16(f[2 * i], f[2 * i + 1]);
        else r[i] = pk_f16(f[2 * i], f[2 * i + 1]);
    }
    return r;
}
// the first n elements of such a vector (0 < n; all of them when n >= vlen), the others zero.  The end of a row is gathered by
// loads that are all on their way at once (behind its last element they repeat that one): a branch per element would wait for
// each of them in turn, and the whole wavefront with it.
template <int DT>
__device__ __forceinline__ u32x4 load_raw(const char* p, int n) {
    constexpr int V = vlen(DT);
    if (n >= V) return load16(p);
    u32x4 r;
    if (DT == BS_DT_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const uint32_t*>(p + min(i, n - 1) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = i < n ? r[i] : 0u;
    } else {
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = *reinterpret_cast<const uint16_t*>(p + min(i, n - 1) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (2 * i < n ? u[2 * i] : 0u) | (2 * i + 1 < n ? u[2 * i + 1] << 16 : 0u);
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void load_vec(const char* p, int n, float* f) { unpack16<DT>(load_raw<DT>(p, n), f); }
template <int DT>
__device__ __forceinline__ void store_vec(char* p, int n, const float* f) {
    constexpr int V = vlen(DT);
    if (n >= V) {
        store16(p, pack16<DT>(f));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) store1<DT>(p + i * esize(DT), f[i]);
    }
}

// store_vec for an output that its launch does not read again, rows of `width` channels: past the L2 (nontemporal), where the inputs
// that are read again stay.  Not for 16-bit rows that are no multiple of 64 bytes: lines written in two pieces cost more than is won
// (25600x256 -> 264 bf16: 21.5 us kept, 23.5 us past; -> 288: 20.8 and 18.4; float32 102400x256 -> 256 131 and 110).  float32 rows that are
// no such multiple go both ways: 102400x256 -> 257 178 and 164, 8192x256 -> 257 24.7 and 23.0, but 25600x256 -> 252 39 and 43,
// 102400x256 -> 100 71 and 82.  All of it a launch over and over by itself; what reads the outputs next is not in it.
template <int DT>
__device__ __forceinline__ void store_out(char* p, int n, const float* f, int width) {
    typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));
    if (n >= vlen(DT) && (DT == BS_DT_F32 || width % 32 == 0)) __builtin_nontemporal_store((u32x4_e)pack16<DT>(f), reinterpret_cast<u32x4_e*>(p));
    else store_vec<DT>(p, n, f);
}

// ---- activations ----------------------------------------------------------------------------------------------------------
// A layer's epilogue has tens of millions of these beside a product that is bound elsewhere; the library's expm1f and erff cost
// more than the product itself (16384 x 2048 x 2048 with GELU: 226 us, 96 of them the product).  Here: one v_exp_f32 where a ratio
// or a slope is wanted (relative error 2^-24 |s| + one step), the series of e^r - 1 on |r| <= ln 2 / 2 for ELU (degree 7: 1.5e-8),
// Hastings' rational form for the normal integral (Abramowitz and Stegun 7.1.26: 1.5e-7 absolute).
__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float expm1_neg(float s) {                // s <= 0
    s = fmaxf(s, -87.0f);                                            // below: -1 to the last bit
    const float n = rintf(s * 1.44269504088896341f);
    float r = fmaf(n, -0.693145751953125f, s);                      // ln 2 in two parts, the first exact in n's products
    r = fmaf(n, -1.42860682030941723e-6f, r);
    float q = 1.0f / 5040.0f;
    q = fmaf(q, r, 1.0f / 720.0f);
    q = fmaf(q, r, 1.0f / 120.0f);
    q = fmaf(q, r, 1.0f / 24.0f);
    q = fmaf(q, r, 1.0f / 6.0f);
    q = fmaf(q, r, 0.5f);
    q = fmaf(q * r, r, r);                                           // e^r - 1
    const float t = bits_f32((uint32_t)((int)n + 127) << 23);        // 2^n, n >= -126
    return fmaf(t, q, t - 1.0f);
}
// the normal integral at s, and e^(-s s / 2)
__device__ __forceinline__ float normal_integral(float s, float* gauss) {
    const float x = fabsf(s) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f)), g = exp_(-x * x);
    float q = 1.061405429f;
    q = fmaf(q, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    const float tail = 0.5f * (q * t) * g;                           // half of erfc(|s| / sqrt 2)
    *gauss = g;
    return s < 0.0f ? tail : 1.0f - tail;
}
// (16-bit results: e^s - 1 as it stands, s + s s / 2 near zero: relative error 2^-14 where the type has 2^-12 at best)
template <int DT>
__device__ __forceinline__ float elu_value(float s) {
    if (DT == BS_DT_F32) return s <= 0.0f ? expm1_neg(s) : s;
    const float e = s > -0.001953125f ? fmaf(0.5f * s, s, s) : exp_(s) - 1.0f;
    return s <= 0.0f ? e : s;
}
__device__ __forceinline__ float silu_value(float s) { return s * __builtin_amdgcn_rcpf(1.0f + exp_(-s)); }
__device__ __forceinline__ float gelu_value(float s) {
    float g;
    return s * normal_integral(s, &g);
}
__device__ __forceinline__ float elu_slope(float s) { return s > 0.0f ? 1.0f : exp_(s); }
__device__ __forceinline__ float silu_slope(float s) {
    const float p = __builtin_amdgcn_rcpf(1.0f + exp_(-s));
    return p * fmaf(s, 1.0f - p, 1.0f);
}
__device__ __forceinline__ float gelu_slope(float s) {
    float g;
    const float p = normal_integral(s, &g);
    return fmaf(s * 0.39894228040143268f, g, p);
}
// N values at once: the choice of the activation is one (uniform) branch for all of them.  A branch per value cost more than the
// activation: 102400 x 256 x 256 in bfloat16 54 us against 39.
template <int DT, int N>
__device__ __forceinline__ void act_values(int act, const float* s, float* y) {
    if (act == BS_ACT_ELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = elu_value<DT>(s[i]);
    } else if (act == BS_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = silu_value(s[i]);
    } else if (act == BS_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = gelu_value(s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = s[i];
    }
}
// d *= act'(s)
template <int N>
__device__ __forceinline__ void act_slopes(int act, const float* s, float* d) {
    if (act == BS_ACT_ELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] *= elu_slope(s[i]);
    } else if (act == BS_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] *= silu_slope(s[i]);
    } else if (act == BS_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] *= gelu_slope(s[i]);
    }
}

// ---- the 8-bit form of a saved activation ---------------------------------------------------------------------------------
// 32 consecutive channels of a row share 2^e, e the smallest exponent >= -126 with amax <= 127 2^e, but no larger than 127 2^e is
// a value of the type (121; float16: 9); code = rint(v 2^-e), at most 127 either way, -128 stands for a value that is not finite
// (and is kept out of amax).  A power of two keeps every step exact: v 2^-e, code 2^e, and
// code 2^e as bfloat16 (7 significant bits), so the gradients' matrix products take the codes as bfloat16 operands unrounded.
constexpr int P8_BLOCK = 32;

template <int DT>
__device__ __forceinline__ int p8_exponent(float amax) {      // amax finite, >= 0
    const uint32_t u = f32_bits(amax);
    const int p = (int)(u >> 23) - 127;                         // amax in [2^p, 2^(p+1)); subnormal: p = -127
    const int e = p - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);        // 1.984375 = 127 / 64
    constexpr int top = DT == BS_DT_F16 ? 9 : 121;
    return e < -126 ? -126 : e > top ? top : e;
}
__device__ __forceinline__ float p8_pow2(int e) { return bits_f32((uint32_t)(e + 127) << 23); }      // e >= -126
__device__ __forceinline__ float p8_value(int code, float step) { return code == -128 ? __builtin_nanf("") : (float)code * step; }

// V codes of a row from channel c on (n of them exist) -> floats
template <int V>
__device__ __forceinline__ void load_codes(const int8_t* __restrict__ codes, const int8_t* __restrict__ exps, int c, int n, float* f) {
    // at most two blocks of 32 channels meet in V <= 8 consecutive channels
    const int b0 = c / P8_BLOCK, b1 = (c + (n < V ? n : V) - 1) / P8_BLOCK;
    const float s0 = p8_pow2(exps[b0]), s1 = p8_pow2(exps[b1]);
    uint32_t w[2] = {0, 0};
    if (n >= V) {
        if (V == 4) w[0] = load4((const char*)codes + c);
        else {
            const u32x2 t = load8((const char*)codes + c);
            w[0] = t[0]; w[1] = t[1];
        }
    } else {
        uint32_t u[V];
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = (uint8_t)codes[c + min(i, n - 1)];
#pragma unroll
        for (int i = 0; i < V; ++i) w[i / 4] |= i < n ? u[i] << (8 * (i % 4)) : 0u;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = p8_value((int)(int8_t)(w[i / 4] >> (8 * (i % 4))), (c + i) / P8_BLOCK == b0 ? s0 : s1);
}

// parts [nparts][n] -> their sums, columns below n0 to out0 and the others to out1 (either may be null); 32 columns x 32 lanes over
// the parts a workgroup, always the same order
static __global__ __launch_bounds__(1024) void k_sum_columns(const float* __restrict__ parts, int64_t nparts, int n, int n0,
                                                     float* __restrict__ out0, float* __restrict__ out1) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, l = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
    float s = 0.0f;
    if (c < n)
#pragma unroll 4
        for (int64_t k = l; k < nparts; k += 32) s += parts[k * n + c];
    red[l][tx] = s;
    __syncthreads();
    s = red[tx][l];                                             // 32 neighbours hold the 32 partial sums of column l
#pragma unroll
    for (int o = 1; o < 32; o *= 2) s += __shfl_xor(s, o);
    const int col = blockIdx.x * 32 + l;
    if (tx == 0 && col < n) {
        if (col < n0) { if (out0) out0[col] = s; }
        else if (out1) out1[col - n0] = s;
    }
}

inline bool bad_type(int dt) { return dt != BS_DT_F32 && dt != BS_DT_BF16 && dt != BS_DT_F16; }
constexpr int64_t MAX_ROWS = (int64_t)1 << 40;
inline hipStream_t rows_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }
// a launch has fewer than 2^32 threads along an axis: a call that would need more is refused before its first launch
inline bool too_many(int64_t blocks, int threads) { return blocks > (int64_t)0xffffffff / threads; }
// a workspace that holds what a call needs; the kernels and their DMA move 16 aligned bytes of it at a time
inline bool bad_workspace(const void* p, int64_t bytes, int64_t need) { return need > 0 && (!p || ((uintptr_t)p & 15) != 0 || bytes < need); }
inline int rows_rc() { return hipGetLastError() == hipSuccess ? BS_OK : BS_ELAUNCH; }

}  // namespace
#endif
