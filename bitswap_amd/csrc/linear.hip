// linear.hip -- products over rows of channels (channels-last activations): s = x w^T + bias (+ res) with its activation, and the
// two products of its backward pass.  One kernel template; what differs is which axis of an operand is contiguous in memory.
//
//   out[q][p] = sum_k P(p, k) Q(q, k)                    p the contiguous axis of the output
//   forward   P = w  [N, K]      (k contiguous)      Q = x  [rows, K]  (k contiguous)
//   dx        P = w^T            (p contiguous)      Q = ds [rows, N]  (k contiguous)
//   dw        P = x^T or codes   (p contiguous)      Q = ds^T          (q contiguous), k = rows, split over workgroups
#include "rows_dev.h"

namespace {

enum { L_KC = 0, L_IC = 1, L_P8 = 2 };                    // k contiguous | index contiguous | index contiguous 8-bit codes
enum { E_LAYER = 0, E_PLAIN = 1, E_PART = 2 };            // bias + residual + activation | one rounding | float32 partial sums

struct GemmArgs {
    const char* P;
    const char* Q;
    const int8_t* Pexp;       // L_P8: exponents [nk, lpe]
    int64_t ldp, ldq;         // row strides in elements
    int lpe;
    int np;
    int64_t nq, nk;
    int64_t kpart;            // k per part (split products), else nk
    int tp;                   // tiles along p
    int64_t tiles;
    const char* bias;
    const char* res;
    int64_t ldr;
    char* out0;               // sum / plain output / partials
    char* out1;               // activation
    int act, bias_f32;
};

template <int DT>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if (DT == BS_DT_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 8 floats -> their three bfloat16 limbs (round to nearest; the three add up to the float exactly)
__device__ __forceinline__ void limbs3(const float* f, u32x4* l) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = f[2 * i], b = f[2 * i + 1];
        const uint32_t h0 = pk_bf16(a, b);
        a -= bits_f32(h0 << 16);
        b -= bits_f32(h0 & 0xffff0000u);
        const uint32_t h1 = pk_bf16(a, b);
        a -= bits_f32(h1 << 16);
        b -= bits_f32(h1 & 0xffff0000u);
        l[0][i] = h0;
        l[1][i] = h1;
        l[2][i] = pk_bf16(a, b);
    }
}

// One operand's tile [BI indexes][BK k]: global -> registers -> shared memory, as 16-byte chunks of 8 consecutive k.  Chunk c of
// index i lies in slot c ^ f(i) of its row, f chosen so that the 8 lanes a 16-byte LDS access serves together touch all banks.
template <int DT, int LAY, int BI, int BK, int NT>
struct Tile {
    static constexpr int LIMBS = (DT == BS_DT_F32 && LAY != L_P8) ? 3 : 1;
    static constexpr int SL = BK / 8, RL = 8 / SL;
    static constexpr int BYTES = LIMBS * BI * BK * 2;
    static constexpr int UNITS = LAY == L_KC ? BI * SL : BI / 4 * SL;
    static constexpr int PER = (UNITS + NT - 1) / NT;
    static constexpr int ES = esize(DT);
    static constexpr int RAWN = LAY == L_KC ? (DT == BS_DT_F32 ? 8 : 4) : LAY == L_IC ? (DT == BS_DT_F32 ? 32 : 16) : 16;
    uint32_t raw[PER][RAWN];

    static __device__ __forceinline__ int slot(int i, int c) { return c ^ (((i / RL) ^ (LAY == L_KC ? 0 : i >> 3)) & (SL - 1)); }
    static __device__ __forceinline__ int lds_at(int limb, int i, int c) { return ((limb * BI + i) * SL + slot(i, c)) * 16; }

    __device__ __forceinline__ void load(const GemmArgs& a, const char* base, int64_t ld, int64_t ni, int64_t i0, int64_t k0, int64_t k1,
                                         int tid) {
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int u = tid + n * NT;
            if (UNITS % NT != 0 && u >= UNITS) break;
            if (LAY == L_KC) {
                int64_t i = i0 + u / SL;
                i = i < ni ? i : ni - 1;                       // rows behind the last: any row, their sums are not stored
                const int64_t k = k0 + (u % SL) * 8;
                const char* p = base + (i * ld + k) * ES;
                const int64_t left = k1 - k;
                if (left >= 8) {
                    const u32x4 v = load16(p);
                    raw[n][0] = v[0]; raw[n][1] = v[1]; raw[n][2] = v[2]; raw[n][3] = v[3];
                    if (DT == BS_DT_F32) {
                        const u32x4 w = load16(p + 16);
                        raw[n][4 % RAWN] = w[0]; raw[n][5 % RAWN] = w[1]; raw[n][6 % RAWN] = w[2]; raw[n][7 % RAWN] = w[3];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint32_t v = 0;
                        if (e < left) v = DT == BS_DT_F32 ? *reinterpret_cast<const uint32_t*>(p + e * 4) : *reinterpret_cast<const uint16_t*>(p + e * 2);
                        if (DT == BS_DT_F32) raw[n][e % RAWN] = v;
                        else raw[n][e / 2] = e % 2 ? (raw[n][e / 2] | (v << 16)) : v;
                    }
                }
            } else {
                const int64_t i = i0 + (u % (BI / 4)) * 4;
                const int64_t kb = k0 + (u / (BI / 4)) * 8;
                const bool whole = i + 4 <= ni;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int64_t k = kb + r < k1 ? kb + r : k1 - 1;           // rows behind the last: zeroed below
                    const bool live = kb + r < k1;
                    if (LAY == L_P8) {
                        const char* p = base + k * ld + i;
                        uint32_t v = 0, e = 0;
                        if (whole) {
                            v = load4(p);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (i + j < ni) v |= (uint32_t)(uint8_t)p[j] << (8 * j);
                        }
                        if (i < ni) e = (uint32_t)(int)a.Pexp[k * a.lpe + i / P8_BLOCK];
                        raw[n][r] = live ? v : 0;
                        raw[n][(8 + r) % RAWN] = e;
                    } else {
                        const char* p = base + (k * ld + i) * ES;
                        uint32_t v[4] = {0, 0, 0, 0};
                        if (whole) {
                            if (DT == BS_DT_F32) {
                                const u32x4 t = load16(p);
                                v[0] = t[0]; v[1] = t[1]; v[2] = t[2]; v[3] = t[3];
                            } else {
                                const u32x2 t = load8(p);
                                v[0] = t[0]; v[1] = t[1];
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (i + j < ni) {
                                    if (DT == BS_DT_F32) v[j] = *reinterpret_cast<const uint32_t*>(p + j * 4);
                                    else v[j / 2] |= (uint32_t) * reinterpret_cast<const uint16_t*>(p + j * 2) << (16 * (j % 2));
                                }
                        }
                        constexpr int W = DT == BS_DT_F32 ? 4 : 2;
#pragma unroll
                        for (int j = 0; j < W; ++j) raw[n][(r * W + j) % RAWN] = live ? v[j] : 0;
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void put(char* lds, int i, int c, const float* f) const {      // 8 floats of consecutive k
        if (LIMBS == 3) {
            u32x4 l[3];
            limbs3(f, l);
#pragma unroll
            for (int b = 0; b < 3; ++b) *reinterpret_cast<u32x4*>(lds + lds_at(b, i, c)) = l[b];
        } else {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = DT == BS_DT_F16 ? pk_f16(f[2 * j], f[2 * j + 1]) : pk_bf16(f[2 * j], f[2 * j + 1]);
            *reinterpret_cast<u32x4*>(lds + lds_at(0, i, c)) = v;
        }
    }

    __device__ __forceinline__ void store(char* lds, int tid) const {
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int u = tid + n * NT;
            if (UNITS % NT != 0 && u >= UNITS) break;
            if (LAY == L_KC) {
                const int i = u / SL, c = u % SL;
                if (DT == BS_DT_F32) {
                    float f[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = bits_f32(raw[n][e % RAWN]);
                    put(lds, i, c, f);
                } else {
                    const u32x4 v = {raw[n][0], raw[n][1], raw[n][2], raw[n][3]};
                    *reinterpret_cast<u32x4*>(lds + lds_at(0, i, c)) = v;
                }
            } else {
                const int i = (u % (BI / 4)) * 4, c = u / (BI / 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (LAY == L_P8) {
                        float f[8];
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            f[r] = p8_value((int)(int8_t)(raw[n][r] >> (8 * j)), p8_pow2((int)raw[n][(8 + r) % RAWN]));
                        put(lds, i + j, c, f);
                    } else if (DT == BS_DT_F32) {
                        float f[8];
#pragma unroll
                        for (int r = 0; r < 8; ++r) f[r] = bits_f32(raw[n][(r * 4 + j) % RAWN]);
                        put(lds, i + j, c, f);
                    } else {
                        u32x4 v;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t lo = raw[n][(4 * r + j / 2) % RAWN], hi = raw[n][(4 * r + 2 + j / 2) % RAWN];
                            v[r] = j % 2 ? ((lo >> 16) | (hi & 0xffff0000u)) : ((lo & 0xffffu) | (hi << 16));
                        }
                        *reinterpret_cast<u32x4*>(lds + lds_at(0, i + j, c)) = v;
                    }
                }
            }
        }
    }
};

// operand element as float, for the sums that are added up again (float32 only)
template <int DT, int LAY>
__device__ __forceinline__ float element(const GemmArgs& a, const char* base, int64_t ld, int64_t i, int64_t k) {
    if (LAY == L_KC) return load1<DT>(base + (i * ld + k) * esize(DT));
    if (LAY == L_IC) return load1<DT>(base + (k * ld + i) * esize(DT));
    return p8_value((int)(int8_t)base[k * ld + i], p8_pow2((int)a.Pexp[k * a.lpe + i / P8_BLOCK]));
}

template <int DT, int PLAY, int QLAY, int EPI, int BP, int BQ, int WP, int WQ, int BK>
__global__ __launch_bounds__((BP / WP) * (BQ / WQ) * 64) void k_rows_gemm(const GemmArgs a) {
    constexpr int NT = (BP / WP) * (BQ / WQ) * 64;
    typedef Tile<DT, PLAY, BP, BK, NT> TP;
    typedef Tile<DT, QLAY, BQ, BK, NT> TQ;
    constexpr int STAGE = TP::BYTES + TQ::BYTES;
    constexpr int NP = WP / 32, NQ = WQ / 32;
    __shared__ __align__(16) char lds[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wp = wave % (BP / WP), wq = wave / (BP / WP);

    // workgroups of one XCD (blockIdx % 8) take a run of tiles, p fastest: the rows of Q that several p tiles read are in its L2
    const int64_t per = (a.tiles + 7) / 8;
    const int64_t t = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (blockIdx.x / 8 >= per || t >= a.tiles) return;
    const int64_t p0 = (t % a.tp) * BP, q0 = (t / a.tp) * BQ;
    const int64_t kb = blockIdx.y * a.kpart;
    const int64_t ke = kb + a.kpart < a.nk ? kb + a.kpart : a.nk;

    f32x16 acc[NP][NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    TP tp;
    TQ tq;
    tp.load(a, a.P, a.ldp, a.np, p0, kb, ke, tid);
    tq.load(a, a.Q, a.ldq, a.nq, q0, kb, ke, tid);
    int buf = 0;
    for (int64_t k = kb; k < ke; k += BK) {
        char* const lp = lds + buf * STAGE;
        char* const lq = lp + TP::BYTES;
        tp.store(lp, tid);
        tq.store(lq, tid);
        __syncthreads();          // one barrier a step: the buffer written next was read before the previous barrier
        if (k + BK < ke) {
            tp.load(a, a.P, a.ldp, a.np, p0, k + BK, ke, tid);
            tq.load(a, a.Q, a.ldq, a.nq, q0, k + BK, ke, tid);
        }
#pragma unroll
        for (int s = 0; s < BK / 16; ++s) {
            u32x4 fp[NP][TP::LIMBS], fq[NQ][TQ::LIMBS];
            const int c = 2 * s + (lane >> 5);
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int l = 0; l < TP::LIMBS; ++l)
                    fp[i][l] = *reinterpret_cast<const u32x4*>(lp + TP::lds_at(l, wp * WP + i * 32 + (lane & 31), c));
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int l = 0; l < TQ::LIMBS; ++l)
                    fq[j][l] = *reinterpret_cast<const u32x4*>(lq + TQ::lds_at(l, wq * WQ + j * 32 + (lane & 31), c));
            // limb products of total order <= 2, small ones first: what is left out is of relative size 2^-24
#pragma unroll
            for (int o = TP::LIMBS + TQ::LIMBS > 2 ? 2 : 0; o >= 0; --o)
#pragma unroll
                for (int lp_ = 0; lp_ < TP::LIMBS; ++lp_)
#pragma unroll
                    for (int i = 0; i < NP; ++i)
#pragma unroll
                        for (int j = 0; j < NQ; ++j)
                            if (o - lp_ >= 0 && o - lp_ < TQ::LIMBS)
                                acc[i][j] = mfma<DT>(fp[i][lp_], fq[j][(o - lp_ >= 0 && o - lp_ < TQ::LIMBS) ? o - lp_ : 0], acc[i][j]);
        }
        buf ^= 1;
    }

    // lane l holds, for q = l % 32 of a 32x32 tile, the p of rows 8 g + 4 (l / 32) + 0..3, g = 0..3: four channels side by side
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int64_t q = q0 + wq * WQ + j * 32 + (lane & 31);
        if (q >= a.nq) continue;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int64_t p = p0 + wp * WP + i * 32 + 8 * g + 4 * (lane >> 5);
                if (p >= a.np) continue;
                const int n = a.np - p < 4 ? (int)(a.np - p) : 4;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = acc[i][j][4 * g + e];
                    if (DT == BS_DT_F32 && e < n && (f32_bits(v[e]) & 0x7f800000u) == 0x7f800000u) {
                        // an infinity or a NaN among the operands (or a limb that overflowed): the sum again, in float32
                        float s = 0.0f;
                        for (int64_t k = kb; k < ke; ++k)
                            s = fmaf(element<DT, PLAY>(a, a.P, a.ldp, p + e, k), element<DT, QLAY>(a, a.Q, a.ldq, q, k), s);
                        v[e] = s;
                    }
                }
                if (EPI == E_PART) {
                    float* o = reinterpret_cast<float*>(a.out0) + ((int64_t)blockIdx.y * a.nq + q) * a.np + p;
                    for (int e = 0; e < n; ++e) o[e] = v[e];
                    continue;
                }
                const int64_t at = (q * a.np + p) * esize(DT);
                if (EPI == E_PLAIN) {
                    for (int e = 0; e < n; ++e) store1<DT>(a.out0 + at + e * esize(DT), v[e]);
                    continue;
                }
                for (int e = 0; e < n; ++e) {
                    float s = v[e];
                    if (a.bias) s += a.bias_f32 ? reinterpret_cast<const float*>(a.bias)[p + e] : load1<DT>(a.bias + (p + e) * esize(DT));
                    if (a.res) s += load1<DT>(a.res + (q * a.ldr + p + e) * esize(DT));
                    if (a.out0) store1<DT>(a.out0 + at + e * esize(DT), s);
                    if (a.out1) store1<DT>(a.out1 + at + e * esize(DT), act_value(a.act, s));
                }
            }
    }
}

// parts [nparts][n] float32 -> their sum, part 0 first, in dtype
template <int DT>
__global__ __launch_bounds__(256) void k_add_parts(const float* __restrict__ parts, int nparts, int64_t n, char* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.0f;
    for (int k = 0; k < nparts; ++k) s += parts[k * n + i];
    store1<DT>(out + i * esize(DT), s);
}

template <int DT>
__global__ __launch_bounds__(256) void k_zero(int64_t n, char* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) store1<DT>(out + i * esize(DT), 0.0f);
}

template <int DT, int PLAY, int QLAY, int EPI>
int launch_gemm(GemmArgs a, int parts, hipStream_t st) {
    constexpr int BP = 128, BQ = 128, BK = DT == BS_DT_F32 ? 16 : 64;
    a.tp = (a.np + BP - 1) / BP;
    a.tiles = (int64_t)a.tp * ((a.nq + BQ - 1) / BQ);
    const int64_t blocks = (a.tiles + 7) / 8 * 8;
    if (blocks > 0x7fffffff) return BS_EINVAL;
    hipLaunchKernelGGL((k_rows_gemm<DT, PLAY, QLAY, EPI, BP, BQ, 64, 64, BK>), dim3((unsigned)blocks, (unsigned)parts), dim3(256), 0, st, a);
    return rows_rc();
}

// how the rows of a weight gradient are cut into parts: enough workgroups to fill the chip twice over, none under 256 rows
void split_rows(int64_t rows, int K, int N, int64_t* part, int64_t* parts) {
    const int64_t tiles = (int64_t)((K + 127) / 128) * ((N + 127) / 128);
    int64_t want = (512 + tiles - 1) / tiles;
    const int64_t most = (rows + 255) / 256;
    if (want > most) want = most;
    if (want < 1) want = 1;
    *part = ((rows + want - 1) / want + 63) / 64 * 64;
    if (*part < 64) *part = 64;                               // no rows
    *parts = rows ? (rows + *part - 1) / *part : 1;
}

}  // namespace

extern "C" {

int bs_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, const void* res,
                  int64_t ldr, void* sum_out, void* act_out, int act, int dtype, int64_t rows, int K, int N, void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1 || act < BS_ACT_NONE || act > BS_ACT_GELU) return BS_EINVAL;
    if (rows == 0) return BS_OK;
    if (!x || !w || ldx < K || ldw < K || (res && ldr < N) || (!sum_out && !act_out)) return BS_EINVAL;
    if (bias && bias_dtype != BS_DT_F32 && bias_dtype != dtype) return BS_EINVAL;
    GemmArgs a = {};
    a.P = (const char*)w; a.ldp = ldw; a.np = N;
    a.Q = (const char*)x; a.ldq = ldx; a.nq = rows;
    a.nk = a.kpart = K;
    a.bias = (const char*)bias; a.bias_f32 = bias_dtype == BS_DT_F32;
    a.res = (const char*)res; a.ldr = ldr;
    a.out0 = (char*)sum_out; a.out1 = (char*)act_out; a.act = act;
    hipStream_t st = rows_stream(stream);
    if (dtype == BS_DT_F32) return launch_gemm<BS_DT_F32, L_KC, L_KC, E_LAYER>(a, 1, st);
    if (dtype == BS_DT_BF16) return launch_gemm<BS_DT_BF16, L_KC, L_KC, E_LAYER>(a, 1, st);
    return launch_gemm<BS_DT_F16, L_KC, L_KC, E_LAYER>(a, 1, st);
}

int bs_linear_grad_x(const void* ds, int64_t ldds, const void* w, int64_t ldw, void* dx, int dtype, int64_t rows, int K, int N,
                     void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1) return BS_EINVAL;
    if (rows == 0) return BS_OK;
    if (!ds || !w || !dx || ldds < N || ldw < K) return BS_EINVAL;
    GemmArgs a = {};
    a.P = (const char*)w; a.ldp = ldw; a.np = K;
    a.Q = (const char*)ds; a.ldq = ldds; a.nq = rows;
    a.nk = a.kpart = N;
    a.out0 = (char*)dx;
    hipStream_t st = rows_stream(stream);
    if (dtype == BS_DT_F32) return launch_gemm<BS_DT_F32, L_IC, L_KC, E_PLAIN>(a, 1, st);
    if (dtype == BS_DT_BF16) return launch_gemm<BS_DT_BF16, L_IC, L_KC, E_PLAIN>(a, 1, st);
    return launch_gemm<BS_DT_F16, L_IC, L_KC, E_PLAIN>(a, 1, st);
}

int64_t bs_linear_grad_w_workspace(int dtype, int64_t rows, int K, int N) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1) return BS_EINVAL;
    int64_t part, parts;
    split_rows(rows, K, N, &part, &parts);
    return parts > 1 ? parts * K * N * 4 : 0;
}

int bs_linear_grad_w(const void* ds, int64_t ldds, const void* x, const int8_t* x_exps, int64_t ldx, void* dw, int dtype,
                     int64_t rows, int K, int N, void* workspace, int64_t workspace_bytes, void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1 || !dw) return BS_EINVAL;
    hipStream_t st = rows_stream(stream);
    const int64_t n = (int64_t)K * N;
    const unsigned blocks = (unsigned)((n + 255) / 256);
    if (rows == 0) {
        if (dtype == BS_DT_F32) hipLaunchKernelGGL(k_zero<BS_DT_F32>, dim3(blocks), dim3(256), 0, st, n, (char*)dw);
        else hipLaunchKernelGGL(k_zero<BS_DT_F16>, dim3(blocks), dim3(256), 0, st, n, (char*)dw);
        return rows_rc();
    }
    if (!ds || !x || ldds < N || ldx < K) return BS_EINVAL;
    int64_t part, parts;
    split_rows(rows, K, N, &part, &parts);
    if (parts > 1 && (!workspace || workspace_bytes < parts * n * 4)) return BS_EINVAL;
    GemmArgs a = {};
    a.P = (const char*)x; a.Pexp = x_exps; a.lpe = (K + P8_BLOCK - 1) / P8_BLOCK; a.ldp = ldx; a.np = K;
    a.Q = (const char*)ds; a.ldq = ldds; a.nq = N;
    a.nk = rows; a.kpart = part;
    a.out0 = (char*)(parts > 1 ? workspace : dw);
    int rc;
#define GRAD_W(DT) (parts > 1 ? (x_exps ? launch_gemm<DT, L_P8, L_IC, E_PART>(a, (int)parts, st) : launch_gemm<DT, L_IC, L_IC, E_PART>(a, (int)parts, st)) \
                              : (x_exps ? launch_gemm<DT, L_P8, L_IC, E_PLAIN>(a, 1, st) : launch_gemm<DT, L_IC, L_IC, E_PLAIN>(a, 1, st)))
    if (dtype == BS_DT_F32) rc = GRAD_W(BS_DT_F32);
    else if (dtype == BS_DT_BF16) rc = GRAD_W(BS_DT_BF16);
    else rc = GRAD_W(BS_DT_F16);
#undef GRAD_W
    if (rc != BS_OK || parts == 1) return rc;
    const float* ws = (const float*)workspace;
    if (dtype == BS_DT_F32) hipLaunchKernelGGL(k_add_parts<BS_DT_F32>, dim3(blocks), dim3(256), 0, st, ws, (int)parts, n, (char*)dw);
    else if (dtype == BS_DT_BF16) hipLaunchKernelGGL(k_add_parts<BS_DT_BF16>, dim3(blocks), dim3(256), 0, st, ws, (int)parts, n, (char*)dw);
    else hipLaunchKernelGGL(k_add_parts<BS_DT_F16>, dim3(blocks), dim3(256), 0, st, ws, (int)parts, n, (char*)dw);
    return rows_rc();
}

}  // extern "C"
