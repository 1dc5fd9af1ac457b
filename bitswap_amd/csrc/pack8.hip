// pack8.hip -- saved activations in 8 bits, and the pointwise part of a layer's backward pass: ds = g_sum + g_act act'(s) with the
// column sums that are the bias gradient.  All bound by memory traffic: one 16-byte access per operand and thread step.
//
//   pack    e = the smallest exponent with max|x| <= 127 2^e over 32 channels of a row, code = rint(x 2^-e)
//   unpack  x = code 2^e
//
// Measured, 102400 x 256 float32 (105 MB, 27 MB of codes): pack 25 us (5.3 TB/s), unpack 20 us (6.7 TB/s: the codes from the caches);
// ds and its column sums of 65536 x 1024 bfloat16 from 8-bit sums (338 MB) 77 us (4.4 TB/s), of 25600 x 256 float32 from both gradients
// 17.7 us (105 MB, 5.9 TB/s).  A large copy runs at 4.9 TB/s.
#include "rows_dev.h"

namespace {

// One thread = 16 bytes of a row; the 32 / V threads of a block of 32 channels are neighbours in a wavefront and take the maximum
// over it together, so that x is read once.
template <int DT>
__global__ __launch_bounds__(256) void k_pack8(const char* __restrict__ x, int64_t ldx, int8_t* __restrict__ codes,
                                               int8_t* __restrict__ exps, int64_t rows, int C, int nb) {
    constexpr int V = vlen(DT), LB = P8_BLOCK / V;
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = t / (nb * LB);
    const int ch = (int)(t - row * (nb * LB));
    const int c = ch * V, left = C - c;
    float f[V];
    float m = 0.0f;
    if (row < rows && left > 0) {
        load_vec<DT>(x + (row * ldx + c) * esize(DT), left, f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float a = fabsf(f[i]);
            m = a < __builtin_inff() ? fmaxf(m, a) : m;                 // false for a NaN as well
        }
    }
#pragma unroll
    for (int o = 1; o < LB; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    if (row >= rows || left <= 0) return;
    const int e = p8_exponent<DT>(m);
    const float inv = p8_pow2(-e);
    uint32_t q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = fabsf(f[i]) < __builtin_inff() ? (uint32_t)(int)fminf(fmaxf(rintf(f[i] * inv), -127.0f), 127.0f) & 255u : 128u;
    int8_t* const out = codes + row * C + c;
    if (left >= V) {
        if (V == 4) {
            const uint32_t w = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
            __builtin_memcpy(out, &w, 4);
        } else {
            const u32x2 w = {q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4 % V] | q[5 % V] << 8 | q[6 % V] << 16 | q[7 % V] << 24};
            store8((char*)out, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < left) out[i] = (int8_t)q[i];
    }
    if (ch % LB == 0) exps[row * nb + ch / LB] = (int8_t)e;
}

template <int DT>
__global__ __launch_bounds__(256) void k_unpack8(const int8_t* __restrict__ codes, const int8_t* __restrict__ exps, char* __restrict__ x,
                                                 int64_t rows, int C, int nb, int cpr) {
    constexpr int V = vlen(DT);
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = t / cpr;
    if (row >= rows) return;
    const int c = (int)(t - row * cpr) * V;
    float f[V];
    load_codes<V>(codes + row * C, exps + row * nb, c, C - c, f);
    store_out<DT>(x + (row * C + c) * esize(DT), C - c, f, C);
}

struct ActGradArgs {
    const char *g_sum, *g_act, *s;
    const int8_t* exps;
    int64_t ldgs, ldga, lds, rows, part;
    int N, nb, act;
    char* ds;
    int64_t ldds;
    float* parts;             // [parts][N]
};

// workgroup = CL threads along the channels x 256 / CL rows at a time, over a part of the rows; every thread keeps the column sums
// of its V channels.  Parts: 2048 workgroups in all, none under 32 rows; their sums are joined in a second launch, always in the same
// order (4 to 5 us, where atomics would change their order from call to call).
// ds is rounded to the type here, once: it is what dres returns, half the bytes of float32, and what 16-bit matrix instructions take.
// dx and dw are products of the rounded ds (65536 x 512 x 1024 bfloat16: off by 0.0023 of their norm; with ds whole 0.0017, for a
// second limb and twice the products' 170 us).  db adds ds up before its rounding.
template <int DT, bool SAVED8>
__global__ __launch_bounds__(256) void k_act_grad(const ActGradArgs a, int cl_log2) {
    constexpr int V = vlen(DT), ES = esize(DT);
    __shared__ float red[256 * V];
    const int CL = 1 << cl_log2, RL = 256 >> cl_log2;
    const int tid = threadIdx.x, cl = tid & (CL - 1), rl = tid >> cl_log2;
    const int c = (blockIdx.x * CL + cl) * V, left = a.N - c;
    const int64_t r0 = (int64_t)blockIdx.y * a.part;
    const int64_t r1 = r0 + a.part < a.rows ? r0 + a.part : a.rows;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    if (left > 0)
        for (int64_t r = r0 + rl; r < r1; r += RL) {
            float d[V];
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = 0.0f;
            if (a.g_act) {
                load_vec<DT>(a.g_act + (r * a.ldga + c) * ES, left, d);
                if (a.act != BS_ACT_NONE) {
                    float s[V];
                    if (SAVED8) load_codes<V>((const int8_t*)a.s + r * a.lds, a.exps + r * a.nb, c, left, s);
                    else load_vec<DT>(a.s + (r * a.lds + c) * ES, left, s);
                    act_slopes<V>(a.act, s, d);
                }
            }
            if (a.g_sum) {
                float g[V];
                load_vec<DT>(a.g_sum + (r * a.ldgs + c) * ES, left, g);
#pragma unroll
                for (int i = 0; i < V; ++i) d[i] += g[i];
            }
            if (a.ds) store_vec<DT>(a.ds + (r * a.ldds + c) * ES, c + V <= a.ldds ? V : left, d);      // (d is 0 behind the last channel)
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] += d[i];
        }
    if (!a.parts) return;
#pragma unroll
    for (int i = 0; i < V; ++i) red[(rl * CL + cl) * V + i] = sum[i];
    __syncthreads();
    for (int i = tid; i < CL * V; i += 256) {
        const int col = blockIdx.x * CL * V + i;
        if (col >= a.N) continue;
        float s = 0.0f;
        for (int r = 0; r < RL; ++r) s += red[r * CL * V + i];
        a.parts[(int64_t)blockIdx.y * a.N + col] = s;
    }
}

void split_rows(int64_t rows, int N, int64_t* part, int64_t* parts) {
    const int slabs = (N + 127) / 128;
    int64_t want = (2048 + slabs - 1) / slabs;
    int lanes = 1;                                            // along the channels, at most (k_act_grad)
    while (lanes < 32 && lanes * 4 < N) lanes *= 2;
    const int64_t most = rows <= 8 * (256 / lanes) ? 1 : (rows + 31) / 32;     // (eight rows a thread: sooner done than joined)
    if (want > most) want = most;
    if (want < 1) want = 1;
    *part = (rows + want - 1) / want;
    *parts = *part ? (rows + *part - 1) / *part : 1;
}

}  // namespace

extern "C" {

int bs_pack8(const void* x, int64_t ldx, int8_t* codes, int8_t* exps, int dtype, int64_t rows, int channels, void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || channels < 1 || channels > (1 << 30)) return BS_EINVAL;
    if (rows == 0) return BS_OK;
    if (!x || !codes || !exps || ldx < channels) return BS_EINVAL;
    const int nb = (channels + P8_BLOCK - 1) / P8_BLOCK;
    if (rows > MAX_ROWS / nb) return BS_EINVAL;
    const int64_t threads = rows * nb * (dtype == BS_DT_F32 ? 8 : 4), blocks = (threads + 255) / 256;
    if (too_many(blocks, 256)) return BS_EINVAL;
    hipStream_t st = rows_stream(stream);
#define PACK(DT) hipLaunchKernelGGL(k_pack8<DT>, dim3((unsigned)blocks), dim3(256), 0, st, (const char*)x, ldx, codes, exps, rows, channels, nb)
    if (dtype == BS_DT_F32) PACK(BS_DT_F32);
    else if (dtype == BS_DT_BF16) PACK(BS_DT_BF16);
    else PACK(BS_DT_F16);
#undef PACK
    return rows_rc();
}

int bs_unpack8(const int8_t* codes, const int8_t* exps, void* x, int dtype, int64_t rows, int channels, void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || channels < 1 || channels > (1 << 30)) return BS_EINVAL;
    if (rows == 0) return BS_OK;
    if (!x || !codes || !exps) return BS_EINVAL;
    const int nb = (channels + P8_BLOCK - 1) / P8_BLOCK, V = dtype == BS_DT_F32 ? 4 : 8, cpr = (channels + V - 1) / V;
    if (rows > MAX_ROWS / cpr) return BS_EINVAL;
    const int64_t blocks = (rows * cpr + 255) / 256;
    if (too_many(blocks, 256)) return BS_EINVAL;
    hipStream_t st = rows_stream(stream);
#define UNPACK(DT) hipLaunchKernelGGL(k_unpack8<DT>, dim3((unsigned)blocks), dim3(256), 0, st, codes, exps, (char*)x, rows, channels, nb, cpr)
    if (dtype == BS_DT_F32) UNPACK(BS_DT_F32);
    else if (dtype == BS_DT_BF16) UNPACK(BS_DT_BF16);
    else UNPACK(BS_DT_F16);
#undef UNPACK
    return rows_rc();
}

int64_t bs_act_grad_workspace(int64_t rows, int N) {
    if (rows < 0 || rows > MAX_ROWS || N < 1) return BS_EINVAL;
    int64_t part, parts;
    split_rows(rows, N, &part, &parts);
    return parts > 1 ? parts * N * 4 : 0;
}

int bs_act_grad(const void* g_sum, int64_t ldgs, const void* g_act, int64_t ldga, const void* s, const int8_t* s_exps, int64_t lds,
                int act, int dtype, int64_t rows, int N, void* ds_out, int64_t ldds, float* db_out, void* workspace,
                int64_t workspace_bytes, void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || N < 1 || N > (1 << 30) || act < BS_ACT_NONE || act > BS_ACT_GELU) return BS_EINVAL;
    hipStream_t st = rows_stream(stream);
    if (rows > 0 && ((!g_sum && !g_act) || (g_sum && ldgs < N) || (g_act && ldga < N) ||
                     (g_act && act != BS_ACT_NONE && (!s || lds < N)))) return BS_EINVAL;
    if (rows == 0 && !db_out) return BS_OK;                  // (an empty ds has no address)
    if ((!ds_out && !db_out) || (ds_out && ldds < N)) return BS_EINVAL;
    int64_t part, parts;
    split_rows(rows, N, &part, &parts);
    if (db_out && parts > 1 && bad_workspace(workspace, workspace_bytes, parts * N * 4)) return BS_EINVAL;
    ActGradArgs a = {};
    a.g_sum = (const char*)g_sum; a.g_act = (const char*)g_act; a.s = (const char*)s; a.exps = s_exps;
    a.ldgs = ldgs; a.ldga = ldga; a.lds = lds; a.rows = rows; a.part = part;
    a.N = N; a.nb = (N + P8_BLOCK - 1) / P8_BLOCK; a.act = act; a.ds = (char*)ds_out; a.ldds = ldds;
    a.parts = db_out ? (parts > 1 ? (float*)workspace : db_out) : nullptr;
    const int V = dtype == BS_DT_F32 ? 4 : 8, chunks = (N + V - 1) / V;
    int cl = 0;
    while ((1 << cl) < chunks && cl < 5) ++cl;
    const dim3 grid((unsigned)((chunks + (1 << cl) - 1) >> cl), (unsigned)parts);
    const bool p8 = s_exps != nullptr;
#define GO(DT) do { if (p8) hipLaunchKernelGGL((k_act_grad<DT, true>), grid, dim3(256), 0, st, a, cl); \
                    else hipLaunchKernelGGL((k_act_grad<DT, false>), grid, dim3(256), 0, st, a, cl); } while (0)
    if (dtype == BS_DT_F32) GO(BS_DT_F32);
    else if (dtype == BS_DT_BF16) GO(BS_DT_BF16);
    else GO(BS_DT_F16);
#undef GO
    if (db_out && parts > 1)
        hipLaunchKernelGGL(k_sum_columns, dim3((unsigned)((N + 31) / 32)), dim3(1024), 0, st, (const float*)workspace, parts, N, N, db_out, (float*)nullptr);
    return rows_rc();
}

}  // extern "C"
