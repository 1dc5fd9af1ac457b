// linear.hip -- products over rows of channels (channels-last activations): s = x w^T + bias (+ res) with its activation, and the
// two products of its backward pass, on the bf16 / f16 matrix cores (v_mfma_f32_32x32x16), float32 sums.
//
//   forward  out[q][p] = sum_k w[p][k] x[q][k]          k = K, the contiguous axis of both: k_rows_dma / k_relay
//   dx       out[q][p] = sum_k w[k][p] ds[q][k]         k = N; as the forward, w turned round first (k_prepare) where rows are many
//   dw       out[q][p] = sum_k x[k][p] ds[k][q]         k = rows, the strided axis of both: k_over_dma, cut into parts of the rows
//
// What bounds them: the bytes of x, residual and outputs where K is a few hundred (a copy runs at 4.9 TB/s here), the matrix cores
// where it is long (a library product reaches 1420 TFLOP/s in bfloat16 at 16384 x 2048 x 2048; float32 costs six such products), and
// below some hundred rows the latency of one load, a chain of matrix instructions and one store.
//
// float32 operands are split into three bfloat16 limbs (their sum is the float exactly from 2^-110 on; of a smaller one the bits below
// 2^-133 are lost, which no bfloat16 has) and multiplied as the six limb products of total order <= 2; what is left out is of relative
// size 2^-24.  Limb products of an infinity or of a value that rounds to one are
// NaN, so a sum that does not come out finite is added up again in float32.
//
// The output channel is the row index of the matrix instruction: a lane then holds, for one row q = lane % 32 of activations, the
// channels 8 g + 4 (lane / 32) + 0..3, g = 0..3, of a 32x32 tile.
#include <type_traits>

#include "rows_dev.h"

namespace {

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2* lds_i32x2;

enum { E_LAYER = 0, E_PLAIN = 1 };                        // bias + residual + activation | one rounding
constexpr int limbs_of(int dt) { return dt == BS_DT_F32 ? 3 : 1; }
constexpr int kb_of(int dt) { return dt == BS_DT_F32 ? 16 : 32; }          // k that lie side by side in a laid out w

template <int DT>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if (DT == BS_DT_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two floats -> their three bfloat16 limbs, round to nearest
__device__ __forceinline__ void limbs2(float a, float b, uint32_t* l) {
    l[0] = pk_bf16(a, b);
    a -= bits_f32(l[0] << 16);
    b -= bits_f32(l[0] & 0xffff0000u);
    l[1] = pk_bf16(a, b);
    a -= bits_f32(l[1] << 16);
    b -= bits_f32(l[1] & 0xffff0000u);
    l[2] = pk_bf16(a, b);
}

// all limb products of a 16-deep block, small ones first: ONE order for every kernel here, so that which kernel takes a product
// does not show in its bits
template <int DT, int LP, int LQ, int NP, int NQ>
__device__ __forceinline__ void multiply(const u32x4 (&fp)[NP][LP], const u32x4 (&fq)[NQ][LQ], f32x16 (&acc)[NP][NQ]) {
#pragma unroll
    for (int o = LP + LQ > 2 ? 2 : 0; o >= 0; --o)
#pragma unroll
        for (int l = 0; l < LP; ++l) {
            if (o - l < 0 || o - l >= LQ) continue;
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int j = 0; j < NQ; ++j) acc[i][j] = mfma<DT>(fp[i][l], fq[j][(o - l >= 0 && o - l < LQ) ? o - l : 0], acc[i][j]);
        }
}

struct RowsArgs {
    const char *x, *w;                 // operands as the caller holds them
    int64_t ldx, ldw;
    const char* xd;                    // x as DMA takes it (rows of whole chunks): x itself or its copy
    int64_t ldxd;
    const char* wl;                    // w as the kernel reads it, 16-bit: laid out (k_prepare), or w itself
    int64_t sp, sk, sl;                // element (limb, p, k) is at limb sl + p sp + k / KB sk + k % KB
    int64_t rows;
    int K, N;
    int Kx;                            // k that rows of x hold in whole 16-byte chunks, zero from K on
    int wt;                            // w is [K, N] (the gradient of x)
    int tp;
    int64_t tiles;
    const char *bias, *res;
    int64_t ldr;
    char *sum, *act_out;               // E_PLAIN: sum
    int act, bias_f32;
};

// the sum once more, in float32 arithmetic
template <int DT>
__device__ __forceinline__ float again(const RowsArgs& a, int64_t q, int64_t p) {
    float s = 0.0f;
    for (int k = 0; k < a.K; ++k)
        s = fmaf(load1<DT>(a.w + (a.wt ? (int64_t)k * a.ldw + p : p * a.ldw + k) * esize(DT)), load1<DT>(a.x + (q * a.ldx + k) * esize(DT)), s);
    return s;
}

// what becomes of V neighbouring channels of a row (n of them exist); bias, r: their bias and residual
template <int DT, int EPI>
__device__ __forceinline__ void finish(const RowsArgs& a, int64_t q, int64_t p, int n, float* v, const float* bias, u32x4 r) {
    constexpr int V = vlen(DT), ES = esize(DT);
    if (DT == BS_DT_F32) {
        bool odd = false;
#pragma unroll
        for (int e = 0; e < V; ++e) odd |= (f32_bits(v[e]) & 0x7f800000u) == 0x7f800000u;
        if (odd) {
            for (int e = 0; e < V; ++e)
                if ((f32_bits(v[e]) & 0x7f800000u) == 0x7f800000u && e < n) v[e] = again<DT>(a, q, p + e);
        }
    }
    const int64_t at = (q * a.N + p) * ES;
    if (EPI == E_LAYER) {
        float t[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += bias[e];
        if (a.res) {
            unpack16<DT>(r, t);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += t[e];
        }
        if (a.sum) store_out<DT>(a.sum + at, n, v, a.N);
        if (a.act_out) {
            act_values<DT, V>(a.act, v, t);
            store_out<DT>(a.act_out + at, n, t, a.N);
        }
    } else {
        store_out<DT>(a.sum + at, n, v, a.N);
    }
}
template <int DT>
__device__ __forceinline__ void load_bias(const RowsArgs& a, int64_t p, float* b) {
    constexpr int V = vlen(DT);
#pragma unroll
    for (int e = 0; e < V; ++e) b[e] = 0.0f;
    if (!a.bias || p >= a.N) return;
    if (DT != BS_DT_F32 && a.bias_f32) {
#pragma unroll
        for (int e = 0; e < V; e += 4)
            if (p + e < a.N) load_vec<BS_DT_F32>(a.bias + (p + e) * 4, a.N - p - e < 4 ? (int)(a.N - p - e) : 4, b + e);
    } else {
        load_vec<DT>(a.bias + p * esize(DT), a.N - p < V ? (int)(a.N - p) : V, b);
    }
}
template <int DT>
__device__ __forceinline__ u32x4 residual(const RowsArgs& a, int64_t q, int64_t p, int n) {
    return load_raw<DT>(a.res + (q * a.ldr + p) * esize(DT), n);
}

// A wavefront's 32 rows x 64 channels from the registers of the matrix instruction to rows of memory, by way of its own piece of
// shared memory (row stride 68 floats: 16 lanes of a 16-byte access touch all banks): whole 16-byte accesses, 128 or 256 bytes of a
// row side by side.
constexpr int turn_bytes(int cols) { return 32 * (cols + 4) * 4; }
// COLS: 64, or 32 where a wavefront has one 32x32 tile across
template <int DT, int EPI, int COLS>
__device__ __forceinline__ void turn_and_finish(const RowsArgs& a, const f32x16& a0, const f32x16& a1, float* mine, int lane, int64_t q0,
                                                int64_t p0, const float* bias) {
    constexpr int V = vlen(DT), LPR = COLS / V, RI = 64 / LPR, NI = 32 / RI, ST = COLS + 4;      // lanes per row, rows at a time
    const int c = (lane % LPR) * V;
    const int64_t p = p0 + c, left = a.N - p;
    const int n = left < V ? (int)left : V;
    u32x4 res[NI];
    if (EPI == E_LAYER && a.res && n > 0) {                                    // all residuals of the piece are asked for at once
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int64_t q = q0 + lane / LPR + i * RI;
            if (q < a.rows) res[i] = residual<DT>(a, q, p, n);
        }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float* const at = mine + (lane & 31) * ST + 8 * g + 4 * (lane >> 5);
        *reinterpret_cast<f32x4*>(at) = f32x4{a0[4 * g], a0[4 * g + 1], a0[4 * g + 2], a0[4 * g + 3]};
        if (COLS == 64) *reinterpret_cast<f32x4*>(at + 32) = f32x4{a1[4 * g], a1[4 * g + 1], a1[4 * g + 2], a1[4 * g + 3]};
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (n > 0) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = lane / LPR + i * RI;
            if (q0 + r >= a.rows) break;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const f32x4 t = *reinterpret_cast<const f32x4*>(mine + r * ST + c + e);
                v[e] = t[0]; v[e + 1] = t[1]; v[e + 2] = t[2]; v[e + 3] = t[3];
            }
            finish<DT, EPI>(a, q0 + r, p, n, v, bias, res[i]);
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---- forward and dx, many rows ------------------------------------------------------------------------------------------------
// Tile of BQ rows x BP channels, BK deep steps.  Both operands come by DMA (rows of x that are no whole aligned 16-byte chunks are
// copied to such first, k_prepare) through a ring of NS buffers with one barrier a step; fragments are read one 16-deep block ahead of
// the matrix instructions.  float32 rows lie in shared memory as they are and are split into limbs after the read, between the
// matrix instructions of the block before: 32 bytes a fragment instead of 48, and nothing goes back to shared memory.  Rows of BK k
// lie there as 16-byte chunks, chunk c in slot c ^ f(row), f such that the 16 lanes a 16-byte read serves together (0-3, 12-15, 20-27;
// the others) touch all 64 banks.
//
// Measured: bfloat16 16384 x 2048 x 2048 with GELU, both outputs 134 us (1025 TFLOP/s; the library's product alone 97 us, what is more
// is the epilogue, which nothing covers with one workgroup a compute unit: 256 x 128 tiles, two of them, 156 us); float32
// 102400 x 256 x 256 with residual and both outputs 120 us where two sets of tensors alternate (3.5 TB/s of 419 MB; 55 us of matrix
// instructions, 86 of traffic, one partly behind the other), 100 to 114 over and over on one set, as the comparisons below are timed;
// bfloat16 25600 x 256 x 256 11.8 us.  Kept after trying the other way: the compiler places the limb splits
// (places given to them: 105 us against 100 for 102400 x 256 x 256); a third block of reads ahead, six buffers or steps twice as
// deep change nothing or cost; 16-bit 128x128 tiles over eight wavefronts of 32 rows, not four of 64 (102400 x 256 x 256 43 and 49 us);
// 64x64 over four of 32x32, not two of 32x64 (4096 x 256 x 256 5.6 and 6.7 us); float32
// 128x128 over four wavefronts of 32 rows x 128 channels, which split a row into limbs once, not of 64x64 (16384 x 1024 x 1024 187 and 192 us).
// Residuals asked for before the sums change nothing (115 and 112 us).
__device__ __forceinline__ constexpr int wait_vm(int v) { return (v & 15) | (7 << 4) | ((v >> 4) << 14); }      // vmcnt(v), lgkmcnt(0)

template <int DT, int EPI, int BQ, int BP, int WQ, int WP, int BK, int NS, int PER_SIMD>
__global__ __launch_bounds__((BQ / WQ) * (BP / WP) * 64, PER_SIMD) void k_rows_dma(const RowsArgs a) {
    constexpr int NW = (BQ / WQ) * (BP / WP), L = limbs_of(DT), ES = esize(DT), CK = 16 / ES;       // CK: k of a chunk of x
    constexpr int XS = BK * ES / 16, WS = BK / 8;                                                    // chunks of a row
    constexpr int XB = BQ * BK * ES, WB = L * BP * BK * 2, STAGE = XB + WB;
    constexpr int XI = XB / 1024 / NW, WI = WB / 1024 / NW;
    constexpr int NP = WP / 32, NQ = WQ / 32;
    static_assert(XB % (1024 * NW) == 0 && WB % (1024 * NW) == 0 && NS * STAGE <= 160 * 1024 && (NP == 1 || NP % 2 == 0), "");
    constexpr int COLS = NP == 1 ? 32 : 64, TURN = turn_bytes(COLS);
    __shared__ __align__(16) char lds[NS * STAGE > NW * TURN ? NS * STAGE : NW * TURN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wp = wave % (BP / WP), wq = wave / (BP / WP);
    auto swz = [](int slots, int row, int c) { return slots == 8 ? (c ^ ((row >> 1) & 7)) : slots == 4 ? (c ^ ((row >> 2) & 3)) : (c ^ ((row >> 3) & 1)); };
    const int64_t per = (a.tiles + 7) / 8;
    const int64_t t = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (t >= a.tiles) return;
    const int64_t q0 = t / a.tp * BQ;
    const int p0 = (int)(t % a.tp) * BP;
    const int steps = (a.K + BK - 1) / BK;
    const char* const xb = a.xd + q0 * a.ldxd * ES;
    const char* const wb = a.wl + p0 * a.sp * 2;
    constexpr int KB = kb_of(DT);
    static_assert(BK % KB == 0, "");
    uint32_t xo[XI], wo[WI];
    int xk[XI];
#pragma unroll
    for (int n = 0; n < XI; ++n) {
        const int row = (wave * XI + n) * (64 / XS) + lane / XS, c = swz(XS, row, lane % XS);
        const int64_t r = q0 + row < a.rows ? row : a.rows - 1 - q0;            // rows behind the last: not stored
        xo[n] = (uint32_t)(r * a.ldxd * ES + c * 16);
        xk[n] = a.Kx - c * CK;
    }
#pragma unroll
    for (int n = 0; n < WI; ++n) {
        const int r = (wave * WI + n) * (64 / WS) + lane / WS, limb = r / BP, row = r % BP;
        const int pr = p0 + row < a.N ? row : a.N - 1 - p0;                       // channels behind the last: not stored
        const int k = swz(WS, row, lane % WS) * 8;
        wo[n] = (uint32_t)((limb * a.sl + pr * a.sp + k / KB * a.sk + k % KB) * 2);
    }
    // a step whose k all exist: no branch among the loads
    auto issue_whole = [&](int s, int slot) {
        char* const st = lds + slot * STAGE;
        const char* const xs = xb + (int64_t)s * BK * ES;
        const char* const ws = wb + (int64_t)s * (BK / KB) * a.sk * 2;
#pragma unroll
        for (int n = 0; n < XI; ++n) {
            const char* const src = xs + xo[n];
            __builtin_amdgcn_global_load_lds(src, (lds_ptr)(st + (wave * XI + n) * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int n = 0; n < WI; ++n) {
            const char* const src = ws + wo[n];
            __builtin_amdgcn_global_load_lds(src, (lds_ptr)(st + XB + (wave * WI + n) * 1024), 16, 0, 0);
        }
    };
    auto issue = [&](int s, int slot) {
        if ((s + 1) * BK <= a.Kx) return issue_whole(s, slot);
        char* const st = lds + slot * STAGE;
        const char* const xs = xb + (int64_t)s * BK * ES;
        const char* const ws = wb + (int64_t)s * (BK / KB) * a.sk * 2;
#pragma unroll
        for (int n = 0; n < XI; ++n) {
            const char* const src = xs + xo[n];
            if (s * BK < xk[n]) __builtin_amdgcn_global_load_lds(src, (lds_ptr)(st + (wave * XI + n) * 1024), 16, 0, 0);
            else *reinterpret_cast<u32x4*>(st + (wave * XI + n) * 1024 + lane * 16) = u32x4{0, 0, 0, 0};       // behind K: zero
        }
#pragma unroll
        for (int n = 0; n < WI; ++n) {
            const char* const src = ws + wo[n];
            __builtin_amdgcn_global_load_lds(src, (lds_ptr)(st + XB + (wave * WI + n) * 1024), 16, 0, 0);
        }
    };
    // fragments of 16 k: w's limbs, x as it lies in shared memory
    struct Frag {
        u32x4 p[NP][L], q[NQ][DT == BS_DT_F32 ? 2 : 1];
    };
    auto read = [&](const char* st, int b, Frag& f) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const int row = wq * WQ + j * 32 + (lane & 31);
#pragma unroll
            for (int h = 0; h < (DT == BS_DT_F32 ? 2 : 1); ++h) {
                const int c = DT == BS_DT_F32 ? 4 * b + 2 * (lane >> 5) + h : 2 * b + (lane >> 5);
                f.q[j][h] = *reinterpret_cast<const u32x4*>(st + row * (BK * ES) + swz(XS, row, c) * 16);
            }
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int row = wp * WP + i * 32 + (lane & 31);
#pragma unroll
            for (int l = 0; l < L; ++l)
                f.p[i][l] = *reinterpret_cast<const u32x4*>(st + XB + (l * BP + row) * (BK * 2) + swz(WS, row, 2 * b + (lane >> 5)) * 16);
        }
    };
    auto split = [&](const Frag& f, u32x4 (&q)[NQ][L]) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            if constexpr (DT == BS_DT_F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t l3[3];
                    limbs2(bits_f32(f.q[j][e / 2][(2 * e) & 3]), bits_f32(f.q[j][e / 2][(2 * e + 1) & 3]), l3);
                    q[j][0][e] = l3[0];
                    q[j][1][e] = l3[1];
                    q[j][2][e] = l3[2];
                }
            } else {
                q[j][0] = f.q[j][0];
            }
        }
    };
    f32x16 acc[NP][NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (s < steps) issue(s, s);
    if (NS <= a.Kx / BK) __builtin_amdgcn_s_waitcnt(wait_vm((NS - 1) * (XI + WI)));      // NS whole steps are on their way
    else __builtin_amdgcn_s_waitcnt(wait_vm(0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    constexpr int SB = BK / 16;
    Frag f;
    u32x4 q[NQ][L];
    read(lds, 0, f);
    split(f, q);
    int slot = 0;
    // One step.  RUN: the step NS ahead exists whole.  The next step has landed for this wavefront once only the DMA of the NS - 2 steps
    // behind it is in flight (near the end everything is waited for), and for all of them after the barrier; what was read of this
    // step is in registers (lgkmcnt), its buffer takes the step NS ahead.  Reads, DMA and the split go between the matrix
    // instructions, which work on what was read a block before.
    auto step = [&](int s, auto run) {
        constexpr bool RUN = decltype(run)::value;
        constexpr int M = (L == 3 ? 6 : 1) * NP * NQ, R = NQ * (DT == BS_DT_F32 ? 2 : 1) + NP * L, D = XI + WI;
        const int next = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
        for (int b = 0; b < SB; ++b) {
            Frag g;
            if (b == SB - 1) {
                if (RUN) __builtin_amdgcn_s_waitcnt(wait_vm((NS - 2) * D));
                else __builtin_amdgcn_s_waitcnt(wait_vm(0));
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (!RUN && s + NS < steps) issue(s + NS, slot);
                __builtin_amdgcn_sched_barrier(0);
                read(lds + next * STAGE, 0, g);               // (behind the last step: not used)
                if (RUN) issue_whole(s + NS, slot);
            } else {
                __builtin_amdgcn_sched_barrier(0);
                read(lds + slot * STAGE, b + 1, g);
            }
            u32x4 qn[NQ][L];
            multiply<DT, L, L, NP, NQ>(f.p, q, acc);
            split(g, qn);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                       // one matrix instruction
                if (m < (R + 1) / 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);                  // two LDS reads
                else if (RUN && b == SB - 1 && m < (R + 1) / 2 + D) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            f = g;
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int l = 0; l < L; ++l) q[j][l] = qn[j][l];
        }
        slot = next;
    };
    const int whole = a.Kx / BK;                               // steps s with s + NS < whole have a whole step NS ahead
    int s = 0;
#pragma unroll SB == 1 ? 2 : 1
    for (; s + NS < whole; ++s) step(s, std::true_type{});
    for (; s < steps; ++s) step(s, std::false_type{});
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(lds + wave * TURN);
#pragma unroll
    for (int i = 0; i < NP; i += COLS / 32) {
        const int p = p0 + wp * WP + i * 32;
        float bias[vlen(DT)];
        if (EPI == E_LAYER) load_bias<DT>(a, p + lane % (COLS / vlen(DT)) * vlen(DT), bias);
#pragma unroll
        for (int j = 0; j < NQ; ++j)
            turn_and_finish<DT, EPI, COLS>(a, acc[i][j], acc[i + COLS / 32 - 1][j], mine, lane, q0 + wq * WQ + j * 32, p, bias);
    }
}

// ---- forward and dx, few rows -------------------------------------------------------------------------------------------------
// One 32x32 tile a workgroup.  Its four wavefronts hold four runs of k in registers, loaded at once straight from memory (the next
// four while these are multiplied), and pass the sums on from run to run (a relay): the order of k_rows_dma, at the latency of
// about one load.  w comes as the caller holds it; dx (WT) gathers 8 rows of it a fragment, a launch less than turning it round first.
// Measured: 1 x 1024 x 1024 float16 7.2 us, 256 x 256 x 256 float32 7.5 us with a residual; bound by that latency (an empty launch
// takes 2 us).
template <int DT, int EPI, bool WT>
__global__ __launch_bounds__(256) void k_relay(const RowsArgs a) {
    constexpr int L = limbs_of(DT), NS = DT == BS_DT_F32 ? 4 : 8, ES = esize(DT), RUN = NS * 16;
    __shared__ __align__(16) char lds[turn_bytes(64)];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t q0 = blockIdx.x / a.tp * 32;
    const int p0 = (int)(blockIdx.x % a.tp) * 32;
    const int64_t q = q0 + (lane & 31) < a.rows ? q0 + (lane & 31) : a.rows - 1;
    const int p = p0 + (lane & 31) < a.N ? p0 + (lane & 31) : a.N - 1;
    const char* const xp = a.x + q * a.ldx * ES;
    const char* const wp = a.w + (WT ? p : (int64_t)p * a.ldw) * ES;
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
    constexpr int RAW = DT == BS_DT_F32 ? 2 : 1;
    auto fetch = [&](const char* base, int k, u32x4* r) {          // 8 values from k on, zero behind K
        const int left = a.K - k;
        const char* const at = base + (int64_t)k * ES;
        r[0] = left > 0 ? load_raw<DT>(at, left) : u32x4{0, 0, 0, 0};
        if (RAW == 2) r[RAW - 1] = left > 4 ? load_raw<DT>(at + 16, left - 4) : u32x4{0, 0, 0, 0};
    };
    auto split = [&](const u32x4* r, u32x4* l) {
        if (DT == BS_DT_F32) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                uint32_t t[3];
                limbs2(bits_f32(r[(n / 2) % RAW][2 * (n & 1)]), bits_f32(r[(n / 2) % RAW][2 * (n & 1) + 1]), t);
#pragma unroll
                for (int b = 0; b < L; ++b) l[b][n] = t[b];
            }
        } else {
            l[0] = r[0];
        }
    };
    auto fetch_turned = [&](int k, u32x4* r) {                     // the same of a column of w [K, N]: neighbouring lanes, neighbouring values
        uint32_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const char* const at = wp + (int64_t)min(k + e, a.K - 1) * a.ldw * ES;
            u[e] = DT == BS_DT_F32 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at);
            if (k + e >= a.K) u[e] = 0;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (DT == BS_DT_F32) {
                r[0][e] = u[e];
                r[RAW - 1][e] = u[4 + e];
            } else {
                r[0][e] = u[2 * e] | u[2 * e + 1] << 16;
            }
        }
    };
    u32x4 xr[NS][RAW], wr[NS][RAW];
    auto ask = [&](int k0) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const int k = k0 + wave * RUN + 8 * (lane >> 5) + n * 16;
            fetch(xp, k, xr[n]);
            if (WT) fetch_turned(k, wr[n]);
            else fetch(wp, k, wr[n]);
        }
    };
    ask(0);
    for (int k0 = 0; k0 < a.K; k0 += 4 * RUN) {
        u32x4 fp[NS][1][L], fq[NS][1][L];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            split(wr[n], fp[n][0]);
            split(xr[n], fq[n][0]);
        }
        if (k0 + 4 * RUN < a.K) ask(k0 + 4 * RUN);                  // on its way while the others take their turns
        for (int turn = 0; turn < 4; ++turn) {
            if (turn == wave && k0 + wave * RUN < a.K) {
                f32x16 one[1][1];
                if (k0 + turn > 0) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const f32x4 t = *reinterpret_cast<const f32x4*>(lds + (e * 64 + lane * 4) * 4);
                        acc[e] = t[0]; acc[e + 1] = t[1]; acc[e + 2] = t[2]; acc[e + 3] = t[3];
                    }
                }
                one[0][0] = acc;
#pragma unroll
                for (int n = 0; n < NS; ++n) multiply<DT, L, L, 1, 1>(fp[n], fq[n], one);
                acc = one[0][0];
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<f32x4*>(lds + (e * 64 + lane * 4) * 4) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
            }
            __syncthreads();
        }
    }
    // the sums lie in shared memory as the last wavefront left them; every wavefront finishes 8 of the 32 rows
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(lds + (e * 64 + lane * 4) * 4);
        acc[e] = t[0]; acc[e + 1] = t[1]; acc[e + 2] = t[2]; acc[e + 3] = t[3];
    }
    __syncthreads();
    float* const turn = reinterpret_cast<float*>(lds);
    if (wave == 0) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(turn + (lane & 31) * 68 + 8 * g + 4 * (lane >> 5)) = f32x4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    }
    __syncthreads();
    constexpr int V = vlen(DT), LPR = 32 / V;
    for (int r = threadIdx.x / LPR; r < 32; r += 256 / LPR) {
        const int c = (threadIdx.x % LPR) * V, left = a.N - p0 - c;
        if (q0 + r >= a.rows || left <= 0) break;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = turn[r * 68 + c + e];
        const int n = left < V ? left : V;
        float bias[V];
        if (EPI == E_LAYER) load_bias<DT>(a, p0 + c, bias);
        finish<DT, EPI>(a, q0 + r, p0 + c, n, v, bias, EPI == E_LAYER && a.res ? residual<DT>(a, q0 + r, p0 + c, n) : u32x4{0, 0, 0, 0});
    }
}

// ---- w laid out for the kernels above -------------------------------------------------------------------------------------------
// out [kp / KB][limb][P][KB] 16-bit: a DMA of neighbouring rows reads whole kilobytes.  w [P, K], or with TURNED w [K, P] turned round;
// zero from K to kp.  16-bit w whose rows are whole aligned multiples of 64 k is read as it lies instead (8192 x 512 x 512 bfloat16
// 11.0 us, laid out first 13.5).  Once per call, not kept from call to call: a caller that trains changes w.  256 x 256 float32 2.7 us,
// 1024 x 512 bfloat16 turned 4.8 us, the better part of each the launch.
struct LayJob {
    const char* w;
    int64_t ldw;
    int P, K;
    char* out;
    int across, blocks;                // blocks along k, all of them
    int chunks;                        // by chunks
};
template <int DT, bool TURNED>
__device__ __forceinline__ void lay_tile(const LayJob& j, int bx, int by) {
    constexpr int ES = esize(DT), L = limbs_of(DT), KB = kb_of(DT);
    const char* const w = j.w;
    const int64_t ldw = j.ldw;
    const int P = j.P, K = j.K;
    char* const out = j.out;
    __shared__ uint32_t tile[32][33];
    const int p0 = by * 32, k0 = bx * 32;                                // 32 p x 32 k
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    uint32_t v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {                                        // (all loads at once: outside, any element, then zero)
        const int r = ty + 8 * n, p = p0 + (TURNED ? tx : r), k = k0 + (TURNED ? r : tx);
        const int pc = min(p, P - 1), kc = min(k, K - 1);
        const char* const src = w + (TURNED ? (int64_t)kc * ldw + pc : (int64_t)pc * ldw + kc) * ES;
        v[n] = DT == BS_DT_F32 ? *reinterpret_cast<const uint32_t*>(src) : *reinterpret_cast<const uint16_t*>(src);
        if (k >= K) v[n] = 0;
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) tile[TURNED ? tx : ty + 8 * n][TURNED ? ty + 8 * n : tx] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 2; ++n) {                                        // two k a thread: words of a row side by side
        const int u = threadIdx.x + n * 256, r = u >> 4, k2 = (u & 15) * 2, p = p0 + r, k = k0 + k2;
        if (p >= P) continue;
        uint32_t l[3];
        if (DT == BS_DT_F32) limbs2(bits_f32(tile[r][k2]), bits_f32(tile[r][k2 + 1]), l);
        else l[0] = tile[r][k2] | (tile[r][k2 + 1] << 16);
#pragma unroll
        for (int b = 0; b < L; ++b) *reinterpret_cast<uint32_t*>(out + ((((int64_t)k / KB * L + b) * P + p) * KB + k % KB) * 2) = l[b];
    }
}

// the same for 16-bit w [P, K] in whole aligned chunks: nothing to turn, a thread moves one chunk of 8 k (2048 x 2048: 6 us, by single
// elements 9)
__device__ __forceinline__ void lay_chunks(const LayJob& j, int bx, int by) {
    constexpr int KB = kb_of(BS_DT_BF16);
    const int p = by * 32 + (threadIdx.x >> 3), k = bx * 64 + (threadIdx.x & 7) * 8;
    if (p >= j.P) return;
    *reinterpret_cast<u32x4*>(j.out + (((int64_t)k / KB * j.P + p) * KB + k % KB) * 2) = k < j.K ? load16(j.w + (p * j.ldw + k) * 2) : u32x4{0, 0, 0, 0};
}

// rows of K elements of ES bytes (1, 2, 4) -> rows of whole 16-byte chunks, zero behind K.  2^lanes_log2 threads a row (a power of two:
// no division); the last chunk of a row comes as its last 16 bytes, moved down.  A copy: 7919 x 252 bfloat16 3 us, 20567 x 963 float32
// 24 us (6.6 TB/s).  The products that went without it, by single elements through registers into shared memory, took 17 us for
// 7919 x 252 x 505 in bfloat16 and 28 for its dw; copied first 16 and 25, and one kernel less of each kind.
struct PadJob {
    const char* in;
    int64_t ld, rows;
    int K;
    char* out;
    int chunks, lanes_log2;
    int64_t blocks;
};
template <int ES>
__device__ __forceinline__ void pad_rows(const PadJob& j, int64_t block) {
    constexpr int V = 16 / ES;
    const char* const in = j.in;
    const int64_t ld = j.ld, rows = j.rows;
    const int K = j.K, chunks = j.chunks, lanes_log2 = j.lanes_log2;
    char* const out = j.out;
    const int64_t row = block * (256 >> lanes_log2) + (threadIdx.x >> lanes_log2);
    if (row >= rows) return;
    for (int c = threadIdx.x & ((1 << lanes_log2) - 1); c < chunks; c += 1 << lanes_log2) {
        const int left = K - c * V;
        const char* const src = in + (row * ld + (int64_t)c * V) * ES;
        u32x4 v;
        if (left >= V) {
            v = load16(src);
        } else if (c > 0) {
            const int down = (V - left) * ES;                            // bytes of the chunk before
            const u32x4 t = load16(src - down);
            const uint64_t lo = t[0] | (uint64_t)t[1] << 32, hi = t[2] | (uint64_t)t[3] << 32;
            const int bits = down * 8;                                   // 8 .. 120
            const uint64_t l = bits < 64 ? (lo >> bits) | (hi << (64 - bits)) : bits == 64 ? hi : hi >> (bits - 64);
            const uint64_t h = bits < 64 ? hi >> bits : 0;
            v = u32x4{(uint32_t)l, (uint32_t)(l >> 32), (uint32_t)h, (uint32_t)(h >> 32)};
        } else {
            uint8_t u[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) u[e] = *reinterpret_cast<const uint8_t*>(src + min(e, left * ES - 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) v[e] |= 4 * e + b < left * ES ? (uint32_t)u[4 * e + b] << (8 * b) : 0u;
            }
        }
        *reinterpret_cast<u32x4*>(out + (row * chunks + c) * 16) = v;
    }
}

// What a product over rows needs first, one launch: w laid out, x in whole rows (either may have no blocks).  bfloat16 7919 x 252 and
// 505 x 252 4.8 us; in two launches 4.5 + 2.9, the whole call 18.5 us instead of 15.5.
template <int DT, bool TURNED>
__global__ __launch_bounds__(256) void k_prepare(const LayJob l, const PadJob x) {
    const int b = blockIdx.x;
    if (b >= l.blocks) pad_rows<esize(DT)>(x, b - l.blocks);
    else if (l.chunks) lay_chunks(l, b % l.across, b / l.across);
    else lay_tile<DT, TURNED>(l, b % l.across, b / l.across);
}

// ---- dw -------------------------------------------------------------------------------------------------------------------------
struct OverArgs {
    const char *x, *ds;                // as the caller holds them
    const char *xd, *dd;               // as DMA takes them
    const int8_t* exps;
    int64_t ldx, ldds, ldxd, lddd, rows, part;
    int K, N, nb, parts;
    int64_t pstride;                   // floats of a part: N K, rounded up to whole 16 bytes
    int tp;
    int64_t tiles;                     // tiles x parts
    char* out;
};
// sums over rows kb..ke that did not come out finite once more, in float32 arithmetic
template <int DT, bool P8>
__device__ __forceinline__ void again_over(const OverArgs& a, int64_t kb, int64_t ke, int p, int q, int n, f32x4& v) {
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= (f32_bits(v[e]) & 0x7f800000u) == 0x7f800000u;
    if (!odd) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if ((f32_bits(v[e]) & 0x7f800000u) == 0x7f800000u && e < n) {
            float s = 0.0f;
            for (int64_t k = kb; k < ke; ++k) {
                const float xv = P8 ? p8_value((int)(int8_t)a.x[k * a.ldx + p + e], p8_pow2(a.exps[k * a.nb + (p + e) / P8_BLOCK]))
                                    : load1<DT>(a.x + (k * a.ldx + p + e) * esize(DT));
                s = fmaf(xv, load1<DT>(a.ds + (k * a.ldds + q) * esize(DT)), s);
            }
            v[e] = s;
        }
}

// x and ds by DMA through a ring, as in k_rows_dma, every tile as it lies in memory: [BK rows][channels].  The transposition that the
// matrix instruction wants (8 rows of one channel side by side) happens in the read from shared memory: transposing reads for 16-bit
// values (4 rows) and for codes (8 rows, turned into bfloat16 / float16 in registers: exact), dword reads along the channels and a
// split into limbs for float32.  steps: 2^e of the codes, laid out [blocks of 32 channels][rows] beforehand (k_prepare_over).
// A part's sums go to the workspace in float32 and are joined in order (k_add_parts); a single part is rounded here.
//
// Measured: bfloat16 x as codes, 65536 x 512 x 1024 100 us (687 TFLOP/s; as bfloat16 85: the codes' conversion, 16 instructions per 8
// values, goes beside the matrix instructions but not for nothing); float32 25600 x 256 x 256 32 us, 8192 x 1024 x 1024 113 us (six
// products: 912 TFLOP/s), bound by the limb splits, 44 instructions a fragment beside its matrix instructions (reads are dwords: no
// transposing read takes 32 bits).
template <int DT, bool P8, int BQ, int BP, int WQ, int WP, int BK, int NS>
__global__ __launch_bounds__((BQ / WQ) * (BP / WP) * 64) void k_over_dma(const OverArgs a, const float* __restrict__ steps, int64_t ldsteps) {
    constexpr int NW = (BQ / WQ) * (BP / WP), ES = esize(DT), XE = P8 ? 1 : ES;
    constexpr int LX = (DT == BS_DT_F32 && !P8) ? 3 : 1, LD = limbs_of(DT);
    constexpr int XR = BP * XE, DR = BQ * ES;                            // bytes of a row
    constexpr int XB = BK * XR, DB = BK * DR, SB = P8 ? BP / 32 * BK * 4 : 0, STAGE = XB + DB + SB;
    constexpr int XI = XB / 1024 / NW, DI = DB / 1024 / NW, SI = P8 ? 1 : 0;
    constexpr int NP = WP / 32, NQ = WQ / 32;
    static_assert(XB % (1024 * NW) == 0 && DB % (1024 * NW) == 0 && NS * STAGE <= 160 * 1024 && NW * turn_bytes(64) <= NS * STAGE, "shared memory");
    static_assert(!P8 || (SB % 256 == 0 && SB / 256 <= NW), "steps: one dword a lane");
    __shared__ __align__(16) char lds[NS * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wp = wave % (BP / WP), wq = wave / (BP / WP);
    // chunk c of row r lies in slot c ^ sx(r): rows that one transposing read gathers then lie in different banks
    // (swap: RB bytes a row; 64 channels of 16 bits are 128 bytes, two rows on the 64 banks)
    auto swap = [](int RB, int r) { return ES == 4 ? 8 * ((r >> 3) & 1) : RB >= 256 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); };
    auto sd = [&](int r) { return swap(DR, r); };
    auto sx = [&](int r) { return P8 ? 2 * ((r >> 1) & 3) : swap(XR, r); };
    static_assert(XR >= 128 && DR >= 128 && (ES == 2 || DR >= 256), "a row takes its swaps");
    const int64_t per = (a.tiles + 7) / 8;
    const int64_t t = (blockIdx.x % 8) * per + blockIdx.x / 8;        // an XCD takes runs of tiles over the same rows
    if (t >= a.tiles) return;
    const int64_t tiles = a.tiles / a.parts;
    const int part = (int)(t / tiles), tile = (int)(t % tiles);
    const int p0 = tile % a.tp * BP, q0 = tile / a.tp * BQ;
    const int64_t kb = part * a.part, ke = kb + a.part < a.rows ? kb + a.part : a.rows;
    const int nk = (int)(ke - kb), count = (nk + BK - 1) / BK;
    const char* const xb = a.xd + (kb * a.ldxd + p0) * XE;
    const char* const db = a.dd + (kb * a.lddd + q0) * ES;
    uint32_t xo[XI], dof[DI];
    int xr[XI], dr[DI];
#pragma unroll
    for (int n = 0; n < XI; ++n) {
        constexpr int CH = XR / 16;
        const int u = (wave * XI + n) * 64 + lane, row = u / CH, c = (u % CH) ^ sx(row);
        xr[n] = row;
        xo[n] = (uint32_t)((int64_t)row * a.ldxd * XE + (p0 + c * (16 / XE) < a.K ? c * 16 : 0));        // channels behind the last: not stored
    }
#pragma unroll
    for (int n = 0; n < DI; ++n) {
        constexpr int CH = DR / 16;
        const int u = (wave * DI + n) * 64 + lane, row = u / CH, c = (u % CH) ^ sd(row);
        dr[n] = row;
        dof[n] = (uint32_t)((int64_t)row * a.lddd * ES + (q0 + c * (16 / ES) < a.N ? c * 16 : 0));
    }
    const float* sp = nullptr;
    if constexpr (P8) {
        const int i = wave % (SB / 256) * 64 + lane, blk = i / BK, nb = (a.K + 31) / 32;
        sp = steps + (int64_t)(p0 / 32 + blk < nb ? p0 / 32 + blk : nb - 1) * ldsteps + kb + i % BK;
    }
    auto issue_whole = [&](int s, int slot) {                             // all its rows exist: no branch among the loads
        char* const st = lds + slot * STAGE;
        const char* const xs = xb + (int64_t)s * BK * a.ldxd * XE;
        const char* const ds = db + (int64_t)s * BK * a.lddd * ES;
#pragma unroll
        for (int n = 0; n < XI; ++n) {
            const char* const src = xs + xo[n];
            __builtin_amdgcn_global_load_lds(src, (lds_ptr)(st + (wave * XI + n) * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int n = 0; n < DI; ++n) {
            const char* const src = ds + dof[n];
            __builtin_amdgcn_global_load_lds(src, (lds_ptr)(st + XB + (wave * DI + n) * 1024), 16, 0, 0);
        }
        if constexpr (P8) {              // (wavefronts beyond the first SB / 256 write the same steps once more: every one counts alike)
            const char* const src = (const char*)(sp + s * BK);
            __builtin_amdgcn_global_load_lds(src, (lds_ptr)(st + XB + DB + wave % (SB / 256) * 256), 4, 0, 0);
        }
    };
    auto issue = [&](int s, int slot) {
        if ((s + 1) * BK <= nk) return issue_whole(s, slot);
        char* const st = lds + slot * STAGE;
        const char* const xs = xb + (int64_t)s * BK * a.ldxd * XE;
        const char* const ds = db + (int64_t)s * BK * a.lddd * ES;
        const int left = nk - s * BK;
#pragma unroll
        for (int n = 0; n < XI; ++n) {
            const char* const src = xs + xo[n];
            char* const dst = st + (wave * XI + n) * 1024;
            if (xr[n] < left) __builtin_amdgcn_global_load_lds(src, (lds_ptr)dst, 16, 0, 0);
            else *reinterpret_cast<u32x4*>(dst + lane * 16) = u32x4{0, 0, 0, 0};                 // rows behind the last: zero
        }
#pragma unroll
        for (int n = 0; n < DI; ++n) {
            const char* const src = ds + dof[n];
            char* const dst = st + XB + (wave * DI + n) * 1024;
            if (dr[n] < left) __builtin_amdgcn_global_load_lds(src, (lds_ptr)dst, 16, 0, 0);
            else *reinterpret_cast<u32x4*>(dst + lane * 16) = u32x4{0, 0, 0, 0};
        }
        if constexpr (P8) {
            const char* const src = (const char*)(sp + s * BK);
            __builtin_amdgcn_global_load_lds(src, (lds_ptr)(st + XB + DB + wave % (SB / 256) * 256), 4, 0, 0);
        }
    };
    uint32_t bad = 0;
    // Fragments as they are read: channel c0 + lane % 32, rows r0 + 8 (lane / 32) + 0..7.  16-bit: two transposing reads of 4 rows,
    // codes: one of 8 rows and the rows' steps, float32: 8 dwords.
    struct Raw16 { u32x4 v; };
    struct Raw32 { float f[8]; };
    struct Raw8 { i32x2 w; f32x4 s[2]; };
    typedef typename std::conditional<P8, Raw8, typename std::conditional<DT == BS_DT_F32, Raw32, Raw16>::type>::type RawX;
    typedef typename std::conditional<DT == BS_DT_F32, Raw32, Raw16>::type RawD;
    constexpr int RX = P8 ? 3 : DT == BS_DT_F32 ? 8 : 2, RD = DT == BS_DT_F32 ? 8 : 2;              // reads of a fragment
    auto read_plain = [&](const char* base, int RB, int r0, int c0, auto& r) {
        if constexpr (DT == BS_DT_F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = r0 + 8 * (lane >> 5) + e, ch = c0 + (lane & 31);
                r.f[e] = *reinterpret_cast<const float*>(base + row * RB + ((ch >> 2) ^ swap(RB, row)) * 16 + (ch & 3) * 4);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = r0 + 8 * (lane >> 5) + 4 * h + ((lane & 15) >> 2), ch = c0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(base + row * RB + (((ch >> 3) ^ swap(RB, row)) * 16) + (ch & 4) * 2));
                const u32x2 w2 = __builtin_bit_cast(u32x2, w);
                r.v[2 * h] = w2[0];
                r.v[2 * h + 1] = w2[1];
            }
        }
    };
    auto turn_plain = [&](const auto& r, auto& l) {
        if constexpr (DT == BS_DT_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t t3[3];
                limbs2(r.f[2 * e], r.f[2 * e + 1], t3);
                l[0][e] = t3[0];
                l[1][e] = t3[1];
                l[2][e] = t3[2];
            }
        } else {
            l[0] = r.v;
        }
    };
    auto read = [&](const char* st, int b, RawX (&x)[NP], RawD (&d)[NQ]) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c0 = wp * WP + i * 32;
            if constexpr (P8) {
                const int row = b * 16 + 8 * (lane >> 5) + ((lane & 15) >> 1), ch = c0 + 16 * ((lane >> 4) & 1) + 8 * (lane & 1);
                x[i].w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2)(st + row * XR + (((ch >> 4) ^ sx(row)) * 16) + (ch & 8)));
                const char* const sb = st + XB + DB + (c0 / 32 * BK + b * 16 + 8 * (lane >> 5)) * 4;
                x[i].s[0] = *reinterpret_cast<const f32x4*>(sb);
                x[i].s[1] = *reinterpret_cast<const f32x4*>(sb + 16);
            } else {
                read_plain(st, XR, b * 16, c0, x[i]);
            }
        }
#pragma unroll
        for (int j = 0; j < NQ; ++j) read_plain(st + XB, DR, b * 16, wq * WQ + j * 32, d[j]);
    };
    auto turn = [&](const RawX (&x)[NP], const RawD (&d)[NQ], u32x4 (&fp)[NP][LX], u32x4 (&fq)[NQ][LD]) {
        if constexpr (P8) {
            uint32_t odd = 0;                                            // a byte 0x80 anywhere: a value that was not finite
            float f[NP][8];
#pragma unroll
            for (int i = 0; i < NP; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[i][e] = (float)(int8_t)((uint32_t)x[i].w[e / 4] >> (8 * (e % 4))) * x[i].s[e / 4][e % 4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t y = (uint32_t)x[i].w[e] ^ 0x80808080u;
                    odd |= (y - 0x01010101u) & ~y & 0x80808080u;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) fp[i][0][e] = DT == BS_DT_F16 ? pk_f16(f[i][2 * e], f[i][2 * e + 1]) : pk_bf16(f[i][2 * e], f[i][2 * e + 1]);
            }
            bad = odd;
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) turn_plain(x[i], fp[i]);
        }
#pragma unroll
        for (int j = 0; j < NQ; ++j) turn_plain(d[j], fq[j]);
    };
    // (rare) the codes 0x80 of what was just turned, as NaN
    auto mend = [&](const RawX (&x)[NP], u32x4 (&fp)[NP][LX]) {
        if constexpr (P8) {
            if (__builtin_expect(__any(bad != 0), 0)) {
#pragma unroll
                for (int i = 0; i < NP; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((((uint32_t)x[i].w[e / 4] >> (8 * (e % 4))) & 255u) == 0x80u) fp[i][0][e / 2] |= e & 1 ? 0x7fff0000u : 0x00007fffu;
            }
        }
    };
    f32x16 acc[NP][NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    const int whole = nk / BK;
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (s < count) issue(s, s);
    constexpr int D = XI + DI + SI, SBK = BK / 16;
    if (NS <= whole) __builtin_amdgcn_s_waitcnt(wait_vm((NS - 1) * D));
    else __builtin_amdgcn_s_waitcnt(wait_vm(0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    RawX x0[NP];
    RawD d0[NQ];
    u32x4 fp[NP][LX], fq[NQ][LD];
    read(lds, 0, x0, d0);
    turn(x0, d0, fp, fq);
    mend(x0, fp);
    int slot = 0;
    // one step, as in k_rows_dma
    auto step = [&](int s, auto run) {
        constexpr bool RUN = decltype(run)::value;
        constexpr int M = (LX == 3 ? 6 : LD == 3 ? 3 : 1) * NP * NQ, R = NP * RX + NQ * RD, RM = (R + M - 1) / M > 2 ? (R + M - 1) / M : 2;
        const int next = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
        for (int b = 0; b < SBK; ++b) {
            RawX xn[NP];
            RawD dn[NQ];
            if (b == SBK - 1) {
                if (RUN) __builtin_amdgcn_s_waitcnt(wait_vm((NS - 2) * D));
                else __builtin_amdgcn_s_waitcnt(wait_vm(0));
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (!RUN && s + NS < count) issue(s + NS, slot);
                __builtin_amdgcn_sched_barrier(0);
                read(lds + next * STAGE, 0, xn, dn);               // (behind the last step: not used)
                if (RUN) issue_whole(s + NS, slot);
            } else {
                __builtin_amdgcn_sched_barrier(0);
                read(lds + slot * STAGE, b + 1, xn, dn);
            }
            u32x4 pn[NP][LX], qn[NQ][LD];
            multiply<DT, LX, LD, NP, NQ>(fp, fq, acc);
            turn(xn, dn, pn, qn);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (m * RM < R) __builtin_amdgcn_sched_group_barrier(0x100, RM, 0);
                if (RUN && b == SBK - 1 && m >= M - D) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            mend(xn, pn);
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int l = 0; l < LX; ++l) fp[i][l] = pn[i][l];
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int l = 0; l < LD; ++l) fq[j][l] = qn[j][l];
        }
        slot = next;
    };
    int s = 0;
#pragma unroll SBK == 1 ? 2 : 1
    for (; s + NS < whole; ++s) step(s, std::true_type{});
    for (; s < count; ++s) step(s, std::false_type{});
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(lds + wave * turn_bytes(64));
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int i = 0; i < NP; i += 2) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float* const at = mine + (lane & 31) * 68 + 8 * g + 4 * (lane >> 5);
                *reinterpret_cast<f32x4*>(at) = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                *reinterpret_cast<f32x4*>(at + 32) = f32x4{acc[i + 1][j][4 * g], acc[i + 1][j][4 * g + 1], acc[i + 1][j][4 * g + 2], acc[i + 1][j][4 * g + 3]};
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int p = p0 + wp * WP + i * 32 + lane % 16 * 4, n = a.K - p;
            if (n > 0)
                for (int r = lane / 16; r < 32; r += 4) {
                    const int q = q0 + wq * WQ + j * 32 + r;
                    if (q >= a.N) break;
                    f32x4 v = *reinterpret_cast<const f32x4*>(mine + r * 68 + lane % 16 * 4);
                    if (DT == BS_DT_F32) again_over<DT, P8>(a, kb, ke, p, q, n, v);
                    if (DT != BS_DT_F32 && a.parts == 1) {                       // nothing to be joined with: rounded here
                        char* const o = a.out + ((int64_t)q * a.K + p) * ES;
                        const u32x2 w = DT == BS_DT_F16 ? u32x2{pk_f16(v[0], v[1]), pk_f16(v[2], v[3])} : u32x2{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
                        if (n >= 4) store8(o, w);
                        else
                            for (int e = 0; e < n; ++e) store1<DT>(o + e * ES, v[e]);
                        continue;
                    }
                    float* const o = reinterpret_cast<float*>(a.out) + part * a.pstride + (int64_t)q * a.K + p;
                    if (n >= 4) store16((char*)o, __builtin_bit_cast(u32x4, v));
                    else
                        for (int e = 0; e < n; ++e) o[e] = v[e];
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
}

// exponents [rows, nb] -> 2^e as floats [nb][ld], zero from rows to ld (65536 x 16: 5.3 us; the products would read each a byte at a
// time, a row apart)
struct StepsJob {
    const int8_t* exps;
    int64_t rows;
    int nb;
    float* out;
    int64_t ld, blocks;
};
__device__ __forceinline__ void lay_steps(const StepsJob& j, int64_t block) {
    const int64_t i = block * 256 + threadIdx.x;
    if (i >= j.ld) return;
    for (int b = 0; b < j.nb; ++b) j.out[b * j.ld + i] = i < j.rows ? p8_pow2(j.exps[i * j.nb + b]) : 0.0f;
}
// What a weight gradient needs first, one launch: the steps of codes, x (codes: bytes) and ds in whole rows.
template <int DT, bool P8>
__global__ __launch_bounds__(256) void k_prepare_over(const StepsJob s, const PadJob x, const PadJob ds) {
    const int64_t b = blockIdx.x;
    if (P8 && b < s.blocks) lay_steps(s, b);
    else if (b < s.blocks + x.blocks) pad_rows<P8 ? 1 : esize(DT)>(x, b - s.blocks);
    else pad_rows<esize(DT)>(ds, b - s.blocks - x.blocks);
}

// parts [nparts][n, rounded up to whole 16 bytes] float32 -> their sum in dtype; 16 threads of four neighbours x 16 lanes over the parts,
// always the same order.  64 parts of 256 x 256 4.7 us, 32 of 512 x 1024 11 us (6.1 TB/s, from the caches)
template <int DT>
__global__ __launch_bounds__(256) void k_add_parts(const float* __restrict__ parts, int nparts, int64_t n, char* __restrict__ out) {
    __shared__ __align__(16) f32x4 red[256];
    const int tx = threadIdx.x & 15, l = threadIdx.x >> 4;
    const int64_t i = ((int64_t)blockIdx.x * 16 + tx) * 4;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i < n) {
        const int64_t stride = (n + 3) / 4 * 4;
#pragma unroll 4
        for (int k = l; k < nparts; k += 16) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(parts + k * stride + i);
            s[0] += v[0]; s[1] += v[1]; s[2] += v[2]; s[3] += v[3];
        }
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (l || i >= n) return;
    float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += red[k * 16 + tx][e];
    for (int e = 0; e < 4 && i + e < n; ++e) store1<DT>(out + (i + e) * esize(DT), t[e]);
}

// ---- which way --------------------------------------------------------------------------------------------------------------------
constexpr int MAX_WIDTH = 1 << 20;
int64_t tiles_of(int64_t rows, int N, int bq, int bp) { return (rows + bq - 1) / bq * ((N + bp - 1) / bp); }
// The tile of a product goes by how many tiles of a size there are for 256 compute units, and by K.  Both sides, in us, at
// (rows, K, N):
//   k_relay up to 256 tiles of 32x32 (16-bit) or 512 (float32), as its workgroups, a tile each, then have the chip for themselves:
//     bf16  (256, 256, 256) 4.6, k_rows_dma 5.2   (512, 512, 512) 6.0 and 6.2    beyond: (1024, 256, 512) 5.9 and 5.4
//     f32   (256, 1024, 1024) 18.6 and 27.3       (1024, 256, 512) 9.4 and 12.0  beyond: (2048, 256, 512) 15.9 and 12.6
bool few(int dtype, int64_t rows, int N) { return tiles_of(rows, N, 32, 32) <= (dtype == BS_DT_F32 ? 512 : 256); }
//   128 channels across (16-bit 128x128, float32 64x128) from 256 tiles on, 64x64 below and for N <= 64:
//     bf16  (8192, 512, 512), 256 tiles, 10.9 and 12.6      (2048, 256, 512), 64 tiles, 8.3 and 5.7
//     f32   (4096, 512, 1024), 512 tiles, 38.3 and 40.4     (1024, 512, 512), 64 tiles, 21.7 and 16.0
bool enough(int64_t rows, int N, int bq, int bp) { return tiles_of(rows, N, bq, bp) >= 256; }
//   the largest tile (16-bit 256x256, one workgroup a compute unit; float32 128x128, two) where K is long enough to pay for its
//   start and end, which nothing covers:
//     bf16  (16384, 2048, 2048) 145 and 168                 (102400, 256, 256) 50 and 43
//     f32   (4942, 832, 1168) 72 and 84                     (40000, 256, 256) 54 and 45,  (8192, 256, 512) 25.5 and 22.3
constexpr int DEEP_K = 512;
//   or, float32, where it saves a round: 512 of its tiles are on the chip at once, 768 of 64x128, a round of which costs 3/4 as much
//     (25600, 256, 256), a round of 400 against two of 800, 35 and 41;   (50000, 64, 128), 391, 23 and 25;   (7400, 300, 1000), 464, 48
//     and 44;   (16384, 256, 512), 512, 39 and 39;   no round saved: (40000, 256, 256), 54 and 45
bool fewer_rounds(int64_t rows, int N) { return 4 * ((tiles_of(rows, N, 128, 128) + 511) / 512) < 3 * ((tiles_of(rows, N, 64, 128) + 767) / 768); }
//   and, 16-bit, where its tiles fill four fifths of the rounds that they take:
//     (16384, 1024, 1024), 256 tiles, 46 and 50             (12288, 512, 1024), 192 tiles, 29 and 23
bool fills(int64_t rows, int N) {
    const int64_t tiles = tiles_of(rows, N, 256, 256), rounds = (tiles + 255) / 256;
    return N > 128 && tiles * 5 >= rounds * 256 * 4;
}

int64_t lay_bytes(int dtype, int K, int P) { return ((int64_t)limbs_of(dtype) * P * ((K + 63) / 64 * 64) * 2 + 255) / 256 * 256; }
int64_t pad_bytes(int es, int64_t rows, int K) { return (rows * (((int64_t)K * es + 15) / 16) * 16 + 255) / 256 * 256; }

// rows that DMA can take: aligned chunks, whole or ended with zeros (zeros), tiles within 31 bits of their first byte
bool whole_rows(const void* p, int64_t ld, int K, int es, int zeros) {
    return ((uintptr_t)p & 15) == 0 && ld * es % 16 == 0 && ((int64_t)K * es % 16 == 0 || (zeros && ld * es >= ((int64_t)K * es + 15) / 16 * 16)) &&
           ld * es < (1 << 22);
}
PadJob pad_job(int es, const void* in, int64_t ld, int64_t rows, int K, char* out) {
    PadJob j = {(const char*)in, ld, rows, K, out, (int)(((int64_t)K * es + 15) / 16), 0, 0};
    while ((1 << j.lanes_log2) < j.chunks && j.lanes_log2 < 8) ++j.lanes_log2;
    j.blocks = (rows + (256 >> j.lanes_log2) - 1) / (256 >> j.lanes_log2);
    return j;
}

// out [rows, N] over K; whole: rows of x that DMA can take
int64_t rows_bytes(int dtype, int64_t rows, int K, int N, bool whole) {
    return few(dtype, rows, N) ? 0 : lay_bytes(dtype, K, N) + (whole ? 0 : pad_bytes(esize(dtype), rows, K));
}
template <int DT, int EPI>
int launch_rows(RowsArgs a, int zeros, void* workspace, int64_t bytes, hipStream_t st) {
    constexpr int ES = esize(DT), CK = 16 / ES;
    const int kp = (a.K + 63) / 64 * 64;
    const bool small = few(DT, a.rows, a.N), whole = whole_rows(a.x, a.ldx, a.K, ES, zeros);
    const bool big = DT != BS_DT_F32 && a.K >= DEEP_K && fills(a.rows, a.N);
    const bool as_is = DT != BS_DT_F32 && !a.wt && a.K % 64 == 0 && a.ldw % 8 == 0 && ((uintptr_t)a.w & 15) == 0 && a.ldw < (1 << 21);
    const int64_t need = rows_bytes(DT, a.rows, a.K, a.N, whole);
    if (bad_workspace(workspace, bytes, need)) return BS_EINVAL;
    if (a.K > MAX_WIDTH || a.N > MAX_WIDTH) return BS_EINVAL;          // 31-bit offsets into a tile's rows, and the grids below
    if (small) {
        a.tp = (a.N + 31) / 32;
        const unsigned blocks = (unsigned)((a.rows + 31) / 32 * a.tp);
        hipLaunchKernelGGL((k_relay<DT, EPI, EPI == E_PLAIN>), dim3(blocks), dim3(256), 0, st, a);      // (E_PLAIN: dx, w [K, N])
        return rows_rc();
    }
    LayJob l = {};
    PadJob x = {};
    a.Kx = (a.K + CK - 1) / CK * CK;
    a.xd = a.x; a.ldxd = a.ldx;
    if (as_is) {
        a.wl = a.w; a.sp = a.ldw; a.sl = 0; a.sk = kb_of(DT);
    } else {
        constexpr int KB = kb_of(DT);
        l = {a.w, a.ldw, a.N, a.K, (char*)workspace, kp / 32, 0, DT != BS_DT_F32 && !a.wt && a.K % 8 == 0 && a.ldw % 8 == 0 && ((uintptr_t)a.w & 15) == 0};
        if (l.chunks) l.across = kp / 64;
        l.blocks = l.across * ((a.N + 31) / 32);
        a.wl = (const char*)workspace; a.sp = KB; a.sl = (int64_t)a.N * KB; a.sk = a.sl * limbs_of(DT);
    }
    if (!whole) {
        x = pad_job(ES, a.x, a.ldx, a.rows, a.K, (char*)workspace + lay_bytes(DT, a.K, a.N));
        a.xd = x.out; a.ldxd = a.Kx;
    }
    if (too_many(l.blocks + x.blocks, 256)) return BS_EINVAL;
    auto prepare = [&] {
        if (l.blocks + x.blocks > 0)
            hipLaunchKernelGGL((k_prepare<DT, EPI == E_PLAIN>), dim3((unsigned)(l.blocks + x.blocks)), dim3(256), 0, st, l, x);
    };
#define ROWS(BQ, BP, WQ, WP, BK, NS, PS) do { a.tp = (a.N + BP - 1) / BP; a.tiles = tiles_of(a.rows, a.N, BQ, BP); \
        const int64_t blocks = (a.tiles + 7) / 8 * 8; if (too_many(blocks, (BQ / WQ) * (BP / WP) * 64)) return BS_EINVAL; \
        prepare(); \
        hipLaunchKernelGGL((k_rows_dma<DT, EPI, BQ, BP, WQ, WP, BK, NS, PS>), dim3((unsigned)blocks), dim3((BQ / WQ) * (BP / WP) * 64), 0, st, a); } while (0)
    if constexpr (DT == BS_DT_F32) {
        if (a.N > 64 && enough(a.rows, a.N, 128, 128) && (a.K >= DEEP_K || fewer_rounds(a.rows, a.N))) ROWS(128, 128, 32, 128, 16, 3, 2);
        else if (a.N > 64 && enough(a.rows, a.N, 64, 128)) ROWS(64, 128, 32, 64, 16, 3, 3);
        else ROWS(64, 64, 32, 32, 32, 4, 1);
    } else {
        if (big) ROWS(256, 256, 128, 64, 32, 4, 1);
        else if (a.N > 64 && enough(a.rows, a.N, 128, 128)) ROWS(128, 128, 32, 64, 32, 3, 4);
        else ROWS(64, 64, 32, 32, 32, 4, 1);
    }
#undef ROWS
    return rows_rc();
}

// How a weight gradient is cut: tiles of 256 x 128 (16-bit) or 128 x 128 (float32) outputs where these and parts of 256 rows come to
// two workgroups a compute unit, else of 64 x 128; the rows into as many parts as give a compute unit two, or one where tiles are small
// and 16-bit (what more parts win the join of them costs again), none under 128 rows.  Both sides, in us, at (rows, K, N):
//   large tiles   bf16 from codes (65536, 512, 1024) 102 and 179    f32 (8192, 1024, 1024) 113 and 124
//                 below: bf16 (8192, 512, 512) 30 and 22            f32 (2048, 256, 256) 16.5 and 12.8
//   parts, large  two a compute unit 102, one 126, four 126 (bf16 from codes (65536, 512, 1024))
//   parts, small  one a compute unit 12.7, two 17.2 (bf16 (8192, 256, 256)); 40 and 37 (f32 (25600, 256, 256), both launches); parts
//                 under 512 rows 12.7, none 22.2 (f32 (2048, 256, 256))
int over_bq(int dtype, int64_t rows, int K, int N) {
    const int big = dtype == BS_DT_F32 ? 128 : 256;
    return 2 * N > big && tiles_of(N, K, big, 128) * ((rows + 255) / 256) >= 512 ? big : 64;
}
void split_rows(int dtype, int64_t rows, int K, int N, int64_t* part, int64_t* parts) {
    const int bq = over_bq(dtype, rows, K, N);
    const int64_t tiles = tiles_of(N, K, bq, 128), groups = bq == 64 && dtype != BS_DT_F32 ? 256 : 512;
    int64_t want = (groups + tiles - 1) / tiles;
    const int64_t most = rows <= 256 ? 1 : (rows + 127) / 128;      // (so few: the launch that joins two parts costs more)
    if (want > most) want = most;
    if (want < 1) want = 1;
    *part = ((rows + want - 1) / want + 63) / 64 * 64;
    if (*part < 64) *part = 64;                               // no rows
    *parts = rows ? (rows + *part - 1) / *part : 1;
}
int64_t steps_bytes(int64_t rows, int K) { return (int64_t)((K + 31) / 32) * ((rows + 63) / 64 * 64) * 4; }
struct OverBytes {
    int64_t steps, x, ds, parts;
    int64_t all() const { return steps + x + ds + parts; }
};
OverBytes over_bytes(int dtype, int64_t rows, int K, int N, bool codes, bool x_whole, bool ds_whole) {
    int64_t part, parts;
    split_rows(dtype, rows, K, N, &part, &parts);
    return {codes ? steps_bytes(rows, K) : 0, x_whole ? 0 : pad_bytes(codes ? 1 : esize(dtype), rows, K), ds_whole ? 0 : pad_bytes(esize(dtype), rows, N),
            parts > 1 ? parts * (((int64_t)K * N + 3) / 4 * 4) * 4 : 0};
}

template <int DT>
int launch_over(OverArgs a, const float* steps, int64_t ld, hipStream_t st) {
#define OVER(P8, BQ, WQ, BK_, NS) do { a.tp = (a.K + 127) / 128; a.tiles = tiles_of(a.N, a.K, BQ, 128) * a.parts; \
        const int64_t blocks = (a.tiles + 7) / 8 * 8; \
        hipLaunchKernelGGL((k_over_dma<DT, P8, BQ, 128, WQ, 64, BK_, NS>), dim3((unsigned)blocks), dim3(256), 0, st, a, steps, ld); } while (0)
    if (a.exps) {
        if constexpr (DT == BS_DT_F32) {
            if (over_bq(DT, a.rows, a.K, a.N) == 128) OVER(true, 128, 64, 32, 3);
            else OVER(true, 64, 32, 32, 3);
        } else if (over_bq(DT, a.rows, a.K, a.N) == 256) OVER(true, 256, 128, 32, 3);
        else OVER(true, 64, 32, 32, 4);
    } else {
        if constexpr (DT == BS_DT_F32) {
            if (over_bq(DT, a.rows, a.K, a.N) == 128) OVER(false, 128, 64, 16, 3);
            else OVER(false, 64, 32, 16, 3);
        } else if (over_bq(DT, a.rows, a.K, a.N) == 256) OVER(false, 256, 128, 32, 3);
        else OVER(false, 64, 32, 32, 4);
    }
#undef OVER
    return rows_rc();
}

}  // namespace

extern "C" {

int64_t bs_linear_workspace(int dtype, int64_t rows, int K, int N, int whole) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1 || K > MAX_WIDTH || N > MAX_WIDTH) return BS_EINVAL;
    return rows_bytes(dtype, rows, K, N, whole != 0);
}

int bs_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, const void* res,
                  int64_t ldr, void* sum_out, void* act_out, int act, int dtype, int64_t rows, int K, int N, void* workspace,
                  int64_t workspace_bytes, void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1 || act < BS_ACT_NONE || act > BS_ACT_GELU) return BS_EINVAL;
    if (rows == 0) return BS_OK;
    if (!x || !w || ldx < K || ldw < K || (res && ldr < N) || (!sum_out && !act_out)) return BS_EINVAL;
    if (bias && bias_dtype != BS_DT_F32 && bias_dtype != dtype) return BS_EINVAL;
    RowsArgs a = {};
    a.x = (const char*)x; a.ldx = ldx; a.w = (const char*)w; a.ldw = ldw; a.rows = rows; a.K = K; a.N = N;
    a.bias = (const char*)bias; a.bias_f32 = bias_dtype == BS_DT_F32;
    a.res = (const char*)res; a.ldr = ldr;
    a.sum = (char*)sum_out; a.act_out = (char*)act_out; a.act = act;
    hipStream_t st = rows_stream(stream);
    if (dtype == BS_DT_F32) return launch_rows<BS_DT_F32, E_LAYER>(a, 0, workspace, workspace_bytes, st);
    if (dtype == BS_DT_BF16) return launch_rows<BS_DT_BF16, E_LAYER>(a, 0, workspace, workspace_bytes, st);
    return launch_rows<BS_DT_F16, E_LAYER>(a, 0, workspace, workspace_bytes, st);
}

int64_t bs_linear_grad_x_workspace(int dtype, int64_t rows, int K, int N, int whole) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1 || K > MAX_WIDTH || N > MAX_WIDTH) return BS_EINVAL;
    return rows_bytes(dtype, rows, N, K, whole != 0);
}

int bs_linear_grad_x(const void* ds, int64_t ldds, int zeros, const void* w, int64_t ldw, void* dx, int dtype, int64_t rows, int K, int N,
                     void* workspace, int64_t workspace_bytes, void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1) return BS_EINVAL;
    if (rows == 0) return BS_OK;
    if (!ds || !w || !dx || ldds < N || ldw < K) return BS_EINVAL;
    RowsArgs a = {};
    a.x = (const char*)ds; a.ldx = ldds; a.w = (const char*)w; a.ldw = ldw; a.rows = rows; a.K = N; a.N = K; a.wt = 1;
    a.sum = (char*)dx;
    hipStream_t st = rows_stream(stream);
    if (dtype == BS_DT_F32) return launch_rows<BS_DT_F32, E_PLAIN>(a, zeros, workspace, workspace_bytes, st);
    if (dtype == BS_DT_BF16) return launch_rows<BS_DT_BF16, E_PLAIN>(a, zeros, workspace, workspace_bytes, st);
    return launch_rows<BS_DT_F16, E_PLAIN>(a, zeros, workspace, workspace_bytes, st);
}

int64_t bs_linear_grad_w_workspace(int dtype, int64_t rows, int K, int N, int codes, int x_whole, int ds_whole) {
    if (bad_type(dtype) || rows < 0 || rows > MAX_ROWS || K < 1 || N < 1 || K > MAX_WIDTH || N > MAX_WIDTH) return BS_EINVAL;
    return over_bytes(dtype, rows, K, N, codes != 0, x_whole != 0, ds_whole != 0).all();
}

int bs_linear_grad_w(const void* ds, int64_t ldds, int zeros, const void* x, const int8_t* x_exps, int64_t ldx, void* dw, int dtype,
                     int64_t rows, int K, int N, void* workspace, int64_t workspace_bytes, void* stream) {
    if (bad_type(dtype) || rows < 0 || rows > (1 << 30) || K < 1 || N < 1 || K > MAX_WIDTH || N > MAX_WIDTH || !dw) return BS_EINVAL;
    if (rows > 0 && (!ds || !x || ldds < N || ldx < K)) return BS_EINVAL;
    hipStream_t st = rows_stream(stream);
    const int64_t n = (int64_t)K * N;
    const int es = esize(dtype), xe = x_exps ? 1 : es;
    const bool x_whole = whole_rows(x, ldx, K, xe, 0), ds_whole = whole_rows(ds, ldds, N, es, zeros);
    const OverBytes b = over_bytes(dtype, rows, K, N, x_exps != nullptr, x_whole, ds_whole);
    int64_t part, parts;
    split_rows(dtype, rows, K, N, &part, &parts);
    if (rows > 0 && bad_workspace(workspace, workspace_bytes, b.all())) return BS_EINVAL;
    char* const ws = (char*)workspace;                       // steps of the codes | copy of x | copy of ds | parts
    const bool joined = parts > 1;
    if (rows > 0) {
        OverArgs a = {};
        a.x = (const char*)x; a.exps = x_exps; a.ldx = ldx; a.ds = (const char*)ds; a.ldds = ldds; a.rows = rows; a.part = part;
        a.K = K; a.N = N; a.nb = (K + P8_BLOCK - 1) / P8_BLOCK; a.parts = (int)parts;
        a.xd = a.x; a.ldxd = ldx; a.dd = a.ds; a.lddd = ldds; a.pstride = (n + 3) / 4 * 4;
        a.out = joined ? ws + b.steps + b.x + b.ds : (char*)dw;
        const int64_t ld = (rows + 63) / 64 * 64;
        StepsJob sj = {};
        PadJob xj = {}, dj = {};
        if (x_exps) sj = {x_exps, rows, a.nb, (float*)ws, ld, (ld + 255) / 256};
        if (!x_whole) {
            xj = pad_job(xe, x, ldx, rows, K, ws + b.steps);
            a.xd = xj.out; a.ldxd = (K + 16 / xe - 1) / (16 / xe) * (16 / xe);
        }
        if (!ds_whole) {
            dj = pad_job(es, ds, ldds, rows, N, ws + b.steps + b.x);
            a.dd = dj.out; a.lddd = (N + 16 / es - 1) / (16 / es) * (16 / es);
        }
        const int64_t first = sj.blocks + xj.blocks + dj.blocks;
        if (too_many(first, 256) || too_many(tiles_of(N, K, over_bq(dtype, rows, K, N), 128) * parts + 7, 256)) return BS_EINVAL;
        if (first > 0) {
#define PREPARE(DT) do { if (x_exps) hipLaunchKernelGGL((k_prepare_over<DT, true>), dim3((unsigned)first), dim3(256), 0, st, sj, xj, dj); \
                         else hipLaunchKernelGGL((k_prepare_over<DT, false>), dim3((unsigned)first), dim3(256), 0, st, sj, xj, dj); } while (0)
            if (dtype == BS_DT_F32) PREPARE(BS_DT_F32);
            else if (dtype == BS_DT_BF16) PREPARE(BS_DT_BF16);
            else PREPARE(BS_DT_F16);
#undef PREPARE
        }
        const int rc = dtype == BS_DT_F32 ? launch_over<BS_DT_F32>(a, (float*)ws, ld, st) : dtype == BS_DT_BF16 ? launch_over<BS_DT_BF16>(a, (float*)ws, ld, st)
                                                                                              : launch_over<BS_DT_F16>(a, (float*)ws, ld, st);
        if (rc != BS_OK || !joined) return rc;
    } else {
        parts = 0;                                            // the sum of no parts
    }
    const float* const from = (const float*)(ws + b.steps + b.x + b.ds);
    constexpr int64_t once = (int64_t)1 << 29;               // values of a launch (only a sum of no parts has more)
    for (int64_t at = 0; at < n; at += once) {
        const int64_t count = n - at < once ? n - at : once;
        const dim3 blocks((unsigned)((count + 63) / 64));
        char* const to = (char*)dw + at * es;
        if (dtype == BS_DT_F32) hipLaunchKernelGGL(k_add_parts<BS_DT_F32>, blocks, dim3(256), 0, st, from, (int)parts, count, to);
        else if (dtype == BS_DT_BF16) hipLaunchKernelGGL(k_add_parts<BS_DT_BF16>, blocks, dim3(256), 0, st, from, (int)parts, count, to);
        else hipLaunchKernelGGL(k_add_parts<BS_DT_F16>, blocks, dim3(256), 0, st, from, (int)parts, count, to);
    }
    return rows_rc();
}

}  // extern "C"
