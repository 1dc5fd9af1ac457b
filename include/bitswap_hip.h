/*
 * bitswap_hip.h -- C ABI of libbitswap_hip.so, the MI355X (gfx950) implementation of the
 * Bit-Swap / BB-ANS entropy-coding hot path.
 *
 * The reference (fhkingma/bitswap) has no FFI layer: its hot path is the Python class
 * `ANS` (mnist_compress.py:13-68, copied verbatim into the five other CLI scripts) plus
 * `logistic_cdf` (utils/torch/rand.py:67-68) and the three-line pmf assembly repeated at
 * every call site (mnist_compress.py:183-185).  Each entry point below names the reference
 * lines it replaces.  INTEGRATION.md shows the ctypes stub a maintainer of the reference
 * would add.
 *
 * Conventions
 *   - every pointer is a DEVICE pointer unless marked host; the caller allocates everything;
 *     the library keeps no global state and may be called from several host threads on
 *     different streams.
 *   - `stream` is a hipStream_t passed as void* (NULL = the null stream); every call only
 *     enqueues work, nothing synchronises.
 *   - return value: BS_OK or a negative BS_E* code for errors detectable on the host at
 *     enqueue time.  Errors that only the device can see (stack underflow ...) are written
 *     to the per-chain `status` array and are sticky: a chain whose status is non-zero is
 *     skipped by every later call until the caller clears it.
 *   - B = number of independent chains (rANS states), D = symbols per chain and call
 *     (latent or pixel dimensions), K = alphabet size (2^quantbits), bits = ANS precision
 *     (the reference hard-codes 31, mnist_compress.py:76).
 *   - a chain's state is {head[b] : uint64 in [2^32, 2^64), stack[b*cap .. b*cap+len[b]) :
 *     uint32 words}; this is the reference's Python list `state` with head = state[-1]
 *     (mnist_compress.py:158-159).
 *   - integer tables: cdf rows hold c_0 = 0 <= c_1 <= ... <= c_K = 2^bits with row stride
 *     `ld` >= K+1 (uint32 units); f_j = c_{j+1} - c_j.  ld == K+1 is the reference layout
 *     (ANS.cdfs, mnist_compress.py:39-40); ld % 4 == 0 (e.g. K+4) selects 16-byte stores.
 */
#ifndef BITSWAP_HIP_H
#define BITSWAP_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* 2: layout argument, BS_LAYOUT_WAVE pivot words, conv-stack epilogue entry points
 * 3: bin_step (CDF spec 2) and status arguments of bs_logistic_tables / bs_logistic_fc; bs_layer_pop64 / _push64
 * 4: BS_LAYOUT_PIVOT and bs_rans_pop_pivot (64 cumulative values per row instead of the whole row)
 * 6: explicit cdf_spec argument (after bin_step) of bs_logistic_tables / _fc, bs_rans_pop_pivot, bs_layer_pop64 / _push64;
 *    CDF spec 3
 * 7: CDF spec 4 accepted wherever a cdf_spec is taken; BS_POP_PIVOT_MAX_D (the pivot pop's documented D limit is what its LDS
 *    allows); bs_wino_gemm_bf16x3 launches its wave-specialised shape by default (same products, same bits)
 * A version changes when what was there changes.  Entry points that are only added (the channels-last layer operators below) leave
 * it as it is: a caller that needs them looks their names up. */
#define BS_ABI_VERSION 7
/* highest version of the deterministic logistic-CDF specification this library implements;
 * a stream written with one CDF spec can only be decoded with the same one.
 *   spec 1: one float64 sigmoid per bin endpoint; any bins.
 *   spec 2: rows of UNIFORM-width bins (bin_step required, K >= 256): one exponential per group of K/64 bins
 *           and a geometric factor per bin; same endpoints, agrees with spec 1 to a few ulp of the cdf.  Defined for
 *           rows with (K/64) * bin_step / scale < 650 (the geometric factors must stay clear of the exponential's clamp:
 *           scale > 5e-5 for the pixel bins, 20x under the reference's floor); a row outside flags BS_ST_BADTABLE.
 *   spec 3: spec 2's denominators 1 + E, inverted per block of min(K/64, 16) bins through a balanced product tree with ONE
 *           correctly rounded reciprocal (54 instead of 144 issue slots per 16 bins); rows with (K/64) * bin_step / scale
 *           >= 8 (peaked pixel rows) are spec 2's bit for bit.  Same domain as spec 2; the default of the codec since round 5.
 *   spec 4: spec 3 with blocks of min(K/64, 8) bins and one residual correction per quotient, c <- fma(fma(-x, c, 1), c, c):
 *           spec 2's accuracy against torch.sigmoid (the correction squares the tree's rounding error away) for 92 instead of
 *           144 issue slots per 16 bins; same domain and the same switch to spec 2's arithmetic for peaked rows as spec 3.
 * Every table-building entry point takes `cdf_spec` (1 .. 4) next to `bin_step`: 1 ignores bin_step; 2, 3 and 4 need it
 * (BS_EINVAL otherwise).  The oracle's C restatements: oracle/bitswap_oracle.c::orc_det_sigmoid / det2_row_cdf / det3_row_cdf /
 * det4_row_cdf. */
#define BS_CDF_SPEC 4

#define BS_OK 0
#define BS_EINVAL (-1)       /* bad argument (null pointer, negative size, ld < K+1 ...)   */
#define BS_EUNSUPPORTED (-2) /* K not supported by the fused logistic kernels              */
#define BS_ELAUNCH (-3)      /* HIP reported a launch error                                */

/* per-chain device status codes */
#define BS_ST_OK 0
#define BS_ST_UNDERFLOW 1 /* pop on an empty stack: "too few initial bits", mnist_compress.py:66,193 */
#define BS_ST_OVERFLOW 2  /* push beyond `cap` words (the reference list is unbounded)               */
#define BS_ST_BADTABLE 3  /* cdf[K] != 2^bits or a zero frequency, the assert at mnist_compress.py:47 */
#define BS_ST_BADSYMBOL 4 /* symbol outside [0, K)                                                    */

#define BS_PARAM_F32 0
#define BS_PARAM_F64 1

/* layout of an integer cdf row
 *   BS_LAYOUT_LINEAR  row[j] = c_j, j = 0..K (the reference's ANS.cdfs row), ld >= K+1
 *   BS_LAYOUT_WAVE    internal hand-off format between bs_logistic_tables and bs_rans_pop /
 *                     bs_rans_push_table (K = 256*n, ld >= K+64, 16-byte aligned rows): the K entries
 *                     c_0..c_{K-1} permuted so that a 64-lane wavefront's 16-byte loads leave entries
 *                     64r..64r+63 in register r across its lanes (entry j at dword ((j/256)*64 + j%64)*4
 *                     + (j/64)%4), followed at [K, K+64) by the pivot words: word r = c_{64r} for
 *                     r < K/64, word K/64 = c_K = 2^bits, the remaining words 0xffffffff.
 *   BS_LAYOUT_PIVOT   internal hand-off format between bs_logistic_tables and bs_rans_pop_pivot for rows of
 *                     uniform-width bins (CDF spec 2 or 3, bin_step != NULL, K = 256*n; ld >= 128 even, 8-byte aligned rows):
 *                     64 pairs of words; pair l = (c_{l K/64}, aux_l) -- the cumulative value at the first bin of group
 *                     l -- with aux_0 = the bin that took the remnant 2^bits - sum f (mnist_compress.py:36) and aux_1 =
 *                     that remnant.  512 bytes per row cross HBM instead of 4 (K + 64): the popping wavefront rebuilds
 *                     the K/64 bins of the one group its symbol falls into from (endpoints, bin_step, mu, scale). */
#define BS_LAYOUT_LINEAR 0
#define BS_LAYOUT_WAVE 1
#define BS_LAYOUT_PIVOT 2

int bs_abi_version(void);
int bs_cdf_spec(void);
const char* bs_strerror(int code);

/*
 * bs_table_rows_f64 -- ANS.__init__ (mnist_compress.py:14-47) for `rows` independent pmf rows.
 *   f_j = trunc(pmf_j * (2^bits - 2^quantbits)) + 1; the first maximal f absorbs
 *   2^bits - sum f; cdf = exclusive prefix sum with cdf[K] = 2^bits.  Bit-exact.
 *   pmf [rows,K] f64; f_out [rows,K] (nullable); cdf_out [rows,ld]; status [rows] (nullable,
 *   BS_ST_BADTABLE when the row violates the reference's asserts).  Any K >= 1.
 */
int bs_table_rows_f64(const double* pmf, int64_t rows, int K, int bits, int quantbits,
                      uint32_t* f_out, uint32_t* cdf_out, int64_t ld, int32_t* status, void* stream);

/*
 * bs_logistic_tables -- logistic_cdf (utils/torch/rand.py:67-68) + pmf assembly
 * (mnist_compress.py:183-185) + ANS.__init__ (:14-47) fused, "decode flavour": writes the full
 * integer cdf row of every (chain, dim) so that bs_rans_pop can search it.
 *   endpoints: row d at endpoints + d*e_stride doubles, K-1 interior bin endpoints, increasing
 *              (zendpoints[zi] has e_stride = K-1; ImageBins / top-layer bins, whose rows are
 *              all equal, may pass e_stride = 0).
 *   mu, scale [B,D] of param_dtype (the reference's Model emits float32 and casts up,
 *              model/mnist_train.py:375-376; both are converted to f64 exactly).
 *   bin_step:  [D] doubles, the bin width h_d = (e[d][K-2] - e[d][0]) / (K-2) of rows whose endpoints are an arithmetic
 *              progression up to rounding (every latent layer but the top one: discretization.py:81-83,105-118);
 *              required by CDF specs 2 and 3 (K >= 256), ignored (may be NULL) by spec 1.
 *   cdf_spec:  1, 2, 3 or 4 (BS_CDF_SPEC above).  The caller decides from the bins alone, so sender and receiver agree.
 *   cdf_out [B,D,ld] in `layout` (BS_LAYOUT_LINEAR, BS_LAYOUT_WAVE or BS_LAYOUT_PIVOT).
 *   status [B] (nullable) receives BS_ST_BADTABLE for a chain with a non-finite mu, a scale that is not a
 *              positive finite number, or a row whose remnant drives a frequency below 1 (mnist_compress.py:46-47).
 * The CDF is evaluated in float64 by the deterministic routine of DESIGN.md (BS_CDF_SPEC);
 * it agrees with torch.sigmoid to a few ulp, everything after it is exact integer work.
 * K must be 64*n, n in {1,2,4,8,16,32}.
 */
int bs_logistic_tables(const double* endpoints, int64_t e_stride, const double* bin_step, int cdf_spec, const void* mu,
                       const void* scale, int param_dtype, int B, int D, int K, int bits, int quantbits,
                       uint32_t* cdf_out, int64_t ld, int layout, int32_t* status, void* stream);

/*
 * bs_logistic_fc -- same fused computation, "encode flavour": given the symbol of every
 * (chain, dim) emit only its frequency f and cumulative start c (what ANS.encode reads at
 * mnist_compress.py:51,55); no table is written.
 *   sym [B,D] int32; f_out, c_out [B,D] uint32; status [B] receives BS_ST_BADSYMBOL / BS_ST_BADTABLE.
 *   bin_step, cdf_spec as in bs_logistic_tables (must be the same choice on both sides of a stream).
 */
int bs_logistic_fc(const double* endpoints, int64_t e_stride, const double* bin_step, int cdf_spec, const void* mu,
                   const void* scale, int param_dtype, const int32_t* sym, int B, int D, int K, int bits,
                   int quantbits, uint32_t* f_out, uint32_t* c_out, int32_t* status, void* stream);

/*
 * bs_rans_push -- ANS.encode (mnist_compress.py:49-56), B chains, symbols i = 0..D-1 in order:
 *   if head >= 2^(64-bits) * f: stack[len++] = low32(head); head >>= 32
 *   head = (head / f) << bits + head % f + c
 *   f, c [B,D] as produced by bs_logistic_fc.
 */
int bs_rans_push(uint64_t* head, uint32_t* stack, int32_t* len, int64_t cap,
                 const uint32_t* f, const uint32_t* c, int B, int D, int bits,
                 int32_t* status, void* stream);

/*
 * bs_rans_push_table -- ANS.encode reading (f, c) from integer cdf rows: row of (b, d) at
 * cdf + b*chain_stride + d*ld (chain_stride = 0 shares one table between all chains, used for
 * the image-independent prior, mnist_compress.py:246-251).  sym [B,D].
 */
int bs_rans_push_table(uint64_t* head, uint32_t* stack, int32_t* len, int64_t cap,
                       const uint32_t* cdf, int64_t chain_stride, int64_t ld, int layout, const int32_t* sym,
                       int B, int D, int K, int bits, int32_t* status, void* stream);

/*
 * bs_rans_pop -- ANS.decode (mnist_compress.py:58-68), B chains, symbols i = D-1..0:
 *   m = head & (2^bits - 1); s = max{j : c_j <= m}; head = f_s * (head >> bits) + m - c_s
 *   if head < 2^32: head = head << 32 | stack[--len]
 * cdf as in bs_rans_push_table.  sym_out [B,D] int32.  If `centres` is non-null (row d at
 * centres + d*c_stride doubles, K entries) the bin centre of every decoded symbol is also
 * written as float32 to centre_out [B,D]: the gather + cast of mnist_compress.py:181,196 and
 * model/mnist_train.py:324,392.
 */
int bs_rans_pop(uint64_t* head, uint32_t* stack, int32_t* len, int64_t cap,
                const uint32_t* cdf, int64_t chain_stride, int64_t ld, int layout, int B, int D, int K,
                int bits, int32_t* sym_out, const double* centres, int64_t c_stride, float* centre_out,
                int32_t* status, void* stream);

/*
 * bs_rans_pop_pivot -- bs_rans_pop on BS_LAYOUT_PIVOT rows (the production pair of the batched codec for every table
 * of uniform-width bins): the same ANS.decode (mnist_compress.py:58-68), the same symbols and words; the integer row of
 * a symbol's group is rebuilt inside the kernel with the operations bs_logistic_tables spent on it (the SAME endpoints,
 * bin_step, cdf_spec (2, 3 or 4), mu, scale, bits, quantbits must be passed), so only 64 cumulative values per row travel through HBM.
 * pivots [B,D,ld] as written by bs_logistic_tables(layout = BS_LAYOUT_PIVOT); D % 64 == 0, D <= BS_POP_PIVOT_MAX_D
 * (a chain's D symbols and the 2 KB parameter block of a 64-row chunk share one 64 KB LDS allocation).
 */
#define BS_POP_PIVOT_MAX_D 15872
int bs_rans_pop_pivot(uint64_t* head, uint32_t* stack, int32_t* len, int64_t cap, const uint32_t* pivots, int64_t ld,
                      const double* endpoints, int64_t e_stride, const double* bin_step, int cdf_spec, const void* mu,
                      const void* scale, int param_dtype, int B, int D, int K, int bits, int quantbits,
                      int32_t* sym_out, const double* centres, int64_t c_stride, float* centre_out, int32_t* status,
                      void* stream);

/*
 * BS_FORMAT_WAVE64 -- opt-in 64-state stream format (no reference counterpart).  A chain owns 64 independent rANS
 * states: head64 [B,64] uint64, stack64 [B,64,cap] uint32, len64 [B,64] int32; symbol d of a coding operation is coded
 * on state d % 64 with the reference's arithmetic and order inside that state (ANS.encode / ANS.decode,
 * mnist_compress.py:49-68: pushes ascending d, pops descending d).  Streams in this format are NOT the reference's
 * word stream (they cost 64 heads instead of one per chain); they exist because the format has no serial chain longer
 * than D/64 symbols, so one launch does the whole of mnist_compress.py:183-188 (or :198-203) -- logistic CDF, integer
 * table, rANS step -- with the table row never leaving the registers of the wavefront that built it.
 *
 * bs_layer_pop64  -- pop D symbols per chain under Logistic(mu, scale) discretised on `endpoints` (arguments as
 *   bs_logistic_tables; p_stride = elements between two chains' mu/scale rows, D normally, 0 = one row set shared by
 *   all chains, the prior); sym_out [B,D], optional bin centres as in bs_rans_pop.  D <= 4096, K in {256, 512, 1024}.
 * bs_layer_push64 -- push sym [B,D] under the same model.
 * status [B]: BS_ST_UNDERFLOW / OVERFLOW / BADTABLE / BADSYMBOL, sticky, whichever state of the chain reports first.
 */
int bs_layer_pop64(uint64_t* head64, uint32_t* stack64, int32_t* len64, int64_t cap, const double* endpoints,
                   int64_t e_stride, const double* bin_step, int cdf_spec, const void* mu, const void* scale, int64_t p_stride,
                   int param_dtype, int B, int D, int K, int bits, int quantbits, int32_t* sym_out, const double* centres,
                   int64_t c_stride, float* centre_out, int32_t* status, void* stream);
int bs_layer_push64(uint64_t* head64, uint32_t* stack64, int32_t* len64, int64_t cap, const double* endpoints,
                    int64_t e_stride, const double* bin_step, int cdf_spec, const void* mu, const void* scale, int64_t p_stride,
                    int param_dtype, const int32_t* sym, int B, int D, int K, int bits, int quantbits, int32_t* status,
                    void* stream);

/*
 * bs_gather_centres -- centre_out[b,d] = (float) centres[d*c_stride + sym[b,d]]
 * (mnist_compress.py:181,196,308 followed by the .float() of model/mnist_train.py:324,392).
 */
int bs_gather_centres(const double* centres, int64_t c_stride, const int32_t* sym, int B, int D, int K,
                      float* centre_out, void* stream);

/*
 * Scheduling helpers (no reference counterpart; round 5): a HIP stream whose kernels run on a subset of the
 * compute units, so that the one-wavefront-per-chain coder kernels can be kept off the CUs the bulk kernels fill.
 * bs_stream_create_cu_mask -- *stream_out = a stream restricted to the n_cus mask bits [first_cu, first_cu + n_cus); the driver
 *   deals the mask bits round the 8 XCDs (bit b = XCD b % 8), so 8 m consecutive bits are m CUs on every XCD.  HOST pointers.
 * bs_stream_destroy -- destroys it.
 * bs_debug_where -- diagnostics: n one-wavefront workgroups that spin spin_cycles and record where they ran
 *   (ids_out[i] = HW_ID[15:0] | XCC_ID << 16, device pointer): how the tests check what a mask really does.
 */
int bs_stream_create_cu_mask(int first_cu, int n_cus, void** stream_out);
int bs_stream_destroy(void* stream);
int bs_debug_where(uint32_t* ids_out, int n, int spin_cycles, void* stream);

/*
 * bs_selftest -- runs the wave-level primitives (DPP scan / reductions) and the deterministic
 * sigmoid against in-kernel scalar restatements; host pointer `failures` receives the number of
 * mismatching lanes.  Synchronises the stream.  For tests only.
 */
int bs_selftest(int64_t* failures_host, void* stream);

/* bs_sigmoid_f64 -- out[i] = deterministic sigmoid(t[i]); exposes the CDF spec for parity tests */
int bs_sigmoid_f64(const double* t, int64_t n, double* out, void* stream);

/*
 * Conv-stack kernels (bitswap_amd/csrc/net_epilogue.hip, wino_gemm.hip).  Since round 3 NO convolution of Model.infer /
 * Model.generate (model/mnist_train.py:315-438) in compress mode is a library call: the ResNet, head and 5x5 input
 * convolutions run in the Winograd domain (bs_wino_fused_f32 transform passes around ONE batched fp32 MFMA product,
 * bs_wino_gemm_f32 / bs_small_k_gemm_f32), the 3x3 input convolutions in bs_conv3_wino_f32 -- every output summed in
 * one fixed order, so (mu, scale) do not depend on how many chains are coded per call.  The two entry points below are the
 * pointwise passes of the unfused fallback routes (narrow test models, BITSWAP_OWN_GEMM=0).
 * NCHW float32, contiguous; N images, C channels, HW pixels.
 *
 * bs_bias_residual_elu_f32 -- s = x + bias[c] (+ res); sum_out = s (nullable); act_out = ELU(s)
 *   (nullable; at least one output).  Covers `act(conv(x))` of the input convs and
 *   `x + conv2(act(conv1(act(x))))` of ResNetLayer (utils/torch/modules.py:216-241): the sum feeds the
 *   next layer's skip connection, its ELU the next conv.  bias and res are nullable; outputs may alias x.
 *
 * bs_head_params_f32 -- x [N,2C,HW] is ONE convolution with the mu and the std filters stacked
 *   (the reference runs two, mnist_train.py:346-349,365-368,423-426); bias [2C].
 *   mu = x[:, :C] + bias[:C];  s = x[:, C:] + bias[C:];
 *   BS_HEAD_SIGMOID : scale = 0.1 + 0.9 * sigmoid(s + 2)                 (inference heads)
 *   BS_HEAD_SOFTPLUS: scale = 0.1 + 0.9 * softplus(s + log(e - 1))       (deep generative heads)
 *   mu, scale [N,C,HW] float32.
 *
 * bs_expand_rows5_f32 -- operand builder for the 5x5 convolutions run as GEMMs on rocBLAS/hipBLASLt
 *   (bitswap_amd/model.py::_conv5_gemm): out [N, C*5, H+4, W],
 *   out[n, c*5+dx, yy, x] = act(in[n, c, yy-2, x+dx-2] + bias[c]) inside the image, 0 outside;
 *   act != 0 applies ELU, bias nullable.  Kernel row dy of the convolution is then one strided-batched
 *   GEMM W_dy [Cout, C*5] x out[n, :, dy:dy+H, :] (leading dimension (H+4)*W).  W % 4 == 0.
 *
 * bs_wino_in_f32 / bs_wino_out_f32 -- the two ends of a Winograd-domain convolution whose middle is ONE
 *   batched GEMM M[t] = U[t] x V[t], t = 0..ts*ts-1 (bitswap_amd/model.py::_res_wino; U = G g G^T is computed
 *   from the folded weights once, bitswap_amd/winograd.py).  (ts, ms) = tile size, tile stride:
 *     (6, 4): F(4x4, 3x3), 'same' padding 1;  (6, 2): F(2x2, 5x5), padding 2;  (8, 4): F(4x4, 5x5), padding 2.
 *   H, W multiples of ms.
 *     in : V [ts*ts, C, N*T] <- B^T d B of the ts x ts windows of act(in [N,C,H,W] + bias[c]);
 *          T = (H/ms)*(W/ms), column = n*T + tile;  act != 0 applies ELU;  bias nullable.
 *     out: s = A^T M A + bias[c] (+ res [N,C,H,W]) from M [ts*ts, C, N*T]; sum_out = s, act_out = ELU(s)
 *          (each nullable, at least one), both [N,C,H,W].
 *
 * bs_wino_fused_f32 -- everything between two batched GEMMs of a ResNet layer in one pass (tile stride 4:
 *   ts 6 = F(4x4,3x3), ts 8 = F(4x4,5x5); H, W multiples of 4 with (H/4)*(W/4) dividing 256):
 *     source: ts_in == 0 ? src = x [N,C,H,W] : src = M [ts_in^2, C, N*T] -> A^T M A
 *     s = source + bias[c] (+ res);  sum_out = s;  a = (act & 1) ? ELU(s) : s;  act_out = a   (outputs nullable)
 *     ts_out != 0: V [ts_out^2, C, N*T] <- B^T a' B, a' = (act & 2) ? ELU(a) : a   (the operand of the next GEMM)
 *   A layer x + conv2(ELU(conv1(ELU(x)) + b1)) + b2 is: GEMM, fused(ts,ts), GEMM, fused(ts,ts | 0).
 *
 * bs_conv3_wino_f32 -- the 3x3 'same' INPUT convolution of a stack (x [N,Cin,H,W], w [C,Cin,3,3], small Cin) fused with
 *   what follows it up to the first GEMM of the next block: h = (act & 1) ? ELU(conv(x) + bias[c]) : conv(x) + bias[c];
 *   act_out [N,C,H,W] = h (nullable); V [ts_out^2, C, N*T] = B^T h' B with h' = (act & 2) ? ELU(h) : h.  ts_out 6 or 8.
 *   H, W multiples of 4 with T = (H/4)*(W/4) dividing 64 (a wavefront covers whole images) and the Cin planes of 64/T
 *   images within the LDS (BS_EUNSUPPORTED otherwise; bitswap_amd.hip.conv3_wino_supported).  Per (image, channel) the
 *   sum runs over ci, then ky, kx in that order: batch-invariant.
 *
 * bs_wino_gemm_f32 -- M [T, Cout, cols] = U [T, Cout, Cin] x V [T, Cin, cols], float32 on the matrix cores
 *   (v_mfma_f32_32x32x2_f32, float32 accumulate): the batched product in the middle of a Winograd-domain convolution
 *   (bitswap_amd/csrc/wino_gemm.hip: persistent workgroups over (t, row tile, 32-column block) units, operands staged by
 *   LDS-DMA).  Every output element is the sum over ci in one fixed order that depends on Cin only: results are bitwise
 *   independent of `cols` (how many blocks are coded together) and of Cout, which no BLAS library promises -- since round 3
 *   every product of the conv stacks takes it, the 16-channel head convolutions included.  Cin % 16 == 0, cols % 4 == 0,
 *   Cin * cols < 2^31, 16-byte aligned operands (BS_EUNSUPPORTED / BS_EINVAL otherwise).
 *
 * bs_wino_gemm_bf16x3 -- the same product with every float32 operand split exactly into three bfloat16 limbs and assembled
 *   from nprod = 6 (limb products down to relative size 2^-16; the three of size 2^-24 dropped) or 9 (all: every product
 *   exact) v_mfma_f32_32x32x16_bf16 per 16-deep k block, float32 accumulation, one fixed order per output that depends on
 *   Cin alone (bitswap_amd/csrc/wino_gemm_bf16x3.hip).  U_frags [T, ceil(Cout/32), Cin/16, 3, 64, 8] bfloat16 bit patterns:
 *   the three limbs of U (U = limb0 + limb1 + limb2 exactly), split and tiled once by the caller as MFMA A fragments --
 *   entry [t, r, kb, i, l, e] = limb i of U[t, 32 r + l % 32, 16 kb + 8 (l / 32) + e], rows beyond Cout zero
 *   (bitswap_amd.hip.frags_bf16x3); V float32 as above, split inside the kernel -- by producer wavefronts of its own in the
 *   default launch shape (one multiplying wavefront per SIMD; bitswap_amd/csrc/wino_gemm_bf16x3.hip), every launch shape adding
 *   the same products in the same order.  The DEFAULT arithmetic of the conv stacks' big products since round 6
 *   (BITSWAP_GEMM_ARITH=fp32 opts out): a different rounding of (mu, scale) than bs_wino_gemm_f32, hence named in the stream
 *   fingerprint -- a receiver takes the arithmetic the record names.  No reference counterpart (the reference's convolutions are
 *   cuDNN float32, utils/torch/modules.py:233-241).  Cin % 16 == 0, cols % 4 == 0, 16-byte aligned operands.
 *
 * bs_small_k_gemm_f32 -- M [T, Cout, cols] = U [T, Cout, Cin] x V [T, Cin, cols] for small Cin (<= 64): the batched product
 *   of the INPUT convolutions of the stacks in the Winograd domain (Cin = zchannels or 4 x image channels); a write of M
 *   with a dozen multiply-adds per element.  cols % 4 == 0, 16-byte aligned operands.
 */
#define BS_HEAD_SIGMOID 0
#define BS_HEAD_SOFTPLUS 1
int bs_bias_residual_elu_f32(const float* x, const float* bias, const float* res, float* sum_out,
                             float* act_out, int64_t N, int C, int HW, void* stream);
int bs_head_params_f32(const float* x, const float* bias, float* mu, float* scale, int64_t N, int C,
                       int HW, int mode, void* stream);
int bs_expand_rows5_f32(const float* in, const float* bias, float* out, int64_t N, int C, int H, int W,
                        int act, void* stream);
int bs_wino_gemm_f32(const float* U, const float* V, float* M, int T, int Cout, int Cin, int64_t cols, void* stream);
int bs_wino_gemm_bf16x3(const uint16_t* U_frags, const float* V, float* M, int T, int Cout, int Cin, int64_t cols,
                        int nprod, void* stream);
int bs_conv3_wino_f32(const float* x, const float* w, const float* bias, int act, float* act_out, float* V, int ts_out,
                      int64_t N, int Cin, int C, int H, int W, void* stream);
int bs_small_k_gemm_f32(const float* U, const float* V, float* M, int T, int Cout, int Cin, int64_t cols, void* stream);
int bs_wino_fused_f32(const float* src, int ts_in, const float* bias, const float* res, int act, float* sum_out,
                      float* act_out, float* V, int ts_out, int64_t N, int C, int H, int W, void* stream);
int bs_wino_in_f32(const float* in, const float* bias, float* V, int64_t N, int C, int H, int W, int ts,
                   int ms, int act, void* stream);
int bs_wino_out_f32(const float* M, const float* bias, const float* res, float* sum_out, float* act_out,
                    int64_t N, int C, int H, int W, int ts, int ms, void* stream);

/*
 * Channels-last layer operators (bitswap_amd/csrc/linear.hip, norm_act.hip, pack8.hip): a layer over rows of channels -- the
 * pixels of channels-last latents, or any [rows, channels] -- and its gradients.  dtype: BS_DT_F32 / BF16 / F16, the type of x, w,
 * res, s, gradients and outputs; bias, gamma and beta may be float32 beside a 16-bit dtype (their own dtype argument).  Row
 * strides (ld*) are in elements, channels of a row are contiguous, addresses need the alignment of an element only.  Sums and
 * statistics are float32; outputs are rounded once, to nearest even.  dx and dw take the ds they are given, of dtype: in 16 bits, where
 * bs_act_grad made it, that is one rounding (of ds) before theirs.
 *
 * bs_linear_act -- s = x w^T + bias (+ res), a = act(s); x [rows, K], w [N, K], bias [N] (nullable), res [rows, N] (nullable);
 *   sum_out = s, act_out = a, contiguous [rows, N] (each nullable, at least one).  act sees s before its rounding.  float32
 *   operands are split into three bfloat16 limbs and multiplied as six limb products (as bs_wino_gemm_bf16x3), here and in the
 *   gradients: operands below 2^-110 keep their bits down to 2^-133 only; a sum that does
 *   not come out finite is added up again in float32, so infinities and NaN arrive as they do in float32 arithmetic.  A row's
 *   bits do not depend on `rows`.  K, N <= 2^20, here and in the gradients.
 *
 * Workspaces: the *_workspace functions give the bytes a call needs (0: none) for w laid out for the kernel, copies of rows that are
 *   not whole, partial sums; their address is a multiple of 16.  Outputs and workspaces overlap no input.  whole: the operand's address, row stride and row are multiples of 16 bytes and the stride is under 4
 *   MiB; rows that are not are copied first.  zeros (of ds): the rows end in zeros up to the next multiple of 16 bytes, which lies
 *   within their stride, as bs_act_grad writes them -- such rows count as whole.
 *
 * bs_act_grad -- ds = g_sum + g_act act'(s) (either gradient nullable, not both), rows [rows, N]: ds_out (row stride ldds,
 *   nullable; where ldds has the room its rows end in zeros up to the next multiple of 16 bytes), db_out [N] float32 = sum over
 *   the rows of ds before its rounding (nullable; workspace of bs_act_grad_workspace bytes then).
 *   s: [rows, N] of dtype (row stride lds), or, if s_exps is given, int8 codes [rows, N] with their exponents (bs_pack8).
 *   act BS_ACT_NONE: s is not read and may be null.
 * bs_linear_grad_x -- dx [rows, K] = ds w;  ds [rows, N] (row stride ldds), w [N, K].
 * bs_linear_grad_w -- dw [N, K] = ds^T x;  x [rows, K] of dtype (row stride ldx) or, if x_exps is given, codes of bs_pack8.  The
 *   rows are split over the chip into parts of a size fixed by (rows, N, K) and the parts added in order: the same call gives the
 *   same bits.  rows <= 2^30.
 *
 * bs_group_norm_act -- x [n, pixels, channels] (strides ldn, ldp), groups dividing channels: mean and biased variance over the
 *   pixels and channels of a group, u = (x - mean) / sqrt(var + eps) * gamma + beta, y = act(u), y contiguous; stats
 *   [n, groups, 2] float32 = (mean, 1 / sqrt(var + eps)) (nullable).  An image's bits do not depend on n.
 *   channels <= 2^20.  workspace: bs_group_norm_workspace bytes (0 for images that fit a workgroup's registers).
 * bs_group_norm_act_grad -- with h = (x - mean) rstd, du = g act'(h gamma + beta), t = du gamma:
 *   dx = rstd (t - mean_g(t) - h mean_g(t h)), dgamma = sum du h, dbeta = sum du (float32 [channels], each nullable).
 *   x [n, pixels, channels] of dtype, or codes of bs_pack8 over [n * pixels, channels] if x_exps is given.
 *
 * bs_pack8 -- x [rows, channels] -> codes int8 [rows, channels] and exps int8 [rows, ceil(channels / 32)]: 32 channels of a row
 *   share 2^e, e the smallest integer >= -126 with max|x| <= 127 2^e, at most 121 (float16: 9: 127 2^e stays a value of the type);
 *   code = rint(x 2^-e) (ties to even) within +-127; -128 marks a value that is not finite (left out of the maximum).
 *   bs_unpack8 -- x = code 2^e, exact in every dtype that held x; -128 gives NaN.
 *
 * All of them: BS_EINVAL for null operands, negative sizes, strides below the row length, unknown types or activations, a
 * workspace that is too small or not aligned, sizes that would take a launch of 2^32 threads or more (operands of tens of gigabytes; nothing has
 * been launched then); rows == 0 or n == 0 is a call without rows (gradients of parameters are then zero).
 */
#define BS_DT_F32 0
#define BS_DT_BF16 1
#define BS_DT_F16 2
#define BS_ACT_NONE 0
#define BS_ACT_ELU 1
#define BS_ACT_SILU 2
#define BS_ACT_GELU 3
int64_t bs_linear_workspace(int dtype, int64_t rows, int K, int N, int whole);
int bs_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, const void* res,
                  int64_t ldr, void* sum_out, void* act_out, int act, int dtype, int64_t rows, int K, int N, void* workspace,
                  int64_t workspace_bytes, void* stream);
int64_t bs_act_grad_workspace(int64_t rows, int N);
int bs_act_grad(const void* g_sum, int64_t ldgs, const void* g_act, int64_t ldga, const void* s, const int8_t* s_exps, int64_t lds,
                int act, int dtype, int64_t rows, int N, void* ds_out, int64_t ldds, float* db_out, void* workspace,
                int64_t workspace_bytes, void* stream);
int64_t bs_linear_grad_x_workspace(int dtype, int64_t rows, int K, int N, int whole);
int bs_linear_grad_x(const void* ds, int64_t ldds, int zeros, const void* w, int64_t ldw, void* dx, int dtype, int64_t rows, int K, int N,
                     void* workspace, int64_t workspace_bytes, void* stream);
int64_t bs_linear_grad_w_workspace(int dtype, int64_t rows, int K, int N, int codes, int x_whole, int ds_whole);
int bs_linear_grad_w(const void* ds, int64_t ldds, int zeros, const void* x, const int8_t* x_exps, int64_t ldx, void* dw, int dtype,
                     int64_t rows, int K, int N, void* workspace, int64_t workspace_bytes, void* stream);
int64_t bs_group_norm_workspace(int dtype, int64_t n, int64_t pixels, int channels, int groups, int grad);
int bs_group_norm_act(const void* x, int64_t ldn, int64_t ldp, const void* gamma, const void* beta, int affine_dtype, float eps,
                      int act, int dtype, int64_t n, int64_t pixels, int channels, int groups, void* y, float* stats,
                      void* workspace, int64_t workspace_bytes, void* stream);
int bs_group_norm_act_grad(const void* g, int64_t ldgn, int64_t ldgp, const void* x, const int8_t* x_exps, int64_t ldn, int64_t ldp,
                           const float* stats, const void* gamma, const void* beta, int affine_dtype, int act, int dtype, int64_t n,
                           int64_t pixels, int channels, int groups, void* dx, float* dgamma, float* dbeta, void* workspace,
                           int64_t workspace_bytes, void* stream);
int bs_pack8(const void* x, int64_t ldx, int8_t* codes, int8_t* exps, int dtype, int64_t rows, int channels, void* stream);
int bs_unpack8(const int8_t* codes, const int8_t* exps, void* x, int dtype, int64_t rows, int channels, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* BITSWAP_HIP_H */
