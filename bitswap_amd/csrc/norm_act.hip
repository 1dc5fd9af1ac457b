// norm_act.hip -- group norm with an activation on channels-last activations, and its gradient.
//
//   m = mean, v = variance of a group (all pixels, channels / groups neighbouring channels);  r = 1 / sqrt(v + eps)
//   h = (x - m) r,  u = h gamma + beta,  y = act(u)
//   du = g act'(u), t = du gamma:   dx = r (t - mean(t) - h mean(t h)),  dgamma = sum du h,  dbeta = sum du
//
// Bound by memory: x (and g) in, y (dx) out.  Where the pixels of a few whole groups fit a workgroup's registers (k_norm,
// k_norm_grad) everything is read once: a thread keeps 32 elements (V neighbouring channels of 32 / V pixels), sums go over its
// pixels, then over the workgroup's pixel lanes and a group's channels, by exchanges between lanes where channels and pixels divide
// into powers of two, else through shared memory; the variance is the mean squared distance from the mean already known.  Larger
// images (k_part, k_join, k_apply) are cut into runs of pixels whose per-channel sums are joined in a second launch and applied in a
// third.  Which way is taken, and every order of addition, follows from (pixels, channels, groups, type) alone: an image's bits do
// not depend on how many there are.
//
// Measured (256 x 256 images in 32 groups; the bytes in and out at 4.9 TB/s in brackets): bfloat16, 400 images 23.8 us [21.5];
// float32, 100 images 9.3 us, their gradient 16.7 us and 3 for the parameters' [17]; one image 6.3 us, bound by the one workgroup's
// load, reduction and store one after the other.
#include "rows_dev.h"

namespace {

struct NormArgs {
    const char *x, *g;
    const int8_t* exps;                 // x in 8 bits
    int64_t ldn, ldp, ldgn, ldgp;
    const char *gamma, *beta;
    int aff_f32, act;
    float eps;
    int64_t n, pixels;
    int C, G, per;
    int pl;                             // pixel lanes of a workgroup
    int cl;                             // lanes along the channels
    int gs;                             // groups of a workgroup
    int slabs;
    int nb;                             // 8-bit blocks of a row
    char* y;
    float* stats;                       // in or out
    float* parts;                       // grad: [n][2][C] sums of du h, du; split: per run of pixels
    int runs;
    int64_t run;
};

template <int DT>
__device__ __forceinline__ void affine(const char* p, int f32, int c, int left, float fill, float* v) {
    constexpr int V = vlen(DT);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = fill;
    if (!p || left <= 0) return;
    if (f32) {
#pragma unroll
        for (int i = 0; i < V; i += 4)
            if (left > i) load_vec<BS_DT_F32>(p + (int64_t)(c + i) * 4, left - i, v + i);
    } else {
        load_vec<DT>(p + (int64_t)c * esize(DT), left, v);
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) v += __shfl_xor(v, o);
    return v;
}

// Workgroups of one XCD (blockIdx % 8) take a run of the work: the slabs of an image, whose rows share cache lines where a slab is no
// multiple of them, go through one L2.  -1: nothing left (the grid is a multiple of 8).
__device__ __forceinline__ int64_t xcd_run(int64_t total) {
    const int64_t at = (blockIdx.x % 8) * ((total + 7) / 8) + blockIdx.x / 8;
    return at < total ? at : -1;
}

// N sums per thread and channel -> sums per group, known to every thread of the workgroup (any channels per group).
//   add_up: over the pixel lanes, in Q parts a channel (red -> part).  groups: over a group's parts, each channel's times its weight
//   (null: 1), a wavefront a group.  channels: a channel's sum, out to memory.
struct SlabSum {
    float *red, *part, *out;
    int ch, PL, Q, gs, per, nthr, tid;           // ch: channels of the slab (lanes x V)
    template <int N, int V>
    __device__ __forceinline__ void add_up(const float (&a)[N][V], int pl, int c, bool live) const {
        if (live)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < V; ++i) red[(n * PL + pl) * ch + c + i] = a[n][i];
        __syncthreads();
        for (int i = tid; i < ch * Q; i += nthr) {
            const int q = i / ch, k = i - q * ch;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float s = 0.0f;
#pragma unroll 4
                for (int p = q; p < PL; p += Q) s += red[(n * PL + p) * ch + k];
                part[n * Q * ch + i] = s;
            }
        }
        __syncthreads();
    }
    template <int N>
    __device__ __forceinline__ void channels(int width, int64_t C, float* to) const {
        for (int k = tid; k < width; k += nthr)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float s = 0.0f;
#pragma unroll 4
                for (int q = 0; q < Q; ++q) s += part[(n * Q + q) * ch + k];
                to[n * C + k] = s;
            }
    }
    template <int N>
    __device__ __forceinline__ void groups(const float* weight) const {
        for (int g = tid >> 6; g < gs; g += nthr >> 6) {
            float s[N];
#pragma unroll
            for (int n = 0; n < N; ++n) s[n] = 0.0f;
            for (int j = tid & 63; j < per * Q; j += 64) {
                const int q = j / per, k = g * per + j - q * per;
                const float w = weight ? weight[k] : 1.0f;
#pragma unroll
                for (int n = 0; n < N; ++n) s[n] = fmaf(part[(n * Q + q) * ch + k], w, s[n]);
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                s[n] = wave_sum(s[n]);
                if ((tid & 63) == 0) out[n * gs + g] = s[n];
            }
        }
        __syncthreads();
    }
};

// ---- images that fit -------------------------------------------------------------------------------------------------------
// Sums of N values over a group where its channels are whole lanes (per % V == 0) and lanes and groups are powers of two: exchanges
// within the wavefront, one barrier, and every thread adds up what the wavefronts left for its group.
template <int N>
struct LaneSum {
    int cl, cpg, CL, gs, rows, row, lane;           // lanes per group and of the slab; wavefronts that hold pixels of one lane
    __device__ __forceinline__ void run(float (&v)[N], float* red) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            for (int o = 1; o < cpg; o *= 2) v[n] += __shfl_xor(v[n], o);
            for (int o = CL; o < 64; o *= 2) v[n] += __shfl_xor(v[n], o);
        }
        const int g = cl / cpg;
        if ((cl & (cpg - 1)) == 0 && (CL >= 64 || lane < CL)) {
#pragma unroll
            for (int n = 0; n < N; ++n) red[(n * rows + row) * gs + g] = v[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = 0.0f;
            for (int r = 0; r < rows; ++r) v[n] += red[(n * rows + r) * gs + g];
        }
    }
};
template <int N>
__device__ __forceinline__ LaneSum<N> lane_sum(const NormArgs& a, int cl, int V, int tid) {
    LaneSum<N> s;
    s.cl = cl; s.cpg = a.per / V; s.CL = a.cl; s.gs = a.gs; s.lane = tid & 63;
    const int wpr = a.cl > 64 ? a.cl / 64 : 1;                       // wavefronts a pixel takes
    const int waves = (a.pl * a.cl + 63) / 64;
    s.rows = waves / wpr;
    s.row = (tid >> 6) / wpr;
    return s;
}

template <int DT, bool LANES>
__global__ __launch_bounds__(1024) void k_norm(const NormArgs a) {
    constexpr int V = vlen(DT), R = 32 / V, ES = esize(DT);
    extern __shared__ __align__(16) float sh[];
    const int PL = a.pl, CL = a.cl, tid = threadIdx.x;
    const int64_t at = xcd_run(a.n * a.slabs);
    if (at < 0) return;
    const int64_t img = at / a.slabs;
    const int slab = (int)(at % a.slabs), c0 = slab * a.gs * a.per;
    const int width = min(a.gs * a.per, a.C - c0);               // channels of this slab
    const int pl = tid / CL, cl = tid - pl * CL, k = cl * V, left = width - k;
    const bool live = pl < PL && left > 0;

    float f[R][V];
    const char* const xp = a.x + (img * a.ldn + c0 + k) * ES;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[r][i] = 0.0f;
        const int64_t p = pl + (int64_t)r * PL;
        if (live && p < a.pixels) load_vec<DT>(xp + p * a.ldp * ES, left, f[r]);
    }
    float ga[V], be[V];
    affine<DT>(a.gamma, a.aff_f32, c0 + k, live ? left : 0, 1.0f, ga);
    affine<DT>(a.beta, a.aff_f32, c0 + k, live ? left : 0, 0.0f, be);
    const float inv = 1.0f / ((float)a.pixels * (float)a.per);
    float m[V], rs[V];
    if (LANES) {
        const LaneSum<1> sum = lane_sum<1>(a, cl, V, tid);
        float t[1] = {0.0f};
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < V; ++i) t[0] += f[r][i];
        sum.run(t, sh);
        const float mean = t[0] * inv;
        t[0] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (live && pl + r * PL < a.pixels) {
#pragma unroll
                for (int i = 0; i < V; ++i) t[0] = fmaf(f[r][i] - mean, f[r][i] - mean, t[0]);
            }
        sum.run(t, sh + 16 * a.gs);
        const float rstd = 1.0f / sqrtf(t[0] * inv + a.eps);
        if (a.stats && live && pl == 0 && k % a.per == 0) {
            float* const o = a.stats + (img * a.G + (c0 + k) / a.per) * 2;
            o[0] = mean;
            o[1] = rstd;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            m[i] = mean;
            rs[i] = rstd;
        }
    } else {
        SlabSum ss;
        ss.ch = CL * V; ss.PL = PL; ss.Q = max(1, PL / V); ss.gs = min(a.gs, a.G - slab * a.gs); ss.per = a.per;
        ss.nthr = blockDim.x; ss.tid = tid;
        ss.red = sh; ss.part = sh + PL * ss.ch; ss.out = ss.part + ss.Q * ss.ch;
        float t[1][V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            t[0][i] = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) t[0][i] += f[r][i];
        }
        int g[V];
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = min(k + i, width - 1) / a.per;
        ss.add_up<1, V>(t, pl, k, live);
        ss.groups<1>(nullptr);
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] = i < left ? ss.out[g[i]] * inv : 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            t[0][i] = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (pl + r * PL < a.pixels) t[0][i] = fmaf(f[r][i] - m[i], f[r][i] - m[i], t[0][i]);
        }
        float* const mean_sh = ss.out;                               // the means stay: the next sums go behind them
        ss.out += ss.gs;
        ss.add_up<1, V>(t, pl, k, live);
        ss.groups<1>(nullptr);
#pragma unroll
        for (int i = 0; i < V; ++i) rs[i] = i < left ? 1.0f / sqrtf(ss.out[g[i]] * inv + a.eps) : 0.0f;
        if (a.stats)                                                 // (16-bit groups of one channel: up to 121 of them for 64 threads)
            for (int j = tid; j < ss.gs; j += ss.nthr) {
                float* const o = a.stats + (img * a.G + slab * a.gs + j) * 2;
                o[0] = mean_sh[j] * inv;
                o[1] = 1.0f / sqrtf(ss.out[j] * inv + a.eps);
            }
    }
    if (!live) return;
    char* const yp = a.y + (img * a.pixels * a.C + c0 + k) * ES;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t p = pl + (int64_t)r * PL;
        if (p >= a.pixels) break;
#pragma unroll
        for (int i = 0; i < V; ++i) f[r][i] = fmaf((f[r][i] - m[i]) * rs[i], ga[i], be[i]);
        act_values<DT, V>(a.act, f[r], f[r]);
        store_out<DT>(yp + p * a.C * ES, left, f[r], a.C);
    }
}

template <int DT, bool SAVED8>
__device__ __forceinline__ void load_x(const NormArgs& a, int64_t img, int64_t p, int c, int left, float* f) {
    constexpr int V = vlen(DT);
    if (SAVED8) {
        const int64_t row = img * a.pixels + p;
        load_codes<V>((const int8_t*)a.x + row * a.C, a.exps + row * a.nb, c, left, f);
    } else {
        load_vec<DT>(a.x + (img * a.ldn + p * a.ldp + c) * esize(DT), left, f);
    }
}

template <int DT, bool SAVED8, bool LANES, int THREADS>
__global__ __launch_bounds__(THREADS) void k_norm_grad(const NormArgs a) {
    constexpr int V = vlen(DT), R = 32 / V, ES = esize(DT);
    extern __shared__ __align__(16) float sh[];
    const int PL = a.pl, CL = a.cl, tid = threadIdx.x;
    const int64_t at = xcd_run(a.n * a.slabs);
    if (at < 0) return;
    const int64_t img = at / a.slabs;
    const int slab = (int)(at % a.slabs), c0 = slab * a.gs * a.per;
    const int width = min(a.gs * a.per, a.C - c0);
    const int pl = tid / CL, cl = tid - pl * CL, k = cl * V, left = width - k;
    const bool live = pl < PL && left > 0;
    SlabSum ss;
    ss.ch = CL * V; ss.PL = PL; ss.Q = max(1, PL / V); ss.gs = min(a.gs, a.G - slab * a.gs); ss.per = a.per;
    ss.nthr = blockDim.x; ss.tid = tid;
    ss.red = sh; ss.part = sh + 2 * PL * ss.ch; ss.out = ss.part + 2 * ss.Q * ss.ch;
    float* const weight = ss.out + 32 * a.gs;

    float h[R][V], d[R][V], m[V], rs[V], ga[V], be[V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < V; ++i) h[r][i] = d[r][i] = 0.0f;
        const int64_t p = pl + (int64_t)r * PL;
        if (live && p < a.pixels) {
            load_x<DT, SAVED8>(a, img, p, c0 + k, left, h[r]);
            load_vec<DT>(a.g + (img * a.ldgn + p * a.ldgp + c0 + k) * ES, left, d[r]);
        }
    }
    if (LANES) {                                                     // the lane's channels are of one group
        const float* const st = a.stats + (img * a.G + (c0 + min(k, width - 1)) / a.per) * 2;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            m[i] = st[0];
            rs[i] = st[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float* const st = a.stats + (img * a.G + (c0 + min(k + i, width - 1)) / a.per) * 2;
            m[i] = st[0];
            rs[i] = st[1];
        }
    }
    affine<DT>(a.gamma, a.aff_f32, c0 + k, live ? left : 0, 1.0f, ga);
    affine<DT>(a.beta, a.aff_f32, c0 + k, live ? left : 0, 0.0f, be);
    float s[2][V];                                                   // sums of du h and of du
#pragma unroll
    for (int i = 0; i < V; ++i) s[0][i] = s[1][i] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (live && pl + r * PL < a.pixels) {
            float u[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[r][i] = (h[r][i] - m[i]) * rs[i];
                u[i] = fmaf(h[r][i], ga[i], be[i]);
            }
            act_slopes<V>(a.act, u, d[r]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[0][i] = fmaf(d[r][i], h[r][i], s[0][i]);
                s[1][i] += d[r][i];
            }
        }
    float* const po = a.parts ? a.parts + img * 2 * a.C + c0 : nullptr;
    const float inv = 1.0f / ((float)a.pixels * (float)a.per);
    float m1[V], m2[V];
    if (LANES) {
        const LaneSum<2> sum = lane_sum<2>(a, cl, V, tid);
        float t[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < V; ++i) {
            t[0] = fmaf(ga[i], s[0][i], t[0]);
            t[1] = fmaf(ga[i], s[1][i], t[1]);
        }
        sum.run(t, ss.out);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            m2[i] = t[0] * inv;
            m1[i] = t[1] * inv;
        }
    } else {
        if (live && pl == 0)
#pragma unroll
            for (int i = 0; i < V; ++i) weight[k + i] = ga[i];
        ss.add_up<2, V>(s, pl, k, live);
        if (po) ss.channels<2>(width, a.C, po);
        ss.groups<2>(weight);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int g = min(k + i, width - 1) / a.per;
            m2[i] = ss.out[g] * inv;
            m1[i] = ss.out[ss.gs + g] * inv;
        }
    }
    if (live) {
        char* const yp = a.y + (img * a.pixels * a.C + c0 + k) * ES;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t p = pl + (int64_t)r * PL;
            if (p >= a.pixels) break;
#pragma unroll
            for (int i = 0; i < V; ++i) d[r][i] = rs[i] * (fmaf(d[r][i], ga[i], -m1[i]) - h[r][i] * m2[i]);
            store_out<DT>(yp + p * a.C * ES, left, d[r], a.C);
        }
    }
    if (LANES && po) {                                               // the channels' sums over the pixels, while dx is on its way out
        ss.add_up<2, V>(s, pl, k, live);
        ss.channels<2>(width, a.C, po);
    }
}

// ---- images that do not: runs of pixels ------------------------------------------------------------------------------------
// workgroup: CL lanes along the channels x PL pixel lanes over one run of pixels of one image.
//   forward: parts [n][runs][2][C] = mean and summed squared distance from it, per channel of the run
//   grad:    parts [n][runs][2][C] = sums of du h and of du
template <int DT, bool SAVED8, bool GRAD>
__global__ __launch_bounds__(256) void k_part(const NormArgs a) {
    constexpr int V = vlen(DT), ES = esize(DT);
    __shared__ float red[256 * V];
    __shared__ float tot[64 * V];
    const int CL = a.cl, PL = 256 / CL, tid = threadIdx.x, pl = tid / CL, cl = tid - pl * CL;
    const int64_t img = blockIdx.x / a.runs;
    const int run = (int)(blockIdx.x % a.runs);
    const int c = (blockIdx.y * CL + cl) * V, left = a.C - c;
    const bool live = pl < PL && left > 0;
    const int64_t p0 = run * a.run, p1 = min(p0 + a.run, a.pixels);
    float* const out = a.parts + (img * a.runs + run) * 2 * a.C;
    float s1[V], s2[V], m[V], rs[V], ga[V], be[V];
    if (GRAD && live) {
        affine<DT>(a.gamma, a.aff_f32, c, left, 1.0f, ga);
        affine<DT>(a.beta, a.aff_f32, c, left, 0.0f, be);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float* const st = a.stats + (img * a.G + min(c + i, a.C - 1) / a.per) * 2;
            m[i] = st[0];
            rs[i] = st[1];
        }
    }
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {              // forward: sums, then squared distances; grad: one pass, two joins
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!GRAD || pass == 0) s1[i] = 0.0f;
            if (pass == 0) s2[i] = 0.0f;
        }
        if (live && (!GRAD || pass == 0))
            for (int64_t p = p0 + pl; p < p1; p += PL) {
                float f[V];
                load_x<DT, SAVED8>(a, img, p, c, left, f);
                if (GRAD) {
                    float g[V];
                    load_vec<DT>(a.g + (img * a.ldgn + p * a.ldgp + c) * ES, left, g);
                    float u[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        f[i] = (f[i] - m[i]) * rs[i];
                        u[i] = fmaf(f[i], ga[i], be[i]);
                    }
                    act_slopes<V>(a.act, u, g);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        s1[i] = fmaf(g[i], f[i], s1[i]);
                        s2[i] += g[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = pass == 0 ? f[i] : f[i] - m[i];
                        s1[i] = pass == 0 ? s1[i] + d : fmaf(d, d, s1[i]);
                    }
                }
            }
        if (pl < PL)
#pragma unroll
            for (int i = 0; i < V; ++i) red[(pl * CL + cl) * V + i] = (GRAD && pass == 1) ? s2[i] : s1[i];
        __syncthreads();
        for (int i = tid; i < CL * V; i += 256) {
            float s = 0.0f;
            for (int p = 0; p < PL; ++p) s += red[p * CL * V + i];
            if (!GRAD && pass == 0) s = s / (float)(p1 - p0);
            tot[i] = s;
            const int col = blockIdx.y * CL * V + i;
            if (col < a.C) out[pass * a.C + col] = s;
        }
        __syncthreads();
        if (!GRAD && pass == 0 && pl < PL)
#pragma unroll
            for (int i = 0; i < V; ++i) m[i] = tot[cl * V + i];
    }
}

// one workgroup per (image, group): joins the runs.  forward: stats; grad: sums [n][G][2] of gamma du h and gamma du
template <bool GRAD>
__global__ __launch_bounds__(256) void k_join(const NormArgs a, int dt, float* __restrict__ out) {
    __shared__ float red[2][4];
    const int64_t img = blockIdx.x / a.G;
    const int g = (int)(blockIdx.x % a.G), tid = threadIdx.x;
    const int64_t items = (int64_t)a.runs * a.per;
    const float* const parts = a.parts + img * a.runs * 2 * a.C + g * a.per;
    auto join = [&](int slot, float v) {
        v = wave_sum(v);
        if ((tid & 63) == 0) red[slot][tid >> 6] = v;
        __syncthreads();
        return (red[slot][0] + red[slot][1]) + (red[slot][2] + red[slot][3]);
    };
    const float count = (float)a.pixels * (float)a.per;
    float s = 0.0f, q = 0.0f;
    if (GRAD) {
        for (int64_t i = tid; i < items; i += 256) {
            const int64_t r = i / a.per;
            const int c = (int)(i - r * a.per), ch = g * a.per + c;
            const float w = !a.gamma ? 1.0f : a.aff_f32 ? reinterpret_cast<const float*>(a.gamma)[ch]
                                      : dt == BS_DT_BF16 ? load1<BS_DT_BF16>(a.gamma + 2 * (int64_t)ch) : load1<BS_DT_F16>(a.gamma + 2 * (int64_t)ch);
            s = fmaf(parts[r * 2 * a.C + c], w, s);
            q = fmaf(parts[(r * 2 + 1) * a.C + c], w, q);
        }
        s = join(0, s);
        q = join(1, q);
        if (tid == 0) {
            out[blockIdx.x * 2] = s / count;
            out[blockIdx.x * 2 + 1] = q / count;
        }
        return;
    }
    for (int64_t i = tid; i < items; i += 256) {
        const int64_t r = i / a.per;
        const float cnt = (float)(min((r + 1) * a.run, a.pixels) - r * a.run);
        s = fmaf(parts[r * 2 * a.C + (i - r * a.per)], cnt, s);
    }
    const float mean = join(0, s) / count;
    for (int64_t i = tid; i < items; i += 256) {
        const int64_t r = i / a.per, c = i - r * a.per;
        const float cnt = (float)(min((r + 1) * a.run, a.pixels) - r * a.run);
        const float d = parts[r * 2 * a.C + c] - mean;
        q += fmaf(d * d, cnt, parts[(r * 2 + 1) * a.C + c]);
    }
    q = join(1, q) / count;
    if (tid == 0) {
        out[blockIdx.x * 2] = mean;
        out[blockIdx.x * 2 + 1] = 1.0f / sqrtf(q + a.eps);
    }
}

// stats known (and, for the gradient, the group means): one pass
template <int DT, bool SAVED8, bool GRAD>
__global__ __launch_bounds__(256) void k_apply(const NormArgs a, const float* __restrict__ stats, const float* __restrict__ means) {
    constexpr int V = vlen(DT), ES = esize(DT);
    const int CL = a.cl, PL = 256 / CL, tid = threadIdx.x, pl = tid / CL, cl = tid - pl * CL;
    const int64_t img = blockIdx.x / a.runs;
    const int run = (int)(blockIdx.x % a.runs);
    const int c = (blockIdx.y * CL + cl) * V, left = a.C - c;
    if (pl >= PL || left <= 0) return;
    const int64_t p0 = run * a.run, p1 = min(p0 + a.run, a.pixels);
    float m[V], rs[V], ga[V], be[V], m1[V], m2[V];
    affine<DT>(a.gamma, a.aff_f32, c, left, 1.0f, ga);
    affine<DT>(a.beta, a.aff_f32, c, left, 0.0f, be);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int64_t at = (img * a.G + min(c + i, a.C - 1) / a.per) * 2;
        m[i] = stats[at];
        rs[i] = stats[at + 1];
        m2[i] = GRAD ? means[at] : 0.0f;
        m1[i] = GRAD ? means[at + 1] : 0.0f;
    }
    for (int64_t p = p0 + pl; p < p1; p += PL) {
        float f[V], g[V];
        load_x<DT, SAVED8>(a, img, p, c, left, f);
        if (GRAD) load_vec<DT>(a.g + (img * a.ldgn + p * a.ldgp + c) * ES, left, g);
        float u[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            f[i] = (f[i] - m[i]) * rs[i];
            u[i] = fmaf(f[i], ga[i], be[i]);
        }
        if (GRAD) {
            act_slopes<V>(a.act, u, g);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = rs[i] * (fmaf(g[i], ga[i], -m1[i]) - f[i] * m2[i]);
        } else {
            act_values<DT, V>(a.act, u, f);
        }
        store_out<DT>(a.y + ((img * a.pixels + p) * a.C + c) * ES, left, f, a.C);
    }
}

// ---- which way, and how it is cut --------------------------------------------------------------------------------------------
// Both sides, in us, at (images, pixels, channels, groups); forward | gradient:
//   registers against three launches   (400, 256, 256, 32) bf16 24 and 66 | 48 and 74    (1, 256, 256, 32) f32 6.3 and 29 | 10 and 34
//     up to 1024 threads               (16, 1024, 256, 8) f32 gradient 17 and 44
//     and 256 pixel lanes, a row of the workgroup under 64 bytes beyond:  (50, 3000, 32, 8) bf16 55 and 16 | 103 and 23
//   exchanges against shared memory    (400, 256, 256, 32) bf16 24 and 39 | 48 and 70    (100, 1024, 64, 8) f32 12 and 26 | 20 and 35
//   groups of a workgroup, until a row of it is 256 bytes or it has 512 threads:
//     256 threads                      (400, 225, 60, 6) f32 16 and 11 | 24 and 19       (37, 289, 252, 28) f32 13 and 11.5 | 18 and 16.5
//     1024 threads                     (400, 256, 256, 32) bf16 32 and 24                (1, 256, 256, 32) bf16 8.2 and 6.3
struct Plan {
    bool fits, lanes;
    int pl, cl, gs, slabs, threads, lds;
    int runs;
    int64_t run;
    int cly;              // split: workgroups along the channels
};

Plan plan(int dtype, int64_t n, int64_t pixels, int C, int G, int grad) {
    Plan p = {};
    const int V = dtype == BS_DT_F32 ? 4 : 8, R = 32 / V, per = C / G, cap = 1024;
    const int64_t need = (pixels + R - 1) / R;              // pixel lanes
    const int one = (per + V - 1) / V;                      // channel lanes of a group
    p.fits = need <= 256 && need * one <= cap;             // (longer columns would leave a row of the workgroup under 64 bytes)
    if (p.fits) {
        auto pow2 = [](int64_t v) { return (v & (v - 1)) == 0; };
        int64_t up = 1;
        while (up < need) up *= 2;
        p.lanes = per % V == 0 && pow2(one) && one <= 64 && up * one <= cap;
        p.pl = (int)(p.lanes ? up : need);
        int gs = 1;
        auto lanes_of = [&](int g) { return (g * per + V - 1) / V; };
        while (gs < G && lanes_of(gs) < 16) {
            const int next = p.lanes ? 2 * gs : gs + 1;
            if (next > G || lanes_of(next) * p.pl > 512) break;
            gs = next;
        }
        p.gs = gs;
        p.cl = lanes_of(gs);
        p.slabs = (G + gs - 1) / gs;
        p.threads = (p.pl * p.cl + 63) / 64 * 64;
        const int ch = p.cl * V, Q = p.pl / V > 1 ? p.pl / V : 1;
        p.lds = ((p.lanes && !grad ? 0 : (grad ? 2 : 1) * (p.pl + Q) * ch) + 32 * gs + (grad ? ch : 0)) * 4;
        if (p.lds <= 160 * 1024) return p;
        p = {};                                             // (over 1020 lanes of 16-bit channels to a pixel lane: the gradient's sums)
    }
    const int chunks = (C + V - 1) / V;
    p.cl = chunks < 32 ? chunks : 32;
    p.cly = (chunks + p.cl - 1) / p.cl;
    p.run = 256;                                        // pixels of a run, more when there would be over 1024 runs
    while ((pixels + p.run - 1) / p.run > 1024) p.run *= 2;
    p.runs = (int)((pixels + p.run - 1) / p.run);
    return p;
}

int bad_norm(int dtype, int64_t n, int64_t pixels, int channels, int groups, int act) {
    return bad_type(dtype) || n < 0 || n > MAX_ROWS || pixels < 0 || pixels > MAX_ROWS || channels < 1 || channels > (1 << 20) || n > MAX_ROWS / channels || groups < 1 ||
           channels % groups || act < BS_ACT_NONE || act > BS_ACT_GELU;
}

void fill(NormArgs* a, const Plan& p) {
    a->pl = p.pl; a->cl = p.cl; a->gs = p.gs; a->slabs = p.slabs; a->runs = p.runs; a->run = p.run;
}

}  // namespace

extern "C" {

int64_t bs_group_norm_workspace(int dtype, int64_t n, int64_t pixels, int channels, int groups, int grad) {
    if (bad_norm(dtype, n, pixels, channels, groups, 0)) return BS_EINVAL;
    const Plan p = plan(dtype, n, pixels, channels, groups, grad);
    if (p.fits) return grad ? n * 2 * channels * 4 : 0;
    return (n * p.runs * 2 * channels + n * groups * 2) * 4;
}

int bs_group_norm_act(const void* x, int64_t ldn, int64_t ldp, const void* gamma, const void* beta, int affine_dtype, float eps,
                      int act, int dtype, int64_t n, int64_t pixels, int channels, int groups, void* y, float* stats,
                      void* workspace, int64_t workspace_bytes, void* stream) {
    if (bad_norm(dtype, n, pixels, channels, groups, act) || !(eps >= 0.0f)) return BS_EINVAL;
    if (n == 0 || pixels == 0) return BS_OK;
    if (!x || !y || ldp < channels || ldn < 0) return BS_EINVAL;
    if ((gamma || beta) && affine_dtype != BS_DT_F32 && affine_dtype != dtype) return BS_EINVAL;
    const Plan p = plan(dtype, n, pixels, channels, groups, 0);
    const int64_t need = bs_group_norm_workspace(dtype, n, pixels, channels, groups, 0);
    if (bad_workspace(workspace, workspace_bytes, need)) return BS_EINVAL;
    NormArgs a = {};
    a.x = (const char*)x; a.ldn = ldn; a.ldp = ldp; a.gamma = (const char*)gamma; a.beta = (const char*)beta;
    a.aff_f32 = affine_dtype == BS_DT_F32; a.act = act; a.eps = eps; a.n = n; a.pixels = pixels;
    a.C = channels; a.G = groups; a.per = channels / groups; a.y = (char*)y; a.stats = stats;
    fill(&a, p);
    hipStream_t st = rows_stream(stream);
    const int64_t blocks = p.fits ? (n * p.slabs + 7) / 8 * 8 : n * p.runs;
    if (p.fits ? too_many(blocks, p.threads) : too_many(blocks, 256) || too_many(n * groups, 256)) return BS_EINVAL;
    if (p.fits) {
#define GO(DT) do { if (p.lanes) hipLaunchKernelGGL((k_norm<DT, true>), dim3((unsigned)blocks), dim3(p.threads), p.lds, st, a); \
                    else hipLaunchKernelGGL((k_norm<DT, false>), dim3((unsigned)blocks), dim3(p.threads), p.lds, st, a); } while (0)
        if (dtype == BS_DT_F32) GO(BS_DT_F32);
        else if (dtype == BS_DT_BF16) GO(BS_DT_BF16);
        else GO(BS_DT_F16);
#undef GO
        return rows_rc();
    }
    a.parts = (float*)workspace;
    float* const own = a.parts + n * p.runs * 2 * channels;
    float* const st_out = stats ? stats : own;
    const dim3 grid((unsigned)blocks, (unsigned)p.cly);
#define GO(DT) do { hipLaunchKernelGGL((k_part<DT, false, false>), grid, dim3(256), 0, st, a); \
                    hipLaunchKernelGGL(k_join<false>, dim3((unsigned)(n * groups)), dim3(256), 0, st, a, dtype, st_out); \
                    hipLaunchKernelGGL((k_apply<DT, false, false>), grid, dim3(256), 0, st, a, (const float*)st_out, (const float*)nullptr); } while (0)
    if (dtype == BS_DT_F32) GO(BS_DT_F32);
    else if (dtype == BS_DT_BF16) GO(BS_DT_BF16);
    else GO(BS_DT_F16);
#undef GO
    return rows_rc();
}

int bs_group_norm_act_grad(const void* g, int64_t ldgn, int64_t ldgp, const void* x, const int8_t* x_exps, int64_t ldn, int64_t ldp,
                           const float* stats, const void* gamma, const void* beta, int affine_dtype, int act, int dtype, int64_t n,
                           int64_t pixels, int channels, int groups, void* dx, float* dgamma, float* dbeta, void* workspace,
                           int64_t workspace_bytes, void* stream) {
    if (bad_norm(dtype, n, pixels, channels, groups, act)) return BS_EINVAL;
    hipStream_t st = rows_stream(stream);
    const dim3 cols((unsigned)((2 * (int64_t)channels + 31) / 32));
    if (n == 0 || pixels == 0) {
        if (dgamma || dbeta) hipLaunchKernelGGL(k_sum_columns, cols, dim3(1024), 0, st, (const float*)nullptr, (int64_t)0, 2 * channels, channels, dgamma, dbeta);
        return rows_rc();
    }
    if (!g || !x || !stats || !dx || ldgp < channels || ldgn < 0 || (!x_exps && (ldp < channels || ldn < 0))) return BS_EINVAL;
    if ((gamma || beta) && affine_dtype != BS_DT_F32 && affine_dtype != dtype) return BS_EINVAL;
    const Plan p = plan(dtype, n, pixels, channels, groups, 1);
    const int64_t need = bs_group_norm_workspace(dtype, n, pixels, channels, groups, 1);
    if (bad_workspace(workspace, workspace_bytes, need)) return BS_EINVAL;
    NormArgs a = {};
    a.g = (const char*)g; a.ldgn = ldgn; a.ldgp = ldgp;
    a.x = (const char*)x; a.exps = x_exps; a.ldn = ldn; a.ldp = ldp; a.nb = (channels + P8_BLOCK - 1) / P8_BLOCK;
    a.gamma = (const char*)gamma; a.beta = (const char*)beta; a.aff_f32 = affine_dtype == BS_DT_F32; a.act = act;
    a.n = n; a.pixels = pixels; a.C = channels; a.G = groups; a.per = channels / groups;
    a.y = (char*)dx; a.stats = (float*)stats; a.parts = (float*)workspace;
    fill(&a, p);
    const int64_t blocks = p.fits ? (n * p.slabs + 7) / 8 * 8 : n * p.runs;
    if (p.fits ? too_many(blocks, p.threads) : too_many(blocks, 256) || too_many(n * groups, 256)) return BS_EINVAL;
    if (p.fits) {
        if (!dgamma && !dbeta) a.parts = nullptr;
        // Builds by the registers that a number of threads leaves, in us at (images, pixels, channels, groups), bf16.  Exchanges: 128,
        // which lets two workgroups of 512 threads share a compute unit, at the cost of a few spilled: (400, 256, 256, 32) 48, 61 with
        // the 131 that it would take; (1, 256, 256, 32) 11.6 and 10.4.  Shared memory: 128 spill 50 to 90, (37, 289, 252, 28) 25, 16
        // with 153; only where 1024 threads leave no more.
#define FIT_T(DT, P8, L, T) hipLaunchKernelGGL((k_norm_grad<DT, P8, L, T>), dim3((unsigned)blocks), dim3(p.threads), p.lds, st, a)
#define FIT(DT, P8) do { if (p.lanes) FIT_T(DT, P8, true, 1024); else if (p.threads > 512) FIT_T(DT, P8, false, 1024); else FIT_T(DT, P8, false, 512); } while (0)
#define GO(DT) do { if (x_exps) FIT(DT, true); else FIT(DT, false); } while (0)
        if (dtype == BS_DT_F32) GO(BS_DT_F32);
        else if (dtype == BS_DT_BF16) GO(BS_DT_BF16);
        else GO(BS_DT_F16);
#undef GO
#undef FIT
#undef FIT_T
    } else {
        float* const means = a.parts + n * p.runs * 2 * channels;
        const dim3 grid((unsigned)blocks, (unsigned)p.cly);
#define STEPS(DT, P8) do { hipLaunchKernelGGL((k_part<DT, P8, true>), grid, dim3(256), 0, st, a); \
                           hipLaunchKernelGGL(k_join<true>, dim3((unsigned)(n * groups)), dim3(256), 0, st, a, dtype, means); \
                           hipLaunchKernelGGL((k_apply<DT, P8, true>), grid, dim3(256), 0, st, a, stats, (const float*)means); } while (0)
#define GO(DT) do { if (x_exps) STEPS(DT, true); else STEPS(DT, false); } while (0)
        if (dtype == BS_DT_F32) GO(BS_DT_F32);
        else if (dtype == BS_DT_BF16) GO(BS_DT_BF16);
        else GO(BS_DT_F16);
#undef GO
#undef STEPS
    }
    if (dgamma || dbeta)
        hipLaunchKernelGGL(k_sum_columns, cols, dim3(1024), 0, st, (const float*)workspace, p.fits ? n : n * p.runs, 2 * channels, channels, dgamma, dbeta);
    return rows_rc();
}

}  // extern "C"
