// Group norm with an activation over channels-last arrays [n, rows, channels] (rows = pixels of a window), forward and backward, as an
// operator of its own: the layer src/train/src/model.py:100-121 applies, on the channels-last features the library exports
// (ttc_forward_taps).  model.hip keeps the planar fused form of the fixed graph.
//
//   m, v = mean, biased variance over (rows, channels of the group);  rstd = 1 / sqrt(v + eps)
//   xh = (x - m) rstd,  z = gamma xh + beta,  y = act(z)
//   dz = dy act'(z);  dbeta = sum dz;  dgamma = sum dz xh;  M = rows * channels / groups
//   dx = rstd (gamma dz - sum_g(gamma dz) / M - xh sum_g(gamma dz xh) / M)
//
// What bounds it: memory, and for 16-bit types with an activation nearly as much the vector ALU.  The statistics need the whole sample before the
// first output.  A sample (or some whole groups of it) that fits the registers of one workgroup is read ONCE, in one launch (k_gn_resident*); a larger
// one is read twice, by two launches.  (Pairs of launches over a few samples at a time, so that the second read finds the first's data in the 256 MB
// last-level cache, measured slower: 36 x 172 x 172 x 64 fp32 in three parts 172 us against 154.)
// A thread owns one vector of channels (up to 16 bytes) and walks rows: the inner loop knows no groups, and a row is read as whole cache lines.
// Numerics: a thread sums (x - x0) and (x - x0)^2 about its own first row in 32 bits, folds into 64-bit sums every 128 values; the forward sums across
// threads are 64-bit, the backward ones 32-bit runs of at most 512 rows (a resident sample: 32-bit trees) joined in 64 bits; the order is fixed (no atomics).
#include <algorithm>

#include "layers_common.h"

namespace {
using namespace layers;

constexpr int NT = 256;             // threads of the streaming kernels
constexpr int RT = 1024, RU = 4;    // threads and vectors per thread of the resident ones
constexpr int SU = 8;                   // loads of the forward sums in flight
constexpr int FOLD = 128;           // values summed in 32 bits before they are folded into the 64-bit sums
constexpr int RUN = 512;            // rows a thread of the backward sums adds in 32 bits: longer ones get more splits

struct NormArgs {
    const void* x; const void* dy;
    const float* gamma; const float* beta;
    void* y;                        // forward: y; backward: dx (contiguous)
    const float* stats_in;          // backward: [n][G][2]
    float* stats;                   // forward, optional: [n][G][2]
    double* part;                   // forward partial sums [n][slots][G][2]
    float* cpart;                   // backward partial sums [n][slots][2][C]
    float* csum;                    // backward sums per sample [n][2][C]
    float* coef;                    // backward [n][G][2]: sum_g(gamma dz) / M, sum_g(gamma dz xh) / M
    float* dgamma; float* dbeta;
    long rows, sn, pitch, dsn, dpitch;   // element strides of x (sample, row) and dy
    int n, C, G, cpg, act;
    int cols, rpb;                  // vector columns per block, rows per block step
    int ctiles;                     // column tiles (blockIdx.z)
    int splits; long rows_per;      // row splits (blockIdx.x) of a sample
    float eps;
};

__device__ __forceinline__ float gam(const NormArgs& a, int c) { return a.gamma ? a.gamma[c] : 1.0f; }
__device__ __forceinline__ float bet(const NormArgs& a, int c) { return a.beta ? a.beta[c] : 0.0f; }

// sum of the slots of one (sample, group) by one wave, the same order every time
__device__ __forceinline__ void wave_sum2(double& s, double& q) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) { s += __shfl_xor(s, m); q += __shfl_xor(q, m); }
}
__device__ __forceinline__ void mean_rstd(double s, double q, double count, float eps, float* mean, float* rstd) {
    const double m = s / count;
    double var = q / count - m * m;
    if (var < 0.0) var = 0.0;                      // rounding only; NaN stays NaN
    *mean = (float)m;
    *rstd = (float)(1.0 / sqrt(var + (double)eps));
}

// ---- forward, pass 1: partial sums per (sample, slot, group) ------------------------------------------------------------------------
// Bound by reading x: 36 x 172 x 172 x 64 fp32 (273 MB) 66 us = 4.1 TB/s, bf16 22 us (6 TB/s, from the last-level cache).
// UNI: a thread's V channels share a group, so one pair of sums (about the thread's first element) serves them all
template <class T, int V, bool UNI>
__global__ __launch_bounds__(NT) void k_gn_sums(NormArgs a) {
    constexpr int NS = UNI ? 1 : V;                // sums a thread keeps
    extern __shared__ double sm[];                 // [rpb][cols * NS][2], row 0 becomes the columns' sums
    const int tid = threadIdx.x, col = tid % a.cols, rl = tid / a.cols;
    const int c0 = (blockIdx.z * a.cols + col) * V;
    const long n = blockIdx.y;
    const long r0 = blockIdx.x * a.rows_per, r1 = min(r0 + a.rows_per, a.rows);
    const int width = a.cols * NS;
    double s[NS], q[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] = q[i] = 0.0;
    long r = r0 + rl;
    if (rl < a.rpb && c0 < a.C && r < r1) {
        const T* x = (const T*)a.x + n * a.sn + c0;
        float x0[V];
        load_vec<T, V>(x + r * a.pitch, x0);
        if (UNI) {
#pragma unroll
            for (int i = 1; i < V; ++i) x0[i] = x0[0];
        }
        double cnt = 0.0;
        while (r < r1) {
            float f[NS], g[NS];
#pragma unroll
            for (int i = 0; i < NS; ++i) f[i] = g[i] = 0.0f;
            auto add = [&](const float (&v)[V]) {
#pragma unroll
                for (int i = 0; i < V; ++i) { const float d = v[i] - x0[i]; f[i % NS] += d; g[i % NS] += d * d; }
            };
            int k = 0;
            constexpr int ROWS = FOLD / (V / NS);
            for (; k + SU <= ROWS && r + (SU - 1) * a.rpb < r1; k += SU, r += SU * a.rpb) {
                float v[SU][V];
#pragma unroll
                for (int u = 0; u < SU; ++u) load_vec<T, V>(x + (r + u * a.rpb) * a.pitch, v[u]);
#pragma unroll
                for (int u = 0; u < SU; ++u) add(v[u]);
            }
            for (; k < ROWS && r < r1; ++k, r += a.rpb) {
                float v[V];
                load_vec<T, V>(x + r * a.pitch, v);
                add(v);
            }
            cnt += k * (V / NS);
#pragma unroll
            for (int i = 0; i < NS; ++i) { s[i] += f[i]; q[i] += g[i]; }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {             // about x0 -> about 0
            const double c = x0[i];
            q[i] += 2.0 * c * s[i] + cnt * c * c;
            s[i] += cnt * c;
        }
    }
    if (rl < a.rpb) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            double* d = sm + ((long)rl * width + col * NS + i) * 2;
            d[0] = s[i]; d[1] = q[i];
        }
    }
    __syncthreads();
    for (int c = tid; c < width; c += NT) {        // rows of the block -> columns
        double t0 = 0.0, t1 = 0.0;
        for (int k = 0; k < a.rpb; ++k) { t0 += sm[((long)k * width + c) * 2]; t1 += sm[((long)k * width + c) * 2 + 1]; }
        sm[2 * c] = t0; sm[2 * c + 1] = t1;        // row 0's own slot, read by this thread alone
    }
    __syncthreads();
    const int per = UNI ? a.cpg / V : a.cpg;       // columns of a group
    const int lo = blockIdx.z * width, hi = min(lo + width, a.C / (V / NS));
    double* out = a.part + ((n * a.splits + blockIdx.x) * a.ctiles + blockIdx.z) * (2L * a.G);
    for (int g = tid; g < a.G; g += NT) {          // columns -> groups; a group of another column tile adds nothing here
        double t0 = 0.0, t1 = 0.0;
        for (int c = max(lo, g * per); c < min(hi, (g + 1) * per); ++c) { t0 += sm[2 * (c - lo)]; t1 += sm[2 * (c - lo) + 1]; }
        out[2 * g] = t0; out[2 * g + 1] = t1;
    }
}

// what a thread needs of its V channels.  UNI: they share a group (channels / groups is a multiple of V): one mean, not V -- registers are occupancy.
template <int V, bool UNI>
struct Chan {
    float mean[UNI ? 1 : V], rstd[UNI ? 1 : V], sc[V], sh[V];       // z = (x - mean) sc + sh
    __device__ __forceinline__ void get(const NormArgs& a, const float* stats, int c0, int g0) {       // stats: (mean, rstd) of groups g0 ..
#pragma unroll
        for (int i = 0; i < (UNI ? 1 : V); ++i) {
            const int g = (c0 + i) / a.cpg - g0;
            mean[i] = stats[2 * g]; rstd[i] = stats[2 * g + 1];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) { sc[i] = rstd[UNI ? 0 : i] * gam(a, c0 + i); sh[i] = bet(a, c0 + i); }
    }
    // (x - mean) first: exact where x is near the mean, which folding the mean into the shift would lose
    __device__ __forceinline__ void center(float (&x)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] -= mean[UNI ? 0 : i];
    }
    __device__ __forceinline__ void out(float (&x)[V], int act) const {
        center(x);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = x[i] * sc[i] + sh[i];
        act_vec<V>(x, act);
    }
    // x -> x - mean, dy -> dz = dy act'(z)
    __device__ __forceinline__ void slope(float (&x)[V], float (&dy)[V], int act) const {
        center(x);
        if (act == TTC_ACT_NONE) return;
        float z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = x[i] * sc[i] + sh[i];
        slope_vec<V>(dy, z, act);
    }
};

// ---- forward, pass 2: y = act(gamma xh + beta) ----------------------------------------------------------------------------------------
// Bound by memory: 36 x 172 x 172 x 64 fp32 swish 88 us = 6.2 TB/s read and written, bf16 49 us = 5.6; 36 x 84 x 84 x 128 bf16 sigmoid 27 us.
template <class T, int V, bool UNI>
__global__ __launch_bounds__(NT) void k_gn_apply(NormArgs a) {
    extern __shared__ float sg[];                  // [G][2]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long n = a.n - 1 - blockIdx.y;   // pass 1 ended on the last sample: walk the samples back
    const int slots = a.splits * a.ctiles;
    for (int g = wave; g < a.G; g += NT / 64) {
        double s = 0.0, q = 0.0;
        for (int i = lane; i < slots; i += 64) {
            const double* p = a.part + ((n * slots + i) * a.G + g) * 2;
            s += p[0]; q += p[1];
        }
        wave_sum2(s, q);
        if (lane == 0) {
            mean_rstd(s, q, (double)a.rows * a.cpg, a.eps, &sg[2 * g], &sg[2 * g + 1]);
            if (a.stats && blockIdx.x == 0 && blockIdx.z == 0) {
                a.stats[(n * a.G + g) * 2] = sg[2 * g];
                a.stats[(n * a.G + g) * 2 + 1] = sg[2 * g + 1];
            }
        }
    }
    __syncthreads();
    const int col = tid % a.cols, rl = tid / a.cols, c0 = (blockIdx.z * a.cols + col) * V;
    if (rl >= a.rpb || c0 >= a.C) return;
    Chan<V, UNI> ch;
    ch.get(a, sg, c0, 0);
    const long r0 = blockIdx.x * a.rows_per, r1 = min(r0 + a.rows_per, a.rows);
    const T* x = (const T*)a.x + n * a.sn + c0;
    T* y = (T*)a.y + n * a.rows * a.C + c0;
    long r = r0 + rl;
    for (; r + 3 * a.rpb < r1; r += 4 * a.rpb) {
        float v[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_vec<T, V>(x + (r + u * a.rpb) * a.pitch, v[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            ch.out(v[u], a.act);
            store_vec<T, V>(y + (r + u * a.rpb) * a.C, v[u]);
        }
    }
    for (; r < r1; r += a.rpb) {
        float v[V];
        load_vec<T, V>(x + r * a.pitch, v);
        ch.out(v, a.act);
        store_vec<T, V>(y + r * a.C, v);
    }
}

// ---- backward, pass 1: sum dz, sum dz xh per (sample, slot, channel) -----------------------------------------------------------------
// 36 x 172 x 172 x 64 bf16 swish: 59 us = 4.6 TB/s of x and dy; the slope costs about 36 us of vector ALU under it.
template <class T, int V, bool UNI>
__global__ __launch_bounds__(NT) void k_gn_bwd_sums(NormArgs a) {
    extern __shared__ float sf[];                  // [rpb][cols * V][2]
    const int tid = threadIdx.x, col = tid % a.cols, rl = tid / a.cols;
    const int c0 = (blockIdx.z * a.cols + col) * V;
    const long n = blockIdx.y;
    const long r0 = blockIdx.x * a.rows_per, r1 = min(r0 + a.rows_per, a.rows);
    const int width = a.cols * V;
    float sa[V], sb[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.0f;
    if (rl < a.rpb && c0 < a.C) {
        Chan<V, UNI> ch;
        ch.get(a, a.stats_in + n * a.G * 2, c0, 0);
        const T* x = (const T*)a.x + n * a.sn + c0;
        const T* dy = (const T*)a.dy + n * a.dsn + c0;
        auto add = [&](float (&xv)[V], float (&dv)[V]) {
            ch.slope(xv, dv, a.act);
#pragma unroll
            for (int i = 0; i < V; ++i) { sa[i] += dv[i]; sb[i] += dv[i] * xv[i]; }
        };
        long r = r0 + rl;
        for (; r + a.rpb < r1; r += 2 * a.rpb) {
            float xv[2][V], dv[2][V];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                load_vec<T, V>(x + (r + u * a.rpb) * a.pitch, xv[u]);
                load_vec<T, V>(dy + (r + u * a.rpb) * a.dpitch, dv[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) add(xv[u], dv[u]);
        }
        for (; r < r1; r += a.rpb) {
            float xv[V], dv[V];
            load_vec<T, V>(x + r * a.pitch, xv);
            load_vec<T, V>(dy + r * a.dpitch, dv);
            add(xv, dv);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sb[i] *= ch.rstd[UNI ? 0 : i];
    }
    if (rl < a.rpb) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float* d = sf + (rl * width + col * V + i) * 2;
            d[0] = sa[i]; d[1] = sb[i];
        }
    }
    __syncthreads();
    float* out = a.cpart + (n * a.splits + blockIdx.x) * 2L * a.C;
    for (int c = tid; c < width; c += NT) {
        const int cc = blockIdx.z * width + c;
        if (cc >= a.C) break;
        double t0 = 0.0, t1 = 0.0;
        for (int r = 0; r < a.rpb; ++r) { t0 += sf[(r * width + c) * 2]; t1 += sf[(r * width + c) * 2 + 1]; }
        out[cc] = (float)t0; out[a.C + cc] = (float)t1;
    }
}

// ---- backward, between: slots -> channels of a sample, and the two group means --------------------------------------------------------
__global__ __launch_bounds__(RT) void k_gn_bwd_mid(NormArgs a) {
    extern __shared__ float sm2[];                 // [lanes][2C] partial sums, then [2C] times gamma
    const long n = blockIdx.x;
    const int w = 2 * a.C, lanes = max(1, RT / w);
    const float* p = a.cpart + n * a.splits * (long)w;
    for (int i = threadIdx.x; i < w * lanes; i += RT) {
        const int c = i % w;
        double t = 0.0;
#pragma unroll 4
        for (int k = i / w; k < a.splits; k += lanes) t += p[(long)k * w + c];
        sm2[i] = (float)t;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < w; c += RT) {
        double t = 0.0;
        for (int l = 0; l < lanes; ++l) t += sm2[l * w + c];
        a.csum[n * w + c] = (float)t;
        sm2[c] = (float)t * gam(a, c < a.C ? c : c - a.C);
    }
    __syncthreads();
    const double m = (double)a.rows * a.cpg;
    for (int g = threadIdx.x; g < 2 * a.G; g += RT) {
        const float* s = sm2 + (g < a.G ? 0 : a.C) + (g < a.G ? g : g - a.G) * a.cpg;
        double t = 0.0;
        for (int c = 0; c < a.cpg; ++c) t += s[c];
        a.coef[(n * a.G + (g < a.G ? g : g - a.G)) * 2 + (g < a.G ? 0 : 1)] = (float)(t / m);
    }
}

// dgamma, dbeta: channels summed over the samples, 16 channels a step, 16 lanes each
__device__ void gn_param_grads(const NormArgs& a, int first, int step) {
    __shared__ double red[16][17][2];
    const int ch = threadIdx.x & 15, l = threadIdx.x >> 4;
    for (int c0 = first * 16; c0 < a.C; c0 += step * 16) {
        const int c = c0 + ch;
        double t0 = 0.0, t1 = 0.0;
        if (c < a.C)
            for (long n = l; n < a.n; n += NT / 16) { t0 += a.csum[n * 2 * a.C + c]; t1 += a.csum[n * 2 * a.C + a.C + c]; }
        red[l][ch][0] = t0; red[l][ch][1] = t1;
        __syncthreads();
        if (l == 0 && c < a.C) {
            for (int i = 1; i < NT / 16; ++i) { t0 += red[i][ch][0]; t1 += red[i][ch][1]; }
            if (a.dbeta) a.dbeta[c] = (float)t0;
            if (a.dgamma) a.dgamma[c] = (float)t1;
        }
        __syncthreads();
    }
}
__global__ __launch_bounds__(NT) void k_gn_param_grads(NormArgs a) { gn_param_grads(a, blockIdx.x, gridDim.x); }

// dx = rstd gamma dz - rstd k1 - (x - mean) rstd^2 k2
template <int V, bool UNI>
struct ChanBwd : Chan<V, UNI> {
    float q0[UNI ? 1 : V], q1[UNI ? 1 : V];
    __device__ __forceinline__ void get_coef(const NormArgs& a, const float* coef, int c0, int g0) {
#pragma unroll
        for (int i = 0; i < (UNI ? 1 : V); ++i) {
            const int g = (c0 + i) / a.cpg - g0;
            q0[i] = this->rstd[i] * coef[2 * g]; q1[i] = this->rstd[i] * this->rstd[i] * coef[2 * g + 1];
        }
    }
    __device__ __forceinline__ void dx(const float (&xc)[V], float (&dz)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) dz[i] = this->sc[i] * dz[i] - (q1[UNI ? 0 : i] * xc[i] + q0[UNI ? 0 : i]);
    }
};

// ---- backward, pass 2: dx, and in blocks of their own (the last of every sample's row) the parameters' gradients --------------------------
// 36 x 172 x 172 x 64 bf16 swish: 77 us = 5.3 TB/s.
template <class T, int V, bool UNI>
__global__ __launch_bounds__(NT) void k_gn_bwd_apply(NormArgs a) {
    if ((int)blockIdx.x == a.splits) {
        if (blockIdx.z == 0) gn_param_grads(a, blockIdx.y, gridDim.y);
        return;
    }
    const int tid = threadIdx.x, col = tid % a.cols, rl = tid / a.cols, c0 = (blockIdx.z * a.cols + col) * V;
    const long n = a.n - 1 - blockIdx.y;   // back to front, as in the forward's second pass
    if (rl >= a.rpb || c0 >= a.C) return;
    ChanBwd<V, UNI> ch;
    ch.get(a, a.stats_in + n * a.G * 2, c0, 0);
    ch.get_coef(a, a.coef + n * a.G * 2, c0, 0);
    const long r0 = blockIdx.x * a.rows_per, r1 = min(r0 + a.rows_per, a.rows);
    const T* x = (const T*)a.x + n * a.sn + c0;
    const T* dy = (const T*)a.dy + n * a.dsn + c0;
    T* dx = (T*)a.y + n * a.rows * a.C + c0;
    long r = r0 + rl;
    for (; r + a.rpb < r1; r += 2 * a.rpb) {
        float xv[2][V], dv[2][V];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            load_vec<T, V>(x + (r + u * a.rpb) * a.pitch, xv[u]);
            load_vec<T, V>(dy + (r + u * a.rpb) * a.dpitch, dv[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            ch.slope(xv[u], dv[u], a.act);
            ch.dx(xv[u], dv[u]);
            store_vec<T, V>(dx + (r + u * a.rpb) * a.C, dv[u]);
        }
    }
    for (; r < r1; r += a.rpb) {
        float xv[V], dv[V];
        load_vec<T, V>(x + r * a.pitch, xv);
        load_vec<T, V>(dy + r * a.dpitch, dv);
        ch.slope(xv, dv, a.act);
        ch.dx(xv, dv);
        store_vec<T, V>(dx + r * a.C, dv);
    }
}

// ---- one launch: a workgroup holds whole groups of a sample ------------------------------------------------------------------------------
// blockIdx.x = slab of a.cols * V channels (whole groups, V divides channels / groups), blockIdx.y = sample; RU vectors a thread stay in registers
// as stored (with 8 vectors a thread 5 x 61 x 47 x 40 fp16 takes 14.6 us instead of 10.5: too few workgroups share the chip).  Bound by latency.
// 14 x 14 x 64 fp32: 4.4 us against 7.8 by two launches; norm_resident has both sides of more sizes.
template <class T, int V>
struct Held {
    static constexpr int W = V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1;
    unsigned w[W];
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(w, p, V * sizeof(T)); }
    // the compiler would rather keep a first pass's 32-bit values (twice the registers of the stored ones: it spills) than convert again
    __device__ __forceinline__ void again() {
#pragma unroll
        for (int i = 0; i < W; ++i) asm volatile("" : "+v"(w[i]));
    }
    __device__ __forceinline__ void get(float (&v)[V]) const {
        T t[V];
        __builtin_memcpy(t, w, V * sizeof(T));
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)t[i];
    }
};

template <class T, int V>
__global__ __launch_bounds__(RT) void k_gn_resident(NormArgs a) {
    __shared__ double red[RT][2];
    __shared__ float sg[2 * RT];                   // (mean, rstd) of the slab's groups: at most one per column
    const int tid = threadIdx.x, col = tid % a.cols, rl = tid / a.cols, cg = a.cpg / V;      // cg: columns of a group
    const long n = blockIdx.y;
    const int cs = blockIdx.x * a.cols * V, c0 = cs + col * V, ng = min(a.cols * V, a.C - cs) / a.cpg;
    const bool on = rl < a.rpb && c0 < a.C;
    const T* x = (const T*)a.x + n * a.sn + c0;
    const int rows = (int)a.rows;
    Held<T, V> h[RU];
#pragma unroll
    for (int u = 0; u < RU; ++u) if (on && rl + u * a.rpb < rows) h[u].load(x + (long)(rl + u * a.rpb) * a.pitch);
    double s = 0.0, q = 0.0;
    if (on && rl < rows) {                         // the thread's channels share a group: one shift, its first element
        float v[V], f = 0.0f, g = 0.0f;
        h[0].get(v);
        const float x0 = v[0];
        int k = 0;
#pragma unroll
        for (int u = 0; u < RU; ++u) {
            if (rl + u * a.rpb < rows) {
                h[u].get(v);
#pragma unroll
                for (int i = 0; i < V; ++i) { const float d = v[i] - x0; f += d; g += d * d; }
                k += V;
            }
        }
        s = k * (double)x0 + f;
        q = (double)g + 2.0 * x0 * f + k * (double)x0 * x0;
    }
    red[tid][0] = s; red[tid][1] = q;
    __syncthreads();
    for (int g = tid >> 6; g < ng; g += blockDim.x >> 6) {
        double t0 = 0.0, t1 = 0.0;
        for (int e = tid & 63; e < cg * a.rpb; e += 64) {
            const int i = e / cg * a.cols + g * cg + e % cg;
            t0 += red[i][0]; t1 += red[i][1];
        }
        wave_sum2(t0, t1);
        if ((tid & 63) == 0) {
            mean_rstd(t0, t1, (double)a.rows * a.cpg, a.eps, &sg[2 * g], &sg[2 * g + 1]);
            if (a.stats) {
                float* st = a.stats + (n * a.G + cs / a.cpg + g) * 2;
                st[0] = sg[2 * g]; st[1] = sg[2 * g + 1];
            }
        }
    }
    __syncthreads();
    if (!on) return;
    Chan<V, true> ch;
    ch.get(a, sg, c0, cs / a.cpg);
    T* y = (T*)a.y + n * a.rows * a.C + c0;
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int r = rl + u * a.rpb;
        if (r < rows) {
            float v[V];
            h[u].again();
            h[u].get(v);
            ch.out(v, a.act);
            store_vec<T, V>(y + (long)r * a.C, v);
        }
    }
}

// the same for the backward pass: x is held, dy read again for dx (holding both spills: its second read comes from the L2); the sums of a channel over
// the rows are a 32-bit tree in LDS.  direct: one sample, so its sums ARE the parameters' gradients
template <class T, int V>
__global__ __launch_bounds__(RT) void k_gn_resident_bwd(NormArgs a, int direct) {
    extern __shared__ float sf[];                  // [rpb][cols * V][2], row 0 becomes the channels' sums, row 1 the groups'
    const int tid = threadIdx.x, col = tid % a.cols, rl = tid / a.cols, width = a.cols * V;
    const long n = blockIdx.y;
    const int cs = blockIdx.x * width, c0 = cs + col * V, nc = min(width, a.C - cs), ng = nc / a.cpg, g0 = cs / a.cpg;
    const bool on = rl < a.rpb && c0 < a.C;
    const T* x = (const T*)a.x + n * a.sn + c0;
    const T* dy = (const T*)a.dy + n * a.dsn + c0;
    const int rows = (int)a.rows;
    Held<T, V> hx[RU];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        if (on && rl + u * a.rpb < rows) hx[u].load(x + (long)(rl + u * a.rpb) * a.pitch);
    }
    ChanBwd<V, true> ch;
    if (on) ch.get(a, a.stats_in + (n * a.G + g0) * 2, c0, g0);
    float sa[V], sb[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.0f;
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int r = rl + u * a.rpb;
        if (on && r < rows) {
            float xv[V], dv[V];
            load_vec<T, V>(dy + (long)r * a.dpitch, dv);
            hx[u].get(xv);
            ch.slope(xv, dv, a.act);
#pragma unroll
            for (int i = 0; i < V; ++i) { sa[i] += dv[i]; sb[i] += dv[i] * xv[i]; }
        }
    }
    if (rl < a.rpb) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float* d = sf + (rl * width + col * V + i) * 2;
            d[0] = sa[i]; d[1] = on ? sb[i] * ch.rstd[0] : 0.0f;
        }
    }
    int top = 1;
    while (top < a.rpb) top *= 2;
    for (int half = top / 2; half; half /= 2) {
        __syncthreads();
        const int cnt = max(0, min(half, a.rpb - half)) * width * 2;
        for (int i = tid; i < cnt; i += blockDim.x) sf[i] += sf[half * width * 2 + i];
    }
    __syncthreads();
    for (int c = tid; c < nc; c += blockDim.x) {
        if (direct) {
            if (a.dbeta) a.dbeta[cs + c] = sf[2 * c];
            if (a.dgamma) a.dgamma[cs + c] = sf[2 * c + 1];
        } else {
            a.csum[n * 2 * a.C + cs + c] = sf[2 * c];
            a.csum[n * 2 * a.C + a.C + cs + c] = sf[2 * c + 1];
        }
    }
    if (!a.y) return;
    float* sk = sf + width * 2;
    for (int g = tid; g < 2 * ng; g += blockDim.x) {
        const int j = g >> 1, w = g & 1;
        double t = 0.0;
        for (int c = j * a.cpg; c < (j + 1) * a.cpg; ++c) t += (double)(sf[2 * c + w] * gam(a, cs + c));
        sk[g] = (float)(t / ((double)a.rows * a.cpg));
    }
    __syncthreads();
    if (!on) return;
    ch.get_coef(a, sk, c0, g0);
    T* dx = (T*)a.y + n * a.rows * a.C + c0;
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int r = rl + u * a.rpb;
        if (r < rows) {
            float xv[V], dv[V];
            load_vec<T, V>(dy + (long)r * a.dpitch, dv);
            hx[u].again();
            hx[u].get(xv);
            ch.slope(xv, dv, a.act);
            ch.dx(xv, dv);
            store_vec<T, V>(dx + (long)r * a.C, dv);
        }
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------
// elements of one access: the widest power of two up to 16 bytes that divides `c` (rows may start anywhere)
int norm_vec(int c, int bytes) {
    int v = 16 / bytes;
    while (c % v) v /= 2;
    return v;
}

// streaming kernels: 1024 blocks of 4 waves; a split keeps at least 4 steps of rows so that its prologue stays small, and backward at most RUN of them
void norm_geometry(NormArgs& a, int V, bool backward) {
    const int cv = a.C / V;
    a.cols = std::min(cv, NT);
    a.rpb = NT / a.cols;
    a.ctiles = (cv + a.cols - 1) / a.cols;
    const long want = std::max<long>(1, 1024 / std::max<long>(1, (long)a.n * a.ctiles));
    const long most = std::max<long>(1, a.rows / (4L * a.rpb));
    const long least = backward ? (a.rows + (long)RUN * a.rpb - 1) / ((long)RUN * a.rpb) : 1;
    a.splits = (int)std::min<long>(std::max(least, std::min(want, most)), 65535);
    a.rows_per = std::max<long>(1, (a.rows + a.splits - 1) / a.splits);
    a.splits = (int)((a.rows + a.rows_per - 1) / a.rows_per);
}

// resident kernels: V divides channels / groups; the slab is all channels, halved (in whole groups) while it does not fit or while the launch has
// fewer than 256 workgroups and the halves still read whole 64-byte pieces.  false: a single group does not fit, or the streaming kernels are faster:
//  - forward: a slab's pieces of a row below 64 bytes, of more than 4 MB in all (lines fetched by several XCDs).  us resident / streaming: fp16 5 x 2867 x 40
//    in groups of 8 8.3 / 10.2, 16 x 2867 x 64 15.4 / 11.3; fp32 8 x 1200 x 64 6.3 / 8.9, 8 x 2048 x 64 8.0 / 8.3, 32 x 2048 x 64 18.5 / 13.0, 32 x 784 x 64
//    (64 bytes) 6.0 / 9.9.
//  - backward: a second round of workgroups (its phases wait for each other; streaming spreads them over the chip: fp16 36 x 1600 x 256 74.5 / 35.7, fp32
//    32 x 2048 x 64 37.7 / 19.7, 1024 x 49 x 64 42.5 / 30.9), and for 16-bit types more than 15 elements a thread (fp32 holds 16 at most).  Mean of resident /
//    streaming over 1, 8 and 32 samples of 64, 128 and 256 channels in 8 groups, by elements a thread: 16-bit 8: 0.94, 12: 0.98, 14: 0.96, 16: 1.01, 20: 1.04,
//    24: 1.07, 32: 1.12 (a few samples are over it from 8 on, 32 of 256 channels below it at 32); fp32 8: 0.88, 12: 0.91, 16: 0.95.  E.g. fp16 1 x 512 x 64
//    12.5 / 12.6, 8 x 512 x 128 15.5 / 15.2, 32 x 512 x 256 21.2 / 24.8; fp32 1 x 1024 x 64 9.5 / 10.4, 8 x 1024 x 64 11.7 / 11.0, 32 x 512 x 256 18.1 / 24.2.
struct Slab { int v, threads, slabs; };
bool norm_resident(NormArgs& a, int bytes, bool backward, Slab* s) {
    s->v = norm_vec(a.cpg, bytes);
    int groups = a.G;
    auto vecs = [&](int g) { return a.rows * (long)g * a.cpg / s->v; };
    auto cols = [&](int g) { return (long)g * a.cpg / s->v; };
    while (groups > 1 && (cols(groups) > RT || vecs(groups) > RT * (long)RU
                          || ((long)a.n * ((a.G + groups - 1) / groups) < 256 && (long)(groups / 2) * a.cpg * bytes >= 64)))
        groups = (groups + 1) / 2;
    if (cols(groups) > RT) return false;
    a.cols = (int)cols(groups);
    a.rpb = RT / a.cols;
    if ((long)a.rpb * RU < a.rows) return false;
    a.rpb = (int)std::min<long>(a.rpb, a.rows);
    s->threads = (a.cols * a.rpb + 63) / 64 * 64;
    s->slabs = (a.G + groups - 1) / groups;
    const long piece = (long)groups * a.cpg;
    if (backward) return (bytes == 4 || a.rows * piece <= 15 * RT) && (long)a.n * s->slabs <= 256;
    return s->slabs == 1 || piece * bytes >= 64 || a.n * a.rows * a.C * bytes <= 4 << 20;
}

struct NormWs { size_t csum, coef, total; };
NormWs norm_ws(const NormArgs& a, bool backward, bool resident) {
    NormWs w{};
    if (!backward) { w.total = resident ? 0 : (size_t)a.n * a.splits * a.ctiles * a.G * 2 * sizeof(double); return w; }
    w.csum = resident ? 0 : (size_t)a.n * a.splits * 2 * a.C * sizeof(float);
    w.coef = w.csum + (size_t)a.n * 2 * a.C * sizeof(float);
    w.total = resident ? w.coef : w.coef + (size_t)a.n * a.G * 2 * sizeof(float);
    return w;
}

const char* norm_check(const ttc_group_norm_desc* d) {
    if (!d) return "no descriptor";
    if (!known_dtype(d->dtype)) return "unknown dtype (TTC_DT_*)";
    if (!known_act(d->activation)) return "unknown activation (TTC_ACT_*)";
    if (d->n < 0 || d->rows < 0 || d->n > 65535) return "n must be in [0, 65535], rows >= 0";
    if (d->channels < 1 || d->channels > 4096) return "channels must be in [1, 4096]";
    if (d->groups < 1 || d->channels % d->groups) return "groups must divide channels";
    if (!(d->eps >= 0.0f) || std::isinf(d->eps)) return "eps must be finite and >= 0";
    const int64_t lim = (int64_t)1 << 46;
    if (d->rows > lim / d->channels / std::max<int64_t>(1, d->n)) return "array too large";
    if (d->rows > 1 && (d->x_pitch < d->channels || d->x_pitch > lim / d->rows)) return "x_pitch must be at least channels";
    if (d->n > 1 && (d->x_stride < 0 || d->x_stride > lim / d->n)) return "x_stride out of range";
    return nullptr;
}

// everything the launches of a call follow from
struct NormPlan {
    NormArgs a{};
    Slab slab{};
    bool resident = false;
    int V = 1;
    NormWs ws{};
};
NormPlan norm_plan(const ttc_group_norm_desc* d, bool backward) {
    NormPlan p;
    NormArgs& a = p.a;
    const int bytes = dtype_bytes(d->dtype);
    a.rows = d->rows; a.n = (int)d->n; a.C = d->channels; a.G = d->groups; a.cpg = d->channels / d->groups;
    a.act = d->activation; a.eps = d->eps;
    a.sn = d->x_stride; a.pitch = d->x_pitch;
    p.resident = d->rows > 0 && norm_resident(a, bytes, backward, &p.slab);
    if (!p.resident) {
        p.V = norm_vec(a.C, bytes);
        norm_geometry(a, p.V, backward);
    }
    p.ws = norm_ws(a, backward, p.resident);
    return p;
}

template <class F>
ttc_status with_vec(int V, F&& f) {
    switch (V) {
        case 1: f(std::integral_constant<int, 1>{}); break;
        case 2: f(std::integral_constant<int, 2>{}); break;
        case 4: f(std::integral_constant<int, 4>{}); break;
        default: f(std::integral_constant<int, 8>{}); break;
    }
    return TTC_OK;
}

}  // namespace

extern "C" {

ttc_status ttc_group_norm_workspace(const ttc_group_norm_desc* d, int32_t backward, size_t* bytes) {
    if (!bytes) return TTC_ERR_ARG;
    *bytes = 0;
    if (norm_check(d)) return TTC_ERR_ARG;
    if (d->n == 0 || d->rows == 0) return TTC_OK;
    *bytes = norm_plan(d, backward != 0).ws.total;
    return TTC_OK;
}

ttc_status ttc_group_norm(ttc_ctx* c, const ttc_group_norm_desc* d, const void* d_x, const float* d_gamma, const float* d_beta, void* d_y,
                          float* d_stats, void* d_ws, size_t ws_bytes, void* stream) {
    if (!c) return TTC_ERR_ARG;
    if (const char* e = norm_check(d)) return c->fail(TTC_ERR_ARG, std::string("group_norm: ") + e);
    if (d->n == 0 || d->rows == 0) return TTC_OK;
    NormPlan p = norm_plan(d, false);
    NormArgs& a = p.a;
    if (!d_x || !d_y || (p.ws.total && !d_ws)) return c->fail(TTC_ERR_ARG, "group_norm: null pointer");
    if ((uintptr_t)d_ws % 16) return c->fail(TTC_ERR_ARG, "group_norm: the workspace must be 16-byte aligned");
    if (ws_bytes < p.ws.total) return c->fail(TTC_ERR_ARG, "group_norm: workspace smaller than ttc_group_norm_workspace asks for");
    a.x = d_x; a.gamma = d_gamma; a.beta = d_beta; a.y = d_y; a.stats = d_stats; a.part = (double*)d_ws;
    DeviceGuard dev(c->device);
    if (!dev.ok) return c->fail(TTC_ERR_HIP, "group_norm: hipSetDevice failed");
    hipStream_t s = (hipStream_t)stream;
    KTimer t(c, "group_norm", s);
    with_dtype(d->dtype, [&](auto tag) {
        using T = decltype(tag);
        return with_vec(p.resident ? p.slab.v : p.V, [&](auto vt) {
            constexpr int V = decltype(vt)::value;
            if constexpr (V * sizeof(T) <= 16) {
                if (p.resident) {
                    hipLaunchKernelGGL((k_gn_resident<T, V>), dim3(p.slab.slabs, a.n), dim3(p.slab.threads), 0, s, a);
                    return;
                }
                const size_t lds = (size_t)a.rpb * a.cols * V * 2 * sizeof(double);
                const dim3 grid(a.splits, a.n, a.ctiles);
                if (a.cpg % V == 0) {
                    hipLaunchKernelGGL((k_gn_sums<T, V, true>), grid, dim3(NT), lds / V, s, a);
                    hipLaunchKernelGGL((k_gn_apply<T, V, true>), grid, dim3(NT), a.G * 2 * sizeof(float), s, a);
                } else {
                    hipLaunchKernelGGL((k_gn_sums<T, V, false>), grid, dim3(NT), lds, s, a);
                    hipLaunchKernelGGL((k_gn_apply<T, V, false>), grid, dim3(NT), a.G * 2 * sizeof(float), s, a);
                }
            }
        });
    });
    TTC_HIP(c, hipGetLastError());
    return TTC_OK;
}

ttc_status ttc_group_norm_backward(ttc_ctx* c, const ttc_group_norm_desc* d, const void* d_dy, int64_t dy_stride, int64_t dy_pitch,
                                   const void* d_x, const float* d_gamma, const float* d_beta, const float* d_stats, void* d_dx,
                                   float* d_dgamma, float* d_dbeta, void* d_ws, size_t ws_bytes, void* stream) {
    if (!c) return TTC_ERR_ARG;
    if (const char* e = norm_check(d)) return c->fail(TTC_ERR_ARG, std::string("group_norm_backward: ") + e);
    const bool params = d_dgamma || d_dbeta, empty = d->n == 0 || d->rows == 0;
    if (!params && (empty || !d_dx)) return TTC_OK;
    const int64_t lim = (int64_t)1 << 46;
    if (!empty && ((d->rows > 1 && (dy_pitch < d->channels || dy_pitch > lim / d->rows)) || (d->n > 1 && (dy_stride < 0 || dy_stride > lim / d->n))))
        return c->fail(TTC_ERR_ARG, "group_norm_backward: dy_pitch must be at least channels, dy_stride in range");
    NormPlan p;
    if (!empty) {
        p = norm_plan(d, true);
        if (!d_x || !d_dy || !d_stats || !d_ws) return c->fail(TTC_ERR_ARG, "group_norm_backward: null pointer");
        if ((uintptr_t)d_ws % 16) return c->fail(TTC_ERR_ARG, "group_norm_backward: the workspace must be 16-byte aligned");
        if (ws_bytes < p.ws.total) return c->fail(TTC_ERR_ARG, "group_norm_backward: workspace smaller than ttc_group_norm_workspace asks for");
    } else {
        p.a.C = d->channels;
    }
    NormArgs& a = p.a;
    a.x = d_x; a.dy = d_dy; a.gamma = d_gamma; a.beta = d_beta; a.y = d_dx; a.stats_in = d_stats;
    a.dsn = dy_stride; a.dpitch = dy_pitch; a.dgamma = d_dgamma; a.dbeta = d_dbeta;
    a.cpart = (float*)d_ws; a.csum = (float*)((char*)d_ws + p.ws.csum); a.coef = (float*)((char*)d_ws + p.ws.coef);
    DeviceGuard dev(c->device);
    if (!dev.ok) return c->fail(TTC_ERR_HIP, "group_norm_backward: hipSetDevice failed");
    hipStream_t s = (hipStream_t)stream;
    KTimer t(c, "group_norm_backward", s);
    auto param_grads = [&] { hipLaunchKernelGGL(k_gn_param_grads, dim3((a.C + 15) / 16), dim3(NT), 0, s, a); };
    if (empty) {
        param_grads();                             // sums over no samples
        TTC_HIP(c, hipGetLastError());
        return TTC_OK;
    }
    with_dtype(d->dtype, [&](auto tag) {
        using T = decltype(tag);
        return with_vec(p.resident ? p.slab.v : p.V, [&](auto vt) {
            constexpr int V = decltype(vt)::value;
            if constexpr (V * sizeof(T) <= 16) {
                if (p.resident) {
                    const size_t lds = (size_t)std::max(a.rpb, 2) * a.cols * V * 2 * sizeof(float);       // <= 64 KB
                    hipLaunchKernelGGL((k_gn_resident_bwd<T, V>), dim3(p.slab.slabs, a.n), dim3(p.slab.threads), lds, s, a, (int)(a.n == 1));
                    if (params && a.n > 1) param_grads();
                    return;
                }
                const size_t lds = (size_t)a.rpb * a.cols * V * 2 * sizeof(float), mid = (size_t)std::max(RT, 2 * a.C) * sizeof(float);
                const dim3 grid(a.splits, a.n, a.ctiles), grid2(a.splits + params, a.n, a.ctiles);
                if (a.cpg % V == 0) hipLaunchKernelGGL((k_gn_bwd_sums<T, V, true>), grid, dim3(NT), lds, s, a);
                else hipLaunchKernelGGL((k_gn_bwd_sums<T, V, false>), grid, dim3(NT), lds, s, a);
                hipLaunchKernelGGL(k_gn_bwd_mid, dim3(a.n), dim3(RT), mid, s, a);
                if (!a.y) param_grads();
                else if (a.cpg % V == 0) hipLaunchKernelGGL((k_gn_bwd_apply<T, V, true>), grid2, dim3(NT), 0, s, a);
                else hipLaunchKernelGGL((k_gn_bwd_apply<T, V, false>), grid2, dim3(NT), 0, s, a);
            }
        });
    });
    TTC_HIP(c, hipGetLastError());
    return TTC_OK;
}

}  // extern "C"
