// Group norm with an activation over channels-last arrays [n, rows, channels] (rows = pixels of a window), forward and backward, as an
// operator of its own: the layer src/train/src/model.py:100-121 applies, on the channels-last features the library exports
// (ttc_forward_taps).  model.hip keeps the planar fused form of the fixed graph.
//
//   m, v = mean, biased variance over (rows, channels of the group);  rstd = 1 / sqrt(v + eps)
//   xh = (x - m) rstd,  z = gamma xh + beta,  y = act(z)
//   dz = dy act'(z);  dbeta = sum dz;  dgamma = sum dz xh;  M = rows * channels / groups
//   dx = rstd (gamma dz - sum_g(gamma dz) / M - xh sum_g(gamma dz xh) / M)
//
// What bounds it: memory.  The statistics need the whole sample before the first output, so a sample that fits no workgroup is read twice.
// A thread owns one vector of channels (16 bytes) and walks rows: the group a channel belongs to never appears in the inner loop, any
// channels / groups ratio costs the same, and a row is read as whole cache lines.
// Numerics: a thread sums (x - x0) and (x - x0)^2 about its own first row in 32 bits, folds into 64-bit sums every 128 rows; everything across
// threads is 64-bit, in a fixed order (no atomics).
#include <algorithm>

#include "layers_common.h"

namespace {
using namespace layers;

constexpr int NT = 256;             // threads of the streaming kernels
constexpr int FOLD = 128;           // rows summed in 32 bits before they are folded into the 64-bit sums

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
template <class T, int V>
__global__ __launch_bounds__(NT) void k_gn_sums(NormArgs a) {
    extern __shared__ double sm[];                 // [rpb][cols * V][2], then per channel
    const int tid = threadIdx.x, col = tid % a.cols, rl = tid / a.cols;
    const int c0 = (blockIdx.z * a.cols + col) * V;
    const long n = blockIdx.y;
    const long r0 = blockIdx.x * a.rows_per, r1 = min(r0 + a.rows_per, a.rows);
    const int width = a.cols * V;
    double s[V], q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = q[i] = 0.0;
    if (rl < a.rpb && c0 < a.C) {
        const T* x = (const T*)a.x + n * a.sn + c0;
        long r = r0 + rl;
        if (r < r1) {
            float x0[V];
            load_vec<T, V>(x + r * a.pitch, x0);
            while (r < r1) {
                float f[V], g[V];
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = g[i] = 0.0f;
                int k = 0;
                for (; k + 4 <= FOLD && r + 3 * a.rpb < r1; k += 4, r += 4 * a.rpb) {
                    float v[4][V];
#pragma unroll
                    for (int u = 0; u < 4; ++u) load_vec<T, V>(x + (r + u * a.rpb) * a.pitch, v[u]);
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int i = 0; i < V; ++i) { const float d = v[u][i] - x0[i]; f[i] += d; g[i] += d * d; }
                }
                for (; k < FOLD && r < r1; ++k, r += a.rpb) {
                    float v[V];
                    load_vec<T, V>(x + r * a.pitch, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) { const float d = v[i] - x0[i]; f[i] += d; g[i] += d * d; }
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const double c = x0[i];
                    s[i] += k * c + f[i];
                    q[i] += (double)g[i] + 2.0 * c * f[i] + k * c * c;
                }
            }
        }
    }
    if (rl < a.rpb) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            double* d = sm + ((long)rl * width + col * V + i) * 2;
            d[0] = s[i]; d[1] = q[i];
        }
    }
    __syncthreads();
    for (int c = tid; c < width; c += NT) {        // rows of the block -> channels
        double t0 = 0.0, t1 = 0.0;
        for (int r = 0; r < a.rpb; ++r) { t0 += sm[((long)r * width + c) * 2]; t1 += sm[((long)r * width + c) * 2 + 1]; }
        sm[2 * c] = t0; sm[2 * c + 1] = t1;        // row 0's own slot, read by this thread alone
    }
    __syncthreads();
    const int lo = blockIdx.z * width, hi = min(lo + width, a.C);      // channels of this block
    double* out = a.part + ((n * a.splits + blockIdx.x) * a.ctiles + blockIdx.z) * (2L * a.G);
    for (int g = tid; g < a.G; g += NT) {          // channels -> groups; a group of another column tile adds nothing here
        double t0 = 0.0, t1 = 0.0;
        for (int c = max(lo, g * a.cpg); c < min(hi, (g + 1) * a.cpg); ++c) { t0 += sm[2 * (c - lo)]; t1 += sm[2 * (c - lo) + 1]; }
        out[2 * g] = t0; out[2 * g + 1] = t1;
    }
}

// ---- forward, pass 2: y = act(gamma xh + beta) ----------------------------------------------------------------------------------------
template <class T, int V>
__global__ __launch_bounds__(NT) void k_gn_apply(NormArgs a) {
    extern __shared__ float sg[];                  // [G][2]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // pass 1 ended on the last sample: walking the samples back finds its tail in the 256 MB last-level cache
    const long n = gridDim.y - 1 - blockIdx.y;
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
    float mean[V], sc[V], sh[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int g = (c0 + i) / a.cpg;
        mean[i] = sg[2 * g]; sc[i] = sg[2 * g + 1] * gam(a, c0 + i); sh[i] = bet(a, c0 + i);
    }
    const long r0 = blockIdx.x * a.rows_per, r1 = min(r0 + a.rows_per, a.rows);
    const T* x = (const T*)a.x + n * a.sn + c0;
    T* y = (T*)a.y + n * a.rows * a.C + c0;
    // (x - mean) first: exact where x is near the mean, which folding the mean into the shift would lose
    long r = r0 + rl;
    for (; r + 3 * a.rpb < r1; r += 4 * a.rpb) {
        float v[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_vec<T, V>(x + (r + u * a.rpb) * a.pitch, v[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[u][i] = (v[u][i] - mean[i]) * sc[i] + sh[i];
            act_vec<V>(v[u], a.act);
            store_vec<T, V>(y + (r + u * a.rpb) * a.C, v[u]);
        }
    }
    for (; r < r1; r += a.rpb) {
        float v[V];
        load_vec<T, V>(x + r * a.pitch, v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (v[i] - mean[i]) * sc[i] + sh[i];
        act_vec<V>(v, a.act);
        store_vec<T, V>(y + r * a.C, v);
    }
}

// dz = dy act'(z) and xh of one vector
template <int V>
__device__ __forceinline__ void norm_slope(const float (&x)[V], const float (&dy)[V], const float (&mean)[V], const float (&rstd)[V],
                                           const float (&ga)[V], const float (&be)[V], int act, float (&dz)[V], float (&xh)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) { xh[i] = (x[i] - mean[i]) * rstd[i]; dz[i] = dy[i]; }
    if (act != TTC_ACT_NONE) {
        float z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = xh[i] * ga[i] + be[i];
        slope_vec<V>(dz, z, act);
    }
}

// ---- backward, pass 1: sum dz, sum dz xh per (sample, slot, channel) -----------------------------------------------------------------
template <class T, int V>
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
        float mean[V], rstd[V], ga[V], be[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float* st = a.stats_in + (n * a.G + (c0 + i) / a.cpg) * 2;
            mean[i] = st[0]; rstd[i] = st[1]; ga[i] = gam(a, c0 + i); be[i] = bet(a, c0 + i);
        }
        const T* x = (const T*)a.x + n * a.sn + c0;
        const T* dy = (const T*)a.dy + n * a.dsn + c0;
        long r = r0 + rl;
        for (; r + a.rpb < r1; r += 2 * a.rpb) {
            float xv[2][V], dv[2][V], dz[V], xh[V];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                load_vec<T, V>(x + (r + u * a.rpb) * a.pitch, xv[u]);
                load_vec<T, V>(dy + (r + u * a.rpb) * a.dpitch, dv[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                norm_slope<V>(xv[u], dv[u], mean, rstd, ga, be, a.act, dz, xh);
#pragma unroll
                for (int i = 0; i < V; ++i) { sa[i] += dz[i]; sb[i] += dz[i] * xh[i]; }
            }
        }
        for (; r < r1; r += a.rpb) {
            float xv[V], dv[V], dz[V], xh[V];
            load_vec<T, V>(x + r * a.pitch, xv);
            load_vec<T, V>(dy + r * a.dpitch, dv);
            norm_slope<V>(xv, dv, mean, rstd, ga, be, a.act, dz, xh);
#pragma unroll
            for (int i = 0; i < V; ++i) { sa[i] += dz[i]; sb[i] += dz[i] * xh[i]; }
        }
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
        const int ch = blockIdx.z * width + c;
        if (ch >= a.C) break;
        double t0 = 0.0, t1 = 0.0;
        for (int r = 0; r < a.rpb; ++r) { t0 += sf[(r * width + c) * 2]; t1 += sf[(r * width + c) * 2 + 1]; }
        out[ch] = (float)t0; out[a.C + ch] = (float)t1;
    }
}

// ---- backward, between: slots -> channels of a sample, and the two group means --------------------------------------------------------
__global__ __launch_bounds__(NT) void k_gn_bwd_mid(NormArgs a) {
    extern __shared__ float sc2[];                 // [2][C]: gamma dz, gamma dz xh
    const long n = blockIdx.x;
    const float* p = a.cpart + n * a.splits * 2L * a.C;
    for (int c = threadIdx.x; c < 2 * a.C; c += NT) {
        double t = 0.0;
        for (int i = 0; i < a.splits; ++i) t += p[(long)i * 2 * a.C + c];
        a.csum[n * 2 * a.C + c] = (float)t;
        sc2[c] = (float)t * gam(a, c < a.C ? c : c - a.C);
    }
    __syncthreads();
    const double m = (double)a.rows * a.cpg;
    for (int g = threadIdx.x; g < 2 * a.G; g += NT) {
        const float* s = sc2 + (g < a.G ? 0 : a.C) + (g < a.G ? g : g - a.G) * a.cpg;
        double t = 0.0;
        for (int c = 0; c < a.cpg; ++c) t += s[c];
        a.coef[(n * a.G + (g < a.G ? g : g - a.G)) * 2 + (g < a.G ? 0 : 1)] = (float)(t / m);
    }
}

// dgamma, dbeta: channels summed over the samples, 16 channels a block, 16 lanes each
__device__ void gn_param_grads(const NormArgs& a, int block) {
    __shared__ double red[16][17][2];
    const int ch = threadIdx.x & 15, l = threadIdx.x >> 4, c = block * 16 + ch;
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
}
__global__ __launch_bounds__(NT) void k_gn_param_grads(NormArgs a) { gn_param_grads(a, blockIdx.x); }

// ---- backward, pass 2: dx --------------------------------------------------------------------------------------------------------------
template <class T, int V>
__global__ __launch_bounds__(NT) void k_gn_bwd_apply(NormArgs a) {
    const int tid = threadIdx.x, col = tid % a.cols, rl = tid / a.cols, c0 = (blockIdx.z * a.cols + col) * V;
    const long n = gridDim.y - 1 - blockIdx.y;     // back to front, as in the forward's second pass
    if (rl >= a.rpb || c0 >= a.C) return;
    float mean[V], rstd[V], ga[V], be[V], k1[V], k2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const long g = n * a.G + (c0 + i) / a.cpg;
        mean[i] = a.stats_in[2 * g]; rstd[i] = a.stats_in[2 * g + 1];
        k1[i] = a.coef[2 * g]; k2[i] = a.coef[2 * g + 1];
        ga[i] = gam(a, c0 + i); be[i] = bet(a, c0 + i);
    }
    const long r0 = blockIdx.x * a.rows_per, r1 = min(r0 + a.rows_per, a.rows);
    const T* x = (const T*)a.x + n * a.sn + c0;
    const T* dy = (const T*)a.dy + n * a.dsn + c0;
    T* dx = (T*)a.y + n * a.rows * a.C + c0;
    long r = r0 + rl;
    for (; r + a.rpb < r1; r += 2 * a.rpb) {
        float xv[2][V], dv[2][V], dz[V], xh[V];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            load_vec<T, V>(x + (r + u * a.rpb) * a.pitch, xv[u]);
            load_vec<T, V>(dy + (r + u * a.rpb) * a.dpitch, dv[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            norm_slope<V>(xv[u], dv[u], mean, rstd, ga, be, a.act, dz, xh);
#pragma unroll
            for (int i = 0; i < V; ++i) dz[i] = rstd[i] * (ga[i] * dz[i] - k1[i] - xh[i] * k2[i]);
            store_vec<T, V>(dx + (r + u * a.rpb) * a.C, dz);
        }
    }
    for (; r < r1; r += a.rpb) {
        float xv[V], dv[V], dz[V], xh[V];
        load_vec<T, V>(x + r * a.pitch, xv);
        load_vec<T, V>(dy + r * a.dpitch, dv);
        norm_slope<V>(xv, dv, mean, rstd, ga, be, a.act, dz, xh);
#pragma unroll
        for (int i = 0; i < V; ++i) dz[i] = rstd[i] * (ga[i] * dz[i] - k1[i] - xh[i] * k2[i]);
        store_vec<T, V>(dx + r * a.C, dz);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------
// elements of one access: the widest power of two up to 16 bytes that divides the channels (rows may start anywhere)
int norm_vec(int C, int bytes) {
    int v = 16 / bytes;
    while (C % v) v /= 2;
    return v;
}

// 2048 blocks of 4 waves fill 256 CUs once; a split keeps at least 4 steps of rows so that its prologue stays small
void norm_geometry(NormArgs& a, int V) {
    const int cv = a.C / V;
    a.cols = std::min(cv, NT);
    a.rpb = NT / a.cols;
    a.ctiles = (cv + a.cols - 1) / a.cols;
    const long want = std::max<long>(1, 2048 / std::max<long>(1, (long)a.n * a.ctiles));
    const long most = std::max<long>(1, a.rows / (4L * a.rpb));
    a.splits = (int)std::min<long>({want, most, 65535});
    a.rows_per = std::max<long>(1, (a.rows + a.splits - 1) / a.splits);
    a.splits = (int)((a.rows + a.rows_per - 1) / a.rows_per);
}

struct NormWs { size_t part, csum, coef, total; };
NormWs norm_ws(const NormArgs& a, bool backward) {
    NormWs w{};
    if (!backward) { w.total = (size_t)a.n * a.splits * a.ctiles * a.G * 2 * sizeof(double); return w; }
    w.csum = (size_t)a.n * a.splits * 2 * a.C * sizeof(float);
    w.coef = w.csum + (size_t)a.n * 2 * a.C * sizeof(float);
    w.total = w.coef + (size_t)a.n * a.G * 2 * sizeof(float);
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
NormArgs norm_args(const ttc_group_norm_desc* d, int V) {
    NormArgs a{};
    a.rows = d->rows; a.n = (int)d->n; a.C = d->channels; a.G = d->groups; a.cpg = d->channels / d->groups;
    a.act = d->activation; a.eps = d->eps;
    a.sn = d->x_stride; a.pitch = d->x_pitch;
    norm_geometry(a, V);
    return a;
}

template <class F>
ttc_status with_vec(int V, F&& f) {
    switch (V) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        default: return f(std::integral_constant<int, 8>{});
    }
}

}  // namespace

extern "C" {

ttc_status ttc_group_norm_workspace(const ttc_group_norm_desc* d, int32_t backward, size_t* bytes) {
    if (!bytes) return TTC_ERR_ARG;
    *bytes = 0;
    if (norm_check(d)) return TTC_ERR_ARG;
    if (d->n == 0 || (d->rows == 0 && !backward)) return TTC_OK;
    *bytes = norm_ws(norm_args(d, norm_vec(d->channels, dtype_bytes(d->dtype))), backward != 0).total;
    return TTC_OK;
}

ttc_status ttc_group_norm(ttc_ctx* c, const ttc_group_norm_desc* d, const void* d_x, const float* d_gamma, const float* d_beta, void* d_y,
                          float* d_stats, void* d_ws, size_t ws_bytes, void* stream) {
    if (!c) return TTC_ERR_ARG;
    if (const char* e = norm_check(d)) return c->fail(TTC_ERR_ARG, std::string("group_norm: ") + e);
    if (d->n == 0 || d->rows == 0) return TTC_OK;
    const int V = norm_vec(d->channels, dtype_bytes(d->dtype));
    NormArgs a = norm_args(d, V);
    const NormWs w = norm_ws(a, false);
    if (!d_x || !d_y || !d_ws) return c->fail(TTC_ERR_ARG, "group_norm: null pointer");
    if (ws_bytes < w.total) return c->fail(TTC_ERR_ARG, "group_norm: workspace smaller than ttc_group_norm_workspace asks for");
    a.x = d_x; a.gamma = d_gamma; a.beta = d_beta; a.y = d_y; a.stats = d_stats; a.part = (double*)d_ws;
    DeviceGuard dev(c->device);
    if (!dev.ok) return c->fail(TTC_ERR_HIP, "group_norm: hipSetDevice failed");
    hipStream_t s = (hipStream_t)stream;
    KTimer t(c, "group_norm", s);
    const ttc_status st = with_dtype(d->dtype, [&](auto tag) {
        using T = decltype(tag);
        return with_vec(V, [&](auto vt) {
            constexpr int VV = decltype(vt)::value;
            if constexpr (VV * sizeof(T) <= 16) {
                const dim3 grid(a.splits, a.n, a.ctiles);
                const size_t lds = (size_t)a.rpb * a.cols * VV * 2 * sizeof(double);
                hipLaunchKernelGGL((k_gn_sums<T, VV>), grid, dim3(NT), lds, s, a);
                hipLaunchKernelGGL((k_gn_apply<T, VV>), grid, dim3(NT), a.G * 2 * sizeof(float), s, a);
            }
            return TTC_OK;
        });
    });
    TTC_HIP(c, hipGetLastError());
    return st;
}

ttc_status ttc_group_norm_backward(ttc_ctx* c, const ttc_group_norm_desc* d, const void* d_dy, int64_t dy_stride, int64_t dy_pitch,
                                   const void* d_x, const float* d_gamma, const float* d_beta, const float* d_stats, void* d_dx,
                                   float* d_dgamma, float* d_dbeta, void* d_ws, size_t ws_bytes, void* stream) {
    if (!c) return TTC_ERR_ARG;
    if (const char* e = norm_check(d)) return c->fail(TTC_ERR_ARG, std::string("group_norm_backward: ") + e);
    const bool params = d_dgamma || d_dbeta, empty = d->n == 0 || d->rows == 0;
    if (empty && !params) return TTC_OK;
    const int64_t lim = (int64_t)1 << 46;
    if (!empty && ((d->rows > 1 && (dy_pitch < d->channels || dy_pitch > lim / d->rows)) || (d->n > 1 && (dy_stride < 0 || dy_stride > lim / d->n))))
        return c->fail(TTC_ERR_ARG, "group_norm_backward: dy_pitch must be at least channels, dy_stride in range");
    const int V = norm_vec(d->channels, dtype_bytes(d->dtype));
    NormArgs a = norm_args(d, V);
    const NormWs w = norm_ws(a, true);
    if (!empty && (!d_x || !d_dy || !d_stats || !d_ws)) return c->fail(TTC_ERR_ARG, "group_norm_backward: null pointer");
    if (!empty && ws_bytes < w.total) return c->fail(TTC_ERR_ARG, "group_norm_backward: workspace smaller than ttc_group_norm_workspace asks for");
    a.x = d_x; a.dy = d_dy; a.gamma = d_gamma; a.beta = d_beta; a.y = d_dx; a.stats_in = d_stats;
    a.dsn = dy_stride; a.dpitch = dy_pitch; a.dgamma = d_dgamma; a.dbeta = d_dbeta;
    a.cpart = (float*)d_ws; a.csum = (float*)((char*)d_ws + w.csum); a.coef = (float*)((char*)d_ws + w.coef);
    if (empty) a.n = 0;
    DeviceGuard dev(c->device);
    if (!dev.ok) return c->fail(TTC_ERR_HIP, "group_norm_backward: hipSetDevice failed");
    hipStream_t s = (hipStream_t)stream;
    KTimer t(c, "group_norm_backward", s);
    ttc_status st = TTC_OK;
    if (!empty)
        st = with_dtype(d->dtype, [&](auto tag) {
            using T = decltype(tag);
            return with_vec(V, [&](auto vt) {
                constexpr int VV = decltype(vt)::value;
                if constexpr (VV * sizeof(T) <= 16) {
                    const dim3 grid(a.splits, a.n, a.ctiles);
                    hipLaunchKernelGGL((k_gn_bwd_sums<T, VV>), grid, dim3(NT), (size_t)a.rpb * a.cols * VV * 2 * sizeof(float), s, a);
                    hipLaunchKernelGGL(k_gn_bwd_mid, dim3(a.n), dim3(NT), (size_t)a.C * 2 * sizeof(float), s, a);
                    if (a.y) hipLaunchKernelGGL((k_gn_bwd_apply<T, VV>), grid, dim3(NT), 0, s, a);
                }
                return TTC_OK;
            });
        });
    if (params) hipLaunchKernelGGL(k_gn_param_grads, dim3((a.C + 15) / 16), dim3(NT), 0, s, a);
    TTC_HIP(c, hipGetLastError());
    return st;
}

}  // extern "C"
