// Product of channels-last rows with a weight matrix, bias, activation and residual in the epilogue -- the 1x1 convolution as an operator of
// its own (the graph's head: src/train/train-model.py:226-231), forward and backward.
//
//   z = x w + b,  y = residual + scale act(z)            x [m, k], w [k, n] (TF layout: the output channel is contiguous)
//   dz = scale dy act'(z);  dx = dz w^T;  dw = x^T dz;  db = column sums of dz
//
// All three products run the one tile kernel k_gemm: C[i, j] = sum_c A(i, c) B(c, j), where each operand is stored either with the contracted index
// contiguous ("KC": x and dz in dx, w in dx) or with its free index contiguous ("FC": w in y, x and dz in dw).
//  - KC tiles lie in LDS as rows of 128 bytes; a lane reads 16 bytes = its 8 (16-bit) or 4 (fp32) values of the contracted index.
//  - FC tiles lie in LDS as stored; 16-bit fragments come through the transposing LDS read (ds_read_tr16_b64), fp32 ones through single words.
//  - the contracted index may be permuted freely as long as both operands agree: that is what makes the 16-byte KC read fit the fp32 instruction.
//  - the matrix instruction gets B's fragment first, so a lane ends up with consecutive OUTPUT CHANNELS of one row (8 for 16-bit types: the rows of
//    fragment pairs are interleaved) and stores 16 bytes at a time.
// LDS slots are XOR-swizzled so that no fragment read has more than a two-way bank conflict.
#include <algorithm>

#include "layers_common.h"

namespace {
using namespace layers;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int NT = 256;

struct GemmArgs {
    const void* A; const void* B;
    long lda, ldb;
    long M; int N; long K;          // C is [M, N], K contracted
    long k_per;                     // contracted range of a split (blockIdx.y)
    void* C; long ldc;              // T, or float partials [split][M][N]
    int partial;
    float alpha;
    // forward epilogue
    int fwd, act;
    const float* bias; const void* res; long ldr; void* preact;
    int mt, nt;                     // tiles
};

// ---- fragments ----------------------------------------------------------------------------------------------------------------------------
template <class T> struct Mma;
template <> struct Mma<f16> {
    typedef vec<f16, 8> Frag;
    static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<bf16> {
    typedef vec<bf16, 8> Frag;
    static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<float> {
    typedef f32x4 Frag;             // 4 values of the contracted index = 4 instructions of 4
    static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// free index (inside a wave's extent) of fragment f, instruction row r.  16-bit, B: fragment pairs interleave so that a lane's 2 x 4 results are 8
// consecutive columns.
template <class T, bool PAIR>
__device__ __forceinline__ int free_of(int f, int r) {
    return PAIR && sizeof(T) == 2 ? 32 * (f >> 1) + 8 * (r >> 2) + 4 * (f & 1) + (r & 3) : 16 * f + r;
}

template <class T> constexpr int BKE = 128 / sizeof(T);      // contracted elements of a tile step
template <class T> constexpr int VE = 16 / sizeof(T);        // elements of 16 bytes

__device__ __forceinline__ int kc_slot(int row, int ch) { return row * 8 + (ch ^ ((row ^ (row >> 3)) & 7)); }   // in 16-byte units

template <class T, int BF>
__device__ __forceinline__ int fc_byte(int k, int f) {       // byte offset of element (k, f) of an FC tile, f a multiple of the read width
    constexpr int NG = BF / 16;
    const int sw = sizeof(T) == 2 ? ((k & 3) | ((k >> 1) & 4)) : ((k >> 2) & 3);
    return k * BF * (int)sizeof(T) + (((f >> 4) ^ (sw & (NG - 1))) << 4) * (int)sizeof(T) + (f & 15) * (int)sizeof(T);
}

// one 16-byte piece of a row with `left` valid elements (zero past them)
template <class T>
__device__ __forceinline__ uint4 load_piece(const T* p, long left) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (left >= VE<T>) { __builtin_memcpy(&v, p, 16); return v; }
    if (left > 0) {
        T t[VE<T>];
#pragma unroll
        for (int i = 0; i < VE<T>; ++i) t[i] = i < left ? p[i] : (T)0.0f;
        __builtin_memcpy(&v, t, 16);
    }
    return v;
}

// the 16-byte pieces of a BF x BKE tile a thread moves, global -> registers -> LDS
template <class T, bool KC, int BF>
struct Stage {
    static constexpr int CNT = BF * 8 / NT;
    uint4 v[CNT];
    __device__ __forceinline__ void load(const T* p, long ld, long f0, long F, long k0, long k1, int tid) {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int id = tid + i * NT;
            if (KC) {
                const long f = f0 + (id >> 3), k = k0 + (id & 7) * VE<T>;
                v[i] = load_piece(p + f * ld + k, f < F ? k1 - k : 0);
            } else {
                constexpr int PR = BF / VE<T>;
                const long k = k0 + id / PR, f = f0 + (id % PR) * VE<T>;
                v[i] = load_piece(p + k * ld + f, k < k1 ? F - f : 0);
            }
        }
    }
    __device__ __forceinline__ void store(char* lds, int tid) const {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int id = tid + i * NT;
            if (KC) {
                reinterpret_cast<uint4*>(lds)[kc_slot(id >> 3, id & 7)] = v[i];
            } else {
                constexpr int PR = BF / VE<T>;
                *reinterpret_cast<uint4*>(lds + fc_byte<T, BF>(id / PR, (id % PR) * VE<T>)) = v[i];
            }
        }
    }
};

template <class T, bool KC, int BF, bool PAIR>
__device__ __forceinline__ typename Mma<T>::Frag frag(const char* lds, int base, int f, int ks, int lane) {
    const int r = lane & 15, q = lane >> 4;
    if constexpr (KC) {
        const uint4 u = reinterpret_cast<const uint4*>(lds)[kc_slot(base + free_of<T, PAIR>(f, r), ks * 4 + q)];
        return __builtin_bit_cast(typename Mma<T>::Frag, u);
    } else if constexpr (sizeof(T) == 2) {
        // transposing read: lane i of 16 names 4 consecutive free elements of row i / 4 and receives free element i of rows 0..3
        const int k = ks * 32 + q * 8 + (r >> 2), c = base + free_of<T, PAIR>(f, 4 * (r & 3));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + fc_byte<T, BF>(k, c)));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + fc_byte<T, BF>(k + 4, c)));
        struct { s16x4 a, b; } u = {lo, hi};
        return __builtin_bit_cast(typename Mma<T>::Frag, u);
    } else {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float*>(lds + fc_byte<T, BF>(ks * 16 + q * 4 + i, base + 16 * f + r));
        return v;
    }
}

// what the backward pass reads back: rounded to T, but never across 0 or to infinity (relu's slope is a matter of the sign, and an infinite value
// would make 0 * inf of the slopes that have long reached their limit)
template <class T>
__device__ __forceinline__ float keep_preact(float z) {
    if constexpr (__is_same(T, f16)) {
        const float m = fabsf(z);
        if (m > 65504.0f) return copysignf(65504.0f, z);
        if (m > 0.0f && m < 5.9604645e-8f) return copysignf(5.9604645e-8f, z);
    }
    return z;
}

// V consecutive columns of one row; `left` of them exist
template <class T, int V>
__device__ __forceinline__ void emit(const GemmArgs& a, long row, long col, int left, float (&v)[V]) {
    if (a.partial) {
        float* p = (float*)a.C + ((long)blockIdx.y * a.M + row) * a.N + col;
        if (left >= V) store_vec<float, V>(p, v);
        else for (int i = 0; i < left; ++i) p[i] = v[i];
        return;
    }
    T* out = (T*)a.C + row * a.ldc + col;
    if (!a.fwd) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= a.alpha;
    } else {
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < V; ++i) if (i < left) v[i] += a.bias[col + i];
        }
        if (a.preact) {
            T* pp = (T*)a.preact + row * a.ldc + col;
            float z[V];
#pragma unroll
            for (int i = 0; i < V; ++i) z[i] = keep_preact<T>(v[i]);
            if (left >= V) store_vec<T, V>(pp, z);
            else
#pragma unroll
                for (int i = 0; i < V; ++i) if (i < left) pp[i] = (T)z[i];
        }
        act_vec<V>(v, a.act);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= a.alpha;
        if (a.res) {
            const T* rp = (const T*)a.res + row * a.ldr + col;
            float r[V];
            if (left >= V) load_vec<T, V>(rp, r);
            else
#pragma unroll
                for (int i = 0; i < V; ++i) r[i] = i < left ? (float)rp[i] : 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += r[i];
        }
    }
    if (left >= V) store_vec<T, V>(out, v);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) if (i < left) out[i] = (T)v[i];
}

// ---- the tile kernel --------------------------------------------------------------------------------------------------------------------
template <class T, bool AKC, bool BKC, int BM, int BN, int WGM>
__global__ __launch_bounds__(NT) void k_gemm(GemmArgs a) {
    constexpr int WGN = 4 / WGM, WM = BM / WGM, WN = BN / WGN, FM = WM / 16, FN = WN / 16, KS = sizeof(T) == 2 ? 2 : 2;
    constexpr int ABYTES = BM * 128, BBYTES = BN * 128;
    __shared__ __attribute__((aligned(16))) char lds[2 * (ABYTES + BBYTES)];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WGN, wn = wave % WGN;
    // workgroups go round the 8 XCDs: give each XCD a contiguous run of tiles (column tiles fastest), so that a row tile's re-reads hit its L2
    const int total = a.mt * a.nt, bid = blockIdx.x, xcd = bid & 7, per = total >> 3, rem = total & 7;
    const int tile = xcd * per + min(xcd, rem) + (bid >> 3);
    const long m0 = (long)(tile / a.nt) * BM;
    const int n0 = (tile % a.nt) * BN;
    const long k0 = blockIdx.y * a.k_per, k1 = min(k0 + a.k_per, a.K);
    const T* A = (const T*)a.A;
    const T* B = (const T*)a.B;
    Stage<T, AKC, BM> sa;
    Stage<T, BKC, BN> sb;
    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    sa.load(A, a.lda, m0, a.M, k0, k1, tid);
    sb.load(B, a.ldb, n0, a.N, k0, k1, tid);
    sa.store(lds, tid);
    sb.store(lds + 2 * ABYTES, tid);
    __syncthreads();
    int cur = 0;
    for (long k = k0; k < k1; k += BKE<T>, cur ^= 1) {
        const bool more = k + BKE<T> < k1;
        if (more) {
            sa.load(A, a.lda, m0, a.M, k + BKE<T>, k1, tid);
            sb.load(B, a.ldb, n0, a.N, k + BKE<T>, k1, tid);
        }
        const char* la = lds + cur * ABYTES;
        const char* lb = lds + 2 * ABYTES + cur * BBYTES;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            typename Mma<T>::Frag fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FM; ++j) fa[j] = frag<T, AKC, BM, false>(la, wm * WM, j, ks, lane);
#pragma unroll
            for (int i = 0; i < FN; ++i) fb[i] = frag<T, BKC, BN, true>(lb, wn * WN, i, ks, lane);
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j) acc[i][j] = Mma<T>::run(fb[i], fa[j], acc[i][j]);
        }
        if (more) {                                // the other half was last read before the previous barrier
            sa.store(lds + (cur ^ 1) * ABYTES, tid);
            sb.store(lds + 2 * ABYTES + (cur ^ 1) * BBYTES, tid);
        }
        __syncthreads();
    }
    const int r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const long row = m0 + wm * WM + j * 16 + r;
        if (row >= a.M) continue;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int p = 0; p < FN / 2; ++p) {
                const int col = n0 + wn * WN + 32 * p + 8 * q;
                if (col >= a.N) continue;
                float v[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) { v[i] = acc[2 * p][j][i]; v[4 + i] = acc[2 * p + 1][j][i]; }
                emit<T, 8>(a, row, col, a.N - col, v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const int col = n0 + wn * WN + 16 * i + 4 * q;
                if (col >= a.N) continue;
                float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                emit<T, 4>(a, row, col, a.N - col, v);
            }
        }
    }
}

// out[i] = alpha * sum of the splits, in split order within 16 interleaved lanes: 64 outputs a block
template <class T>
__global__ __launch_bounds__(NT) void k_gemm_reduce(const float* __restrict__ part, int splits, long cnt, float alpha, T* __restrict__ out) {
    __shared__ float red[16][64];
    const int e = threadIdx.x & 15, l = threadIdx.x >> 4;
    const long i0 = (long)blockIdx.x * 64 + e * 4;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (i0 + 4 <= cnt) {
        for (int k = l; k < splits; k += 16) {
            float v[4];
            load_vec<float, 4>(part + k * cnt + i0, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += v[i];
        }
    } else {
        for (int k = l; k < splits; k += 16)
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i0 + i < cnt) s[i] += part[k * cnt + i0 + i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) red[l][e * 4 + i] = s[i];
    __syncthreads();
    const long o = (long)blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x < 64 && o < cnt) {
        float t = 0.0f;
        for (int k = 0; k < 16; ++k) t += red[k][threadIdx.x];
        out[o] = (T)(t * alpha);
    }
}

// ---- dz = scale dy act'(z), and the column sums of dz -----------------------------------------------------------------------------------
struct DzArgs {
    const void* dy; const void* z; void* dz; float* part;
    long rows, dpitch; int N, act; float scale;
    int cols, rpb; long rows_per;
};
template <class T, int V>
__global__ __launch_bounds__(NT) void k_dz(DzArgs a) {
    extern __shared__ float sf[];
    const int tid = threadIdx.x, col = tid % a.cols, rl = tid / a.cols, width = a.cols * V;
    const int c0 = (blockIdx.y * a.cols + col) * V;
    const long r0 = blockIdx.x * a.rows_per, r1 = min(r0 + a.rows_per, a.rows);
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.0f;
    if (rl < a.rpb && c0 < a.N)
        for (long r = r0 + rl; r < r1; r += a.rpb) {
            float d[V], z[V];
            load_vec<T, V>((const T*)a.dy + r * a.dpitch + c0, d);
            if (a.act != TTC_ACT_NONE) load_vec<T, V>((const T*)a.z + r * a.N + c0, z);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                d[i] *= a.scale;
                if (a.act != TTC_ACT_NONE) d[i] *= act_slope(z[i], a.act);
                s[i] += d[i];
            }
            if (a.dz) store_vec<T, V>((T*)a.dz + r * a.N + c0, d);   // the products take operands of their type: dz is rounded to it once
        }
    if (!a.part) return;
    if (rl < a.rpb)
#pragma unroll
        for (int i = 0; i < V; ++i) sf[rl * width + col * V + i] = s[i];
    __syncthreads();
    for (int c = tid; c < width; c += NT) {
        const int ch = blockIdx.y * width + c;
        if (ch >= a.N) break;
        double t = 0.0;
        for (int r = 0; r < a.rpb; ++r) t += sf[r * width + c];
        a.part[(long)blockIdx.x * a.N + ch] = (float)t;
    }
}
// column sums of [rows][N], 16 columns a block
__global__ __launch_bounds__(NT) void k_col_reduce(const float* __restrict__ part, int rows, int N, float* __restrict__ out) {
    __shared__ double red[16][17];
    const int ch = threadIdx.x & 15, l = threadIdx.x >> 4, c = blockIdx.x * 16 + ch;
    double t = 0.0;
    if (c < N) for (int r = l; r < rows; r += NT / 16) t += part[(long)r * N + c];
    red[l][ch] = t;
    __syncthreads();
    if (l == 0 && c < N) {
        for (int i = 1; i < NT / 16; ++i) t += red[i][ch];
        out[c] = (float)t;
    }
}
template <class T>
__global__ void k_fill0(T* p, long n) {
    const long i = (long)blockIdx.x * NT + threadIdx.x;
    if (i < n) p[i] = (T)0.0f;
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------
template <class T, bool AKC, bool BKC>
void gemm_launch(GemmArgs a, int splits, hipStream_t s) {
    a.mt = (int)((a.M + 127) / 128);
    auto go = [&](auto fn, int bn) {
        a.nt = (a.N + bn - 1) / bn;
        hipLaunchKernelGGL(fn, dim3((unsigned)(a.mt * a.nt), splits), dim3(NT), 0, s, a);
    };
    // narrower column tiles only where the wide one would be mostly padding
    if (a.N <= 32) go(k_gemm<T, AKC, BKC, 128, 32, 4>, 32);
    else if (a.N <= 64) go(k_gemm<T, AKC, BKC, 128, 64, 2>, 64);
    else go(k_gemm<T, AKC, BKC, 128, 128, 2>, 128);
}

// splits of the contracted rows of dw: enough workgroups for two per CU, at least 512 rows each, partials of at most 64 MB
int dw_splits(const ttc_linear_desc* d) {
    const long tiles = ((d->cin + 127L) / 128) * ((d->cout + 127L) / 128);
    const long fit = std::max<long>(1, (64L << 20) / ((long)d->cin * d->cout * 4));
    return (int)std::max<long>(1, std::min<long>({512 / tiles, d->rows / 512, fit}));
}
int col_vec(int N, int bytes) {
    int v = 16 / bytes;
    while (N % v) v /= 2;
    return v;
}
void dz_geometry(DzArgs& a, int V, int* blocks, int* tiles) {
    const int cv = a.N / V;
    a.cols = std::min(cv, NT);
    a.rpb = NT / a.cols;
    *tiles = (cv + a.cols - 1) / a.cols;
    const long want = std::max<long>(1, 2048 / *tiles), most = std::max<long>(1, a.rows / (4L * a.rpb));
    long b = std::min(want, most);
    a.rows_per = std::max<long>(1, (a.rows + b - 1) / b);
    *blocks = (int)((a.rows + a.rows_per - 1) / a.rows_per);
}

struct BwdWs { size_t dz, sums, dw, total; int blocks; };
BwdWs linear_ws(const ttc_linear_desc* d) {
    const auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    BwdWs w{};
    DzArgs z{};
    z.rows = d->rows; z.N = d->cout;
    int tiles;
    dz_geometry(z, col_vec(d->cout, dtype_bytes(d->dtype)), &w.blocks, &tiles);
    w.sums = d->activation != TTC_ACT_NONE ? up((size_t)d->rows * d->cout * dtype_bytes(d->dtype)) : 0;
    w.dw = w.sums + up((size_t)w.blocks * d->cout * sizeof(float));
    const int sp = dw_splits(d);
    w.total = w.dw + (sp > 1 ? (size_t)sp * d->cin * d->cout * sizeof(float) : 0);
    return w;
}

const char* linear_check(const ttc_linear_desc* d) {
    if (!d) return "no descriptor";
    if (!known_dtype(d->dtype)) return "unknown dtype (TTC_DT_*)";
    if (!known_act(d->activation)) return "unknown activation (TTC_ACT_*)";
    if (d->rows < 0 || d->rows > (1L << 31) - 1) return "rows must be in [0, 2^31)";
    if (d->cin < 1 || d->cin > 65536 || d->cout < 1 || d->cout > 65536) return "cin and cout must be in [1, 65536]";
    if (((d->rows + 127) / 128) * ((d->cout + 31) / 32) > (1L << 31) - 1 || ((d->rows + 127) / 128) * ((d->cin + 31) / 32) > (1L << 31) - 1)
        return "array too large";
    const int64_t lim = (int64_t)1 << 30;
    if ((d->rows > 1 && d->x_pitch < d->cin) || d->x_pitch > lim) return "x_pitch must be at least cin";
    if ((d->cin > 1 && d->w_pitch < d->cout) || d->w_pitch > lim) return "w_pitch must be at least cout";
    if (!std::isfinite(d->scale)) return "scale must be finite";
    return nullptr;
}

}  // namespace

extern "C" {

ttc_status ttc_linear_workspace(const ttc_linear_desc* d, int32_t backward, size_t* bytes) {
    if (!bytes) return TTC_ERR_ARG;
    *bytes = 0;
    if (linear_check(d)) return TTC_ERR_ARG;
    if (backward && d->rows > 0) *bytes = linear_ws(d).total;
    return TTC_OK;
}

ttc_status ttc_linear(ttc_ctx* c, const ttc_linear_desc* d, const void* d_x, const void* d_w, const float* d_bias, const void* d_residual,
                      void* d_y, void* d_preact, void* d_ws, size_t ws_bytes, void* stream) {
    (void)d_ws; (void)ws_bytes;
    if (!c) return TTC_ERR_ARG;
    if (const char* e = linear_check(d)) return c->fail(TTC_ERR_ARG, std::string("linear: ") + e);
    if (d_residual && ((d->rows > 1 && d->res_pitch < d->cout) || d->res_pitch > (1L << 30)))
        return c->fail(TTC_ERR_ARG, "linear: res_pitch must be at least cout");
    if (d->rows == 0) return TTC_OK;
    if (!d_x || !d_w || !d_y) return c->fail(TTC_ERR_ARG, "linear: null pointer");
    DeviceGuard dev(c->device);
    if (!dev.ok) return c->fail(TTC_ERR_HIP, "linear: hipSetDevice failed");
    GemmArgs a{};
    a.A = d_x; a.lda = d->x_pitch; a.B = d_w; a.ldb = d->w_pitch;
    a.M = d->rows; a.N = d->cout; a.K = d->cin; a.k_per = d->cin;
    a.C = d_y; a.ldc = d->cout; a.alpha = d->scale;
    a.fwd = 1; a.act = d->activation; a.bias = d_bias; a.res = d_residual; a.ldr = d->res_pitch; a.preact = d_preact;
    hipStream_t s = (hipStream_t)stream;
    KTimer t(c, "linear", s);
    const ttc_status st = with_dtype(d->dtype, [&](auto tag) {
        gemm_launch<decltype(tag), true, false>(a, 1, s);
        return TTC_OK;
    });
    TTC_HIP(c, hipGetLastError());
    return st;
}

ttc_status ttc_linear_backward(ttc_ctx* c, const ttc_linear_desc* d, const void* d_dy, const void* d_x, const void* d_w, const void* d_preact,
                               void* d_dx, void* d_dw, float* d_dbias, void* d_ws, size_t ws_bytes, void* stream) {
    if (!c) return TTC_ERR_ARG;
    if (const char* e = linear_check(d)) return c->fail(TTC_ERR_ARG, std::string("linear_backward: ") + e);
    if ((d->rows > 1 && d->dy_pitch < d->cout) || d->dy_pitch > (1L << 30)) return c->fail(TTC_ERR_ARG, "linear_backward: dy_pitch must be at least cout");
    if (!d_dx && !d_dw && !d_dbias) return TTC_OK;
    DeviceGuard dev(c->device);
    if (!dev.ok) return c->fail(TTC_ERR_HIP, "linear_backward: hipSetDevice failed");
    hipStream_t s = (hipStream_t)stream;
    KTimer t(c, "linear_backward", s);
    const ttc_status st = with_dtype(d->dtype, [&](auto tag) {
        using T = decltype(tag);
        if (d->rows == 0) {
            const long n = (long)d->cin * d->cout;
            if (d_dw) hipLaunchKernelGGL((k_fill0<T>), dim3((unsigned)((n + NT - 1) / NT)), dim3(NT), 0, s, (T*)d_dw, n);
            if (d_dbias) hipLaunchKernelGGL((k_fill0<float>), dim3((d->cout + NT - 1) / NT), dim3(NT), 0, s, d_dbias, (long)d->cout);
            return TTC_OK;
        }
        const bool act = d->activation != TTC_ACT_NONE;
        const BwdWs w = linear_ws(d);
        if (!d_dy || (d_dw && !d_x) || (d_dx && !d_w) || (act && !d_preact) || (w.total && !d_ws))
            return c->fail(TTC_ERR_ARG, "linear_backward: null pointer (an activation needs d_preact)");
        if (ws_bytes < w.total) return c->fail(TTC_ERR_ARG, "linear_backward: workspace smaller than ttc_linear_workspace asks for");
        char* ws = (char*)d_ws;
        const T* dz = act ? (const T*)ws : (const T*)d_dy;
        const long dz_pitch = act ? d->cout : d->dy_pitch;
        const float alpha = act ? 1.0f : d->scale;           // without an activation dz is dy itself and the scale moves into the epilogues
        if (act || d_dbias) {
            DzArgs z{};
            z.dy = d_dy; z.z = d_preact; z.dz = act && (d_dx || d_dw) ? ws : nullptr; z.part = d_dbias ? (float*)(ws + w.sums) : nullptr;
            z.rows = d->rows; z.dpitch = d->dy_pitch; z.N = d->cout; z.act = d->activation; z.scale = d->scale;
            const int V = col_vec(d->cout, sizeof(T));
            int blocks, tiles;
            dz_geometry(z, V, &blocks, &tiles);
            auto go = [&](auto fn) { hipLaunchKernelGGL(fn, dim3(blocks, tiles), dim3(NT), (size_t)z.rpb * z.cols * V * sizeof(float), s, z); };
            if (V == 1) go(k_dz<T, 1>);
            else if (V == 2) go(k_dz<T, 2>);
            else if (V == 4) go(k_dz<T, 4>);
            else if constexpr (sizeof(T) == 2) go(k_dz<T, 8>);
            if (d_dbias) hipLaunchKernelGGL(k_col_reduce, dim3((d->cout + 15) / 16), dim3(NT), 0, s, z.part, blocks, d->cout, d_dbias);
        }
        if (d_dx) {
            GemmArgs a{};
            a.A = dz; a.lda = dz_pitch; a.B = d_w; a.ldb = d->w_pitch;
            a.M = d->rows; a.N = d->cin; a.K = d->cout; a.k_per = d->cout;
            a.C = d_dx; a.ldc = d->cin; a.alpha = alpha;
            gemm_launch<T, true, true>(a, 1, s);
        }
        if (d_dw) {
            int sp = dw_splits(d);
            GemmArgs a{};
            a.A = d_x; a.lda = d->x_pitch; a.B = dz; a.ldb = dz_pitch;
            a.M = d->cin; a.N = d->cout; a.K = d->rows;
            const long step = BKE<T>;
            a.k_per = ((d->rows + sp - 1) / sp + step - 1) / step * step;
            sp = (int)((d->rows + a.k_per - 1) / a.k_per);
            a.C = d_dw; a.ldc = d->cout; a.alpha = alpha;
            if (sp > 1) { a.C = ws + w.dw; a.partial = 1; }
            gemm_launch<T, false, false>(a, sp, s);
            if (sp > 1) {
                const long n = (long)d->cin * d->cout;
                hipLaunchKernelGGL((k_gemm_reduce<T>), dim3((unsigned)((n + 63) / 64)), dim3(NT), 0, s, (const float*)(ws + w.dw), sp, n, alpha,
                                   (T*)d_dw);
            }
        }
        return TTC_OK;
    });
    TTC_HIP(c, hipGetLastError());
    return st;
}

}  // extern "C"
