// Product of channels-last rows with a weight matrix, bias, activation and residual in the epilogue -- the 1x1 convolution as an operator of
// its own (the graph's head: src/train/train-model.py:226-231), forward and backward.
//
//   z = x w + b,  y = residual + scale act(z)            x [m, k], w [k, n] (TF layout: the output channel is contiguous)
//   dz = scale dy act'(z);  dx = dz w^T;  dw = x^T dz;  db = column sums of dz
//
// A product is C[i, j] = sum_c A(i, c) B(c, j), where each operand is stored either with the contracted index contiguous ("KC": x and dz in dx, w in dx) or
// with its free index contiguous ("FC": w in y, x and dz in dw).  By size (host code at the end):
//   k_narrow, k_narrow_bwd   up to 128 columns, weights in LDS: bound by the rows' bytes forward in 16 bits; the backward pass in one pass over the rows
//   k_few                    a few rows: bound by reading w
//   k_gemm_wide              many 256 x 256 / 256 x 128 tiles of aligned rows: bound by the matrix cores
//   k_gemm                   everything else; with few tiles the contracted index is split and k_join adds the parts
// All but k_few share the fragments:
//  - KC tiles lie in LDS as rows of 128 bytes; a lane reads 16 bytes = its 8 (16-bit) or 4 (fp32) values of the contracted index.
//  - FC tiles lie in LDS as stored; 16-bit fragments come through the transposing LDS read (ds_read_tr16_b64), fp32 ones through single words.
//  - the contracted index may be permuted freely as long as both operands agree: that is what makes the 16-byte KC read fit the fp32 instruction.
//  - the matrix instruction gets B's fragment first, so a lane ends up with consecutive OUTPUT CHANNELS of one row (8 for 16-bit types: the rows of
//    fragment pairs are interleaved) and stores 16 bytes at a time.
//  - LDS slots are XOR-swizzled against bank conflicts.
#include <algorithm>

#include "layers_common.h"

namespace {
using namespace layers;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int NT = 256;

struct GemmArgs {
    const void* A; const void* B;
    const void* Alo; const void* Blo;   // the low halves of a pair (dz_pair), of A or of B, in the same strides; or none
    long lda, ldb;
    long M; int N; long K;          // C is [M, N], K contracted
    long k_per;                     // contracted range of a split (blockIdx.y)
    void* C; long ldc;              // T, or float partials [split][M][N]
    int partial;
    float alpha;
    // forward epilogue
    int fwd, act;
    const float* bias; const void* res; long ldr; float* preact;
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
    typedef f32x4 Frag;             // 4 values of the contracted index = 4 instructions of 4 (mma_block)
};

// acc[i][j] += b[i] a[j]: the instructions of one accumulator are as far apart as there are accumulators (fp32: four per pair; back to back each waited
// for the one before)
template <class T, int I, int J>
__device__ __forceinline__ void mma_block(f32x4 (&acc)[I][J], const typename Mma<T>::Frag (&b)[I], const typename Mma<T>::Frag (&a)[J]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < I; ++i)
#pragma unroll
                for (int j = 0; j < J; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[i][c], a[j][c], acc[i][j], 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) acc[i][j] = Mma<T>::run(b[i], a[j], acc[i][j]);
    }
}

// dz = dy act'(z) is a 32-bit value and an operand of two products in the arrays' type.  In 16 bits it goes in as the pair hi + lo / LO_UP, multiplied one
// after the other: rounded once instead, dx and dw were 1.4 times as far from their 64-bit values as their own rounding takes them (bf16 2.35e-3 against 1.66e-3).
// The pair holds 16 (bf16) or 22 bits (fp16).  fp16 has a narrow range: the value is halved, so that a slope up to 1.13 does not overflow it, and its low
// half, 11 bits further down, comes up by 2^11, out of the subnormals (smallest piece 2^-35).
// relu's slope is 0 or 1: dz has the arrays' bits as it is, and a low half of 0 would turn the infinite dw of an infinite x into NaN.
template <class T> inline bool dz_is_pair(int act) { return sizeof(T) == 2 && act != TTC_ACT_NONE && act != TTC_ACT_RELU; }
template <class T> constexpr float DZ_DOWN = std::is_same_v<T, f16> ? 0.5f : 1.0f;      // undone by the products' alpha
template <class T> constexpr float LO_UP = std::is_same_v<T, f16> ? 2048.0f : 1.0f;
template <class T>
__device__ __forceinline__ void dz_pair(float v, T* hi, T* lo) {
    *hi = (T)v;
    const float d = (v - (float)*hi) * LO_UP<T>;
    *lo = (T)(fabsf(d) < INFINITY ? d : 0.0f);     // an infinite or NaN v stays in hi alone
}

// the products of the low halves are summed: down to the high ones' scale
template <class T, int I, int J>
__device__ __forceinline__ void lo_done(f32x4 (&acc)[I][J]) {
    if constexpr (LO_UP<T> != 1.0f) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) acc[i][j] *= 1.0f / LO_UP<T>;
    }
}

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

// drop the first `n` elements of 16 bytes (all of them for n >= VE), zeros come in
template <class T>
__device__ __forceinline__ uint4 drop_front(uint4 v, int n) {
    const int bits = min(n, VE<T>) * 8 * (int)sizeof(T);
    unsigned long lo = v.x | (unsigned long)v.y << 32, hi = v.z | (unsigned long)v.w << 32;
    if (bits >= 64) { lo = hi; hi = 0; }
    const int b = bits & 63;
    if (b) { lo = lo >> b | hi << (64 - b); hi >>= b; }
    if (bits >= 128) lo = 0;
    return make_uint4((unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32));
}

// the 16-byte pieces of a BF x BKE tile a thread moves, global -> registers -> LDS.  Inside the array the loads are plain.  In an edge tile a piece that
// sticks out of its row is read so that it ENDS with the row and shifted down, one wholly outside reads something valid and becomes zero: no
// element-by-element path (rows shorter than 16 bytes apart).  The shift happens on the way to LDS, so that the loads stay in flight.
template <class T, bool KC, int BF>
struct Stage {
    static constexpr int CNT = BF * 8 / NT, PR = BF / VE<T>;
    uint4 v[CNT];
    static __device__ __forceinline__ int line(int id) { return KC ? id >> 3 : id / PR; }                      // row of the tile as stored
    static __device__ __forceinline__ int along(int id) { return (KC ? id & 7 : id % PR) * VE<T>; }            // first element in it
    // rows [r0, R), elements [e0, E) of the array remain
    static __device__ __forceinline__ bool edge(long r0, long R, long e0, long E) { return r0 + (KC ? BF : BKE<T>) > R || e0 + (KC ? BKE<T> : BF) > E; }
    __device__ __forceinline__ void load(const T* p, long ld, long f0, long F, long k0, long K, int tid) {
        const long r0 = KC ? f0 : k0, R = KC ? F : K, e0 = KC ? k0 : f0, E = KC ? K : F;
        if (!edge(r0, R, e0, E)) {
            p += r0 * ld + e0;
#pragma unroll
            for (int i = 0; i < CNT; ++i) __builtin_memcpy(&v[i], p + line(tid + i * NT) * ld + along(tid + i * NT), 16);
        } else if (E >= VE<T>) {
#pragma unroll
            for (int i = 0; i < CNT; ++i)
                __builtin_memcpy(&v[i], p + min(r0 + line(tid + i * NT), R - 1) * ld + min(e0 + along(tid + i * NT), E - VE<T>), 16);
        } else {
#pragma unroll
            for (int i = 0; i < CNT; ++i) {
                const long r = r0 + line(tid + i * NT), e = e0 + along(tid + i * NT);
                v[i] = load_piece(p + r * ld + e, r < R ? E - e : 0);
            }
        }
    }
    __device__ __forceinline__ void store(char* lds, long f0, long F, long k0, long K, int tid) const {
        const long r0 = KC ? f0 : k0, R = KC ? F : K, e0 = KC ? k0 : f0, E = KC ? K : F;
        const bool fix = edge(r0, R, e0, E) && E >= VE<T>;
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int id = tid + i * NT;
            uint4 t = v[i];
            if (fix) {
                const long e = e0 + along(id);
                t = drop_front<T>(t, r0 + line(id) < R ? (int)(e - min(e, E - VE<T>)) : VE<T>);
            }
            if (KC) reinterpret_cast<uint4*>(lds)[kc_slot(id >> 3, id & 7)] = t;
            else *reinterpret_cast<uint4*>(lds + fc_byte<T, BF>(line(id), along(id))) = t;
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

// V consecutive columns of one row, `left` of them exist
template <class T, int V>
__device__ __forceinline__ void store_part(T* p, int left, const float (&v)[V]) {
    if (left >= V) { store_vec<T, V>(p, v); return; }
#pragma unroll
    for (int i = 0; i < V; ++i) if (i < left) p[i] = (T)v[i];
}
template <class T, int V>
__device__ __forceinline__ void load_part(const T* p, int left, float (&v)[V]) {
    if (left >= V) { load_vec<T, V>(p, v); return; }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < left ? (float)p[i] : 0.0f;
}
template <class T, int V>
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[V]) {
    T t[V];
    __builtin_memcpy(t, &u, sizeof t);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)t[i];
}
// Whole cache lines for the stores.  A lane holds pieces of ONE row r = lane & 15 of 16: piece a of columns [0, 4V), piece b of [4V, 8V) by its quarter
// q = lane >> 4 -- a store of either would write half lines of 16 rows.  Lanes r and r ^ 8 trade pieces: then a lane has columns of ONE half, for rows
// (r & 7) in a and (r & 7) + 8 in b, and each of the two stores writes 8 whole runs of 8V columns.  (898704 rows, 64 -> 64, bf16: 54.7 -> 45.0 us.)
__device__ __forceinline__ unsigned ror8(unsigned v) { return __builtin_amdgcn_update_dpp(0u, v, 0x128, 0xf, 0xf, false); }
template <class R, int V>
__device__ __forceinline__ void trade(R (&a)[V], R (&b)[V], bool hi) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const unsigned x = __builtin_bit_cast(unsigned, a[i]), y = __builtin_bit_cast(unsigned, b[i]);
        const unsigned got = ror8(hi ? x : y);
        a[i] = __builtin_bit_cast(R, hi ? got : x);
        b[i] = __builtin_bit_cast(R, hi ? y : got);
    }
}
template <class T, int V>
__device__ __forceinline__ void finish(const GemmArgs& a, long row, int col, int left, float (&v)[V], const float (&bias)[V], const float (&res)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += bias[i];
    if (a.preact) store_part<float, V>(a.preact + row * a.ldc + col, left, v);    // in 32 bits: the bias gradient sums slopes taken from it
    if (!a.C) return;
    act_vec<V>(v, a.act);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = v[i] * a.alpha + res[i];
    store_part<T, V>((T*)a.C + row * a.ldc + col, left, v);
}
template <class T, int V>
__device__ __forceinline__ void emit(const GemmArgs& a, long row, int col, int left, float (&v)[V]) {
    if (!a.fwd) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= a.alpha;
        store_part<T, V>((T*)a.C + row * a.ldc + col, left, v);
    } else {
        float bias[V], res[V];
#pragma unroll
        for (int i = 0; i < V; ++i) bias[i] = res[i] = 0.0f;
        if (a.bias) load_part<float, V>(a.bias + col, left, bias);
        if (a.res) load_part<T, V>((const T*)a.res + row * a.ldr + col, left, res);
        finish<T, V>(a, row, col, left, v, bias, res);
    }
}

// A wave's accumulators (FN fragments of columns, FM of rows) from row m0, column n0, through its own piece of LDS (free after the last step), JC row
// fragments at a time.  There a lane finds whole 16-byte runs of a row, its columns (and its bias) the same for every row, and 64 lanes whole lines: no
// trade.  And the epilogue is a LOOP: unrolled over the accumulators, with its five activations, it was 100 KB and more of code that every wave ran once,
// fetched from the L2 (bf16 without activation, 8192 x 1024 -> 4096: 86 -> 77 us, 57600 x 256 -> 256: 25 -> 20).  16-byte slots are XOR-swizzled by row.
template <class T, int FN, int FM, int JC>
__device__ __forceinline__ void store_tile(const GemmArgs& a, const f32x4 (&acc)[FN][FM], long m0, int n0, int lane, char* lds) {
    constexpr int V = VE<T>, WN = FN * 16, CPR = WN / 4, LPR = WN / V, RPI = 64 / LPR;      // slots of a row, lanes of a row, rows of a loop step
    const int r = lane & 15, q = lane >> 4, cl = lane % LPR, rl = lane / LPR;
    const int col = n0 + cl * V, left = a.N - col;
    float bias[V];
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = 0.0f;
    if (a.fwd && a.bias && left > 0) load_part<float, V>(a.bias + col, left, bias);
#pragma unroll
    for (int j0 = 0; j0 < FM; j0 += JC) {
#pragma unroll
        for (int j = 0; j < JC; ++j)
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                const int slot = sizeof(T) == 2 ? 8 * (f >> 1) + 2 * q + (f & 1) : 4 * f + q, row = j * 16 + r;
                *reinterpret_cast<f32x4*>(lds + (row * CPR + (slot ^ (row & (CPR - 1)))) * 16) = acc[f][j0 + j];
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the wave's own piece: LDS serves one wave in order
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int it = 0; it < JC * 16 / RPI; ++it) {
            const int lr = it * RPI + rl;
            const long row = m0 + j0 * 16 + lr;
            float v[V];
#pragma unroll
            for (int u = 0; u < V / 4; ++u) {
                const f32x4 t = *reinterpret_cast<const f32x4*>(lds + (lr * CPR + ((cl * (V / 4) + u) ^ (lr & (CPR - 1)))) * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * u + i] = t[i];
            }
            if (row >= a.M || left <= 0) continue;
            if (a.partial) {
                store_part<float, V>((float*)a.C + ((long)blockIdx.y * a.M + row) * a.N + col, left, v);
            } else if (!a.fwd) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] *= a.alpha;
                store_part<T, V>((T*)a.C + row * a.ldc + col, left, v);
            } else {
                float res[V];
#pragma unroll
                for (int i = 0; i < V; ++i) res[i] = 0.0f;
                if (a.res) load_part<T, V>((const T*)a.res + row * a.ldr + col, left, res);
                finish<T, V>(a, row, col, left, v, bias, res);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- the tile kernel --------------------------------------------------------------------------------------------------------------------
// Any size, alignment and type: 128 (64) rows by 128 (64, 32) columns, 4 waves, two stages of 128-byte steps; tiles pass through registers, where edge pieces
// are trimmed.  Bound by the matrix cores for large sizes (8192 x 1024 -> 4096: fp32 603 us = 114 TFLOP/s, bf16 133 us), by latency for small ones
// (5003 x 177 -> 93 fp16: y 10.0, dx 6.4, dw 8.4 + 4.2 us to join 39 splits).
// PAIR: A or B comes as a pair of 16-bit halves (dz): the range is walked twice, the low halves first
template <class T, bool AKC, bool BKC, int BM, int BN, int WGM, bool PAIR>
__global__ __launch_bounds__(NT) void k_gemm(GemmArgs a) {
    constexpr int WGN = 4 / WGM, WM = BM / WGM, WN = BN / WGN, FM = WM / 16, FN = WN / 16;
    constexpr int ABYTES = BM * 128, BBYTES = BN * 128;
    __shared__ __attribute__((aligned(16))) char lds[2 * (ABYTES + BBYTES)];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WGN, wn = wave % WGN;
    // workgroups go round the 8 XCDs: give each XCD a contiguous run of tiles (column tiles fastest), so that a row tile's re-reads hit its L2
    const int total = a.mt * a.nt, bid = blockIdx.x, xcd = bid & 7, per = total >> 3, rem = total & 7;
    const int tile = xcd * per + min(xcd, rem) + (bid >> 3);
    const long m0 = (long)(tile / a.nt) * BM;
    const int n0 = (tile % a.nt) * BN;
    const long k0 = blockIdx.y * a.k_per, k1 = min(k0 + a.k_per, a.K);
    const T* A = (const T*)(PAIR && a.Alo ? a.Alo : a.A);
    const T* B = (const T*)(PAIR && a.Blo ? a.Blo : a.B);
    bool low = PAIR;
    Stage<T, AKC, BM> sa;
    Stage<T, BKC, BN> sb;
    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    sa.load(A, a.lda, m0, a.M, k0, k1, tid);
    sb.load(B, a.ldb, n0, a.N, k0, k1, tid);
    sa.store(lds, m0, a.M, k0, k1, tid);
    sb.store(lds + 2 * ABYTES, n0, a.N, k0, k1, tid);
    __syncthreads();
    int cur = 0;
    for (long k = k0;; cur ^= 1) {
        const bool turn = low && k + BKE<T> >= k1;           // a pair's last low step: the high halves follow from k0
        const bool more = turn || k + BKE<T> < k1;
        k = turn ? k0 : k + BKE<T>;
        if (PAIR && turn) { A = (const T*)a.A; B = (const T*)a.B; }
        if (more) {
            sa.load(A, a.lda, m0, a.M, k, k1, tid);
            sb.load(B, a.ldb, n0, a.N, k, k1, tid);
        }
        const char* la = lds + cur * ABYTES;
        const char* lb = lds + 2 * ABYTES + cur * BBYTES;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            typename Mma<T>::Frag fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FM; ++j) fa[j] = frag<T, AKC, BM, false>(la, wm * WM, j, ks, lane);
#pragma unroll
            for (int i = 0; i < FN; ++i) fb[i] = frag<T, BKC, BN, true>(lb, wn * WN, i, ks, lane);
            mma_block<T>(acc, fb, fa);
        }
        if (PAIR && turn) { lo_done<T>(acc); low = false; }
        if (more) {                                // the other half was last read before the previous barrier
            sa.store(lds + (cur ^ 1) * ABYTES, m0, a.M, k, k1, tid);
            sb.store(lds + 2 * ABYTES + (cur ^ 1) * BBYTES, n0, a.N, k, k1, tid);
        }
        __syncthreads();
        if (!more) break;
    }
    static_assert(4 * WM * WN * 4 <= 2 * (ABYTES + BBYTES), "the waves' tiles fit the stages");
    store_tile<T, FN, FM, FM>(a, acc, m0 + wm * WM, n0 + wn * WN, lane, lds + wave * (WM * WN * 4));
}

// ---- the wide tile kernel: 256 x 256 (16-bit) or 256 x 128 ------------------------------------------------------------------------------------
// One workgroup of 8 waves per CU, two stages in LDS (16-bit 256 x 256: a wave's 128 x 64 outputs read 24 KB of LDS fragments per step against 64 matrix
// instructions, 3/4 of the LDS rate; 8192 x 4096 x 4096 bf16 measured 1.1 - 1.35 PFLOP/s, the library's product 1.3).  Tiles go from memory to LDS
// without passing registers, 16 bytes a lane; the swizzle is in which piece of its row a lane fetches.  A stage is fetched while the other is
// multiplied; one barrier a step.  Rows and columns past the array fetch the last ones (not stored); the contracted range is whole steps and every row
// 16-byte aligned: other calls take k_gemm.
// The copy is written out because the compiler, which cannot tell the stages apart, waits for every copy in flight before each LDS read.  It has no
// register result; the wait for it is the explicit one in front of the barrier.
template <class T, bool KC, int BF>
struct WideTile {
    static constexpr int CNT = BF / 64, PR = BF / VE<T>, PG = sizeof(T);     // pieces a lane, pieces of a row as stored (FC), pieces of a swizzled run
    unsigned off[CNT];                             // a lane's pieces, bytes from the step's base
    __device__ __forceinline__ void init(long ld, long f0, long F, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int id = (i * 8 + wave) * 64 + lane;
            if (KC) {
                const int row = id >> 3, ch = (id & 7) ^ ((row ^ (row >> 3)) & 7);
                off[i] = (unsigned)min((long)row, F - 1 - f0) * (unsigned)(ld * (long)sizeof(T)) + ch * 16;
            } else {
                const int k = id / PR, c = id % PR, sw = sizeof(T) == 2 ? (k & 3) | ((k >> 1) & 4) : (k >> 2) & 3;
                const int col = ((c / PG) ^ (sw & (BF / 16 - 1))) * 16 + (c % PG) * VE<T>;
                off[i] = (unsigned)k * (unsigned)(ld * (long)sizeof(T)) + (unsigned)min((long)col, F - VE<T> - f0) * (unsigned)sizeof(T);
            }
        }
    }
    __device__ __forceinline__ void fetch(const T* p, long ld, long f0, long k, unsigned lds, int wave) const {
        const T* base = KC ? p + f0 * ld + k : p + k * ld + f0;
#pragma unroll
        for (int i = 0; i < CNT; ++i)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds + (i * 8 + wave) * 1024u), "v"(off[i]), "s"(base) : "memory", "m0");
    }
};
constexpr int WIDE_LDS(int bn) { return 2 * (256 + bn) * 128; }
template <class T, bool AKC, bool BKC, int BN, bool PAIR>
__global__ __launch_bounds__(512) void k_gemm_wide(GemmArgs a) {
    extern __shared__ __attribute__((aligned(16))) char wide_lds[];      // A0 A1 B0 B1
    constexpr int TA = 256 * 128, TB = BN * 128, WGN = BN / 64, WM = 256 / (8 / WGN), FM = WM / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WGN, wn = wave % WGN;
    const int total = a.mt * a.nt, bid = blockIdx.x, xcd = bid & 7, per = total >> 3, rem = total & 7;
    const int tile = xcd * per + min(xcd, rem) + (bid >> 3);
    const long m0 = (long)(tile / a.nt) * 256;
    const int n0 = (tile % a.nt) * BN;
    const long k0 = blockIdx.y * a.k_per, k1 = min(k0 + a.k_per, a.K);
    const T* A = (const T*)(PAIR && a.Alo ? a.Alo : a.A);
    const T* B = (const T*)(PAIR && a.Blo ? a.Blo : a.B);
    bool low = PAIR;
    f32x4 acc[4][FM];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)wide_lds;
    WideTile<T, AKC, 256> ta;
    WideTile<T, BKC, BN> tb;
    ta.init(a.lda, m0, a.M, wave, lane);
    tb.init(a.ldb, n0, a.N, wave, lane);
    ta.fetch(A, a.lda, m0, k0, lds0, wave);
    tb.fetch(B, a.ldb, n0, k0, lds0 + 2 * TA, wave);
    __builtin_amdgcn_s_waitcnt(0x0f70);            // vmcnt(0): this wave's pieces have landed; the barrier makes that everyone's
    __syncthreads();
    int cur = 0;
    for (long k = k0;; cur ^= 1) {
        const bool turn = low && k + BKE<T> >= k1, more = turn || k + BKE<T> < k1;           // as in k_gemm
        k = turn ? k0 : k + BKE<T>;
        if (PAIR && turn) { A = (const T*)a.A; B = (const T*)a.B; }
        if (more) {                                // the other stage was last read before the barrier
            ta.fetch(A, a.lda, m0, k, lds0 + (cur ^ 1) * TA, wave);
            tb.fetch(B, a.ldb, n0, k, lds0 + 2 * TA + (cur ^ 1) * TB, wave);
        }
        const char* la = wide_lds + cur * TA;
        const char* lb = wide_lds + 2 * TA + cur * TB;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            typename Mma<T>::Frag fa[FM], fb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) fb[i] = frag<T, BKC, BN, true>(lb, wn * 64, i, ks, lane);
#pragma unroll
            for (int j = 0; j < FM; ++j) fa[j] = frag<T, AKC, 256, false>(la, wm * WM, j, ks, lane);
            mma_block<T>(acc, fb, fa);
        }
        if (PAIR && turn) { lo_done<T>(acc); low = false; }
        __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
        if (!more) break;
    }
    store_tile<T, 4, FM, FM / 2>(a, acc, m0 + wm * WM, n0 + wn * 64, lane, wide_lds + wave * (WM / 2 * 256));
}

// ---- joining the splits of the contracted index: C = epilogue(sum of the partials), 4 columns a thread, L lanes over the splits -------------------
// part: [splits][rec] floats, the M x N block first; `tail` further floats of a record (the column sums of dz) go to `tail_out`, times alpha
template <class T, int L>
__global__ __launch_bounds__(NT) void k_join(GemmArgs a, const float* __restrict__ part, long rec, int splits, int tail, float* __restrict__ tail_out) {
    constexpr int E = NT / L;
    __shared__ float red[4][E * 4];                    // one partial of each wave
    const int e = threadIdx.x % E, l = threadIdx.x / E;
    const int nv = (a.N + 3) / 4;
    const long vecs = a.M * nv, id = (long)blockIdx.x * E + e;
    long off = 0, row = 0;
    int col = 0, left = 0;
    if (id < vecs) { row = id / nv; col = (int)(id % nv) * 4; off = row * a.N + col; left = min(4, a.N - col); }
    else { col = (int)min((id - vecs) * 4, (long)tail); off = a.M * a.N + col; left = min(4, tail - col); }
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int U = L == 64 ? 8 : 4;                 // loads in flight: past the last split they read it again and are dropped
    auto sum = [&](auto load) {
        for (int k = l; k < splits; k += U * L) {
            float v[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) load(part + min(k + u * L, splits - 1) * rec + off, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] += k + u * L < splits ? v[u][i] : 0.0f;
        }
    };
    if (left == 4) {
        sum([](const float* p, float (&v)[4]) { load_vec<float, 4>(p, v); });
    } else if (left > 0) {
        sum([&](const float* p, float (&v)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = p[min(i, left - 1)];
        });
    }
    if constexpr (L > 1) {                             // a wave holds 64 / E of the L lanes of an output: a tree, then the four waves in order
#pragma unroll
        for (int m = E; m < 64; m <<= 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += __shfl_xor(s[i], m);
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) < E)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[wave][e * 4 + i] = s[i];
        __syncthreads();
        if (l) return;
#pragma unroll
        for (int k = 1; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += red[k][e * 4 + i];
    }
    if (left <= 0) return;
    if (id >= vecs) {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < left) tail_out[col + i] = s[i] * a.alpha;
    } else if (a.C || a.preact) {
        emit<T, 4>(a, row, col, left, s);
    }
}

// ---- a few rows: the weights pass once, straight through the vector ALU ------------------------------------------------------------------
// y of MR rows is bound by reading w (and, for one row, by the launch).  A lane owns 16 bytes of columns and every KL-th row of w, so a workgroup
// covers `lanes` x 16 bytes of columns and the whole contracted index: no partials in memory, one launch.  Narrow column runs give enough
// workgroups; those that share a cache line of w run on one XCD and meet in its L2.  The KL partial sums of a column are a tree in LDS.
// 1 x 1024 -> 4096 bf16: 5.0 us (8.4 MB: 1.7 us at the memory's rate; the rest is the launch and one round of latency).
template <class T, int MR>
__global__ __launch_bounds__(NT) void k_few(GemmArgs a, int lanes) {
    constexpr int V = VE<T>;
    __shared__ float red[NT * MR * V];
    const int total = gridDim.x, bid = blockIdx.x, xcd = bid & 7, per = total >> 3, rem = total & 7;
    const int tile = xcd * per + min(xcd, rem) + (bid >> 3);
    const int tid = threadIdx.x, cl = tid & (lanes - 1), kl = tid / lanes, KL = NT / lanes;
    const int col = (tile * lanes + cl) * V, left = a.N - col;
    float acc[MR][V];
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[m][i] = 0.0f;
    if (left > 0) {
        const T* w = (const T*)a.B + col;
        const T* x = (const T*)a.A;
        const int K = (int)a.K;
        if (left >= V) {
#pragma unroll 8
            for (int k = kl; k < K; k += KL) {
                float wv[V];
                load_vec<T, V>(w + (long)k * a.ldb, wv);
#pragma unroll
                for (int m = 0; m < MR; ++m) {
                    const float xv = (float)x[min((long)m, a.M - 1) * a.lda + k];
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[m][i] += xv * wv[i];
                }
            }
        } else {
            for (int k = kl; k < K; k += KL)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i < left) {
                        const float wv = (float)w[(long)k * a.ldb + i];
#pragma unroll
                        for (int m = 0; m < MR; ++m) acc[m][i] += (float)x[min((long)m, a.M - 1) * a.lda + k] * wv;
                    }
        }
    }
    const int width = lanes * MR * V;                        // [kl][row][column]
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int i = 0; i < V; ++i) red[kl * width + (m * lanes + cl) * V + i] = acc[m][i];
    for (int half = KL / 2; half; half /= 2) {
        __syncthreads();
        for (int i = tid; i < half * width; i += NT) red[i] += red[half * width + i];
    }
    __syncthreads();
    for (int i = tid; i < lanes * MR; i += NT) {
        const int m = i / lanes, c = (tile * lanes + (i & (lanes - 1))) * V;
        if (m >= a.M || c >= a.N) continue;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = red[i * V + j];
        emit<T, V>(a, m, c, a.N - c, v);
    }
}

// ---- narrow products: the weights stay in LDS ------------------------------------------------------------------------------------------------
// x w for cin <= 16-byte steps KS of the contracted index, cout <= 16 FN: bound by the rows' bytes.  A wave takes 16 rows at a time and needs no
// other wave: x goes from memory straight into fragments (a lane's 16 bytes ARE the fragment), the next rows' while this row's products run, and
// only the weights sit in LDS, loaded once per workgroup.  16-row steps read KS * FN KB of LDS per KS KB of x: 1/6 of the LDS rate at the memory's.
// Measured, 898704 rows: 64 -> 64 bf16 with swish and residual 62 - 66 us = 5.2 - 5.6 TB/s, 64 -> 1 fp32 37 us (x partly cached; 44 cold = 5.3 TB/s).
template <class T> constexpr int KSTEP = 4 * VE<T>;           // contracted elements of one fragment step: 32 or 16

// 16 rows of an array: the wave's row 0 is a scalar base, a lane's place in them a 32-bit byte offset that never changes (the narrow kernels take pitches
// up to 2^24 elements).  Rows past the last read the last row: nothing of them is stored or summed.
struct Rows16 {
    const char* p;
    long pitch;                     // bytes
    long rows;
    __device__ __forceinline__ const char* base(long r0) const { return p + min(r0, rows - 1) * pitch; }
    __device__ __forceinline__ unsigned row(long r0, int r) const {      // of row r0 + r, from base(r0)
        const long left = rows - 1 - min(r0, rows - 1);
        return (unsigned)(left >= 15 ? r : min(r, (int)left)) * (unsigned)pitch;
    }
};
template <class T>
__device__ __forceinline__ Rows16 rows16(const void* p, long pitch, long rows) { return {(const char*)p, pitch * (long)sizeof(T), rows}; }

// One row's fragment pieces (zero past K).  A piece that sticks out of the row is read so that it ENDS with the row and shifted down: no lane takes an
// element-by-element path (rows shorter than 16 bytes apart).
// FULL: K is exactly the fragment's width.
template <class T, int KS, bool FULL>
struct RowFrag {
    uint4 v[KS];
    __device__ __forceinline__ void load(const Rows16& a, long r0, int r, int K, int q) {
        const char* p = a.base(r0);
        const unsigned o = a.row(r0, r);
        if (FULL || K == KS * KSTEP<T>) {
#pragma unroll
            for (int s = 0; s < KS; ++s) __builtin_memcpy(&v[s], p + (o + q * 16u) + s * 64, 16);
        } else if (K >= VE<T>) {
#pragma unroll
            for (int s = 0; s < KS; ++s) __builtin_memcpy(&v[s], p + (o + (unsigned)min(s * KSTEP<T> + q * VE<T>, K - VE<T>) * (unsigned)sizeof(T)), 16);
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) v[s] = load_piece((const T*)(p + o), s || q ? 0 : K);
        }
    }
    // after the load has arrived (kept apart from it so that the next rows' loads stay in flight)
    __device__ __forceinline__ void trim(int K, int q) {
        if (FULL || K == KS * KSTEP<T> || K < VE<T>) return;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int c = s * KSTEP<T> + q * VE<T>;
            v[s] = drop_front<T>(v[s], c - min(c, K - VE<T>));
        }
    }
};

// rows x cols of a weight matrix into an FC image [KP][NP], zero outside
template <class T, int NP>
__device__ __forceinline__ void load_image(char* lds, const T* w, long ld, int K, int N, int KP, int tid, int nthreads) {
    constexpr int PR = NP / VE<T>;
    for (int id = tid; id < KP * PR; id += nthreads) {
        const int k = id / PR, f = (id % PR) * VE<T>;
        *reinterpret_cast<uint4*>(lds + fc_byte<T, NP>(k, f)) = load_piece(w + (long)k * ld + f, k < K ? N - f : 0);
    }
}

// FULL: cout is exactly 16 FN and no preact leaves: no lane sits out but in the last rows.  A kernel of its own, because the ragged epilogue's
// addresses and masks cost 50 registers (898704 rows, 64 -> 64 with residual, bf16: 165 registers, 3 waves per SIMD, 77 us against 122, 4 and 65 us).
template <class T, int KS, int FN, bool FULL>
__global__ __launch_bounds__(NT) void k_narrow(GemmArgs a) {
    constexpr int NP = FN * 16;
    constexpr bool PAIR = sizeof(T) == 2 && FN > 1;
    constexpr int V = PAIR ? 8 : 4, NV = NP / (4 * V);        // columns a lane stores at once, such runs per row
    __shared__ __attribute__((aligned(16))) char lw[KS * KSTEP<T> * NP * sizeof(T)];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), K = (int)a.K;
    const long groups = (a.M + 15) / 16, step = (long)gridDim.x * 4;
    long g = (long)blockIdx.x * 4 + wave;
    constexpr int NG = NV == 1 ? 1 : NV / 2, NR = NV == 1 ? 1 : 2;        // column runs of a lane after the trade, rows of each
    const int hi = NV == 1 ? 0 : r >> 3, r0 = NV == 1 ? r : r & 7;
    const int c0 = hi * 4 * V + q * V;                        // first column of a lane's run p: NR * p * 4 V further
    const Rows16 ax = rows16<T>(a.A, a.lda, a.M), ar = rows16<T>(a.res, a.ldr, a.M);
    RowFrag<T, KS, false> x0, x1;
    uint4 res0[NG][NR], res1[NG][NR];                         // V elements of the residual each
    auto load_res = [&](uint4 (&to)[NG][NR], long row) {
        const char* p = ar.base(row);
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            const unsigned o = ar.row(row, r0 + 8 * u) + c0 * (unsigned)sizeof(T);
#pragma unroll
            for (int i = 0; i < NG; ++i) __builtin_memcpy(&to[i][u], p + o + i * NR * 4 * V * (int)sizeof(T), V * sizeof(T));
        }
    };
    x0.load(ax, g * 16, r, K, q);
    if (FULL && a.res) load_res(res0, g * 16);
    load_image<T, NP>(lw, (const T*)a.B, a.ldb, K, a.N, KS * KSTEP<T>, tid, NT);
    float bias[NG][V];
#pragma unroll
    for (int p = 0; p < NG; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int col = NR * p * 4 * V + c0 + i;
            bias[p][i] = a.bias && col < a.N ? a.bias[col] : 0.0f;
        }
    __syncthreads();
    // two register sets in turn: a copy between them would wait for the loads it is there to overlap
    auto rows = [&](RowFrag<T, KS, false>& x, uint4 (&res)[NG][NR], RowFrag<T, KS, false>& nx, uint4 (&nres)[NG][NR]) {
        const long base = g * 16;
        nx.load(ax, base + step * 16, r, K, q);
        if (FULL && a.res) load_res(nres, base + step * 16);
        x.trim(K, q);
        int here = 0;
        // the weights are read from LDS for every 16 rows: kept in registers they cost a wave per SIMD (fp32 64 -> 64: 144 -> 135 us)
        asm volatile("" : "+v"(here));
        f32x4 acc[FN][1];
#pragma unroll
        for (int f = 0; f < FN; ++f) acc[f][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            typename Mma<T>::Frag fw[FN];
            const typename Mma<T>::Frag fx[1] = {__builtin_bit_cast(typename Mma<T>::Frag, x.v[s])};
#pragma unroll
            for (int f = 0; f < FN; ++f) fw[f] = frag<T, false, NP, PAIR>(lw + here, 0, f, s, lane);
            mma_block<T>(acc, fw, fx);
        }
        const int left = (int)min(a.M - base, 16L);
#pragma unroll
        for (int p = 0; p < NG; ++p) {
            float v[NR][V];
#pragma unroll
            for (int u = 0; u < NR; ++u)
#pragma unroll
                for (int i = 0; i < V; ++i) v[u][i] = acc[V == 8 ? 2 * (NR * p + u) + i / 4 : NR * p + u][0][i & 3];
            if constexpr (NR == 2) trade(v[0], v[1], hi);
            const int col = NR * p * 4 * V + c0;
#pragma unroll
            for (int u = 0; u < NR; ++u) {
                if constexpr (FULL) {
                    if (r0 + 8 * u >= left) continue;
#pragma unroll
                    for (int i = 0; i < V; ++i) v[u][i] += bias[p][i];
                    act_vec<V>(v[u], a.act);
                    if (a.res) {
                        float rv[V];
                        unpack<T, V>(res[p][u], rv);
#pragma unroll
                        for (int i = 0; i < V; ++i) v[u][i] = v[u][i] * a.alpha + rv[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < V; ++i) v[u][i] *= a.alpha;
                    }
                    store_vec<T, V>((T*)((char*)a.C + base * NP * (long)sizeof(T) + (unsigned)(((r0 + 8 * u) * NP + col) * (int)sizeof(T))), v[u]);
                    continue;
                }
                const long row = base + r0 + 8 * u;
                if (r0 + 8 * u >= left || col >= a.N) continue;
                float rv[V];
#pragma unroll
                for (int i = 0; i < V; ++i) rv[i] = 0.0f;
                if (a.res) load_part<T, V>((const T*)a.res + row * a.ldr + col, a.N - col, rv);
                finish<T, V>(a, row, col, a.N - col, v[u], bias[p], rv);
            }
        }
        g += step;
    };
    for (;;) {
        if (g >= groups) break;
        rows(x0, res0, x1, res1);
        if (g >= groups) break;
        rows(x1, res1, x0, res0);
    }
}

// ---- narrow products: the whole backward pass in one pass over the rows ----------------------------------------------------------------------
// One wave owns RW rows (the contracted length of one matrix instruction over rows) and does everything for them:
//   z = x w + b again from the x it reads anyway (cheaper than 4 bytes per output to write and read),  dz = dy act'(z),
//   dx = dz w^T: a lane's results of the first product are 8 (4) consecutive columns of one row = exactly the operand fragment of this one,
//   dw += x^T dz: both tiles go through a wave-private piece of LDS and come back transposed; the sums stay in registers for the whole kernel.
// In 16 bits with an activation dz is a pair (dz_pair): the last two products run on its low half too, with the same fragments of w and x.
// x and dy are read once, dx written once; per workgroup one record [cin][cout] + column sums of dz leaves for k_join.  Bound by memory and, with an
// activation, by how few waves its registers leave (2 per SIMD): 898704 x 64 -> 64 bf16 without an activation 73 us = 4.7 TB/s, with swish 94 - 102 (80 - 84 on a
// single rounded dz); fp32 219 - 229 us, 2/3 of the fp32 matrix rate (3 products of 7.4 GFLOP).
struct NarrowBwd {
    const void* x; const void* dy; const void* w; const float* bias; const float* z; void* dx; float* part;
    long M, ldx, ldy, ldw; int K, N, act; float scale;
    int want_dw;
};
// image of w | per wave a tile of x, one of dz, of a pair one of the low halves | bias; at the end the sums of all four waves
template <class T, int KS, int NS, bool PAIR>
constexpr int NARROW_BWD_LDS() {
    const int kp = KS * KSTEP<T>, np = NS * KSTEP<T>, rows = sizeof(T) == 2 ? 32 : 16;
    const int run = (kp * np + 4 * rows * (kp + (PAIR ? 2 : 1) * np)) * (int)sizeof(T) + np * 4, red = (kp * np + np) * 4;
    return run > red ? run : red;
}
// FULL: cin and cout are exactly the padded sides and the preact is formed again (as in k_narrow: no masks, no second set of addresses).
// PAIR: 16-bit with an activation but relu (dz_is_pair).
template <class T, int KS, int NS, bool FULL, bool PAIR>
__global__ __launch_bounds__(NT, KS * NS <= (sizeof(T) == 2 ? 4 : 8) ? 2 : 1) void k_narrow_bwd(NarrowBwd a) {
    constexpr int KP = KS * KSTEP<T>, NP = NS * KSTEP<T>, FK = KP / 16, FN = NP / 16;
    constexpr bool H16 = sizeof(T) == 2;
    static_assert(H16 || !PAIR);
    constexpr int RF = H16 ? 2 : 1, RW = 16 * RF, V = VE<T>;
    typedef typename Mma<T>::Frag Frag;
    constexpr int TX = RW * KP * sizeof(T), TZ = RW * NP * sizeof(T), IMG = KP * NP * sizeof(T);
    extern __shared__ __attribute__((aligned(16))) char lds[];       // NARROW_BWD_LDS
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, q = lane >> 4;
    const Rows16 ax = rows16<T>(a.x, a.ldx, a.M), ad = rows16<T>(a.dy, a.ldy, a.M);
    char* lw = lds;
    char* lx = lds + IMG + wave * (TX + (PAIR ? 2 : 1) * TZ);
    char* lz = lx + TX;                                      // the pair's high tile, then its low one
    const long groups = (a.M + RW - 1) / RW, step = (long)gridDim.x * 4;
    long g = (long)blockIdx.x * 4 + wave;
    RowFrag<T, KS, FULL> x0[RF], x1[RF];
    RowFrag<T, NS, FULL> d0[RF], d1[RF];
#pragma unroll
    for (int h = 0; h < RF; ++h) {
        x0[h].load(ax, g * RW + h * 16, r, a.K, q);
        d0[h].load(ad, g * RW + h * 16, r, a.N, q);
    }
    load_image<T, NP>(lw, (const T*)a.w, a.ldw, a.K, a.N, KP, tid, NT);
    float* lb = reinterpret_cast<float*>(lds + IMG + 4 * (TX + (PAIR ? 2 : 1) * TZ));        // bias: beside the sums its registers spill
    for (int i = tid; i < NP; i += NT) lb[i] = a.bias && i < a.N ? a.bias[i] : 0.0f;
    float db[NS][V];
#pragma unroll
    for (int p = 0; p < NS; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) db[p][i] = 0.0f;
    f32x4 dw[FN][FK];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FK; ++j) dw[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    // two register sets in turn: a copy between them would wait for the loads it is there to overlap
    auto rows = [&](RowFrag<T, KS, FULL> (&x)[RF], RowFrag<T, NS, FULL> (&d)[RF], RowFrag<T, KS, FULL> (&nx)[RF], RowFrag<T, NS, FULL> (&nd)[RF]) {
#pragma unroll
        for (int h = 0; h < RF; ++h) {
            nx[h].load(ax, (g + step) * RW + h * 16, r, a.K, q);
            nd[h].load(ad, (g + step) * RW + h * 16, r, a.N, q);
        }
#pragma unroll
        for (int h = 0; h < RF; ++h) {
            const long row = g * RW + h * 16 + r;
            x[h].trim(a.K, q);
            d[h].trim(a.N, q);
            const int left = (int)max(min(a.M - (g * RW + h * 16), 16L), 0L);
            if (r >= left) {                                 // no row there: nothing of what was read instead may reach dw (0 x inf is not 0)
#pragma unroll
                for (int p = 0; p < NS; ++p) d[h].v[p] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int s = 0; s < KS; ++s) x[h].v[s] = make_uint4(0, 0, 0, 0);
            }
            Frag dz[NS], dl[NS];                             // dl: the pair's low halves
            if (!PAIR && a.act == TTC_ACT_NONE) {
#pragma unroll
                for (int p = 0; p < NS; ++p) {
                    dz[p] = __builtin_bit_cast(Frag, d[h].v[p]);
#pragma unroll
                    for (int i = 0; i < V; ++i) db[p][i] += (float)dz[p][i];
                }
            } else {
                f32x4 z[FN][1];
                if (!FULL && a.z) {
#pragma unroll
                    for (int p = 0; p < NS; ++p) {
                        const int col = p * KSTEP<T> + q * V, cols = r < left ? a.N - col : 0;
#pragma unroll
                        for (int u = 0; u < V / 4; ++u) {
                            const uint4 t = load_piece(a.z + row * a.N + col + 4 * u, (long)cols - 4 * u);
                            z[p * (V / 4) + u][0] = __builtin_bit_cast(f32x4, t);
                        }
                    }
                } else {
#pragma unroll
                    for (int f = 0; f < FN; ++f) z[f][0] = *reinterpret_cast<const f32x4*>(lb + (H16 ? 32 * (f >> 1) + 8 * q + 4 * (f & 1) : 16 * f + 4 * q));
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        Frag fw[FN];
                        const Frag fr[1] = {__builtin_bit_cast(Frag, x[h].v[s])};
#pragma unroll
                        for (int f = 0; f < FN; ++f) fw[f] = frag<T, false, NP, true>(lw, 0, f, s, lane);
                        mma_block<T>(z, fw, fr);
                    }
                }
#pragma unroll
                for (int p = 0; p < NS; ++p) {
                    const Frag dv = __builtin_bit_cast(Frag, d[h].v[p]);
                    float t[V], zz[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) { t[i] = (float)dv[i]; zz[i] = z[H16 ? 2 * p + i / 4 : p][0][i & 3]; }
                    slope_vec<V>(t, zz, H16 && !PAIR ? TTC_ACT_RELU : a.act);
                    int cols = FULL ? V : a.N - p * KSTEP<T> - q * V;
                    if (!FULL) asm volatile("" : "+v"(cols));           // compared where it is used: as masks kept over the loop it is 16 registers
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        // a padded column: its zero weights make z NaN where x is infinite, and that times its zero dy would reach every dx of the row
                        if (!FULL && i >= cols) t[i] = 0.0f;
                        if (PAIR) t[i] *= DZ_DOWN<T>;
                        db[p][i] += t[i];
                        if constexpr (PAIR) {
                            T hi, lo;
                            dz_pair<T>(t[i], &hi, &lo);
                            dz[p][i] = hi; dl[p][i] = lo;
                        } else {
                            dz[p][i] = (T)t[i];
                        }
                    }
                }
            }
            if (a.dx) {
                f32x4 o[FK][1];
#pragma unroll
                for (int f = 0; f < FK; ++f) o[f][0] = f32x4{0.f, 0.f, 0.f, 0.f};
                auto times_w = [&](const Frag (&z)[NS]) {
#pragma unroll
                    for (int p = 0; p < NS; ++p) {
                        Frag fw[FK];
                        const Frag fr[1] = {z[p]};
#pragma unroll
                        for (int f = 0; f < FK; ++f)
                            fw[f] = __builtin_bit_cast(Frag, *reinterpret_cast<const uint4*>(lw + fc_byte<T, NP>(free_of<T, true>(f, r), p * KSTEP<T> + q * V)));
                        mma_block<T>(o, fw, fr);
                    }
                };
                if constexpr (PAIR) { times_w(dl); lo_done<T>(o); }
                times_w(dz);
                const int hi = KS == 1 ? 0 : r >> 3;
#pragma unroll
                for (int p = 0; p < KS; p += 2) {
                    unsigned v[2][4];
#pragma unroll
                    for (int u = 0; u < (KS == 1 ? 1 : 2); ++u) {
                        T t[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) t[i] = (T)(o[H16 ? 2 * (p + u) + i / 4 : p + u][0][i & 3] * a.scale);
                        __builtin_memcpy(v[u], t, 16);
                    }
                    if constexpr (KS > 1) trade(v[0], v[1], hi);
                    const int col = (p + hi) * KSTEP<T> + q * V;
#pragma unroll
                    for (int u = 0; u < (KS == 1 ? 1 : 2); ++u) {
                        const int rr = KS == 1 ? r : (r & 7) + 8 * u;
                        if (rr >= left) continue;
                        if constexpr (FULL) {
                            __builtin_memcpy((char*)a.dx + (g * RW + h * 16) * KP * (long)sizeof(T) + (unsigned)((rr * KP + col) * (int)sizeof(T)), v[u], 16);
                            continue;
                        }
                        if (col >= a.K) continue;
                        T* out = (T*)a.dx + (g * RW + h * 16 + rr) * a.K + col;
                        if (col + V <= a.K) { __builtin_memcpy(out, v[u], 16); continue; }
                        T t[V];
                        __builtin_memcpy(t, v[u], 16);
#pragma unroll
                        for (int i = 0; i < V; ++i) if (col + i < a.K) out[i] = t[i];
                    }
                }
            }
            if (a.want_dw) {
#pragma unroll
                for (int s = 0; s < KS; ++s) *reinterpret_cast<uint4*>(lx + fc_byte<T, KP>(h * 16 + r, s * KSTEP<T> + q * V)) = x[h].v[s];
#pragma unroll
                for (int p = 0; p < NS; ++p) *reinterpret_cast<uint4*>(lz + fc_byte<T, NP>(h * 16 + r, p * KSTEP<T> + q * V)) = __builtin_bit_cast(uint4, dz[p]);
                if constexpr (PAIR)
#pragma unroll
                    for (int p = 0; p < NS; ++p) *reinterpret_cast<uint4*>(lz + TZ + fc_byte<T, NP>(h * 16 + r, p * KSTEP<T> + q * V)) = __builtin_bit_cast(uint4, dl[p]);
            }
        }
        if (a.want_dw) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the tiles are this wave's own: LDS serves one wave in order
            __builtin_amdgcn_wave_barrier();
            Frag fx[FK];
#pragma unroll
            for (int j = 0; j < FK; ++j) fx[j] = frag<T, false, KP, false>(lx, 0, j, 0, lane);
            Frag fz[FN];
#pragma unroll
            for (int i = 0; i < FN; ++i) fz[i] = frag<T, false, NP, false>(lz, 0, i, 0, lane);
            mma_block<T>(dw, fz, fx);
            if constexpr (PAIR) {
                // the low halves' scale goes to x here: a scaled copy of the sums would cost their registers again.  x 2^-11 is exact down to 2^-3 and
                // off by at most 2^-25, on a term that is 2^-11 of the high one.
                if constexpr (LO_UP<T> != 1.0f)
#pragma unroll
                    for (int j = 0; j < FK; ++j) fx[j] *= (T)(1.0f / LO_UP<T>);
#pragma unroll
                for (int i = 0; i < FN; ++i) fz[i] = frag<T, false, NP, false>(lz + TZ, 0, i, 0, lane);
                mma_block<T>(dw, fz, fx);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        g += step;
    };
    for (;;) {
        if (g >= groups) break;
        rows(x0, d0, x1, d1);
        if (g >= groups) break;
        rows(x1, d1, x0, d0);
    }
    if (!a.part) return;
    // the four waves' sums, in wave order: column sums over the 16 rows of a lane column first
    float* red = reinterpret_cast<float*>(lds);
    float* rdb = red + KP * NP;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1)
#pragma unroll
        for (int p = 0; p < NS; ++p)
#pragma unroll
            for (int i = 0; i < V; ++i) db[p][i] += __shfl_xor(db[p][i], m);
    for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (wave != w) continue;
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FK; ++j) {
                f32x4* c = reinterpret_cast<f32x4*>(red + (16 * j + r) * NP + 16 * i + 4 * q);
                *c = w ? *c + dw[i][j] : dw[i][j];
            }
        if (r == 0)
#pragma unroll
            for (int p = 0; p < NS; ++p)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float* c = rdb + p * KSTEP<T> + q * V + i;
                    *c = w ? *c + db[p][i] : db[p][i];
                }
    }
    __syncthreads();
    float* out = a.part + (long)blockIdx.x * ((long)a.K * a.N + a.N);
    for (int i = tid; i < KP * NP; i += NT) {
        const int k = i / NP, n = i % NP;
        if (k < a.K && n < a.N) out[k * a.N + n] = red[i];
    }
    for (int n = tid; n < a.N; n += NT) out[a.K * a.N + n] = rdb[n];
}

// ---- wide backward: dz = dy act'(z), and the column sums of dz -----------------------------------------------------------------------------------
// Bound by memory: 57600 x 128 fp32 17 - 21 us = 4.2 - 5.3 TB/s (the plain products then read dz twice; forming it inside them would read dy and z as often).
struct DzArgs {
    const void* dy; const float* z; void* dz; void* lo; float* part;      // lo: the pair's low halves (16-bit types)
    long rows, dpitch; int N, act;
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
    if (rl < a.rpb && c0 < a.N) {
        const T* dy = (const T*)a.dy + c0;
#pragma unroll 4
        for (long r = r0 + rl; r < r1; r += a.rpb) {
            float d[V], z[V];
            load_vec<T, V>(dy + r * a.dpitch, d);
            if (a.act != TTC_ACT_NONE) {
                load_vec<float, V>(a.z + r * a.N + c0, z);
                slope_vec<V>(d, z, a.act);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] += d[i];
            if (!a.dz) continue;
            if (sizeof(T) == 4 || !a.lo) {
                store_vec<T, V>((T*)a.dz + r * a.N + c0, d);
            } else {
                T hi[V], lo[V];
#pragma unroll
                for (int i = 0; i < V; ++i) dz_pair<T>(d[i] * DZ_DOWN<T>, &hi[i], &lo[i]);
                __builtin_memcpy((T*)a.dz + r * a.N + c0, hi, sizeof hi);
                __builtin_memcpy((T*)a.lo + r * a.N + c0, lo, sizeof lo);
            }
        }
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
template <class T>
__global__ void k_fill0(T* p, long n) {
    for (long i = (long)blockIdx.x * NT + threadIdx.x; i < n; i += (long)gridDim.x * NT) p[i] = (T)0.0f;
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------
int bn_of(long N) { return N <= 32 ? 32 : N <= 64 ? 64 : 128; }       // column tile: narrower only where the wide one would be mostly padding
// row tile: 64 rows where 128 would leave CUs without a tile (5003 x 93 -> 177: 8.7 -> 6.2 us; but 8192 x 1024 -> 4096: 133 -> 159, twice the reads of w)
int bm_of(long M, long N) { return bn_of(N) == 128 && ((M + 127) / 128) * ((N + 127) / 128) < 256 ? 64 : 128; }
// the wide kernel's columns (0: not for this product): 256 for 16-bit types where its tiles fill the CUs, or do with the contracted index split into
// runs of at least 1024; 128 where those fill most of them (4096 x 1024 -> 1024, 128 tiles: bf16 25 -> 20 us, but fp32, bound by the matrix cores, 94 -> 129)
constexpr long WIDE_PITCH = 1L << 21;                         // 256 rows of them fit a 32-bit byte offset
long wide_tiles(long M, long N, long bn) { return ((M + 255) / 256) * ((N + bn - 1) / bn); }
int wide_cols(long M, long N, long K, int bytes) {
    if (K % (128 / bytes) || M < 256 || N < 128) return 0;
    const long runs = std::max<long>(1, K / 1024);
    if (bytes == 2 && N >= 256 && wide_tiles(M, N, 256) * runs >= 192) return 256;
    return wide_tiles(M, N, 128) >= (bytes == 2 ? 96 : 192) ? 128 : 0;
}
// how many ways the contracted index is split: one where the tiles fill the CUs; else so that one workgroup per CU runs, two where the index is long
// (4096 x 1024 -> 1024 bf16: y 23 us with one, 34 with two; dw of 65536 x 512 -> 256: 76 us with one, 56 with two), and the partials stay under 64 MB.
// A split and its join cost about 5 us.  16-bit products below 384 take none (dx of 1000 x 1024 -> 256: 7.0 us against 12.7) and up to 4096 as many as
// keep the partials under 4 MB (64 x 1024 -> 4096: 12.0 us by four, 13.9 by eight), two of a thousand in any case (dw of 1500 x 1000 -> 1000: 23 us against
// 31); fp32, with a quarter of their matrix rate, splits down to 64 (64 x 512 -> 512: 9.8 us against 12.0 at 128; 16 x 1024 -> 4096 by eight 14, four 19)
int gemm_splits(long M, long N, long K, int bytes) {
    const long bytes_one = M * N * 4;
    long fit = std::max<long>(1, (64L << 20) / bytes_one);
    if (const int wn = wide_cols(M, N, K, bytes)) return (int)std::max<long>(1, std::min<long>({256 / wide_tiles(M, N, wn), K / 1024, fit}));
    if (bytes == 2 && K < 384) return 1;
    if (bytes == 2 && K <= 4096) fit = std::min(fit, std::max<long>(K >= 1024 ? 2 : 1, (4L << 20) / bytes_one));
    const long bm = bm_of(M, N), tiles = ((M + bm - 1) / bm) * ((N + bn_of(N) - 1) / bn_of(N));
    return (int)std::max<long>(1, std::min<long>({(K > 4096 ? 512 : 256) / tiles, K / (bytes == 2 ? 128 : 64), fit}));
}

template <class T>
void join_launch(const GemmArgs& a, const float* part, long rec, int splits, int tail, float* tail_out, hipStream_t s) {
    const long vecs = a.M * ((a.N + 3) / 4) + (tail + 3) / 4;
    // more lanes on the splits where there are few outputs to spread over the chip
    if (splits > 128 && vecs < 2048) hipLaunchKernelGGL((k_join<T, 64>), dim3((unsigned)((vecs + 3) / 4)), dim3(NT), 0, s, a, part, rec, splits, tail, tail_out);
    else if (splits > 16) hipLaunchKernelGGL((k_join<T, 16>), dim3((unsigned)((vecs + 15) / 16)), dim3(NT), 0, s, a, part, rec, splits, tail, tail_out);
    else hipLaunchKernelGGL((k_join<T, 1>), dim3((unsigned)((vecs + NT - 1) / NT)), dim3(NT), 0, s, a, part, rec, splits, tail, tail_out);
}

// C = epilogue(A B) by tiles; ws: splits * M * N floats when splits > 1
template <class T, bool AKC, bool BKC, bool PAIR = false>
void gemm_launch(GemmArgs a, int splits, float* ws, hipStream_t s) {
    if constexpr (sizeof(T) == 2 && AKC == BKC && !PAIR)     // dx, dw
        if (a.Alo || a.Blo) return gemm_launch<T, AKC, BKC, true>(a, splits, ws, s);
    GemmArgs j = a;
    a.k_per = a.K;
    if (splits > 1) {
        a.k_per = ((a.K + splits - 1) / splits + BKE<T> - 1) / BKE<T> * BKE<T>;
        splits = (int)((a.K + a.k_per - 1) / a.k_per);
    }
    if (splits > 1) { a.C = ws; a.partial = 1; }
    if (const int wn = wide_cols(a.M, a.N, a.K, sizeof(T));
        wn && a.lda % VE<T> == 0 && a.ldb % VE<T> == 0 && a.lda <= WIDE_PITCH && a.ldb <= WIDE_PITCH && (uintptr_t)a.A % 16 == 0 && (uintptr_t)a.B % 16 == 0
        && (AKC || a.M % VE<T> == 0) && (BKC || a.N % VE<T> == 0)) {
        auto go = [&](auto fn, LdsConfig& cfg) {
            if (cfg.ensure(fn, WIDE_LDS(wn)) != hipSuccess) {
                (void)hipGetLastError();                     // the LDS size was refused: the smaller tiles do it
                return false;
            }
            a.mt = (int)((a.M + 255) / 256);
            a.nt = (a.N + wn - 1) / wn;
            hipLaunchKernelGGL(fn, dim3((unsigned)(a.mt * a.nt), splits), dim3(512), WIDE_LDS(wn), s, a);
            if (splits > 1) join_launch<T>(j, ws, a.M * a.N, splits, 0, nullptr, s);
            return true;
        };
        static LdsConfig c128, c256;
        if (wn == 128 && go(k_gemm_wide<T, AKC, BKC, 128, PAIR>, c128)) return;
        if constexpr (sizeof(T) == 2)
            if (wn == 256 && go(k_gemm_wide<T, AKC, BKC, 256, PAIR>, c256)) return;
    }
    const int bn = bn_of(a.N), bm = bm_of(a.M, a.N);
    a.mt = (int)((a.M + bm - 1) / bm);
    a.nt = (a.N + bn - 1) / bn;
    auto go = [&](auto fn) { hipLaunchKernelGGL(fn, dim3((unsigned)(a.mt * a.nt), splits), dim3(NT), 0, s, a); };
    if (bn == 32) go(k_gemm<T, AKC, BKC, 128, 32, 4, PAIR>);
    else if (bn == 64) go(k_gemm<T, AKC, BKC, 128, 64, 2, PAIR>);
    else if (bm == 64) go(k_gemm<T, AKC, BKC, 64, 128, 1, PAIR>);
    else go(k_gemm<T, AKC, BKC, 128, 128, 2, PAIR>);
    if (splits > 1) join_launch<T>(j, ws, a.M * a.N, splits, 0, nullptr, s);
}

// the narrow kernels: weights of at most 32 KB as an LDS image whose padded sides are powers of two of 16-byte steps (57600 x 256 -> 128 bf16, 64 KB:
// 32 us against 15 by tiles)
int pow2_at_least(int v) { int p = 1; while (p < v) p *= 2; return p; }
constexpr long NARROW_PITCH = 1L << 24;                       // 15 rows of them fit a 32-bit byte offset
bool narrow_fwd(const ttc_linear_desc* d) {
    if (d->x_pitch > NARROW_PITCH || d->res_pitch > NARROW_PITCH) return false;
    const int step = d->dtype == TTC_DT_F32 ? 16 : 32;
    return d->cin <= 8 * step && d->cout <= 128 && pow2_at_least((d->cin + step - 1) / step) * pow2_at_least((d->cout + 15) / 16) <= 32;
}
bool narrow_bwd(const ttc_linear_desc* d) {
    if (d->x_pitch > NARROW_PITCH || d->dy_pitch > NARROW_PITCH) return false;
    if (d->dtype == TTC_DT_F32) return d->cin <= 64 && d->cout <= 64;
    return d->cin <= 128 && d->cout <= 128 && (d->cin <= 64 || d->cout <= 64);
}
template <class T, int KS>
void narrow_launch_k(const GemmArgs& a, hipStream_t s) {
    const long groups = (a.M + 15) / 16;
    const dim3 grid((unsigned)std::min<long>((groups + 3) / 4, 2048));
    auto go = [&](auto fn) {
        constexpr int FN = decltype(fn)::value;
        if (a.N == FN * 16 && !a.preact) hipLaunchKernelGGL((k_narrow<T, KS, FN, true>), grid, dim3(NT), 0, s, a);
        else hipLaunchKernelGGL((k_narrow<T, KS, FN, false>), grid, dim3(NT), 0, s, a);
    };
    if (a.N <= 16) go(std::integral_constant<int, 1>{});
    else if (a.N <= 32) go(std::integral_constant<int, 2>{});
    else if (a.N <= 64) go(std::integral_constant<int, 4>{});
    else if constexpr (KS < 8) go(std::integral_constant<int, 8>{});         // weights of at most 32 KB
}
template <class T>
void narrow_launch(const GemmArgs& a, hipStream_t s) {
    const int ks = (int)((a.K + KSTEP<T> - 1) / KSTEP<T>);
    if (ks <= 1) narrow_launch_k<T, 1>(a, s);
    else if (ks <= 2) narrow_launch_k<T, 2>(a, s);
    else if (ks <= 4) narrow_launch_k<T, 4>(a, s);
    else narrow_launch_k<T, 8>(a, s);
}
// a few rows that are not narrow: k_few.  1024 -> 4096, us by k_few / by split tiles: bf16 1 row 5.0 / 9.2, 4 rows 7.2 / 8.1, 8 rows 10.0 / 8.1;
// fp32 8 rows 8.8 / 13.5 (half the columns a lane, so half the sums a row costs it)
bool few_rows(const ttc_linear_desc* d) { return d->rows <= (d->dtype == TTC_DT_F32 ? 8 : 4) && !narrow_fwd(d); }
template <class T>
void few_launch(const GemmArgs& a, hipStream_t s) {
    const long runs = (a.N + VE<T> - 1) / VE<T>;             // 16-byte column runs
    int lanes = 2;                                           // 32 bytes of columns a workgroup, wider where that makes more than 1024 of them
    while (lanes < 64 && runs / lanes > 1024) lanes *= 2;
    const dim3 grid((unsigned)((runs + lanes - 1) / lanes));
    if (a.M <= 1) hipLaunchKernelGGL((k_few<T, 1>), grid, dim3(NT), 0, s, a, lanes);
    else if (a.M <= 2) hipLaunchKernelGGL((k_few<T, 2>), grid, dim3(NT), 0, s, a, lanes);
    else if (a.M <= 4) hipLaunchKernelGGL((k_few<T, 4>), grid, dim3(NT), 0, s, a, lanes);
    else if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((k_few<T, 8>), grid, dim3(NT), 0, s, a, lanes);
}
int narrow_bwd_blocks(const ttc_linear_desc* d) {
    const long rw = d->dtype == TTC_DT_F32 ? 64 : 128;        // rows of a workgroup's step
    return (int)std::min<long>((d->rows + rw - 1) / rw, 512);
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
    const long want = std::max<long>(1, 1024 / *tiles), most = std::max<long>(1, a.rows / (4L * a.rpb));
    const long b = std::min(want, most);
    a.rows_per = std::max<long>(1, (a.rows + b - 1) / b);
    *blocks = (int)((a.rows + a.rows_per - 1) / a.rows_per);
}

// workspace of the backward pass: z (where it is formed again) | dz | its low halves (16-bit types) | column sums | partial products, each 256-byte aligned
struct BwdWs { size_t dz, lo, sums, part, total; int blocks, dx_splits, dw_splits; };
BwdWs linear_ws(const ttc_linear_desc* d, bool have_z) {
    const auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    BwdWs w{};
    const size_t cells = (size_t)d->rows * d->cout;
    if (narrow_bwd(d)) {
        w.blocks = narrow_bwd_blocks(d);
        w.total = (size_t)w.blocks * ((size_t)d->cin * d->cout + d->cout) * sizeof(float);
        return w;
    }
    const bool act = d->activation != TTC_ACT_NONE;
    DzArgs z{};
    z.rows = d->rows; z.N = d->cout;
    int tiles;
    dz_geometry(z, col_vec(d->cout, dtype_bytes(d->dtype)), &w.blocks, &tiles);
    w.dz = act && !have_z ? up(cells * sizeof(float)) : 0;
    w.lo = w.dz + (act ? up(cells * dtype_bytes(d->dtype)) : 0);
    w.sums = w.lo + (d->dtype != TTC_DT_F32 && dz_is_pair<f16>(d->activation) ? up(cells * 2) : 0);
    w.part = w.sums + up((size_t)w.blocks * d->cout * sizeof(float));
    const size_t zs = act && !have_z ? (size_t)gemm_splits(d->rows, d->cout, d->cin, dtype_bytes(d->dtype)) : 1;
    w.dx_splits = gemm_splits(d->rows, d->cin, d->cout, dtype_bytes(d->dtype));
    w.dw_splits = gemm_splits(d->cin, d->cout, d->rows, dtype_bytes(d->dtype));
    size_t part = 0;
    if (zs > 1) part = zs * cells;
    if (w.dx_splits > 1) part = std::max(part, (size_t)w.dx_splits * d->rows * d->cin);
    if (w.dw_splits > 1) part = std::max(part, (size_t)w.dw_splits * d->cin * d->cout);
    w.total = w.part + part * sizeof(float);
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
GemmArgs fwd_args(const ttc_linear_desc* d, const void* x, const void* w) {
    GemmArgs a{};
    a.A = x; a.lda = d->x_pitch; a.B = w; a.ldb = d->w_pitch;
    a.M = d->rows; a.N = d->cout; a.K = d->cin; a.ldc = d->cout;
    return a;
}

template <class T>
void dz_launch(const DzArgs& z, int V, int blocks, int tiles, hipStream_t s) {
    auto go = [&](auto fn) { hipLaunchKernelGGL(fn, dim3(blocks, tiles), dim3(NT), (size_t)z.rpb * z.cols * V * sizeof(float), s, z); };
    if (V == 1) go(k_dz<T, 1>);
    else if (V == 2) go(k_dz<T, 2>);
    else if (V == 4) go(k_dz<T, 4>);
    else if constexpr (sizeof(T) == 2) go(k_dz<T, 8>);
}

template <class T>
hipError_t narrow_bwd_launch(const NarrowBwd& a, int blocks, hipStream_t s) {
    auto launch = [&](auto fn, int lds, LdsConfig& cfg) {
        if (const hipError_t e = cfg.ensure(fn, lds); e != hipSuccess) return e;
        hipLaunchKernelGGL(fn, dim3(blocks), dim3(NT), lds, s, a);
        return hipSuccess;
    };
    auto go = [&](auto ks, auto ns) {
        constexpr int KS = decltype(ks)::value, NS = decltype(ns)::value;
        auto pick = [&](auto pair) {
            constexpr bool PAIR = decltype(pair)::value;
            static LdsConfig full, ragged;
            if (a.K == KS * KSTEP<T> && a.N == NS * KSTEP<T> && !a.z) return launch(k_narrow_bwd<T, KS, NS, true, PAIR>, NARROW_BWD_LDS<T, KS, NS, PAIR>(), full);
            return launch(k_narrow_bwd<T, KS, NS, false, PAIR>, NARROW_BWD_LDS<T, KS, NS, PAIR>(), ragged);
        };
        if constexpr (sizeof(T) == 2)
            if (dz_is_pair<T>(a.act)) return pick(std::true_type{});
        return pick(std::false_type{});
    };
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 4> four{};
    const int half = 2 * KSTEP<T>;
    if constexpr (sizeof(T) == 2)                  // a head: half the padding (898704 x 64 -> 1 sigmoid 121 us -> 70, 64 -> 32 swish 154 -> 59)
        if (a.K <= half && a.N <= KSTEP<T>) return go(two, std::integral_constant<int, 1>{});
    if (a.K <= half && a.N <= half) return go(two, two);
    if (a.K <= half) return go(two, four);
    if (a.N <= half) return go(four, two);
    if constexpr (sizeof(T) == 4) return go(four, four);
    return hipErrorInvalidValue;                   // narrow_bwd has no such sizes
}

}  // namespace

extern "C" {

ttc_status ttc_linear_workspace(const ttc_linear_desc* d, int32_t backward, size_t* bytes) {
    if (!bytes) return TTC_ERR_ARG;
    *bytes = 0;
    if (linear_check(d)) return TTC_ERR_ARG;
    if (d->rows == 0) return TTC_OK;
    if (backward) { *bytes = linear_ws(d, backward == TTC_LINEAR_HAVE_PREACT).total; return TTC_OK; }
    const int sp = narrow_fwd(d) || few_rows(d) ? 1 : gemm_splits(d->rows, d->cout, d->cin, dtype_bytes(d->dtype));
    if (sp > 1) *bytes = (size_t)sp * d->rows * d->cout * sizeof(float);
    return TTC_OK;
}

int32_t ttc_linear_wants_preact(const ttc_linear_desc* d) {
    return !linear_check(d) && d->activation != TTC_ACT_NONE && !narrow_bwd(d);
}

ttc_status ttc_linear(ttc_ctx* c, const ttc_linear_desc* d, const void* d_x, const void* d_w, const float* d_bias, const void* d_residual,
                      void* d_y, float* d_preact, void* d_ws, size_t ws_bytes, void* stream) {
    if (!c) return TTC_ERR_ARG;
    if (const char* e = linear_check(d)) return c->fail(TTC_ERR_ARG, std::string("linear: ") + e);
    if (d_residual && ((d->rows > 1 && d->res_pitch < d->cout) || d->res_pitch > (1L << 30)))
        return c->fail(TTC_ERR_ARG, "linear: res_pitch must be at least cout");
    if (d->rows == 0) return TTC_OK;
    const bool narrow = narrow_fwd(d), few = few_rows(d);
    const int sp = narrow || few ? 1 : gemm_splits(d->rows, d->cout, d->cin, dtype_bytes(d->dtype));
    if (!d_x || !d_w || !d_y || (sp > 1 && !d_ws)) return c->fail(TTC_ERR_ARG, "linear: null pointer");
    if (sp > 1 && (uintptr_t)d_ws % 16) return c->fail(TTC_ERR_ARG, "linear: the workspace must be 16-byte aligned");
    if (sp > 1 && ws_bytes < (size_t)sp * d->rows * d->cout * sizeof(float))
        return c->fail(TTC_ERR_ARG, "linear: workspace smaller than ttc_linear_workspace asks for");
    DeviceGuard dev(c->device);
    if (!dev.ok) return c->fail(TTC_ERR_HIP, "linear: hipSetDevice failed");
    GemmArgs a = fwd_args(d, d_x, d_w);
    a.C = d_y; a.alpha = d->scale;
    a.fwd = 1; a.act = d->activation; a.bias = d_bias; a.res = d_residual; a.ldr = d->res_pitch; a.preact = d_preact;
    hipStream_t s = (hipStream_t)stream;
    KTimer t(c, "linear", s);
    const ttc_status st = with_dtype(d->dtype, [&](auto tag) {
        using T = decltype(tag);
        if (narrow) narrow_launch<T>(a, s);
        else if (few) few_launch<T>(a, s);
        else gemm_launch<T, true, false>(a, sp, (float*)d_ws, s);
        return TTC_OK;
    });
    TTC_HIP(c, hipGetLastError());
    return st;
}

ttc_status ttc_linear_backward(ttc_ctx* c, const ttc_linear_desc* d, const void* d_dy, const void* d_x, const void* d_w, const float* d_bias,
                               const float* d_preact, void* d_dx, void* d_dw, float* d_dbias, void* d_ws, size_t ws_bytes, void* stream) {
    if (!c) return TTC_ERR_ARG;
    if (const char* e = linear_check(d)) return c->fail(TTC_ERR_ARG, std::string("linear_backward: ") + e);
    if ((d->rows > 1 && d->dy_pitch < d->cout) || d->dy_pitch > (1L << 30)) return c->fail(TTC_ERR_ARG, "linear_backward: dy_pitch must be at least cout");
    if (!d_dx && !d_dw && !d_dbias) return TTC_OK;
    const bool act = d->activation != TTC_ACT_NONE, again = act && !d_preact;
    BwdWs w{};
    if (d->rows > 0) {
        w = linear_ws(d, !again);
        if (!d_dy || !d_x || !d_w || !d_ws) return c->fail(TTC_ERR_ARG, "linear_backward: null pointer");
        if ((uintptr_t)d_ws % 16) return c->fail(TTC_ERR_ARG, "linear_backward: the workspace must be 16-byte aligned");
        if (ws_bytes < w.total) return c->fail(TTC_ERR_ARG, "linear_backward: workspace smaller than ttc_linear_workspace asks for");
    }
    DeviceGuard dev(c->device);
    if (!dev.ok) return c->fail(TTC_ERR_HIP, "linear_backward: hipSetDevice failed");
    hipStream_t s = (hipStream_t)stream;
    KTimer t(c, "linear_backward", s);
    const ttc_status st = with_dtype(d->dtype, [&](auto tag) {
        using T = decltype(tag);
        if (d->rows == 0) {
            const long n = (long)d->cin * d->cout;
            // at most 2^16 workgroups: a launch is limited to 2^32 threads, and dw may have as many elements
            if (d_dw) hipLaunchKernelGGL((k_fill0<T>), dim3((unsigned)std::min<long>((n + NT - 1) / NT, 1 << 16)), dim3(NT), 0, s, (T*)d_dw, n);
            if (d_dbias) hipLaunchKernelGGL((k_fill0<float>), dim3((d->cout + NT - 1) / NT), dim3(NT), 0, s, d_dbias, (long)d->cout);
            return TTC_OK;
        }
        char* ws = (char*)d_ws;
        const bool pair = dz_is_pair<T>(d->activation);
        const float alpha = d->scale / (pair ? DZ_DOWN<T> : 1.0f);
        GemmArgs o{};                                        // dw [cin, cout], scaled where the splits are joined
        o.M = d->cin; o.N = d->cout; o.C = d_dw; o.ldc = d->cout; o.alpha = alpha;
        if (narrow_bwd(d)) {
            NarrowBwd a{};
            a.x = d_x; a.dy = d_dy; a.w = d_w; a.bias = d_bias; a.z = act ? d_preact : nullptr; a.dx = d_dx;
            a.part = d_dw || d_dbias ? (float*)ws : nullptr;
            a.M = d->rows; a.ldx = d->x_pitch; a.ldy = d->dy_pitch; a.ldw = d->w_pitch;
            a.K = d->cin; a.N = d->cout; a.act = d->activation; a.scale = alpha; a.want_dw = d_dw != nullptr;
            TTC_HIP(c, narrow_bwd_launch<T>(a, w.blocks, s));
            if (a.part) join_launch<T>(o, a.part, (long)d->cin * d->cout + d->cout, w.blocks, d_dbias ? d->cout : 0, d_dbias, s);
            return TTC_OK;
        }
        const float* z = d_preact;
        if (again) {                                         // x w + bias in 32 bits
            GemmArgs a = fwd_args(d, d_x, d_w);
            GemmArgs zf = a;
            zf.fwd = 1; zf.act = TTC_ACT_NONE; zf.alpha = 1.0f; zf.bias = d_bias; zf.C = nullptr; zf.preact = (float*)ws;
            gemm_launch<T, true, false>(zf, gemm_splits(d->rows, d->cout, d->cin, dtype_bytes(d->dtype)), (float*)(ws + w.part), s);
            z = (const float*)ws;
        }
        const T* dz = act ? (const T*)(ws + w.dz) : (const T*)d_dy;     // without an activation dz is dy itself; the scale is in the epilogues either way
        void* dz_lo = pair ? ws + w.lo : nullptr;
        const long dz_pitch = act ? d->cout : d->dy_pitch;
        if (act || d_dbias) {
            DzArgs q{};
            q.dy = d_dy; q.z = z; q.dz = act && (d_dx || d_dw) ? ws + w.dz : nullptr; q.lo = dz_lo; q.part = d_dbias ? (float*)(ws + w.sums) : nullptr;
            q.rows = d->rows; q.dpitch = d->dy_pitch; q.N = d->cout; q.act = d->activation;
            const int V = col_vec(d->cout, sizeof(T));
            int blocks, tiles;
            dz_geometry(q, V, &blocks, &tiles);
            dz_launch<T>(q, V, blocks, tiles, s);
            if (d_dbias) {
                GemmArgs b{};
                b.M = 0; b.N = d->cout; b.alpha = d->scale;
                join_launch<float>(b, q.part, d->cout, blocks, d->cout, d_dbias, s);
            }
        }
        if (d_dx) {
            GemmArgs a{};
            a.A = dz; a.Alo = dz_lo; a.lda = dz_pitch; a.B = d_w; a.ldb = d->w_pitch;
            a.M = d->rows; a.N = d->cin; a.K = d->cout;
            a.C = d_dx; a.ldc = d->cin; a.alpha = alpha;
            gemm_launch<T, true, true>(a, w.dx_splits, (float*)(ws + w.part), s);
        }
        if (d_dw) {
            GemmArgs a = o;
            a.A = d_x; a.lda = d->x_pitch; a.B = dz; a.Blo = dz_lo; a.ldb = dz_pitch; a.K = d->rows;
            gemm_launch<T, false, false>(a, w.dw_splits, (float*)(ws + w.part), s);
        }
        return TTC_OK;
    });
    TTC_HIP(c, hipGetLastError());
    return st;
}

}  // extern "C"
