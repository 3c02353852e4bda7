// The gated delta rule, forward and backward in chunks of 64 time steps, on matrix instructions.
//
// One head, with keys and queries of Dk values, values of Dv, a decay e^{g_t} (g_t <= 0) and a rate beta_t:
//
//     S_t = e^{g_t} S_{t-1} + beta_t k_t (v_t - e^{g_t} S_{t-1}^T k_t)^T,     o_t = scale * S_t^T q_t
//
// The state S [Dk, Dv] is an associative memory: it decays, what it holds under key k_t is replaced by v_t at rate
// beta_t, and it is read with q_t.  Rows of a chunk written as matrices, c_i the sum of g over the chunk up to row i,
// a_i = e^{c_i}, d_i = e^{c_last - c_i}, G_ij = e^{c_i - c_j} (i >= j; never above one), S the state before the chunk:
//
//     A_ij = beta_i (k_i . k_j) G_ij  (i > j)          Tm = (I + A)^-1        (unit lower triangular)
//     X = beta (V - a K S)                             R = Tm X               (what each row adds to the memory)
//     P_ij = scale (q_i . k_j) G_ij  (i >= j)          O = scale a (Q S) + P R
//     S' = a_last S + K^T (d R)
//
// Only X, R and S' hang on the state of the chunk before.  Backwards, with dS' the gradient of the state after:
//
//     dR = P^T dO + d (K dS')          dX = Tm^T dR        dS = a_last dS' + Q^T (scale a dO) - K^T (beta a dX)
//     dV = beta dX      Y1 = dX S^T    Y2 = dO S^T    Y3 = R dS'^T
//     dA = -dX R^T (i > j)     M = beta_i dA G         dP = dO R^T (i >= j)     N = scale dP G
//     dQ = scale a Y2 + N K            dK = -beta a Y1 + d Y3 + (M + M^T) K + N^T Q
//     dbeta_i = v_i . dX_i - a_i k_i . Y1_i + sum_j dA_ij (k_i . k_j) G_ij
//     dc_i = sum_j (dA A + dP P)_ij - sum_j (dA A + dP P)_ji - beta_i a_i k_i . Y1_i + scale a_i q_i . Y2_i - e_i,
//     e_i = d_i k_i . Y3_i;   dc_last += sum e + a_last <S, dS'>;   dg = sums of dc from the row to the end of the chunk
//
// Kernels.  Everything that does not hang on the state runs over all chunks and heads at once; the two passes that do
// (delta_state_kernel forwards, delta_state_grad_kernel backwards) walk the chunks of a head, one workgroup per head
// and 32 columns of the state, which they hold in accumulators.
//   forward    delta_inverse_kernel -> Tm;   delta_state_kernel -> S of every chunk, R, last state;   delta_output_kernel -> O
//   backward   delta_inner_grad_kernel -> P^T dO;   delta_state_grad_kernel -> dS' of every chunk, dX;
//              delta_input_grad_kernel -> the gradients;   delta_shared_grad_kernel where heads share keys
// The state passes are bound by the latency of a chunk's chain of products (three forward, three backward, each
// through LDS), the others by memory.
//
// Numbers.  States, R, Tm, dX and every sum are fp32.  In bf16 storage the products run on the bf16 matrix
// instructions; an input is exact there, and everything derived (Tm, X, R, P, the state, ...) is given as two bf16
// parts, value and remainder, which together keep 16 bits: rounding it once would cost a relative 2^-9 in each
// product and show up in the fp32 gradients and states.  The product of the two remainders is left out (2^-18).
// In fp32 storage they run on the fp32 matrix instructions.  The sums c are held in 64 bits: G needs differences.
//
// Time steps at or behind a sequence's length have no row: they leave the state alone and their outputs are zero.
#ifndef SNNLIF_SEQ_DELTA_H
#define SNNLIF_SEQ_DELTA_H

#include "seq_common.h"

namespace snnseq {

constexpr int kChunk = 64;
constexpr int kStateCols = 32;  // columns of the state a workgroup of the state passes holds

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- operands of the matrix instructions --------------------------------------------------------
//
// A fragment is 16 rows (or columns) times 32 steps of the contraction; lane l holds index l % 16, steps
// (l / 16) * 8 .. + 7.  A 16 x 16 product leaves rows (l / 16) * 4 + i, column l % 16 in lane l's element i.

template <int N> struct FragH { bf16x8 p[N]; };   // the sum of N bf16 parts
struct FragF { float v[8]; };

template <int NA, int NB>
__device__ __forceinline__ f32x4 mma(const FragH<NA>& a, const FragH<NB>& b, f32x4 c) {
    constexpr int most = NA > NB ? NA : NB;
#pragma unroll
    for (int i = NA - 1; i >= 0; --i)
#pragma unroll
        for (int j = NB - 1; j >= 0; --j)
            if (i + j < most) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ f32x4 mma(const FragF& a, const FragF& b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ uint16_t bits_of(float v) {
    const __bf16 r = static_cast<__bf16>(v);
    return __builtin_bit_cast(uint16_t, r);
}
__device__ __forceinline__ float value_of(uint16_t bits) {
    return __builtin_bit_cast(float, static_cast<uint32_t>(bits) << 16);
}

// A matrix in LDS as N bf16 parts, row-major; 16 bytes of padding per row spread the rows over the banks.
template <int N, int ROWS, int COLS>
struct TileH {
    static constexpr int ld = COLS + 8;
    uint16_t v[N][ROWS * ld];

    // n consecutive columns, c a multiple of 4
    template <int n>
    __device__ __forceinline__ void put(int r, int c, const float (&x)[n]) {
        float rest[n];
#pragma unroll
        for (int j = 0; j < n; ++j) rest[j] = x[j];
#pragma unroll
        for (int part = 0; part < N; ++part) {
            uint32_t words[n / 2];
#pragma unroll
            for (int j = 0; j < n; j += 2) {
                const uint16_t lo = bits_of(rest[j]), hi = bits_of(rest[j + 1]);
                words[j / 2] = lo | static_cast<uint32_t>(hi) << 16;
                rest[j] -= value_of(lo);
                rest[j + 1] -= value_of(hi);
            }
            uint16_t* p = &v[part][r * ld + c];
            if constexpr (n == 8) *reinterpret_cast<u32x4*>(p) = u32x4{words[0], words[1], words[2], words[3]};
            else *reinterpret_cast<u32x2*>(p) = u32x2{words[0], words[1]};
        }
    }
    __device__ __forceinline__ void put(int r, int c, float x) {
#pragma unroll
        for (int part = 0; part < N; ++part) {
            const uint16_t b = bits_of(x);
            v[part][r * ld + c] = b;
            x -= value_of(b);
        }
    }
    __device__ __forceinline__ void put_raw(int r, int c, u32x4 raw) {
        static_assert(N == 1, "raw storage is one part");
        *reinterpret_cast<u32x4*>(&v[0][r * ld + c]) = raw;
    }
    __device__ __forceinline__ float get(int r, int c) const {
        float x = 0.f;
#pragma unroll
        for (int part = 0; part < N; ++part) x += value_of(v[part][r * ld + c]);
        return x;
    }
    // operand indexed by rows r0 .., contracted over columns k0 ..
    __device__ __forceinline__ FragH<N> rows(int r0, int k0) const {
        const int lane = threadIdx.x & 63;
        FragH<N> f;
#pragma unroll
        for (int part = 0; part < N; ++part)
            f.p[part] = *reinterpret_cast<const bf16x8*>(&v[part][(r0 + (lane & 15)) * ld + k0 + (lane >> 4) * 8]);
        return f;
    }
    // operand indexed by columns c0 .., contracted over rows k0 ..: the transposing LDS read hands 16 lanes that
    // point at 4 rows of 16 columns the 4 values of a column each
    __device__ __forceinline__ FragH<N> cols(int c0, int k0) const {
        const int lane = threadIdx.x & 63;
        FragH<N> f;
#pragma unroll
        for (int part = 0; part < N; ++part) {
            s16x4 half[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint16_t* p = &v[part][(k0 + (lane >> 4) * 8 + h * 4 + ((lane >> 2) & 3)) * ld + c0 + (lane & 3) * 4];
                half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4*)(const_cast<uint16_t*>(p)));
            }
            f.p[part] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return f;
    }
};

// The same in fp32.
template <int ROWS, int COLS>
struct TileF {
    static constexpr int ld = COLS + 4;
    float v[ROWS * ld];

    template <int n>
    __device__ __forceinline__ void put(int r, int c, const float (&x)[n]) {
#pragma unroll
        for (int j = 0; j < n; j += 4)
            *reinterpret_cast<f32x4*>(&v[r * ld + c + j]) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
    }
    __device__ __forceinline__ void put(int r, int c, float x) { v[r * ld + c] = x; }
    __device__ __forceinline__ float get(int r, int c) const { return v[r * ld + c]; }
    __device__ __forceinline__ FragF rows(int r0, int k0) const {
        const int lane = threadIdx.x & 63;
        const float* p = &v[(r0 + (lane & 15)) * ld + k0 + (lane >> 4) * 8];
        FragF f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4 q = *reinterpret_cast<const f32x4*>(p + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) f.v[4 * h + j] = q[j];
        }
        return f;
    }
    __device__ __forceinline__ FragF cols(int c0, int k0) const {
        const int lane = threadIdx.x & 63;
        FragF f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f.v[j] = v[(k0 + (lane >> 4) * 8 + j) * ld + c0 + (lane & 15)];
        return f;
    }
};

// What a storage type computes with: tiles of inputs and of derived values.
template <typename E> struct Mode;
template <> struct Mode<bf16_t> {
    template <int R, int C> using Input = TileH<1, R, C>;
    template <int R, int C> using Derived = TileH<2, R, C>;
};
template <> struct Mode<float> {
    template <int R, int C> using Input = TileF<R, C>;
    template <int R, int C> using Derived = TileF<R, C>;
};

// ---- arguments ----------------------------------------------------------------------------------

// A [T, B, heads, D] tensor whose rows of D values are dense.
struct DeltaTensor {
    const void* p;
    int64_t t, b, h;   // strides in elements
    int wide;          // every row begins on 16 bytes and D is a multiple of 8
};

struct DeltaArgs {
    int T, B, Hk, Hv, Dk, Dv;
    int chunks;                 // ceil(T / 64)
    int cols;                   // Dv rounded up to 32: row length of the workspace's matrices
    float scale;
    const int32_t* lengths;     // [B] or nullptr
    DeltaTensor q, k, v, grad_o;
    const float *g, *beta;      // [T, B, Hv]
    const float *state, *grad_state;   // [B, Hv, Dk, Dv] or nullptr: the initial state, the gradient of the last one
    void* o;                    // [T, B, Hv, Dv]
    float* state_out;           // [B, Hv, Dk, Dv] or nullptr
    // per (batch entry, value head, chunk)
    float* inverse;             // [64, 64] Tm
    float* added;               // [64, cols] R
    float* states;              // [DKP, cols] state before the chunk
    // backward
    float* inner;               // [64, cols] P^T dO, then dX
    float* state_grads;         // [DKP, cols] gradient of the state after the chunk
    void *grad_q, *grad_k;      // [T, B, Hk, Dk] of the storage type, or fp32 [T, B, Hv, Dk] where heads share keys
    void* grad_v;               // [T, B, Hv, Dv]
    float *grad_g, *grad_beta;  // [T, B, Hv]
    float* grad_initial;        // [B, Hv, Dk, Dv] or nullptr
};

struct DeltaWhere {  // the chunk (or head) a workgroup works on
    int b, hv, hk, chunk, head;
    int t0, rows;    // first step and how many of its 64 rows exist
};

__device__ __forceinline__ int delta_length(const DeltaArgs& a, int b) {
    if (a.lengths == nullptr) return a.T;
    const int n = a.lengths[b];
    return n < 0 ? 0 : n > a.T ? a.T : n;
}

__device__ __forceinline__ DeltaWhere delta_where(const DeltaArgs& a, int head, int chunk) {
    DeltaWhere w;
    w.head = head;
    w.b = head / a.Hv;
    w.hv = head - w.b * a.Hv;
    w.hk = w.hv / (a.Hv / a.Hk);
    w.chunk = chunk;
    w.t0 = chunk * kChunk;
    const int left = delta_length(a, w.b) - w.t0;
    w.rows = left < 0 ? 0 : left > kChunk ? kChunk : left;
    return w;
}

// ---- staging ------------------------------------------------------------------------------------

// Eight consecutive values of a row, zero behind `valid`.
template <typename E>
__device__ __forceinline__ void load8(const E* row, int c, int valid, bool wide, float (&x)[8]) {
    constexpr int per = 16 / static_cast<int>(sizeof(E));
    if (wide) {
        if (c < valid) {
#pragma unroll
            for (int h = 0; h < 8 / per; ++h) {
                const Vec<E, 16> v = load_vec<E, 16>(row + c + h * per);
#pragma unroll
                for (int j = 0; j < per; ++j) x[h * per + j] = widen(v.e[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = c + j < valid ? widen(row[c + j]) : 0.f;
    }
}

// ROWS x COLS of a tensor with `stride` values from row to row, of which `rows` x `valid` exist.
template <int ROWS, int COLS, int THREADS, typename E, typename Tile>
__device__ __forceinline__ void stage(Tile& tile, const E* base, int64_t stride, int rows, int valid, bool wide) {
#pragma unroll
    for (int i = 0; i < ROWS * COLS / 8; i += THREADS) {
        const int seg = i + threadIdx.x;
        if (ROWS * COLS / 8 % THREADS != 0 && seg >= ROWS * COLS / 8) break;
        const int r = seg / (COLS / 8), c = seg % (COLS / 8) * 8;
        float x[8];
        load8<E>(base + (r < rows ? r : 0) * stride, c, r < rows ? valid : 0, wide, x);
        tile.put(r, c, x);
    }
}

template <typename E>
__device__ __forceinline__ const E* row_of(const DeltaTensor& x, const DeltaWhere& w, int head) {
    return static_cast<const E*>(x.p) + w.t0 * x.t + w.b * x.b + head * x.h;
}

// Decay of a chunk: sums c (64 bits), a = e^c, d = e^{c_last - c}, and beta; by the first wavefront.  A row that does
// not exist has g = 0 and beta = 0.
struct Decay {
    double c[kChunk];
    float a[kChunk], d[kChunk], beta[kChunk];
    float a_last;
};

__device__ __forceinline__ void decay_of(const DeltaArgs& args, const DeltaWhere& w, Decay& out) {
    const int lane = threadIdx.x;
    if (lane >= 64) return;
    float g = 0.f, beta = 0.f;
    if (lane < w.rows) {
        const int64_t at = (static_cast<int64_t>(w.t0 + lane) * args.B + w.b) * args.Hv + w.hv;
        g = args.g[at];
        beta = args.beta[at];
        g = g < -1e4f ? -1e4f : g;   // e^-10000 is zero; sums and differences stay finite (a NaN stays)
    }
    double c = g;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double other = __shfl_up(c, s);
        if (lane >= s) c += other;
    }
    const double last = __shfl(c, 63);
    out.c[lane] = c;
    out.a[lane] = expf(static_cast<float>(c));
    out.d[lane] = expf(static_cast<float>(last - c));
    out.beta[lane] = beta;
    if (lane == 63) out.a_last = expf(static_cast<float>(c));
}

__device__ __forceinline__ float gap(const Decay& y, int i, int j) {  // G_ij
    return expf(static_cast<float>(y.c[i] - y.c[j]));
}

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

// ---- Tm = (I + A)^-1 ----------------------------------------------------------------------------

struct Square { float v[kChunk][kChunk + 4]; };

// 16 x 16 products of blocks of fp32 squares on the fp32 matrix instructions (16 x 16 x 4).
__device__ __forceinline__ f32x4 block_product(const Square& x, int xr, int xc, const Square& y, int yr, int yc, f32x4 acc) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < 16; k += 4)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[xr + (lane & 15)][xc + k + (lane >> 4)],
                                                   y.v[yr + k + (lane >> 4)][yc + (lane & 15)], acc, 0, 0, 0);
    return acc;
}

// Four wavefronts.  Diagonal blocks of 16 by substitution, one column per lane; then the blocks below, one distance
// from the diagonal at a time: T_ij = -T_ii sum_{j <= k < i} A_ik T_kj.
__device__ __forceinline__ void invert_unit_lower(const Square& a, Square& t, Square& scratch) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < 16) {
        float x[16];
        const int o = wave * 16;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == lane ? 1.f : 0.f;
#pragma unroll
            for (int j = 0; j < i; ++j) s -= a.v[o + i][o + j] * x[j];
            x[i] = s;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) t.v[o + i][o + lane] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int far = 1; far < 4; ++far) {
        const int j = wave, i = wave + far;
        if (i < 4) {
            f32x4 acc = zero4();
            for (int k = j; k < i; ++k) acc = block_product(a, i * 16, k * 16, t, k * 16, j * 16, acc);
#pragma unroll
            for (int e = 0; e < 4; ++e) scratch.v[i * 16 + (lane >> 4) * 4 + e][j * 16 + (lane & 15)] = -acc[e];
        }
        __syncthreads();
        if (i < 4) {
            const f32x4 acc = block_product(t, i * 16, i * 16, scratch, i * 16, j * 16, zero4());
#pragma unroll
            for (int e = 0; e < 4; ++e) t.v[i * 16 + (lane >> 4) * 4 + e][j * 16 + (lane & 15)] = acc[e];
        }
        __syncthreads();
    }
}

template <typename E, int DKP>
__global__ void __launch_bounds__(256) delta_inverse_kernel(DeltaArgs args) {
    using M = Mode<E>;
    __shared__ typename M::template Input<kChunk, DKP> k;
    __shared__ Square a, t, scratch;
    __shared__ Decay y;
    const DeltaWhere w = delta_where(args, blockIdx.y, blockIdx.x);
    if (w.rows == 0) return;
    stage<kChunk, DKP, 256>(k, row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk, args.k.wide != 0);
    decay_of(args, w, y);
    for (int i = threadIdx.x; i < kChunk * (kChunk + 4); i += 256) (&t.v[0][0])[i] = 0.f;
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int block = 0; block <= wave; ++block) {
        f32x4 acc = zero4();
#pragma unroll
        for (int s = 0; s < DKP; s += 32) acc = mma(k.rows(wave * 16, s), k.rows(block * 16, s), acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = wave * 16 + (lane >> 4) * 4 + e, j = block * 16 + (lane & 15);
            a.v[i][j] = i > j ? y.beta[i] * acc[e] * gap(y, i, j) : 0.f;
        }
    }
    __syncthreads();
    invert_unit_lower(a, t, scratch);
    float* out = args.inverse + (static_cast<int64_t>(w.head) * args.chunks + w.chunk) * (kChunk * kChunk);
#pragma unroll
    for (int i = 0; i < kChunk * kChunk / 4; i += 256) {
        const int r = (i + threadIdx.x) / 16, c = (i + threadIdx.x) % 16 * 4;
        *reinterpret_cast<f32x4*>(out + r * kChunk + c) = *reinterpret_cast<const f32x4*>(&t.v[r][c]);
    }
}

// ---- the state, forwards ------------------------------------------------------------------------

constexpr int kStateThreads = 512;

template <typename E, int DKP>
__global__ void __launch_bounds__(kStateThreads) delta_state_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kStateCols, TILES = DKP / 16 * (NV / 16) / 8;  // state tiles per wavefront
    __shared__ typename M::template Input<kChunk, DKP> k;
    __shared__ typename M::template Derived<kChunk, kChunk> inverse;
    __shared__ typename M::template Derived<NV, DKP> state;     // transposed
    __shared__ typename M::template Derived<NV, kChunk> x, r;   // transposed
    __shared__ Decay y;
    const int head = blockIdx.y, v0 = blockIdx.x * NV;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lr = (lane >> 4) * 4, lc = lane & 15;
    const DeltaWhere first = delta_where(args, head, 0);
    const int chunks = (delta_length(args, first.b) + kChunk - 1) / kChunk;

    f32x4 s[TILES];
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        const int tile = wave + 8 * i, row = tile / 2 * 16 + lr, col = v0 + tile % 2 * 16 + lc;
        float v4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v4[e] = 0.f;
            if (args.state != nullptr && row + e < args.Dk && col < args.Dv)
                v4[e] = args.state[(static_cast<int64_t>(head) * args.Dk + row + e) * args.Dv + col];
            s[i][e] = v4[e];
        }
        state.put(tile % 2 * 16 + lc, row, v4);
    }
    const int rt = wave / 2 * 16, ct = wave % 2 * 16;   // this wavefront's tile of the chunk's rows
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const DeltaWhere w = delta_where(args, head, chunk);
        const int64_t at = static_cast<int64_t>(head) * args.chunks + chunk;
        __syncthreads();
        stage<kChunk, DKP, kStateThreads>(k, row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk, args.k.wide != 0);
        stage<kChunk, kChunk, kStateThreads>(inverse, const_cast<const float*>(args.inverse) + at * (kChunk * kChunk),
                                             kChunk, kChunk, kChunk, true);
        decay_of(args, w, y);
        const int col = v0 + ct + lc;
        float v[4];
        const E* pv = row_of<E>(args.v, w, w.hv);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = rt + lr + e < w.rows && col < args.Dv ? widen(pv[(rt + lr + e) * args.v.t + col]) : 0.f;
        float* ps = args.states + at * DKP * args.cols + v0;
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int tile = wave + 8 * i;
#pragma unroll
            for (int e = 0; e < 4; ++e) ps[(tile / 2 * 16 + lr + e) * static_cast<int64_t>(args.cols) + tile % 2 * 16 + lc] = s[i][e];
        }
        __syncthreads();
        f32x4 acc = zero4();
#pragma unroll
        for (int c = 0; c < DKP; c += 32) acc = mma(k.rows(rt, c), state.rows(ct, c), acc);
        float out[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = y.beta[rt + lr + e] * (v[e] - y.a[rt + lr + e] * acc[e]);
        x.put(ct + lc, rt + lr, out);
        __syncthreads();
        acc = zero4();
        for (int c = 0; c < rt + 16; c += 32) acc = mma(inverse.rows(rt, c), x.rows(ct, c), acc);
        float* pr = args.added + at * kChunk * args.cols + v0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            pr[(rt + lr + e) * static_cast<int64_t>(args.cols) + ct + lc] = acc[e];
            out[e] = y.d[rt + lr + e] * acc[e];
        }
        r.put(ct + lc, rt + lr, out);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int tile = wave + 8 * i;
            f32x4 next;
#pragma unroll
            for (int e = 0; e < 4; ++e) next[e] = y.a_last * s[i][e];
#pragma unroll
            for (int c = 0; c < kChunk; c += 32) next = mma(k.cols(tile / 2 * 16, c), r.rows(tile % 2 * 16, c), next);
            s[i] = next;
            float v4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v4[e] = next[e];
            state.put(tile % 2 * 16 + lc, tile / 2 * 16 + lr, v4);
        }
    }
    if (args.state_out != nullptr) {
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int tile = wave + 8 * i, row = tile / 2 * 16 + lr, col = v0 + tile % 2 * 16 + lc;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row + e < args.Dk && col < args.Dv)
                    args.state_out[(static_cast<int64_t>(head) * args.Dk + row + e) * args.Dv + col] = s[i][e];
        }
    }
}

// ---- the output ---------------------------------------------------------------------------------

// P of a chunk from staged Q and K, by four wavefronts; blocks above the diagonal are zero.
template <int DKP, typename TQ, typename TK, typename TP>
__device__ __forceinline__ void scores_of(const TQ& q, const TK& k, const Decay& y, float scale, TP& p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int block = 0; block < 4; ++block) {
        f32x4 acc = zero4();
        if (block <= wave) {
#pragma unroll
            for (int s = 0; s < DKP; s += 32) acc = mma(q.rows(wave * 16, s), k.rows(block * 16, s), acc);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = wave * 16 + (lane >> 4) * 4 + e, j = block * 16 + (lane & 15);
            p.put(i, j, i >= j ? scale * acc[e] * gap(y, i, j) : 0.f);
        }
    }
}

template <typename E, int DKP>
__global__ void __launch_bounds__(256) delta_output_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kStateCols;
    __shared__ typename M::template Input<kChunk, DKP> q;
    __shared__ typename M::template Derived<kChunk, kChunk> p;
    __shared__ Decay y;
    struct Columns {
        typename M::template Derived<DKP, NV> state;
        typename M::template Derived<kChunk, NV> r;
    };
    union Later {   // K is done with before the columns come
        typename M::template Input<kChunk, DKP> k;
        Columns c;
        __device__ Later() {}
    };
    __shared__ Later u;
    const DeltaWhere w = delta_where(args, blockIdx.y, blockIdx.x);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lr = wave * 16 + (lane >> 4) * 4, lc = lane & 15;
    E* out = static_cast<E*>(args.o) + (static_cast<int64_t>(w.t0) * args.B * args.Hv + w.head) * args.Dv;
    const int64_t out_stride = static_cast<int64_t>(args.B) * args.Hv * args.Dv;
    const int present = args.T - w.t0 < kChunk ? args.T - w.t0 : kChunk;
    if (w.rows == 0) {
        for (int i = threadIdx.x; i < present * args.Dv; i += 256) out[i / args.Dv * out_stride + i % args.Dv] = narrow<E>(0.f);
        return;
    }
    stage<kChunk, DKP, 256>(q, row_of<E>(args.q, w, w.hk), args.q.t, w.rows, args.Dk, args.q.wide != 0);
    stage<kChunk, DKP, 256>(u.k, row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk, args.k.wide != 0);
    decay_of(args, w, y);
    __syncthreads();
    scores_of<DKP>(q, u.k, y, args.scale, p);
    const int64_t at = static_cast<int64_t>(w.head) * args.chunks + w.chunk;
    for (int v0 = 0; v0 < args.cols; v0 += NV) {
        __syncthreads();
        stage<DKP, NV, 256>(u.c.state, const_cast<const float*>(args.states) + at * DKP * args.cols + v0, args.cols, DKP, NV, true);
        stage<kChunk, NV, 256>(u.c.r, const_cast<const float*>(args.added) + at * kChunk * args.cols + v0, args.cols, kChunk, NV, true);
        __syncthreads();
        f32x4 acc[2] = {zero4(), zero4()};
#pragma unroll
        for (int s = 0; s < DKP; s += 32) {
            const auto f = q.rows(wave * 16, s);
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[c] = mma(f, u.c.state.cols(c * 16, s), acc[c]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][e] *= args.scale * y.a[lr + e];
        for (int s = 0; s < wave * 16 + 16; s += 32) {
            const auto f = p.rows(wave * 16, s);
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[c] = mma(f, u.c.r.cols(c * 16, s), acc[c]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = v0 + c * 16 + lc;
                if (lr + e < present && col < args.Dv)
                    out[(lr + e) * out_stride + col] = narrow<E>(lr + e < w.rows ? acc[c][e] : 0.f);
            }
    }
}

// ---- backward: P^T dO ---------------------------------------------------------------------------

template <typename E, int DKP>
__global__ void __launch_bounds__(256) delta_inner_grad_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kStateCols;
    __shared__ typename M::template Input<kChunk, DKP> q, k;
    __shared__ typename M::template Derived<kChunk, kChunk> p;
    __shared__ typename M::template Input<kChunk, NV> go;
    __shared__ Decay y;
    const DeltaWhere w = delta_where(args, blockIdx.y, blockIdx.x);
    if (w.rows == 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lr = wave * 16 + (lane >> 4) * 4, lc = lane & 15;
    stage<kChunk, DKP, 256>(q, row_of<E>(args.q, w, w.hk), args.q.t, w.rows, args.Dk, args.q.wide != 0);
    stage<kChunk, DKP, 256>(k, row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk, args.k.wide != 0);
    decay_of(args, w, y);
    __syncthreads();
    scores_of<DKP>(q, k, y, args.scale, p);
    const int64_t at = static_cast<int64_t>(w.head) * args.chunks + w.chunk;
    const E* pg = row_of<E>(args.grad_o, w, w.hv);
    for (int v0 = 0; v0 < args.cols; v0 += NV) {
        __syncthreads();
        stage<kChunk, NV, 256>(go, pg + v0, args.grad_o.t, w.rows, args.Dv - v0, args.grad_o.wide != 0);
        __syncthreads();
        f32x4 acc[2] = {zero4(), zero4()};
        for (int s = wave * 16 / 32 * 32; s < kChunk; s += 32) {
            const auto f = p.cols(wave * 16, s);
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[c] = mma(f, go.cols(c * 16, s), acc[c]);
        }
        float* out = args.inner + at * kChunk * args.cols + v0;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) out[static_cast<int64_t>(lr + e) * args.cols + c * 16 + lc] = acc[c][e];
    }
}

// ---- the state, backwards -----------------------------------------------------------------------

template <typename E, int DKP>
__global__ void __launch_bounds__(kStateThreads) delta_state_grad_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kStateCols, TILES = DKP / 16 * (NV / 16) / 8;
    __shared__ typename M::template Input<kChunk, DKP> q, k;
    __shared__ typename M::template Derived<kChunk, kChunk> inverse;
    __shared__ typename M::template Derived<NV, DKP> state;       // gradient of the state, transposed
    __shared__ typename M::template Derived<NV, kChunk> r, x, go; // dR, beta a dX, scale a dO, transposed
    __shared__ Decay y;
    const int head = blockIdx.y, v0 = blockIdx.x * NV;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lr = (lane >> 4) * 4, lc = lane & 15;
    const DeltaWhere first = delta_where(args, head, 0);
    const int chunks = (delta_length(args, first.b) + kChunk - 1) / kChunk;

    f32x4 s[TILES];
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        const int tile = wave + 8 * i, row = tile / 2 * 16 + lr, col = v0 + tile % 2 * 16 + lc;
        float v4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v4[e] = 0.f;
            if (args.grad_state != nullptr && row + e < args.Dk && col < args.Dv)
                v4[e] = args.grad_state[(static_cast<int64_t>(head) * args.Dk + row + e) * args.Dv + col];
            s[i][e] = v4[e];
        }
        state.put(tile % 2 * 16 + lc, row, v4);
    }
    const int rt = wave / 2 * 16, ct = wave % 2 * 16;
    for (int chunk = chunks - 1; chunk >= 0; --chunk) {
        const DeltaWhere w = delta_where(args, head, chunk);
        const int64_t at = static_cast<int64_t>(head) * args.chunks + chunk;
        __syncthreads();
        stage<kChunk, DKP, kStateThreads>(q, row_of<E>(args.q, w, w.hk), args.q.t, w.rows, args.Dk, args.q.wide != 0);
        stage<kChunk, DKP, kStateThreads>(k, row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk, args.k.wide != 0);
        stage<kChunk, kChunk, kStateThreads>(inverse, const_cast<const float*>(args.inverse) + at * (kChunk * kChunk),
                                             kChunk, kChunk, kChunk, true);
        decay_of(args, w, y);
        const int col = v0 + ct + lc;
        float g[4], out[4];
        const E* pg = row_of<E>(args.grad_o, w, w.hv);
        float* px = args.inner + at * kChunk * args.cols + v0;
        f32x4 acc;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            g[e] = rt + lr + e < w.rows && col < args.Dv ? widen(pg[(rt + lr + e) * args.grad_o.t + col]) : 0.f;
            acc[e] = px[(rt + lr + e) * static_cast<int64_t>(args.cols) + ct + lc];
        }
        float* ps = args.state_grads + at * DKP * args.cols + v0;
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int tile = wave + 8 * i;
#pragma unroll
            for (int e = 0; e < 4; ++e) ps[(tile / 2 * 16 + lr + e) * static_cast<int64_t>(args.cols) + tile % 2 * 16 + lc] = s[i][e];
        }
        __syncthreads();
        f32x4 from_state = zero4();
#pragma unroll
        for (int c = 0; c < DKP; c += 32) from_state = mma(k.rows(rt, c), state.rows(ct, c), from_state);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = rt + lr + e;
            out[e] = acc[e] + y.d[i] * from_state[e];
            g[e] *= args.scale * y.a[i];
        }
        r.put(ct + lc, rt + lr, out);
        go.put(ct + lc, rt + lr, g);
        __syncthreads();
        acc = zero4();
        for (int c = rt / 32 * 32; c < kChunk; c += 32) acc = mma(inverse.cols(rt, c), r.rows(ct, c), acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = rt + lr + e;
            px[i * static_cast<int64_t>(args.cols) + ct + lc] = acc[e];
            out[e] = -y.beta[i] * y.a[i] * acc[e];
        }
        x.put(ct + lc, rt + lr, out);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int tile = wave + 8 * i;
            f32x4 next;
#pragma unroll
            for (int e = 0; e < 4; ++e) next[e] = y.a_last * s[i][e];
#pragma unroll
            for (int c = 0; c < kChunk; c += 32) {
                next = mma(q.cols(tile / 2 * 16, c), go.rows(tile % 2 * 16, c), next);
                next = mma(k.cols(tile / 2 * 16, c), x.rows(tile % 2 * 16, c), next);
            }
            s[i] = next;
            float v4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v4[e] = next[e];
            state.put(tile % 2 * 16 + lc, tile / 2 * 16 + lr, v4);
        }
    }
    if (args.grad_initial != nullptr) {
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int tile = wave + 8 * i, row = tile / 2 * 16 + lr, col = v0 + tile % 2 * 16 + lc;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row + e < args.Dk && col < args.Dv)
                    args.grad_initial[(static_cast<int64_t>(head) * args.Dk + row + e) * args.Dv + col] = s[i][e];
        }
    }
}

// ---- backward: the gradients of the inputs ------------------------------------------------------

__device__ __forceinline__ float row_sum16(float v) {  // over the 16 lanes that share rows
    v += __shfl_xor(v, 1);
    v += __shfl_xor(v, 2);
    v += __shfl_xor(v, 4);
    v += __shfl_xor(v, 8);
    return v;
}

// QO: type of grad_q and grad_k (the storage type, or float partial gradients where value heads share a key head).
template <typename E, typename QO, int DKP>
__global__ void __launch_bounds__(256) delta_input_grad_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kStateCols, KT = DKP / 16;
    struct Columns {
        typename M::template Derived<kChunk, NV> x, r;
        typename M::template Input<kChunk, NV> go;
        typename M::template Derived<DKP, NV> s, ds;
    };
    struct Rows {
        typename M::template Input<kChunk, DKP> q, k;
        typename M::template Derived<kChunk, kChunk> m, n;
    };
    union Shared {
        Columns c;
        Rows w;
        __device__ Shared() {}
    };
    __shared__ Shared u;
    __shared__ Decay y;
    __shared__ float row_beta[kChunk], row_c[kChunk], row_e[kChunk], col_c[4][kChunk], dot_v[kChunk], inner[4];
    const DeltaWhere w = delta_where(args, blockIdx.y, blockIdx.x);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lr = wave * 16 + (lane >> 4) * 4, lc = lane & 15;
    const int present = args.T - w.t0 < kChunk ? args.T - w.t0 : kChunk;
    // rows of the dense outputs: (t, b, head) of Hv heads; grad_q / grad_k per value head or, unshared, per key head
    const int64_t row0 = static_cast<int64_t>(w.t0) * args.B * args.Hv + w.head, row_step = static_cast<int64_t>(args.B) * args.Hv;
    E* gv = static_cast<E*>(args.grad_v) + row0 * args.Dv;
    QO* gq = static_cast<QO*>(args.grad_q) + row0 * args.Dk;
    QO* gk = static_cast<QO*>(args.grad_k) + row0 * args.Dk;
    if (w.rows == 0) {
        for (int i = threadIdx.x; i < present * args.Dv; i += 256)
            gv[i / args.Dv * row_step * args.Dv + i % args.Dv] = narrow<E>(0.f);
        for (int i = threadIdx.x; i < present * args.Dk; i += 256) {
            gq[i / args.Dk * row_step * args.Dk + i % args.Dk] = narrow<QO>(0.f);
            gk[i / args.Dk * row_step * args.Dk + i % args.Dk] = narrow<QO>(0.f);
        }
        for (int i = threadIdx.x; i < present; i += 256) {
            args.grad_g[row0 + i * row_step] = 0.f;
            args.grad_beta[row0 + i * row_step] = 0.f;
        }
        return;
    }
    decay_of(args, w, y);
    const int64_t at = static_cast<int64_t>(w.head) * args.chunks + w.chunk;
    const E* pv = row_of<E>(args.v, w, w.hv);
    const E* pg = row_of<E>(args.grad_o, w, w.hv);

    f32x4 y1[KT], y2[KT], y3[KT], da[4], dp[4];
#pragma unroll
    for (int i = 0; i < KT; ++i) y1[i] = y2[i] = y3[i] = zero4();
#pragma unroll
    for (int i = 0; i < 4; ++i) da[i] = dp[i] = zero4();
    float v_dot = 0.f, s_dot = 0.f;
    for (int v0 = 0; v0 < args.cols; v0 += NV) {
        __syncthreads();
        {   // dX: 64 rows of 4 times 8 columns, one each; with it dV and v . dX
            const int i = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8;
            float x[8], v[8];
            load8<float>(args.inner + (at * kChunk + i) * args.cols, v0 + c, args.cols, true, x);
            u.c.x.put(i, c, x);
            load8<E>(pv + (i < w.rows ? i : 0) * args.v.t, v0 + c, i < w.rows ? args.Dv : 0, args.v.wide != 0, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v_dot += v[j] * x[j];
            if (i < present) {
                const float beta = i < w.rows ? y.beta[i] : 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (v0 + c + j < args.Dv) gv[i * row_step * args.Dv + v0 + c + j] = narrow<E>(i < w.rows ? beta * x[j] : 0.f);
            }
        }
        stage<kChunk, NV, 256>(u.c.r, const_cast<const float*>(args.added) + at * kChunk * args.cols + v0, args.cols, kChunk, NV, true);
        stage<kChunk, NV, 256>(u.c.go, pg + v0, args.grad_o.t, w.rows, args.Dv - v0, args.grad_o.wide != 0);
#pragma unroll
        for (int i = 0; i < DKP * NV / 8; i += 256) {
            const int seg = i + threadIdx.x, row = seg / (NV / 8), c = seg % (NV / 8) * 8;
            float s[8], ds[8];
            load8<float>(args.states + (at * DKP + row) * args.cols, v0 + c, args.cols, true, s);
            load8<float>(args.state_grads + (at * DKP + row) * args.cols, v0 + c, args.cols, true, ds);
            u.c.s.put(row, c, s);
            u.c.ds.put(row, c, ds);
#pragma unroll
            for (int j = 0; j < 8; ++j) s_dot += s[j] * ds[j];
        }
        __syncthreads();
        const auto fx = u.c.x.rows(wave * 16, 0);
        const auto fg = u.c.go.rows(wave * 16, 0);
        const auto fr = u.c.r.rows(wave * 16, 0);
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            const auto fs = u.c.s.rows(i * 16, 0);
            y1[i] = mma(fx, fs, y1[i]);
            y2[i] = mma(fg, fs, y2[i]);
            y3[i] = mma(fr, u.c.ds.rows(i * 16, 0), y3[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i <= wave) {
                const auto f = u.c.r.rows(i * 16, 0);
                da[i] = mma(fx, f, da[i]);
                dp[i] = mma(fg, f, dp[i]);
            }
    }
    // v . dX: four threads share a row;  <S, dS'>: the whole workgroup
    v_dot += __shfl_xor(v_dot, 1);
    v_dot += __shfl_xor(v_dot, 2);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s_dot += __shfl_xor(s_dot, d);
    __syncthreads();
    if ((threadIdx.x & 3) == 0) dot_v[threadIdx.x >> 2] = v_dot;
    if (lane == 0) inner[wave] = s_dot;
    stage<kChunk, DKP, 256>(u.w.q, row_of<E>(args.q, w, w.hk), args.q.t, w.rows, args.Dk, args.q.wide != 0);
    stage<kChunk, DKP, 256>(u.w.k, row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk, args.k.wide != 0);
    __syncthreads();

    // M, N and the sums over their products with A and P
    float sum_beta[4] = {}, sum_c[4] = {};
#pragma unroll
    for (int block = 0; block < 4; ++block) {
        f32x4 kk = zero4(), qk = zero4();
        if (block <= wave) {
#pragma unroll
            for (int s = 0; s < DKP; s += 32) {
                const auto f = u.w.k.rows(block * 16, s);
                kk = mma(u.w.k.rows(wave * 16, s), f, kk);
                qk = mma(u.w.q.rows(wave * 16, s), f, qk);
            }
        }
        float col = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = lr + e, j = block * 16 + lc;
            const float decay = i >= j ? gap(y, i, j) : 0.f;
            const float a_grad = i > j ? -da[block][e] * decay : 0.f;
            const float p_grad = i >= j ? dp[block][e] * decay * args.scale : 0.f;
            const float m = a_grad * y.beta[i];
            const float both = m * kk[e] + p_grad * qk[e];
            sum_beta[e] += a_grad * kk[e];
            sum_c[e] += both;
            col += both;
            u.w.m.put(i, j, m);
            u.w.n.put(i, j, p_grad);
        }
        col += __shfl_xor(col, 16);
        col += __shfl_xor(col, 32);
        if (lane < 16) col_c[wave][block * 16 + lc] = col;
    }
    // k . Y1, q . Y2, k . Y3 by row
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float d1 = 0.f, d2 = 0.f, d3 = 0.f;
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            const float kv = u.w.k.get(lr + e, i * 16 + lc), qv = u.w.q.get(lr + e, i * 16 + lc);
            d1 += kv * y1[i][e];
            d2 += qv * y2[i][e];
            d3 += kv * y3[i][e];
        }
        const float a = y.a[lr + e], beta = y.beta[lr + e];
        const float rest = row_sum16(sum_c[e] - beta * a * d1 + args.scale * a * d2);
        const float e_row = y.d[lr + e] * row_sum16(d3);
        const float b_row = row_sum16(sum_beta[e] - a * d1);
        if (lc == 0) {
            row_c[lr + e] = rest - e_row;
            row_e[lr + e] = e_row;
            row_beta[lr + e] = b_row;
        }
    }
    __syncthreads();
    if (wave == 0) {
        const int i = lane;
        const bool here = i < w.rows;
        double e_sum = here ? row_e[i] : 0.0;
        double dc = row_c[i];
#pragma unroll
        for (int o = 0; o < 4; ++o) dc -= col_c[o][i];
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) e_sum += __shfl_xor(e_sum, d);
        if (i == 63)
            dc += e_sum + static_cast<double>(y.a_last) * (static_cast<double>(inner[0]) + inner[1] + inner[2] + inner[3]);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {   // sums from the row to the end
            const double other = __shfl_down(dc, d);
            if (i + d < 64) dc += other;
        }
        if (i < present) {
            args.grad_g[row0 + i * row_step] = here ? static_cast<float>(dc) : 0.f;
            args.grad_beta[row0 + i * row_step] = here ? row_beta[i] + dot_v[i] : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < KT; ++i) {
        f32x4 q, k;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = y.a[lr + e];
            q[e] = args.scale * a * y2[i][e];
            k[e] = y.d[lr + e] * y3[i][e] - y.beta[lr + e] * a * y1[i][e];
        }
#pragma unroll
        for (int s = 0; s < kChunk; s += 32) {
            const auto fk = u.w.k.cols(i * 16, s);
            if (s <= wave * 16) {   // rows of this wavefront against columns up to the diagonal
                q = mma(u.w.n.rows(wave * 16, s), fk, q);
                k = mma(u.w.m.rows(wave * 16, s), fk, k);
            }
            if (s + 32 > wave * 16) {
                k = mma(u.w.m.cols(wave * 16, s), fk, k);
                k = mma(u.w.n.cols(wave * 16, s), u.w.q.cols(i * 16, s), k);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = i * 16 + lc;
            if (lr + e < present && col < args.Dk) {
                const bool here = lr + e < w.rows;
                gq[(lr + e) * row_step * args.Dk + col] = narrow<QO>(here ? q[e] : 0.f);
                gk[(lr + e) * row_step * args.Dk + col] = narrow<QO>(here ? k[e] : 0.f);
            }
        }
    }
}

// grad[row, hk, :] = sum over the value heads that share key head hk, in order.
template <typename E>
__global__ void __launch_bounds__(256)
delta_shared_grad_kernel(const float* __restrict__ part_q, const float* __restrict__ part_k, E* __restrict__ grad_q,
                         E* __restrict__ grad_k, int64_t rows, int Dk, int share) {
    const float* part = blockIdx.y == 0 ? part_q : part_k;
    E* grad = blockIdx.y == 0 ? grad_q : grad_k;
    const int64_t total = rows * Dk;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / Dk;
        const int c = static_cast<int>(i - row * Dk);
        float sum = 0.f;
        for (int h = 0; h < share; ++h) sum += part[(row * share + h) * Dk + c];
        grad[i] = narrow<E>(sum);
    }
}

// ---- launches -----------------------------------------------------------------------------------

hipError_t delta_forward_f32(const DeltaArgs& a, hipStream_t st);
hipError_t delta_forward_bf16(const DeltaArgs& a, hipStream_t st);
hipError_t delta_backward_f32(const DeltaArgs& a, void* grad_q, void* grad_k, hipStream_t st);
hipError_t delta_backward_bf16(const DeltaArgs& a, void* grad_q, void* grad_k, hipStream_t st);

template <typename E, int DKP>
hipError_t delta_forward_as(const DeltaArgs& a, hipStream_t st) {
    const dim3 pieces(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.B * a.Hv));
    const dim3 columns(static_cast<unsigned>(a.cols / kStateCols), static_cast<unsigned>(a.B * a.Hv));
    hipError_t err = hipSuccess;
    if (a.chunks > 0) err = launch(delta_inverse_kernel<E, DKP>, pieces, dim3(256), st, a);
    if (err == hipSuccess) err = launch(delta_state_kernel<E, DKP>, columns, dim3(kStateThreads), st, a);
    if (err == hipSuccess && a.chunks > 0) err = launch(delta_output_kernel<E, DKP>, pieces, dim3(256), st, a);
    return err;
}

// grad_q, grad_k: where the gradients go in the end (a.grad_q and a.grad_k are partial ones where heads share keys)
template <typename E, int DKP>
hipError_t delta_backward_as(const DeltaArgs& a, void* grad_q, void* grad_k, hipStream_t st) {
    const dim3 pieces(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.B * a.Hv));
    const dim3 columns(static_cast<unsigned>(a.cols / kStateCols), static_cast<unsigned>(a.B * a.Hv));
    hipError_t err = hipSuccess;
    if (a.chunks > 0) err = launch(delta_inner_grad_kernel<E, DKP>, pieces, dim3(256), st, a);
    if (err == hipSuccess) err = launch(delta_state_grad_kernel<E, DKP>, columns, dim3(kStateThreads), st, a);
    if (err != hipSuccess || a.chunks == 0) return err;
    if (a.Hv == a.Hk) return launch(delta_input_grad_kernel<E, E, DKP>, pieces, dim3(256), st, a);
    err = launch(delta_input_grad_kernel<E, float, DKP>, pieces, dim3(256), st, a);
    if (err != hipSuccess) return err;
    const int64_t rows = static_cast<int64_t>(a.T) * a.B * a.Hk;
    const int64_t blocks = ceil_div(rows * a.Dk, 256);
    return launch(delta_shared_grad_kernel<E>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096), 2), dim3(256),
                  st, static_cast<const float*>(a.grad_q), static_cast<const float*>(a.grad_k), static_cast<E*>(grad_q),
                  static_cast<E*>(grad_k), rows, a.Dk, a.Hv / a.Hk);
}

// Keys of up to 64 values, and of up to 128.
#define SNNSEQ_DEFINE_DELTA(NAME, E)                                                                         \
    hipError_t delta_forward_##NAME(const DeltaArgs& a, hipStream_t st) {                                    \
        return a.Dk <= 64 ? delta_forward_as<E, 64>(a, st) : delta_forward_as<E, 128>(a, st);                \
    }                                                                                                        \
    hipError_t delta_backward_##NAME(const DeltaArgs& a, void* grad_q, void* grad_k, hipStream_t st) {       \
        return a.Dk <= 64 ? delta_backward_as<E, 64>(a, grad_q, grad_k, st)                                  \
                          : delta_backward_as<E, 128>(a, grad_q, grad_k, st);                                \
    }

}  // namespace snnseq

#endif  // SNNLIF_SEQ_DELTA_H
