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
// and 16 columns of the state, which they hold in accumulators.
//   forward    delta_inverse_kernel -> Tm;   delta_state_kernel -> S of every chunk, R, last state;   delta_output_kernel -> O
//              without a backward to come: delta_inverse_kernel -> Tm, P;   delta_state_kernel -> O, last state
//   backward   delta_inner_grad_kernel -> P^T dO;   delta_state_grad_kernel -> dS' of every chunk, dX;
//              delta_input_grad_kernel -> the gradients;   delta_shared_grad_kernel where heads share keys
// The state passes are bound by the latency of a chunk's chain of products (three forward, three backward, each
// through LDS), the others by memory.
//
// Measured, keys and values of 128 in bf16.  (a) 2048 steps of 4 sequences of 8 heads, with a backward: inverse 26 us
// (98 MB: 3.7 TB/s), state 57 (1.8 per chunk), output 37 (147 MB: 4.0 TB/s), inner gradients 27 (98 MB: 3.7 TB/s), state
// gradients 91 (2.9 per chunk), input gradients 112 (311 MB: 2.8 TB/s, one workgroup of 129 KB of LDS per CU).
// (b) 8192 steps of one sequence of 16 heads, nothing kept: inverse 52, state and output 234 (1.8 per chunk); in fp32 112
// and 399.
//
// Numbers.  States, R, Tm, dX and every sum are fp32.  In bf16 storage the products run on the bf16 matrix
// instructions; an input is exact there, and what is derived (Tm, X, R, P, the state, ...) is given as a sum of three
// bf16 parts, which keep all 24 bits.  With two parts errors came out ten times those of an fp32 evaluation (4e-6
// against 4e-7), and bf16 results were 1.2e-4 by norm from an fp32 evaluation's, 4e-5 with three, as more of them rounded
// the other way; the third part costs 12 us of 274 on a prompt of 8192 steps.  Products of parts below the last bit kept
// are left out.  In fp32 storage the products run on the fp32 matrix instructions.  The sums c are held in 64 bits: G
// needs their differences.
//
// Time steps at or behind a sequence's length have no row: they leave the state alone and their outputs are zero.
#ifndef SNNLIF_SEQ_DELTA_H
#define SNNLIF_SEQ_DELTA_H

#include "seq_common.h"

namespace snnseq {

constexpr int kChunk = 64;
constexpr int kStateCols = 16;  // columns of the state a workgroup of the state passes holds
constexpr int kCols = 32;       // columns of the state the other kernels take at a time

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

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

// Eight consecutive values as they lie in memory.
template <typename E> struct Raw8 { u32x4 r[sizeof(E) / 2]; };

// n values as bf16 parts: words[part][j] holds values 2j and 2j + 1.
template <int N, int n>
__device__ __forceinline__ void split(const float (&x)[n], uint32_t (&words)[N][n / 2]) {
    float rest[n];
#pragma unroll
    for (int j = 0; j < n; ++j) rest[j] = x[j];
#pragma unroll
    for (int part = 0; part < N; ++part)
#pragma unroll
        for (int j = 0; j < n; j += 2) {
            const bf16x2 pair = __builtin_convertvector(f32x2{rest[j], rest[j + 1]}, bf16x2);   // one instruction
            const uint32_t word = __builtin_bit_cast(uint32_t, pair);
            words[part][j / 2] = word;
            if (part + 1 < N) {
                rest[j] -= __builtin_bit_cast(float, word << 16);
                rest[j + 1] -= __builtin_bit_cast(float, word & 0xffff0000u);
            }
        }
}

// A matrix in LDS as N bf16 parts, row-major; 16 bytes of padding per row spread the rows over the banks.  Read and
// written in vectors of 16 bytes, like every struct below that lies in LDS: each asks for that alignment.
template <int N, int ROWS, int COLS>
struct TileH {
    static constexpr int ld = COLS + 8;
    alignas(16) uint16_t v[N][ROWS * ld];

    // n consecutive columns, c a multiple of 4
    template <int n>
    __device__ __forceinline__ void put(int r, int c, const float (&x)[n]) {
        uint32_t words[N][n / 2];
        split<N, n>(x, words);
#pragma unroll
        for (int part = 0; part < N; ++part) {
            uint16_t* p = &v[part][r * ld + c];
            if constexpr (n == 8) *reinterpret_cast<u32x4*>(p) = u32x4{words[part][0], words[part][1], words[part][2], words[part][3]};
            else *reinterpret_cast<u32x2*>(p) = u32x2{words[part][0], words[part][1]};
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
    __device__ __forceinline__ void put(int r, int c, const Raw8<bf16_t>& x) {
        static_assert(N == 1, "what lies in memory is one part");
        *reinterpret_cast<u32x4*>(&v[0][r * ld + c]) = x.r[0];
    }
    // rows r0 + (l / 16) * 4 .. + 3 of column c0 + l % 16, the layout of a 16 x 16 product; by the transposing read
    __device__ __forceinline__ f32x4 block(int r0, int c0) const {
        const int lane = threadIdx.x & 63;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int part = N - 1; part >= 0; --part) {
            const uint16_t* p = &v[part][(r0 + (lane >> 2)) * ld + c0 + (lane & 3) * 4];
            const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(const_cast<uint16_t*>(p)));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const short bits = w[e];
                x[e] += value_of(static_cast<uint16_t>(bits));
            }
        }
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
    alignas(16) float v[ROWS * ld];

    template <int n>
    __device__ __forceinline__ void put(int r, int c, const float (&x)[n]) {
#pragma unroll
        for (int j = 0; j < n; j += 4)
            *reinterpret_cast<f32x4*>(&v[r * ld + c + j]) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
    }
    __device__ __forceinline__ void put(int r, int c, float x) { v[r * ld + c] = x; }
    __device__ __forceinline__ void put(int r, int c, const Raw8<float>& x) {
        *reinterpret_cast<u32x4*>(&v[r * ld + c]) = x.r[0];
        *reinterpret_cast<u32x4*>(&v[r * ld + c + 4]) = x.r[1];
    }
    __device__ __forceinline__ f32x4 block(int r0, int c0) const {
        const int lane = threadIdx.x & 63;
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[(r0 + (lane >> 4) * 4 + e) * ld + c0 + (lane & 15)];
        return x;
    }
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

static_assert(alignof(TileH<1, 16, 32>) == 16 && alignof(TileF<16, 32>) == 16, "tiles are accessed in vectors of 16 bytes");

// Fragments in memory: 64 lanes times 16 bytes are one run, so that a wavefront reads an operand of its products
// straight into registers, one access of 1 KiB per part, without LDS and with one address.
template <typename F> constexpr int frag_bytes() { return static_cast<int>(sizeof(F)) * 64; }

template <typename F>
__device__ __forceinline__ F load_frag(const char* base, int index) {
    const u32x4* p = reinterpret_cast<const u32x4*>(base + index * frag_bytes<F>()) + (threadIdx.x & 63);
    struct Words { u32x4 x[sizeof(F) / 16]; } w;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(F) / 16); ++i) w.x[i] = p[i * 64];
    return __builtin_bit_cast(F, w);
}

template <typename F>
__device__ __forceinline__ void store_frag(char* base, int index, const F& f) {
    u32x4* p = reinterpret_cast<u32x4*>(base + index * frag_bytes<F>()) + (threadIdx.x & 63);
    struct Words { u32x4 x[sizeof(F) / 16]; };
    const Words w = __builtin_bit_cast(Words, f);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(F) / 16); ++i) p[i * 64] = w.x[i];
}

// Eight fp32 values as a fragment's values.
__device__ __forceinline__ void frag_of(const float (&x)[8], FragH<3>& f) {
    uint32_t words[3][4];
    split<3, 8>(x, words);
#pragma unroll
    for (int part = 0; part < 3; ++part)
        f.p[part] = __builtin_bit_cast(bf16x8, u32x4{words[part][0], words[part][1], words[part][2], words[part][3]});
}
__device__ __forceinline__ void frag_of(const float (&x)[8], FragF& f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = x[j];
}

// What a storage type computes with: tiles of inputs, and of derived values (Fine).
template <typename E> struct Mode;
template <> struct Mode<bf16_t> {
    template <int R, int C> using Input = TileH<1, R, C>;
    template <int R, int C> using Fine = TileH<3, R, C>;
    using InputFrag = FragH<1>;
    using FineFrag = FragH<3>;
};
template <> struct Mode<float> {
    template <int R, int C> using Input = TileF<R, C>;
    template <int R, int C> using Fine = TileF<R, C>;
    using InputFrag = FragF;
    using FineFrag = FragF;
};

// Bytes of a chunk's operands in this form: keys (or queries) by rows or transposed, and a 64 x 64 matrix.
template <typename E> constexpr int keys_bytes(int dkp) { return dkp / 8 * frag_bytes<typename Mode<E>::InputFrag>(); }
template <typename E> constexpr int square_bytes() { return 8 * frag_bytes<typename Mode<E>::FineFrag>(); }

// ---- arguments ----------------------------------------------------------------------------------

// A [T, B, heads, D] tensor whose rows of D values are dense.
struct DeltaTensor {
    const void* p;
    int64_t t, b, h;   // strides in elements
    int wide;          // D is a multiple of 8
};

// Decay of a chunk: the sums c in 64 bits and in units of log 2, a = e^c, d = e^{c_last - c}, and beta.  A row that
// does not exist has g = 0 and beta = 0.
struct alignas(16) Decay {
    double c[kChunk];
    float a[kChunk], d[kChunk], beta[kChunk];
};

struct DeltaArgs {
    int T, B, Hk, Hv, Dk, Dv;
    int chunks;                 // ceil(T / 64)
    int cols;                   // Dv rounded up to 32: columns of the matrices below
    float scale;
    const int32_t* lengths;     // [B] or nullptr
    DeltaTensor q, k, v, grad_o;
    const float *g, *beta;      // [T, B, Hv]
    const float *state, *grad_state;   // [B, Hv, Dk, Dv] or nullptr: the initial state, the gradient of the last one
    void* o;                    // [T, B, Hv, Dv]
    float* state_out;           // [B, Hv, Dk, Dv] or nullptr
    // per (batch entry, value head, chunk); matrices with a column of the state are transposed, as the state passes
    // hold them: each column of theirs is one run of memory
    Decay* decay;
    char *inverse, *inverse_t;  // Tm and its transpose, fragments (band of 16 rows, 32 columns of it); the latter or nullptr
    char *keys, *keys_t;        // per (batch entry, key head, chunk): K by rows, and transposed, fragments
    float* added;               // R, [cols, 64]
    float* states;              // state before the chunk, [cols, DKP]
    // a forward with its output in the state pass: Q by rows as keys, and P as Tm; else nullptr
    char *queries, *scores;
    // backward
    char* queries_t;            // as keys_t
    float* inner;               // P^T dO, then dX, [cols, 64]
    float* state_grads;         // gradient of the state after the chunk, [cols, DKP]
    void *grad_q, *grad_k;      // [T, B, Hk, Dk] of the storage type, or fp32 [T, B, Hv, Dk] where heads share keys
    void* grad_v;               // [T, B, Hv, Dv]
    float *grad_g, *grad_beta;  // [T, B, Hv]
    float* grad_initial;        // [B, Hv, Dk, Dv] or nullptr
};

struct DeltaWhere {  // the chunk (or head) a workgroup works on
    int b, hv, hk, chunk, head;
    int t0, rows;    // first step and how many of its 64 rows exist
    int64_t at;      // its place among the matrices of the value heads
    int64_t key_at;  // and of the key heads
};

__device__ __forceinline__ int delta_length(const DeltaArgs& a, int b) {
    if (a.lengths == nullptr) return a.T;
    const int n = a.lengths[b];
    return n < 0 ? 0 : n > a.T ? a.T : n;
}

// `length` of the head's sequence, where it is known already
__device__ __forceinline__ DeltaWhere delta_where(const DeltaArgs& a, int head, int chunk, int length = -1) {
    DeltaWhere w;
    w.head = head;
    w.b = head / a.Hv;
    w.hv = head - w.b * a.Hv;
    w.hk = w.hv / (a.Hv / a.Hk);
    w.chunk = chunk;
    w.t0 = chunk * kChunk;
    const int left = (length < 0 ? delta_length(a, w.b) : length) - w.t0;
    w.rows = left < 0 ? 0 : left > kChunk ? kChunk : left;
    w.at = static_cast<int64_t>(head) * a.chunks + chunk;
    w.key_at = (static_cast<int64_t>(w.b) * a.Hk + w.hk) * a.chunks + chunk;
    return w;
}

// ---- staging ------------------------------------------------------------------------------------

// Eight consecutive values of a row, from any element on.  Without a look at the values, so that all loads of a thread
// are under way together.  WIDE: rows of a multiple of eight values; what lies behind `valid` is read at the row's
// beginning, and keep_valid takes it out later.  Otherwise the eight that would reach over the row's end are the last
// eight instead, and keep_valid moves them to their places.
template <bool WIDE, typename E>
__device__ __forceinline__ Raw8<E> load_raw8(const E* row, int c, int valid) {
    using memory_t = u32x4 __attribute__((aligned(sizeof(E))));
    Raw8<E> x;
    if (WIDE || valid >= 8) {
        const int at = WIDE ? (c < valid ? c : 0) : (c < valid - 8 ? c : valid - 8);
        const memory_t* p = reinterpret_cast<const memory_t*>(row + at);
#pragma unroll
        for (int h = 0; h < static_cast<int>(sizeof(E) / 2); ++h) x.r[h] = p[h];
    } else {   // fewer than eight: those behind are in front, and moved out
        uint32_t bits[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const E v = row[valid - 8 + j > 0 ? valid - 8 + j : 0];
            if constexpr (sizeof(E) == 4) bits[j] = __builtin_bit_cast(uint32_t, v);
            else bits[j] = v.bits;
        }
        if constexpr (sizeof(E) == 4) {
            x.r[0] = u32x4{bits[0], bits[1], bits[2], bits[3]};
            x.r[1] = u32x4{bits[4], bits[5], bits[6], bits[7]};
        } else {
            x.r[0] = u32x4{bits[0] | bits[1] << 16, bits[2] | bits[3] << 16, bits[4] | bits[5] << 16, bits[6] | bits[7] << 16};
        }
    }
    return x;
}

// Zero at and behind `valid`, and everywhere where the row does not exist.
template <bool WIDE, typename E>
__device__ __forceinline__ Raw8<E> keep_valid(Raw8<E> x, int c, int valid, bool exists) {
    constexpr int words = 2 * static_cast<int>(sizeof(E)), per = 4 / static_cast<int>(sizeof(E));   // values per word
    if constexpr (WIDE) {
#pragma unroll
        for (int h = 0; h < words / 4; ++h) x.r[h] = exists && c < valid ? x.r[h] : u32x4{0, 0, 0, 0};
    } else {
        const int last = valid - 8, by = exists ? (c > last ? c - last : 0) : 8;   // places to move down, zeros behind
        uint32_t w[words];
#pragma unroll
        for (int j = 0; j < words; ++j) w[j] = by < 8 ? x.r[j / 4][j % 4] : 0u;
#pragma unroll
        for (int step = 4; step >= per; step >>= 1)
#pragma unroll
            for (int j = 0; j < words; ++j) {
                const uint32_t from = j + step / per < words ? w[j + step / per] : 0u;
                w[j] = by & step ? from : w[j];
            }
        if constexpr (per == 2) {
#pragma unroll
            for (int j = 0; j < words; ++j) {
                const uint32_t above = j + 1 < words ? w[j + 1] : 0u;
                w[j] = by & 1 ? w[j] >> 16 | above << 16 : w[j];
            }
        }
#pragma unroll
        for (int j = 0; j < words; ++j) x.r[j / 4][j % 4] = w[j];
    }
    return x;
}

__device__ __forceinline__ void values_of(const Raw8<bf16_t>& x, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __builtin_bit_cast(float, x.r[0][j] << 16);
        v[2 * j + 1] = __builtin_bit_cast(float, x.r[0][j] & 0xffff0000u);
    }
}
__device__ __forceinline__ void values_of(const Raw8<float>& x, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t bits = x.r[j / 4][j % 4];   // a bit cast of the vector's element itself reads element 0
        v[j] = __builtin_bit_cast(float, bits);
    }
}

// ROWS x COLS of a tensor, eight values of a row per access, requested now (load) and put into LDS later (store), so
// that a product can run in between.
template <bool WIDE, typename E, int ROWS, int COLS, int THREADS>
struct Ahead {
    static constexpr int total = ROWS * COLS / 8, n = (total + THREADS - 1) / THREADS;
    Raw8<E> x[n];
    int rows, valid;
    // rows `stride` values apart, of which `rows_` x `valid_` exist (one at least of each)
    __device__ __forceinline__ void load(const E* base, int64_t stride, int rows_, int valid_) {
        rows = rows_;
        valid = valid_;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int seg = i * THREADS + threadIdx.x, r = seg / (COLS / 8), c = seg % (COLS / 8) * 8;
            x[i] = load_raw8<WIDE, E>(base + (r < rows ? r : 0) * stride, c, valid);
        }
    }
    __device__ __forceinline__ Raw8<E> get(int i) const {
        const int seg = i * THREADS + threadIdx.x, r = seg / (COLS / 8), c = seg % (COLS / 8) * 8;
        return keep_valid<WIDE, E>(x[i], c, valid, r < rows);
    }
    template <typename Tile>
    __device__ __forceinline__ void store(Tile& tile) const {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int seg = i * THREADS + threadIdx.x;
            if (total % THREADS != 0 && seg >= total) break;
            tile.put(seg / (COLS / 8), seg % (COLS / 8) * 8, get(i));
        }
    }
};

// ROWS x COLS of an fp32 matrix without gaps, stored as the parts a tile keeps.
template <int ROWS, int COLS, int THREADS>
struct MatrixAhead {
    static constexpr int total = ROWS * COLS / 8, n = (total + THREADS - 1) / THREADS;
    Raw8<float> x[n];
    __device__ __forceinline__ static bool mine(int i) {
        return total % THREADS == 0 || i * THREADS + static_cast<int>(threadIdx.x) < total;
    }
    __device__ __forceinline__ void load(const float* base) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int seg = mine(i) ? i * THREADS + threadIdx.x : 0;
            x[i] = load_raw8<true, float>(base, seg * 8, total * 8);
        }
    }
    template <typename Tile>
    __device__ __forceinline__ void store(Tile& tile) const {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int seg = i * THREADS + threadIdx.x;
            if (!mine(i)) break;
            float v[8];
            values_of(x[i], v);
            tile.put(seg / (COLS / 8), seg % (COLS / 8) * 8, v);
        }
    }
};

template <typename E>
__device__ __forceinline__ const E* row_of(const DeltaTensor& x, const DeltaWhere& w, int head) {
    return static_cast<const E*>(x.p) + w.t0 * x.t + w.b * x.b + head * x.h;
}

// By the first wavefront.
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
    double c = g * 1.4426950408889634;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double other = __shfl_up(c, s);
        if (lane >= s) c += other;
    }
    const double last = __shfl(c, 63);
    out.c[lane] = c;
    out.a[lane] = exp2f(static_cast<float>(c));
    out.d[lane] = exp2f(static_cast<float>(last - c));
    out.beta[lane] = beta;
}

struct DecayAhead {
    static constexpr unsigned n = sizeof(Decay) / 16;
    u32x4 x;
    __device__ __forceinline__ void load(const DeltaArgs& args, int64_t at) {
        x = reinterpret_cast<const u32x4*>(args.decay + at)[threadIdx.x < n ? threadIdx.x : 0];
    }
    __device__ __forceinline__ void store(Decay& out) const {
        if (threadIdx.x < n) reinterpret_cast<u32x4*>(&out)[threadIdx.x] = x;
    }
};
static_assert(alignof(Decay) == 16, "a Decay is copied in vectors");

__device__ __forceinline__ float gap(const Decay& y, int i, int j) {  // G_ij
    return __builtin_amdgcn_exp2f(static_cast<float>(y.c[i] - y.c[j]));
}

// What a later kernel reads: the non-temporal hint.  A load waits for the stores before it, and without the hint the
// state pass over 8192 steps of 16 heads (350 MB of matrices) took 259 us instead of 228.
__device__ __forceinline__ void store_later(float* p, f32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p)); }

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

// Workgroups go to the eight XCDs in turn, each with an L2 of its own: the workgroups of a head, which read the same
// keys and matrices, are given to one XCD.
__device__ __forceinline__ int piece_in_l2(int total) {
    const int per = total / 8, id = blockIdx.x;
    return id < per * 8 ? (id % 8) * per + id / 8 : id;
}

// The transpose of staged keys or queries, as fragments (16 key columns, half of the rows), by WAVES wavefronts.
template <typename E, int DKP, int WAVES, typename Tile>
__device__ __forceinline__ void store_transposed(const Tile& tile, char* out) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < DKP / 8; i += WAVES) {
        const int index = i + wave;
        if (DKP / 8 % WAVES != 0 && index >= DKP / 8) break;
        store_frag(out, index, tile.cols(index / 2 * 16, index % 2 * 32));
    }
}

// ---- Tm = (I + A)^-1 ----------------------------------------------------------------------------

struct Square { alignas(16) float v[kChunk][kChunk + 4]; };

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

// OUTPUT: and what the state pass needs for the output, the queries and P.
template <typename E, bool WIDE, int DKP, bool OUTPUT>
__global__ void __launch_bounds__(256) delta_inverse_kernel(DeltaArgs args) {
    using M = Mode<E>;
    union First {   // K is done with when the inversion needs its scratch
        typename M::template Input<kChunk, DKP> k;
        Square scratch;
        __device__ First() {}
    };
    union Second {  // and P is in memory
        typename M::template Fine<kChunk, kChunk> p;
        Square t;
        __device__ Second() {}
    };
    __shared__ First u;
    __shared__ Second z;
    __shared__ Square a;
    __shared__ typename M::template Input<OUTPUT ? kChunk : 1, DKP> q;
    __shared__ Decay y;
    Square& t = z.t;
    const DeltaWhere w = delta_where(args, blockIdx.y, blockIdx.x);
    if (w.rows == 0) return;
    Ahead<WIDE, E, kChunk, DKP, 256> k;
    k.load(row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk);
    if constexpr (OUTPUT) {
        Ahead<WIDE, E, kChunk, DKP, 256> q_next;
        q_next.load(row_of<E>(args.q, w, w.hk), args.q.t, w.rows, args.Dk);
        q_next.store(q);
    }
    decay_of(args, w, y);
    k.store(u.k);
    __syncthreads();
    if (threadIdx.x < sizeof(Decay) / 16)
        reinterpret_cast<u32x4*>(args.decay + w.at)[threadIdx.x] = reinterpret_cast<const u32x4*>(&y)[threadIdx.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (w.hv % (args.Hv / args.Hk) == 0) {   // the first of the value heads that share these keys
#pragma unroll
        for (int s = 0; s < DKP / 32; ++s)
            store_frag(args.keys + w.key_at * keys_bytes<E>(DKP), wave * (DKP / 32) + s, u.k.rows(wave * 16, s * 32));
        store_transposed<E, DKP, 4>(u.k, args.keys_t + w.key_at * keys_bytes<E>(DKP));
        if constexpr (OUTPUT) {
#pragma unroll
            for (int s = 0; s < DKP / 32; ++s)
                store_frag(args.queries + w.key_at * keys_bytes<E>(DKP), wave * (DKP / 32) + s, q.rows(wave * 16, s * 32));
        }
    }
    if constexpr (OUTPUT) {
#pragma unroll
        for (int block = 0; block < 4; ++block) {
            f32x4 acc = zero4();
            if (block <= wave) {
#pragma unroll
                for (int s = 0; s < DKP; s += 32) acc = mma(q.rows(wave * 16, s), u.k.rows(block * 16, s), acc);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = wave * 16 + (lane >> 4) * 4 + e, j = block * 16 + (lane & 15);
                z.p.put(i, j, i >= j ? args.scale * acc[e] * gap(y, i, j) : 0.f);
            }
        }
        // a wavefront reads back its own rows only
#pragma unroll
        for (int s = 0; s < 2; ++s)
            store_frag(args.scores + w.at * square_bytes<E>(), wave * 2 + s, z.p.rows(wave * 16, s * 32));
        __syncthreads();
    }
    for (int i = threadIdx.x; i < kChunk * (kChunk + 4); i += 256) (&t.v[0][0])[i] = 0.f;
    for (int block = 0; block <= wave; ++block) {
        f32x4 acc = zero4();
#pragma unroll
        for (int s = 0; s < DKP; s += 32) acc = mma(u.k.rows(wave * 16, s), u.k.rows(block * 16, s), acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = wave * 16 + (lane >> 4) * 4 + e, j = block * 16 + (lane & 15);
            a.v[i][j] = i > j ? y.beta[i] * acc[e] * gap(y, i, j) : 0.f;
        }
    }
    __syncthreads();
    invert_unit_lower(a, t, u.scratch);
    // fragment (band of rows or columns, half of the contraction): a wavefront writes both halves of its band
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int r = wave * 16 + (lane & 15), c = s * 32 + (lane >> 4) * 8;
        float x[8];
        typename M::FineFrag f;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = t.v[r][c + j];
        frag_of(x, f);
        store_frag(args.inverse + w.at * square_bytes<E>(), wave * 2 + s, f);
        if (args.inverse_t != nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = t.v[c + j][r];
            frag_of(x, f);
            store_frag(args.inverse_t + w.at * square_bytes<E>(), wave * 2 + s, f);
        }
    }
}

// ---- the state passes ---------------------------------------------------------------------------
//
// A workgroup of four wavefronts holds kStateCols columns of a head's state: wavefront w rows 16 w.. of the chunk in
// the first two products, DKP / 64 tiles of 16 state rows in the last one.  The chain from chunk to chunk -- three
// products, each through LDS to the next -- is all that counts, so nothing else is on it: keys and matrices come as
// fragments, straight into registers, and LDS holds only what the wavefronts exchange.  The next chunk's operand is
// requested as soon as a product has used this one's, into the same registers: a chunk's time ahead, while the matrix
// instructions run.  (Requested all together, or before the products, they cost the chain 1900 cycles of 4800: each
// occupies the memory path of the CU for 16.)  Loads are never under a condition, which would make every wait one for
// all of them; behind the last chunk they fetch it once more.

constexpr int kStateThreads = 256;

// The 4 x TILES state values of a lane: state rows tile_row(i) .. + 3 of column v0 + lane % 16, kept transposed in LDS.
template <int DKP>
struct StateTiles {
    static constexpr int n = DKP / 64;
    f32x4 s[n];
    __device__ __forceinline__ static int row(int i) {
        return ((threadIdx.x >> 6) + 4 * i) * 16 + ((threadIdx.x & 63) >> 4) * 4;
    }
    template <typename Tile>
    __device__ __forceinline__ void put(Tile& tile) const {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            float v4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v4[e] = s[i][e];
            tile.put(threadIdx.x & 15, row(i), v4);
        }
    }
    __device__ __forceinline__ void load(const float* state, int64_t head, int Dk, int Dv, int col) {
#pragma unroll
        for (int i = 0; i < n; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[i][e] = state != nullptr && row(i) + e < Dk && col < Dv ? state[(head * Dk + row(i) + e) * Dv + col] : 0.f;
    }
    __device__ __forceinline__ void save(float* state, int64_t head, int Dk, int Dv, int col) const {
        if (state == nullptr || col >= Dv) return;
#pragma unroll
        for (int i = 0; i < n; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row(i) + e < Dk) state[(head * Dk + row(i) + e) * Dv + col] = s[i][e];
    }
    __device__ __forceinline__ void keep(float* matrix, int col) const {   // matrix [cols, DKP]
#pragma unroll
        for (int i = 0; i < n; ++i) store_later(matrix + static_cast<int64_t>(col) * DKP + row(i), s[i]);
    }
};

// Four rows of one column of a strided input, in the layout of a product; requested and looked at apart, as above.
template <typename E>
struct ColumnAhead {
    E x[4];
    int rows;
    __device__ __forceinline__ void load(const DeltaTensor& t, const DeltaWhere& w, int head, int row, int col, int valid) {
        rows = col < valid ? w.rows - row : 0;
        const E* p = row_of<E>(t, w, head) + (rows > 0 ? row * t.t + col : 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = p[min(e, max(rows - 1, 0)) * t.t];
    }
    __device__ __forceinline__ float get(int e) const { return e < rows ? widen(x[e]) : 0.f; }
};

// What the forward pass takes from memory for a chunk.
template <typename E, int DKP, bool OUTPUT>
struct StateOperands {
    using M = Mode<E>;
    typename M::InputFrag k[DKP / 32], kt[DKP / 64][2], q[OUTPUT ? DKP / 32 : 1];
    typename M::FineFrag inverse[2];
    typename M::FineFrag p[OUTPUT ? 2 : 1];
    f32x4 a, d, beta;
    float a_last;
    ColumnAhead<E> v;
    __device__ __forceinline__ void load_keys(const DeltaArgs& args, const DeltaWhere& w) {
        load_rows(k, args.keys + w.key_at * keys_bytes<E>(DKP));
        if constexpr (OUTPUT) load_rows(q, args.queries + w.key_at * keys_bytes<E>(DKP));
    }
    __device__ __forceinline__ static void load_rows(typename M::InputFrag (&x)[DKP / 32], const char* matrix) {
#pragma unroll
        for (int s = 0; s < DKP / 32; ++s) x[s] = load_frag<typename M::InputFrag>(matrix, (threadIdx.x >> 6) * (DKP / 32) + s);
    }
    __device__ __forceinline__ void load_inverse(const DeltaArgs& args, const DeltaWhere& w) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
            inverse[s] = load_frag<typename M::FineFrag>(args.inverse + w.at * square_bytes<E>(), (threadIdx.x >> 6) * 2 + s);
    }
    __device__ __forceinline__ void load_factors(const DeltaArgs& args, const DeltaWhere& w, int row, int col) {
        const Decay* y = args.decay + w.at;
        a = *reinterpret_cast<const f32x4*>(y->a + row);
        d = *reinterpret_cast<const f32x4*>(y->d + row);
        beta = *reinterpret_cast<const f32x4*>(y->beta + row);
        a_last = y->a[kChunk - 1];
        v.load(args.v, w, w.hv, row, col, args.Dv);
    }
    __device__ __forceinline__ void load_transposed(const DeltaArgs& args, const DeltaWhere& w) {
#pragma unroll
        for (int i = 0; i < DKP / 64; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s)
                kt[i][s] = load_frag<typename M::InputFrag>(args.keys_t + w.key_at * keys_bytes<E>(DKP), ((threadIdx.x >> 6) + 4 * i) * 2 + s);
    }
    __device__ __forceinline__ void load_scores(const DeltaArgs& args, const DeltaWhere& w) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
            p[s] = load_frag<typename M::FineFrag>(args.scores + w.at * square_bytes<E>(), (threadIdx.x >> 6) * 2 + s);
    }
};

// OUTPUT: with the output, for a forward that leaves nothing for a backward; the states and R then never reach memory.
template <typename E, int DKP, bool OUTPUT>
__global__ void __launch_bounds__(kStateThreads) delta_state_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kStateCols;
    __shared__ typename M::template Fine<NV, DKP> state;     // transposed
    __shared__ typename M::template Fine<NV, kChunk> x, r;   // transposed; X and d R
    __shared__ typename M::template Fine<NV, OUTPUT ? kChunk : 32> plain_r;
    const int tiles = args.cols / NV;
    const int piece = piece_in_l2(args.B * args.Hv * tiles), head = piece / tiles, v0 = (piece - head * tiles) * NV;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lc = lane & 15, row = wave * 16 + (lane >> 4) * 4, col = v0 + lc;
    const int length = delta_length(args, head / args.Hv), chunks = (length + kChunk - 1) / kChunk;

    StateOperands<E, DKP, OUTPUT> now;
    if (chunks > 0) {
        const DeltaWhere w = delta_where(args, head, 0, length);
        now.load_keys(args, w);
        now.load_factors(args, w, row, col);
        now.load_inverse(args, w);
        now.load_transposed(args, w);
        if constexpr (OUTPUT) now.load_scores(args, w);
    }
    StateTiles<DKP> s;
    s.load(args.state, head, args.Dk, args.Dv, col);
    s.put(state);
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const DeltaWhere w = delta_where(args, head, chunk + 1 < chunks ? chunk + 1 : chunk, length);   // the next one
        const int64_t at = static_cast<int64_t>(head) * args.chunks + chunk;
        __syncthreads();
        f32x4 acc[2] = {zero4(), zero4()}, o = zero4();   // o sums in the order of delta_output_kernel
        typename M::FineFrag f[DKP / 32];
#pragma unroll
        for (int c = 0; c < DKP / 32; ++c) f[c] = state.rows(0, c * 32);
#pragma unroll
        for (int c = 0; c < DKP / 32; ++c) acc[c % 2] = mma(now.k[c], f[c], acc[c % 2]);
        if constexpr (OUTPUT) {
#pragma unroll
            for (int c = 0; c < DKP / 32; ++c) o = mma(now.q[c], f[c], o);
        }
        __builtin_amdgcn_sched_barrier(0);
        now.load_keys(args, w);
        __builtin_amdgcn_sched_barrier(0);
        float out[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = now.beta[e] * (now.v.get(e) - now.a[e] * (acc[0][e] + acc[1][e]));
        x.put(lc, row, out);
        if constexpr (OUTPUT) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] *= args.scale * now.a[e];
        } else {
            s.keep(args.states + at * DKP * args.cols, col);
        }
        __syncthreads();
        f[0] = x.rows(0, 0);
        f[1] = x.rows(0, 32);
        acc[0] = mma(now.inverse[0], f[0], zero4());
        if (wave >= 2) {   // rows below 32 have nothing right of column 32
            acc[1] = mma(now.inverse[1], f[1], zero4());
            acc[0] += acc[1];
        }
        __builtin_amdgcn_sched_barrier(0);
        now.load_inverse(args, w);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 next_s[s.n];
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = now.d[e] * acc[0][e];
        r.put(lc, row, out);
        if constexpr (OUTPUT) {
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = acc[0][e];
            plain_r.put(lc, row, out);
        } else {
            store_later(args.added + (at * args.cols + col) * kChunk + row, acc[0]);
        }
#pragma unroll
        for (int i = 0; i < s.n; ++i) next_s[i] = now.a_last * s.s[i];
        __builtin_amdgcn_sched_barrier(0);
        now.load_factors(args, w, row, col);
        __syncthreads();
        f[0] = r.rows(0, 0);
        f[1] = r.rows(0, 32);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < s.n; ++i) next_s[i] = mma(now.kt[i][c], f[c], next_s[i]);
        __builtin_amdgcn_sched_barrier(0);
        now.load_transposed(args, w);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < s.n; ++i) s.s[i] = next_s[i];
        s.put(state);
        if constexpr (OUTPUT) {
            o = mma(now.p[0], plain_r.rows(0, 0), o);
            if (wave >= 2) o = mma(now.p[1], plain_r.rows(0, 32), o);
            now.load_scores(args, w);
            const int t0 = chunk * kChunk;
            E* p = static_cast<E*>(args.o) + ((static_cast<int64_t>(t0) + row) * args.B * args.Hv + head) * args.Dv + col;
            const int64_t stride = static_cast<int64_t>(args.B) * args.Hv * args.Dv;
            if (col < args.Dv) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (t0 + row + e < args.T) p[e * stride] = narrow<E>(t0 + row + e < length ? o[e] : 0.f);
            }
        }
    }
    if constexpr (OUTPUT) {   // steps in chunks that no row of the sequence reaches
        for (int t = chunks * kChunk + static_cast<int>(threadIdx.x >> 4); t < args.T; t += kStateThreads / 16) {
            const int c = v0 + (threadIdx.x & 15);
            if (c < args.Dv)
                static_cast<E*>(args.o)[(static_cast<int64_t>(t) * args.B * args.Hv + head) * args.Dv + c] = narrow<E>(0.f);
        }
    }
    s.save(args.state_out, head, args.Dk, args.Dv, col);
}

// ---- the output ---------------------------------------------------------------------------------
//
// Where a backward follows, the states are in memory for it anyway, and the output is cheaper here, over all chunks at
// once, than on the state pass's chain.  Bound by memory: mostly the fp32 state of a chunk and R.
//
// The kernels over all chunks have eight wavefronts: wavefront w works on rows 16 (w % 4) .. of the chunk and on half
// (w / 4) of the columns.

constexpr int kPieceThreads = 512;

// P of a chunk from staged Q and K; blocks above the diagonal are zero.
template <int DKP, typename TQ, typename TK, typename TP>
__device__ __forceinline__ void scores_of(const TQ& q, const TK& k, const Decay& y, float scale, TP& p) {
    const int lane = threadIdx.x & 63, band = threadIdx.x >> 6 & 3, half = threadIdx.x >> 8;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int block = b * 2 + half;   // both halves get one block of every pair
        f32x4 acc = zero4();
        if (block <= band) {
#pragma unroll
            for (int s = 0; s < DKP; s += 32) acc = mma(q.rows(band * 16, s), k.rows(block * 16, s), acc);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = band * 16 + (lane >> 4) * 4 + e, j = block * 16 + (lane & 15);
            p.put(i, j, i >= j ? scale * acc[e] * gap(y, i, j) : 0.f);
        }
    }
}

template <typename E, bool WIDE, int DKP>
__global__ void __launch_bounds__(kPieceThreads) delta_output_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kCols;
    struct Columns {
        typename M::template Fine<NV, DKP> state;
        typename M::template Fine<NV, kChunk> r;
    };
    struct Scores {
        typename M::template Input<kChunk, DKP> k;
        typename M::template Fine<kChunk, kChunk> p;
    };
    union Later {   // K is done with before the columns come, and P is in registers
        Scores s;
        Columns c;
        __device__ Later() {}
    };
    __shared__ typename M::template Input<kChunk, DKP> q;
    __shared__ Decay y;
    __shared__ Later u;
    const DeltaWhere w = delta_where(args, blockIdx.y, blockIdx.x);
    const int lane = threadIdx.x & 63, band = threadIdx.x >> 6 & 3, half = threadIdx.x >> 8;
    const int lr = band * 16 + (lane >> 4) * 4, lc = lane & 15;
    E* out = static_cast<E*>(args.o) + (static_cast<int64_t>(w.t0) * args.B * args.Hv + w.head) * args.Dv;
    const int64_t out_stride = static_cast<int64_t>(args.B) * args.Hv * args.Dv;
    const int present = args.T - w.t0 < kChunk ? args.T - w.t0 : kChunk;
    if (w.rows == 0) {
        for (int i = threadIdx.x; i < present * args.Dv; i += kPieceThreads)
            out[i / args.Dv * out_stride + i % args.Dv] = narrow<E>(0.f);
        return;
    }
    MatrixAhead<NV, DKP, kPieceThreads> state_next;
    MatrixAhead<NV, kChunk, kPieceThreads> r_next;
    const auto request = [&](int v0) {
        state_next.load(args.states + (w.at * args.cols + v0) * DKP);
        r_next.load(args.added + (w.at * args.cols + v0) * kChunk);
    };
    {
        Ahead<WIDE, E, kChunk, DKP, kPieceThreads> q_next, k_next;
        q_next.load(row_of<E>(args.q, w, w.hk), args.q.t, w.rows, args.Dk);
        k_next.load(row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk);
        DecayAhead y_next;
        y_next.load(args, w.at);
        request(0);
        y_next.store(y);
        q_next.store(q);
        k_next.store(u.s.k);
    }
    __syncthreads();
    scores_of<DKP>(q, u.s.k, y, args.scale, u.s.p);
    __syncthreads();
    const typename M::FineFrag p[2] = {u.s.p.rows(band * 16, 0), u.s.p.rows(band * 16, 32)};
    for (int v0 = 0; v0 < args.cols; v0 += NV) {
        __syncthreads();
        state_next.store(u.c.state);
        r_next.store(u.c.r);
        __syncthreads();
        if (v0 + NV < args.cols) request(v0 + NV);
        f32x4 acc = zero4();
#pragma unroll
        for (int s = 0; s < DKP; s += 32) acc = mma(q.rows(band * 16, s), u.c.state.rows(half * 16, s), acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= args.scale * y.a[lr + e];
        acc = mma(p[0], u.c.r.rows(half * 16, 0), acc);
        if (band >= 2) acc = mma(p[1], u.c.r.rows(half * 16, 32), acc);   // rows below 32 have nothing right of column 32
        const int col = v0 + half * 16 + lc;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (lr + e < present && col < args.Dv)
                out[(lr + e) * out_stride + col] = narrow<E>(lr + e < w.rows ? acc[e] : 0.f);
    }
}

// ---- backward: P^T dO ---------------------------------------------------------------------------
//
// All of dR that does not wait for the state, and the transposed queries as fragments for the state pass.  Bound by
// memory: q, k and dO read, as much written in fp32.

template <typename E, bool WIDE, int DKP>
__global__ void __launch_bounds__(kPieceThreads) delta_inner_grad_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kCols;
    struct Scores {
        typename M::template Input<kChunk, DKP> q, k;
    };
    union Later {   // Q and K are done with before dO comes
        Scores s;
        typename M::template Input<kChunk, NV> go;
        __device__ Later() {}
    };
    __shared__ Later u;
    __shared__ typename M::template Fine<kChunk, kChunk> p;
    __shared__ Decay y;
    const DeltaWhere w = delta_where(args, blockIdx.y, blockIdx.x);
    if (w.rows == 0) return;
    const int lane = threadIdx.x & 63, band = threadIdx.x >> 6 & 3, half = threadIdx.x >> 8;
    const int lr = band * 16 + (lane >> 4) * 4, lc = lane & 15;
    Ahead<WIDE, E, kChunk, NV, kPieceThreads> go_next;
    const E* pg = row_of<E>(args.grad_o, w, w.hv);
    const auto request = [&](int v0) {
        go_next.load(pg + v0, args.grad_o.t, w.rows, args.Dv - v0);
    };
    {
        Ahead<WIDE, E, kChunk, DKP, kPieceThreads> q_next, k_next;
        q_next.load(row_of<E>(args.q, w, w.hk), args.q.t, w.rows, args.Dk);
        k_next.load(row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk);
        DecayAhead y_next;
        y_next.load(args, w.at);
        request(0);
        y_next.store(y);
        q_next.store(u.s.q);
        k_next.store(u.s.k);
    }
    __syncthreads();
    if (w.hv % (args.Hv / args.Hk) == 0)
        store_transposed<E, DKP, kPieceThreads / 64>(u.s.q, args.queries_t + w.key_at * keys_bytes<E>(DKP));
    scores_of<DKP>(u.s.q, u.s.k, y, args.scale, p);
    for (int v0 = 0; v0 < args.cols; v0 += NV) {
        __syncthreads();
        go_next.store(u.go);
        __syncthreads();
        if (v0 + NV < args.cols) request(v0 + NV);
        f32x4 acc = zero4();
        for (int s = band * 16 / 32 * 32; s < kChunk; s += 32) acc = mma(p.cols(band * 16, s), u.go.cols(half * 16, s), acc);
        *reinterpret_cast<f32x4*>(args.inner + (w.at * args.cols + v0 + half * 16 + lc) * kChunk + lr) = acc;
    }
}

// ---- the state, backwards -----------------------------------------------------------------------

template <typename E, int DKP>
struct StateGradOperands {
    using M = Mode<E>;
    typename M::InputFrag k[DKP / 32], kt[DKP / 64][2], qt[DKP / 64][2];
    typename M::FineFrag inverse[2];   // transposed
    f32x4 a, d, beta, inner;
    float a_last;
    ColumnAhead<E> go;
    __device__ __forceinline__ void load_keys(const DeltaArgs& args, const DeltaWhere& w) {
#pragma unroll
        for (int s = 0; s < DKP / 32; ++s)
            k[s] = load_frag<typename M::InputFrag>(args.keys + w.key_at * keys_bytes<E>(DKP), (threadIdx.x >> 6) * (DKP / 32) + s);
    }
    __device__ __forceinline__ void load_inverse(const DeltaArgs& args, const DeltaWhere& w) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
            inverse[s] = load_frag<typename M::FineFrag>(args.inverse_t + w.at * square_bytes<E>(), (threadIdx.x >> 6) * 2 + s);
    }
    __device__ __forceinline__ void load_transposed(typename M::InputFrag (&x)[DKP / 64][2], const char* matrix, const DeltaWhere& w) {
#pragma unroll
        for (int i = 0; i < DKP / 64; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s)
                x[i][s] = load_frag<typename M::InputFrag>(matrix + w.key_at * keys_bytes<E>(DKP), ((threadIdx.x >> 6) + 4 * i) * 2 + s);
    }
    __device__ __forceinline__ void load_factors(const DeltaArgs& args, const DeltaWhere& w, int row, int col) {
        const Decay* y = args.decay + w.at;
        a = *reinterpret_cast<const f32x4*>(y->a + row);
        d = *reinterpret_cast<const f32x4*>(y->d + row);
        beta = *reinterpret_cast<const f32x4*>(y->beta + row);
        a_last = y->a[kChunk - 1];
        inner = *reinterpret_cast<const f32x4*>(args.inner + (w.at * args.cols + col) * kChunk + row);
        go.load(args.grad_o, w, w.hv, row, col, args.Dv);
    }
};

template <typename E, int DKP>
__global__ void __launch_bounds__(kStateThreads) delta_state_grad_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kStateCols;
    __shared__ typename M::template Fine<NV, DKP> state;       // gradient of the state, transposed
    __shared__ typename M::template Fine<NV, kChunk> r, x, go; // dR, -beta a dX, scale a dO, transposed
    const int tiles = args.cols / NV;
    const int piece = piece_in_l2(args.B * args.Hv * tiles), head = piece / tiles, v0 = (piece - head * tiles) * NV;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lc = lane & 15, row = wave * 16 + (lane >> 4) * 4, col = v0 + lc;
    const int length = delta_length(args, head / args.Hv), chunks = (length + kChunk - 1) / kChunk;

    StateGradOperands<E, DKP> now;
    if (chunks > 0) {
        const DeltaWhere w = delta_where(args, head, chunks - 1, length);
        now.load_factors(args, w, row, col);
        now.load_keys(args, w);
        now.load_inverse(args, w);
        now.load_transposed(now.qt, args.queries_t, w);
        now.load_transposed(now.kt, args.keys_t, w);
    }
    StateTiles<DKP> s;
    s.load(args.grad_state, head, args.Dk, args.Dv, col);
    s.put(state);
    for (int chunk = chunks - 1; chunk >= 0; --chunk) {
        const DeltaWhere w = delta_where(args, head, chunk > 0 ? chunk - 1 : 0, length);   // the next one
        const int64_t at = static_cast<int64_t>(head) * args.chunks + chunk;
        float out[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = args.scale * now.a[e] * now.go.get(e);
        go.put(lc, row, out);   // its readers of the chunk before are behind a barrier
        __syncthreads();
        f32x4 acc[2] = {zero4(), zero4()};
        typename M::FineFrag f[DKP / 32];
#pragma unroll
        for (int c = 0; c < DKP / 32; ++c) f[c] = state.rows(0, c * 32);
#pragma unroll
        for (int c = 0; c < DKP / 32; ++c) acc[c % 2] = mma(now.k[c], f[c], acc[c % 2]);
        __builtin_amdgcn_sched_barrier(0);
        now.load_keys(args, w);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = now.inner[e] + now.d[e] * (acc[0][e] + acc[1][e]);
        r.put(lc, row, out);
        s.keep(args.state_grads + at * DKP * args.cols, col);
        __syncthreads();
        f[0] = r.rows(0, 0);
        f[1] = r.rows(0, 32);
        acc[1] = mma(now.inverse[1], f[1], zero4());
        if (wave < 2) {   // columns from 32 on have nothing above row 32
            acc[0] = mma(now.inverse[0], f[0], zero4());
            acc[1] += acc[0];
        }
        __builtin_amdgcn_sched_barrier(0);
        now.load_inverse(args, w);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = -now.beta[e] * now.a[e] * acc[1][e];
        x.put(lc, row, out);
        store_later(args.inner + (at * args.cols + col) * kChunk + row, acc[1]);
        f[0] = go.rows(0, 0);   // does not wait for dX
        f[1] = go.rows(0, 32);
        f32x4 next_s[s.n];
#pragma unroll
        for (int i = 0; i < s.n; ++i) next_s[i] = now.a_last * s.s[i];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < s.n; ++i) next_s[i] = mma(now.qt[i][c], f[c], next_s[i]);
        __builtin_amdgcn_sched_barrier(0);
        now.load_transposed(now.qt, args.queries_t, w);
        now.load_factors(args, w, row, col);
        __syncthreads();
        f[0] = x.rows(0, 0);
        f[1] = x.rows(0, 32);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < s.n; ++i) next_s[i] = mma(now.kt[i][c], f[c], next_s[i]);
        __builtin_amdgcn_sched_barrier(0);
        now.load_transposed(now.kt, args.keys_t, w);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < s.n; ++i) s.s[i] = next_s[i];
        s.put(state);
    }
    s.save(args.grad_initial, head, args.Dk, args.Dv, col);
}

// ---- backward: the gradients of the inputs ------------------------------------------------------
//
// One workgroup per chunk and head takes 32 columns of the values at a time; dA, dP and the three Y stay in
// accumulators over them.  Reads everything that the passes left (states, their gradients, R, dX: 2 to 4 times the
// inputs' bytes); the tiles of a step are requested during the products of the one before.

__device__ __forceinline__ float row_sum16(float v) {  // over the 16 lanes that share rows
    v += __shfl_xor(v, 1);
    v += __shfl_xor(v, 2);
    v += __shfl_xor(v, 4);
    v += __shfl_xor(v, 8);
    return v;
}

// QO: type of grad_q and grad_k (the storage type, or float partial gradients where value heads share a key head).
template <typename E, bool WIDE, typename QO, int DKP>
__global__ void __launch_bounds__(kPieceThreads) delta_input_grad_kernel(DeltaArgs args) {
    using M = Mode<E>;
    constexpr int NV = kCols, KT = DKP / 32;   // tiles of 16 key columns per wavefront
    struct Columns {
        typename M::template Fine<NV, kChunk> x, r;   // transposed, like s and ds
        typename M::template Input<kChunk, NV> go, v;
        typename M::template Fine<NV, DKP> s, ds;
    };
    struct Squares {
        typename M::template Fine<kChunk, kChunk> m, n;   // transposed
    };
    union Shared {   // the columns are done with when M and N come
        Columns c;
        Squares w;
        __device__ Shared() {}
    };
    __shared__ typename M::template Input<kChunk, DKP> q_rows, k_rows;
    __shared__ Shared u;
    __shared__ Decay y;
    // sums of a row from both halves of the workgroup, of a column from every band
    __shared__ float row_beta[2][kChunk], row_c[2][kChunk], row_e[2][kChunk], col_c[4][kChunk], dot_v[kChunk], inner[8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, band = wave & 3, half = wave >> 2;
    const int lr = band * 16 + (lane >> 4) * 4, lc = lane & 15;
    // rows of the dense outputs: (t, b, head) of Hv heads; grad_q / grad_k per value head or, unshared, per key head
    const int64_t row_step = static_cast<int64_t>(args.B) * args.Hv;

    MatrixAhead<NV, kChunk, kPieceThreads> x_next, r_next;
    MatrixAhead<NV, DKP, kPieceThreads> s_next, ds_next;
    Ahead<WIDE, E, kChunk, NV, kPieceThreads> go_next, v_next;
    DecayAhead y_next;
    const auto request = [&](const DeltaWhere& w, int v0) {
        x_next.load(args.inner + (w.at * args.cols + v0) * kChunk);
        r_next.load(args.added + (w.at * args.cols + v0) * kChunk);
        go_next.load(row_of<E>(args.grad_o, w, w.hv) + v0, args.grad_o.t, w.rows, args.Dv - v0);
        v_next.load(row_of<E>(args.v, w, w.hv) + v0, args.v.t, w.rows, args.Dv - v0);
        s_next.load(args.states + (w.at * args.cols + v0) * DKP);
        ds_next.load(args.state_grads + (w.at * args.cols + v0) * DKP);
    };
    const DeltaWhere w = delta_where(args, blockIdx.y, blockIdx.x);
    const int present = args.T - w.t0 < kChunk ? args.T - w.t0 : kChunk;
    const int64_t row0 = static_cast<int64_t>(w.t0) * args.B * args.Hv + w.head;
    E* gv = static_cast<E*>(args.grad_v) + row0 * args.Dv;
    QO* gq = static_cast<QO*>(args.grad_q) + row0 * args.Dk;
    QO* gk = static_cast<QO*>(args.grad_k) + row0 * args.Dk;
    if (w.rows == 0) {
        for (int i = threadIdx.x; i < present * args.Dv; i += kPieceThreads)
            gv[i / args.Dv * row_step * args.Dv + i % args.Dv] = narrow<E>(0.f);
        for (int i = threadIdx.x; i < present * args.Dk; i += kPieceThreads) {
            gq[i / args.Dk * row_step * args.Dk + i % args.Dk] = narrow<QO>(0.f);
            gk[i / args.Dk * row_step * args.Dk + i % args.Dk] = narrow<QO>(0.f);
        }
        for (int i = threadIdx.x; i < present; i += kPieceThreads) {
            args.grad_g[row0 + i * row_step] = 0.f;
            args.grad_beta[row0 + i * row_step] = 0.f;
        }
        return;
    }
    {
        Ahead<WIDE, E, kChunk, DKP, kPieceThreads> q_next, k_next;
        q_next.load(row_of<E>(args.q, w, w.hk), args.q.t, w.rows, args.Dk);
        k_next.load(row_of<E>(args.k, w, w.hk), args.k.t, w.rows, args.Dk);
        y_next.load(args, w.at);
        request(w, 0);
        q_next.store(q_rows);
        k_next.store(k_rows);
        y_next.store(y);
    }

    f32x4 y1[KT], y2[KT], y3[KT], da[2], dp[2], v_dx = zero4();
#pragma unroll
    for (int i = 0; i < KT; ++i) y1[i] = y2[i] = y3[i] = zero4();
#pragma unroll
    for (int i = 0; i < 2; ++i) da[i] = dp[i] = zero4();
    float s_dot = 0.f;
    for (int v0 = 0; v0 < args.cols; v0 += NV) {
        __syncthreads();
        x_next.store(u.c.x);
        r_next.store(u.c.r);
        go_next.store(u.c.go);
        v_next.store(u.c.v);
        s_next.store(u.c.s);
        ds_next.store(u.c.ds);
#pragma unroll
        for (int i = 0; i < s_next.n; ++i) {
            float a[8], b[8];
            values_of(s_next.x[i], a);
            values_of(ds_next.x[i], b);
            if (s_next.mine(i)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) s_dot += a[j] * b[j];
            }
        }
        __syncthreads();
        if (v0 + NV < args.cols) request(w, v0 + NV);
        {   // dV: 16 rows times 16 columns per wavefront, four columns of a row per lane
            const f32x4 dx = u.c.x.block(half * 16, band * 16);
            const int i = band * 16 + lc, at = v0 + half * 16 + (lane >> 4) * 4;
            const float beta = y.beta[i];
            Vec<E, 4 * sizeof(E)> out;
#pragma unroll
            for (int j = 0; j < 4; ++j) out.e[j] = narrow<E>(i < w.rows ? beta * dx[j] : 0.f);
            if (i < present && at < args.Dv) {
                E* p = gv + i * row_step * args.Dv + at;
                if (at + 4 <= args.Dv) {
                    store_vec<E, 4 * sizeof(E)>(p, out);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (at + j < args.Dv) p[j] = out.e[j];
                }
            }
        }
        const auto fx = u.c.x.cols(band * 16, 0);
        const auto fg = u.c.go.rows(band * 16, 0);
        const auto fr = u.c.r.cols(band * 16, 0);
        if (half == 0) v_dx = mma(u.c.v.rows(band * 16, 0), fx, v_dx);   // v . dX is its diagonal
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            const auto fs = u.c.s.cols((half * KT + i) * 16, 0);
            y1[i] = mma(fx, fs, y1[i]);
            y2[i] = mma(fg, fs, y2[i]);
            y3[i] = mma(fr, u.c.ds.cols((half * KT + i) * 16, 0), y3[i]);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
            if (b * 2 + half <= band) {
                const auto f = u.c.r.cols((b * 2 + half) * 16, 0);
                da[b] = mma(fx, f, da[b]);
                dp[b] = mma(fg, f, dp[b]);
            }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s_dot += __shfl_xor(s_dot, d);   // <S, dS'>
    if (lane == 0) inner[wave] = s_dot;
    if (half == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if ((lane >> 4) * 4 + e == lc) dot_v[lr + e] = v_dx[e];
    }
    __syncthreads();
    // M, N and the sums over their products with A and P
    f32x4 sum_beta = zero4(), sum_c = zero4();
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int block = b * 2 + half, j = block * 16 + lc;
        f32x4 kk = zero4(), qk = zero4();
        if (block <= band) {
#pragma unroll
            for (int s = 0; s < DKP; s += 32) {
                const auto f = k_rows.rows(block * 16, s);
                kk = mma(k_rows.rows(band * 16, s), f, kk);
                qk = mma(q_rows.rows(band * 16, s), f, qk);
            }
        }
        float col = 0.f, m4[4], n4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = lr + e;
            const float decay = i >= j ? gap(y, i, j) : 0.f;
            const float a_grad = i > j ? -da[b][e] * decay : 0.f;
            n4[e] = i >= j ? dp[b][e] * decay * args.scale : 0.f;
            m4[e] = a_grad * y.beta[i];
            const float both = m4[e] * kk[e] + n4[e] * qk[e];
            sum_beta[e] += a_grad * kk[e];
            sum_c[e] += both;
            col += both;
        }
        u.w.m.put(j, lr, m4);
        u.w.n.put(j, lr, n4);
        col += __shfl_xor(col, 16);
        col += __shfl_xor(col, 32);
        if (lane < 16) col_c[band][j] = col;
    }
    // k . Y1, q . Y2, k . Y3 by row
    f32x4 d1 = zero4(), d2 = zero4(), d3 = zero4();
#pragma unroll
    for (int i = 0; i < KT; ++i) {
        const f32x4 kv = k_rows.block(band * 16, (half * KT + i) * 16), qv = q_rows.block(band * 16, (half * KT + i) * 16);
        d1 += kv * y1[i];
        d2 += qv * y2[i];
        d3 += kv * y3[i];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float a = y.a[lr + e], beta = y.beta[lr + e];
        const float rest = row_sum16(sum_c[e] - beta * a * d1[e] + args.scale * a * d2[e]);
        const float e_row = y.d[lr + e] * row_sum16(d3[e]);
        const float b_row = row_sum16(sum_beta[e] - a * d1[e]);
        if (lc == 0) {
            row_c[half][lr + e] = rest - e_row;
            row_e[half][lr + e] = e_row;
            row_beta[half][lr + e] = b_row;
        }
    }
    __syncthreads();
    if (wave == 0) {
        const int i = lane;
        const bool here = i < w.rows;
        double e_sum = here ? static_cast<double>(row_e[0][i]) + row_e[1][i] : 0.0;
        double dc = static_cast<double>(row_c[0][i]) + row_c[1][i];
#pragma unroll
        for (int o = 0; o < 4; ++o) dc -= col_c[o][i];
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) e_sum += __shfl_xor(e_sum, d);
        if (i == 63) {
            double dot = 0.0;
#pragma unroll
            for (int o = 0; o < 8; ++o) dot += inner[o];
            dc += e_sum + static_cast<double>(y.a[kChunk - 1]) * dot;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {   // sums from the row to the end
            const double other = __shfl_down(dc, d);
            if (i + d < 64) dc += other;
        }
        if (i < present) {
            args.grad_g[row0 + i * row_step] = here ? static_cast<float>(dc) : 0.f;
            args.grad_beta[row0 + i * row_step] = here ? row_beta[0][i] + row_beta[1][i] + dot_v[i] : 0.f;
        }
    }
    f32x4 a4, ad, ab;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a4[e] = args.scale * y.a[lr + e];
        ad[e] = y.d[lr + e];
        ab[e] = y.beta[lr + e] * y.a[lr + e];
    }
#pragma unroll
    for (int i = 0; i < KT; ++i) {   // from here y2 is dQ and y1 dK
        y2[i] = a4 * y2[i];
        y1[i] = ad * y3[i] - ab * y1[i];
    }
#pragma unroll
    for (int s = 0; s < kChunk; s += 32) {
        const bool left = s <= band * 16, below = s + 32 > band * 16;   // rows of the band end at the diagonal
        if (left) {
            const auto fn = u.w.n.cols(band * 16, s), fm = u.w.m.cols(band * 16, s);
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                const auto fk = k_rows.cols((half * KT + i) * 16, s);
                y2[i] = mma(fn, fk, y2[i]);
                y1[i] = mma(fm, fk, y1[i]);
            }
        }
        if (below) {
            const auto fn = u.w.n.rows(band * 16, s), fm = u.w.m.rows(band * 16, s);
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                y1[i] = mma(fm, k_rows.cols((half * KT + i) * 16, s), y1[i]);
                y1[i] = mma(fn, q_rows.cols((half * KT + i) * 16, s), y1[i]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (lr + e >= present) continue;
        QO *pq = gq + (lr + e) * row_step * args.Dk + half * KT * 16 + lc, *pk = gk + (lr + e) * row_step * args.Dk + half * KT * 16 + lc;
        const bool here = lr + e < w.rows;
#pragma unroll
        for (int i = 0; i < KT; ++i)
            if ((half * KT + i) * 16 + lc < args.Dk) {
                pq[i * 16] = narrow<QO>(here ? y2[i][e] : 0.f);
                pk[i * 16] = narrow<QO>(here ? y1[i][e] : 0.f);
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

template <typename E, bool WIDE, int DKP>
hipError_t delta_forward_as(const DeltaArgs& a, hipStream_t st) {
    const dim3 pieces(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.B * a.Hv));
    const dim3 columns(static_cast<unsigned>(a.cols / kStateCols * a.B * a.Hv));
    hipError_t err = hipSuccess;
    if (a.scores != nullptr) {
        if (a.chunks > 0) err = launch(delta_inverse_kernel<E, WIDE, DKP, true>, pieces, dim3(256), st, a);
        if (err == hipSuccess) err = launch(delta_state_kernel<E, DKP, true>, columns, dim3(kStateThreads), st, a);
        return err;
    }
    if (a.chunks > 0) err = launch(delta_inverse_kernel<E, WIDE, DKP, false>, pieces, dim3(256), st, a);
    if (err == hipSuccess) err = launch(delta_state_kernel<E, DKP, false>, columns, dim3(kStateThreads), st, a);
    if (err == hipSuccess && a.chunks > 0) err = launch(delta_output_kernel<E, WIDE, DKP>, pieces, dim3(kPieceThreads), st, a);
    return err;
}

// grad_q, grad_k: where the gradients go in the end (a.grad_q and a.grad_k are partial ones where heads share keys)
template <typename E, bool WIDE, int DKP>
hipError_t delta_backward_as(const DeltaArgs& a, void* grad_q, void* grad_k, hipStream_t st) {
    const dim3 pieces(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.B * a.Hv));
    const dim3 columns(static_cast<unsigned>(a.cols / kStateCols * a.B * a.Hv));
    hipError_t err = hipSuccess;
    if (a.chunks > 0) err = launch(delta_inner_grad_kernel<E, WIDE, DKP>, pieces, dim3(kPieceThreads), st, a);
    if (err == hipSuccess) err = launch(delta_state_grad_kernel<E, DKP>, columns, dim3(kStateThreads), st, a);
    if (err != hipSuccess || a.chunks == 0) return err;
    if (a.Hv == a.Hk) return launch(delta_input_grad_kernel<E, WIDE, E, DKP>, pieces, dim3(kPieceThreads), st, a);
    err = launch(delta_input_grad_kernel<E, WIDE, float, DKP>, pieces, dim3(kPieceThreads), st, a);
    if (err != hipSuccess) return err;
    const int64_t rows = static_cast<int64_t>(a.T) * a.B * a.Hk;
    const int64_t blocks = ceil_div(rows * a.Dk, 256);
    return launch(delta_shared_grad_kernel<E>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096), 2), dim3(256),
                  st, static_cast<const float*>(a.grad_q), static_cast<const float*>(a.grad_k), static_cast<E*>(grad_q),
                  static_cast<E*>(grad_k), rows, a.Dk, a.Hv / a.Hk);
}

// Keys of up to 64 values and of up to 128; rows of a multiple of eight values, and any others.
#define SNNSEQ_DEFINE_DELTA(NAME, E)                                                                           \
    hipError_t delta_forward_##NAME(const DeltaArgs& a, hipStream_t st) {                                      \
        const bool wide = a.q.wide && a.k.wide;                                                                \
        if (a.Dk <= 64)                                                                                        \
            return wide ? delta_forward_as<E, true, 64>(a, st) : delta_forward_as<E, false, 64>(a, st);        \
        return wide ? delta_forward_as<E, true, 128>(a, st) : delta_forward_as<E, false, 128>(a, st);          \
    }                                                                                                          \
    hipError_t delta_backward_##NAME(const DeltaArgs& a, void* grad_q, void* grad_k, hipStream_t st) {         \
        const bool wide = a.q.wide && a.k.wide && a.v.wide && a.grad_o.wide;                                   \
        if (a.Dk <= 64)                                                                                        \
            return wide ? delta_backward_as<E, true, 64>(a, grad_q, grad_k, st)                                \
                        : delta_backward_as<E, false, 64>(a, grad_q, grad_k, st);                              \
        return wide ? delta_backward_as<E, true, 128>(a, grad_q, grad_k, st)                                   \
                    : delta_backward_as<E, false, 128>(a, grad_q, grad_k, st);                                 \
    }

}  // namespace snnseq

#endif  // SNNLIF_SEQ_DELTA_H
