// Group norm with an activation, channels last: x [S, P, C], C = G groups of cpg consecutive channels, statistics
// per (sample, group) over the P * cpg values of the group.
//
//   forward    xhat = (x - mean) * rstd,  z = xhat * w + b,  y = act(z)
//   backward   gz = grad_y * act'(z);  per channel  B = sum gz,  A = sum gz * xhat;  per group, n = P * cpg
//              c1 = sum_c w B / n,  c2 = sum_c w A / n;   grad_x = rstd * (gz * w - c1 - xhat * c2)
//
// Bound by memory: 2 passes over the activation forward (read x, write y), 3 backward (read x and grad_y, write
// grad_x).  Three layouts reach or approach that:
//   rows   P == 1 and a group of at most 4 vectors per lane: a group is one run of memory.  L lanes (a power of two)
//          own it, hold it in registers and reduce by shuffles.  In the backward a lane keeps its channels over many
//          samples, so the channel sums stay in registers.  [16384, 8 groups of 128] bf16 silu: forward 21 us (67 MB:
//          3.2 TB/s), backward 32 us (101 MB: 3.2 TB/s); without an activation 18 and 28 us.  Bound by arithmetic: vector
//          instructions are under way 85 % and 78 % of the time (77 % and 69 % without the activation).
//   slab   the P rows of a bundle of groups fit the registers of a workgroup: read once, reduced through LDS, written
//          once.  A bundle is as many groups as make a row segment of 128 bytes, a memory line (64 where 128 do not fit).
//          [8 64 32 32 128] fp32: forward 97 us (537 MB: 5.5 TB/s), backward 219 us (805 MB: 3.7 TB/s; 1024 threads with
//          all their registers, one workgroup per CU, so that a sample's loads overlap only with the sums before).
//   split  larger: partial sums over slices of the positions, a small kernel that combines them, and a second read
//          of the inputs in the pass that writes.  [32 samples of 4096 positions, 8 groups of 32] silu: fp32 forward 100 us
//          (403 MB), backward 159 us (671 MB); bf16 55 and 85 us.  The backward of [8 64 32 32 128] in 32 groups bf16, whose
//          sums do not fit the slab's registers, takes 160 us here (671 MB: 4.2 TB/s); its slab forward 78 us.
// Statistics and sums are held in 32 bits (64 for double storage, and in the split layout's statistics); the variance is taken
// around the mean, in a second sweep over the registers, or around one of the group's values in 64 bits (split).
// Every sum has a fixed order.  Groups of any size, wherever they lie, are covered by vectors of 16 bytes (Spot): [7455,
// 32 groups of 111] fp32 takes 134 us forward and backward, 235 with single values.
#include "seq_common.h"

namespace snnseq {
namespace {

// Two instructions, off by a unit in the last place and |v| * 2^-24: that of v's own rounding.  The library's exponential
// takes four times as many, and instructions are what the norm of bf16 tokens is bound by.
__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896341f); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float erf_of(float v) { return erff(v); }
__device__ __forceinline__ double erf_of(double v) { return erf(v); }
__device__ __forceinline__ float inverse(float v) { return __builtin_amdgcn_rcpf(v); }  // 1 ulp
__device__ __forceinline__ double inverse(double v) { return 1.0 / v; }
__device__ __forceinline__ float inverse_root(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return 1.0 / sqrt(v); }

template <typename A>
__device__ __forceinline__ A act_value(A z, int act) {
    switch (act) {
        case SNNSEQ_ACT_RELU: return z < A(0) ? A(0) : z;  // NaN stays
        case SNNSEQ_ACT_SILU: return z * inverse(A(1) + exp_of(-z));
        case SNNSEQ_ACT_GELU: return A(0.5) * z * (A(1) + erf_of(z * A(0.70710678118654752440)));
        default: return z;
    }
}

template <typename A>
__device__ __forceinline__ A act_slope(A z, int act) {
    switch (act) {
        case SNNSEQ_ACT_RELU: return z > A(0) ? A(1) : A(0);
        case SNNSEQ_ACT_SILU: {
            const A s = inverse(A(1) + exp_of(-z));
            // z * (1 - s) is inf * 0 where exp overflows; the slope there is 0
            return s == A(0) ? A(0) : s * (A(1) + z * (A(1) - s));
        }
        case SNNSEQ_ACT_GELU:
            return A(0.5) * (A(1) + erf_of(z * A(0.70710678118654752440))) +
                   z * A(0.39894228040143267794) * exp_of(A(-0.5) * z * z);
        default: return A(1);
    }
}

// Sum over `lanes` (a power of two) neighbouring lanes, left in all of them.
template <typename A>
__device__ __forceinline__ A lanes_sum(A v, int lanes) {
    for (int d = 1; d < lanes; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// The product rounds by itself, as it did in c1's sum: in a group of one value they are equal, and the gradient is 0.
template <typename A>
__device__ __forceinline__ A input_grad(A gz, A w, A c1, A xhat, A c2, A rstd) {
    A h;
    {
#pragma clang fp contract(off)
        h = gz * w;
    }
    return rstd * (h - c1 - xhat * c2);
}

// The `index`-th vector of a group of cpg channels: its first channel within the group, and how many of its values the
// vector before has too.  Those are computed and stored by both, and counted in sums by the one before.
// RAGGED: cpg is no multiple of the vector; otherwise `skip` is 0 and costs nothing.
template <int n, bool RAGGED>
struct Spot {
    int first, skip;
    __device__ __forceinline__ Spot(int index, int cpg) {
        const int c = index * n;
        first = RAGGED && c > cpg - n ? cpg - n : c;
        skip = c - first;
    }
    template <typename A>
    __device__ __forceinline__ A counted(int j, A value) const { return RAGGED && j < skip ? A(0) : value; }
    __device__ __forceinline__ bool counts(int j) const { return !RAGGED || j >= skip; }
};

// ---- rows ---------------------------------------------------------------------------------------

constexpr int kRowsBlock = 256;

// U items (sample, group), `step` apart, per group of L lanes: all of them requested before the first is looked at.
// `step` is a multiple of G, so that they share their channels' weights.
template <typename E, int BYTES, bool RAGGED, int K, int U>
__global__ void __launch_bounds__(kRowsBlock)
gn_rows_forward_kernel(const E* __restrict__ x, const E* __restrict__ weight, const E* __restrict__ bias,
                       E* __restrict__ y, arith_t<E>* __restrict__ mean, arith_t<E>* __restrict__ rstd, int64_t items,
                       int64_t step, int G, int cpg, arith_t<E> eps, int act, int lanes_log2) {
    using A = arith_t<E>;
    constexpr int n = Vec<E, BYTES>::n;
    const int L = 1 << lanes_log2;
    const int lane = threadIdx.x & (L - 1);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kRowsBlock >> lanes_log2) + (threadIdx.x >> lanes_log2);
    if (first >= step) return;  // whole groups of lanes
    const int g = static_cast<int>(first % G);
    Vec<E, BYTES> v[U][K], w[K], b[K];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t item = first + u * step;
            v[u][k] = load_or_zero<E, BYTES>(x, item * cpg + Spot<n, RAGGED>(k * L + lane, cpg).first,
                                             (k * L + lane) * n < cpg && item < items, true);
        }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = Spot<n, RAGGED>(k * L + lane, cpg).first;
        w[k] = load_or_zero<E, BYTES>(weight, g * cpg + c, (k * L + lane) * n < cpg, false);
        b[k] = load_or_zero<E, BYTES>(bias, g * cpg + c, (k * L + lane) * n < cpg, false);
    }
    const A per = A(1) / A(cpg);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t item = first + u * step;
        if (item >= items) return;
        A sum = A(0);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Spot<n, RAGGED> spot(k * L + lane, cpg);
#pragma unroll
            for (int j = 0; j < n; ++j) sum += spot.counted(j, widen(v[u][k].e[j]));  // absent values are zero
        }
        const A m = lanes_sum(sum, L) * per;
        A sq = A(0);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if ((k * L + lane) * n < cpg) {
                const Spot<n, RAGGED> spot(k * L + lane, cpg);
#pragma unroll
                for (int j = 0; j < n; ++j) {
                    const A d = widen(v[u][k].e[j]) - m;
                    sq += spot.counted(j, d * d);
                }
            }
        const A r = inverse_root(lanes_sum(sq, L) * per + eps);
        if (lane == 0) {
            mean[item] = m;
            rstd[item] = r;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if ((k * L + lane) * n >= cpg) continue;
            Vec<E, BYTES> o;
#pragma unroll
            for (int j = 0; j < n; ++j)
                o.e[j] = narrow<E>(act_value((widen(v[u][k].e[j]) - m) * r * widen(w[k].e[j]) + widen(b[k].e[j]), act));
            store_vec<E, BYTES>(y + item * cpg + Spot<n, RAGGED>(k * L + lane, cpg).first, o);
        }
    }
}

// Groups of L lanes: `gpb` groups of channels (blockIdx.y names which) times `spb` samples at a time; blockIdx.x is
// the sample slice.  part [slices][2][C]: sums of gz * xhat, then of gz.
template <typename E, int BYTES, bool RAGGED, int K>
__global__ void __launch_bounds__(kRowsBlock)
gn_rows_backward_kernel(const E* __restrict__ x, const E* __restrict__ weight, const E* __restrict__ bias,
                        const arith_t<E>* __restrict__ mean, const arith_t<E>* __restrict__ rstd,
                        const E* __restrict__ grad, E* __restrict__ grad_x, arith_t<E>* __restrict__ part, int64_t S,
                        int G, int cpg, int act, int lanes_log2, int gpb, int spb) {
    using A = arith_t<E>;
    constexpr int n = Vec<E, BYTES>::n;
    __shared__ A shared[kRowsBlock];
    const int L = 1 << lanes_log2;
    const int lane = threadIdx.x & (L - 1);
    const int sub = threadIdx.x >> lanes_log2;
    const int sample = sub / gpb;
    const int g = blockIdx.y * gpb + sub - sample * gpb;
    const bool here = sample < spb && g < G;
    A acc_a[K * n] = {}, acc_b[K * n] = {};
    if (here) {
        Vec<E, BYTES> w[K], b[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = Spot<n, RAGGED>(k * L + lane, cpg).first;
            w[k].raw = b[k].raw = typename Vec<E, BYTES>::raw_t(0);
            if ((k * L + lane) * n < cpg) {
                w[k] = load_vec<E, BYTES>(weight + g * cpg + c);
                b[k] = load_vec<E, BYTES>(bias + g * cpg + c);
            }
        }
        const int64_t hop = static_cast<int64_t>(gridDim.x) * spb;
        int64_t s = static_cast<int64_t>(blockIdx.x) * spb + sample;
        Vec<E, BYTES> v_next[K], d_next[K];
        A m_next = A(0), r_next = A(0);
        const auto request = [&](int64_t at) {   // the sample after this one is under way while this one is worked on
            const int64_t item = (at < S ? at : s) * G + g;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = Spot<n, RAGGED>(k * L + lane, cpg).first;
                v_next[k].raw = d_next[k].raw = typename Vec<E, BYTES>::raw_t(0);
                if ((k * L + lane) * n < cpg) {
                    v_next[k] = load_vec_once<E, BYTES>(x + item * cpg + c);
                    d_next[k] = load_vec_once<E, BYTES>(grad + item * cpg + c);
                }
            }
            m_next = mean[item];
            r_next = rstd[item];
        };
        if (s < S) request(s);
        for (; s < S; s += hop) {
            const int64_t item = s * G + g;
            Vec<E, BYTES> v[K], d[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                v[k] = v_next[k];
                d[k] = d_next[k];
            }
            const A m = m_next, r = r_next;
            request(s + hop);
            A gz[K * n], c1 = A(0), c2 = A(0);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Spot<n, RAGGED> spot(k * L + lane, cpg);
#pragma unroll
                for (int j = 0; j < n; ++j) {
                    const A xhat = (widen(v[k].e[j]) - m) * r;
                    const A t = widen(d[k].e[j]) * act_slope(xhat * widen(w[k].e[j]) + widen(b[k].e[j]), act);
                    gz[k * n + j] = t;  // zero where there is no channel
                    if ((k * L + lane) * n < cpg && spot.counts(j)) {
                        acc_a[k * n + j] += t * xhat;
                        acc_b[k * n + j] += t;
                        c1 += t * widen(w[k].e[j]);
                        c2 += t * widen(w[k].e[j]) * xhat;
                    }
                }
            }
            c1 = lanes_sum(c1, L) / A(cpg);
            c2 = lanes_sum(c2, L) / A(cpg);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if ((k * L + lane) * n >= cpg) continue;
                Vec<E, BYTES> o;
#pragma unroll
                for (int j = 0; j < n; ++j) {
                    const A xhat = (widen(v[k].e[j]) - m) * r;
                    o.e[j] = narrow<E>(input_grad(gz[k * n + j], widen(w[k].e[j]), c1, xhat, c2, r));
                }
                store_vec<E, BYTES>(grad_x + item * cpg + Spot<n, RAGGED>(k * L + lane, cpg).first, o);
            }
        }
    }
    // the spb samples that shared the workgroup, in order
    const int C = G * cpg;
    A* row = part + static_cast<int64_t>(blockIdx.x) * 2 * C;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < n; ++j)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                A v = which == 0 ? acc_a[k * n + j] : acc_b[k * n + j];
                if (spb > 1) {
                    __syncthreads();
                    shared[threadIdx.x] = v;
                    __syncthreads();
                    if (sample == 0)
                        for (int o = 1; o < spb; ++o) v += shared[threadIdx.x + o * gpb * L];
                }
                const Spot<n, RAGGED> spot(k * L + lane, cpg);
                if (here && sample == 0 && (k * L + lane) * n < cpg && spot.counts(j))
                    row[which * C + g * cpg + spot.first + j] = v;
            }
}

// grad_weight, grad_bias from `rows` partial rows [2][C]: 32 columns times 32 groups of rows per workgroup.
template <typename E>
__global__ void __launch_bounds__(1024)
gn_parameters_kernel(const arith_t<E>* __restrict__ part, E* __restrict__ grad_weight, E* __restrict__ grad_bias,
                     int64_t rows, int C) {
    using A = arith_t<E>;
    __shared__ A shared[1024];
    const int column = blockIdx.x * 32 + (threadIdx.x & 31), group = threadIdx.x >> 5;
    A acc = A(0);
    if (column < 2 * C) {
#pragma unroll 8
        for (int64_t r = group; r < rows; r += 32) acc += part[r * 2 * C + column];
    }
    shared[threadIdx.x] = acc;
    __syncthreads();
    if (group == 0 && column < 2 * C) {
        for (int o = 1; o < 32; ++o) acc += shared[threadIdx.x + 32 * o];
        (column < C ? grad_weight : grad_bias)[column < C ? column : column - C] = narrow<E>(acc);
    }
}

// ---- slab ---------------------------------------------------------------------------------------

// Values a thread holds of each input: 32 (64 registers of x and grad_y), half as many where a thread of a
// 1024-thread workgroup, limited to 128 registers, holds both inputs, and half as many doubles; in at most 16 vectors
// (8 there), each of which costs an address.
constexpr int held_vectors(int element_bytes, int vector_values, int block, bool backward) {
    const bool tight = backward && block == 1024;
    const int values = (element_bytes == 8 ? 16 : 32) / (tight ? 2 : 1), most = tight ? 8 : 16;
    const int k = values / vector_values;
    return k > most ? most : k;
}

// Workgroups go to the eight XCDs in turn, each with an L2 of its own: consecutive pieces of work are given to one
// XCD, so that the bundles of a sample, which share memory lines, meet in one L2.
__device__ __forceinline__ int64_t piece_of_work() {
    const unsigned per = gridDim.x / 8;
    return blockIdx.x < per * 8 ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
}

// sm[q][tid] (q < Q, rows of `cols` threads): adds the rows up; the sums are left in sm[q][0 .. cols).  Eight rows become
// one in a step.  All threads share the Q * kept * cols sums of a step, and the values of one are requested together:
// with Q sums one after another in the threads that keep a row, the backward of [205 samples, 220 positions, 9 groups
// of 43] bf16 took 171 us instead of 82.  The forward's single sum has too few to share and wants its registers.
template <typename A, int Q, int BT>
__device__ __forceinline__ void fold_rows(A (*sm)[BT], int rows, int cols, int tid) {
    __syncthreads();
    while (rows > 1) {
        const int kept = (rows + 7) >> 3, slots = kept * cols, end = rows * cols;
        if constexpr (Q == 1) {
            if (tid < slots) {
                A s = sm[0][tid];
                for (int r = tid + slots; r < end; r += slots) s += sm[0][r];
                sm[0][tid] = s;
            }
        } else {
            for (int i = tid; i < Q * slots; i += BT) {
                const int q = i / slots, slot = i - q * slots;
                A s = sm[q][slot], v[7];
#pragma unroll
                for (int r = 0; r < 7; ++r) {
                    const int at = slot + (r + 1) * slots;
                    v[r] = at < end ? sm[q][at] : A(0);
                }
#pragma unroll
                for (int r = 0; r < 7; ++r) s += v[r];
                sm[q][slot] = s;
            }
        }
        rows = kept;
        __syncthreads();
    }
}

// Sum over the columns of this thread's group.
template <typename A>
__device__ __forceinline__ A group_sum(const A* column_sums, int first, int count) {
    A s = A(0);
    for (int i = 0; i < count; ++i) s += column_sums[first + i];
    return s;
}

struct Bundle {  // which columns and rows of the slab a thread holds
    int first_group, cols, rows, col, row, group;
    bool here;
};

template <int BT>
__device__ __forceinline__ Bundle bundle_of(int bundle, int gpb, int G, int vpg) {
    Bundle b;
    b.first_group = bundle * gpb;
    const int groups = G - b.first_group < gpb ? G - b.first_group : gpb;
    b.cols = groups * vpg;
    b.rows = BT / b.cols;
    b.row = threadIdx.x / b.cols;
    b.col = threadIdx.x - b.row * b.cols;
    b.here = b.row < b.rows;
    b.group = b.col / vpg;
    return b;
}

// Workgroup (sample, bundle of `gpb` groups); vpg = vectors per group and position.
template <typename E, int BYTES, bool RAGGED, int BT>
__global__ void __launch_bounds__(BT)
gn_slab_forward_kernel(const E* __restrict__ x, const E* __restrict__ weight, const E* __restrict__ bias,
                       E* __restrict__ y, arith_t<E>* __restrict__ mean, arith_t<E>* __restrict__ rstd, int bundles,
                       int P, int G, int cpg, int gpb, arith_t<E> eps, int act) {
    using A = arith_t<E>;
    constexpr int n = Vec<E, BYTES>::n, K = held_vectors(sizeof(E), n, BT, false);
    __shared__ A sm[1][BT];
    const int vpg = (cpg + n - 1) / n, C = G * cpg;
    const int64_t piece = piece_of_work();
    const int64_t s = piece / bundles;
    const Bundle t = bundle_of<BT>(static_cast<int>(piece - s * bundles), gpb, G, vpg);
    const Spot<n, RAGGED> spot(t.col - t.group * vpg, cpg);
    const int c = (t.first_group + t.group) * cpg + spot.first;
    const E* px = x + s * P * C;  // one sample is below 2 GiB: 32-bit offsets from here
    Vec<E, BYTES> v[K];
    A sum = A(0);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int p = t.row + k * t.rows;
        v[k] = load_or_zero<E, BYTES>(px, static_cast<uint32_t>(p * C + c), t.here && p < P, true);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < n; ++j) sum += spot.counted(j, widen(v[k].e[j]));
    sm[0][threadIdx.x] = sum;
    fold_rows<A, 1, BT>(sm, t.rows, t.cols, threadIdx.x);
    const A count = A(P) * A(cpg);
    const A m = group_sum(sm[0], t.group * vpg < t.cols ? t.group * vpg : 0, vpg) / count;
    __syncthreads();
    A sq = A(0);
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (t.here && t.row + k * t.rows < P) {
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const A d = widen(v[k].e[j]) - m;
                sq += spot.counted(j, d * d);
            }
        }
    sm[0][threadIdx.x] = sq;
    fold_rows<A, 1, BT>(sm, t.rows, t.cols, threadIdx.x);
    if (!t.here) return;
    const A r = inverse_root(group_sum(sm[0], t.group * vpg, vpg) / count + eps);
    if (t.row == 0 && t.col == t.group * vpg) {
        mean[s * G + t.first_group + t.group] = m;
        rstd[s * G + t.first_group + t.group] = r;
    }
    const Vec<E, BYTES> w = load_vec<E, BYTES>(weight + c), b = load_vec<E, BYTES>(bias + c);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int p = t.row + k * t.rows;
        if (p >= P) continue;
        Vec<E, BYTES> o;
#pragma unroll
        for (int j = 0; j < n; ++j)
            o.e[j] = narrow<E>(act_value((widen(v[k].e[j]) - m) * r * widen(w.e[j]) + widen(b.e[j]), act));
        store_vec<E, BYTES>(y + s * P * C + static_cast<uint32_t>(p * C + c), o);
    }
}

// Workgroup (slice of the samples, bundle): samples slice, slice + slices, ...; part [slices][2][C].
template <typename E, int BYTES, bool RAGGED, int BT>
__global__ void __launch_bounds__(BT)
gn_slab_backward_kernel(const E* __restrict__ x, const E* __restrict__ weight, const E* __restrict__ bias,
                        const arith_t<E>* __restrict__ mean, const arith_t<E>* __restrict__ rstd,
                        const E* __restrict__ grad, E* __restrict__ grad_x, arith_t<E>* __restrict__ part, int64_t S,
                        int bundles, int slices, int P, int G, int cpg, int gpb, int act) {
    using A = arith_t<E>;
    constexpr int n = Vec<E, BYTES>::n, K = held_vectors(sizeof(E), n, BT, true);
    __shared__ A sm[2 * n][BT];
    const int vpg = (cpg + n - 1) / n, C = G * cpg;
    const int64_t piece = piece_of_work();
    const int slice = static_cast<int>(piece / bundles);
    const Bundle t = bundle_of<BT>(static_cast<int>(piece - static_cast<int64_t>(slice) * bundles), gpb, G, vpg);
    const Spot<n, RAGGED> spot(t.col - t.group * vpg, cpg);
    const int c = (t.first_group + t.group) * cpg + spot.first;
    const int first_col = t.here ? t.group * vpg : 0;
    const A count = A(P) * A(cpg);
    Vec<E, BYTES> w, b;
    w.raw = b.raw = typename Vec<E, BYTES>::raw_t(0);
    if (t.here) {
        w = load_vec<E, BYTES>(weight + c);
        b = load_vec<E, BYTES>(bias + c);
    }
    A total_a[n] = {}, total_b[n] = {};
    Vec<E, BYTES> v[K], d[K];
    A m_next = A(0), r_next = A(0);
    // The one workgroup of 1024 threads that a CU holds requests a sample while the one before is summed up and stored
    // ([8 64 32 32 128] fp32, with the sums one after another: 267 us, 301 without); smaller ones overlap each other, and the registers are theirs.
    // What does not exist is read at the slab's beginning and left out below.
    // Narrow vectors (more addresses) and counting have no registers for it.
    constexpr bool kRequestAhead = BT == 1024 && sizeof(E) == 4 && BYTES == 16 && !RAGGED;
    const auto request = [&](int64_t s) {
        const E *px = x + s * P * C, *pg = grad + s * P * C;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int p = t.row + k * t.rows;
            const uint32_t at = t.here && p < P ? static_cast<uint32_t>(p * C + c) : 0u;
            v[k] = load_vec<E, BYTES>(px + at);
            d[k] = load_vec<E, BYTES>(pg + at);
        }
        const int64_t item = s * G + (t.here ? t.first_group + t.group : 0);
        m_next = mean[item];
        r_next = rstd[item];
    };
    if (kRequestAhead && slice < S) request(slice);
    for (int64_t s = slice; s < S; s += slices) {
        if (!kRequestAhead) request(s);
        const A m = m_next, r = r_next;
        // xhat and gz take the registers of x and grad_y: 64 at most, within the 128 of a 1024-thread workgroup
        A xh[K * n], gz[K * n], acc_a[n] = {}, acc_b[n] = {};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            __builtin_amdgcn_sched_barrier(0);  // one vector's activation at a time: no registers for the next one's
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const A xhat = (widen(v[k].e[j]) - m) * r;
                const A q = widen(d[k].e[j]) * act_slope(xhat * widen(w.e[j]) + widen(b.e[j]), act);
                const bool valid = t.here && t.row + k * t.rows < P && spot.counts(j);
                xh[k * n + j] = xhat;
                gz[k * n + j] = q;
                acc_a[j] += valid ? q * xhat : A(0);
                acc_b[j] += valid ? q : A(0);
            }
        }
        if (kRequestAhead) request(s + slices < S ? s + slices : s);
        __syncthreads();  // the sums of the sample before have been read
#pragma unroll
        for (int j = 0; j < n; ++j) {
            sm[j][threadIdx.x] = acc_a[j];
            sm[n + j][threadIdx.x] = acc_b[j];
        }
        fold_rows<A, 2 * n, BT>(sm, t.rows, t.cols, threadIdx.x);
        A pa = A(0), pb = A(0);
        if (static_cast<int>(threadIdx.x) < t.cols) {
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const A a = sm[j][threadIdx.x], bsum = sm[n + j][threadIdx.x];
                total_a[j] += a;
                total_b[j] += bsum;
                pa += widen(w.e[j]) * a;
                pb += widen(w.e[j]) * bsum;
            }
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < t.cols) {
            sm[0][threadIdx.x] = pa;
            sm[1][threadIdx.x] = pb;
        }
        __syncthreads();
        const A c2 = group_sum(sm[0], first_col, vpg) / count, c1 = group_sum(sm[1], first_col, vpg) / count;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int p = t.row + k * t.rows;
            if (!t.here || p >= P) continue;
            Vec<E, BYTES> o;
#pragma unroll
            for (int j = 0; j < n; ++j) {
                o.e[j] = narrow<E>(input_grad(gz[k * n + j], widen(w.e[j]), c1, xh[k * n + j], c2, r));
            }
            store_vec<E, BYTES>(grad_x + s * P * C + static_cast<uint32_t>(p * C + c), o);
        }
    }
    if (static_cast<int>(threadIdx.x) < t.cols) {
        A* row = part + static_cast<int64_t>(slice) * 2 * C;
#pragma unroll
        for (int j = 0; j < n; ++j) {
            if (!spot.counts(j)) continue;
            row[c + j] = total_a[j];
            row[C + c + j] = total_b[j];
        }
    }
}

// ---- split --------------------------------------------------------------------------------------

constexpr int kSplitBlock = 256;

// Columns (vectors) blockIdx.z * cols .., positions [slice * span, (slice + 1) * span), samples blockIdx.x.
struct Patch {
    int col, row, rows, begin, end;
    bool here;
};

__device__ __forceinline__ Patch patch_of(int cols, int columns, int span, int P) {
    Patch t;
    t.rows = kSplitBlock / cols;
    t.row = threadIdx.x / cols;
    t.col = blockIdx.z * cols + threadIdx.x - t.row * cols;
    t.begin = blockIdx.y * span;
    t.end = t.begin + span < P ? t.begin + span : P;
    t.here = t.row < t.rows && t.col < columns;
    return t;
}

// part [S][slices][2][columns]: sums of d and d * d, d = x - (the group's first value), in 64 bits.
template <typename E, int BYTES, bool RAGGED>
__global__ void __launch_bounds__(kSplitBlock)
gn_split_statistics_kernel(const E* __restrict__ x, double* __restrict__ part, int P, int C, int cpg, int cols,
                           int span) {
    constexpr int n = Vec<E, BYTES>::n;
    __shared__ double sm[2][kSplitBlock];
    const int vpg = (cpg + n - 1) / n, columns = C / cpg * vpg;
    const Patch t = patch_of(cols, columns, span, P);
    const int group = t.col / vpg;
    const Spot<n, RAGGED> spot(t.col - group * vpg, cpg);
    const int64_t s = blockIdx.x;
    const E* px = x + s * P * C;
    double sum = 0.0, sq = 0.0;
    if (t.here) {
        const double shift = static_cast<double>(widen(px[group * cpg]));
        constexpr int U = 4;
        for (int p0 = t.begin + t.row; p0 < t.end; p0 += U * t.rows) {
            Vec<E, BYTES> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = p0 + u * t.rows;
                v[u] = load_vec<E, BYTES>(px + static_cast<int64_t>(p < t.end ? p : p0) * C + group * cpg + spot.first);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (p0 + u * t.rows < t.end) {
#pragma unroll
                    for (int j = 0; j < n; ++j) {
                        const double d = spot.counted(j, static_cast<double>(widen(v[u].e[j])) - shift);
                        sum += d;
                        sq += d * d;
                    }
                }
        }
    }
    sm[0][threadIdx.x] = sum;
    sm[1][threadIdx.x] = sq;
    fold_rows<double, 2, kSplitBlock>(sm, t.rows, cols, threadIdx.x);
    if (static_cast<int>(threadIdx.x) < cols && t.here) {
        double* q = part + (s * gridDim.y + blockIdx.y) * 2 * columns;
        q[t.col] = sm[0][threadIdx.x];
        q[columns + t.col] = sm[1][threadIdx.x];
    }
}

// One wavefront per (sample, group).
template <typename E>
__global__ void __launch_bounds__(64)
gn_split_finish_kernel(const E* __restrict__ x, const double* __restrict__ part, arith_t<E>* __restrict__ mean,
                       arith_t<E>* __restrict__ rstd, int P, int C, int G, int columns, int slices, double eps) {
    const int64_t item = blockIdx.x;
    const int64_t s = item / G;
    const int g = static_cast<int>(item - s * G);
    const int vpg = columns / G, cpg = C / G;
    double sum = 0.0, sq = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < slices * vpg; i += 64) {
        const int slice = i / vpg, col = g * vpg + i - slice * vpg;
        const double* q = part + (s * slices + slice) * 2 * columns;
        sum += q[col];
        sq += q[columns + col];
    }
    sum = lanes_sum(sum, 64);
    sq = lanes_sum(sq, 64);
    if (threadIdx.x == 0) {
        const double n = static_cast<double>(P) * cpg;
        const double m = sum / n;
        double var = sq / n - m * m;
        var = var < 0.0 ? 0.0 : var;  // rounding only; a NaN stays
        mean[item] = static_cast<arith_t<E>>(static_cast<double>(widen(x[s * P * C + g * cpg])) + m);
        rstd[item] = static_cast<arith_t<E>>(1.0 / sqrt(var + eps));
    }
}

// coefficients == nullptr: y = act(z).  Otherwise grad_x, with coefficients [S][G][2] = (c1, c2).
template <typename E, int BYTES, bool RAGGED>
__global__ void __launch_bounds__(kSplitBlock)
gn_split_apply_kernel(const E* __restrict__ x, const E* __restrict__ weight, const E* __restrict__ bias,
                      const arith_t<E>* __restrict__ mean, const arith_t<E>* __restrict__ rstd,
                      const E* __restrict__ grad, const arith_t<E>* __restrict__ coefficients, E* __restrict__ out,
                      int P, int C, int G, int cols, int span, int act) {
    using A = arith_t<E>;
    constexpr int n = Vec<E, BYTES>::n;
    const int cpg = C / G, vpg = (cpg + n - 1) / n;
    const Patch t = patch_of(cols, G * vpg, span, P);
    if (!t.here) return;
    const int64_t s = blockIdx.x;
    const int g = t.col / vpg, c = g * cpg + Spot<n, RAGGED>(t.col - g * vpg, cpg).first;
    const int64_t base = s * P * C + c;
    const Vec<E, BYTES> w = load_vec<E, BYTES>(weight + c), b = load_vec<E, BYTES>(bias + c);
    const A m = mean[s * G + g], r = rstd[s * G + g];
    A c1 = A(0), c2 = A(0);
    if (coefficients != nullptr) {
        c1 = coefficients[(s * G + g) * 2];
        c2 = coefficients[(s * G + g) * 2 + 1];
    }
    constexpr int U = 4;
    for (int p0 = t.begin + t.row; p0 < t.end; p0 += U * t.rows) {
        Vec<E, BYTES> v[U], d[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + u * t.rows;
            const int64_t at = base + static_cast<int64_t>(p < t.end ? p : p0) * C;
            v[u] = load_vec_once<E, BYTES>(x + at);
            d[u].raw = typename Vec<E, BYTES>::raw_t(0);
            if (coefficients != nullptr) d[u] = load_vec_once<E, BYTES>(grad + at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + u * t.rows;
            if (p >= t.end) continue;
            Vec<E, BYTES> o;
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const A xhat = (widen(v[u].e[j]) - m) * r;
                const A z = xhat * widen(w.e[j]) + widen(b.e[j]);
                o.e[j] = narrow<E>(coefficients == nullptr
                                       ? act_value(z, act)
                                       : input_grad(widen(d[u].e[j]) * act_slope(z, act), widen(w.e[j]), c1, xhat, c2, r));
            }
            store_vec<E, BYTES>(out + base + static_cast<int64_t>(p) * C, o);
        }
    }
}

// part [S][slices][2][C]: sums of gz * xhat and of gz.
template <typename E, int BYTES, bool RAGGED>
__global__ void __launch_bounds__(kSplitBlock)
gn_split_sums_kernel(const E* __restrict__ x, const E* __restrict__ weight, const E* __restrict__ bias,
                     const arith_t<E>* __restrict__ mean, const arith_t<E>* __restrict__ rstd,
                     const E* __restrict__ grad, arith_t<E>* __restrict__ part, int P, int C, int G, int cols, int span,
                     int act) {
    using A = arith_t<E>;
    constexpr int n = Vec<E, BYTES>::n;
    __shared__ A sm[2 * n][kSplitBlock];
    const int cpg = C / G, vpg = (cpg + n - 1) / n;
    const Patch t = patch_of(cols, G * vpg, span, P);
    const int64_t s = blockIdx.x;
    const int g = t.col / vpg;
    const Spot<n, RAGGED> spot(t.col - g * vpg, cpg);
    const int c = g * cpg + spot.first;
    A acc_a[n] = {}, acc_b[n] = {};
    if (t.here) {
        const int64_t base = s * P * C + c;
        const Vec<E, BYTES> w = load_vec<E, BYTES>(weight + c), b = load_vec<E, BYTES>(bias + c);
        const A m = mean[s * G + g], r = rstd[s * G + g];
        constexpr int U = 4;
        for (int p0 = t.begin + t.row; p0 < t.end; p0 += U * t.rows) {
            Vec<E, BYTES> v[U], d[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = p0 + u * t.rows;
                const int64_t at = base + static_cast<int64_t>(p < t.end ? p : p0) * C;
                v[u] = load_vec<E, BYTES>(x + at);
                d[u] = load_vec<E, BYTES>(grad + at);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (p0 + u * t.rows < t.end) {
#pragma unroll
                    for (int j = 0; j < n; ++j) {
                        const A xhat = (widen(v[u].e[j]) - m) * r;
                        const A q = widen(d[u].e[j]) * act_slope(xhat * widen(w.e[j]) + widen(b.e[j]), act);
                        acc_a[j] += q * xhat;
                        acc_b[j] += q;
                    }
                }
        }
    }
#pragma unroll
    for (int j = 0; j < n; ++j) {
        sm[j][threadIdx.x] = acc_a[j];
        sm[n + j][threadIdx.x] = acc_b[j];
    }
    fold_rows<A, 2 * n, kSplitBlock>(sm, t.rows, cols, threadIdx.x);
    if (static_cast<int>(threadIdx.x) < cols && t.here) {
        A* q = part + (s * gridDim.y + blockIdx.y) * 2 * C;
#pragma unroll
        for (int j = 0; j < n; ++j) {
            if (!spot.counts(j)) continue;
            q[c + j] = sm[j][threadIdx.x];
            q[C + c + j] = sm[n + j][threadIdx.x];
        }
    }
}

// One wavefront per (sample, group): (c1, c2).
template <typename E>
__global__ void __launch_bounds__(64)
gn_split_coefficients_kernel(const arith_t<E>* __restrict__ part, const E* __restrict__ weight,
                             arith_t<E>* __restrict__ coefficients, int P, int C, int G, int slices) {
    using A = arith_t<E>;
    const int64_t item = blockIdx.x;
    const int64_t s = item / G;
    const int cpg = C / G, first = static_cast<int>(item - s * G) * cpg;
    A c1 = A(0), c2 = A(0);
#pragma unroll 8
    for (int i = threadIdx.x; i < slices * cpg; i += 64) {
        const int slice = i / cpg, c = first + i - slice * cpg;
        const A* q = part + (s * slices + slice) * 2 * C;
        c2 += widen(weight[c]) * q[c];
        c1 += widen(weight[c]) * q[C + c];
    }
    c1 = lanes_sum(c1, 64);
    c2 = lanes_sum(c2, 64);
    if (threadIdx.x == 0) {
        const A count = A(P) * A(cpg);
        coefficients[item * 2] = c1 / count;
        coefficients[item * 2 + 1] = c2 / count;
    }
}

// ---- host ---------------------------------------------------------------------------------------

enum class Way { rows, slab, split };

struct Plan {
    Way way;
    // rows
    int lanes_log2, vectors, gpb, spb, group_blocks;
    // slab
    int block, bundles;
    // split
    int cols, col_blocks, span, slices;
    int64_t part_rows;         // backward: partial rows [2][C] of the parameter gradients
    size_t part, coefficients, bytes;
};

// A vector never leaves its group.
Plan plan_of(int dtype, int64_t S, int64_t P, int64_t C, int64_t G, bool backward) {
    Plan p{};
    const int64_t es = static_cast<int64_t>(element_size(dtype));
    const size_t arith = dtype == SNNLIF_DTYPE_F64 ? 8 : 4;
    const int64_t cpg = C / G, n = widest_vector(cpg, es) / es, vpg = ceil_div(cpg, n);
    if (P == 1 && vpg <= 64 * 4) {
        p.way = Way::rows;
        while ((1 << p.lanes_log2) < vpg && p.lanes_log2 < 6) ++p.lanes_log2;
        const int64_t per_lane = ceil_div(vpg, int64_t(1) << p.lanes_log2);
        p.vectors = per_lane == 1 ? 1 : per_lane == 2 ? 2 : 4;
        const int64_t subs = kRowsBlock >> p.lanes_log2;
        p.gpb = static_cast<int>(G < subs ? G : subs);
        p.spb = static_cast<int>(subs / p.gpb);
        p.group_blocks = static_cast<int>(ceil_div(G, p.gpb));
        // four workgroups per CU, each over several samples: enough requests in flight, and few partial rows
        const int64_t wanted = ceil_div(1024, p.group_blocks), most = ceil_div(S, p.spb);
        p.part_rows = wanted < most ? wanted : most;
    } else {
        p.way = Way::split;
        // 1024 threads only where 256 cannot hold the slab: more workgroups per CU overlap loads with stores.  Segments
        // of 32 bytes, which 256 threads could hold, cost twice the time ([8 64 32 32 128] fp32: backward 475 us against 276, both with the sums one after another)
        const bool small_sample = P * C * es < (int64_t(1) << 31);
        for (int64_t segment = 128; segment >= 64 && p.way == Way::split && small_sample; segment >>= 1) {
            int64_t gpb = ceil_div(segment, cpg * es);
            gpb = gpb < G ? gpb : G;
            const int64_t cols = gpb * vpg;
            for (int block : {256, 1024}) {
                if (backward && block == 1024 && es == 8) continue;  // 64-bit sums do not fit 128 registers
                const int held = held_vectors(static_cast<int>(es), static_cast<int>(n), block, backward);
                if (cols > block || ceil_div(P, block / cols) > held) continue;
                if (!backward && S * ceil_div(G, gpb) * block > (int64_t(1) << 31)) continue;   // more threads than a launch
                p.way = Way::slab;
                p.block = block;
                p.gpb = static_cast<int>(gpb);
                p.bundles = static_cast<int>(ceil_div(G, gpb));
                break;
            }
        }
        if (p.way == Way::slab) {
            const int64_t wanted = ceil_div(p.block == 256 ? 2048 : 512, p.bundles);
            p.part_rows = wanted < S ? wanted : S;
        } else {
            const int64_t columns = G * vpg;
            p.cols = static_cast<int>(columns < 64 ? columns : 64);
            p.col_blocks = static_cast<int>(ceil_div(columns, p.cols));
            const int64_t rows = kSplitBlock / p.cols;
            int64_t slices = ceil_div(4096, S * p.col_blocks);
            const int64_t most = ceil_div(P, rows * 4);
            slices = slices < most ? slices : most;
            p.span = static_cast<int>(ceil_div(P, slices));
            p.slices = static_cast<int>(ceil_div(P, p.span));
            p.part_rows = S * p.slices;
        }
    }
    if (backward) {
        p.bytes = round_up(static_cast<size_t>(p.part_rows) * 2 * static_cast<size_t>(C) * arith, 16);
        p.coefficients = p.bytes;
        if (p.way == Way::split) p.bytes += static_cast<size_t>(S) * static_cast<size_t>(G) * 2 * arith;
    } else if (p.way == Way::split) {
        p.bytes = static_cast<size_t>(S) * p.slices * 2 * static_cast<size_t>(G * vpg) * sizeof(double);
    }
    return p;
}

struct Call {
    const void *x, *weight, *bias, *mean, *rstd, *grad;
    void *out, *mean_out, *rstd_out, *grad_weight, *grad_bias;
    int64_t S, P, C, G;
    double eps;
    int act;
    char* ws;
    hipStream_t stream;
};

template <typename E, int BYTES, bool RAGGED, int K, int U>
hipError_t rows_forward_by(const Call& a, const Plan& p) {
    using A = arith_t<E>;
    const int64_t items = a.S * a.G, step = ceil_div(a.S, U) * a.G;
    return launch(gn_rows_forward_kernel<E, BYTES, RAGGED, K, U>,
                  dim3(static_cast<unsigned>(ceil_div(step, kRowsBlock >> p.lanes_log2))), dim3(kRowsBlock), a.stream,
                  static_cast<const E*>(a.x), static_cast<const E*>(a.weight), static_cast<const E*>(a.bias),
                  static_cast<E*>(a.out), static_cast<A*>(a.mean_out), static_cast<A*>(a.rstd_out), items, step,
                  static_cast<int>(a.G), static_cast<int>(a.C / a.G), static_cast<A>(a.eps), a.act, p.lanes_log2);
}

template <typename E, int BYTES, bool RAGGED, int K>
hipError_t rows_forward(const Call& a, const Plan& p) {
    // four samples per group of lanes where that leaves eight workgroups for every CU: more requests in flight
    // ([16384, 8 groups of 128] bf16 silu: 21.5 us); fewer samples want the workgroups
    if (K == 1 && a.S * a.G >= int64_t(4) * 8 * 256 * (kRowsBlock >> p.lanes_log2)) return rows_forward_by<E, BYTES, RAGGED, K, 4>(a, p);
    return rows_forward_by<E, BYTES, RAGGED, K, 1>(a, p);
}

template <typename E, int BYTES, bool RAGGED, int K>
hipError_t rows_backward(const Call& a, const Plan& p) {
    using A = arith_t<E>;
    return launch(gn_rows_backward_kernel<E, BYTES, RAGGED, K>,
                  dim3(static_cast<unsigned>(p.part_rows), static_cast<unsigned>(p.group_blocks)), dim3(kRowsBlock),
                  a.stream, static_cast<const E*>(a.x), static_cast<const E*>(a.weight), static_cast<const E*>(a.bias),
                  static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd), static_cast<const E*>(a.grad),
                  static_cast<E*>(a.out), reinterpret_cast<A*>(a.ws), a.S, static_cast<int>(a.G),
                  static_cast<int>(a.C / a.G), a.act, p.lanes_log2, p.gpb, p.spb);
}

template <typename E, int BYTES, bool RAGGED, int BT>
hipError_t slab_forward(const Call& a, const Plan& p) {
    using A = arith_t<E>;
    return launch(gn_slab_forward_kernel<E, BYTES, RAGGED, BT>, dim3(static_cast<unsigned>(a.S * p.bundles)), dim3(BT),
                  a.stream, static_cast<const E*>(a.x), static_cast<const E*>(a.weight), static_cast<const E*>(a.bias),
                  static_cast<E*>(a.out), static_cast<A*>(a.mean_out), static_cast<A*>(a.rstd_out), p.bundles,
                  static_cast<int>(a.P), static_cast<int>(a.G), static_cast<int>(a.C / a.G), p.gpb,
                  static_cast<A>(a.eps), a.act);
}

template <typename E, int BYTES, bool RAGGED, int BT>
hipError_t slab_backward(const Call& a, const Plan& p) {
    using A = arith_t<E>;
    return launch(gn_slab_backward_kernel<E, BYTES, RAGGED, BT>, dim3(static_cast<unsigned>(p.part_rows * p.bundles)),
                  dim3(BT), a.stream, static_cast<const E*>(a.x), static_cast<const E*>(a.weight),
                  static_cast<const E*>(a.bias), static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd),
                  static_cast<const E*>(a.grad), static_cast<E*>(a.out), reinterpret_cast<A*>(a.ws), a.S, p.bundles,
                  static_cast<int>(p.part_rows), static_cast<int>(a.P), static_cast<int>(a.G),
                  static_cast<int>(a.C / a.G), p.gpb, a.act);
}

template <typename E, int BYTES, bool RAGGED>
hipError_t split_forward(const Call& a, const Plan& p) {
    using A = arith_t<E>;
    const int P = static_cast<int>(a.P), C = static_cast<int>(a.C), G = static_cast<int>(a.G);
    const dim3 grid(static_cast<unsigned>(a.S), static_cast<unsigned>(p.slices), static_cast<unsigned>(p.col_blocks));
    const E* x = static_cast<const E*>(a.x);
    double* part = reinterpret_cast<double*>(a.ws);
    hipError_t err = launch(gn_split_statistics_kernel<E, BYTES, RAGGED>, grid, dim3(kSplitBlock), a.stream, x, part, P, C,
                            C / G, p.cols, p.span);
    if (err == hipSuccess)
        err = launch(gn_split_finish_kernel<E>, dim3(static_cast<unsigned>(a.S * a.G)), dim3(64), a.stream, x,
                     const_cast<const double*>(part), static_cast<A*>(a.mean_out), static_cast<A*>(a.rstd_out), P, C, G,
                     G * static_cast<int>(ceil_div(C / G, Vec<E, BYTES>::n)), p.slices, a.eps);
    if (err == hipSuccess)
        err = launch(gn_split_apply_kernel<E, BYTES, RAGGED>, grid, dim3(kSplitBlock), a.stream, x,
                     static_cast<const E*>(a.weight), static_cast<const E*>(a.bias),
                     static_cast<const A*>(a.mean_out), static_cast<const A*>(a.rstd_out),
                     static_cast<const E*>(nullptr), static_cast<const A*>(nullptr), static_cast<E*>(a.out), P, C, G,
                     p.cols, p.span, a.act);
    return err;
}

template <typename E, int BYTES, bool RAGGED>
hipError_t split_backward(const Call& a, const Plan& p) {
    using A = arith_t<E>;
    const int P = static_cast<int>(a.P), C = static_cast<int>(a.C), G = static_cast<int>(a.G);
    const dim3 grid(static_cast<unsigned>(a.S), static_cast<unsigned>(p.slices), static_cast<unsigned>(p.col_blocks));
    const E *x = static_cast<const E*>(a.x), *weight = static_cast<const E*>(a.weight),
            *bias = static_cast<const E*>(a.bias), *grad = static_cast<const E*>(a.grad);
    const A *mean = static_cast<const A*>(a.mean), *rstd = static_cast<const A*>(a.rstd);
    A* part = reinterpret_cast<A*>(a.ws);
    A* coefficients = reinterpret_cast<A*>(a.ws + p.coefficients);
    hipError_t err = launch(gn_split_sums_kernel<E, BYTES, RAGGED>, grid, dim3(kSplitBlock), a.stream, x, weight, bias, mean,
                            rstd, grad, part, P, C, G, p.cols, p.span, a.act);
    if (err == hipSuccess)
        err = launch(gn_split_coefficients_kernel<E>, dim3(static_cast<unsigned>(a.S * a.G)), dim3(64), a.stream,
                     const_cast<const A*>(part), weight, coefficients, P, C, G, p.slices);
    if (err == hipSuccess)
        err = launch(gn_split_apply_kernel<E, BYTES, RAGGED>, grid, dim3(kSplitBlock), a.stream, x, weight, bias, mean, rstd,
                     grad, const_cast<const A*>(coefficients), static_cast<E*>(a.out), P, C, G, p.cols, p.span, a.act);
    return err;
}

template <typename E, int BYTES, bool RAGGED>
hipError_t run_as(const Call& a, const Plan& p, bool backward) {
    hipError_t err;
    if (p.way == Way::rows) {
        if (p.vectors == 1) err = backward ? rows_backward<E, BYTES, RAGGED, 1>(a, p) : rows_forward<E, BYTES, RAGGED, 1>(a, p);
        else if (p.vectors == 2) err = backward ? rows_backward<E, BYTES, RAGGED, 2>(a, p) : rows_forward<E, BYTES, RAGGED, 2>(a, p);
        else err = backward ? rows_backward<E, BYTES, RAGGED, 4>(a, p) : rows_forward<E, BYTES, RAGGED, 4>(a, p);
    } else if (p.way == Way::slab) {
        if (p.block == 256) err = backward ? slab_backward<E, BYTES, RAGGED, 256>(a, p) : slab_forward<E, BYTES, RAGGED, 256>(a, p);
        else if constexpr (sizeof(E) == 8) err = slab_forward<E, BYTES, RAGGED, 1024>(a, p);
        else err = backward ? slab_backward<E, BYTES, RAGGED, 1024>(a, p) : slab_forward<E, BYTES, RAGGED, 1024>(a, p);
    } else {
        err = backward ? split_backward<E, BYTES, RAGGED>(a, p) : split_forward<E, BYTES, RAGGED>(a, p);
    }
    if (err == hipSuccess && backward)
        err = launch(gn_parameters_kernel<E>, dim3(static_cast<unsigned>(ceil_div(2 * a.C, 32))), dim3(1024), a.stream,
                     reinterpret_cast<const arith_t<E>*>(a.ws), static_cast<E*>(a.grad_weight),
                     static_cast<E*>(a.grad_bias), p.part_rows, static_cast<int>(a.C));
    return err;
}

template <typename E, int BYTES>
hipError_t run_by(const Call& a, const Plan& p, bool backward) {
    if constexpr (BYTES > static_cast<int>(sizeof(E)))
        if (a.C / a.G % Vec<E, BYTES>::n != 0) return run_as<E, BYTES, true>(a, p, backward);
    return run_as<E, BYTES, false>(a, p, backward);
}

hipError_t run(int dtype, const Call& a, const Plan& p, bool backward) {
    const int bytes = widest_vector(a.C / a.G, element_size(dtype));
    if (dtype == SNNLIF_DTYPE_F32)
        return bytes == 16  ? run_by<float, 16>(a, p, backward)
               : bytes == 8 ? run_by<float, 8>(a, p, backward)
                            : run_by<float, 4>(a, p, backward);
    if (dtype == SNNLIF_DTYPE_F64)
        return bytes == 16 ? run_by<double, 16>(a, p, backward) : run_by<double, 8>(a, p, backward);
    return bytes == 16  ? run_by<bf16_t, 16>(a, p, backward)
           : bytes == 8 ? run_by<bf16_t, 8>(a, p, backward)
           : bytes == 4 ? run_by<bf16_t, 4>(a, p, backward)
                        : run_by<bf16_t, 2>(a, p, backward);
}

int gn_shape_error(int dtype, int64_t S, int64_t P, int64_t C, int64_t G, int act) {
    if (element_size(dtype) == 0) return SNNLIF_ERR_DTYPE;
    if (S < 0 || P < 0 || C < 0 || G < 1 || C > SNNSEQ_MAX_CHANNELS || C % G != 0) return SNNLIF_ERR_ARG;
    if (act < SNNSEQ_ACT_NONE || act > SNNSEQ_ACT_GELU) return SNNLIF_ERR_ARG;
    // samples times groups and positions are launch sizes or 32-bit numbers on the device
    if (S > SNNSEQ_MAX_TOKENS / G || P > SNNSEQ_MAX_TOKENS) return SNNLIF_ERR_ARG;
    if (S > 0 && (P == 0 || C == 0)) return SNNLIF_ERR_ARG;
    return SNNLIF_OK;
}

}  // namespace
}  // namespace snnseq

using namespace snnseq;

extern "C" size_t snnseq_gn_act_workspace_bytes(int dtype, int64_t S, int64_t P, int64_t C, int64_t G, int backward) {
    if (gn_shape_error(dtype, S, P, C, G, SNNSEQ_ACT_NONE) != SNNLIF_OK || S == 0) return 0;
    return plan_of(dtype, S, P, C, G, backward != 0).bytes;
}

extern "C" int snnseq_gn_act_fp(const void* x, const void* weight, const void* bias, void* y, void* mean, void* rstd,
                                int dtype, int64_t S, int64_t P, int64_t C, int64_t G, double eps, int act,
                                void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = gn_shape_error(dtype, S, P, C, G, act);
    if (bad != SNNLIF_OK) return bad;
    if (S == 0) return SNNLIF_OK;
    if (x == nullptr || weight == nullptr || bias == nullptr || y == nullptr || mean == nullptr || rstd == nullptr)
        return SNNLIF_ERR_ARG;
    const size_t es = element_size(dtype), as = es == 8 ? 8 : 4;
    if (!aligned_to(x, es) || !aligned_to(weight, es) || !aligned_to(bias, es) || !aligned_to(y, es) ||
        !aligned_to(mean, as) || !aligned_to(rstd, as) || !aligned_to(workspace, 16))
        return SNNLIF_ERR_ALIGN;
    const Plan p = plan_of(dtype, S, P, C, G, false);
    if (p.bytes > 0 && (workspace == nullptr || workspace_bytes < p.bytes)) return SNNLIF_ERR_WORKSPACE;
    Call a{};
    a.x = x; a.weight = weight; a.bias = bias; a.out = y; a.mean_out = mean; a.rstd_out = rstd;
    a.S = S; a.P = P; a.C = C; a.G = G; a.eps = eps; a.act = act;
    a.ws = static_cast<char*>(workspace);
    a.stream = static_cast<hipStream_t>(stream);
    return static_cast<int>(run(dtype, a, p, false));
}

extern "C" int snnseq_gn_act_bp(const void* x, const void* weight, const void* bias, const void* mean,
                                const void* rstd, const void* grad_y, void* grad_x, void* grad_weight, void* grad_bias,
                                int dtype, int64_t S, int64_t P, int64_t C, int64_t G, int act, void* workspace,
                                size_t workspace_bytes, void* stream) {
    const int bad = gn_shape_error(dtype, S, P, C, G, act);
    if (bad != SNNLIF_OK) return bad;
    if (S == 0) return SNNLIF_OK;
    if (x == nullptr || weight == nullptr || bias == nullptr || mean == nullptr || rstd == nullptr ||
        grad_y == nullptr || grad_x == nullptr || grad_weight == nullptr || grad_bias == nullptr)
        return SNNLIF_ERR_ARG;
    const size_t es = element_size(dtype), as = es == 8 ? 8 : 4;
    if (!aligned_to(x, es) || !aligned_to(weight, es) || !aligned_to(bias, es) || !aligned_to(grad_y, es) ||
        !aligned_to(grad_x, es) || !aligned_to(grad_weight, es) || !aligned_to(grad_bias, es) ||
        !aligned_to(mean, as) || !aligned_to(rstd, as) || !aligned_to(workspace, 16))
        return SNNLIF_ERR_ALIGN;
    const Plan p = plan_of(dtype, S, P, C, G, true);
    if (workspace == nullptr || workspace_bytes < p.bytes) return SNNLIF_ERR_WORKSPACE;
    Call a{};
    a.x = x; a.weight = weight; a.bias = bias; a.mean = mean; a.rstd = rstd; a.grad = grad_y; a.out = grad_x;
    a.grad_weight = grad_weight; a.grad_bias = grad_bias;
    a.S = S; a.P = P; a.C = C; a.G = G; a.act = act;
    a.ws = static_cast<char*>(workspace);
    a.stream = static_cast<hipStream_t>(stream);
    return static_cast<int>(run(dtype, a, p, true));
}
