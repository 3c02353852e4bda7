// Embedding lookup with a scale, and its gradient by sorted tokens.
//
//   forward    y[n, :] = scale * W[token[n], :]                       (a token outside [0, V): a row of zeros)
//   backward   dW[v, :] = scale * sum over n with token[n] = v, in ascending n, of g[n, :]
//
// Both are bound by memory.  The forward reads and writes each row once (32768 tokens of 1024 bf16 columns: 17 us, 67 MB
// written, most rows read from the caches).  The backward reads g once and
// writes all V rows of dW (most of them zero for a large vocabulary); sums are held in 32 bits (64 for
// double storage), always in the same order, so results are reproducible.
//
// The gradient takes three launches:
//   1. sort.  Positions ordered by token, equal tokens in ascending position, without any exchange between
//      workgroups: each workgroup owns R consecutive rows of the table, reads all N tokens (they stay in L2), counts
//      those below its rows -- where its part of the order begins -- and keeps those of its rows in LDS, from where
//      it places them.  A wavefront that meets more of them than it can keep reads its tokens once more instead.
//      32768 tokens, 50000 rows: 40 us with the second reading for all, 14 us with the lists.
//   2. rows and pieces.  A row with at most a piece's positions is summed by the threads that own its columns.
//      The positions of longer rows (frequent words) are cut at multiples of a piece in the sorted order;
//      every piece is summed by a workgroup of its own, in the same launch.
//      The same sizes, 1024 bf16 columns: 43 us (67 MB read, 102 MB written: 3.9 TB/s; a row's few reads follow each
//      other, so a group of threads begins four rows at a time).
//   3. merge.  The pieces of each long row, in order (6 us).  Not launched where N cannot hold a long row.
#include "seq_common.h"

namespace snnseq {
namespace {

constexpr int kBlock = 256;
constexpr int kSortBlock = 1024;
constexpr int kSortWaves = kSortBlock / 64;
constexpr int kRowsInFlight = 4;  // rows requested before the first is used
constexpr int kRowsTogether = 4;  // rows of the gradient whose first tokens are requested together

// The last vector of a row shares columns with the one before: both write the same values there.
__device__ __forceinline__ int at_most(int a, int b) { return a < b ? a : b; }

template <typename I>
__device__ __forceinline__ int row_of(const I* tokens, int64_t n, int V) {
    const int64_t t = static_cast<int64_t>(tokens[n]);
    return static_cast<uint64_t>(t) < static_cast<uint64_t>(V) ? static_cast<int>(t) : -1;
}

// ---- forward ------------------------------------------------------------------------------------

// `tpr` threads (a power of two) share a row, kBlock / tpr rows at a time.
template <typename E, int BYTES, typename I>
__global__ void __launch_bounds__(kBlock)
embed_forward_kernel(const I* __restrict__ tokens, const E* __restrict__ weight, E* __restrict__ out,
                     int64_t N, int V, int C, int64_t row_stride, arith_t<E> scale, int tpr_log2) {
    constexpr int n = Vec<E, BYTES>::n;
    const int tpr = 1 << tpr_log2;
    const int lane = threadIdx.x & (tpr - 1);
    const int rows = kBlock >> tpr_log2;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * rows * kRowsInFlight + (threadIdx.x >> tpr_log2);
    int row[kRowsInFlight];
#pragma unroll
    for (int r = 0; r < kRowsInFlight; ++r) {   // all requested at once: none under a condition
        const int64_t i = first + static_cast<int64_t>(r) * rows;
        row[r] = row_of(tokens, i < N ? i : N - 1, V);
    }
    for (int c0 = lane * n; c0 < C; c0 += tpr * n) {
        const int c = at_most(c0, C - n);
        Vec<E, BYTES> v[kRowsInFlight];
#pragma unroll
        for (int r = 0; r < kRowsInFlight; ++r) {
            v[r].raw = typename Vec<E, BYTES>::raw_t(0);
            if (row[r] >= 0) v[r] = load_vec<E, BYTES>(weight + row[r] * row_stride + c);
        }
#pragma unroll
        for (int r = 0; r < kRowsInFlight; ++r) {
            const int64_t i = first + static_cast<int64_t>(r) * rows;
            if (i >= N) continue;
            // a zero row is written as it is: scale * 0 would be NaN for an infinite scale
            if (row[r] >= 0) {
#pragma unroll
                for (int j = 0; j < n; ++j) v[r].e[j] = narrow<E>(scale * widen(v[r].e[j]));
            }
            store_vec<E, BYTES>(out + i * C + c, v[r]);
        }
    }
}

// ---- backward: the order ------------------------------------------------------------------------

// Lanes of the wavefront that hold the same `key` (BITS wide) among those that are `in`.
template <int BITS>
__device__ __forceinline__ uint64_t same_key(int key, bool in) {
    uint64_t mask = __ballot(in);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const bool bit = (key >> b) & 1;
        const uint64_t with = __ballot(bit);
        mask &= bit ? with : ~with;
    }
    return mask;
}

// Workgroup blockIdx.x owns table rows [lo, lo + 2^RBITS).  Wavefront w reads tokens [w*span, (w+1)*span).
//   start[v]   first place of row v in the order (start[V] = number of positions in the order)
//   position[] positions by (token, position);  row[] their tokens
template <int RBITS, typename I>
__global__ void __launch_bounds__(kSortBlock)
embed_sort_kernel(const I* __restrict__ tokens, int64_t N, int V, int* __restrict__ start,
                  int* __restrict__ position, int* __restrict__ row) {
    constexpr int R = 1 << RBITS;
    constexpr int kAhead = 8;     // token groups requested at once
    constexpr int kKept = 256;    // tokens of its rows a wavefront keeps
    __shared__ int count[kSortWaves][R];
    __shared__ int total[R];
    __shared__ int kept_at[kSortWaves][kKept];
    __shared__ uint16_t kept_row[kSortWaves][kKept];
    __shared__ int below_of[kSortWaves];
    __shared__ int scan_of[kSortWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint64_t before = (uint64_t(1) << lane) - 1;
    const int lo = blockIdx.x * R;
    const int64_t span = (N + kSortBlock - 1) / kSortBlock * 64;
    const int64_t begin = wave * span;
    const int64_t end = begin + span < N ? begin + span : N;

    for (int i = tid; i < kSortWaves * R; i += kSortBlock) (&count[0][0])[i] = 0;
    __syncthreads();

    int below = 0, found = 0;
    for (int64_t i0 = begin; i0 < end; i0 += 64 * kAhead) {
        int key[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int64_t i = i0 + a * 64 + lane;
            key[a] = row_of(tokens, i < end ? i : end - 1, V);
            if (i >= end) key[a] = -1;
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            below += __popcll(__ballot(key[a] >= 0 && key[a] < lo));
            const bool in = key[a] >= lo && key[a] - lo < R;
            const uint64_t mine = __ballot(in);
            if (mine == 0) continue;
            if (in) {
                const int place = found + __popcll(mine & before);
                atomicAdd(&count[wave][key[a] - lo], 1);
                if (place < kKept) {
                    kept_at[wave][place] = static_cast<int>(i0 + a * 64 + lane);
                    kept_row[wave][place] = static_cast<uint16_t>(key[a] - lo);
                }
            }
            found += __popcll(mine);
        }
    }
    if (lane == 0) below_of[wave] = below;
    __syncthreads();

    // total[r] = positions of row lo + r;  count[w][r] = those that earlier wavefronts hold
    for (int r = tid; r < R; r += kSortBlock) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const int c = count[w][r];
            count[w][r] = sum;
            sum += c;
        }
        total[r] = sum;
    }
    int base = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) base += below_of[w];
    __syncthreads();

    // exclusive scan of total[] (one value per thread, R <= kSortBlock), added to count[]
    const int mine = tid < R ? total[tid] : 0;
    int inclusive = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(inclusive, d);
        if (lane >= d) inclusive += other;
    }
    if (lane == 63) scan_of[wave] = inclusive;
    __syncthreads();
    int offset = base + inclusive - mine;
    for (int w = 0; w < wave; ++w) offset += scan_of[w];
    if (tid < R) {
        if (lo + tid <= V) start[lo + tid] = offset;   // row V, in the last workgroup: the number of positions
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) count[w][tid] += offset;
    }
    __syncthreads();

    // 64 positions in ascending order, each with its row r if it is `in`
    const auto place_group = [&](bool in, int r, int at) {
        const uint64_t same = same_key<RBITS>(r, in);
        const int leader = in ? __ffsll(static_cast<unsigned long long>(same)) - 1 : lane;
        int place = 0;
        if (in && lane == leader) place = atomicAdd(&count[wave][r], __popcll(same));
        place = __shfl(place, leader) + __popcll(same & before);
        if (in) {
            position[place] = at;
            row[place] = lo + r;
        }
    };
    if (found <= kKept) {
        for (int k0 = 0; k0 < found; k0 += 64) {
            const bool in = k0 + lane < found;
            const int k = in ? k0 + lane : k0;
            place_group(in, kept_row[wave][k], kept_at[wave][k]);
        }
        return;
    }
    for (int64_t i0 = begin; i0 < end; i0 += 64 * kAhead) {
        int key[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int64_t i = i0 + a * 64 + lane;
            key[a] = row_of(tokens, i < end ? i : end - 1, V);
            if (i >= end) key[a] = -1;
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const bool in = key[a] >= lo && key[a] - lo < R;
            if (__ballot(in) != 0) place_group(in, in ? key[a] - lo : 0, static_cast<int>(i0 + a * 64 + lane));
        }
    }
}

// ---- backward: the sums -------------------------------------------------------------------------

// Adds g[position[j], c .. c+n) for j in [from, to) step `step`.
template <typename E, int BYTES>
__device__ __forceinline__ void add_rows(const E* __restrict__ grad, const int* __restrict__ position, int from,
                                         int to, int step, int C, int c, arith_t<E> (&acc)[Vec<E, BYTES>::n]) {
    constexpr int n = Vec<E, BYTES>::n;
    int j = from;
    for (; j + (kRowsInFlight - 1) * step < to; j += kRowsInFlight * step) {
        Vec<E, BYTES> v[kRowsInFlight];
#pragma unroll
        for (int r = 0; r < kRowsInFlight; ++r)
            v[r] = load_vec_once<E, BYTES>(grad + static_cast<int64_t>(position[j + r * step]) * C + c);
#pragma unroll
        for (int r = 0; r < kRowsInFlight; ++r)
#pragma unroll
            for (int k = 0; k < n; ++k) acc[k] += widen(v[r].e[k]);
    }
    for (; j < to; j += step) {
        const Vec<E, BYTES> v = load_vec_once<E, BYTES>(grad + static_cast<int64_t>(position[j]) * C + c);
#pragma unroll
        for (int k = 0; k < n; ++k) acc[k] += widen(v.e[k]);
    }
}

template <typename E, int BYTES>
__device__ __forceinline__ void store_row(E* p, const arith_t<E> (&acc)[Vec<E, BYTES>::n], arith_t<E> scale) {
    Vec<E, BYTES> v;
#pragma unroll
    for (int k = 0; k < Vec<E, BYTES>::n; ++k) v.e[k] = narrow<E>(scale * acc[k]);
    store_vec_once<E, BYTES>(p, v);
}

// The groups of a workgroup each hold a sum over every (kBlock/tpr)-th row of the same columns: adds them in order.
template <typename A, int n>
__device__ __forceinline__ void add_groups(A (&acc)[n], A (*shared)[kBlock], int tpr, int group, int groups) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < n; ++k) shared[k][threadIdx.x] = acc[k];
    __syncthreads();
    if (group == 0) {
        for (int o = 1; o < groups; ++o)
#pragma unroll
            for (int k = 0; k < n; ++k) acc[k] += shared[k][threadIdx.x + o * tpr];
    }
}

// Workgroups below row_blocks: whole rows.  The others: one piece of the order each; piece p leaves the sum over
// its first long row in part[p][0] and over the long row it ends in (if another) in part[p][1].
template <typename E, int BYTES, int TOGETHER>
__global__ void __launch_bounds__(kBlock)
embed_sum_kernel(const E* __restrict__ grad, const int* __restrict__ start, const int* __restrict__ position,
                 const int* __restrict__ row, E* __restrict__ grad_weight, arith_t<E>* __restrict__ part, int V,
                 int C, arith_t<E> scale, int row_blocks, int tpr_log2, int piece_log2) {
    using A = arith_t<E>;
    constexpr int n = Vec<E, BYTES>::n;
    __shared__ A shared[n][kBlock];
    const int tpr = 1 << tpr_log2;
    const int lane = threadIdx.x & (tpr - 1), group = threadIdx.x >> tpr_log2, groups = kBlock >> tpr_log2;
    const int c0 = (blockIdx.y * tpr + lane) * n, c = at_most(c0, C - n), piece = 1 << piece_log2;
    if (static_cast<int>(blockIdx.x) < row_blocks) {
        // rows far apart: frequent words are often neighbours
        const int64_t v0 = static_cast<int64_t>(blockIdx.x) * groups + group, hop = static_cast<int64_t>(row_blocks) * groups;
        if (v0 >= V || c0 >= C) return;
        int from[TOGETHER], count[TOGETHER], at[TOGETHER];
        Vec<E, BYTES> first[TOGETHER];
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
            const int64_t v = v0 + i * hop < V ? v0 + i * hop : V - 1;
            from[i] = start[v];
            count[i] = start[v + 1] - from[i];
        }
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
            if (v0 + i * hop >= V) count[i] = piece + 1;   // as the long rows: not written here
            at[i] = count[i] > 0 && count[i] <= piece ? position[from[i]] : -1;
        }
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
            first[i].raw = typename Vec<E, BYTES>::raw_t(0);
            if (at[i] >= 0) first[i] = load_vec_once<E, BYTES>(grad + static_cast<int64_t>(at[i]) * C + c);
        }
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
            if (count[i] > piece) continue;
            A acc[n];
#pragma unroll
            for (int k = 0; k < n; ++k) acc[k] = widen(first[i].e[k]);
            if (count[i] > 1) add_rows<E, BYTES>(grad, position, from[i] + 1, from[i] + count[i], 1, C, c, acc);
            // a row without a token is zero: scale * 0 would be NaN for an infinite scale
            store_row<E, BYTES>(grad_weight + (v0 + i * hop) * C + c, acc, count[i] > 0 ? scale : A(0));
        }
        return;
    }
    const int p = blockIdx.x - row_blocks;
    const int end = start[V];
    const int first = p * piece;
    if (first >= end) return;
    const int last = first + piece < end ? first + piece : end;
    const int row_a = row[first], row_b = row[last - 1];
    for (int side = 0; side < 2; ++side) {
        const int r = side == 0 ? row_a : row_b;
        if (side == 1 && row_b == row_a) break;
        const int r_from = start[r], r_to = start[r + 1];
        if (r_to - r_from <= piece) continue;
        const int from = r_from > first ? r_from : first, to = r_to < last ? r_to : last;
        A acc[n] = {};
        if (c0 < C) add_rows<E, BYTES>(grad, position, from + group, to, groups, C, c, acc);
        if (groups > 1) add_groups<A, n>(acc, shared, tpr, group, groups);
        if (group == 0 && c0 < C) {
            A* dst = part + (static_cast<int64_t>(p) * 2 + side) * C + c;
#pragma unroll
            for (int k = 0; k < n; ++k) dst[k] = acc[k];
        }
    }
}

// Most workgroups find no row and cost their launch, which wide ones are fewer for (32768 tokens of 1024 bf16 columns,
// the whole gradient: 87.7 us with 128 columns each, 92.3 with 32); narrower ones have more threads for a long sum.
constexpr int kMergeColumns = 128;

// Workgroup p: the long row that begins in piece p, if one does (the last row of the piece: a row of more
// positions than a piece ends behind the piece it begins in).
template <typename E>
__global__ void __launch_bounds__(kBlock)
embed_merge_kernel(const int* __restrict__ start, const int* __restrict__ row, E* __restrict__ grad_weight,
                   const arith_t<E>* __restrict__ part, int V, int C, arith_t<E> scale, int piece_log2) {
    using A = arith_t<E>;
    constexpr int kColumns = kMergeColumns, kGroups = kBlock / kColumns;
    __shared__ A shared[1][kBlock];
    const int p = blockIdx.x, piece = 1 << piece_log2;
    const int end = start[V];
    const int first = p * piece;
    if (first >= end) return;
    const int last = first + piece < end ? first + piece : end;
    const int r = row[last - 1];
    const int r_from = start[r], r_to = start[r + 1];
    if (r_to - r_from <= piece || r_from < first) return;
    const int lane = threadIdx.x & (kColumns - 1), group = threadIdx.x / kColumns;
    const int side = r_from == first ? 0 : 1;     // the row opens the piece or follows others
    const int pieces = ((r_to - 1) >> piece_log2) - p + 1;
    const int c = blockIdx.y * kColumns + lane;
    A acc[1] = {A(0)};
    if (c < C) {
#pragma unroll 8
        for (int j = group; j < pieces; j += kGroups)
            acc[0] += part[(static_cast<int64_t>(p + j) * 2 + (j == 0 ? side : 0)) * C + c];
    }
    add_groups<A, 1>(acc, shared, kColumns, group, kGroups);
    if (group == 0 && c < C) grad_weight[static_cast<int64_t>(r) * C + c] = narrow<E>(scale * acc[0]);
}

// ---- host ---------------------------------------------------------------------------------------

// Threads that share a row: one vector of columns each, at most a workgroup.
int log2_threads_per_row(int64_t vectors) {
    int l = 0;
    while ((1 << l) < vectors && (1 << l) < kBlock) ++l;
    return l;
}

template <typename E, int BYTES, typename I>
hipError_t forward_as(const void* tokens, const void* weight, void* out, int64_t N, int64_t V, int64_t C,
                      int64_t row_stride, double scale, hipStream_t st) {
    const int l = log2_threads_per_row(ceil_div(C, Vec<E, BYTES>::n));
    const int64_t rows = int64_t(kBlock >> l) * kRowsInFlight;
    return launch(embed_forward_kernel<E, BYTES, I>, dim3(static_cast<unsigned>(ceil_div(N, rows))), dim3(kBlock), st,
                  static_cast<const I*>(tokens), static_cast<const E*>(weight), static_cast<E*>(out), N,
                  static_cast<int>(V), static_cast<int>(C), row_stride, static_cast<arith_t<E>>(scale), l);
}

struct Layout {  // byte offsets into the workspace
    size_t start, position, row, part, bytes;
    int64_t pieces;
    int piece_log2;
};

// Positions of a row that one group of threads adds up by itself, one after another.  With few tokens the longest such
// sum is all there is to wait for, with many the sums of the pieces cost more than they save.  Backward with pieces of
// 16, 32 and 64: 1805 tokens of 2002 bf16 columns 20.6, 24 and 31 us, 6270 of 973 fp32 columns 39, 41 and 48, 16384 of
// 1024 bf16 columns 67, 64 and 66, 32768 of them 100, 92 and 91.
int piece_log2_of(int64_t N) { return N <= 8192 ? 4 : 5; }

Layout layout_of(int64_t N, int64_t V, int64_t C, size_t arith) {
    Layout w;
    w.piece_log2 = piece_log2_of(N);
    w.pieces = N > 1 << w.piece_log2 ? ceil_div(N, 1 << w.piece_log2) : 0;
    w.start = 0;
    w.position = round_up(w.start + sizeof(int) * static_cast<size_t>(V + 1), 16);
    w.row = round_up(w.position + sizeof(int) * static_cast<size_t>(N), 16);
    w.part = round_up(w.row + sizeof(int) * static_cast<size_t>(N), 16);
    w.bytes = w.part + static_cast<size_t>(w.pieces) * 2 * static_cast<size_t>(C) * arith;
    return w;
}

template <typename E, int BYTES>
hipError_t sums_as(const void* grad, void* grad_weight, char* ws, const Layout& w, int64_t V, int64_t C, double scale,
                   hipStream_t st) {
    using A = arith_t<E>;
    const int l = log2_threads_per_row(ceil_div(C, Vec<E, BYTES>::n));
    const int64_t groups = kBlock >> l;
    // where that leaves eight workgroups for every CU: 32768 tokens, 50000 rows of 512 fp32 columns, the whole gradient
    // 79 us, 86 with a row each
    const bool many = V >= kRowsTogether * groups * 2048;
    const int64_t row_blocks = ceil_div(V, many ? kRowsTogether * groups : groups);
    const int* start = reinterpret_cast<int*>(ws + w.start);
    const int* position = reinterpret_cast<int*>(ws + w.position);
    const int* row = reinterpret_cast<int*>(ws + w.row);
    A* part = reinterpret_cast<A*>(ws + w.part);
    const dim3 grid(static_cast<unsigned>(row_blocks + w.pieces),
                    static_cast<unsigned>(ceil_div(C, int64_t(Vec<E, BYTES>::n) << l)));
    hipError_t err = launch(many ? embed_sum_kernel<E, BYTES, kRowsTogether> : embed_sum_kernel<E, BYTES, 1>, grid, dim3(kBlock), st, static_cast<const E*>(grad), start, position, row,
                            static_cast<E*>(grad_weight), part, static_cast<int>(V), static_cast<int>(C),
                            static_cast<A>(scale), static_cast<int>(row_blocks), l, w.piece_log2);
    if (err == hipSuccess && w.pieces > 0)
        err = launch(embed_merge_kernel<E>, dim3(static_cast<unsigned>(w.pieces), static_cast<unsigned>(ceil_div(C, kMergeColumns))),
                     dim3(kBlock), st, start, row, static_cast<E*>(grad_weight), const_cast<const A*>(part),
                     static_cast<int>(V), static_cast<int>(C), static_cast<A>(scale), w.piece_log2);
    return err;
}

template <typename I>
hipError_t order_as(const void* tokens, int64_t N, int64_t V, char* ws, const Layout& w, hipStream_t st) {
    int* start = reinterpret_cast<int*>(ws + w.start);
    int* position = reinterpret_cast<int*>(ws + w.position);
    int* row = reinterpret_cast<int*>(ws + w.row);
    const I* t = static_cast<const I*>(tokens);
    // Every workgroup reads all tokens, so their number bounds the L2 traffic: 256 rows each up to 512
    // workgroups (two per CU), 1024 rows each for larger tables.  start[] has V + 1 entries.
    if (V < 512 * 256)
        return launch(embed_sort_kernel<8, I>, dim3(static_cast<unsigned>(ceil_div(V + 1, 256))), dim3(kSortBlock), st,
                      t, N, static_cast<int>(V), start, position, row);
    return launch(embed_sort_kernel<10, I>, dim3(static_cast<unsigned>(ceil_div(V + 1, 1024))), dim3(kSortBlock), st, t,
                  N, static_cast<int>(V), start, position, row);
}

int embed_shape_error(int dtype, int token_dtype, int64_t N, int64_t V, int64_t C) {
    if (element_size(dtype) == 0) return SNNLIF_ERR_DTYPE;
    if (token_dtype != SNNSEQ_TOKEN_I32 && token_dtype != SNNSEQ_TOKEN_I64) return SNNLIF_ERR_DTYPE;
    // positions, rows and columns are 32-bit numbers on the device; offsets are not
    if (N < 0 || V < 1 || C < 0 || N > SNNSEQ_MAX_TOKENS || V > SNNSEQ_MAX_TOKENS || C > SNNSEQ_MAX_CHANNELS)
        return SNNLIF_ERR_ARG;
    return SNNLIF_OK;
}

}  // namespace
}  // namespace snnseq

using namespace snnseq;

extern "C" int snnseq_embed_fp(const void* tokens, const void* weight, void* out, int dtype, int token_dtype,
                               int64_t N, int64_t V, int64_t C, int64_t row_stride, double scale, void* stream) {
    const int bad = embed_shape_error(dtype, token_dtype, N, V, C);
    if (bad != SNNLIF_OK) return bad;
    if (N == 0 || C == 0) return SNNLIF_OK;
    if (tokens == nullptr || weight == nullptr || out == nullptr || row_stride < 0) return SNNLIF_ERR_ARG;
    const size_t es = element_size(dtype);
    if (!aligned_to(tokens, token_dtype == SNNSEQ_TOKEN_I32 ? 4 : 8) || !aligned_to(weight, es) || !aligned_to(out, es))
        return SNNLIF_ERR_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int bytes = widest_vector(C, es);
    const bool wide = token_dtype == SNNSEQ_TOKEN_I64;
#define SNNSEQ_FORWARD(E, B)                                                                                     \
    (wide ? forward_as<E, B, int64_t>(tokens, weight, out, N, V, C, row_stride, scale, st)                       \
          : forward_as<E, B, int32_t>(tokens, weight, out, N, V, C, row_stride, scale, st))
    hipError_t err;
    if (dtype == SNNLIF_DTYPE_F32)
        err = bytes == 16 ? SNNSEQ_FORWARD(float, 16) : bytes == 8 ? SNNSEQ_FORWARD(float, 8) : SNNSEQ_FORWARD(float, 4);
    else if (dtype == SNNLIF_DTYPE_F64)
        err = bytes == 16 ? SNNSEQ_FORWARD(double, 16) : SNNSEQ_FORWARD(double, 8);
    else
        err = bytes == 16  ? SNNSEQ_FORWARD(bf16_t, 16)
              : bytes == 8 ? SNNSEQ_FORWARD(bf16_t, 8)
              : bytes == 4 ? SNNSEQ_FORWARD(bf16_t, 4)
                           : SNNSEQ_FORWARD(bf16_t, 2);
#undef SNNSEQ_FORWARD
    return static_cast<int>(err);
}

extern "C" size_t snnseq_embed_bp_workspace_bytes(int dtype, int64_t N, int64_t V, int64_t C) {
    if (embed_shape_error(dtype, SNNSEQ_TOKEN_I64, N, V, C) != SNNLIF_OK) return 0;
    return layout_of(N, V, C, dtype == SNNLIF_DTYPE_F64 ? 8 : 4).bytes;
}

extern "C" int snnseq_embed_bp(const void* tokens, const void* grad, void* grad_weight, int dtype, int token_dtype,
                               int64_t N, int64_t V, int64_t C, double scale, void* workspace, size_t workspace_bytes,
                               void* stream) {
    const int bad = embed_shape_error(dtype, token_dtype, N, V, C);
    if (bad != SNNLIF_OK) return bad;
    if (C == 0) return SNNLIF_OK;
    if ((N > 0 && (tokens == nullptr || grad == nullptr)) || grad_weight == nullptr) return SNNLIF_ERR_ARG;
    const size_t es = element_size(dtype);
    if (!aligned_to(tokens, token_dtype == SNNSEQ_TOKEN_I32 ? 4 : 8) || !aligned_to(grad, es) ||
        !aligned_to(grad_weight, es) || !aligned_to(workspace, 16))
        return SNNLIF_ERR_ALIGN;
    const Layout w = layout_of(N, V, C, dtype == SNNLIF_DTYPE_F64 ? 8 : 4);
    if (workspace == nullptr || workspace_bytes < w.bytes) return SNNLIF_ERR_WORKSPACE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    hipError_t err = token_dtype == SNNSEQ_TOKEN_I64 ? order_as<int64_t>(tokens, N, V, ws, w, st)
                                                     : order_as<int32_t>(tokens, N, V, ws, w, st);
    if (err != hipSuccess) return static_cast<int>(err);
    const int bytes = widest_vector(C, es);
#define SNNSEQ_SUMS(E, B) sums_as<E, B>(grad, grad_weight, ws, w, V, C, scale, st)
    if (dtype == SNNLIF_DTYPE_F32)
        err = bytes == 16 ? SNNSEQ_SUMS(float, 16) : bytes == 8 ? SNNSEQ_SUMS(float, 8) : SNNSEQ_SUMS(float, 4);
    else if (dtype == SNNLIF_DTYPE_F64)
        err = bytes == 16 ? SNNSEQ_SUMS(double, 16) : SNNSEQ_SUMS(double, 8);
    else
        err = bytes == 16  ? SNNSEQ_SUMS(bf16_t, 16)
              : bytes == 8 ? SNNSEQ_SUMS(bf16_t, 8)
              : bytes == 4 ? SNNSEQ_SUMS(bf16_t, 4)
                           : SNNSEQ_SUMS(bf16_t, 2);
#undef SNNSEQ_SUMS
    return static_cast<int>(err);
}
