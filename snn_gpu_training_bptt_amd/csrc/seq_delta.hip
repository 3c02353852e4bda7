// Entry points of the gated delta rule, and its form for single tokens.
#include "seq_delta.h"

namespace snnseq {
namespace {

// ---- one token ----------------------------------------------------------------------------------
//
// o = scale S'^T q with S' = a S + k e^T, e = beta (v - a S^T k):  S^T k and S^T q are taken in one sweep over the
// state, and S'^T q = a S^T q + (k . q) e, so the state is read once, held in registers, and written once: 8 bytes
// per value, the bound.  A workgroup owns 64 columns of a head's state: 16 lanes of four columns share a row, eight
// rows at a time, and the sums over the rows go through shuffles and LDS.  A thread of 128 holds sixteen vectors of
// a state of 128 rows (with 256 threads and eight vectors each, 64 sequences of 16 heads took 38 us); registers for
// four wavefronts per SIMD.  With a state of 128 x 128: 64 sequences of 16 heads 24.6 us (134 MB: 5.5 TB/s), 512 of
// them 189 us (1.07 GB: 5.7 TB/s); of 64 x 64, 64 sequences 6.7 us and 512 of them 45 us (with a condition around each
// load the compiler waited for one after another: 9.7 and 79 us).

constexpr int kStepCols = 64, kStepThreads = 128, kStepLanes = kStepCols / 4, kStepRows = kStepThreads / kStepLanes;

struct StepArgs {
    int B, Hk, Hv, Dk, Dv;
    float scale;
    const void *q, *k, *v;
    int64_t q_b, q_h, k_b, k_h, v_b, v_h;
    const float *g, *beta, *state;
    void* o;
    float* state_out;
};

template <typename E, int ROWS, bool WIDE>   // ROWS: rows of the state per thread;  WIDE: four columns in one access
__global__ void __launch_bounds__(kStepThreads, WIDE ? 4 : 3) delta_step_kernel(StepArgs a) {
    static_assert(ROWS * kStepRows <= kStepThreads);
    __shared__ __align__(16) float qs[kStepThreads], ks[kStepThreads];
    __shared__ float part[2][kStepThreads / 64][kStepCols];
    const int head = blockIdx.y, b = head / a.Hv, hv = head - b * a.Hv, hk = hv / (a.Hv / a.Hk);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * kStepCols + (threadIdx.x % kStepLanes) * 4, r0 = threadIdx.x / kStepLanes * ROWS;
    const bool whole = a.Dk == ROWS * kStepRows;
    const E* q = static_cast<const E*>(a.q) + b * a.q_b + hk * a.q_h;
    const E* k = static_cast<const E*>(a.k) + b * a.k_b + hk * a.k_h;
    const E* v = static_cast<const E*>(a.v) + b * a.v_b + hv * a.v_h;
    const int at = static_cast<int>(threadIdx.x) < a.Dk ? static_cast<int>(threadIdx.x) : a.Dk - 1;
    const E q_in = q[at], k_in = k[at];
    E v_in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v_in[j] = v[c + j < a.Dv ? c + j : 0];
    const float g = a.g[head], beta = a.beta[head];
    const int64_t base = static_cast<int64_t>(head) * a.Dk * a.Dv;
    const uint32_t end = static_cast<uint32_t>(a.Dk) * a.Dv, row0 = static_cast<uint32_t>(r0) * a.Dv;   // below 2^23
    f32x4 s[ROWS];   // requested all at once: none under a condition, absent ones read what is there
    if (WIDE) {
        const uint32_t last = end - a.Dv + (c < a.Dv ? c : 0);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const uint32_t x = row0 + i * static_cast<uint32_t>(a.Dv) + c;
            s[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(a.state + base + (x < last ? x : last)));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t last = end - a.Dv + (c + j < a.Dv ? c + j : 0);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const uint32_t x = row0 + i * static_cast<uint32_t>(a.Dv) + c + j;
                s[i][j] = a.state[base + (x < last ? x : last)];
            }
        }
    }
    qs[threadIdx.x] = static_cast<int>(threadIdx.x) < a.Dk ? widen(q_in) : 0.f;
    ks[threadIdx.x] = static_cast<int>(threadIdx.x) < a.Dk ? widen(k_in) : 0.f;
    __syncthreads();
    f32x4 sk = zero4(), sq = zero4();
    float kq = 0.f;
    if (!whole) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
            if (r0 + i >= a.Dk) s[i] = zero4();
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const float kr = ks[r0 + i], qr = qs[r0 + i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sk[j] += kr * s[i][j];
            sq[j] += qr * s[i][j];
        }
        kq += kr * qr;
    }
#pragma unroll
    for (int d = kStepLanes; d < 64; d <<= 1) {
        kq += __shfl_xor(kq, d);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sk[j] += __shfl_xor(sk[j], d);
            sq[j] += __shfl_xor(sq[j], d);
        }
    }
    __shared__ float kq_part[kStepThreads / 64];
    if (lane < kStepLanes) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            part[0][wave][lane * 4 + j] = sk[j];
            part[1][wave][lane * 4 + j] = sq[j];
        }
        if (lane == 0) kq_part[wave] = kq;
    }
    __syncthreads();
    const float decay = expf(g);
    f32x4 add;
    float out[4];
    float kq_all = 0.f;
#pragma unroll
    for (int w = 0; w < kStepThreads / 64; ++w) kq_all += kq_part[w];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int col = (threadIdx.x % kStepLanes) * 4 + j;
        float k_sum = 0.f, q_sum = 0.f;
#pragma unroll
        for (int w = 0; w < kStepThreads / 64; ++w) {
            k_sum += part[0][w][col];
            q_sum += part[1][w][col];
        }
        add[j] = beta * (widen(v_in[j]) - decay * k_sum);
        out[j] = a.scale * (decay * q_sum + kq_all * add[j]);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const float kr = ks[r0 + i];
        f32x4 n;
#pragma unroll
        for (int j = 0; j < 4; ++j) n[j] = decay * s[i][j] + kr * add[j];
        if (!whole && r0 + i >= a.Dk) continue;
        float* p = a.state_out + base + (row0 + i * static_cast<uint32_t>(a.Dv) + c);
        if (WIDE) {
            if (c < a.Dv) __builtin_nontemporal_store(n, reinterpret_cast<f32x4*>(p));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < a.Dv) p[j] = n[j];
        }
    }
    if (threadIdx.x < kStepLanes) {
        E* o = static_cast<E*>(a.o) + static_cast<int64_t>(head) * a.Dv + c;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < a.Dv) o[j] = narrow<E>(out[j]);
    }
}

template <typename E>
hipError_t step_as(const StepArgs& a, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(ceil_div(a.Dv, kStepCols)), static_cast<unsigned>(a.B * a.Hv));
    const bool wide = a.Dv % 4 == 0 && aligned_to(a.state, 16) && aligned_to(a.state_out, 16);
    // the rows a thread holds cost registers and, where the head has fewer, loads that do nothing
    if (a.Dk <= 64)
        return wide ? launch(delta_step_kernel<E, 64 / kStepRows, true>, grid, dim3(kStepThreads), st, a)
                    : launch(delta_step_kernel<E, 64 / kStepRows, false>, grid, dim3(kStepThreads), st, a);
    return wide ? launch(delta_step_kernel<E, 128 / kStepRows, true>, grid, dim3(kStepThreads), st, a)
                : launch(delta_step_kernel<E, 128 / kStepRows, false>, grid, dim3(kStepThreads), st, a);
}

// ---- arguments ----------------------------------------------------------------------------------

int delta_error(const snnseq_delta* c) {
    if (c == nullptr) return SNNLIF_ERR_ARG;
    if (c->dtype == SNNLIF_DTYPE_F64) return SNNLIF_ERR_UNSUPPORTED;
    if (element_size(c->dtype) == 0) return SNNLIF_ERR_DTYPE;
    if (c->T < 0 || c->B < 0 || c->Hk < 1 || c->Hv < 1 || c->Hv % c->Hk != 0) return SNNLIF_ERR_ARG;
    if (c->T > SNNSEQ_MAX_TOKENS || c->Dk < 1 || c->Dk > SNNSEQ_MAX_KEY || c->Dv < 1 || c->Dv > SNNSEQ_MAX_VALUE)
        return SNNLIF_ERR_ARG;
    if (c->Hv > SNNSEQ_MAX_HEADS || c->B > SNNSEQ_MAX_HEADS / c->Hv) return SNNLIF_ERR_ARG;  // B * Hv is a grid size
    return SNNLIF_OK;
}

// The passes over the chunks launch a workgroup of 256 per head and 16 columns: what a launch can hold.
int chunked_error(const snnseq_delta* c) {
    const int bad = delta_error(c);
    if (bad != SNNLIF_OK) return bad;
    return c->B * c->Hv * ceil_div(c->Dv, kCols) * (kCols / kStateCols) > SNNSEQ_MAX_TOKENS ? SNNLIF_ERR_ARG : SNNLIF_OK;
}

bool empty(const snnseq_delta* c) { return c->B == 0; }

int missing(const snnseq_delta* c) {
    if (c->T > 0 && (c->q == nullptr || c->k == nullptr || c->v == nullptr || c->g == nullptr || c->beta == nullptr))
        return SNNLIF_ERR_ARG;
    const size_t es = element_size(c->dtype);
    if (!aligned_to(c->q, es) || !aligned_to(c->k, es) || !aligned_to(c->v, es) || !aligned_to(c->g, 4) ||
        !aligned_to(c->beta, 4) || !aligned_to(c->state, 4) || !aligned_to(c->lengths, 4))
        return SNNLIF_ERR_ALIGN;
    return SNNLIF_OK;
}

DeltaTensor tensor_of(const void* p, const int64_t* strides, int64_t D) {
    DeltaTensor x{p, strides[0], strides[1], strides[2], 0};
    x.wide = D % 8 == 0;
    return x;
}

struct Sizes {
    int64_t pieces, heads, chunks, cols, dkp;
    size_t decay, inverse, keys, added, states;  // bytes of what the forward leaves behind (inverse and keys: twice)
    size_t scores;                               // of a forward that leaves nothing behind
    size_t inner, state_grads, queries, partial; // of the backward's
    size_t saved, workspace;                     // in all
};

Sizes sizes_of(const snnseq_delta* c, bool for_backward) {
    Sizes s;
    s.chunks = ceil_div(c->T, kChunk);
    s.heads = c->B * c->Hv;
    s.pieces = s.chunks * s.heads;
    s.cols = ceil_div(c->Dv, kCols) * kCols;
    s.dkp = c->Dk <= 64 ? 64 : 128;
    const size_t n = static_cast<size_t>(s.pieces) * sizeof(float);
    s.decay = static_cast<size_t>(s.pieces) * sizeof(Decay);
    const bool f32 = c->dtype == SNNLIF_DTYPE_F32;
    s.inverse = static_cast<size_t>(s.pieces) * (f32 ? square_bytes<float>() : square_bytes<bf16_t>());
    s.keys = s.queries = static_cast<size_t>(c->B * c->Hk * s.chunks) *
                         (f32 ? keys_bytes<float>(static_cast<int>(s.dkp)) : keys_bytes<bf16_t>(static_cast<int>(s.dkp)));
    s.added = s.inner = n * kChunk * static_cast<size_t>(s.cols);
    s.states = s.state_grads = n * static_cast<size_t>(s.dkp * s.cols);
    s.partial = c->Hv == c->Hk ? 0 : round_up(static_cast<size_t>(c->T * s.heads * c->Dk) * sizeof(float), 16);
    s.scores = static_cast<size_t>(s.pieces) * (f32 ? square_bytes<float>() : square_bytes<bf16_t>());
    s.saved = s.decay + s.inverse + 2 * s.keys + (for_backward ? s.inverse + s.added + s.states : s.queries + s.scores);
    s.workspace = s.inner + s.state_grads + s.queries + 2 * s.partial;
    return s;
}

DeltaArgs args_of(const snnseq_delta* c, const Sizes& s, void* saved, bool for_backward) {
    const size_t es = element_size(c->dtype);
    DeltaArgs a{};
    a.T = static_cast<int>(c->T); a.B = static_cast<int>(c->B);
    a.Hk = static_cast<int>(c->Hk); a.Hv = static_cast<int>(c->Hv);
    a.Dk = static_cast<int>(c->Dk); a.Dv = static_cast<int>(c->Dv);
    a.chunks = static_cast<int>(s.chunks); a.cols = static_cast<int>(s.cols);
    a.scale = static_cast<float>(c->scale);
    a.lengths = c->lengths;
    a.q = tensor_of(c->q, c->q_strides, c->Dk);
    a.k = tensor_of(c->k, c->k_strides, c->Dk);
    a.v = tensor_of(c->v, c->v_strides, c->Dv);
    a.g = c->g; a.beta = c->beta; a.state = c->state;
    char* p = static_cast<char*>(saved);
    a.decay = reinterpret_cast<Decay*>(p);
    a.inverse = p + s.decay;
    a.keys = a.inverse + s.inverse;
    a.keys_t = a.keys + s.keys;
    char* rest = a.keys_t + s.keys;
    if (for_backward) {
        a.inverse_t = rest;
        a.added = reinterpret_cast<float*>(rest + s.inverse);
        a.states = reinterpret_cast<float*>(rest + s.inverse + s.added);
    } else {
        a.queries = rest;
        a.scores = rest + s.queries;
    }
    return a;
}

}  // namespace
}  // namespace snnseq

using namespace snnseq;

extern "C" size_t snnseq_gated_delta_saved_bytes(const snnseq_delta* call, int for_backward) {
    if (chunked_error(call) != SNNLIF_OK || empty(call)) return 0;
    return sizes_of(call, for_backward != 0).saved;
}

extern "C" int snnseq_gated_delta_fp(const snnseq_delta* call, void* o, float* state_out, void* saved,
                                     size_t saved_bytes, int for_backward, void* stream) {
    const int bad = chunked_error(call);
    if (bad != SNNLIF_OK) return bad;
    if (empty(call)) return SNNLIF_OK;
    const int lost = missing(call);
    if (lost != SNNLIF_OK) return lost;
    if (call->T > 0 && o == nullptr) return SNNLIF_ERR_ARG;
    if (!aligned_to(o, element_size(call->dtype)) || !aligned_to(state_out, 4) || !aligned_to(saved, 16))
        return SNNLIF_ERR_ALIGN;
    const Sizes s = sizes_of(call, for_backward != 0);
    if (s.pieces > 0 && (saved == nullptr || saved_bytes < s.saved)) return SNNLIF_ERR_WORKSPACE;
    DeltaArgs a = args_of(call, s, saved, for_backward != 0);
    a.o = o;
    a.state_out = state_out;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return static_cast<int>(call->dtype == SNNLIF_DTYPE_F32 ? delta_forward_f32(a, st) : delta_forward_bf16(a, st));
}

extern "C" size_t snnseq_gated_delta_bp_workspace_bytes(const snnseq_delta* call) {
    if (chunked_error(call) != SNNLIF_OK || empty(call)) return 0;
    return sizes_of(call, true).workspace;
}

extern "C" int snnseq_gated_delta_bp(const snnseq_delta* call, const void* saved, size_t saved_bytes,
                                     const void* grad_o, const int64_t* grad_o_strides, const float* grad_state_out,
                                     void* grad_q, void* grad_k, void* grad_v, float* grad_g, float* grad_beta,
                                     float* grad_state, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = chunked_error(call);
    if (bad != SNNLIF_OK) return bad;
    if (empty(call)) return SNNLIF_OK;
    const int lost = missing(call);
    if (lost != SNNLIF_OK) return lost;
    if (grad_o_strides == nullptr) return SNNLIF_ERR_ARG;
    if (call->T > 0 && (grad_o == nullptr || grad_q == nullptr || grad_k == nullptr || grad_v == nullptr ||
                        grad_g == nullptr || grad_beta == nullptr))
        return SNNLIF_ERR_ARG;
    const size_t es = element_size(call->dtype);
    if (!aligned_to(grad_o, es) || !aligned_to(grad_q, es) || !aligned_to(grad_k, es) || !aligned_to(grad_v, es) ||
        !aligned_to(grad_g, 4) || !aligned_to(grad_beta, 4) || !aligned_to(grad_state, 4) ||
        !aligned_to(grad_state_out, 4) || !aligned_to(saved, 16) || !aligned_to(workspace, 16))
        return SNNLIF_ERR_ALIGN;
    const Sizes s = sizes_of(call, true);
    if (s.pieces > 0 && (saved == nullptr || saved_bytes < s.saved || workspace == nullptr ||
                         workspace_bytes < s.workspace))
        return SNNLIF_ERR_WORKSPACE;
    DeltaArgs a = args_of(call, s, const_cast<void*>(saved), true);
    char* p = static_cast<char*>(workspace);
    a.grad_o = tensor_of(grad_o, grad_o_strides, call->Dv);
    a.grad_state = grad_state_out;
    a.inner = reinterpret_cast<float*>(p);
    a.state_grads = reinterpret_cast<float*>(p + s.inner);
    a.queries_t = p + s.inner + s.state_grads;
    a.grad_q = s.partial ? a.queries_t + s.queries : grad_q;
    a.grad_k = s.partial ? a.queries_t + s.queries + s.partial : grad_k;
    a.grad_v = grad_v;
    a.grad_g = grad_g;
    a.grad_beta = grad_beta;
    a.grad_initial = grad_state;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return static_cast<int>(call->dtype == SNNLIF_DTYPE_F32 ? delta_backward_f32(a, grad_q, grad_k, st)
                                                            : delta_backward_bf16(a, grad_q, grad_k, st));
}

extern "C" int snnseq_gated_delta_step(const snnseq_delta* call, void* o, float* state_out, void* stream) {
    const int bad = delta_error(call);
    if (bad != SNNLIF_OK) return bad;
    if (call->T != 1 || call->lengths != nullptr) return SNNLIF_ERR_ARG;
    if (empty(call)) return SNNLIF_OK;
    const int lost = missing(call);
    if (lost != SNNLIF_OK) return lost;
    if (call->state == nullptr || state_out == nullptr || o == nullptr) return SNNLIF_ERR_ARG;
    if (!aligned_to(o, element_size(call->dtype)) || !aligned_to(state_out, 4)) return SNNLIF_ERR_ALIGN;
    StepArgs a{};
    a.B = static_cast<int>(call->B); a.Hk = static_cast<int>(call->Hk); a.Hv = static_cast<int>(call->Hv);
    a.Dk = static_cast<int>(call->Dk); a.Dv = static_cast<int>(call->Dv);
    a.scale = static_cast<float>(call->scale);
    a.q = call->q; a.q_b = call->q_strides[1]; a.q_h = call->q_strides[2];
    a.k = call->k; a.k_b = call->k_strides[1]; a.k_h = call->k_strides[2];
    a.v = call->v; a.v_b = call->v_strides[1]; a.v_h = call->v_strides[2];
    a.g = call->g; a.beta = call->beta; a.state = call->state;
    a.o = o;
    a.state_out = state_out;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return static_cast<int>(call->dtype == SNNLIF_DTYPE_F32 ? step_as<float>(a, st) : step_as<bf16_t>(a, st));
}
