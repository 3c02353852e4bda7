// Shared pieces of the token-layer kernels (embedding, group norm, gated delta rule) for MI355X:
// storage types, vectors of a few bytes, launches that report their own error.
//
// Unlike the fire kernels, which reproduce separately rounded products and sums bit for bit, these
// operators have no bit pattern to match: products and sums contract to fused multiply-adds.
#ifndef SNNLIF_SEQ_COMMON_H
#define SNNLIF_SEQ_COMMON_H

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "snnlib_seq.h"

#pragma clang fp contract(fast)

namespace snnseq {

struct bf16_t {
    uint16_t bits;
};

// Storage type -> type its values are computed in, and the conversions (round to nearest even).
template <typename E> struct Arith { using type = float; };
template <> struct Arith<double> { using type = double; };
template <typename E> using arith_t = typename Arith<E>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(bf16_t v) {
    return __builtin_bit_cast(float, static_cast<uint32_t>(v.bits) << 16);
}

template <typename E> __device__ __forceinline__ E narrow(arith_t<E> v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ double narrow<double>(double v) { return v; }
template <> __device__ __forceinline__ bf16_t narrow<bf16_t>(float v) {
    const __bf16 r = static_cast<__bf16>(v);
    return bf16_t{__builtin_bit_cast(uint16_t, r)};
}

// BYTES consecutive bytes of storage type E, moved with one memory instruction, from any element on.
template <int BYTES> struct RawOf;
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint32_t __attribute__((ext_vector_type(2))); };
template <> struct RawOf<16> { using type = uint32_t __attribute__((ext_vector_type(4))); };

template <typename E, int BYTES>
struct Vec {
    static constexpr int n = BYTES / static_cast<int>(sizeof(E));
    using raw_t = typename RawOf<BYTES>::type;
    using memory_t = raw_t __attribute__((aligned(sizeof(E))));
    union {
        raw_t raw;
        E e[n];
    };
};

template <typename E, int BYTES>
__device__ __forceinline__ Vec<E, BYTES> load_vec(const E* p) {
    Vec<E, BYTES> v;
    v.raw = *reinterpret_cast<const typename Vec<E, BYTES>::memory_t*>(p);
    return v;
}

// Read once (or written for somebody else): the non-temporal hint keeps it from displacing what is read again.
template <typename E, int BYTES>
__device__ __forceinline__ Vec<E, BYTES> load_vec_once(const E* p) {
    Vec<E, BYTES> v;
    v.raw = __builtin_nontemporal_load(reinterpret_cast<const typename Vec<E, BYTES>::memory_t*>(p));
    return v;
}

// The vector at p[at], zero where it is absent; p[0] has to be there all the same.  Loads of two bytes go into half
// of a register, which the compiler waits for at the end of a condition, and it has put waits between conditional loads
// of four: narrow ones are under none.
template <typename E, int BYTES, typename I>
__device__ __forceinline__ Vec<E, BYTES> load_or_zero(const E* p, I at, bool present, bool once) {
    using raw_t = typename Vec<E, BYTES>::raw_t;
    Vec<E, BYTES> v;
    if constexpr (BYTES > 4) {
        v.raw = raw_t(0);
        if (present) v = once ? load_vec_once<E, BYTES>(p + at) : load_vec<E, BYTES>(p + at);
    } else {
        v = load_vec<E, BYTES>(p + (present ? at : I(0)));
        v.raw = present ? v.raw : raw_t(0);
    }
    return v;
}

template <typename E, int BYTES>
__device__ __forceinline__ void store_vec(E* p, const Vec<E, BYTES>& v) {
    *reinterpret_cast<typename Vec<E, BYTES>::memory_t*>(p) = v.raw;
}

template <typename E, int BYTES>
__device__ __forceinline__ void store_vec_once(E* p, const Vec<E, BYTES>& v) {
    __builtin_nontemporal_store(v.raw, reinterpret_cast<typename Vec<E, BYTES>::memory_t*>(p));
}

// Bytes of the widest vector that `count` elements hold.  Rows and groups of any size are covered by such vectors: the
// last begins where it ends with them, and shares elements with the one before.
inline int widest_vector(int64_t count, size_t element_bytes) {
    int bytes = 16;
    while (bytes > count * static_cast<int64_t>(element_bytes)) bytes /= 2;
    return bytes;
}

inline uint64_t address(const void* p) { return reinterpret_cast<uint64_t>(p); }
inline bool aligned_to(const void* p, size_t bytes) { return address(p) % bytes == 0; }

inline size_t element_size(int dtype) {
    switch (dtype) {
        case SNNLIF_DTYPE_F32: return 4;
        case SNNLIF_DTYPE_F64: return 8;
        case SNNLIF_DTYPE_BF16: return 2;
        default: return 0;
    }
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t round_up(size_t n, size_t to) { return (n + to - 1) / to * to; }

// Launches and returns this launch's own error (an error some earlier call left behind stays there).
template <typename... P, typename... A>
inline hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, A... args) {
    struct Slots {
        static hipError_t run(void (*k)(P...), dim3 g, dim3 b, hipStream_t s, P... p) {
            void* pointers[] = {const_cast<void*>(static_cast<const void*>(&p))...};
            return hipLaunchKernel(reinterpret_cast<const void*>(k), g, b, pointers, 0, s);
        }
    };
    return Slots::run(kernel, grid, block, stream, static_cast<P>(args)...);
}

}  // namespace snnseq

#endif  // SNNLIF_SEQ_COMMON_H
