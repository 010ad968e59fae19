// Element types of the operators that take 32- and 16-bit floats: conversions to and from fp32 and accesses of several
// consecutive elements at once.
#pragma once

#include "cn_internal.h"

namespace cn {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

template <typename T, int N>
struct Pack {
    typedef T type __attribute__((ext_vector_type(N)));
};
template <typename T>
struct Pack<T, 1> {
    typedef T type;
};

// N consecutive elements at p (aligned to N elements) as fp32: exact.
template <int N, typename T>
__device__ __forceinline__ void load_f32(const T *p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = (float)*p;
    } else {
        const auto w = *reinterpret_cast<const typename Pack<T, N>::type *>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)w[i];
    }
}
// fp32 to N consecutive elements, each rounded to nearest even once.  STREAM: past the caches, for what is not read again soon.
template <int N, bool STREAM = false, typename T>
__device__ __forceinline__ void store_f32(T *p, const float (&v)[N]) {
    typename Pack<T, N>::type w;
    if constexpr (N == 1) {
        w = (T)v[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = (T)v[i];
    }
    if constexpr (STREAM && N > 1) __builtin_nontemporal_store(w, reinterpret_cast<typename Pack<T, N>::type *>(p));
    else *reinterpret_cast<typename Pack<T, N>::type *>(p) = w;
}

inline bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline size_t dtype_bytes(int dtype) { return dtype == CN_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == CN_F32 || dtype == CN_F16 || dtype == CN_BF16; }

// A launch has fewer than 2^32 work items in x and 2^16 workgroups in y.
inline bool launchable(int64_t blocks, int threads, int64_t slabs = 1) { return blocks <= 0xffffffffLL / threads && slabs <= 65535; }

// Device memory a caller hands over, dealt out in 256-byte steps.
struct Carver {
    char *base;
    size_t used = 0;
    explicit Carver(void *p) : base(static_cast<char *>(p)) {}
    template <typename T>
    T *take(size_t n) {
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += (n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

}  // namespace cn
