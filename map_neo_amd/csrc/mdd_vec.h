// Shared by the document-vector kernels (mdd_vec.hip, mdd_mx.hip): element types, eight-element loads and stores, wave sums.
#ifndef MDD_VEC_H
#define MDD_VEC_H

#include "mdd_common.h"

namespace mddi {

// Restores the caller's current device: the entry points below switch to the context's GPU and must leave no trace of it.
struct DeviceGuard {
    int prev = -1;
    hipError_t err;
    explicit DeviceGuard(int dev) {
        err = hipGetDevice(&prev);
        if (err == hipSuccess && prev != dev) err = hipSetDevice(dev);
        else prev = -1;
    }
    ~DeviceGuard() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};
#define ON_DEVICE(ctx)                     \
    mddi::DeviceGuard guard_((ctx)->device); \
    if (guard_.err != hipSuccess) return mddi::fail(MDD_ERR_HIP, "selecting device %d failed: %s", (ctx)->device, hipGetErrorString(guard_.err))

inline bool aligned_to(const void* p, uint64_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline uint64_t round_up(uint64_t x, uint64_t m) { return (x + m - 1) / m * m; }
inline uint32_t type_bytes(int t) { return t == MDD_F32 ? 4u : (t == MDD_BF16 || t == MDD_F16) ? 2u : 0u; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Rows start where the caller's stride puts them, so an eight-element access may begin at any element: gfx950 serves
// 16-byte accesses at any byte address (unaligned access mode), and only a row's last 1..7 elements go one by one.
template <typename T>
struct vec8;
template <>
struct vec8<float> {
    typedef float raw __attribute__((ext_vector_type(8)));
    typedef float raw_any __attribute__((ext_vector_type(8), aligned(4)));
};
template <>
struct vec8<__bf16> {
    typedef __bf16 raw __attribute__((ext_vector_type(8)));
    typedef __bf16 raw_any __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct vec8<_Float16> {
    typedef _Float16 raw __attribute__((ext_vector_type(8)));
    typedef _Float16 raw_any __attribute__((ext_vector_type(8), aligned(2)));
};

template <typename T>
__device__ __forceinline__ typename vec8<T>::raw load8_raw(const T* __restrict__ p, uint32_t n) {
    typename vec8<T>::raw v;
    if (n >= 8) {
        v = *reinterpret_cast<const typename vec8<T>::raw_any*>(p);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) v[k] = k < n ? p[k] : (T)0.0f;
    }
    return v;
}
template <typename T>
__device__ __forceinline__ f32x8 load8(const T* __restrict__ p, uint32_t n) {
    return __builtin_convertvector(load8_raw<T>(p, n), f32x8);
}
// each element is rounded once, to the nearest (ties to even)
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, uint32_t n, f32x8 v) {
    typename vec8<T>::raw r = __builtin_convertvector(v, typename vec8<T>::raw);
    if (n >= 8) {
        *reinterpret_cast<typename vec8<T>::raw_any*>(p) = r;
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 8; k++)
            if (k < n) p[k] = r[k];
    }
}

// for data that is written once and whole: past the caches, which keep what is used again
template <typename T>
__device__ __forceinline__ void store8_once(T* __restrict__ p, uint32_t n, f32x8 v) {
    if (n >= 8) {
        typename vec8<T>::raw r = __builtin_convertvector(v, typename vec8<T>::raw);
        __builtin_nontemporal_store(r, reinterpret_cast<typename vec8<T>::raw_any*>(p));
    } else {
        store8<T>(p, n, v);
    }
}

// What a call moves beyond the last-level cache goes past it (ONCE): below that the next kernel finds it there
constexpr uint64_t LAST_LEVEL = 256u << 20;
template <typename T, bool ONCE>
__device__ __forceinline__ void store8_or_once(T* __restrict__ p, uint32_t n, f32x8 v) {
    if constexpr (ONCE) store8_once<T>(p, n, v);
    else store8<T>(p, n, v);
}

// Blocks go to the eight XCDs in turn: place of block b of n in a list of which each XCD then takes a run of neighbours
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t n) {
    const uint32_t per = n / 8;  // the last n % 8 keep their place
    return b < per * 8 ? (b % 8) * per + b / 8 : b;
}

// runs body(T()) for the element type `t`
#define MDD_FOR_TYPE(t, T, ...)                                   \
    do {                                                          \
        if ((t) == MDD_F32) {                                     \
            typedef float T;                                      \
            __VA_ARGS__;                                          \
        } else if ((t) == MDD_BF16) {                             \
            typedef __bf16 T;                                     \
            __VA_ARGS__;                                          \
        } else {                                                  \
            typedef _Float16 T;                                   \
            __VA_ARGS__;                                          \
        }                                                         \
    } while (0)

}  // namespace mddi
#endif  // MDD_VEC_H
