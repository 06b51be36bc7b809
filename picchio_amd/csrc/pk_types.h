// pk_types.h — the element types of activations and paged caches (PK_T_*), for
// the kernels and their launchers.
#pragma once

#include "pk_dev.h"

inline int pk_type_size(int t) { return t == PK_T_F32 ? 4 : t == PK_T_F16 || t == PK_T_BF16 ? 2 : 0; }

typedef _Float16 pk_f16;
typedef __bf16 pk_bf16;
typedef pk_f16 pk_f16x8 __attribute__((ext_vector_type(8)));
typedef pk_bf16 pk_bf16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct pk_vec8;
template <> struct pk_vec8<pk_f16> { typedef pk_f16x8 type; };
template <> struct pk_vec8<pk_bf16> { typedef pk_bf16x8 type; };

// Eight neighbouring elements (16-byte aligned) to and from fp32; conversions
// to 16 bits round to nearest even, once.
template <typename T>
__device__ __forceinline__ void pk_load8(const T *p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const pk_f32x4 a = reinterpret_cast<const pk_f32x4 *>(p)[0], b = reinterpret_cast<const pk_f32x4 *>(p)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
        const auto a = *reinterpret_cast<const typename pk_vec8<T>::type *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
}
template <typename T>
__device__ __forceinline__ void pk_store8(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<pk_f32x4 *>(p)[0] = pk_f32x4{v[0], v[1], v[2], v[3]};
        reinterpret_cast<pk_f32x4 *>(p)[1] = pk_f32x4{v[4], v[5], v[6], v[7]};
    } else {
        typename pk_vec8<T>::type a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
        *reinterpret_cast<typename pk_vec8<T>::type *>(p) = a;
    }
}

// Calls f(activation type, cache type) for the pairs that the paged operators take:
// equal types, or fp32 activations over any cache.
#define PK_BY_TYPES(act, cache, CALL)                                                   \
    do {                                                                                \
        if ((act) == PK_T_F16) CALL(pk_f16, pk_f16);                                    \
        else if ((act) == PK_T_BF16) CALL(pk_bf16, pk_bf16);                            \
        else if ((cache) == PK_T_F32) CALL(float, float);                               \
        else if ((cache) == PK_T_F16) CALL(float, pk_f16);                              \
        else CALL(float, pk_bf16);                                                      \
    } while (0)

// The device of an engine for the length of a call: kernels go to the engine's
// stream whatever device the caller has current.
struct pk_device_scope {
    int cur = -1, rc = PK_OK;
    explicit pk_device_scope(int device);
    ~pk_device_scope();
};

// The checks that the paged operators share.
int pk_check_pages(const pk_pages &p, int act_type);
int pk_check_rows(const void *p, int64_t stride, int heads, int hd, const char *what);
