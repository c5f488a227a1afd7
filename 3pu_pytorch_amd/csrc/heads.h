// heads.h -- what the kernels over attention heads share (norm_rotate.hip, block_select.hip, block_attn.hip): element
// types, eight-channel loads and stores of a row, checks of a tpu3_heads argument.
#pragma once
#include "tpu3_dev.h"

typedef float hd_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 hd_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 hd_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 hd_bf4 __attribute__((ext_vector_type(4)));
typedef _Float16 hd_h4 __attribute__((ext_vector_type(4)));
struct __attribute__((aligned(16))) hd_f8 {
    float v[8];
    __device__ __forceinline__ float operator[](int i) const { return v[i]; }
};

// eight consecutive channels of a row: one 16-byte access for the 16-bit types, two for fp32
template <typename T> struct hd_vec;
template <> struct hd_vec<__bf16> { typedef hd_bf8 v8; typedef hd_bf4 v4; };
template <> struct hd_vec<_Float16> { typedef hd_h8 v8; typedef hd_h4 v4; };
template <> struct hd_vec<float> { typedef hd_f8 v8; typedef hd_f4 v4; };

template <typename T> __device__ __forceinline__ void hd_load8(const T *p, float *x)
{
    const typename hd_vec<T>::v8 v = *(const typename hd_vec<T>::v8 *)p;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = (float)v[i];
}
template <typename T> __device__ __forceinline__ void hd_store8(T *p, const float *x)
{
    typename hd_vec<T>::v8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = (T)x[i];                     // one rounding to nearest even, the only one on the way to memory
    *(typename hd_vec<T>::v8 *)p = v;
}
template <> __device__ __forceinline__ void hd_store8<float>(float *p, const float *x)
{
    *(hd_f4 *)p = hd_f4{x[0], x[1], x[2], x[3]};
    *(hd_f4 *)(p + 4) = hd_f4{x[4], x[5], x[6], x[7]};
}

// the same, past the caches
template <typename T> __device__ __forceinline__ void hd_stream8(T *p, const float *x)
{
    if constexpr (sizeof(T) == 4) {
        __builtin_nontemporal_store(hd_f4{x[0], x[1], x[2], x[3]}, (hd_f4 *)p);
        __builtin_nontemporal_store(hd_f4{x[4], x[5], x[6], x[7]}, (hd_f4 *)(p + 4));
    } else {
        typename hd_vec<T>::v8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = (T)x[i];
        __builtin_nontemporal_store(v, (typename hd_vec<T>::v8 *)p);
    }
}

static inline int hd_type_size(int type) { return type == TPU3_TYPE_F32 ? 4 : 2; }
static inline bool hd_type_ok(int type) { return type == TPU3_TYPE_F32 || type == TPU3_TYPE_F16 || type == TPU3_TYPE_BF16; }
// a (b, rows, heads, d) argument: every row of d channels starts on 16 bytes
static inline bool hd_rows_ok(const tpu3_heads *t, int type)
{
    const int64_t per = 16 / hd_type_size(type);
    return t && t->data && t->heads > 0 && ((uintptr_t)t->data & 15) == 0 && t->sb % per == 0 && t->sr % per == 0 &&
           t->sh % per == 0;
}
