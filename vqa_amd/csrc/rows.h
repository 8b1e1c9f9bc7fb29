// What the row operators (logprob.hip, sample.hip, dropout.hip) share: element types, 16-byte accesses, reductions over a
// wave.
#pragma once
#include "vqa_dev.h"
#include "plan.h"
#include <string>

#define ROWS_CHECK_LAUNCH(name)                                                               \
    do {                                                                                      \
        hipError_t e_ = hipGetLastError();                                                    \
        if (e_ != hipSuccess) {                                                               \
            vqa_set_error(std::string(name ": ") + hipGetErrorString(e_));                    \
            return VQA_ELAUNCH;                                                               \
        }                                                                                     \
    } while (0)

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// rows of an odd length start at any element: 16-byte accesses that promise 2-byte alignment only (the hardware takes them
// at any address; a wave's contiguous kilobyte then touches one more cache line)
typedef u32x4 u32x4u __attribute__((aligned(2)));

// DT: VQA_BF16, VQA_F16 or VQA_F32
template <int DT> struct Elem {
    typedef uint16_t type;
    static constexpr int N = 8;                       // elements in 16 bytes
};
template <> struct Elem<VQA_F32> {
    typedef float type;
    static constexpr int N = 4;
};

template <int DT> __device__ __forceinline__ float elem_get(const typename Elem<DT>::type* p) {
    if constexpr (DT == VQA_BF16) return bf2f(*p);
    else if constexpr (DT == VQA_F16) return (float)__builtin_bit_cast(_Float16, *p);
    else return *p;
}
template <int DT> __device__ __forceinline__ void elem_put(typename Elem<DT>::type* p, float v) {
    if constexpr (DT == VQA_BF16) *p = f2bf(v);
    else if constexpr (DT == VQA_F16) *p = __builtin_bit_cast(uint16_t, (_Float16)v);
    else *p = v;
}
template <int DT> __device__ __forceinline__ u32x4 vec_load(const typename Elem<DT>::type* p) {
    return *(const u32x4u*)p;
}
// NT: past the last-level cache, for what will not be there any more when it is read again
template <int DT, bool NT> __device__ __forceinline__ u32x4 vec_load_as(const typename Elem<DT>::type* p) {
    if constexpr (NT) return __builtin_nontemporal_load((const u32x4u*)p);
    else return *(const u32x4u*)p;
}
template <int DT, bool NT> __device__ __forceinline__ void vec_store_as(typename Elem<DT>::type* p, u32x4 v) {
    if constexpr (NT) __builtin_nontemporal_store(v, (u32x4u*)p);
    else *(u32x4u*)p = v;
}
template <int DT> __device__ __forceinline__ void vec_store(typename Elem<DT>::type* p, u32x4 v) { *(u32x4u*)p = v; }
// element i of a 16-byte piece as a float
template <int DT> __device__ __forceinline__ float vec_get(u32x4 v, int i) {
    if constexpr (DT == VQA_BF16) return __uint_as_float((i & 1) ? (v[i >> 1] & 0xFFFF0000u) : (v[i >> 1] << 16));
    else if constexpr (DT == VQA_F16)
        return (float)__builtin_bit_cast(_Float16, (uint16_t)((i & 1) ? (v[i >> 1] >> 16) : (v[i >> 1] & 0xFFFFu)));
    else return __uint_as_float(v[i]);
}
// a 16-byte piece from floats, one rounding (to nearest, ties to even) each
template <int DT> __device__ __forceinline__ u32x4 vec_make(const float* f) {
    u32x4 v;
    if constexpr (DT == VQA_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == VQA_BF16) v[i] = cvt_pk_bf16((f32x2){f[2 * i], f[2 * i + 1]});
            else v[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i]) |
                        ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i + 1]) << 16);
        }
    }
    return v;
}

// waits until what this wave has stored (and loaded) before has arrived, atomic stores at the scope that they were made for
__device__ __forceinline__ void wait_for_stores() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

static inline bool rows_dtype_ok(int32_t dt) { return dt == VQA_BF16 || dt == VQA_F16 || dt == VQA_F32; }
