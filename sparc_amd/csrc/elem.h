// Element types of the table lookup and the gradient norm: 16-byte vectors of float, bfloat16 or half in memory, float32
// in registers.  Rows and views may start at any element, so the vectors carry the alignment of one element (global
// memory instructions take any address).
#pragma once
#include "common.h"

// What the 256 MB Infinity Cache is left to keep from one pass over the data to the next.
constexpr int64_t SPARC_KEEP_BYTES = 192000000;

template <int DT>
struct Elem;
template <>
struct Elem<SPARC_F32> {
    typedef float type;
    static __device__ __forceinline__ float up(const float x) { return x; }
    static __device__ __forceinline__ float down(const float x) { return x; }
};
template <>
struct Elem<SPARC_BF16> {
    typedef __bf16 type;
    static __device__ __forceinline__ float up(const __bf16 x) { return static_cast<float>(x); }
    static __device__ __forceinline__ __bf16 down(const float x) { return static_cast<__bf16>(x); }   // to nearest even
};
template <>
struct Elem<SPARC_F16> {
    typedef _Float16 type;
    static __device__ __forceinline__ float up(const _Float16 x) { return static_cast<float>(x); }
    static __device__ __forceinline__ _Float16 down(const float x) { return static_cast<_Float16>(x); }
};

// VE consecutive elements: one memory instruction each way when VE fills 16 bytes.
template <int DT, int VE>
struct Vec {
    typedef typename Elem<DT>::type T;
    typedef T mem __attribute__((ext_vector_type(VE), aligned(sizeof(T))));
    mem v;
    // STREAM: nontemporal.  A template parameter, because the compiler merges two branches that differ in nothing else.
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (STREAM) v = __builtin_nontemporal_load(reinterpret_cast<const mem*>(p));
        else v = *reinterpret_cast<const mem*>(p);
    }
    template <bool STREAM = false>
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<mem*>(p));
        else *reinterpret_cast<mem*>(p) = v;
    }
    __device__ __forceinline__ float get(const int i) const { return Elem<DT>::up(v[i]); }
    __device__ __forceinline__ void set(const int i, const float x) { v[i] = Elem<DT>::down(x); }
};
template <int DT>
struct Vec<DT, 1> {
    typedef typename Elem<DT>::type T;
    T v;
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (STREAM) v = __builtin_nontemporal_load(p);
        else v = *p;
    }
    template <bool STREAM = false>
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (STREAM) __builtin_nontemporal_store(v, p);
        else *p = v;
    }
    __device__ __forceinline__ float get(int) const { return Elem<DT>::up(v); }
    __device__ __forceinline__ void set(int, const float x) { v = Elem<DT>::down(x); }
};
