// Element types of the training operators (float32, bfloat16, float16): 128-bit loads and stores of
// eight or four elements, conversion to float32, in which everything is computed.  A result is rounded
// to its type once, to nearest even, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace tpb {

template <class T> struct Elem;

template <> struct Elem<float> {
    static constexpr int N = 4;   // elements of a 16-byte vector
    static constexpr uint32_t kNegInf = 0xff800000u;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
    static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
        f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};

template <> struct Elem<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr uint32_t kNegInf = 0xff80u;
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
    // a bfloat16 is the upper half of a float32
    static __device__ __forceinline__ void two(uint32_t w, float* f) {
        f[0] = __uint_as_float(w << 16);
        f[1] = __uint_as_float(w & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t both(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        uint32_t w;
        memcpy(&w, &v, 4);
        return w;
    }
    static __device__ __forceinline__ void unpack(const uint4& v, float* f) { two(v.x, f); two(v.y, f + 2); two(v.z, f + 4); two(v.w, f + 6); }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return make_uint4(both(f[0], f[1]), both(f[2], f[3]), both(f[4], f[5]), both(f[6], f[7]));
    }
};

template <> struct Elem<__half> {
    static constexpr int N = 8;
    static constexpr uint32_t kNegInf = 0xfc00u;
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ void two(uint32_t w, float* f) {
        __half2 v;
        memcpy(&v, &w, 4);
        const float2 r = __half22float2(v);
        f[0] = r.x;
        f[1] = r.y;
    }
    static __device__ __forceinline__ uint32_t both(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        uint32_t w;
        memcpy(&w, &v, 4);
        return w;
    }
    static __device__ __forceinline__ void unpack(const uint4& v, float* f) { two(v.x, f); two(v.y, f + 2); two(v.z, f + 4); two(v.w, f + 6); }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return make_uint4(both(f[0], f[1]), both(f[2], f[3]), both(f[4], f[5]), both(f[6], f[7]));
    }
};

// 16-byte loads and stores with a place in L2's order of eviction.  Streams go first: what is read or written
// once must not push out what is read again (the logits between two sweeps, the rows of a neighbouring
// kernel).  Measured on the gradient of [4096,50016] bf16 logits: 5.88 TB/s without, 6.22 TB/s with; on the
// policy loss, whose second sweep finds its row in L2, 3.97 and 4.97 TB/s of one read and one write.
__device__ __forceinline__ unsigned long long l2_first() {
    unsigned long long p;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ unsigned long long l2_last() {
    unsigned long long p;
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint4 ld_policy16_raw(const void* p, unsigned long long policy) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p), "l"(policy));
    return v;
}
__device__ __forceinline__ void st_stream16_raw(void* p, const uint4& v) {
    asm volatile("st.global.L1::no_allocate.L2::cache_hint.v4.u32 [%0], {%1,%2,%3,%4}, %5;"
                 ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "l"(l2_first()) : "memory");
}
#define ld_policy16(p, policy) ::tpb::ld_policy16_raw(TPB_CKN((p), 16), (policy))
#define ld_once16(p) ::tpb::ld_policy16_raw(TPB_CKN((p), 16), ::tpb::l2_first())
#define st_out16(p, v) ::tpb::st_stream16_raw(TPB_CKN((p), 16), (v))

// Eight consecutive elements, 16-byte aligned: one vector of a 16-bit type, two of float32.
template <class T>
__device__ __forceinline__ void load8(const T* p, float* f) {
    if constexpr (sizeof(T) == 2) {
        Elem<T>::unpack(ld_once16(p), f);
    } else {
        const uint4 a = ld_once16(p), b = ld_once16(p + 4);
        Elem<T>::unpack(a, f);
        Elem<T>::unpack(b, f + 4);
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float* f) {
    if constexpr (sizeof(T) == 2) {
        st_out16(p, Elem<T>::pack(f));
    } else {
        st_out16(p, Elem<T>::pack(f));
        st_out16(p + 4, Elem<T>::pack(f + 4));
    }
}

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
    return v;
}
__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
    return v;
}

}  // namespace tpb
