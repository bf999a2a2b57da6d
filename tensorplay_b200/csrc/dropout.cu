// Dropout from a counter-based generator behind tpb200_dropout: y = x * factor(i), the factor of element
// i being 0 or 1 / (1 - p) as philox.cuh says.  The backward pass is the same call on the gradient.
// Bound by memory (one read and one write of the tensor).
#define TPB_FILE_ID 9
#include "host_util.h"
#include "lowp.cuh"
#include "philox.cuh"

#include <algorithm>

namespace tpb {

// `n` elements one after the other on both sides, 16-byte aligned: a block of the generator per step.  With 32
// registers, and so 64 warps on an SM, [16384,8192] takes 104.8 us in bfloat16 (5.1 TB/s: the generator's ten rounds are
// some sixty integer instructions for eight elements) and 172 us in float32 (6.2 TB/s); with 44 registers 118.9 and
// 176; two vectors in flight per thread gain nothing on top.
#ifdef TPB200_CHECKED
constexpr int kDropCtas = 6;     // the checker's own function needs 38 registers
#else
constexpr int kDropCtas = 8;
#endif
template <class T>
__global__ void __launch_bounds__(256, kDropCtas)
dropout_flat_kernel(const T* __restrict__ x, T* __restrict__ y, long long n, DropSpec d) {
    const long long blocks = n >> 3, step = (long long)gridDim.x * blockDim.x;
    for (long long b = (long long)blockIdx.x * blockDim.x + threadIdx.x; b < blocks; b += step) {
        float v[8];
        load8(x + 8 * b, v);
        if (d.units) drop8((unsigned long long)b, d, v);
        store8(y + 8 * b, v);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0 && (n & 7)) {
        const unsigned keep = d.units ? keep_bits8((unsigned long long)blocks, d) : 0xffu;
        for (int c = 0; c < (int)(n & 7); ++c) {
            const long long i = (blocks << 3) + c;
            *TPB_CK(&y[i]) = Elem<T>::put(keep >> c & 1 ? Elem<T>::get(*TPB_CK(&x[i])) * d.factor : 0.0f);
        }
    }
}

// Rows of any stride and alignment: a thread takes the eight elements of one block of the generator.
template <class T>
__global__ void __launch_bounds__(256)
dropout_rows_kernel(const T* __restrict__ x, T* __restrict__ y, long long n, long long inner, long long width,
                    long long s0, long long s1, DropSpec d) {
    const long long blocks = (n + 7) >> 3;
    for (long long b = (long long)blockIdx.x * blockDim.x + threadIdx.x; b < blocks; b += (long long)gridDim.x * blockDim.x) {
        const unsigned keep = d.units ? keep_bits8((unsigned long long)b, d) : 0xffu;
        long long r = (b << 3) / width, c = (b << 3) - r * width;
        long long o = r / inner, q = r - o * inner;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const long long i = (b << 3) + e;
            if (i < n) *TPB_CK(&y[i]) = Elem<T>::put(keep >> e & 1 ? Elem<T>::get(*TPB_CK(&x[o * s0 + q * s1 + c])) * d.factor : 0.0f);
            if (++c == width) {
                c = 0;
                if (++q == inner) { q = 0; ++o; }
            }
        }
    }
}

template <class T>
int dropout_run(const void* x, long long outer, long long inner, long long width, long long s0, long long s1, const DropSpec& d,
                void* y, cudaStream_t st) {
    const long long n = outer * inner * width;
    const bool flat = (inner == 1 || s1 == width) && (outer == 1 || s0 == inner * width) && (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    const long long ctas = std::max(1LL, std::min(ceil_div(ceil_div(n, 8), 256), 64LL * sm_count()));
    const dim3 grid((unsigned)ctas);
    if (flat) TPB_LAUNCH("dropout_flat_kernel", dropout_flat_kernel<T>, grid, 256, 0, st, (const T*)x, (T*)y, n, d);
    else TPB_LAUNCH("dropout_rows_kernel", dropout_rows_kernel<T>, grid, 256, 0, st, (const T*)x, (T*)y, n, inner, width, s0, s1, d);
    return TPB200_OK;
}

}  // namespace tpb

using namespace tpb;

extern "C" int tpb200_dropout(const void* x, int dtype, int64_t outer, int64_t inner, int64_t width, const int64_t* strides,
                              double p, uint64_t seed, uint64_t offset, void* y, void* stream) {
    if (dtype_bytes(dtype) == 0) return fail(TPB200_ERR_UNSUPPORTED, "dropout: only float32, bfloat16 and float16 are supported (dtype code %d)", dtype);
    if (outer < 0 || inner < 0 || width < 0) return fail(TPB200_ERR_INVALID, "dropout: negative size");
    long long n = 0;
    if (__builtin_mul_overflow((long long)outer, (long long)inner, &n) || __builtin_mul_overflow(n, (long long)width, &n) || n > (1LL << 60))
        return fail(TPB200_ERR_UNSUPPORTED, "dropout: too many elements");
    DropSpec d;
    if (!make_drop(p, seed, offset, &d)) return fail(TPB200_ERR_INVALID, "dropout: p must lie in [0, 1]");
    if (!strides) return fail(TPB200_ERR_INVALID, "strides must not be NULL");
    if (n == 0) return TPB200_OK;
    if (!x || !y) return fail(TPB200_ERR_INVALID, "NULL pointer argument");
    cudaStream_t st = (cudaStream_t)stream;
    const int64_t size = dtype_bytes(dtype);
    TPB_CHECK_RANGES(st, rows_range(x, outer, inner, width, strides, size), HostRange{y, (size_t)(n * size)});
    switch (dtype) {
        case TPB200_F32: return dropout_run<float>(x, outer, inner, width, strides[0], strides[1], d, y, st);
        case TPB200_BF16: return dropout_run<__nv_bfloat16>(x, outer, inner, width, strides[0], strides[1], d, y, st);
        default: return dropout_run<__half>(x, outer, inner, width, strides[0], strides[1], d, y, st);
    }
}
