// The residual path of a block, forward and backward, behind tpb200_block_residual*, tpb200_rms_norm*.
//
// Forward, per row of `width` elements (hat(v) = v * rstd(v), rstd(v) = 1 / sqrt(mean v^2 + eps)):
//     n = hat(h) * w_post                     the norm after the block (or n = h)
//     x' = x + scale * gate * drop(n)         gate, dropout and residual scale
//     y = hat(x') * w_next                    the norm before the next block (or no y)
// Backward, from g_x = dL/dx' and g_y = dL/dy:
//     a = g_y * w_next,  t = g_x + rstd_next * (a - hat(x') * mean(a * hat(x')))       = dL/dx
//     d = scale * gate * factor * t,  dgate = scale * factor * n * t
//     b = d * w_post,  dh = rstd_post * (b - hat(h) * mean(b * hat(h)))
//     dw_next = sum over rows of g_y * hat(x'),  dw_post = sum over rows of d * hat(h)
// rms_norm is the part with w_next alone.  All of it is float32 between the loads and the one rounding of
// each output; y and rstd_next go by the x' before it is rounded.  The backward pass takes x' from the forward
// call's x, h and gate again, operation by operation (the same bits), or, where it is given x_out instead, as
// it was rounded there: dw_next of a 16-bit type is then a second rounding of x' off (bfloat16, [2048,4096]:
// 2.3e-3 of its norm against 1.6e-3).
#define TPB_FILE_ID 8
#include "host_util.h"
#include "lowp.cuh"
#include "philox.cuh"

#include <algorithm>

namespace tpb {

constexpr int kMaxWidth = 16384;

// Row (a, b) of a [outer, inner, width] view; strides of 0 broadcast.
template <class T>
struct RowView {
    T* p;
    long long s0, s1;
    __device__ __forceinline__ T* row(long long a, long long b) const { return p + a * s0 + b * s1; }
};

template <class T>
struct ForwardArgs {
    RowView<const T> x, h, gate;     // h.p NULL: rms_norm alone; gate.p NULL: no gate
    const T *post, *next;            // NULL: no such norm
    T *x_out, *y;                    // contiguous
    float *rstd_post, *rstd_next;
    long long rows, inner;
    int width;
    float scale, eps;
    DropSpec drop;
};

// Eight elements of a row per thread and step: consecutive ones (VEC: 16-byte vectors), or `nthr` apart.
template <bool VEC>
__device__ __forceinline__ int at(int u, int c, int tid, int nthr) {
    return VEC ? (u * nthr + tid) * 8 + c : (u * 8 + c) * nthr + tid;
}
template <class T, bool VEC>
__device__ __forceinline__ void fetch8(const T* p, int u, int tid, int nthr, int width, float* f) {
    if (VEC) {
        const int e = at<VEC>(u, 0, tid, nthr);
        if (e < width) load8(p + e, f);
        else {
#pragma unroll
            for (int c = 0; c < 8; ++c) f[c] = 0.0f;
        }
    } else {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int e = at<VEC>(u, c, tid, nthr);
            f[c] = e < width ? Elem<T>::get(*TPB_CK(&p[e])) : 0.0f;
        }
    }
}
template <class T, bool VEC>
__device__ __forceinline__ void put8(T* p, int u, int tid, int nthr, int width, const float* f) {
    if (VEC) {
        const int e = at<VEC>(u, 0, tid, nthr);
        if (e < width) store8(p + e, f);
    } else {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int e = at<VEC>(u, c, tid, nthr);
            if (e < width) *TPB_CK(&p[e]) = Elem<T>::put(f[c]);
        }
    }
}
// Rows that are no whole blocks of the generator (any width that is no multiple of 8): the threads of a row draw
// the blocks that it touches into shared memory, one byte for eight elements, `base` = the row's first element.
template <bool WARP>
__device__ __forceinline__ void draw_row(const DropSpec& d, unsigned long long base, int width, int tid, int nthr, unsigned char* keep) {
    if (WARP) __syncwarp();      // the row before has been read (a CTA's rows are a barrier apart anyway)
    const unsigned long long first = base >> 3, last = (base + (unsigned)width - 1) >> 3;
    for (unsigned long long b = first + tid; b <= last; b += nthr) keep[b - first] = (unsigned char)keep_bits8(b, d);
    if (WARP) __syncwarp();
    else __syncthreads();
}
// v := dropout(v) for eight elements whose bits in `keep` say which stay
__device__ __forceinline__ void drop_by8(const DropSpec& d, unsigned keep, float* v) {
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = keep >> c & 1 ? v[c] * d.factor : 0.0f;
}
// v := dropout(v) for a thread's eight elements of row r
template <bool VEC>
__device__ __forceinline__ void drop_row8(const DropSpec& d, long long r, int u, int tid, int nthr, int width, const unsigned char* keep, float* v) {
    if (VEC) {
        drop8((unsigned long long)(r * (width >> 3) + (u * nthr + tid)), d, v);
    } else {
        const int skip = (int)((unsigned long long)(r * width) & 7);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int i = at<VEC>(u, c, tid, nthr);
            if (i < width) v[c] = keep[(skip + i) >> 3] >> ((skip + i) & 7) & 1 ? v[c] * d.factor : 0.0f;
        }
    }
}
__host__ __device__ constexpr int keep_bytes(int width) { return width / 8 + 16; }

// Sum over the threads of a row: a warp, or the CTA (`red` then has 32 slots that the next call must not reuse).
template <bool WARP>
__device__ __forceinline__ float row_add(float v, float* red) {
    v = warp_add(v);
    if (WARP) return v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return warp_add(lane < nw ? red[lane] : 0.0f);
}

#ifdef TPB200_CHECKED
template <int NV> constexpr int kForwardCtas = 1;                  // the checker's own function needs 38 registers
#else
template <int NV> constexpr int kForwardCtas = NV == 1 ? 2 : 1;    // 32 registers, 64 warps on an SM
#endif
template <class T, int NV, bool VEC, bool WARP>
__global__ void __launch_bounds__(1024, kForwardCtas<NV>)
block_forward_kernel(ForwardArgs<T> k) {
    extern __shared__ unsigned char keep_mem[];      // keep_bytes per row of the CTA, without VEC and with dropout
    __shared__ float red[2][32];
    const int tid = WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x, nthr = WARP ? 32 : (int)blockDim.x;
    const unsigned r = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && r >= k.rows) return;
    const unsigned a = r / (unsigned)k.inner, b = r - a * (unsigned)k.inner;
    const float inv_width = 1.0f / (float)k.width;
    float x[NV][8], h[NV][8];
    const T *px = k.x.row(a, b), *ph = k.h.p ? k.h.row(a, b) : nullptr, *pg = k.gate.p ? k.gate.row(a, b) : nullptr;
    if (ph) {
#pragma unroll
        for (int u = 0; u < NV; ++u) fetch8<T, VEC>(ph, u, tid, nthr, k.width, h[u]);
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) fetch8<T, VEC>(px, u, tid, nthr, k.width, x[u]);
    if (ph) {
        float rstd = 1.0f;
        if (k.post) {
            float s = 0.0f;
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int c = 0; c < 8; ++c) s = fmaf(h[u][c], h[u][c], s);
            rstd = rsqrtf(row_add<WARP>(s, red[0]) * inv_width + k.eps);
            if (tid == 0) *TPB_CK(&k.rstd_post[r]) = rstd;
        }
        unsigned char* keep = keep_mem + (WARP ? (threadIdx.x >> 5) * keep_bytes(k.width) : 0);
        if (!VEC && k.drop.units) draw_row<WARP>(k.drop, (unsigned long long)r * k.width, k.width, tid, nthr, keep);
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            if (k.post) {
                float w[8];
                fetch8<T, VEC>(k.post, u, tid, nthr, k.width, w);
#pragma unroll
                for (int c = 0; c < 8; ++c) h[u][c] = h[u][c] * rstd * w[c];
            }
            if (k.drop.units) drop_row8<VEC>(k.drop, r, u, tid, nthr, k.width, keep, h[u]);
            if (pg) {
                float g[8];
                fetch8<T, VEC>(pg, u, tid, nthr, k.width, g);
#pragma unroll
                for (int c = 0; c < 8; ++c) h[u][c] *= g[c];
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) x[u][c] = fmaf(k.scale, h[u][c], x[u][c]);
            put8<T, VEC>(k.x_out + (long long)r * k.width, u, tid, nthr, k.width, x[u]);
        }
    }
    if (!k.next) return;
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int c = 0; c < 8; ++c) s = fmaf(x[u][c], x[u][c], s);   // elements past the width are zero
    const float rstd = rsqrtf(row_add<WARP>(s, red[1]) * inv_width + k.eps);
    if (tid == 0) *TPB_CK(&k.rstd_next[r]) = rstd;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        float w[8];
        fetch8<T, VEC>(k.next, u, tid, nthr, k.width, w);
#pragma unroll
        for (int c = 0; c < 8; ++c) w[c] *= x[u][c] * rstd;
        put8<T, VEC>(k.y + (long long)r * k.width, u, tid, nthr, k.width, w);
    }
}

// ---------------------------------------------------------------- staged rows ----------------
// 16-byte aligned rows of up to 8192 elements, one eight-element vector per thread: persistent CTAs, whose threads
// copy their warp's vectors of the next row into shared memory (cp.async; no barrier over the CTA) while they work
// on this one, so that a row's reductions over the CTA do not wait for memory.  [16384,4096] bf16 with an element gate:
// 119 us without dropout (5.6 TB/s; a CTA per row and no prefetch took 147), 159 us with it (some sixty integer
// instructions of the generator for eight elements).
constexpr int kStages = 2;

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)),
                 "l"(TPB_CKN(src, 16)), "l"(l2_first()) : "memory");
}
// One stage.  A warp's 32 vectors of an array are 32 * kVec consecutive 16-byte pieces in memory and in the stage;
// lane l copies the pieces l, l + 32, so that a float32 row is read in whole sectors too (each lane copying its
// own 32 bytes took twice the time), and reads its own pieces back.
template <class T>
struct Staged {
    static constexpr int kVec = 8 * sizeof(T) / 16;       // pieces of a thread's vector
    uint4* warp_at;     // the warp's first piece of array 0
    int nthr;
    __device__ __forceinline__ Staged(uint4* mem, int stage, int arrays, int n)
        : warp_at(mem + (size_t)stage * arrays * kVec * n + (threadIdx.x & ~31u) * kVec), nthr(n) {}
    __device__ __forceinline__ void fill(int array, const T* row, int width) const {
        const int lane = threadIdx.x & 31, first = (int)(threadIdx.x & ~31u) * kVec;
        const uint4* p = reinterpret_cast<const uint4*>(row) + first;
#pragma unroll
        for (int j = 0; j < kVec; ++j)
            if ((first + j * 32 + lane) * Elem<T>::N < width) copy_async16(warp_at + (size_t)array * kVec * nthr + j * 32 + lane, p + j * 32 + lane);
    }
    __device__ __forceinline__ void read(int array, float* f) const {
#pragma unroll
        for (int j = 0; j < kVec; ++j) Elem<T>::unpack(warp_at[(size_t)array * kVec * nthr + (threadIdx.x & 31) * kVec + j], f + j * Elem<T>::N);
    }
    // what the lanes of a warp have copied is there for all of them, or has been read by all of them
    static __device__ __forceinline__ void sync() {
        if (kVec > 1) __syncwarp();
    }
};

constexpr int kForwardArrays = 3;      // h, x, gate
template <class T>
__global__ void __launch_bounds__(1024, kForwardCtas<1>)
block_forward_staged_kernel(ForwardArgs<T> k) {
    extern __shared__ __align__(16) uint4 stage_mem[];
    __shared__ float red[2][2][32];
    const int tid = threadIdx.x, nthr = blockDim.x, e = tid * 8;
    const bool mine = e < k.width;
    const float inv_width = 1.0f / (float)k.width;
    const unsigned rows = (unsigned)k.rows, step = gridDim.x;
    int turn = 0;
    const auto prefetch = [&](unsigned r, int t) {
        if (r < rows) {
            const unsigned a = r / (unsigned)k.inner, b = r - a * (unsigned)k.inner;
            const Staged<T> st(stage_mem, t & 1, kForwardArrays, nthr);
            Staged<T>::sync();
            if (k.h.p) st.fill(0, k.h.row(a, b), k.width);
            st.fill(1, k.x.row(a, b), k.width);
            if (k.gate.p) st.fill(2, k.gate.row(a, b), k.width);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    prefetch(blockIdx.x, 0);
    for (unsigned r = blockIdx.x; r < rows; r += step, ++turn) {       // rows + step stays below 2^32
        prefetch(r + step, turn + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        Staged<T>::sync();
        const Staged<T> st(stage_mem, turn & 1, kForwardArrays, nthr);
        float* sums = red[turn & 1][0];        // alternates: whoever writes it again has passed a barrier of the row between
        float v[8], w[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = 0.0f;
        if (k.h.p) {
            float rstd = 1.0f;
            if (mine) st.read(0, v);
            if (k.post) {
                float s = 0.0f;
#pragma unroll
                for (int c = 0; c < 8; ++c) s = fmaf(v[c], v[c], s);
                rstd = rsqrtf(row_add<false>(s, sums) * inv_width + k.eps);
                if (tid == 0) *TPB_CK(&k.rstd_post[r]) = rstd;
                if (mine) {
                    load8(k.post + e, w);
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[c] = v[c] * rstd * w[c];
                }
            }
            if (mine) {
                if (k.drop.units) drop8((unsigned long long)r * (k.width >> 3) + tid, k.drop, v);
                if (k.gate.p) {
                    st.read(2, w);
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[c] *= w[c];
                }
                st.read(1, w);
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = fmaf(k.scale, v[c], w[c]);
                store8(k.x_out + (long long)r * k.width + e, v);
            }
        } else if (mine) {
            st.read(1, v);
        }
        if (!k.next) continue;
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) s = fmaf(v[c], v[c], s);
        const float rstd = rsqrtf(row_add<false>(s, sums + 32) * inv_width + k.eps);
        if (tid == 0) *TPB_CK(&k.rstd_next[r]) = rstd;
        if (mine) {
            load8(k.next + e, w);
#pragma unroll
            for (int c = 0; c < 8; ++c) w[c] *= v[c] * rstd;
            store8(k.y + (long long)r * k.width + e, w);
        }
    }
}

template <class T>
struct BackwardArgs {
    RowView<const T> grad_x, grad_y, h, x_out, gate;   // grad_x.p NULL: zero; grad_y.p / x_out.p go with next
    int from_x;                        // 1: x_out holds the forward call's x (with h and next)
    const T *post, *next;
    const float *rstd_post, *rstd_next;
    T *dx, *dh, *dgate;                // contiguous; dgate: [groups, width], or all rows (gate_rows)
    float *part_post, *part_next, *part_gate;   // [workers, width] sums over a worker's rows
    long long rows, inner;
    // worker k takes the rows [lo, hi) of split k % splits of group k / splits (group_len rows each,
    // split_len rows per split), or, with groups_per_worker > 0, that many whole groups
    long long group_len, split_len, groups_per_worker;
    int splits, workers, width;
    int gate_rows;                     // 1: the gate has a row for every row
    float scale;
    DropSpec drop;
};

template <class T, int NV, bool VEC, bool WARP>
__global__ void __launch_bounds__(1024)
block_backward_kernel(BackwardArgs<T> k) {
    extern __shared__ unsigned char keep_mem[];      // as in the forward kernel
    __shared__ float red[2][32];
    const int tid = WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x, nthr = WARP ? 32 : (int)blockDim.x;
    const int worker = WARP ? (int)(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) : (int)blockIdx.x;
    if (WARP && worker >= k.workers) return;
    const float inv_width = 1.0f / (float)k.width;
    long long lo, hi;
    if (k.groups_per_worker > 0) {
        lo = (long long)worker * k.groups_per_worker * k.group_len;
        hi = lo + k.groups_per_worker * k.group_len;
        if (hi > k.rows) hi = k.rows;
    } else {
        const long long g = worker / k.splits, s = worker - g * k.splits;
        lo = s * k.split_len;
        hi = lo + k.split_len;
        if (hi > k.group_len) hi = k.group_len;
        lo += g * k.group_len;
        hi += g * k.group_len;
    }
    const bool sum_gate = k.gate.p && !k.gate_rows;
    float acc_post[NV][8], acc_next[NV][8], acc_gate[NV][8];
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int c = 0; c < 8; ++c) acc_post[u][c] = acc_next[u][c] = acc_gate[u][c] = 0.0f;
    for (long long r = lo; r < hi; ++r) {
        const long long a = r / k.inner, b = r - a * k.inner;
        float t[NV][8], h[NV][8];
        if (k.grad_x.p) {
#pragma unroll
            for (int u = 0; u < NV; ++u) fetch8<T, VEC>(k.grad_x.row(a, b), u, tid, nthr, k.width, t[u]);
        } else {
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int c = 0; c < 8; ++c) t[u][c] = 0.0f;
        }
        if (k.h.p) {
#pragma unroll
            for (int u = 0; u < NV; ++u) fetch8<T, VEC>(k.h.row(a, b), u, tid, nthr, k.width, h[u]);
        }
        unsigned char* keep = keep_mem + (WARP ? (threadIdx.x >> 5) * keep_bytes(k.width) : 0);
        const float rstd_post = k.post && k.h.p ? *TPB_CK(&k.rstd_post[r]) : 1.0f;
        if (!VEC && k.h.p && k.drop.units) draw_row<WARP>(k.drop, (unsigned long long)r * k.width, k.width, tid, nthr, keep);
        if (k.next) {
            const float rstd = *TPB_CK(&k.rstd_next[r]);
            float xh[NV][8], g[NV][8], s = 0.0f;
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                float w[8];
                fetch8<T, VEC>(k.x_out.row(a, b), u, tid, nthr, k.width, xh[u]);
                if (k.from_x) {            // x' before it was rounded, by the forward kernel's operations
                    float n[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) n[c] = h[u][c];
                    if (k.post) {
                        fetch8<T, VEC>(k.post, u, tid, nthr, k.width, w);
#pragma unroll
                        for (int c = 0; c < 8; ++c) n[c] = n[c] * rstd_post * w[c];
                    }
                    if (k.drop.units) drop_row8<VEC>(k.drop, r, u, tid, nthr, k.width, keep, n);
                    if (k.gate.p) {
                        fetch8<T, VEC>(k.gate.row(a, b), u, tid, nthr, k.width, w);
#pragma unroll
                        for (int c = 0; c < 8; ++c) n[c] *= w[c];
                    }
#pragma unroll
                    for (int c = 0; c < 8; ++c) xh[u][c] = fmaf(k.scale, n[c], xh[u][c]);
                }
                fetch8<T, VEC>(k.grad_y.row(a, b), u, tid, nthr, k.width, g[u]);
                fetch8<T, VEC>(k.next, u, tid, nthr, k.width, w);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    xh[u][c] *= rstd;
                    acc_next[u][c] = fmaf(g[u][c], xh[u][c], acc_next[u][c]);
                    g[u][c] *= w[c];
                    s = fmaf(g[u][c], xh[u][c], s);
                }
            }
            const float m = row_add<WARP>(s, red[0]) * inv_width;
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int c = 0; c < 8; ++c) t[u][c] = fmaf(rstd, g[u][c] - xh[u][c] * m, t[u][c]);
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) put8<T, VEC>(k.dx + r * k.width, u, tid, nthr, k.width, t[u]);
        if (k.h.p) {
            float s = 0.0f;
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                float w[8], g[8];
                if (k.post) fetch8<T, VEC>(k.post, u, tid, nthr, k.width, w);
                if (k.drop.units) drop_row8<VEC>(k.drop, r, u, tid, nthr, k.width, keep, t[u]);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    h[u][c] *= rstd_post;
                    t[u][c] *= k.scale;                                // scale * factor * t
                }
                if (k.gate.p) {
                    fetch8<T, VEC>(k.gate.row(a, b), u, tid, nthr, k.width, g);
                    float dg[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float n = k.post ? h[u][c] * w[c] : h[u][c];
                        dg[c] = n * t[u][c];
                        acc_gate[u][c] += dg[c];
                        t[u][c] *= g[c];
                    }
                    if (k.gate_rows) put8<T, VEC>(k.dgate + r * k.width, u, tid, nthr, k.width, dg);
                }
                if (k.post) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        acc_post[u][c] = fmaf(t[u][c], h[u][c], acc_post[u][c]);
                        t[u][c] *= w[c];
                        s = fmaf(t[u][c], h[u][c], s);
                    }
                }
            }
            if (k.post) {
                const float m = row_add<WARP>(s, red[1]) * inv_width;
#pragma unroll
                for (int u = 0; u < NV; ++u)
#pragma unroll
                    for (int c = 0; c < 8; ++c) t[u][c] = rstd_post * (t[u][c] - h[u][c] * m);
            }
#pragma unroll
            for (int u = 0; u < NV; ++u) put8<T, VEC>(k.dh + r * k.width, u, tid, nthr, k.width, t[u]);
            if (sum_gate && k.groups_per_worker > 0 && (r + 1) % k.group_len == 0) {   // the group is complete
                const long long g = r / k.group_len;
#pragma unroll
                for (int u = 0; u < NV; ++u) {
                    put8<T, VEC>(k.dgate + g * k.width, u, tid, nthr, k.width, acc_gate[u]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) acc_gate[u][c] = 0.0f;
                }
            }
        }
        if (!WARP) __syncthreads();   // the slots of row_add are free again
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        if (k.post && k.h.p) put8<float, VEC>(k.part_post + (long long)worker * k.width, u, tid, nthr, k.width, acc_post[u]);
        if (k.next) put8<float, VEC>(k.part_next + (long long)worker * k.width, u, tid, nthr, k.width, acc_next[u]);
        if (sum_gate && k.groups_per_worker == 0) put8<float, VEC>(k.part_gate + (long long)worker * k.width, u, tid, nthr, k.width, acc_gate[u]);
    }
}

// ---------------------------------------------------------------- staged backward ------------
// The same for 16-byte aligned rows of up to 8192 elements; the next row's vectors of grad_x, grad_y, x_out, h and gate
// arrive while this one is worked on.  [16384,4096] bf16 with an element gate: 229 us without dropout (4.7 TB/s), 268 us
// with it; with FROM_X 257 and 302 us, three more reads of shared memory and x' formed again in front of the row's
// first sum.  Bound by issue: 104 thread instructions per element (121 with FROM_X) keep the schedulers 74 to 76 % busy with
// the 27 warps on an SM that 64 registers and two stages of five arrays allow.  The kernel
// above, which loads a row when it comes to it, took some 400 us.
constexpr int kStageArrays = 5;

template <class T, bool SUM_GATE, bool FROM_X>
__global__ void __launch_bounds__(1024, 1)
block_backward_staged_kernel(BackwardArgs<T> k) {
    extern __shared__ __align__(16) uint4 stage_mem[];
    __shared__ float red[2][2][32];
    const int tid = threadIdx.x, nthr = blockDim.x, worker = blockIdx.x;
    const float inv_width = 1.0f / (float)k.width;
    long long lo, hi;
    if (k.groups_per_worker > 0) {
        lo = (long long)worker * k.groups_per_worker * k.group_len;
        hi = lo + k.groups_per_worker * k.group_len;
        if (hi > k.rows) hi = k.rows;
    } else {
        const long long g = worker / k.splits, s = worker - g * k.splits;
        lo = s * k.split_len;
        hi = lo + k.split_len;
        if (hi > k.group_len) hi = k.group_len;
        lo += g * k.group_len;
        hi += g * k.group_len;
    }
    const bool mine = tid * 8 < k.width;
    const int e = tid * 8;
    // the thread's part of both weights lies behind the stages: 16 float32 registers are not to spare
    const Staged<T> weights(stage_mem, kStages, kStageArrays, nthr);
    const auto prefetch = [&](long long r) {
        if (r < hi) {
            const unsigned a = (unsigned)r / (unsigned)k.inner, b = (unsigned)r - a * (unsigned)k.inner;
            const Staged<T> st(stage_mem, (int)(r & 1), kStageArrays, nthr);
            Staged<T>::sync();
            if (k.grad_x.p) st.fill(0, k.grad_x.row(a, b), k.width);
            if (k.next) {
                st.fill(1, k.grad_y.row(a, b), k.width);
                st.fill(2, k.x_out.row(a, b), k.width);
            }
            if (k.h.p) st.fill(3, k.h.row(a, b), k.width);
            if (k.gate.p) st.fill(4, k.gate.row(a, b), k.width);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // and behind them the gate's running sums
    float4* gate_sum = reinterpret_cast<float4*>(stage_mem + (size_t)((kStages * kStageArrays + 2) * Staged<T>::kVec) * nthr) + tid;
    if (SUM_GATE) gate_sum[0] = gate_sum[nthr] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto store_gate = [&](auto* dst) {
        const float4 p = gate_sum[0], q = gate_sum[nthr];
        const float v[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
        if (mine) store8(dst, v);
    };
    float acc_post[8], acc_next[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) acc_post[c] = acc_next[c] = 0.0f;
    if (k.next) weights.fill(0, k.next, k.width);
    if (k.post) weights.fill(1, k.post, k.width);
    prefetch(lo);
    for (long long r = lo; r < hi; ++r) {
        prefetch(r + 1);
        const float rstd_next = k.next ? *TPB_CK(&k.rstd_next[r]) : 1.0f, rstd_post = k.post ? *TPB_CK(&k.rstd_post[r]) : 1.0f;
        // with FROM_X drawn here, while the row is on its way, because both halves of the work need it
        const unsigned keep = FROM_X && k.drop.units ? keep_bits8((unsigned long long)(r * (k.width >> 3) + tid), k.drop) : 0xffu;
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        Staged<T>::sync();
        const Staged<T> st(stage_mem, (int)(r & 1), kStageArrays, nthr);
        float t[8], u[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) t[c] = 0.0f;
        float* sums = red[r & 1][0];
        if (k.next) {
            float xh[8], s = 0.0f;
            if (mine) {
                if (FROM_X) {              // x' before it was rounded, by the forward kernel's operations
                    st.read(3, xh);
                    if (k.post) {
                        weights.read(1, u);
#pragma unroll
                        for (int c = 0; c < 8; ++c) xh[c] = xh[c] * rstd_post * u[c];
                    }
                    if (k.drop.units) drop_by8(k.drop, keep, xh);
                    if (k.gate.p) {
                        st.read(4, u);
#pragma unroll
                        for (int c = 0; c < 8; ++c) xh[c] *= u[c];
                    }
                    st.read(2, u);
#pragma unroll
                    for (int c = 0; c < 8; ++c) xh[c] = fmaf(k.scale, xh[c], u[c]);
                } else {
                    st.read(2, xh);
                }
                st.read(1, u);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    xh[c] *= rstd_next;
                    acc_next[c] = fmaf(u[c], xh[c], acc_next[c]);
                }
                float w[8];
                weights.read(0, w);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    u[c] *= w[c];
                    s = fmaf(u[c], xh[c], s);
                }
            }
            const float m = row_add<false>(s, sums) * inv_width;
            if (mine) {
                if (k.grad_x.p) st.read(0, t);
#pragma unroll
                for (int c = 0; c < 8; ++c) t[c] = fmaf(rstd_next, u[c] - xh[c] * m, t[c]);
            }
        } else if (mine && k.grad_x.p) {
            st.read(0, t);
        }
        if (mine) store8(k.dx + r * k.width + e, t);
        if (k.h.p) {
            float s = 0.0f, hat[8];
            if (mine) {
                st.read(3, hat);
                if (k.drop.units) {
                    if (FROM_X) drop_by8(k.drop, keep, t);
                    else drop8((unsigned long long)(r * (k.width >> 3) + tid), k.drop, t);
                }
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    hat[c] *= rstd_post;
                    t[c] *= k.scale;                               // scale * factor * t
                }
                float w[8];
                if (k.post) weights.read(1, w);
                if (k.gate.p) {
                    float g[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) u[c] = (k.post ? hat[c] * w[c] : hat[c]) * t[c];
                    if (SUM_GATE) {
                        float4 q = gate_sum[0];
                        gate_sum[0] = make_float4(q.x + u[0], q.y + u[1], q.z + u[2], q.w + u[3]);
                        q = gate_sum[nthr];
                        gate_sum[nthr] = make_float4(q.x + u[4], q.y + u[5], q.z + u[6], q.w + u[7]);
                    } else {
                        store8(k.dgate + r * k.width + e, u);
                    }
                    st.read(4, g);
#pragma unroll
                    for (int c = 0; c < 8; ++c) t[c] *= g[c];
                }
                if (k.post) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        acc_post[c] = fmaf(t[c], hat[c], acc_post[c]);
                        t[c] *= w[c];
                        s = fmaf(t[c], hat[c], s);
                    }
                }
            }
            if (k.post) {
                const float m = row_add<false>(s, sums + 32) * inv_width;
                if (mine) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) t[c] = rstd_post * (t[c] - hat[c] * m);
                }
            }
            if (mine) store8(k.dh + r * k.width + e, t);
            if (SUM_GATE && k.groups_per_worker > 0 && (r + 1) % k.group_len == 0) {   // the group is complete
                store_gate(k.dgate + (r / k.group_len) * k.width + e);
                gate_sum[0] = gate_sum[nthr] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        // `sums` alternates by the row: whoever writes it again has passed a barrier of the row between, which
        // everybody reaches after reading it
    }
    if (mine) {
        if (k.post && k.h.p) store8(k.part_post + (long long)worker * k.width + e, acc_post);
        if (k.next) store8(k.part_next + (long long)worker * k.width + e, acc_next);
        if (SUM_GATE && k.groups_per_worker == 0) store_gate(k.part_gate + (long long)worker * k.width + e);
    }
}

// Column sums of the workers' partial sums in a fixed order: 32 columns by 8 slots at a time.
// blockIdx.y: 0 w_post, 1 w_next, 2 + g the gate's group g (slots g * splits ...).
template <class T>
__global__ void __launch_bounds__(256)
block_sums_kernel(const float* __restrict__ part_post, const float* __restrict__ part_next, const float* __restrict__ part_gate,
                  T* __restrict__ dpost, T* __restrict__ dnext, T* __restrict__ dgate, int workers, int splits, int width) {
    __shared__ double red[8][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x >> 5;
    const int what = (int)blockIdx.y;
    const float* src = what == 0 ? part_post : (what == 1 ? part_next : part_gate + (long long)(what - 2) * splits * width);
    T* dst = what == 0 ? dpost : (what == 1 ? dnext : dgate + (long long)(what - 2) * width);
    if (!src || !dst) return;
    const int n = what < 2 ? workers : splits;
    double s = 0.0;
    if (c < width)
        for (int i = y; i < n; i += 8) s += (double)*TPB_CK(&src[(long long)i * width + c]);
    red[y][threadIdx.x & 31] = s;
    __syncthreads();
    if (y == 0 && c < width) {
        s = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += red[j][threadIdx.x & 31];
        *TPB_CK(&dst[c]) = Elem<T>::put((float)s);
    }
}

// ---------------------------------------------------------------- host side -------------------
struct RowPlan {
    bool vec, warp;
    int nv, threads;   // threads of a CTA
};
inline RowPlan plan_rows(int64_t width, bool vec) {
    RowPlan p;
    p.vec = vec;
    p.warp = width <= 512;
    p.nv = width <= 256 || (width > 512 && width <= 8192) ? 1 : 2;
    p.threads = p.warp ? 256 : (int)std::min<long long>(1024, round_up(ceil_div(width, 8 * p.nv), 32));
    return p;
}

// Shared memory of the staged kernels: two stages of the arrays; for the backward pass both weights and the gate's
// sums.  They take rows of up to 8192 elements as long as that fits (backward, float32: up to some 4.5 K elements).
inline int staged_threads(int64_t width) { return (int)round_up(ceil_div(width, 8), 32); }
inline size_t backward_bytes(int64_t width, size_t elem, bool sum_gate) {
    return (size_t)staged_threads(width) * ((kStages * kStageArrays + 2) * 8 * elem + (sum_gate ? 32 : 0));
}
// CTAs of a persistent kernel that an SM holds: its threads by registers, 227 KB of shared memory, 32 CTAs.
// One more than fits would run after the others, with the rows dealt out twice the time.
inline int resident_ctas(int threads, int most_threads, size_t smem) {
    const size_t each = (size_t)round_up((long long)(smem + 512 + 1024), 1024);      // static and reserved shared memory
    return (int)std::max<size_t>(1, std::min<size_t>({32, (size_t)(most_threads / threads), (227 * 1024 + 1024) / each}));
}

// How the rows are shared out for the backward pass; depends on sizes only, for the workspace query.
struct Sharing {
    long long groups, group_len, split_len, groups_per_worker;
    int splits, workers;
};
inline Sharing share_rows(long long rows, long long groups, int64_t width, size_t elem, bool sum_gate) {
    const long long most = (long long)sm_count() * (width <= 8192 ? resident_ctas(staged_threads(width), 1024, backward_bytes(width, elem, sum_gate)) : 1);
    Sharing s{groups, rows / groups, 0, 0, 1, 1};
    if (groups > 1 && groups >= most) {
        s.groups_per_worker = ceil_div(groups, most);
        s.workers = (int)ceil_div(groups, s.groups_per_worker);
        return s;
    }
    const long long want = std::max(1LL, std::min(most / groups, s.group_len));
    s.split_len = ceil_div(s.group_len, want);
    s.splits = (int)ceil_div(s.group_len, s.split_len);
    s.workers = (int)(groups * s.splits);
    return s;
}

template <class T, class K>
bool aligned_row(const RowView<K>& v) { return (((uintptr_t)v.p) & 15) == 0 && (v.s0 * (long long)sizeof(T)) % 16 == 0 && (v.s1 * (long long)sizeof(T)) % 16 == 0; }
inline bool aligned16(const void* p) { return (((uintptr_t)p) & 15) == 0; }

// Rows that are not staged, with element loads.
#define TPB_ELEMENT_LAUNCH(KERNEL, T, plan, grid, smem, st, args)                                                          \
    do {                                                                                                                   \
        if ((plan).warp) {                                                                                                 \
            if ((plan).nv == 1) TPB_LAUNCH(#KERNEL, (KERNEL<T, 1, false, true>), grid, (plan).threads, (smem), st, args);  \
            else TPB_LAUNCH(#KERNEL, (KERNEL<T, 2, false, true>), grid, (plan).threads, (smem), st, args);                 \
        } else {                                                                                                           \
            if ((plan).nv == 1) TPB_LAUNCH(#KERNEL, (KERNEL<T, 1, false, false>), grid, (plan).threads, (smem), st, args); \
            else TPB_LAUNCH(#KERNEL, (KERNEL<T, 2, false, false>), grid, (plan).threads, (smem), st, args);                \
        }                                                                                                                  \
    } while (0)

// shared memory for the kept elements of the CTA's rows, where rows are no whole blocks of the generator
inline size_t mask_bytes(const RowPlan& p, int width, const DropSpec& d) {
    return p.vec || d.units == 0 ? 0 : (size_t)keep_bytes(width) * (p.warp ? p.threads / 32 : 1);
}

template <class T>
int forward_run(const ForwardArgs<T>& k, cudaStream_t st) {
    const bool vec = k.width % 8 == 0 && aligned_row<T>(k.x) && (!k.h.p || aligned_row<T>(k.h)) && (!k.gate.p || aligned_row<T>(k.gate)) &&
                     aligned16(k.post) && aligned16(k.next) && aligned16(k.x_out) && aligned16(k.y);
    if (vec && k.width > 256 && k.width <= 8192) {
        const int threads = staged_threads(k.width);
        const size_t smem = (size_t)threads * kStages * kForwardArrays * 8 * sizeof(T);
        const int rc = allow_shared((const void*)block_forward_staged_kernel<T>, smem);
        if (rc != TPB200_OK) return rc;
        const long long ctas = std::min<long long>(k.rows, (long long)sm_count() * resident_ctas(threads, 2048, smem));
        TPB_LAUNCH("block_forward_staged_kernel", block_forward_staged_kernel<T>, dim3((unsigned)ctas), threads, smem, st, k);
        return TPB200_OK;
    }
    const RowPlan p = plan_rows(k.width, vec);
    const dim3 grid((unsigned)(p.warp ? ceil_div(k.rows, p.threads / 32) : k.rows));
    // aligned rows are short ones or longer than the staged kernel takes
    if (vec && p.warp) TPB_LAUNCH("block_forward_kernel", (block_forward_kernel<T, 1, true, true>), grid, p.threads, 0, st, k);
    else if (vec) TPB_LAUNCH("block_forward_kernel", (block_forward_kernel<T, 2, true, false>), grid, p.threads, 0, st, k);
    else TPB_ELEMENT_LAUNCH(block_forward_kernel, T, p, grid, mask_bytes(p, k.width, k.drop), st, k);
    return TPB200_OK;
}

template <class T>
int backward_run(const BackwardArgs<T>& k, T* dpost, T* dnext, long long gate_groups, cudaStream_t st) {
    const bool vec = k.width % 8 == 0 && (!k.grad_x.p || aligned_row<T>(k.grad_x)) && (!k.grad_y.p || aligned_row<T>(k.grad_y)) &&
                     (!k.h.p || aligned_row<T>(k.h)) && (!k.x_out.p || aligned_row<T>(k.x_out)) && (!k.gate.p || aligned_row<T>(k.gate)) &&
                     aligned16(k.post) && aligned16(k.next) && aligned16(k.dx) && aligned16(k.dh) && aligned16(k.dgate);
    RowPlan p = plan_rows(k.width, vec);
    const dim3 grid((unsigned)(p.warp ? ceil_div(k.workers, p.threads / 32) : k.workers));
    const size_t smem = backward_bytes(k.width, sizeof(T), k.gate.p && !k.gate_rows);
    if (vec && k.width <= 8192 && smem <= 226 * 1024) {
        const int threads = staged_threads(k.width);
        const bool sums = k.gate.p && !k.gate_rows;
        const auto kernel = k.from_x ? (sums ? block_backward_staged_kernel<T, true, true> : block_backward_staged_kernel<T, false, true>)
                                     : (sums ? block_backward_staged_kernel<T, true, false> : block_backward_staged_kernel<T, false, false>);
        const int rc = allow_shared((const void*)kernel, smem);
        if (rc != TPB200_OK) return rc;
        TPB_LAUNCH("block_backward_staged_kernel", kernel, dim3((unsigned)k.workers), threads, smem, st, k);
    } else {
        // aligned rows are longer than the staged kernel takes: more than 8192 elements, or a float32 row whose stages do not fit
        static_assert(sizeof(T) == 4 || 1024 * ((kStages * kStageArrays + 2) * 8 * sizeof(T) + 32) <= 226 * 1024, "16-bit rows of 8192 elements are staged");
        auto kernel = block_backward_kernel<T, 2, true, false>;
        if (!vec) {
            TPB_ELEMENT_LAUNCH(block_backward_kernel, T, p, grid, mask_bytes(p, k.width, k.drop), st, k);
        } else {
            if constexpr (sizeof(T) == 4) {
                if (p.nv == 1) kernel = block_backward_kernel<T, 1, true, false>;
            }
            TPB_LAUNCH("block_backward_kernel", kernel, grid, p.threads, 0, st, k);
        }
    }
    const bool sum_gate = k.gate.p && !k.gate_rows && k.groups_per_worker == 0;
    if (!dpost && !dnext && !sum_gate) return TPB200_OK;
    const dim3 sums((unsigned)ceil_div(k.width, 32), (unsigned)(2 + (sum_gate ? gate_groups : 0)));
    TPB_LAUNCH("block_sums_kernel", block_sums_kernel<T>, sums, 256, 0, st, (const float*)k.part_post, (const float*)k.part_next,
               (const float*)k.part_gate, dpost, dnext, sum_gate ? k.dgate : (T*)nullptr, k.workers, k.splits, k.width);
    return TPB200_OK;
}

template <class T>
RowView<const T> view_of(const void* p, const int64_t* s) {
    return RowView<const T>{(const T*)p, p && s ? s[0] : 0, p && s ? s[1] : 0};
}

int check_block(const char* what, int dtype, int64_t outer, int64_t inner, int64_t width) {
    TPB_TRY_ROWS(what, dtype, outer, inner, width);
    if (width > kMaxWidth) return fail(TPB200_ERR_UNSUPPORTED, "%s: rows of at most %d elements (got %lld)", what, kMaxWidth, (long long)width);
    return TPB200_OK;
}

// Rows of no elements have no mean square: their rstd is NaN (all bits set).
inline int empty_rows(long long rows, float* rstd_a, float* rstd_b, cudaStream_t st) {
    for (float* p : {rstd_a, rstd_b})
        if (rows > 0 && p) TPB_CUDA_OK(cudaMemsetAsync(p, 0xff, (size_t)rows * sizeof(float), st));
    return TPB200_OK;
}

// groups of rows that share a row of the gate, by the gate's kind
inline long long gate_groups_of(int kind, int64_t outer) { return kind == TPB200_GATE_SEQUENCE ? outer : 1; }

struct BlockPointers { float *post, *next, *gate; size_t bytes; };
inline BlockPointers block_workspace(void* ws, const Sharing& s, int64_t width, bool post, bool next, bool gate) {
    BlockPointers b{nullptr, nullptr, nullptr, 0};
    const size_t each = (size_t)round_up((long long)s.workers * width * 4, 256);
    if (post) { b.post = (float*)((char*)ws + b.bytes); b.bytes += each; }
    if (next) { b.next = (float*)((char*)ws + b.bytes); b.bytes += each; }
    if (gate && s.groups_per_worker == 0) { b.gate = (float*)((char*)ws + b.bytes); b.bytes += each; }
    return b;
}

template <class T>
int forward_call(const void* x, const int64_t* xs, const void* h, const int64_t* hs, const void* gate, const int64_t* gs, const void* post,
                 const void* next, int64_t outer, int64_t inner, int64_t width, double scale, double eps, const DropSpec& drop, void* x_out,
                 void* y, float* rstd_post, float* rstd_next, cudaStream_t st) {
    ForwardArgs<T> k{};
    k.x = view_of<T>(x, xs);
    k.h = view_of<T>(h, hs);
    k.gate = view_of<T>(gate, gs);
    k.post = (const T*)post;
    k.next = (const T*)next;
    k.x_out = (T*)x_out;
    k.y = (T*)y;
    k.rstd_post = rstd_post;
    k.rstd_next = rstd_next;
    k.rows = outer * inner;
    k.inner = inner;
    k.width = (int)width;
    k.scale = (float)scale;
    k.eps = (float)eps;
    k.drop = drop;
    return forward_run<T>(k, st);
}

struct BackwardCall {
    const void *grad_x, *grad_y, *h, *x_out, *gate, *post, *next;
    const int64_t *gxs, *gys, *hs, *xs, *gs;
    const float *rstd_post, *rstd_next;
    void *dx, *dh, *dgate, *dpost, *dnext;
    int64_t outer, inner, width;
    int gate_kind, from_x;
    double scale;
    DropSpec drop;
    Sharing share;
    BlockPointers ws;
};
template <class T>
int backward_call(const BackwardCall& c, cudaStream_t st) {
    BackwardArgs<T> k{};
    k.grad_x = view_of<T>(c.grad_x, c.gxs);
    k.grad_y = view_of<T>(c.grad_y, c.gys);
    k.h = view_of<T>(c.h, c.hs);
    k.x_out = view_of<T>(c.x_out, c.xs);
    k.from_x = c.from_x;
    k.gate = view_of<T>(c.gate, c.gs);
    k.post = (const T*)c.post;
    k.next = (const T*)c.next;
    k.rstd_post = c.rstd_post;
    k.rstd_next = c.rstd_next;
    k.dx = (T*)c.dx;
    k.dh = (T*)c.dh;
    k.dgate = (T*)c.dgate;
    k.part_post = c.ws.post;
    k.part_next = c.ws.next;
    k.part_gate = c.ws.gate;
    k.rows = c.outer * c.inner;
    k.inner = c.inner;
    k.group_len = c.share.group_len;
    k.split_len = c.share.split_len;
    k.groups_per_worker = c.share.groups_per_worker;
    k.splits = c.share.splits;
    k.workers = c.share.workers;
    k.width = (int)c.width;
    k.gate_rows = c.gate_kind == TPB200_GATE_ELEMENT;
    k.scale = (float)c.scale;
    k.drop = c.drop;
    return backward_run<T>(k, (T*)c.dpost, (T*)c.dnext, c.share.groups, st);
}

}  // namespace tpb

using namespace tpb;

extern "C" int tpb200_rms_norm(const void* x, int dtype, int64_t outer, int64_t inner, int64_t width, const int64_t* strides,
                               const void* weight, double eps, void* y, float* rstd, void* stream) {
    const int rc = check_block("rms_norm", dtype, outer, inner, width);
    if (rc != TPB200_OK) return rc;
    if (!(eps >= 0.0)) return fail(TPB200_ERR_INVALID, "rms_norm: eps must not be negative");
    if (outer * inner * width == 0) return empty_rows(outer * inner, rstd, nullptr, (cudaStream_t)stream);
    if (!x || !strides || !weight || !y || !rstd) return fail(TPB200_ERR_INVALID, "rms_norm: NULL pointer argument");
    cudaStream_t st = (cudaStream_t)stream;
    [[maybe_unused]] const int64_t e = dtype_bytes(dtype), n = outer * inner;
    TPB_CHECK_RANGES(st, rows_range(x, outer, inner, width, strides, e), HostRange{weight, (size_t)(width * e)}, HostRange{y, (size_t)(n * width * e)},
                     HostRange{rstd, (size_t)n * 4});
    const DropSpec none{0, 0, 0, 0, 1.0f};
    if (dtype == TPB200_F32) return forward_call<float>(x, strides, nullptr, nullptr, nullptr, nullptr, nullptr, weight, outer, inner, width, 1.0, eps, none, nullptr, y, nullptr, rstd, st);
    if (dtype == TPB200_BF16) return forward_call<__nv_bfloat16>(x, strides, nullptr, nullptr, nullptr, nullptr, nullptr, weight, outer, inner, width, 1.0, eps, none, nullptr, y, nullptr, rstd, st);
    return forward_call<__half>(x, strides, nullptr, nullptr, nullptr, nullptr, nullptr, weight, outer, inner, width, 1.0, eps, none, nullptr, y, nullptr, rstd, st);
}

extern "C" int tpb200_block_residual(const void* x, const int64_t* x_strides, const void* h, const int64_t* h_strides, const void* gate,
                                     const int64_t* gate_strides, const void* post_weight, const void* next_weight, int dtype,
                                     int64_t outer, int64_t inner, int64_t width, double scale, double eps, double p, uint64_t seed,
                                     uint64_t offset, void* x_out, void* y, float* rstd_post, float* rstd_next, void* stream) {
    const int rc = check_block("block_residual", dtype, outer, inner, width);
    if (rc != TPB200_OK) return rc;
    if (!(eps >= 0.0)) return fail(TPB200_ERR_INVALID, "block_residual: eps must not be negative");
    DropSpec drop;
    if (!make_drop(p, seed, offset, &drop)) return fail(TPB200_ERR_INVALID, "block_residual: p must lie in [0, 1]");
    // (weights of no elements may be NULL: the outputs say which norms there are)
    if (outer * inner * width == 0) return empty_rows(outer * inner, rstd_post, rstd_next, (cudaStream_t)stream);
    if (!x || !h || !x_out || !x_strides || !h_strides || (gate && !gate_strides) || (post_weight && !rstd_post) || (next_weight && (!y || !rstd_next)))
        return fail(TPB200_ERR_INVALID, "block_residual: NULL pointer argument");
    cudaStream_t st = (cudaStream_t)stream;
    [[maybe_unused]] const int64_t e = dtype_bytes(dtype), n = outer * inner;
    TPB_CHECK_RANGES(st, rows_range(x, outer, inner, width, x_strides, e), rows_range(h, outer, inner, width, h_strides, e),
                     rows_range(gate, outer, inner, width, gate_strides, e), HostRange{post_weight, (size_t)(width * e)},
                     HostRange{next_weight, (size_t)(width * e)}, HostRange{x_out, (size_t)(n * width * e)}, HostRange{y, y ? (size_t)(n * width * e) : 0},
                     HostRange{rstd_post, (size_t)n * 4}, HostRange{rstd_next, (size_t)n * 4});
    if (dtype == TPB200_F32) return forward_call<float>(x, x_strides, h, h_strides, gate, gate_strides, post_weight, next_weight, outer, inner, width, scale, eps, drop, x_out, y, rstd_post, rstd_next, st);
    if (dtype == TPB200_BF16) return forward_call<__nv_bfloat16>(x, x_strides, h, h_strides, gate, gate_strides, post_weight, next_weight, outer, inner, width, scale, eps, drop, x_out, y, rstd_post, rstd_next, st);
    return forward_call<__half>(x, x_strides, h, h_strides, gate, gate_strides, post_weight, next_weight, outer, inner, width, scale, eps, drop, x_out, y, rstd_post, rstd_next, st);
}

extern "C" size_t tpb200_block_residual_backward_workspace_bytes(int64_t outer, int64_t inner, int64_t width, int has_post, int has_next,
                                                                 int gate_kind) {
    if (outer <= 0 || inner <= 0 || width <= 0 || outer > 0x7fffffffLL || inner > 0x7fffffffLL || outer * inner > 0x7fffffffLL || width > kMaxWidth) return 0;
    // the element type is not known here: the workers of the smallest take the most
    const bool sum_gate = gate_kind == TPB200_GATE_VECTOR || gate_kind == TPB200_GATE_SEQUENCE;
    const Sharing s = share_rows(outer * inner, gate_groups_of(gate_kind, outer), width, 2, sum_gate);
    return block_workspace(nullptr, s, width, has_post != 0, has_next != 0, sum_gate).bytes;
}

static int backward_entry(const void* grad_x_out, const int64_t* grad_x_strides, const void* grad_y,
                          const int64_t* grad_y_strides, const void* h, const int64_t* h_strides, const void* x_out,
                          const int64_t* x_out_strides, const void* gate, const int64_t* gate_strides, int gate_kind,
                          const void* post_weight, const void* next_weight, const float* rstd_post,
                          const float* rstd_next, int dtype, int64_t outer, int64_t inner, int64_t width, double scale,
                          double p, uint64_t seed, uint64_t offset, void* grad_x, void* grad_h, void* grad_post,
                          void* grad_next, void* grad_gate, void* workspace, size_t workspace_bytes, void* stream, int from_x) {
    const int rc = check_block("block_residual_backward", dtype, outer, inner, width);
    if (rc != TPB200_OK) return rc;
    if (gate_kind < TPB200_GATE_NONE || gate_kind > TPB200_GATE_ELEMENT) return fail(TPB200_ERR_INVALID, "block_residual_backward: unknown gate kind %d", gate_kind);
    BackwardCall c{};
    if (!make_drop(p, seed, offset, &c.drop)) return fail(TPB200_ERR_INVALID, "block_residual_backward: p must lie in [0, 1]");
    const int64_t n = outer * inner, e = dtype_bytes(dtype);
    cudaStream_t st = (cudaStream_t)stream;
    const bool gated = gate_kind != TPB200_GATE_NONE && h;
    if (n * width == 0) {   // sums over no rows are zero
        if (width > 0 && post_weight && grad_post) TPB_CUDA_OK(cudaMemsetAsync(grad_post, 0, (size_t)(width * e), st));
        if (width > 0 && next_weight && grad_next) TPB_CUDA_OK(cudaMemsetAsync(grad_next, 0, (size_t)(width * e), st));
        if (width > 0 && grad_gate && gate_kind == TPB200_GATE_VECTOR) TPB_CUDA_OK(cudaMemsetAsync(grad_gate, 0, (size_t)(width * e), st));
        if (width > 0 && grad_gate && gate_kind == TPB200_GATE_SEQUENCE && outer > 0) TPB_CUDA_OK(cudaMemsetAsync(grad_gate, 0, (size_t)(outer * width * e), st));
        return TPB200_OK;
    }
    if (!grad_x || (grad_x_out && !grad_x_strides) || (next_weight && (!grad_y || !grad_y_strides || !x_out || !x_out_strides || !rstd_next || !grad_next)) ||
        (h && (!h_strides || !grad_h)) || (h && post_weight && (!rstd_post || !grad_post)) || (gated && (!gate || !gate_strides || !grad_gate)))
        return fail(TPB200_ERR_INVALID, "block_residual_backward: NULL pointer argument");
    c.share = share_rows(n, gated ? gate_groups_of(gate_kind, outer) : 1, width, (size_t)e, gated && gate_kind != TPB200_GATE_ELEMENT);
    c.ws = block_workspace(workspace, c.share, width, h && post_weight, next_weight != nullptr, gated && gate_kind != TPB200_GATE_ELEMENT);
    if (c.ws.bytes > 0 && (!workspace || workspace_bytes < c.ws.bytes))
        return fail(TPB200_ERR_WORKSPACE, "block_residual_backward: workspace missing or too small (%zu of %zu bytes)", workspace_bytes, c.ws.bytes);
    c.grad_x = grad_x_out; c.gxs = grad_x_strides;
    c.grad_y = next_weight ? grad_y : nullptr; c.gys = grad_y_strides;
    c.h = h; c.hs = h_strides;
    c.x_out = next_weight ? x_out : nullptr; c.xs = x_out_strides;
    c.gate = gated ? gate : nullptr; c.gs = gate_strides;
    c.post = h ? post_weight : nullptr; c.next = next_weight;
    c.rstd_post = rstd_post; c.rstd_next = rstd_next;
    c.dx = grad_x; c.dh = grad_h; c.dgate = gated ? grad_gate : nullptr;
    c.dpost = c.post ? grad_post : nullptr; c.dnext = next_weight ? grad_next : nullptr;
    c.outer = outer; c.inner = inner; c.width = width;
    c.gate_kind = gated ? gate_kind : TPB200_GATE_NONE;
    c.from_x = from_x && next_weight;
    c.scale = scale;
    const int64_t gate_rows = gate_kind == TPB200_GATE_ELEMENT ? n : gate_groups_of(gate_kind, outer);
    TPB_CHECK_RANGES(st, rows_range(c.grad_x, outer, inner, width, grad_x_strides, e), rows_range(c.grad_y, outer, inner, width, grad_y_strides, e),
                     rows_range(h, outer, inner, width, h_strides, e), rows_range(c.x_out, outer, inner, width, x_out_strides, e),
                     rows_range(c.gate, outer, inner, width, gate_strides, e), HostRange{post_weight, (size_t)(width * e)},
                     HostRange{next_weight, (size_t)(width * e)}, HostRange{rstd_post, (size_t)n * 4}, HostRange{rstd_next, (size_t)n * 4},
                     HostRange{grad_x, (size_t)(n * width * e)}, HostRange{c.h ? grad_h : nullptr, (size_t)(n * width * e)},
                     HostRange{c.dgate, (size_t)(gate_rows * width * e)}, HostRange{c.dpost, (size_t)(width * e)},
                     HostRange{c.dnext, (size_t)(width * e)}, HostRange{workspace, c.ws.bytes});
    if (dtype == TPB200_F32) return backward_call<float>(c, st);
    if (dtype == TPB200_BF16) return backward_call<__nv_bfloat16>(c, st);
    return backward_call<__half>(c, st);
}

extern "C" int tpb200_block_residual_backward(
    const void* grad_x_out, const int64_t* grad_x_strides, const void* grad_y, const int64_t* grad_y_strides, const void* h,
    const int64_t* h_strides, const void* x_out, const int64_t* x_out_strides, const void* gate, const int64_t* gate_strides, int gate_kind,
    const void* post_weight, const void* next_weight, const float* rstd_post, const float* rstd_next, int dtype, int64_t outer, int64_t inner,
    int64_t width, double scale, double p, uint64_t seed, uint64_t offset, void* grad_x, void* grad_h, void* grad_post, void* grad_next,
    void* grad_gate, void* workspace, size_t workspace_bytes, void* stream) {
    return backward_entry(grad_x_out, grad_x_strides, grad_y, grad_y_strides, h, h_strides, x_out, x_out_strides, gate, gate_strides, gate_kind, post_weight,
                          next_weight, rstd_post, rstd_next, dtype, outer, inner, width, scale, p, seed, offset, grad_x, grad_h, grad_post,
                          grad_next, grad_gate, workspace, workspace_bytes, stream, 0);
}

extern "C" int tpb200_block_residual_backward_from_x(
    const void* grad_x_out, const int64_t* grad_x_strides, const void* grad_y, const int64_t* grad_y_strides, const void* h,
    const int64_t* h_strides, const void* x, const int64_t* x_strides, const void* gate, const int64_t* gate_strides, int gate_kind,
    const void* post_weight, const void* next_weight, const float* rstd_post, const float* rstd_next, int dtype, int64_t outer, int64_t inner,
    int64_t width, double scale, double p, uint64_t seed, uint64_t offset, void* grad_x, void* grad_h, void* grad_post, void* grad_next,
    void* grad_gate, void* workspace, size_t workspace_bytes, void* stream) {
    if (!h && outer * inner * width != 0) return fail(TPB200_ERR_INVALID, "block_residual_backward: NULL pointer argument");
    return backward_entry(grad_x_out, grad_x_strides, grad_y, grad_y_strides, h, h_strides, x, x_strides, gate, gate_strides, gate_kind, post_weight,
                          next_weight, rstd_post, rstd_next, dtype, outer, inner, width, scale, p, seed, offset, grad_x, grad_h, grad_post,
                          grad_next, grad_gate, workspace, workspace_bytes, stream, 1);
}

extern "C" size_t tpb200_rms_norm_backward_workspace_bytes(int64_t outer, int64_t inner, int64_t width) {
    return tpb200_block_residual_backward_workspace_bytes(outer, inner, width, 0, 1, TPB200_GATE_NONE);
}

extern "C" int tpb200_rms_norm_backward(const void* grad_y, const int64_t* grad_strides, const void* x, const int64_t* strides, int dtype,
                                        int64_t outer, int64_t inner, int64_t width, const void* weight, const float* rstd, void* grad_x,
                                        void* grad_weight, void* workspace, size_t workspace_bytes, void* stream) {
    if (!weight && outer * inner * width != 0) return fail(TPB200_ERR_INVALID, "rms_norm_backward: NULL pointer argument");
    return tpb200_block_residual_backward(nullptr, nullptr, grad_y, grad_strides, nullptr, nullptr, x, strides, nullptr, nullptr, TPB200_GATE_NONE,
                                          nullptr, weight, nullptr, rstd, dtype, outer, inner, width, 1.0, 0.0, 0, 0, grad_x, nullptr, nullptr,
                                          grad_weight, nullptr, workspace, workspace_bytes, stream);
}
