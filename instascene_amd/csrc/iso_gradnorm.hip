// The global norm of many gradient tensors and their clipping (declared in include/instascene_ops.h).
//
//   norm = (sum |g|^p)^(1/p), p = 1, 2, or max |g|;   coef = min(1, max_norm / (norm + 1e-6));   g *= coef
//
// Bound by memory: the norm reads every gradient once, the scaling reads and writes once more - and nothing where coef is 1
// (a whole launch leaves after it has read the partial sums).  The tensors are cut into chunks of GN_CHUNK elements; a table of at
// most GN_TENSORS tensors travels in the kernel's arguments, so that no copy to the device precedes a launch and a captured graph holds
// all of it.  Workgroup b sums chunks b, b + grid, ... in 64 bits (no overflow, and long sums lose nothing) into partial b: no atomics, the
// order of every sum is fixed by the sizes alone.  The scaling kernel's workgroups each add the partials up for themselves (at most
// GN_PARTS of them, from L2) instead of waiting for a launch of their own that does.
#pragma once
#include <hip/hip_runtime.h>

namespace iso {

constexpr int GN_TENSORS = 128, GN_PARTS = 1024, GN_CHUNK = 8192, GN_THREADS = 256;
enum { GN_F32 = 0, GN_BF16 = 1, GN_F16 = 2 };
struct GradTable {
    void* p[GN_TENSORS];
    long long n[GN_TENSORS];
    unsigned first[GN_TENSORS + 1];     // first chunk of tensor i; first[count] = number of chunks
    unsigned char type[GN_TENSORS];
    int count;
};
// the tensor that holds chunk c
__device__ __forceinline__ int grad_tensor(const GradTable& tb, unsigned c) {
    int lo = 0, hi = tb.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tb.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// P = 1, 2: sums; 0: the largest magnitude (a NaN stays)
template <int P> __device__ __forceinline__ void norm_add(double& acc, float v) {
    if (P == 2) acc += (double)v * (double)v;
    else if (P == 1) acc += (double)__builtin_fabsf(v);
    else { const double m = (double)__builtin_fabsf(v); if (m > acc || m != m) acc = m; }
}
template <int P> __device__ __forceinline__ double norm_join(double a, double b) {
    if (P != 0) return a + b;
    return (b > a || b != b) ? b : a;
}
template <int P> __device__ __forceinline__ double norm_block(double v) {
    __shared__ double lds[GN_THREADS / 64];
    for (int o = 32; o >= 1; o >>= 1) v = norm_join<P>(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int i = 1; i < GN_THREADS / 64; i++) v = norm_join<P>(v, lds[i]);
    return v;
}
template <class T> struct GradVec { static constexpr int N = 16 / (int)sizeof(T); typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); };

template <int P, class T> __device__ __forceinline__ void chunk_norm(double& acc, const T* p, int n) {
    constexpr int N = GradVec<T>::N;
    typedef typename GradVec<T>::type V;
    int i = threadIdx.x * N;
    for (; i + N <= n; i += GN_THREADS * N) {
        const V q = *reinterpret_cast<const V*>(p + i);
#pragma unroll
        for (int e = 0; e < N; e++) norm_add<P>(acc, (float)q[e]);
    }
    for (int e = i; e < n && e < i + N; e++) norm_add<P>(acc, (float)p[e]);
}
template <class T> __device__ __forceinline__ void chunk_scale(T* p, int n, float coef) {
    constexpr int N = GradVec<T>::N;
    typedef typename GradVec<T>::type V;
    int i = threadIdx.x * N;
    for (; i + N <= n; i += GN_THREADS * N) {
        V q = *reinterpret_cast<const V*>(p + i);
#pragma unroll
        for (int e = 0; e < N; e++) q[e] = (T)((float)q[e] * coef);
        *reinterpret_cast<V*>(p + i) = q;
    }
    for (int e = i; e < n && e < i + N; e++) p[e] = (T)((float)p[e] * coef);
}

// out[0] = norm, out[1] = coef
__device__ __forceinline__ void norm_finish(double sum, int p, float max_norm, float& norm, float& coef) {
    norm = (float)(p == 2 ? __builtin_sqrt(sum) : sum);
    const float c = max_norm / (norm + 1e-6f);
    coef = c > 1.0f ? 1.0f : c;             // (a NaN stays)
}
template <int P> __device__ __forceinline__ double partials_join(const double* part, int n) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += GN_THREADS) v = norm_join<P>(v, part[i]);
    return norm_block<P>(v);
}

template <int P> __global__ __launch_bounds__(GN_THREADS) void grad_norm_kernel(GradTable tb, double* __restrict__ part) {
    const unsigned chunks = tb.first[tb.count];
    double acc = 0.0;
    for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int k = grad_tensor(tb, c);
        const long long at = (long long)(c - tb.first[k]) * GN_CHUNK, left = tb.n[k] - at;
        const int n = (int)(left < GN_CHUNK ? left : GN_CHUNK);
        if (tb.type[k] == GN_F32) chunk_norm<P>(acc, (const float*)tb.p[k] + at, n);
        else if (tb.type[k] == GN_BF16) chunk_norm<P>(acc, (const __bf16*)tb.p[k] + at, n);
        else chunk_norm<P>(acc, (const _Float16*)tb.p[k] + at, n);
    }
    acc = norm_block<P>(acc);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}
template <int P> __global__ __launch_bounds__(GN_THREADS) void grad_norm_finish_kernel(const double* __restrict__ part, int n, float max_norm, float* __restrict__ out) {
    const double sum = partials_join<P>(part, n);
    if (threadIdx.x == 0) norm_finish(sum, P, max_norm, out[0], out[1]);
}
template <int P> __global__ __launch_bounds__(GN_THREADS) void grad_clip_kernel(GradTable tb, const double* __restrict__ part, int n, float max_norm, float* __restrict__ out) {
    float norm, coef;
    norm_finish(partials_join<P>(part, n), P, max_norm, norm, coef);
    if (blockIdx.x == 0 && threadIdx.x == 0) { out[0] = norm; out[1] = coef; }
    if (coef == 1.0f) return;
    const unsigned chunks = tb.first[tb.count];
    for (unsigned b = blockIdx.x; b < chunks; b += gridDim.x) {
        const unsigned c = chunks - 1 - b;         // backwards: what the norm read last is still in the caches
        const int k = grad_tensor(tb, c);
        const long long at = (long long)(c - tb.first[k]) * GN_CHUNK, left = tb.n[k] - at;
        const int m = (int)(left < GN_CHUNK ? left : GN_CHUNK);
        if (tb.type[k] == GN_F32) chunk_scale((float*)tb.p[k] + at, m, coef);
        else if (tb.type[k] == GN_BF16) chunk_scale((__bf16*)tb.p[k] + at, m, coef);
        else chunk_scale((_Float16*)tb.p[k] + at, m, coef);
    }
}

}  // namespace iso
