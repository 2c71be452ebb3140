// The global norm of many gradient tensors and their clipping (declared in include/instascene_ops.h).
//
//   norm = (sum |g|^p)^(1/p), p = 1, 2, or max |g|;   coef = min(1, max_norm / (norm + 1e-6));   g *= coef
//
// Bound by memory: the norm reads every gradient once, the scaling reads and writes once more - and nothing where coef is 1
// (a whole launch leaves after it has read the partial sums).  The tensors are cut into chunks of GN_CHUNK elements; a table of at
// most GN_TENSORS tensors travels in the kernel's arguments, so that no copy to the device precedes a launch and a captured graph holds
// all of it.  Workgroup b sums chunks b, b + grid, ... in 64 bits (no overflow, and long sums lose nothing) into partial b: no atomics, the
// order of every sum is fixed by the sizes and alignments alone.  The scaling kernel's workgroups each add the partials up for themselves (at most
// GN_PARTS of them, from L2) instead of waiting for a launch of their own that does.
#pragma once
#include <hip/hip_runtime.h>

namespace iso {

constexpr int GN_TENSORS = 128, GN_PARTS = 1024, GN_CHUNK = 16384, GN_THREADS = 512, GN_SMALL = 16384;
enum { GN_F32 = 0, GN_BF16 = 1, GN_F16 = 2 };
struct GradTable {
    void* p[GN_TENSORS];
    long long n[GN_TENSORS];
    unsigned first[GN_TENSORS + 1];     // first chunk of tensor i; first[count] = number of chunks
    unsigned char type[GN_TENSORS];
    unsigned char head[GN_TENSORS];     // elements in front of the first 16-byte boundary; they go with chunk 0, the chunks count from there
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
template <int P, int THREADS> __device__ __forceinline__ double norm_block(double v) {
    __shared__ double lds[THREADS / 64];
    for (int o = 32; o >= 1; o >>= 1) v = norm_join<P>(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int i = 1; i < THREADS / 64; i++) v = norm_join<P>(v, lds[i]);
    return v;
}
template <class T> struct GradVec { static constexpr int N = 16 / (int)sizeof(T); typedef T type __attribute__((ext_vector_type(16 / sizeof(T)))); };
// the elements of chunk c of a tensor: `head` of them in front of the first 16-byte boundary (with chunk 0), n from p on
template <class T> struct Chunk { T* front; int head; T* p; int n; };
template <class T> __device__ __forceinline__ Chunk<T> grad_chunk(const GradTable& tb, int k, unsigned c) {
    T* t = (T*)tb.p[k];
    const long long at = (long long)(c - tb.first[k]) * GN_CHUNK, left = tb.n[k] - tb.head[k] - at;
    return {t, at == 0 ? tb.head[k] : 0, t + tb.head[k] + at, (int)(left < GN_CHUNK ? left : GN_CHUNK)};
}
// U vectors per thread in flight; a chunk is at most U or 2 U of them per thread
template <int P, class T, int THREADS> __device__ __forceinline__ void chunk_norm(double& acc, const Chunk<T>& c) {
    constexpr int N = GradVec<T>::N, U = 4;
    typedef typename GradVec<T>::type V;
    const int vecs = c.n / N;
    const V* p = reinterpret_cast<const V*>(c.p);
    for (int j = threadIdx.x; j < vecs; j += U * THREADS) {
        V q[U];
#pragma unroll
        for (int u = 0; u < U; u++) q[u] = p[min(j + u * THREADS, vecs - 1)];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < N; e++) norm_add<P>(acc, j + u * THREADS < vecs ? (float)q[u][e] : 0.0f);
    }
    if ((int)threadIdx.x < c.n - vecs * N) norm_add<P>(acc, (float)c.p[vecs * N + threadIdx.x]);
    if ((int)threadIdx.x < c.head) norm_add<P>(acc, (float)c.front[threadIdx.x]);
}
template <class T, int THREADS> __device__ __forceinline__ void chunk_scale(const Chunk<T>& c, float coef) {
    constexpr int N = GradVec<T>::N, U = 4;
    typedef typename GradVec<T>::type V;
    const int vecs = c.n / N;
    V* p = reinterpret_cast<V*>(c.p);
    for (int j = threadIdx.x; j < vecs; j += U * THREADS) {
        V q[U];
#pragma unroll
        for (int u = 0; u < U; u++) q[u] = p[min(j + u * THREADS, vecs - 1)];
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int e = 0; e < N; e++) q[u][e] = (T)((float)q[u][e] * coef);
            if (j + u * THREADS < vecs) p[j + u * THREADS] = q[u];
        }
    }
    const int last = vecs * N + threadIdx.x;
    if (last < c.n) c.p[last] = (T)((float)c.p[last] * coef);
    if ((int)threadIdx.x < c.head) c.front[threadIdx.x] = (T)((float)c.front[threadIdx.x] * coef);
}
template <int P, int THREADS> __device__ __forceinline__ void grad_chunk_norm(const GradTable& tb, unsigned c, double& acc) {
    const int k = grad_tensor(tb, c);
    if (tb.type[k] == GN_F32) chunk_norm<P, float, THREADS>(acc, grad_chunk<float>(tb, k, c));
    else if (tb.type[k] == GN_BF16) chunk_norm<P, __bf16, THREADS>(acc, grad_chunk<__bf16>(tb, k, c));
    else chunk_norm<P, _Float16, THREADS>(acc, grad_chunk<_Float16>(tb, k, c));
}
template <int THREADS> __device__ __forceinline__ void grad_chunk_scale(const GradTable& tb, unsigned c, float coef) {
    const int k = grad_tensor(tb, c);
    if (tb.type[k] == GN_F32) chunk_scale<float, THREADS>(grad_chunk<float>(tb, k, c), coef);
    else if (tb.type[k] == GN_BF16) chunk_scale<__bf16, THREADS>(grad_chunk<__bf16>(tb, k, c), coef);
    else chunk_scale<_Float16, THREADS>(grad_chunk<_Float16>(tb, k, c), coef);
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
    return norm_block<P, GN_THREADS>(v);
}

template <int P> __global__ __launch_bounds__(GN_THREADS) void grad_norm_kernel(GradTable tb, double* __restrict__ part) {
    const unsigned chunks = tb.first[tb.count];
    double acc = 0.0;
    for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) grad_chunk_norm<P, GN_THREADS>(tb, c, acc);
    acc = norm_block<P, GN_THREADS>(acc);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}
// A few small tensors (GN_SMALL elements at most) in one workgroup: the norm and the scaling in one launch (six tensors, 4 000 / 16 000 elements
// together: 7.0 / 8.0 us a call; two launches 7.9 for the norm, 8.5 with clipping, and one workgroup 10 us at 58 000)
template <int P> __global__ __launch_bounds__(1024) void grad_small_kernel(GradTable tb, int clip, float max_norm, float* __restrict__ out) {
    const unsigned chunks = tb.first[tb.count];
    double acc = 0.0;
    for (unsigned c = 0; c < chunks; c++) grad_chunk_norm<P, 1024>(tb, c, acc);
    float norm, coef;
    norm_finish(norm_block<P, 1024>(acc), P, max_norm, norm, coef);
    if (threadIdx.x == 0) { out[0] = norm; out[1] = coef; }
    if (!clip || coef == 1.0f) return;
    for (unsigned c = 0; c < chunks; c++) grad_chunk_scale<1024>(tb, c, coef);
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
        grad_chunk_scale<GN_THREADS>(tb, chunks - 1 - b, coef);        // backwards: what the norm read last is still in the caches
    }
}

// The norm of the RAW parameters' gradients of a Gaussian model, from the gradients of the activated tensors that the rasterizer gives
// (iso_gaussian_adam_step's chain rule, in the same 32-bit arithmetic): opacity g s (1 - s), s = sigmoid(p); scaling g exp(p); rotation, with
// q = p / max(|p|, 1e-12), (g - q <q, g>) / max(|p|, 1e-12); position and spherical harmonics as they are.  One pass over the 59 floats per
// Gaussian (degree 3) and the 7 of the parameters; the spherical harmonics are a flat stream.
struct GaussNormArgs {
    long long P, sh;        // Gaussians, spherical-harmonics floats in all
    const float *xyz, *shs, *opa, *scale, *rot;             // gradients; NULL: no part in the norm
    const float *p_opa, *p_scale, *p_rot;                   // raw parameters
};
__device__ __forceinline__ void flat_squares(double& acc, const float* p, long long n) {
    typedef float V __attribute__((ext_vector_type(4), aligned(4)));
    const long long vecs = n / 4, step = (long long)gridDim.x * GN_THREADS;
    for (long long j = (long long)blockIdx.x * GN_THREADS + threadIdx.x; j < vecs; j += 4 * step) {
        V q[4];
#pragma unroll
        for (int u = 0; u < 4; u++) q[u] = reinterpret_cast<const V*>(p)[min(j + u * step, vecs - 1)];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) norm_add<2>(acc, j + u * step < vecs ? q[u][e] : 0.0f);
    }
    if (blockIdx.x == 0 && (long long)threadIdx.x < n - 4 * vecs) norm_add<2>(acc, p[4 * vecs + threadIdx.x]);
}
__global__ __launch_bounds__(GN_THREADS) void gaussian_norm_kernel(GaussNormArgs a, double* __restrict__ part) {
    double acc = 0.0;
    if (a.shs) flat_squares(acc, a.shs, a.sh);
    if (a.xyz) flat_squares(acc, a.xyz, 3 * a.P);
    const long long step = (long long)gridDim.x * GN_THREADS;
    for (long long i = (long long)blockIdx.x * GN_THREADS + threadIdx.x; i < a.P; i += step) {
        if (a.opa) {
            const float s = 1.0f / (1.0f + expf(-a.p_opa[i]));
            norm_add<2>(acc, a.opa[i] * (s * (1.0f - s)));
        }
        if (a.scale) {
            norm_add<2>(acc, a.scale[2 * i] * expf(a.p_scale[2 * i]));
            norm_add<2>(acc, a.scale[2 * i + 1] * expf(a.p_scale[2 * i + 1]));
        }
        if (a.rot) {
            typedef float V __attribute__((ext_vector_type(4), aligned(4)));
            const V q = reinterpret_cast<const V*>(a.p_rot)[i], g = reinterpret_cast<const V*>(a.rot)[i];
            const float n = fmaxf(__builtin_sqrtf(q.x * q.x + q.y * q.y + q.z * q.z + q.w * q.w), 1e-12f), r = 1.0f / n;
            const float4 y = make_float4(q.x * r, q.y * r, q.z * r, q.w * r);
            const float d = y.x * g.x + y.y * g.y + y.z * g.z + y.w * g.w;
            norm_add<2>(acc, (g.x - y.x * d) * r);
            norm_add<2>(acc, (g.y - y.y * d) * r);
            norm_add<2>(acc, (g.z - y.z * d) * r);
            norm_add<2>(acc, (g.w - y.w * d) * r);
        }
    }
    acc = norm_block<2, GN_THREADS>(acc);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

}  // namespace iso
