// Rows of a table: root-mean-square norm (with the residual's addition, its backward pass, an output in 8 bits with scales) and
// the 8-bit row table (written from rows, read back).  Declared in include/instascene_ops.h.
//
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
//   8 bits, per group of G columns:  t = s w,  top = max |t|,  code = round(t Q / top),  scale = top rstd / Q
//       (Q = 448: e4m3, 127: int8; rstd > 0 is common to the row, so it cancels in the codes and only the scale carries it)
//   backward:  h = s rstd,  c = mean(gy w h),  ds = rstd (gy w - h c) + gs,  dw = sum over rows of gy h
//
// All of it is bound by memory: every element is read once, kept in registers between the reduction and the output, and
// written once.  `tpr` threads (a power of two) share a row, NV vectors of 16 input bytes each, vector j = t + k tpr, so
// that a wave's loads are contiguous; rows longer than the registers hold are read a second time (the *_long kernels).
// Sums of squares are held in 64 bits (two instructions per element, hidden behind the loads): no overflow for any finite row.
#pragma once
#include <hip/hip_runtime.h>

namespace iso {

constexpr float ROWS_TINY = 0x1p-116f;      // a group whose largest magnitude lies below is stored as zeros: Q / top and top / Q stay normal

template <class T> struct RowVec { static constexpr int N = 16 / (int)sizeof(T); };
// (alignment of one element: rows of odd widths and views of buckets start anywhere; gfx950 loads unaligned vectors)
template <class T, int N> struct Unaligned { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };

// v[i] = p[i] for i < left, 0 beyond
template <class T, int N> __device__ __forceinline__ void row_load(const T* p, int left, float (&v)[N]) {
    if (left >= N) {
        const typename Unaligned<T, N>::type q = *reinterpret_cast<const typename Unaligned<T, N>::type*>(p);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (float)q[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = i < left ? (float)p[i] : 0.0f;
    }
}
template <class T, int N> __device__ __forceinline__ void row_store(T* p, int left, const float (&v)[N]) {
    if (left >= N) {
        typename Unaligned<T, N>::type q;
#pragma unroll
        for (int i = 0; i < N; i++) q[i] = (T)v[i];          // round to nearest even
        *reinterpret_cast<typename Unaligned<T, N>::type*>(p) = q;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left) p[i] = (T)v[i];
    }
}
// the gain: 32 bits or the rows' type; NULL = 1
template <class T, int N> __device__ __forceinline__ void gain_load(const void* w, int w32, int at, int left, float (&v)[N]) {
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = 1.0f;
    } else if (w32) row_load<float, N>((const float*)w + at, left, v);
    else row_load<T, N>((const T*)w + at, left, v);
}

// ---- sums and maxima over the tpr threads of a row; `lds` has two slots per wave, `turn` alternates between them so that one barrier
// per reduction is enough
__device__ __forceinline__ double row_sum(double v, int tpr, double (*lds)[16], int turn) {
    for (int o = min(tpr, 64) >> 1; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if (tpr > 64) {
        const int wave = threadIdx.x >> 6, first = (threadIdx.x / tpr) * (tpr >> 6), n = tpr >> 6;
        if ((threadIdx.x & 63) == 0) lds[turn][wave] = v;
        __syncthreads();
        v = 0.0;
        for (int i = 0; i < n; i++) v += lds[turn][first + i];
    }
    return v;
}
__device__ __forceinline__ unsigned row_max(unsigned v, int tpr, double (*lds)[16], int turn) {
    for (int o = min(tpr, 64) >> 1; o >= 1; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o));
    if (tpr > 64) {
        const int wave = threadIdx.x >> 6, first = (threadIdx.x / tpr) * (tpr >> 6), n = tpr >> 6;
        if ((threadIdx.x & 63) == 0) lds[turn][wave] = (double)v;          // (exact: 32 bits)
        __syncthreads();
        v = 0;
        for (int i = 0; i < n; i++) v = max(v, (unsigned)lds[turn][first + i]);
    }
    return v;
}
// 1 / sqrt(ss / F + eps); mean squares beyond the range of 32 bits go through 64
__device__ __forceinline__ float rms_inverse(double ss, double inv_F, float eps) {
    const double m = ss * inv_F + (double)eps;
    if (m < 1e37) return 1.0f / __builtin_sqrtf((float)m);
    return (float)(1.0 / __builtin_sqrt(m));
}

// ---- 8-bit codes -----------------------------------------------------------------------------------------------------------------
enum { CODE_INT8 = 1, CODE_E4M3 = 2 };
template <int CODE> struct Code8;
template <> struct Code8<CODE_INT8> {
    static constexpr float Q = 127.0f;
    static __device__ __forceinline__ unsigned pack4(const float* p) {
        unsigned r = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) r |= ((unsigned)(int)__builtin_rintf(p[i]) & 0xffu) << (8 * i);
        return r;
    }
    static __device__ __forceinline__ float one(unsigned c) { return (float)(signed char)c; }
    static __device__ __forceinline__ void unpack4(unsigned c, float* v) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (float)(signed char)(c >> (8 * i));
    }
};
template <> struct Code8<CODE_E4M3> {
    static constexpr float Q = 448.0f;
    static __device__ __forceinline__ unsigned pack4(const float* p) {
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(p[0], p[1], 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(p[2], p[3], r, true);
    }
    static __device__ __forceinline__ float one(unsigned c) { return __builtin_amdgcn_cvt_f32_fp8((int)c, 0); }
    static __device__ __forceinline__ void unpack4(unsigned c, float* v) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
        v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
    }
};

// The codes of four values of a group: t Q / top rounded to the nearest code, ties to even, as if the quotient were exact.  The 32-bit
// product t (Q / top) is off by at most 2^-23 of itself; where a border between two codes lies that near (the codes of the
// product scaled by 1 -+ 2^-21 differ: one value in 1e5) both sides of the comparison |t| Q <> border top are formed exactly in 64 bits.
template <int CODE> __device__ __forceinline__ unsigned encode4(const float* t, float inv, float top) {
    using C = Code8<CODE>;
    float p[4], lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; i++) { p[i] = inv > 0.0f ? t[i] * inv : 0.0f; lo[i] = p[i] * (1.0f - 0x1p-21f); hi[i] = p[i] * (1.0f + 0x1p-21f); }
    unsigned in = C::pack4(lo);
    const unsigned out = C::pack4(hi);
    if (in != out) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned a = (in >> (8 * i)) & 0xffu, b = (out >> (8 * i)) & 0xffu;
            if (a == b) continue;
            const double border = 0.5 * (fabs((double)C::one(a)) + fabs((double)C::one(b))) * (double)top;
            const double value = fabs((double)t[i]) * (double)C::Q;
            if (value > border || (value == border && (a & 1u))) in = (in & ~(0xffu << (8 * i))) | (b << (8 * i));
        }
    }
    return in;
}
// Q / top and top / Q of a group from the bits of its largest magnitude
template <int CODE> __device__ __forceinline__ void group_scale(unsigned top_bits, float& top, float& inv, float& scale) {
    top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) { inv = 0.0f; scale = __uint_as_float(0x7fc00000u); }        // an infinity or NaN: the group reads back as NaN
    else if (top < ROWS_TINY) { inv = 0.0f; scale = 0.0f; }
    else { inv = Code8<CODE>::Q / top; scale = top / Code8<CODE>::Q; }
}
template <int N> __device__ __forceinline__ void code_store(unsigned char* p, int left, const unsigned (&c)[N / 4]) {
    if (left >= N) __builtin_memcpy(p, c, N);
    else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left) p[i] = (unsigned char)(c[i / 4] >> (8 * (i & 3)));
    }
}

// ---- where a written row goes ----------------------------------------------------------------------------------------------------
// index == NULL: row first + i.  Otherwise row index[i]; of equal indices the last one is kept, indices outside [0, P) write nothing.
// owner == NULL: the row looks through the entries behind it (few rows).  owner [P], all -1 between calls: row_claim_kernel has left
// the largest i per row there; the winner puts the -1 back (a loser reads either another i or -1).
struct RowTarget {
    long long P, first;
    const void* index;
    int is64;
    int* owner;
};
__device__ __forceinline__ long long target_index(const RowTarget& d, long long i) {
    return d.is64 ? ((const long long*)d.index)[i] : (long long)((const int*)d.index)[i];
}
__global__ __launch_bounds__(256) void row_claim_kernel(long long n, RowTarget d) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long r = target_index(d, i);
    if (r >= 0 && r < d.P) atomicMax(d.owner + r, (int)i);
}
// the row that row i goes to, -1: none; the tpr threads of a row call it together
__device__ __forceinline__ long long row_target(const RowTarget& d, long long i, long long n, int t, int tpr, double (*lds)[16]) {
    if (d.index == nullptr) return i < n ? d.first + i : -1;
    long long r = i < n ? target_index(d, i) : -1;
    if (r < 0 || r >= d.P) r = -1;
    unsigned lost = 0;
    if (d.owner != nullptr) {
        if (r >= 0) lost = d.owner[r] != (int)i;
        if (tpr > 64) __syncthreads();              // everybody has read before the winner's store
        if (r >= 0 && !lost && t == 0) d.owner[r] = -1;
    } else {
        if (r >= 0)
            for (long long j = i + 1 + t; j < n; j += tpr) lost |= target_index(d, j) == r;
        lost = row_max(lost, tpr, lds, 1);
        if (tpr > 64) __syncthreads();              // (the slot is used again by the caller)
    }
    return lost ? -1 : r;
}

// ---- forward ---------------------------------------------------------------------------------------------------------------------
// OUT = 0: y in T, else codes and scales.  norm = 0: no statistics (rstd = 1), the plain writing of a table.
struct RmsArgs {
    long long rows, row0;   // this launch starts at row row0
    int F, tpr, norm, w32;
    int groups, gshift;     // groups per row and log2 of their columns; one group: 1 and 31
    float eps;
    double inv_F;
    const void* x;
    long long ldx;
    const void* res;        // or NULL
    long long ldr;
    const void* w;          // or NULL
    void* y;                // OUT = 0: [rows, F]
    void* s;                // or NULL: [rows, F]
    float* rstd;            // or NULL: [rows]
    unsigned char* codes;   // [P, F]
    float* scales;          // [P, groups]
    RowTarget to;
};
template <class T, int NV, int OUT> __global__ __launch_bounds__(512) void rms_forward_kernel(RmsArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x & (tpr - 1);
    const long long i = a.row0 + (long long)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
    const bool on = i < a.rows;
    const T* x = (const T*)a.x + (on ? i : 0) * a.ldx;
    const T* res = a.res ? (const T*)a.res + (on ? i : 0) * a.ldr : nullptr;
    float v[NV][N];
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * N, left = on ? a.F - at : 0;
        if (left <= 0) {
#pragma unroll
            for (int e = 0; e < N; e++) v[k][e] = 0.0f;
            continue;
        }
        row_load<T, N>(x + at, left, v[k]);
        if (res) {
            float r[N];
            row_load<T, N>(res + at, left, r);
#pragma unroll
            for (int e = 0; e < N; e++) v[k][e] += r[e];
        }
    }
    if (a.norm) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < N; e++) ss += (double)v[k][e] * (double)v[k][e];
        ss = row_sum(ss, tpr, lds, 0);
    }
    const float rstd = a.norm ? rms_inverse(ss, a.inv_F, a.eps) : 1.0f;
    if (a.rstd && on && t == 0) a.rstd[i] = rstd;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * N, left = on ? a.F - at : 0;
        if (left <= 0) continue;
        if (a.s) row_store<T, N>((T*)a.s + i * a.F + at, left, v[k]);
        float w[N];
        gain_load<T, N>(a.w, a.w32, at, left, w);
#pragma unroll
        for (int e = 0; e < N; e++) v[k][e] = OUT == 0 ? v[k][e] * rstd * w[e] : v[k][e] * w[e];
        if (OUT == 0) row_store<T, N>((T*)a.y + i * a.F + at, left, v[k]);
    }
    if constexpr (OUT != 0) {
        const long long row = row_target(a.to, i, a.rows, t, tpr, lds);
        const int seg = a.groups == 1 ? 0 : (1 << a.gshift) / N;
        unsigned top_bits = 0;
        if (seg == 0) {
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int e = 0; e < N; e++) top_bits = max(top_bits, __float_as_uint(v[k][e]) & 0x7fffffffu);
            top_bits = row_max(top_bits, tpr, lds, 1);
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int at = (t + k * tpr) * N, left = a.F - at;
            if (seg != 0) {             // a group's vectors lie in `seg` neighbouring lanes of one wave
                top_bits = 0;
#pragma unroll
                for (int e = 0; e < N; e++) top_bits = max(top_bits, __float_as_uint(v[k][e]) & 0x7fffffffu);
                for (int o = seg >> 1; o >= 1; o >>= 1) top_bits = max(top_bits, (unsigned)__shfl_xor((int)top_bits, o));
            }
            float top, inv, scale;
            group_scale<OUT>(top_bits, top, inv, scale);
            if (row < 0 || left <= 0) continue;
            unsigned c[N / 4];
#pragma unroll
            for (int q = 0; q < N / 4; q++) c[q] = encode4<OUT>(&v[k][4 * q], inv, top);
            code_store<N>(a.codes + row * a.F + at, left, c);
            if ((at & ((1u << a.gshift) - 1u)) == 0) a.scales[row * a.groups + (at >> a.gshift)] = scale * rstd;
        }
    }
}

// The same for rows that the registers do not hold: one workgroup per row, read twice.
template <class T, int OUT> __global__ __launch_bounds__(512) void rms_forward_long_kernel(RmsArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x;
    const long long i = a.row0 + blockIdx.x;
    const T* x = (const T*)a.x + i * a.ldx;
    const T* res = a.res ? (const T*)a.res + i * a.ldr : nullptr;
    const long long row = OUT != 0 ? row_target(a.to, i, a.rows, t, tpr, lds) : i;
    double ss = 0.0;
    unsigned row_top = 0;
    const bool by_row = OUT != 0 && a.groups == 1;
    for (int at = t * N; at < a.F; at += tpr * N) {
        float v[N], r[N], w[N];
        row_load<T, N>(x + at, a.F - at, v);
        if (res) {
            row_load<T, N>(res + at, a.F - at, r);
#pragma unroll
            for (int e = 0; e < N; e++) v[e] += r[e];
        }
#pragma unroll
        for (int e = 0; e < N; e++) ss += (double)v[e] * (double)v[e];
        if (by_row) {
            gain_load<T, N>(a.w, a.w32, at, a.F - at, w);
#pragma unroll
            for (int e = 0; e < N; e++) row_top = max(row_top, __float_as_uint(v[e] * w[e]) & 0x7fffffffu);
        }
    }
    float rstd = 1.0f;
    if (a.norm) rstd = rms_inverse(row_sum(ss, tpr, lds, 0), a.inv_F, a.eps);
    if (by_row) row_top = row_max(row_top, tpr, lds, 1);
    if (a.rstd && t == 0) a.rstd[i] = rstd;
    const int seg = OUT == 0 || by_row ? 0 : (1 << a.gshift) / N;
    // (all threads of a wave take every step together: the groups' maxima are shuffled)
    for (int base = 0; base < a.F; base += tpr * N) {
        const int at = base + t * N, left = a.F - at;
        float v[N], r[N], w[N];
        row_load<T, N>(x + (left > 0 ? at : 0), left > 0 ? left : 0, v);
        if (res) {
            row_load<T, N>(res + (left > 0 ? at : 0), left > 0 ? left : 0, r);
#pragma unroll
            for (int e = 0; e < N; e++) v[e] += r[e];
        }
        if (a.s && left > 0) row_store<T, N>((T*)a.s + i * a.F + at, left, v);
        if (left > 0) gain_load<T, N>(a.w, a.w32, at, left, w);
        else {
#pragma unroll
            for (int e = 0; e < N; e++) w[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = OUT == 0 ? v[e] * rstd * w[e] : v[e] * w[e];
        if constexpr (OUT == 0) {
            if (left > 0) row_store<T, N>((T*)a.y + i * a.F + at, left, v);
        } else {
            unsigned top_bits = row_top;
            if (seg != 0) {
                top_bits = 0;
#pragma unroll
                for (int e = 0; e < N; e++) top_bits = max(top_bits, __float_as_uint(v[e]) & 0x7fffffffu);
                for (int o = seg >> 1; o >= 1; o >>= 1) top_bits = max(top_bits, (unsigned)__shfl_xor((int)top_bits, o));
            }
            float top, inv, scale;
            group_scale<OUT>(top_bits, top, inv, scale);
            if (row >= 0 && left > 0) {
                unsigned c[N / 4];
#pragma unroll
                for (int q = 0; q < N / 4; q++) c[q] = encode4<OUT>(&v[4 * q], inv, top);
                code_store<N>(a.codes + row * a.F + at, left, c);
                if ((at & ((1u << a.gshift) - 1u)) == 0) a.scales[row * a.groups + (at >> a.gshift)] = scale * rstd;
            }
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------
struct RmsBackArgs {
    long long rows, row0;   // row0: of the *_long kernel
    int F, tpr, w32;
    const void* s;
    long long lds_;
    const void* w;          // or NULL
    const float* rstd;
    const void* gy;
    long long ldg;
    const void* gs;         // or NULL
    long long ldgs;
    void* ds;               // or NULL: [rows, F]
    float* dw_part;         // or NULL: [gridDim.x, F]
};
template <class T, int NV> __global__ __launch_bounds__(512) void rms_backward_kernel(RmsBackArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    __shared__ float part[8][64 * N];       // the waves' sums of one vector slot
    const int tpr = a.tpr, t = threadIdx.x & (tpr - 1), rpb = blockDim.x / tpr;
    float dw[NV][N], w[NV][N];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * N, left = a.F - at;
#pragma unroll
        for (int e = 0; e < N; e++) { dw[k][e] = 0.0f; w[k][e] = 0.0f; }
        if (left > 0) gain_load<T, N>(a.w, a.w32, at, left, w[k]);
    }
    int turn = 0;
    for (long long r0 = (long long)blockIdx.x * rpb; r0 < a.rows; r0 += (long long)gridDim.x * rpb, turn ^= 1) {
        const long long i = r0 + threadIdx.x / tpr;
        const bool on = i < a.rows;
        const float rstd = on ? a.rstd[i] : 0.0f;
        const T* s = (const T*)a.s + (on ? i : 0) * a.lds_;
        const T* gy = (const T*)a.gy + (on ? i : 0) * a.ldg;
        float h[NV][N], g[NV][N];
        float c = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int at = (t + k * tpr) * N, left = on ? a.F - at : 0;
#pragma unroll
            for (int e = 0; e < N; e++) { h[k][e] = 0.0f; g[k][e] = 0.0f; }
            if (left <= 0) continue;
            row_load<T, N>(s + at, left, h[k]);
            row_load<T, N>(gy + at, left, g[k]);
        }
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                h[k][e] *= rstd;
                dw[k][e] += g[k][e] * h[k][e];
                g[k][e] *= w[k][e];
                c += g[k][e] * h[k][e];
            }
        const float mean = (float)row_sum((double)c, tpr, lds, turn) / (float)a.F;
        if (a.ds == nullptr) continue;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int at = (t + k * tpr) * N, left = on ? a.F - at : 0;
            if (left <= 0) continue;
            float d[N];
#pragma unroll
            for (int e = 0; e < N; e++) d[e] = rstd * (g[k][e] - h[k][e] * mean);
            if (a.gs) {
                float q[N];
                row_load<T, N>((const T*)a.gs + i * a.ldgs + at, left, q);
#pragma unroll
                for (int e = 0; e < N; e++) d[e] += q[e];
            }
            row_store<T, N>((T*)a.ds + i * a.F + at, left, d);
        }
    }
    if (a.dw_part == nullptr) return;
    // the rows of a wave first, then the waves, in a fixed order
    const int lanes = min(tpr, 64);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        for (int o = 32; o >= lanes; o >>= 1)
#pragma unroll
            for (int e = 0; e < N; e++) dw[k][e] += __shfl_xor(dw[k][e], o);
        const int at = (t + k * tpr) * N;
        if (rpb == 1) {
            if (at < a.F) row_store<float, N>(a.dw_part + (long long)blockIdx.x * a.F + at, a.F - at, dw[k]);
            continue;
        }
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, per_row = max(1, tpr >> 6), n = (int)(blockDim.x >> 6) / per_row;
        __syncthreads();
        if (lane < lanes)
#pragma unroll
            for (int e = 0; e < N; e++) part[wave][lane * N + e] = dw[k][e];
        __syncthreads();
        if (threadIdx.x < tpr && at < a.F) {
            float sum[N];
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] = 0.0f;
            for (int q = 0; q < n; q++)
#pragma unroll
                for (int e = 0; e < N; e++) sum[e] += part[q * per_row + wave][lane * N + e];
            row_store<float, N>(a.dw_part + (long long)blockIdx.x * a.F + at, a.F - at, sum);
        }
    }
}
// rows beyond the registers: ds by one workgroup per row (read twice), dw by columns
template <class T> __global__ __launch_bounds__(512) void rms_backward_long_kernel(RmsBackArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x;
    const long long i = a.row0 + blockIdx.x;
    const T* s = (const T*)a.s + i * a.lds_;
    const T* gy = (const T*)a.gy + i * a.ldg;
    const float rstd = a.rstd[i];
    double c = 0.0;
    for (int at = t * N; at < a.F; at += tpr * N) {
        float h[N], g[N], w[N];
        row_load<T, N>(s + at, a.F - at, h);
        row_load<T, N>(gy + at, a.F - at, g);
        gain_load<T, N>(a.w, a.w32, at, a.F - at, w);
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++)
            if (at + e < a.F) p += g[e] * w[e] * (h[e] * rstd);
        c += (double)p;
    }
    const float mean = (float)row_sum(c, tpr, lds, 0) / (float)a.F;
    for (int at = t * N; at < a.F; at += tpr * N) {
        float h[N], g[N], w[N], d[N];
        row_load<T, N>(s + at, a.F - at, h);
        row_load<T, N>(gy + at, a.F - at, g);
        gain_load<T, N>(a.w, a.w32, at, a.F - at, w);
#pragma unroll
        for (int e = 0; e < N; e++) d[e] = rstd * (g[e] * w[e] - h[e] * rstd * mean);
        if (a.gs) {
            float q[N];
            row_load<T, N>((const T*)a.gs + i * a.ldgs + at, a.F - at, q);
#pragma unroll
            for (int e = 0; e < N; e++) d[e] += q[e];
        }
        row_store<T, N>((T*)a.ds + i * a.F + at, a.F - at, d);
    }
}
template <class T> __global__ __launch_bounds__(256) void rms_dw_columns_kernel(RmsBackArgs a, int slices) {
    const long long col = (long long)blockIdx.x * 256 + threadIdx.x;
    if (col >= a.F) return;
    float sum = 0.0f;
    for (long long i = blockIdx.y; i < a.rows; i += slices)
        sum += (float)((const T*)a.gy)[i * a.ldg + col] * ((float)((const T*)a.s)[i * a.lds_ + col] * a.rstd[i]);
    a.dw_part[(long long)blockIdx.y * a.F + col] = sum;
}
// dw = the sum of n partial rows, in a fixed order: 32 columns and 8 slices of the partials per workgroup
template <class T> __global__ __launch_bounds__(256) void rms_dw_sum_kernel(int F, int n, const float* __restrict__ part, T* __restrict__ dw) {
    __shared__ float lds[8][33];
    const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * 32 + c;
    float sum = 0.0f;
    if (col < F)
        for (int i = q; i < n; i += 8) sum += part[(long long)i * F + col];
    lds[q][c] = sum;
    __syncthreads();
    if (q == 0 && col < F) {
        for (int i = 1; i < 8; i++) sum += lds[i][c];
        dw[col] = (T)sum;
    }
}

// ---- reading 8-bit rows back -------------------------------------------------------------------------------------------------------
// out[i] = the values of row (first + i | index[i]); norm: divided by (|row|_2 + eps).  Rows outside [0, P) are zeros.
struct ReadArgs {
    long long rows, row0, P, first;
    int F, tpr, groups, gshift, norm, is64;
    float eps;
    const unsigned char* codes;
    const float* scales;
    const void* index;      // or NULL
    void* out;              // [rows, F]
};
template <int CODE> __device__ __forceinline__ void code_load(const unsigned char* p, int left, float (&v)[8]) {
    if (left >= 8) {
        unsigned c[2];
        __builtin_memcpy(c, p, 8);
        Code8<CODE>::unpack4(c[0], v);
        Code8<CODE>::unpack4(c[1], v + 4);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < left ? Code8<CODE>::one(p[e]) : 0.0f;
    }
}
__device__ __forceinline__ float l2_inverse(double ss, float eps) {
    const float n = ss < 1e37 ? __builtin_sqrtf((float)ss) : (float)__builtin_sqrt(ss);
    return 1.0f / (n + eps);
}
template <class T, int CODE, int NV> __global__ __launch_bounds__(512) void rows_read_kernel(ReadArgs a) {
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x & (tpr - 1);
    const long long i = a.row0 + (long long)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
    long long row = -1;
    if (i < a.rows) row = a.index == nullptr ? a.first + i : a.is64 ? ((const long long*)a.index)[i] : (long long)((const int*)a.index)[i];
    if (row >= a.P) row = -1;
    float v[NV][8];
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * 8, left = row >= 0 ? a.F - at : 0;
#pragma unroll
        for (int e = 0; e < 8; e++) v[k][e] = 0.0f;
        if (left <= 0) continue;
        code_load<CODE>(a.codes + row * a.F + at, left, v[k]);
        const float scale = a.scales[row * a.groups + (at >> a.gshift)];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[k][e] = e < left ? v[k][e] * scale : 0.0f;
            ss += (double)v[k][e] * (double)v[k][e];
        }
    }
    float inv = 1.0f;
    if (a.norm) inv = l2_inverse(row_sum(ss, tpr, lds, 0), a.eps);
    if (row < 0) inv = 0.0f;
    if (i >= a.rows) return;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * 8, left = a.F - at;
        if (left <= 0) continue;
#pragma unroll
        for (int e = 0; e < 8; e++) v[k][e] *= inv;
        row_store<T, 8>((T*)a.out + i * a.F + at, left, v[k]);
    }
}
template <class T, int CODE> __global__ __launch_bounds__(512) void rows_read_long_kernel(ReadArgs a) {
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x;
    const long long i = a.row0 + blockIdx.x;
    long long row = a.index == nullptr ? a.first + i : a.is64 ? ((const long long*)a.index)[i] : (long long)((const int*)a.index)[i];
    if (row >= a.P) row = -1;
    float inv = 1.0f;
    if (a.norm) {
        double ss = 0.0;
        if (row >= 0)
            for (int at = t * 8; at < a.F; at += tpr * 8) {
                float v[8];
                code_load<CODE>(a.codes + row * a.F + at, a.F - at, v);
                const float scale = a.scales[row * a.groups + (at >> a.gshift)];
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (at + e < a.F) ss += (double)(v[e] * scale) * (double)(v[e] * scale);
            }
        inv = l2_inverse(row_sum(ss, tpr, lds, 0), a.eps);
    }
    for (int at = t * 8; at < a.F; at += tpr * 8) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.0f;
        if (row >= 0) {
            code_load<CODE>(a.codes + row * a.F + at, a.F - at, v);
            const float scale = a.scales[row * a.groups + (at >> a.gshift)];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = v[e] * scale * inv;
        }
        row_store<T, 8>((T*)a.out + i * a.F + at, a.F - at, v);
    }
}

}  // namespace iso
