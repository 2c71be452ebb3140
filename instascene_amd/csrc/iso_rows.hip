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
// v = x + res (res may be NULL)
template <class T, int N> __device__ __forceinline__ void sum_load(const T* x, const T* res, int left, float (&v)[N]) {
    row_load<T, N>(x, left, v);
    if (res) {
        float r[N];
        row_load<T, N>(res, left, r);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += r[i];
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

// ---- sums and maxima over the tpr threads of a row.  Within 16 lanes by DPP (quad_perm, then the mirrors of 8 and 16 lanes: every lane of
// a half already holds its half's value), across 16 and 32 lanes by the permlane swaps: no trip through LDS.  All lanes of the wave have to
// be active.  Between waves `lds` has two slots per wave; `turn` alternates between them so that one barrier per reduction is enough.
template <int CTRL> __device__ __forceinline__ unsigned lane_dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
// the value of the partner at distance 1, 2, 4, 8 (STEP 0..3; 4 and 8 mirrored), 16, 32
template <int STEP> __device__ __forceinline__ unsigned lane_partner(unsigned v) {
    if constexpr (STEP == 0) return lane_dpp<0xB1>(v);
    else if constexpr (STEP == 1) return lane_dpp<0x4E>(v);
    else if constexpr (STEP == 2) return lane_dpp<0x141>(v);
    else if constexpr (STEP == 3) return lane_dpp<0x140>(v);
    else {
        const bool up = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)) & (STEP == 4 ? 16u : 32u);
        const auto q = STEP == 4 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return up ? q[0] : q[1];
    }
}
template <int STEP> __device__ __forceinline__ double lane_partner(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = lane_partner<STEP>((unsigned)b), hi = lane_partner<STEP>((unsigned)(b >> 32));
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
// over the lanes of aligned segments of n (a power of two) lanes of a wave
__device__ __forceinline__ double lanes_sum(double v, int n) {
    if (n > 1) v += lane_partner<0>(v);
    if (n > 2) v += lane_partner<1>(v);
    if (n > 4) v += lane_partner<2>(v);
    if (n > 8) v += lane_partner<3>(v);
    if (n > 16) v += lane_partner<4>(v);
    if (n > 32) v += lane_partner<5>(v);
    return v;
}
__device__ __forceinline__ unsigned lanes_max(unsigned v, int n) {
    if (n > 1) v = max(v, lane_partner<0>(v));
    if (n > 2) v = max(v, lane_partner<1>(v));
    if (n > 4) v = max(v, lane_partner<2>(v));
    if (n > 8) v = max(v, lane_partner<3>(v));
    if (n > 16) v = max(v, lane_partner<4>(v));
    if (n > 32) v = max(v, lane_partner<5>(v));
    return v;
}
__device__ __forceinline__ double row_sum(double v, int tpr, double (*lds)[16], int turn) {
    v = lanes_sum(v, tpr);
    if (tpr > 64) {
        const int wave = threadIdx.x >> 6, n = tpr >> 6, first = wave & ~(n - 1);
        if ((threadIdx.x & 63) == 0) lds[turn][wave] = v;
        __syncthreads();
        v = 0.0;
        for (int i = 0; i < n; i++) v += lds[turn][first + i];
    }
    return v;
}
__device__ __forceinline__ unsigned row_max(unsigned v, int tpr, double (*lds)[16], int turn) {
    v = lanes_max(v, tpr);
    if (tpr > 64) {
        const int wave = threadIdx.x >> 6, n = tpr >> 6, first = wave & ~(n - 1);
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
        // + 1.5 2^23 rounds to a whole number, ties to even, whose low byte is the code
        const unsigned a = __float_as_uint(p[0] + 12582912.0f), b = __float_as_uint(p[1] + 12582912.0f);
        const unsigned c = __float_as_uint(p[2] + 12582912.0f), d = __float_as_uint(p[3] + 12582912.0f);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
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

// What encodes a group: its largest magnitude, Q / top a little below and above, the scale top / Q.
struct Group8 { float top, lo, hi, scale; };
// From the bits of the largest magnitude.  Q / top by v_rcp_f32 (within 2^-21.6 with the roundings around it; encode4 allows 2^-21), top / Q correctly rounded: the
// product with 1 / Q, corrected once by its exact remainder.
template <int CODE> __device__ __forceinline__ Group8 group_scale(unsigned top_bits) {
    constexpr float Q = Code8<CODE>::Q, rq = 1.0f / Q;
    Group8 g;
    g.top = __uint_as_float(top_bits);
    const float s = g.top * rq, inv = __builtin_amdgcn_rcpf(s);         // (of top / Q: of top itself it would be below the normal numbers)
    g.lo = inv * (1.0f - 0x1p-21f);
    g.hi = inv * (1.0f + 0x1p-21f);
    g.scale = __builtin_fmaf(__builtin_fmaf(-s, Q, g.top), rq, s);
    if (g.top < ROWS_TINY || top_bits >= 0x7f800000u) {
        g.lo = g.hi = 0.0f;
        g.scale = top_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : 0.0f;      // an infinity or NaN: the group reads back as NaN
    }
    return g;
}
// The codes of four values of a group: t Q / top rounded to the nearest code, ties to even, as if the quotient were exact.  The 32-bit
// products t lo and t hi bracket it; where they round to different codes (one value in 1e5) a border lies between them, and both sides of
// |t| Q <> border top are formed exactly in 64 bits.
template <int CODE> __device__ __forceinline__ unsigned encode4(const float* t, const Group8& g) {
    using C = Code8<CODE>;
    float lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; i++) { lo[i] = t[i] * g.lo; hi[i] = t[i] * g.hi; }
    unsigned in = C::pack4(lo);
    const unsigned out = C::pack4(hi);
    if (g.hi == 0.0f) return 0;                 // (an infinity or NaN times 0)
    if (in != out) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned a = (in >> (8 * i)) & 0xffu, b = (out >> (8 * i)) & 0xffu;
            if (a == b) continue;
            const double border = 0.5 * (fabs((double)C::one(a)) + fabs((double)C::one(b))) * (double)g.top;
            const double value = fabs((double)t[i]) * (double)C::Q;
            if (value > border || (value == border && (a & 1u))) in = (in & ~(0xffu << (8 * i))) | (b << (8 * i));
        }
    }
    return in;
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
    int F, tpr, tsh, norm, w32;     // tpr = 1 << tsh threads per row
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
    const long long i = a.row0 + (long long)blockIdx.x * (blockDim.x >> a.tsh) + (threadIdx.x >> a.tsh);
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
        sum_load<T, N>(x + at, res ? res + at : nullptr, left, v[k]);
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
                top_bits = lanes_max(top_bits, seg);
            }
            const Group8 g = group_scale<OUT>(top_bits);
            if (row < 0 || left <= 0) continue;
            unsigned c[N / 4];
#pragma unroll
            for (int q = 0; q < N / 4; q++) c[q] = encode4<OUT>(&v[k][4 * q], g);
            code_store<N>(a.codes + row * a.F + at, left, c);
            if ((at & ((1u << a.gshift) - 1u)) == 0) a.scales[row * a.groups + (at >> a.gshift)] = g.scale * rstd;
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
        float v[N], w[N];
        sum_load<T, N>(x + at, res ? res + at : nullptr, a.F - at, v);
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
        float v[N], w[N];
        sum_load<T, N>(x + at, res ? res + at : nullptr, left, v);          // (left <= 0: nothing is read)
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
                top_bits = lanes_max(top_bits, seg);
            }
            const Group8 g = group_scale<OUT>(top_bits);
            if (row >= 0 && left > 0) {
                unsigned c[N / 4];
#pragma unroll
                for (int q = 0; q < N / 4; q++) c[q] = encode4<OUT>(&v[4 * q], g);
                code_store<N>(a.codes + row * a.F + at, left, c);
                if ((at & ((1u << a.gshift) - 1u)) == 0) a.scales[row * a.groups + (at >> a.gshift)] = g.scale * rstd;
            }
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------
struct RmsBackArgs {
    long long rows, row0;   // row0: of the *_long kernel
    int F, tpr, tsh, w32;
    const void* x;          // s = x + res
    long long ldx;
    const void* res;        // or NULL
    long long ldr;
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
    const int tpr = a.tpr, t = threadIdx.x & (tpr - 1), rpb = blockDim.x >> a.tsh;
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
        const long long i = r0 + (threadIdx.x >> a.tsh);
        const bool on = i < a.rows;
        const float rstd = on ? a.rstd[i] : 0.0f;
        const T* x = (const T*)a.x + (on ? i : 0) * a.ldx;
        const T* res = a.res ? (const T*)a.res + (on ? i : 0) * a.ldr : nullptr;
        const T* gy = (const T*)a.gy + (on ? i : 0) * a.ldg;
        float h[NV][N], g[NV][N];
        float c = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int at = (t + k * tpr) * N, left = on ? a.F - at : 0;
#pragma unroll
            for (int e = 0; e < N; e++) { h[k][e] = 0.0f; g[k][e] = 0.0f; }
            if (left <= 0) continue;
            sum_load<T, N>(x + at, res ? res + at : nullptr, left, h[k]);
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
    const T* x = (const T*)a.x + i * a.ldx;
    const T* res = a.res ? (const T*)a.res + i * a.ldr : nullptr;
    const T* gy = (const T*)a.gy + i * a.ldg;
    const float rstd = a.rstd[i];
    double c = 0.0;
    for (int at = t * N; at < a.F; at += tpr * N) {
        float h[N], g[N], w[N];
        sum_load<T, N>(x + at, res ? res + at : nullptr, a.F - at, h);
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
        sum_load<T, N>(x + at, res ? res + at : nullptr, a.F - at, h);
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
    for (long long i = blockIdx.y; i < a.rows; i += slices) {
        float v = (float)((const T*)a.x)[i * a.ldx + col];
        if (a.res) v += (float)((const T*)a.res)[i * a.ldr + col];
        sum += (float)((const T*)a.gy)[i * a.ldg + col] * (v * a.rstd[i]);
    }
    a.dw_part[(long long)blockIdx.y * a.F + col] = sum;
}
// dw = the sum of n partial rows, in a fixed order: 32 columns and 32 slices of the partials per workgroup, eight loads in flight each (a
// narrow table has one workgroup here and up to 2048 partials: what counts is the number of loads that wait for each other)
template <class T> __global__ __launch_bounds__(1024) void rms_dw_sum_kernel(int F, int n, const float* __restrict__ part, T* __restrict__ dw) {
    __shared__ float lds[32][33];
    const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * 32 + c;
    float sum = 0.0f;
    if (col < F)
        for (int i = q; i < n; i += 256) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = i + 32 * u < n ? part[(long long)(i + 32 * u) * F + col] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; u++) sum += v[u];
        }
    lds[q][c] = sum;
    __syncthreads();
    if (q == 0 && col < F) {
        for (int i = 1; i < 32; i++) sum += lds[i][c];
        dw[col] = (T)sum;
    }
}

// ---- reading 8-bit rows back -------------------------------------------------------------------------------------------------------
// out[i] = the values of row (first + i | index[i]); norm: divided by (|row|_2 + eps).  Rows outside [0, P) are zeros.
struct ReadArgs {
    long long rows, row0, P, first;
    int F, tpr, tsh, groups, gshift, norm, is64;
    float eps;
    const unsigned char* codes;
    const float* scales;
    const void* index;      // or NULL
    void* out;              // [rows, F]
};
template <int CODE, int N> __device__ __forceinline__ void code_load(const unsigned char* p, int left, float (&v)[N]) {
    if (left >= N) {
        unsigned c[N / 4];
        __builtin_memcpy(c, p, N);
#pragma unroll
        for (int q = 0; q < N / 4; q++) Code8<CODE>::unpack4(c[q], v + 4 * q);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = e < left ? Code8<CODE>::one(p[e]) : 0.0f;
    }
}
__device__ __forceinline__ float l2_inverse(double ss, float eps) {
    const float n = ss < 1e37 ? __builtin_sqrtf((float)ss) : (float)__builtin_sqrt(ss);
    return 1.0f / (n + eps);
}
template <class T, int CODE, int NV> __global__ __launch_bounds__(512) void rows_read_kernel(ReadArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x & (tpr - 1);
    const long long i = a.row0 + (long long)blockIdx.x * (blockDim.x >> a.tsh) + (threadIdx.x >> a.tsh);
    long long row = -1;
    if (i < a.rows) row = a.index == nullptr ? a.first + i : a.is64 ? ((const long long*)a.index)[i] : (long long)((const int*)a.index)[i];
    if (row >= a.P) row = -1;
    float v[NV][N];
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * N, left = row >= 0 ? a.F - at : 0;
#pragma unroll
        for (int e = 0; e < N; e++) v[k][e] = 0.0f;
        if (left <= 0) continue;
        code_load<CODE, N>(a.codes + row * a.F + at, left, v[k]);
        const float scale = a.scales[row * a.groups + (at >> a.gshift)];
#pragma unroll
        for (int e = 0; e < N; e++) {
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
        const int at = (t + k * tpr) * N, left = a.F - at;
        if (left <= 0) continue;
#pragma unroll
        for (int e = 0; e < N; e++) v[k][e] *= inv;
        row_store<T, N>((T*)a.out + i * a.F + at, left, v[k]);
    }
}
template <class T, int CODE> __global__ __launch_bounds__(512) void rows_read_long_kernel(ReadArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x;
    const long long i = a.row0 + blockIdx.x;
    long long row = a.index == nullptr ? a.first + i : a.is64 ? ((const long long*)a.index)[i] : (long long)((const int*)a.index)[i];
    if (row >= a.P) row = -1;
    float inv = 1.0f;
    if (a.norm) {
        double ss = 0.0;
        if (row >= 0)
            for (int at = t * N; at < a.F; at += tpr * N) {
                float v[N];
                code_load<CODE, N>(a.codes + row * a.F + at, a.F - at, v);
                const float scale = a.scales[row * a.groups + (at >> a.gshift)];
#pragma unroll
                for (int e = 0; e < N; e++)
                    if (at + e < a.F) ss += (double)(v[e] * scale) * (double)(v[e] * scale);
            }
        inv = l2_inverse(row_sum(ss, tpr, lds, 0), a.eps);
    }
    for (int at = t * N; at < a.F; at += tpr * N) {
        float v[N];
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = 0.0f;
        if (row >= 0) {
            code_load<CODE, N>(a.codes + row * a.F + at, a.F - at, v);
            const float scale = a.scales[row * a.groups + (at >> a.gshift)];
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = v[e] * scale * inv;
        }
        row_store<T, N>((T*)a.out + i * a.F + at, a.F - at, v);
    }
}

}  // namespace iso
