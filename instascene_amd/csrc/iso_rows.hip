// Rows of a table: root-mean-square norm (with the residual's addition, its backward pass, an output in 8 bits with scales) and
// the 8-bit row table (written from rows, read back).  Declared in include/instascene_ops.h.
//
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
//   8 bits, per group of G columns:  t = s w,  top = max |t|,  code = round(t Q / top),  scale = top rstd / Q
//       (Q = 448: e4m3, 127: int8; rstd > 0 is common to the row, so it cancels in the codes and only the scale carries it)
//   backward:  h = s rstd,  c = mean(gy w h),  ds = rstd (gy w - h c) + gs,  dw = sum over rows of gy h
//
// All of it is bound by memory: every element is read once, kept in registers between the reduction and the output, and
// written once.  `tpr` threads share a row (a power of two up to a wave, beyond it a workgroup of whole waves), NV vectors of 16 input bytes
// each, vector j = t + k tpr, so that a wave's loads are contiguous; rows longer than the registers hold are read a second time (the *_long kernels).
// Sums of squares are held in 32 bits, in short chains (a vector's elements side by side, then a tree); a row whose sum leaves
// [1e-30, 1e37] is summed again in 64 bits, so that no finite row overflows or vanishes.  (64 bits throughout cost a quarter of the time of
// narrow rows: conversions and 64-bit additions run at a fraction of the rate.)
#pragma once
#include <hip/hip_runtime.h>

namespace iso {

constexpr float ROWS_TINY = 0x1p-116f;      // a group whose largest magnitude lies below is stored as zeros: Q / top and top / Q stay normal

template <class T> struct RowVec { static constexpr int N = 16 / (int)sizeof(T); };
// (alignment of one element: rows of odd widths and views of buckets start anywhere; gfx950 loads unaligned vectors)
template <class T, int N> struct Unaligned { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };

// ---- sixteen bytes of a row as they lie in memory.  EVEN: F is a multiple of the vector, so a vector lies in the row or behind it.  TAIL: the
// row's last vector sticks out; where it does, the row's last N elements are loaded instead and moved down when they are used.  NARROW: the
// row is shorter than a vector: element by element (whose code, next to the others', made every load wait: [32k, 1021] bfloat16 backward
// 152 us, 76 so).
enum { EVEN = 0, TAIL = 1, NARROW = 2 };
typedef unsigned Quad __attribute__((ext_vector_type(4)));
// q without its first n elements of B bytes (0 <= n < 16 / B), zeros behind
template <int B> __device__ __forceinline__ Quad quad_drop(Quad q, int n) {
    const int bytes = n * B;
    if (bytes & 8) q = Quad{q.z, q.w, 0u, 0u};
    if (bytes & 4) q = Quad{q.y, q.z, q.w, 0u};
    if (B == 2 && (bytes & 2))
        q = Quad{__builtin_amdgcn_alignbit(q.y, q.x, 16), __builtin_amdgcn_alignbit(q.z, q.y, 16), __builtin_amdgcn_alignbit(q.w, q.z, 16), q.w >> 16};
    return q;
}
// the vector at `at` from what raw_fetch loaded: the part behind the row gone
template <class T, int N, int FIT> __device__ __forceinline__ typename Unaligned<T, N>::type raw_use(typename Unaligned<T, N>::type q, int at, int F) {
    if constexpr (FIT == TAIL)
        if (at < F && at + N > F)
            q = __builtin_bit_cast(typename Unaligned<T, N>::type, quad_drop<(int)sizeof(T)>(__builtin_bit_cast(Quad, q), at + N - F));
    return q;
}
// A load that may stay in flight: q keeps what it held where there is nothing to load (to drop a value is to wait for it: the backward pass of
// [n, 2944] rows took 150 us instead of 100).  NT: past the caches (a stream that is longer than they are and not read again).
template <class T, int N, int FIT, bool NT> __device__ __forceinline__ void raw_fetch(typename Unaligned<T, N>::type& q, const T* row, int at, int F, bool on) {
    typedef typename Unaligned<T, N>::type V;
    if constexpr (FIT != NARROW) {
        if (on && at < F) {
            const V* p = reinterpret_cast<const V*>(row + (FIT == EVEN ? at : min(at, F - N)));
            if constexpr (NT) q = __builtin_nontemporal_load(p);
            else q = *p;
        }
    } else if (on) {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (at + i < F) q[i] = row[at + i];
    }
}
// the vector at `at`, zeros behind the row and for rows that are off: the address is drawn back into the row and the value dropped, without a branch
template <class T, int N, int FIT, bool NT = false> __device__ __forceinline__ typename Unaligned<T, N>::type raw_load(const T* row, int at, int F, bool on) {
    typedef typename Unaligned<T, N>::type V;
    V q = {};
    if constexpr (FIT != NARROW) {
        const V* p = reinterpret_cast<const V*>(row + min(at, F - N));
        if constexpr (NT) q = __builtin_nontemporal_load(p);
        else q = *p;
        if (!on || at >= F) q = V{};
    } else raw_fetch<T, N, FIT, NT>(q, row, at, F, on);
    return raw_use<T, N, FIT>(q, at, F);
}
template <class T, int N> __device__ __forceinline__ void raw_float(const typename Unaligned<T, N>::type& q, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = (float)q[i];
}
template <class T, int N, int FIT, bool NT = false> __device__ __forceinline__ void row_load(const T* row, int at, int F, bool on, float (&v)[N]) {
    raw_float<T, N>(raw_load<T, N, FIT, NT>(row, at, F, on), v);
}
// v = x + res (res may be NULL)
template <class T, int N, int FIT, bool NT = false> __device__ __forceinline__ void sum_load(const T* x, const T* res, int at, int F, bool on, float (&v)[N]) {
    row_load<T, N, FIT, NT>(x, at, F, on, v);
    if (res) {
        float r[N];
        row_load<T, N, FIT, NT>(res, at, F, on, r);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += r[i];
    }
}
// row[at + i] = v[i], rounded to nearest even, within the row (at < F)
template <class T, int N, int FIT, bool NT = false> __device__ __forceinline__ void row_store(T* row, int at, int F, const float (&v)[N]) {
    typedef typename Unaligned<T, N>::type V;
    V q;
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = (T)v[i];
    if (FIT == EVEN || at + N <= F) {
        if constexpr (NT) __builtin_nontemporal_store(q, reinterpret_cast<V*>(row + at));
        else *reinterpret_cast<V*>(row + at) = q;
    } else {                        // the bits of the number of bytes that are left
        Quad w = __builtin_bit_cast(Quad, q);
        unsigned char* p = reinterpret_cast<unsigned char*>(row + at);
        const int bytes = (F - at) * (int)sizeof(T);
        if (bytes & 8) { __builtin_memcpy(p, &w, 8); p += 8; w = Quad{w.z, w.w, 0u, 0u}; }
        if (bytes & 4) { __builtin_memcpy(p, &w, 4); p += 4; w = Quad{w.y, w.z, w.w, 0u}; }
        if (sizeof(T) == 2 && (bytes & 2)) { const unsigned short h = (unsigned short)w.x; __builtin_memcpy(p, &h, 2); }
    }
}
// the gain: 32 bits or the rows' type; NULL = 1
template <class T, int N, int FIT> __device__ __forceinline__ void gain_load(const void* w, int w32, int at, int F, float (&v)[N]) {
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = 1.0f;
    } else if (w32) {
#pragma unroll
        for (int h = 0; h < N; h += 4) {
            float u[4];
            row_load<float, 4, FIT>((const float*)w, at + h, F, true, u);
#pragma unroll
            for (int i = 0; i < 4; i++) v[h + i] = u[i];
        }
    } else row_load<T, N, FIT>((const T*)w, at, F, true, v);
}

// ---- sums and maxima over the tpr threads of a row.  Within 16 lanes by DPP (quad_perm, then the mirrors of 8 and 16 lanes: every lane of
// a half already holds its half's value), across 16 and 32 lanes by the permlane swaps: no trip through LDS.  All lanes of the wave have to
// be active.  Between waves (tpr > 64: the workgroup is one row) `lds` has two slots per wave; `turn` alternates between them so that one
// barrier per reduction is enough.
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
template <int STEP> __device__ __forceinline__ float lane_partner(float v) { return __uint_as_float(lane_partner<STEP>(__float_as_uint(v))); }
template <int STEP> __device__ __forceinline__ double lane_partner(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = lane_partner<STEP>((unsigned)b), hi = lane_partner<STEP>((unsigned)(b >> 32));
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
// over the lanes of aligned segments of n (a power of two) lanes of a wave
template <class S> __device__ __forceinline__ S lanes_sum(S v, int n) {
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
__device__ __forceinline__ int row_waves(int tpr) { return tpr >> 6; }
template <class S> __device__ __forceinline__ S row_sum(S v, int tpr, double (*lds)[16], int turn) {
    v = lanes_sum(v, tpr);
    if (tpr > 64) {
        if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x >> 6] = (double)v;          // (exact)
        __syncthreads();
        v = (S)0;
        for (int i = 0; i < row_waves(tpr); i++) v += (S)lds[turn][i];
    }
    return v;
}
__device__ __forceinline__ unsigned row_max(unsigned v, int tpr, double (*lds)[16], int turn) {
    v = lanes_max(v, tpr);
    if (tpr > 64) {
        if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x >> 6] = (double)v;          // (exact: 32 bits)
        __syncthreads();
        v = 0;
        for (int i = 0; i < row_waves(tpr); i++) v = max(v, (unsigned)lds[turn][i]);
    }
    return v;
}
// The sum of squares of a row of which this thread holds v[NV][N]; `on`: the row is one (the others may be anything).  Where the 32-bit sum
// is no good the 64-bit one is in `wide` (else wide < 0).  The test is the same in all threads of a row; a wave that shares several rows
// repeats the sum for all of them.
template <int NV, int N> __device__ __forceinline__ float row_squares(const float (&v)[NV][N], bool on, int tpr, double (*lds)[16], double& wide) {
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = v[0][e] * v[0][e];
#pragma unroll
    for (int k = 1; k < NV; k++)
#pragma unroll
        for (int e = 0; e < N; e++) acc[e] = __builtin_fmaf(v[k][e], v[k][e], acc[e]);
#pragma unroll
    for (int o = N / 2; o >= 1; o >>= 1)
#pragma unroll
        for (int e = 0; e < o; e++) acc[e] += acc[e + o];
    const float ss = row_sum(acc[0], tpr, lds, 0);
    const bool odd = on && !(ss > 1e-30f && ss < 1e37f);
    wide = -1.0;
    if (__any(odd)) {           // (tpr > 64: one row, all of its waves agree)
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < N; e++) s += (double)v[k][e] * (double)v[k][e];
        if (tpr > 64) __syncthreads();          // slot 0 has been read by everybody
        s = row_sum(s, tpr, lds, 0);
        if (odd) wide = s;
    }
    return ss;
}
// 1 / sqrt(ss / F + eps): v_rsq_f32 is within one step
__device__ __forceinline__ float rms_inverse(float ss, double wide, double inv_F, float eps) {
    if (__builtin_expect(wide >= 0.0 || wide != wide, 0)) return (float)(1.0 / __builtin_sqrt(wide * inv_F + (double)eps));
    return __builtin_amdgcn_rsqf(__builtin_fmaf(ss, (float)inv_F, eps));
}
// A row's values over its length + eps: v inv, corrected once by its exact remainder v - q d (as a division rounds; the product alone is a step
// further off).  `small`: the inverse lies below the normal numbers, whose spacing would cost bits (3e-5 of the value for rows of 33 000 columns
// near the largest float); d is then 2^64 times smaller than it is, for values divided by 2^64.
struct Length { float d, inv; bool small; };
__device__ __forceinline__ Length l2_length(float ss, double wide, float eps) {
    const bool odd = wide >= 0.0 || wide != wide;
    if (__builtin_expect(odd || eps > 0x1p100f, 0)) {
        const double d = __builtin_sqrt(odd ? wide : (double)ss) + (double)eps;
        const bool small = d > 0x1p126;
        const double e = small ? d * 0x1p-64 : d;
        return {(float)e, e > 0.0 && e < 0x1p-126 ? 0.0f : (float)(1.0 / e), small};           // (so short: a row of zeros, and an eps below the normal numbers)
    }
    const float d = __builtin_sqrtf(ss) + eps;
    return {d, 1.0f / d, false};
}
__device__ __forceinline__ float over_length(float v, const Length& l) {
    const float q = v * l.inv;
    return __builtin_fmaf(__builtin_fmaf(-q, l.d, v), l.inv, q);
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
template <int N, int FIT> __device__ __forceinline__ void code_store(unsigned char* row, int at, int F, const unsigned (&c)[N / 4]) {
    typedef unsigned V __attribute__((ext_vector_type(N / 4), aligned(1)));
    if (FIT == EVEN || at + N <= F) {
        V q;
#pragma unroll
        for (int i = 0; i < N / 4; i++) q[i] = c[i];
        *reinterpret_cast<V*>(row + at) = q;
    } else {                        // the bits of the number of bytes that are left
        unsigned char* p = row + at;
        const int bytes = F - at;
        unsigned w = c[0];
        if (N == 8 && (bytes & 4)) { __builtin_memcpy(p, &w, 4); p += 4; w = c[N / 4 - 1]; }
        if (bytes & 2) { const unsigned short h = (unsigned short)w; __builtin_memcpy(p, &h, 2); p += 2; w >>= 16; }
        if (bytes & 1) *p = (unsigned char)w;
    }
}
template <int N> __device__ __forceinline__ unsigned top_bits_of(const float (&v)[N]) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < N; e++) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
    return m;
}

// s w beyond the largest float although s is finite: the vector is loaded again and formed as (s 2^-64) (w 2^-65), its scale times 2^129.  The
// scaling changes no code: what it loses to small numbers lies below top 2^-20, whose code is 0.  Rare, so behind a branch that whole
// waves take.
constexpr unsigned BEYOND = 0x7f800000u;
template <int N> __device__ __forceinline__ void scaled_product(const float (&s)[N], const float (&w)[N], float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = (s[e] * 0x1p-64f) * (w[e] * 0x1p-65f);
}
__device__ __forceinline__ float stored_scale(float scale, float rstd, bool scaled) {
    return scaled ? (float)((double)scale * (double)rstd * 0x1p129) : scale * rstd;
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
    int F, norm, w32;
    int tpr, mask, tsh, rpb;        // threads per row and how they are told apart (RowShape)
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
// NT: the rows are read past the caches.  GAIN (8 bits): there is one, so that a product may leave the floats (whose rare branch costs the
// writing of a table, which has no gain, 4 %: 258 us for [5 M, 64], 269 with it).
template <class T, int NV, int OUT, int FIT, bool NT, bool GAIN> __global__ __launch_bounds__(512) void rms_forward_kernel(RmsArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x & a.mask;
    const long long i = a.row0 + (long long)blockIdx.x * a.rpb + (threadIdx.x >> a.tsh);
    const bool on = i < a.rows;
    const T* x = (const T*)a.x + (on ? i : 0) * a.ldx;
    const T* res = a.res ? (const T*)a.res + (on ? i : 0) * a.ldr : nullptr;
    float v[NV][N];
#pragma unroll
    for (int k = 0; k < NV; k++) sum_load<T, N, FIT, NT>(x, res, (t + k * tpr) * N, a.F, on, v[k]);
    float rstd = 1.0f;
    if (a.norm) {
        double wide;
        const float ss = row_squares(v, on, tpr, lds, wide);
        rstd = rms_inverse(ss, wide, a.inv_F, a.eps);
    }
    if (a.rstd && on && t == 0) a.rstd[i] = rstd;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * N;
        if (at >= a.F || !on) continue;
        if (a.s) row_store<T, N, FIT>((T*)a.s + i * a.F, at, a.F, v[k]);
        if constexpr (OUT == 0 || GAIN) {
            float w[N];
            gain_load<T, N, FIT>(a.w, a.w32, at, a.F, w);
#pragma unroll
            for (int e = 0; e < N; e++) v[k][e] = OUT == 0 ? v[k][e] * rstd * w[e] : v[k][e] * w[e];
        }
        if constexpr (OUT == 0) row_store<T, N, FIT>((T*)a.y + i * a.F, at, a.F, v[k]);
    }
    if constexpr (OUT != 0) {
        const long long row = row_target(a.to, i, a.rows, t, tpr, lds);
        const int seg = a.groups == 1 ? 0 : (1 << a.gshift) / N;
        unsigned tops[NV], top = 0;
        if (seg == 0) {
#pragma unroll
            for (int k = 0; k < NV; k++) top = max(top, top_bits_of(v[k]));
            top = row_max(top, tpr, lds, 1);
#pragma unroll
            for (int k = 0; k < NV; k++) tops[k] = top;
        } else {
#pragma unroll
            for (int k = 0; k < NV; k++) {          // a group's vectors lie in `seg` neighbouring lanes of one wave
                tops[k] = lanes_max(top_bits_of(v[k]), seg);
                top = max(top, tops[k]);
            }
        }
        bool scaled[NV] = {};
        if constexpr (GAIN) {
            auto again = [&](int k) {
                const int at = (t + k * tpr) * N;
                float s[N], w[N];
                sum_load<T, N, FIT>(x, res, at, a.F, on, s);
#pragma unroll
                for (int e = 0; e < N; e++) w[e] = 0.0f;
                if (at < a.F) gain_load<T, N, FIT>(a.w, a.w32, at, a.F, w);
                scaled_product(s, w, v[k]);
            };
            if (__any(top >= BEYOND)) {             // (per row and tpr > 64: one row, all of its waves agree)
                unsigned small = 0;
#pragma unroll
                for (int k = 0; k < NV; k++) {
                    scaled[k] = tops[k] >= BEYOND;
                    if (scaled[k]) again(k);
                    small = max(small, top_bits_of(v[k]));
                }
                if (seg == 0) {
                    if (tpr > 64) __syncthreads();  // slot 1 has been read by everybody
                    small = row_max(small, tpr, lds, 1);
                }
#pragma unroll
                for (int k = 0; k < NV; k++) {
                    if (seg != 0) small = lanes_max(top_bits_of(v[k]), seg);
                    tops[k] = scaled[k] ? small : tops[k];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int at = (t + k * tpr) * N;
            const Group8 g = group_scale<OUT>(tops[k]);
            if (row < 0 || at >= a.F) continue;
            unsigned c[N / 4];
#pragma unroll
            for (int q = 0; q < N / 4; q++) c[q] = encode4<OUT>(&v[k][4 * q], g);
            code_store<N, FIT>(a.codes + row * a.F, at, a.F, c);
            if ((at & ((1u << a.gshift) - 1u)) == 0) a.scales[row * a.groups + (at >> a.gshift)] = stored_scale(g.scale, rstd, scaled[k]);
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
    const bool by_row = OUT != 0 && a.groups == 1;
    double ss = 0.0;
    unsigned row_top = 0;
    for (int at = t * N; at < a.F; at += tpr * N) {
        float v[N], w[N];
        sum_load<T, N, TAIL>(x, res, at, a.F, true, v);
#pragma unroll
        for (int e = 0; e < N; e++) ss += (double)v[e] * (double)v[e];
        if (by_row) {
            gain_load<T, N, TAIL>(a.w, a.w32, at, a.F, w);
#pragma unroll
            for (int e = 0; e < N; e++) v[e] *= w[e];
            row_top = max(row_top, top_bits_of(v));
        }
    }
    float rstd = 1.0f;
    if (a.norm) rstd = rms_inverse(0.0f, row_sum(ss, tpr, lds, 0), a.inv_F, a.eps);
    if (by_row) row_top = row_max(row_top, tpr, lds, 1);
    const bool row_scaled = by_row && a.w && row_top >= BEYOND;
    if (row_scaled) {                           // (the workgroup is the row)
        row_top = 0;
        for (int at = t * N; at < a.F; at += tpr * N) {
            float v[N], w[N];
            sum_load<T, N, TAIL>(x, res, at, a.F, true, v);
            gain_load<T, N, TAIL>(a.w, a.w32, at, a.F, w);
            scaled_product(v, w, v);
            row_top = max(row_top, top_bits_of(v));
        }
        __syncthreads();                        // slot 1 has been read by everybody
        row_top = row_max(row_top, tpr, lds, 1);
    }
    if (a.rstd && t == 0) a.rstd[i] = rstd;
    const int seg = OUT == 0 || by_row ? 0 : (1 << a.gshift) / N;
    // (all threads of a wave take every step together: the groups' maxima go from lane to lane)
    for (int base = 0; base < a.F; base += tpr * N) {
        const int at = base + t * N;
        const bool in = at < a.F;
        float v[N], w[N];
        sum_load<T, N, TAIL>(x, res, at, a.F, in, v);
        if (a.s && in) row_store<T, N, TAIL>((T*)a.s + i * a.F, at, a.F, v);
#pragma unroll
        for (int e = 0; e < N; e++) w[e] = 0.0f;
        if (in) gain_load<T, N, TAIL>(a.w, a.w32, at, a.F, w);
        if constexpr (OUT == 0) {
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = v[e] * rstd * w[e];
            if (in) row_store<T, N, TAIL>((T*)a.y + i * a.F, at, a.F, v);
        } else {
            float s[N];
#pragma unroll
            for (int e = 0; e < N; e++) { s[e] = v[e]; v[e] *= w[e]; }
            unsigned top = row_top;
            bool scaled = row_scaled;
            if (seg != 0) {
                top = lanes_max(top_bits_of(v), seg);
                scaled = a.w && top >= BEYOND;
            }
            if (a.w && __any(scaled)) {
                if (scaled) scaled_product(s, w, v);
                const unsigned small = seg != 0 ? lanes_max(top_bits_of(v), seg) : row_top;
                if (scaled) top = small;
            }
            const Group8 g = group_scale<OUT>(top);
            if (row >= 0 && in) {
                unsigned c[N / 4];
#pragma unroll
                for (int q = 0; q < N / 4; q++) c[q] = encode4<OUT>(&v[4 * q], g);
                code_store<N, TAIL>(a.codes + row * a.F, at, a.F, c);
                if ((at & ((1u << a.gshift) - 1u)) == 0) a.scales[row * a.groups + (at >> a.gshift)] = stored_scale(g.scale, rstd, scaled);
            }
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------
struct RmsBackArgs {
    long long rows, row0;   // row0: of the *_long kernel
    int F, w32;
    int tpr, mask, tsh, rpb;
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
// Up to 512 threads the next row's loads are in flight while a row is reduced and written; 1024 threads (the widest rows) have no registers for
// that, nor for the gain (read again for every row, from the caches), but as many waves to hide behind.
template <class T, int NV, int FIT, bool NT, int MOST> __global__ __launch_bounds__(MOST) void rms_backward_kernel(RmsBackArgs a) {
    constexpr bool AHEAD = MOST <= 512;
    constexpr int N = RowVec<T>::N;
    typedef typename Unaligned<T, N>::type V;
    __shared__ double lds[2][16];
    __shared__ float part[4][64 * N];       // the waves' sums of one vector slot
    const int tpr = a.tpr, t = threadIdx.x & a.mask, rpb = a.rpb;
    float dw[NV][N], w[NV][N];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * N;
#pragma unroll
        for (int e = 0; e < N; e++) { dw[k][e] = 0.0f; w[k][e] = 0.0f; }
        if (AHEAD && at < a.F) gain_load<T, N, FIT>(a.w, a.w32, at, a.F, w[k]);
    }
    const long long step = (long long)gridDim.x * rpb;
    long long i = (long long)blockIdx.x * rpb + (threadIdx.x >> a.tsh);
    V xq[NV] = {}, rq[NV] = {}, gq[NV] = {}, sq[NV] = {};
    float rstd;
    auto fetch = [&](long long row) {           // (rows beyond the last are off)
        const bool on = row < a.rows;
        const long long r = on ? row : 0;
        rstd = on ? a.rstd[r] : 0.0f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int at = (t + k * tpr) * N;
            raw_fetch<T, N, FIT, NT>(xq[k], (const T*)a.x + r * a.ldx, at, a.F, on);
            raw_fetch<T, N, FIT, NT>(gq[k], (const T*)a.gy + r * a.ldg, at, a.F, on);
            if (a.res) raw_fetch<T, N, FIT, NT>(rq[k], (const T*)a.res + r * a.ldr, at, a.F, on);
            if (a.gs) raw_fetch<T, N, FIT, NT>(sq[k], (const T*)a.gs + r * a.ldgs, at, a.F, on);
        }
    };
    if (AHEAD) fetch(i);
    int turn = 0;
    for (long long r0 = (long long)blockIdx.x * rpb; r0 < a.rows; r0 += step, i += step, turn ^= 1) {
        const bool on = i < a.rows;
        if constexpr (!AHEAD) {
            // the raw vectors stay, h and gy w are formed twice
#pragma unroll
            for (int k = 0; k < NV; k++) xq[k] = rq[k] = gq[k] = sq[k] = V{};
            fetch(i);
            float c[N];
#pragma unroll
            for (int e = 0; e < N; e++) c[e] = 0.0f;
            auto terms = [&](int k, float (&h)[N], float (&g)[N]) {
                raw_float<T, N>(xq[k], h);
                raw_float<T, N>(gq[k], g);
                if (a.res) {
                    float r[N];
                    raw_float<T, N>(rq[k], r);
#pragma unroll
                    for (int e = 0; e < N; e++) h[e] += r[e];
                }
#pragma unroll
                for (int e = 0; e < N; e++) h[e] *= rstd;
            };
            auto times_gain = [&](int at, float (&g)[N]) {
                float u[N];
                gain_load<T, N, FIT>(a.w, a.w32, at, a.F, u);
#pragma unroll
                for (int e = 0; e < N; e++) g[e] *= u[e];
            };
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int at = (t + k * tpr) * N;
                if (at >= a.F) continue;
                xq[k] = raw_use<T, N, FIT>(xq[k], at, a.F);
                gq[k] = raw_use<T, N, FIT>(gq[k], at, a.F);
                rq[k] = raw_use<T, N, FIT>(rq[k], at, a.F);
                float h[N], g[N];
                terms(k, h, g);
#pragma unroll
                for (int e = 0; e < N; e++) dw[k][e] = __builtin_fmaf(g[e], h[e], dw[k][e]);        // (the workgroup is one row: on)
                times_gain(at, g);
#pragma unroll
                for (int e = 0; e < N; e++) c[e] = __builtin_fmaf(g[e], h[e], c[e]);
            }
#pragma unroll
            for (int o = N / 2; o >= 1; o >>= 1)
#pragma unroll
                for (int e = 0; e < o; e++) c[e] += c[e + o];
            const float mean = row_sum(c[0], tpr, lds, turn) / (float)a.F;
            if (a.ds == nullptr) continue;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int at = (t + k * tpr) * N;
                if (at >= a.F) continue;
                float h[N], g[N];
                terms(k, h, g);
                times_gain(at, g);
#pragma unroll
                for (int e = 0; e < N; e++) g[e] = rstd * (g[e] - h[e] * mean);
                if (a.gs) {
                    raw_float<T, N>(raw_use<T, N, FIT>(sq[k], at, a.F), h);
#pragma unroll
                    for (int e = 0; e < N; e++) g[e] += h[e];
                }
                row_store<T, N, FIT, NT>((T*)a.ds + i * a.F, at, a.F, g);
            }
            continue;
        }
        const float rs = rstd;
        float h[NV][N], g[NV][N], c[N];
        V q[NV];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int at = (t + k * tpr) * N;
            raw_float<T, N>(raw_use<T, N, FIT>(xq[k], at, a.F), h[k]);
            raw_float<T, N>(raw_use<T, N, FIT>(gq[k], at, a.F), g[k]);
            if (a.gs) q[k] = raw_use<T, N, FIT>(sq[k], at, a.F);
            if (a.res) {
                float r[N];
                raw_float<T, N>(raw_use<T, N, FIT>(rq[k], at, a.F), r);
#pragma unroll
                for (int e = 0; e < N; e++) h[k][e] += r[e];
            }
        }
        fetch(i + step);                        // in flight while this row is reduced and written
#pragma unroll
        for (int e = 0; e < N; e++) c[e] = 0.0f;
        // (a vector behind the row holds zeros; a row that is off holds an earlier one and has no part in dw)
#pragma unroll
        for (int k = 0; k < NV; k++) {
#pragma unroll
            for (int e = 0; e < N; e++) {
                h[k][e] *= rs;
                if (on) dw[k][e] = __builtin_fmaf(g[k][e], h[k][e], dw[k][e]);
                g[k][e] *= w[k][e];
                c[e] = __builtin_fmaf(g[k][e], h[k][e], c[e]);
            }
        }
#pragma unroll
        for (int o = N / 2; o >= 1; o >>= 1)
#pragma unroll
            for (int e = 0; e < o; e++) c[e] += c[e + o];
        const float mean = row_sum(c[0], tpr, lds, turn) / (float)a.F;
        if (a.ds == nullptr) continue;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int at = (t + k * tpr) * N;
            if (at >= a.F || !on) continue;
            float d[N];
#pragma unroll
            for (int e = 0; e < N; e++) d[e] = rs * (g[k][e] - h[k][e] * mean);
            if (a.gs) {
                float u[N];
                raw_float<T, N>(q[k], u);
#pragma unroll
                for (int e = 0; e < N; e++) d[e] += u[e];
            }
            row_store<T, N, FIT, NT>((T*)a.ds + i * a.F, at, a.F, d);
        }
    }
    if (a.dw_part == nullptr) return;
    // the rows of a wave first, then the waves, in a fixed order
    float* out = a.dw_part + (long long)blockIdx.x * a.F;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        for (int o = 32; o >= tpr; o >>= 1)
#pragma unroll
            for (int e = 0; e < N; e++) dw[k][e] += __shfl_xor(dw[k][e], o);
        const int at = (t + k * tpr) * N;
        if (rpb > 1) {                          // (tpr <= 64: every wave has sums of the same columns)
            const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
            __syncthreads();
            if (lane < tpr)
#pragma unroll
                for (int e = 0; e < N; e++) part[wave][lane * N + e] = dw[k][e];
            __syncthreads();
            if ((int)threadIdx.x < tpr)
                for (int q = 1; q < (int)(blockDim.x >> 6); q++)
#pragma unroll
                    for (int e = 0; e < N; e++) dw[k][e] += part[q][lane * N + e];
        }
        if ((int)threadIdx.x < tpr)
#pragma unroll
            for (int h = 0; h < N; h += 4)
                if (at + h < a.F) {
                    const float d[4] = {dw[k][h], dw[k][h + 1], dw[k][h + 2], dw[k][h + 3]};
                    row_store<float, 4, FIT>(out, at + h, a.F, d);
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
        sum_load<T, N, TAIL>(x, res, at, a.F, true, h);
        row_load<T, N, TAIL>(gy, at, a.F, true, g);
        gain_load<T, N, TAIL>(a.w, a.w32, at, a.F, w);
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) p += g[e] * w[e] * (h[e] * rstd);
        c += (double)p;
    }
    const float mean = (float)row_sum(c, tpr, lds, 0) / (float)a.F;
    for (int at = t * N; at < a.F; at += tpr * N) {
        float h[N], g[N], w[N], d[N];
        sum_load<T, N, TAIL>(x, res, at, a.F, true, h);
        row_load<T, N, TAIL>(gy, at, a.F, true, g);
        gain_load<T, N, TAIL>(a.w, a.w32, at, a.F, w);
#pragma unroll
        for (int e = 0; e < N; e++) d[e] = rstd * (g[e] * w[e] - h[e] * rstd * mean);
        if (a.gs) {
            float q[N];
            row_load<T, N, TAIL>((const T*)a.gs + i * a.ldgs, at, a.F, true, q);
#pragma unroll
            for (int e = 0; e < N; e++) d[e] += q[e];
        }
        row_store<T, N, TAIL>((T*)a.ds + i * a.F, at, a.F, d);
    }
}
template <class T> __global__ __launch_bounds__(256) void rms_dw_columns_kernel(RmsBackArgs a, int slices) {
    constexpr int N = RowVec<T>::N;
    const int at = ((int)blockIdx.x * 256 + (int)threadIdx.x) * N;
    if (at >= a.F) return;
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; e++) sum[e] = 0.0f;
    for (long long i = blockIdx.y; i < a.rows; i += slices) {
        const float rstd = a.rstd[i];
        float h[N], g[N];
        sum_load<T, N, TAIL>((const T*)a.x + i * a.ldx, a.res ? (const T*)a.res + i * a.ldr : nullptr, at, a.F, true, h);
        row_load<T, N, TAIL>((const T*)a.gy + i * a.ldg, at, a.F, true, g);
#pragma unroll
        for (int e = 0; e < N; e++) sum[e] += g[e] * (h[e] * rstd);
    }
#pragma unroll
    for (int h = 0; h < N; h += 4)
        if (at + h < a.F) {
            const float d[4] = {sum[h], sum[h + 1], sum[h + 2], sum[h + 3]};
            row_store<float, 4, TAIL>(a.dw_part + (long long)blockIdx.y * a.F, at + h, a.F, d);
        }
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
    int F, groups, gshift, norm, is64;
    int tpr, mask, tsh, rpb;
    float eps;
    const unsigned char* codes;
    const float* scales;
    const void* index;      // or NULL
    void* out;              // [rows, F]
};
// the codes of N columns and their scale as values, zeros beyond the row and for rows that are off
template <int CODE, int N, int FIT> __device__ __forceinline__ void code_load(const ReadArgs& a, long long row, int at, float (&v)[N]) {
    const unsigned char* codes = a.codes + (row >= 0 ? row : 0) * a.F;
    const bool in = row >= 0 && at < a.F;
    const int p = FIT != NARROW ? min(at, a.F - N) : at;
    float scale = 0.0f;
    unsigned c[N / 4] = {};
    if (a.P > 0) {          // (an empty table has nothing to draw the address back to)
        scale = a.scales[(row >= 0 ? row : 0) * a.groups + (min(at, a.F - 1) >> a.gshift)];
        if (FIT != NARROW) __builtin_memcpy(c, codes + p, N);
        else if (in)
            for (int e = 0; e < N && at + e < a.F; e++) c[e / 4] |= (unsigned)codes[at + e] << (8 * (e & 3));
        if (FIT == TAIL && in && at > p) {        // the row's last N codes: those in front of `at` go
            unsigned long long w = 0;
            __builtin_memcpy(&w, c, N);
            w >>= 8 * (at - p);
            __builtin_memcpy(c, &w, N);
        }
    }
#pragma unroll
    for (int q = 0; q < N / 4; q++) Code8<CODE>::unpack4(c[q], v + 4 * q);
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = in && (FIT == EVEN || at + e < a.F) ? v[e] * scale : 0.0f;
}
__device__ __forceinline__ long long read_row(const ReadArgs& a, long long i) {
    const long long row = a.index == nullptr ? a.first + i : a.is64 ? ((const long long*)a.index)[i] : (long long)((const int*)a.index)[i];
    return row < a.P ? row : -1;
}
// NT: written past the caches.
template <class T, int CODE, int NV, int FIT, bool NT> __global__ __launch_bounds__(512) void rows_read_kernel(ReadArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x & a.mask;
    const long long i = a.row0 + (long long)blockIdx.x * a.rpb + (threadIdx.x >> a.tsh);
    const long long row = i < a.rows ? read_row(a, i) : -1;
    float v[NV][N];
#pragma unroll
    for (int k = 0; k < NV; k++) code_load<CODE, N, FIT>(a, row, (t + k * tpr) * N, v[k]);
    if (a.norm) {
        double wide;
        const float ss = row_squares(v, row >= 0, tpr, lds, wide);
        const Length l = row >= 0 ? l2_length(ss, wide, a.eps) : Length{0.0f, 0.0f, false};
        if (l.small)
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int e = 0; e < N; e++) v[k][e] *= 0x1p-64f;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < N; e++) v[k][e] = over_length(v[k][e], l);
    }
    if (i >= a.rows) return;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int at = (t + k * tpr) * N;
        if (at < a.F) row_store<T, N, FIT, NT>((T*)a.out + i * a.F, at, a.F, v[k]);
    }
}
template <class T, int CODE> __global__ __launch_bounds__(512) void rows_read_long_kernel(ReadArgs a) {
    constexpr int N = RowVec<T>::N;
    __shared__ double lds[2][16];
    const int tpr = a.tpr, t = threadIdx.x;
    const long long i = a.row0 + blockIdx.x, row = read_row(a, i);
    Length l = {1.0f, 1.0f, false};
    if (a.norm) {
        double ss = 0.0;
        for (int at = t * N; at < a.F; at += tpr * N) {
            float v[N];
            code_load<CODE, N, TAIL>(a, row, at, v);
#pragma unroll
            for (int e = 0; e < N; e++) ss += (double)v[e] * (double)v[e];
        }
        ss = row_sum(ss, tpr, lds, 0);
        l = row >= 0 ? l2_length(0.0f, ss, a.eps) : Length{0.0f, 0.0f, false};
    }
    for (int at = t * N; at < a.F; at += tpr * N) {
        float v[N];
        code_load<CODE, N, TAIL>(a, row, at, v);
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = over_length(l.small ? v[e] * 0x1p-64f : v[e], l);
        row_store<T, N, TAIL>((T*)a.out + i * a.F, at, a.F, v);
    }
}

}  // namespace iso
