// C-ABI entry points of libinstascene_hip.so for rows and gradients (declared in include/instascene_ops.h): the root-mean-square
// norm, the 8-bit row table, the global gradient norm.  Host-side only: argument checking and launches on the caller's stream; no
// allocation, no synchronisation, nothing recorded that a captured graph could not replay.
#include <algorithm>
#include "isr_host.hpp"
#include "iso_rows.hip"
#include "iso_gradnorm.hip"

using namespace isr;

namespace {

constexpr long long MAX_THREADS = 1ll << 31;       // per launch (the grid times the workgroup has to stay below 2^32)

bool row_type(int t) { return t >= 0 && t <= 2; }       // 0 float32, 1 bfloat16, 2 float16
int type_bytes(int t) { return t == 0 ? 4 : 2; }
bool code_type(int c) { return c == iso::CODE_INT8 || c == iso::CODE_E4M3; }
// columns of a group: the whole row, or 32 / 64 / 128 dividing it
bool group_ok(int F, int group) { return group == F || ((group == 32 || group == 64 || group == 128) && F % group == 0); }
int group_shift(int F, int group) { return group == F ? 31 : group == 32 ? 5 : group == 64 ? 6 : 7; }

// From this many bytes on a stream goes past the caches (256 MB in front of the memory), from which the next kernel would find little:
// the backward pass reads and writes so (forward + backward per stream of 32 / 48 / 64 / 96 MB: [n, 32] float32 47.2 / 65.8 / 89.3 / 134 us, with
// cached lines 44.6 / 71.5 / 95.4 / 147; [n, 4096] bfloat16 56.5 / 79.6 / 107 / 157, cached 51.6 / 74.9 / 110 / 176), 8-bit rows are written from and
// read to (the table of [5 M, 64] 530 us, cached 550; [16384, 4096] bfloat16 quantised 86, cached 94; at 92 MB 61 and 68 with 40 and 46 at 64 MB the
// other way round).  A forward pass, whose outputs the next kernel reads, loses (128 -> 134) and keeps its lines.
constexpr long long NT_BACKWARD = 64ll << 20, NT_CODES = 128ll << 20;

// How a kernel lays rows of `vecs` vectors over its threads: tpr threads and nv vectors per thread for each (nv = 0: the *_long form), thread t of
// the row = threadIdx.x & mask, row of the workgroup = threadIdx.x >> tsh, rpb rows per workgroup.
// Up to a wave: a power of two, `least` vectors per thread where there are rows enough to fill the chip all the same: 2 for 8-bit rows, whose work
// per row (scales, the norm) weighs less then ([5 M, 64]: written 283 -> 258 us, read 359 -> 252; 4 are slower again, 64-byte pieces), 1 for the
// norm ([1.5 M, 32]: 128 us, 160 with 2).  Beyond: a workgroup of whole waves per row, 2 vectors per thread ([8192, 8192] bfloat16: 240 us forward
// and backward, 333 with 4, 456 with 8), as many waves as the row needs.  Where there are so few rows that the chip would stand idle, 1 vector
// per thread.
struct RowShape { int tpr, mask, tsh, rpb, nv, block; };
RowShape row_shape(int vecs, long long rows, int least, int max_nv, int max_waves = 8) {
    int tsh = 0;
    while ((1 << tsh) < vecs && tsh < 6) tsh++;
    while (tsh > 0 && (vecs + (1 << (tsh - 1)) - 1) >> (tsh - 1) <= least && (rows << (tsh - 1)) >= 2048 * 256) tsh--;
    const int per_lane = (vecs + (1 << tsh) - 1) >> tsh;
    if (per_lane <= (tsh == 6 && rows * 64 < 256 * 256 ? 1 : 2)) return {1 << tsh, (1 << tsh) - 1, tsh, 256 >> tsh, per_lane, 256};
    for (int nv = rows * ((vecs + 1) / 2) < 256 * 256 ? 1 : 2; nv <= max_nv; nv *= 2) {
        const int waves = (vecs + 64 * nv - 1) / (64 * nv);
        if (waves <= (nv == max_nv ? max_waves : 8)) return {64 * waves, 0x7fffffff, 31, 1, nv, 64 * waves};
    }
    return {512, 0x7fffffff, 31, 1, 0, 512};
}
template <class A> void set_shape(A& a, const RowShape& r) { a.tpr = r.tpr; a.mask = r.mask; a.tsh = r.tsh; a.rpb = r.rpb; }

#define ROWS_NV(nv, fit, call, call_long) \
    do { if (fit == iso::NARROW) { call(1, iso::NARROW); } else if (nv == 0) { call_long; } \
         else if (fit == iso::EVEN) { if (nv == 1) { call(1, iso::EVEN); } else if (nv == 2) { call(2, iso::EVEN); } else if (nv == 4) { call(4, iso::EVEN); } else { call(8, iso::EVEN); } } \
         else { if (nv == 1) { call(1, iso::TAIL); } else if (nv == 2) { call(2, iso::TAIL); } else if (nv == 4) { call(4, iso::TAIL); } else { call(8, iso::TAIL); } } } while (0)
template <class T> int row_fit(int F) { return F < iso::RowVec<T>::N ? iso::NARROW : F % iso::RowVec<T>::N ? iso::TAIL : iso::EVEN; }

template <class T, int OUT> void launch_forward(iso::RmsArgs a, hipStream_t s) {
    constexpr int N = iso::RowVec<T>::N;
    const RowShape sh = row_shape((a.F + N - 1) / N, a.rows, OUT == 0 ? 1 : 2, 8);
    set_shape(a, sh);
    const int nv = sh.nv;
    // (past the caches only whole 128-byte lines per load: [8 M, 32] float32 224 us so with 4 threads per row, 174 cached)
    const bool nt = OUT != 0 && a.tpr >= 8 && a.rows * a.F * (long long)sizeof(T) >= NT_CODES;
    const int fit = row_fit<T>(a.F);
    const int block = sh.block, rpb = sh.rpb;
    const long long step = MAX_THREADS / block * rpb;
    for (a.row0 = 0; a.row0 < a.rows; a.row0 += step) {
        const long long n = std::min(step, a.rows - a.row0);
        const dim3 grid((unsigned)((n + rpb - 1) / rpb));
// (so many bytes with one vector per thread do not occur: there are rows enough for two)
#define FWD_AS(NV, FIT, NT, GAIN) hipLaunchKernelGGL((iso::rms_forward_kernel<T, NV, OUT, FIT, NT, GAIN>), grid, dim3(block), 0, s, a)
#define FWD(NV, FIT) do { constexpr bool NT = OUT != 0 && NV > 1, GAIN = OUT != 0; \
                           if (nt && a.w) FWD_AS(NV, FIT, NT, GAIN); \
                           else if (nt) FWD_AS(NV, FIT, NT, false); \
                           else if (a.w) FWD_AS(NV, FIT, false, GAIN); \
                           else FWD_AS(NV, FIT, false, false); } while (0)
#define FWD_LONG hipLaunchKernelGGL((iso::rms_forward_long_kernel<T, OUT>), grid, dim3(block), 0, s, a)
        ROWS_NV(nv, fit, FWD, FWD_LONG);
#undef FWD
#undef FWD_AS
#undef FWD_LONG
    }
}
template <int OUT> void launch_forward_type(int type, const iso::RmsArgs& a, hipStream_t s) {
    if (type == 0) launch_forward<float, OUT>(a, s);
    else if (type == 1) launch_forward<__bf16, OUT>(a, s);
    else launch_forward<_Float16, OUT>(a, s);
}
void launch_codes(int code, int type, const iso::RmsArgs& a, hipStream_t s) {
    if (code == iso::CODE_INT8) launch_forward_type<iso::CODE_INT8>(type, a, s);
    else launch_forward_type<iso::CODE_E4M3>(type, a, s);
}

// workgroups of the backward pass = partial rows of dw: enough to keep the memory busy (two of 256 threads per compute unit do for wide rows:
// 768 and 1024 workgroups took 1 to 14 % longer at [n, 2048..4096] float32), few enough that the partials stay small against the rows
template <class T> RowShape backward_shape(long long rows, int F, int& grid) {
    const RowShape sh = row_shape((F + iso::RowVec<T>::N - 1) / iso::RowVec<T>::N, rows, 1, 2, 16);       // (what the registers hold)
    if (sh.nv == 0) {           // slices of the columns' sums: 1024 workgroups with those that the columns need
        const int cols = 256 * iso::RowVec<T>::N;
        grid = (int)std::max<long long>(1, std::min<long long>(rows, std::max(16, 1024 / ((F + cols - 1) / cols))));
        return sh;
    }
    const long long need = (rows + sh.rpb - 1) / sh.rpb, most = std::max<long long>(512, std::min<long long>(2048, (1 << 20) / F));
    grid = (int)std::max<long long>(1, std::min(need, most));
    return sh;
}
RowShape backward_shape_type(int type, long long rows, int F, int& grid) {
    return type == 0 ? backward_shape<float>(rows, F, grid) : type == 1 ? backward_shape<__bf16>(rows, F, grid) : backward_shape<_Float16>(rows, F, grid);
}
template <class T, int FIT, bool NT> void launch_backward_fit(const iso::RmsBackArgs& a, int nv, int block, int grid, hipStream_t s) {
    if (block > 512) hipLaunchKernelGGL((iso::rms_backward_kernel<T, 2, FIT, NT, 1024>), dim3(grid), dim3(block), 0, s, a);
    else if (nv == 1) hipLaunchKernelGGL((iso::rms_backward_kernel<T, 1, FIT, NT, 512>), dim3(grid), dim3(block), 0, s, a);
    else hipLaunchKernelGGL((iso::rms_backward_kernel<T, 2, FIT, NT, 512>), dim3(grid), dim3(block), 0, s, a);
}
template <class T> void launch_backward(iso::RmsBackArgs a, int nv, int block, int grid, hipStream_t s) {
    if (nv != 0) {
        const int fit = row_fit<T>(a.F);
        const bool nt = a.rows * a.F * (long long)sizeof(T) >= NT_BACKWARD;
        if (fit == iso::NARROW) hipLaunchKernelGGL((iso::rms_backward_kernel<T, 1, iso::NARROW, false, 512>), dim3(grid), dim3(block), 0, s, a);
        else if (fit == iso::EVEN && nt) launch_backward_fit<T, iso::EVEN, true>(a, nv, block, grid, s);
        else if (fit == iso::EVEN) launch_backward_fit<T, iso::EVEN, false>(a, nv, block, grid, s);
        else if (nt) launch_backward_fit<T, iso::TAIL, true>(a, nv, block, grid, s);
        else launch_backward_fit<T, iso::TAIL, false>(a, nv, block, grid, s);
        return;
    }
    if (a.ds)
        for (a.row0 = 0; a.row0 < a.rows; a.row0 += MAX_THREADS / 512)
            hipLaunchKernelGGL((iso::rms_backward_long_kernel<T>), dim3((unsigned)std::min(MAX_THREADS / 512, a.rows - a.row0)), dim3(512), 0, s, a);
    if (a.dw_part) hipLaunchKernelGGL((iso::rms_dw_columns_kernel<T>), dim3((a.F + 256 * iso::RowVec<T>::N - 1) / (256 * iso::RowVec<T>::N), grid), dim3(256), 0, s, a, grid);
}
template <class T, int CODE> void launch_read(iso::ReadArgs a, hipStream_t s) {
    constexpr int N = iso::RowVec<T>::N;
    const RowShape sh = row_shape((a.F + N - 1) / N, a.rows, 2, 8);
    set_shape(a, sh);
    const int nv = sh.nv;
    const int fit = row_fit<T>(a.F);
    const bool nt = a.rows * a.F * (long long)sizeof(T) >= NT_CODES;
    const int block = sh.block, rpb = sh.rpb;
    const long long step = MAX_THREADS / block * rpb;
    for (a.row0 = 0; a.row0 < a.rows; a.row0 += step) {
        const long long n = std::min(step, a.rows - a.row0);
        const dim3 grid((unsigned)((n + rpb - 1) / rpb));
#define READ(NV, FIT) do { if (nt) hipLaunchKernelGGL((iso::rows_read_kernel<T, CODE, NV, FIT, (NV > 1 || FIT != iso::TAIL)>), grid, dim3(block), 0, s, a); \
                            else hipLaunchKernelGGL((iso::rows_read_kernel<T, CODE, NV, FIT, false>), grid, dim3(block), 0, s, a); } while (0)
#define READ_LONG hipLaunchKernelGGL((iso::rows_read_long_kernel<T, CODE>), grid, dim3(block), 0, s, a)
        ROWS_NV(nv, fit, READ, READ_LONG);
#undef READ
#undef READ_LONG
    }
}
template <class T> void launch_read_code(int code, const iso::ReadArgs& a, hipStream_t s) {
    if (code == iso::CODE_INT8) launch_read<T, iso::CODE_INT8>(a, s);
    else launch_read<T, iso::CODE_E4M3>(a, s);
}

int check_rows(const char* what, int type, long long rows, int F) {
    if (!row_type(type)) return fail(ISR_EINVAL, "%s: type %d is none of 0 (float32), 1 (bfloat16), 2 (float16)", what, type);
    if (rows < 0 || F < 1 || F > (1 << 24)) return fail(ISR_EINVAL, "%s: needs rows >= 0 and 1 <= F <= 2^24", what);
    return ISR_OK;
}

}  // namespace

extern "C" {

int iso_rms_norm_forward(int type, long long rows, int F, const void* x, long long x_stride, const void* residual,
                         long long residual_stride, const void* weight, int weight_is_float, float eps, void* y, void* s_out,
                         float* rstd, void* stream) {
    if (const int e = check_rows("rms_norm_forward", type, rows, F)) return e;
    if (rows == 0) return ISR_OK;
    if (!x || !y || !(eps > 0.0f)) return fail(ISR_EINVAL, "rms_norm_forward: null pointer, or eps not positive");
    iso::RmsArgs a = {};
    a.rows = rows; a.F = F; a.norm = 1; a.w32 = weight_is_float; a.eps = eps; a.inv_F = 1.0 / F;
    a.x = x; a.ldx = x_stride; a.res = residual; a.ldr = residual_stride; a.w = weight; a.y = y; a.s = s_out; a.rstd = rstd;
    launch_forward_type<0>(type, a, (hipStream_t)stream);
    ISR_LAUNCH_CHECK_S("iso_rms_norm_forward", (hipStream_t)stream);
    return ISR_OK;
}

int iso_rms_norm_quant(int type, int code, long long rows, int F, int group, const void* x, long long x_stride, const void* residual,
                       long long residual_stride, const void* weight, int weight_is_float, float eps, void* codes, float* scales,
                       void* s_out, void* stream) {
    if (const int e = check_rows("rms_norm_quant", type, rows, F)) return e;
    if (!code_type(code)) return fail(ISR_EINVAL, "rms_norm_quant: code %d is neither 1 (int8) nor 2 (e4m3)", code);
    if (!group_ok(F, group)) return fail(ISR_EINVAL, "rms_norm_quant: groups of %d columns do not fit rows of %d", group, F);
    if (rows == 0) return ISR_OK;
    if (!x || !codes || !scales || !(eps > 0.0f)) return fail(ISR_EINVAL, "rms_norm_quant: null pointer, or eps not positive");
    iso::RmsArgs a = {};
    a.rows = rows; a.F = F; a.norm = 1; a.w32 = weight_is_float; a.eps = eps; a.inv_F = 1.0 / F;
    a.x = x; a.ldx = x_stride; a.res = residual; a.ldr = residual_stride; a.w = weight; a.s = s_out;
    a.codes = (unsigned char*)codes; a.scales = scales; a.groups = F / group; a.gshift = group_shift(F, group);
    a.to.P = rows;
    launch_codes(code, type, a, (hipStream_t)stream);
    ISR_LAUNCH_CHECK_S("iso_rms_norm_quant", (hipStream_t)stream);
    return ISR_OK;
}

size_t iso_rms_norm_scratch_bytes(int type, long long rows, int F) {
    if (!row_type(type) || rows <= 0 || F < 1 || F > (1 << 24)) return 0;
    int grid;
    backward_shape_type(type, rows, F, grid);
    return (size_t)grid * (size_t)F * sizeof(float);
}

int iso_rms_norm_backward(int type, long long rows, int F, const void* x, long long x_stride, const void* residual,
                          long long residual_stride, const void* weight, int weight_is_float,
                          const float* rstd, const void* gy, long long gy_stride, const void* gs, long long gs_stride, void* ds,
                          void* dw, void* scratch, size_t scratch_bytes, void* stream) {
    if (const int e = check_rows("rms_norm_backward", type, rows, F)) return e;
    hipStream_t s = (hipStream_t)stream;
    if (rows == 0) return ISR_OK;
    if (!x || !rstd || !gy || (!ds && !dw)) return fail(ISR_EINVAL, "rms_norm_backward: null pointer");
    if (dw && (!scratch || scratch_bytes < iso_rms_norm_scratch_bytes(type, rows, F))) return fail(ISR_EINVAL, "rms_norm_backward: scratch too small");
    iso::RmsBackArgs a = {};
    a.rows = rows; a.F = F; a.w32 = weight_is_float; a.x = x; a.ldx = x_stride; a.res = residual; a.ldr = residual_stride; a.w = weight; a.rstd = rstd;
    a.gy = gy; a.ldg = gy_stride; a.gs = gs; a.ldgs = gs_stride; a.ds = ds; a.dw_part = dw ? (float*)scratch : nullptr;
    int grid;
    const RowShape sh = backward_shape_type(type, rows, F, grid);
    set_shape(a, sh);
    const int nv = sh.nv, block = sh.block;
    if (type == 0) launch_backward<float>(a, nv, block, grid, s);
    else if (type == 1) launch_backward<__bf16>(a, nv, block, grid, s);
    else launch_backward<_Float16>(a, nv, block, grid, s);
    ISR_LAUNCH_CHECK("iso_rms_norm_backward");
    if (dw) {
        const dim3 cols((F + 31) / 32);
        if (weight_is_float || type == 0) hipLaunchKernelGGL((iso::rms_dw_sum_kernel<float>), cols, dim3(1024), 0, s, F, grid, (const float*)scratch, (float*)dw);
        else if (type == 1) hipLaunchKernelGGL((iso::rms_dw_sum_kernel<__bf16>), cols, dim3(1024), 0, s, F, grid, (const float*)scratch, (__bf16*)dw);
        else hipLaunchKernelGGL((iso::rms_dw_sum_kernel<_Float16>), cols, dim3(1024), 0, s, F, grid, (const float*)scratch, (_Float16*)dw);
        ISR_LAUNCH_CHECK("iso_rms_norm_backward");
    }
    return ISR_OK;
}

int iso_rows8_write(int type, int code, long long n, int F, int group, long long P, const void* rows, long long row_stride, long long first,
                    const void* index, int index_is_int64, int* owner, void* codes, float* scales, void* stream) {
    if (const int e = check_rows("rows8_write", type, n, F)) return e;
    hipStream_t s = (hipStream_t)stream;
    if (!code_type(code)) return fail(ISR_EINVAL, "rows8_write: code %d is neither 1 (int8) nor 2 (e4m3)", code);
    if (!group_ok(F, group)) return fail(ISR_EINVAL, "rows8_write: groups of %d columns do not fit rows of %d", group, F);
    if (index && n > 0x7fffffffll) return fail(ISR_EINVAL, "rows8_write: at most 2^31 - 1 indices in one call");
    if (P < 0 || (!index && (first < 0 || first > P || n > P - first))) return fail(ISR_EINVAL, "rows8_write: rows [%lld, %lld) of a table of %lld", first, first + n, P);
    if (n == 0 || P == 0) return ISR_OK;
    if (!rows || !codes || !scales) return fail(ISR_EINVAL, "rows8_write: null pointer");
    if (index && n > ISO_ROWS8_SCAN && !owner) return fail(ISR_EINVAL, "rows8_write: more than %d indices need the owner table", ISO_ROWS8_SCAN);
    iso::RmsArgs a = {};
    a.rows = n; a.F = F; a.x = rows; a.ldx = row_stride;
    a.codes = (unsigned char*)codes; a.scales = scales; a.groups = F / group; a.gshift = group_shift(F, group);
    a.to.P = P; a.to.first = first; a.to.index = index; a.to.is64 = index_is_int64;
    if (index && n > ISO_ROWS8_SCAN) {
        a.to.owner = owner;
        hipLaunchKernelGGL(iso::row_claim_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, n, a.to);
        ISR_LAUNCH_CHECK("row_claim_kernel");
    }
    launch_codes(code, type, a, s);
    ISR_LAUNCH_CHECK("iso_rows8_write");
    return ISR_OK;
}

int iso_rows8_read(int type, int code, long long n, int F, int group, long long P, const void* codes, const float* scales, long long first,
                   const void* index, int index_is_int64, int normalize, float eps, void* out, void* stream) {
    if (const int e = check_rows("rows8_read", type, n, F)) return e;
    hipStream_t s = (hipStream_t)stream;
    if (!code_type(code)) return fail(ISR_EINVAL, "rows8_read: code %d is neither 1 (int8) nor 2 (e4m3)", code);
    if (!group_ok(F, group)) return fail(ISR_EINVAL, "rows8_read: groups of %d columns do not fit rows of %d", group, F);
    if (P < 0 || (!index && (first < 0 || first > P || n > P - first))) return fail(ISR_EINVAL, "rows8_read: rows [%lld, %lld) of a table of %lld", first, first + n, P);
    if (n == 0) return ISR_OK;
    if (!out || (P > 0 && (!codes || !scales))) return fail(ISR_EINVAL, "rows8_read: null pointer");
    iso::ReadArgs a = {};
    a.rows = n; a.P = P; a.first = first; a.F = F; a.groups = F / group; a.gshift = group_shift(F, group);
    a.norm = normalize; a.is64 = index_is_int64; a.eps = eps; a.codes = (const unsigned char*)codes; a.scales = scales; a.index = index; a.out = out;
    if (type == 0) launch_read_code<float>(code, a, s);
    else if (type == 1) launch_read_code<__bf16>(code, a, s);
    else launch_read_code<_Float16>(code, a, s);
    ISR_LAUNCH_CHECK("iso_rows8_read");
    return ISR_OK;
}

size_t iso_grad_norm_scratch_bytes(int count, const long long* sizes) {
    // one partial sum per workgroup, at most GN_PARTS of them for each GN_TENSORS tensors
    (void)sizes;
    return ((size_t)(std::max(count, 0) + iso::GN_TENSORS - 1) / iso::GN_TENSORS + 1) * iso::GN_PARTS * sizeof(double);
}

int iso_grad_norm(int count, void* const* tensors, const long long* sizes, const int* types, int norm_type, float max_norm, int clip,
                  float* out, void* scratch, size_t scratch_bytes, void* stream) {
    hipStream_t s = (hipStream_t)stream;
    if (count < 0 || (count > 0 && (!tensors || !sizes || !types)) || !out) return fail(ISR_EINVAL, "grad_norm: null argument");
    if (norm_type != 0 && norm_type != 1 && norm_type != 2) return fail(ISR_EINVAL, "grad_norm: norm type %d is none of 0 (maximum), 1, 2", norm_type);
    if (clip && !(max_norm >= 0.0f)) return fail(ISR_EINVAL, "grad_norm: max_norm must not be negative");
    if (!scratch || scratch_bytes < iso_grad_norm_scratch_bytes(count, sizes)) return fail(ISR_EINVAL, "grad_norm: scratch too small");
    for (int i = 0; i < count; i++) {
        if (sizes[i] < 0 || !row_type(types[i])) return fail(ISR_EINVAL, "grad_norm: tensor %d has size %lld, type %d", i, sizes[i], types[i]);
        if (sizes[i] > 0 && !tensors[i]) return fail(ISR_EINVAL, "grad_norm: tensor %d is null", i);
    }
    if (clip) {             // scaled in place: no element may belong to two of the tensors
        struct Span { uintptr_t from, to; };
        Span few[64];
        Span* span = count <= 64 ? few : (Span*)malloc((size_t)count * sizeof(Span));
        if (!span) return fail(ISR_EINVAL, "grad_norm: out of host memory");
        int n = 0;
        for (int i = 0; i < count; i++)
            if (sizes[i] > 0) span[n++] = {(uintptr_t)tensors[i], (uintptr_t)tensors[i] + (uintptr_t)sizes[i] * type_bytes(types[i])};
        std::sort(span, span + n, [](const Span& a, const Span& b) { return a.from < b.from; });
        bool overlap = false;
        for (int i = 1; i < n; i++) overlap |= span[i].from < span[i - 1].to;
        if (span != few) free(span);
        if (overlap) return fail(ISR_EINVAL, "grad_norm: two of the tensors to be clipped share memory");
    }
    double* part = (double*)scratch;
    int parts = 0, filled = 0;
    long long total = 0;
    for (int i = 0; i < count; i++) {
        filled += sizes[i] > 0;
        total = std::min(total + sizes[i], 1ll << 40);
    }
    const bool small = filled <= 16 && total <= iso::GN_SMALL;       // one workgroup, one launch
    for (int pass = 0; pass < (clip ? 2 : 1); pass++) {
        bool launched = false;
        for (int i = 0; i < count;) {
            iso::GradTable tb;
            unsigned long long chunks = 0;
            tb.count = 0;
            for (; i < count && tb.count < iso::GN_TENSORS; i++) {
                if (sizes[i] == 0) continue;
                const int size = type_bytes(types[i]);
                const long long head = std::min<long long>((16 - ((uintptr_t)tensors[i] & 15)) % 16 / size, sizes[i]);
                const unsigned long long c = std::max<unsigned long long>(1, ((unsigned long long)(sizes[i] - head) + iso::GN_CHUNK - 1) / iso::GN_CHUNK);
                tb.head[tb.count] = (unsigned char)head;
                if (chunks + c > 0xffffffffull) return fail(ISR_EINVAL, "grad_norm: too many elements");
                tb.p[tb.count] = tensors[i]; tb.n[tb.count] = sizes[i]; tb.type[tb.count] = (unsigned char)types[i];
                tb.first[tb.count++] = (unsigned)chunks;
                chunks += c;
            }
            if (tb.count == 0) break;
            tb.first[tb.count] = (unsigned)chunks;
            launched = true;
            if (small) {
                if (norm_type == 2) hipLaunchKernelGGL(iso::grad_small_kernel<2>, dim3(1), dim3(1024), 0, s, tb, clip, max_norm, out);
                else if (norm_type == 1) hipLaunchKernelGGL(iso::grad_small_kernel<1>, dim3(1), dim3(1024), 0, s, tb, clip, max_norm, out);
                else hipLaunchKernelGGL(iso::grad_small_kernel<0>, dim3(1), dim3(1024), 0, s, tb, clip, max_norm, out);
                ISR_LAUNCH_CHECK("iso_grad_norm");
                return ISR_OK;
            }
            if (pass == 0) {
                const int grid = (int)std::min<unsigned long long>(chunks, iso::GN_PARTS);
                if (norm_type == 2) hipLaunchKernelGGL(iso::grad_norm_kernel<2>, dim3(grid), dim3(iso::GN_THREADS), 0, s, tb, part + parts);
                else if (norm_type == 1) hipLaunchKernelGGL(iso::grad_norm_kernel<1>, dim3(grid), dim3(iso::GN_THREADS), 0, s, tb, part + parts);
                else hipLaunchKernelGGL(iso::grad_norm_kernel<0>, dim3(grid), dim3(iso::GN_THREADS), 0, s, tb, part + parts);
                parts += grid;
            } else {
                const int grid = (int)std::min<unsigned long long>(chunks, 1024);
                if (norm_type == 2) hipLaunchKernelGGL(iso::grad_clip_kernel<2>, dim3(grid), dim3(iso::GN_THREADS), 0, s, tb, part, parts, max_norm, out);
                else if (norm_type == 1) hipLaunchKernelGGL(iso::grad_clip_kernel<1>, dim3(grid), dim3(iso::GN_THREADS), 0, s, tb, part, parts, max_norm, out);
                else hipLaunchKernelGGL(iso::grad_clip_kernel<0>, dim3(grid), dim3(iso::GN_THREADS), 0, s, tb, part, parts, max_norm, out);
            }
            ISR_LAUNCH_CHECK("iso_grad_norm");
        }
        if (pass == 0 && (!clip || !launched)) {
            if (norm_type == 2) hipLaunchKernelGGL(iso::grad_norm_finish_kernel<2>, dim3(1), dim3(iso::GN_THREADS), 0, s, part, parts, max_norm, out);
            else if (norm_type == 1) hipLaunchKernelGGL(iso::grad_norm_finish_kernel<1>, dim3(1), dim3(iso::GN_THREADS), 0, s, part, parts, max_norm, out);
            else hipLaunchKernelGGL(iso::grad_norm_finish_kernel<0>, dim3(1), dim3(iso::GN_THREADS), 0, s, part, parts, max_norm, out);
            ISR_LAUNCH_CHECK("iso_grad_norm");
            break;
        }
    }
    return ISR_OK;
}

int iso_gaussian_grad_norm(int P, int M, float* const params[6], const float* g_xyz, const float* g_shs, const float* g_opacity,
                           const float* g_scale, const float* g_rotation, float max_norm, float* out, void* scratch, size_t scratch_bytes,
                           void* stream) {
    hipStream_t s = (hipStream_t)stream;
    if (P < 0 || M < 1 || M > 64) return fail(ISR_EINVAL, "gaussian_grad_norm: bad sizes P=%d M=%d", P, M);
    if (!params || !out || !(max_norm >= 0.0f)) return fail(ISR_EINVAL, "gaussian_grad_norm: null argument, or max_norm negative");
    if (!scratch || scratch_bytes < iso_grad_norm_scratch_bytes(1, nullptr)) return fail(ISR_EINVAL, "gaussian_grad_norm: scratch too small");
    if (P > 0 && ((g_opacity && !params[3]) || (g_scale && !params[4]) || (g_rotation && !params[5]))) return fail(ISR_EINVAL, "gaussian_grad_norm: a gradient without its parameter");
    double* part = (double*)scratch;
    int parts = 0;
    if (P > 0) {
        iso::GaussNormArgs a = {P, 3ll * M * P, g_xyz, g_shs, g_opacity, g_scale, g_rotation, params[3], params[4], params[5]};
        parts = (int)std::min<long long>(iso::GN_PARTS, std::max<long long>(1, (3ll * M * P / 4 + iso::GN_THREADS - 1) / iso::GN_THREADS));
        hipLaunchKernelGGL(iso::gaussian_norm_kernel, dim3(parts), dim3(iso::GN_THREADS), 0, s, a, part);
        ISR_LAUNCH_CHECK("iso_gaussian_grad_norm");
    }
    hipLaunchKernelGGL(iso::grad_norm_finish_kernel<2>, dim3(1), dim3(iso::GN_THREADS), 0, s, part, parts, max_norm, out);
    ISR_LAUNCH_CHECK("iso_gaussian_grad_norm");
    return ISR_OK;
}

}  // extern "C"
