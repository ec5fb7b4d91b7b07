// mx_quantise.hip -- rows of 16- or 32-bit values to MX blocks and back, and the root-mean-square
// norm that ends in MX blocks.
//
// A lane holds 8 consecutive values (one 16-byte load of a 16-bit type), so 4 lanes hold a block:
// its largest magnitude is two DPP steps away, and no value passes through LDS.  All kernels here
// are one pass over their data, bound by HBM: 8192 x 8192 bfloat16 to FP4 (170 MB) in 36 us, 4.7 TB/s;
// the norm of 16384 x 8192 with residual (943 MB) in 195 us a call among others, 4.8 TB/s (traced
// alone 198 to 210).  A copy of such size reaches 4.7 to 5.3.
#include "internal.hpp"
#include "mx.hpp"

#include "../../include/vcsrmc.h"

namespace vcsrmc {
namespace {

constexpr int kQuantThreads = 256;

// Stores the codes and scale of unit u (8 values) of a row.  The four lanes of a block call this
// together; units at or past the row's padded codes only write scale padding.
__device__ __forceinline__ void put_unit(unsigned char* codes, unsigned char* scales, int u,
                                         int code_units, int scale_units, const float (&v)[8],
                                         int fmt) {
    const int e = mx_scale_of(max_of_quad(absmax8(v)), fmt);
    if (u < code_units) {
        const uint2 c = mx_codes8(v, e, fmt);
        if (fmt == kMxFp8) *(uint2*)(codes + 8ll * u) = c;
        else *(unsigned*)(codes + 4ll * u) = c.x;
    }
    if ((u & 3) == 0 && u < scale_units) scales[u >> 2] = (unsigned char)e;
}

// One thread a unit; units of all rows in one flat order, so short rows share a work-group.
template <typename T>
__global__ void k_mx_quantise(const typename T::Raw* x, long long rows, int cols, long long ldx,
                              bool vec, int fmt, unsigned char* codes, unsigned char* scales) {
    const int code_units = (int)(mx_padded(cols) / 8), scale_units = (int)mx_scale_bytes(cols) * 4;
    const long long first = group_index() * kQuantThreads;
    const long long row0 = first / scale_units;
    const unsigned in = (unsigned)(first - row0 * scale_units) + threadIdx.x;
    const long long row = row0 + in / (unsigned)scale_units;
    const int u = (int)(in % (unsigned)scale_units);
    if (row >= rows) return;  // whole blocks leave together: a row has a multiple of 64 units
    float v[8];
    load8<T>(x + row * ldx + 8ll * u, vec, cols - 8 * u, v);
    put_unit(codes + row * mx_code_bytes(cols, fmt), scales + row * mx_scale_bytes(cols), u,
             code_units, scale_units, v, fmt);
}

template <typename T>
__global__ void k_mx_dequantise(const unsigned char* codes, const unsigned char* scales,
                                long long rows, int cols, int fmt, typename T::Raw* out,
                                long long ldo, bool vec) {
    const int units = (cols + 7) / 8;
    const long long first = group_index() * kQuantThreads;
    const long long row0 = first / units;
    const unsigned in = (unsigned)(first - row0 * units) + threadIdx.x;
    const long long row = row0 + in / (unsigned)units;
    const int u = (int)(in % (unsigned)units);
    if (row >= rows) return;
    const int e = scales[row * mx_scale_bytes(cols) + (u >> 2)];
    const float s = e == 255 ? __uint_as_float(0x7fc00000u) : mx_scale_value(e);
    const unsigned char* p = codes + row * mx_code_bytes(cols, fmt);
    float v[8];
    if (fmt == kMxFp8) {
        const uint2 c = *(const uint2*)(p + 8ll * u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned w = i < 2 ? c.x : c.y;
            const mx_v2f d = (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.f, true)
                                     : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.f, false);
            v[2 * i] = d[0] * s;
            v[2 * i + 1] = d[1] * s;
        }
    } else {
        const unsigned w = *(const unsigned*)(p + 4ll * u);
        mx_v2f d[4];
        d[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0);
        d[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
        d[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2);
        d[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = d[i / 2][i & 1] * s;
    }
    store8<T>(out + row * ldo + 8ll * u, vec, cols - 8 * u, v);
}

// ---- root-mean-square norm --------------------------------------------------------------------
// h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight, then MX blocks of y.  One work-group a
// row, h in registers between the sum and the output, so x and the residual are read once and the
// statistic costs one barrier.  The norm is of the unrounded 32-bit h: rounding h to its type is
// for the copy that is written alone.  Everything after h is in 64 bits, whose vector rate is that of
// 32 bits: y then reaches its 8 or 4 bits with one rounding, where a y in 32 bits falls on the wrong
// side of a rounding boundary a few times in a million.
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Sum over the work-group; every thread gets it.
__device__ __forceinline__ double group_sum(double v, double* part) {
    v = wave_sum(v);
    const int waves = blockDim.x / kWave;
    if (waves == 1) return v;
    if (lane_id() == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    double s = 0;
    for (int w = 0; w < waves; ++w) s += part[w];
    return s;
}

template <typename T>
__device__ __forceinline__ void load_h(const RmsNormArgs& a, long long row, int u, bool vec,
                                       float (&h)[8]) {
    const int n = (int)a.cols - 8 * u;
    load8<T>((const typename T::Raw*)a.x + row * a.ldx + 8ll * u, vec, n, h);
    if (a.residual) {
        float r[8];
        load8<T>((const typename T::Raw*)a.residual + row * a.ldr + 8ll * u, vec, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
}

// v in 32 bits such that rounding the result to fewer bits is rounding v: the nearest number, or,
// where that is even and not v, its neighbour on v's side.  (Boundaries of shorter formats are even.)
// What rounds past the largest 32-bit number stays an infinity, which makes its block NaN: its
// neighbour would be a finite value far below v.
__device__ __forceinline__ float round_to_odd(double v) {
    const float f = (float)v;
    const double d = v - (double)f;  // not finite where f is not
    constexpr int kFiniteNonzero = 0x198;  // classes: normal and subnormal numbers of either sign
    const unsigned u = __float_as_uint(f);
    if ((u & 1) || !__builtin_amdgcn_class(d, kFiniteNonzero)) return f;
    return __uint_as_float((d > 0) == !(u >> 31) ? u + 1 : u - 1);
}

template <typename T, typename W>
__device__ __forceinline__ void norm_unit(const RmsNormArgs& a, long long row, int u, bool vec,
                                          bool wvec, double scale, float (&h)[8]) {
    float w[8];
    load8<W>((const typename W::Raw*)a.weight + 8ll * u, wvec, (int)a.cols - 8 * u, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = round_to_odd((double)h[i] * scale * (double)w[i]);
    put_unit(a.codes + row * mx_code_bytes(a.cols, a.fmt), a.scales + row * mx_scale_bytes(a.cols),
             u, (int)(mx_padded(a.cols) / 8), (int)mx_scale_bytes(a.cols) * 4, h, a.fmt);
}

__device__ __forceinline__ double norm_scale(double ss, const RmsNormArgs& a) {
    return 1.0 / sqrt(ss / (double)a.cols + (double)a.eps);
}

// V units a thread; the work-group covers the row's scale units (V * blockDim.x of them).
template <typename T, typename W, int V>
__global__ void __launch_bounds__(1024) k_rms_norm_mx(RmsNormArgs a, bool vec, bool wvec) {
    __shared__ double part[16];
    const long long row = group_index();
    if (row >= a.rows) return;
    float h[V][8];
    double ss = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int u = threadIdx.x + k * blockDim.x;
        load_h<T>(a, row, u, vec, h[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fma((double)h[k][i], (double)h[k][i], ss);
    }
    const double scale = norm_scale(group_sum(ss, part), a);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int u = threadIdx.x + k * blockDim.x;
        if (a.residual_out)
            store8<T>((typename T::Raw*)a.residual_out + row * a.ldro + 8ll * u, vec,
                      (int)a.cols - 8 * u, h[k]);
        norm_unit<T, W>(a, row, u, vec, wvec, scale, h[k]);
    }
}

// Rows too long for registers: h is formed twice.  The residual's copy is written in the second
// pass, so that it may take the place of x or of the residual.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) k_rms_norm_mx_long(RmsNormArgs a, bool vec, bool wvec) {
    __shared__ double part[16];
    const long long row = group_index();
    if (row >= a.rows) return;
    const int units = (int)mx_scale_bytes(a.cols) * 4;
    double ss = 0;
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
        float h[8];
        load_h<T>(a, row, u, vec, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fma((double)h[i], (double)h[i], ss);
    }
    const double scale = norm_scale(group_sum(ss, part), a);
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
        float h[8];
        load_h<T>(a, row, u, vec, h);
        if (a.residual_out)
            store8<T>((typename T::Raw*)a.residual_out + row * a.ldro + 8ll * u, vec,
                      (int)a.cols - 8 * u, h);
        norm_unit<T, W>(a, row, u, vec, wvec, scale, h);
    }
}

bool aligned16(const void* p, long long ld, int size) {
    return ((uintptr_t)p | (uintptr_t)(ld * size)) % 16 == 0;
}

int size_of(int type) { return type == kTypeF32 ? 4 : 2; }

template <typename T, typename W>
void launch_norm(const RmsNormArgs& a, hipStream_t st) {
    const int size = sizeof(typename T::Raw);
    const bool vec = aligned16(a.x, a.ldx, size) &&
                     (!a.residual || aligned16(a.residual, a.ldr, size)) &&
                     (!a.residual_out || aligned16(a.residual_out, a.ldro, size));
    const bool wvec = aligned16(a.weight, 0, sizeof(typename W::Raw));
    const dim3 grid = grid_of(a.rows);
    const long long units = mx_scale_bytes(a.cols) * 4;  // a multiple of 64
    // Units a thread, kernels traced alone: 16384 rows of 8192 bfloat16 take 205 us with 2, 238 with 1
    // (fewer rows on a CU at once) and 232 with 4; 256 rows 7.1, 7.2 and 9.0 us.
    auto threads = [&](int v) { return (int)((units / v + 63) / 64 * 64); };
    if (units < 512) k_rms_norm_mx<T, W, 1><<<grid, threads(1), 0, st>>>(a, vec, wvec);
    else if (units <= 2048) k_rms_norm_mx<T, W, 2><<<grid, threads(2), 0, st>>>(a, vec, wvec);
    else if (units <= 4096) k_rms_norm_mx<T, W, 4><<<grid, threads(4), 0, st>>>(a, vec, wvec);
    else k_rms_norm_mx_long<T, W><<<grid, 1024, 0, st>>>(a, vec, wvec);
    VCSRMC_HIP(hipGetLastError());
}

template <typename Fn>
void by_type(int type, Fn&& fn) {
    if (type == kTypeF32) fn(F32{});
    else if (type == kTypeF16) fn(F16{});
    else fn(BF16{});
}

}  // namespace

void mx_quantise(const void* x, int type, long long rows, long long cols, long long ldx, int fmt,
                 unsigned char* codes, unsigned char* scales, hipStream_t st) {
    if (rows == 0) return;
    const long long units = rows * mx_scale_bytes(cols) * 4;
    const dim3 grid = grid_of((units + kQuantThreads - 1) / kQuantThreads);
    const bool vec = aligned16(x, ldx, size_of(type));
    by_type(type, [&](auto t) {
        using T = decltype(t);
        k_mx_quantise<T><<<grid, kQuantThreads, 0, st>>>((const typename T::Raw*)x, rows, (int)cols,
                                                         ldx, vec, fmt, codes, scales);
    });
    VCSRMC_HIP(hipGetLastError());
}

void mx_dequantise(const MxOperand& q, void* out, int type, long long ldo, hipStream_t st) {
    if (q.rows == 0) return;
    const long long units = q.rows * ((q.cols + 7) / 8);
    const dim3 grid = grid_of((units + kQuantThreads - 1) / kQuantThreads);
    const bool vec = aligned16(out, ldo, size_of(type));
    by_type(type, [&](auto t) {
        using T = decltype(t);
        k_mx_dequantise<T><<<grid, kQuantThreads, 0, st>>>(q.codes, q.scales, q.rows, (int)q.cols,
                                                           q.fmt, (typename T::Raw*)out, ldo, vec);
    });
    VCSRMC_HIP(hipGetLastError());
}

void rms_norm_mx(const RmsNormArgs& a, hipStream_t st) {
    if (a.rows == 0) return;
    if (a.type == kTypeF32) launch_norm<F32, F32>(a, st);
    else if (a.type == kTypeF16 && a.weight_type == kTypeF32) launch_norm<F16, F32>(a, st);
    else if (a.type == kTypeF16) launch_norm<F16, F16>(a, st);
    else if (a.weight_type == kTypeF32) launch_norm<BF16, F32>(a, st);
    else launch_norm<BF16, BF16>(a, st);
}

}  // namespace vcsrmc
