// mx.hpp -- the microscaled (MX) formats on gfx950: layout, conversions, matrix steps.
//
// A row of `cols` values is cut into blocks of 32 along the row; a block holds 32 codes and one
// scale byte e, which stands for 2^(e - 127) (255: NaN).  Codes are E4M3 bytes (FP8) or E2M1
// nibbles (FP4, even element in the low nibble).  A row's codes are padded with zeros to a
// multiple of 128 values (one matrix step) and its scales to a multiple of 16 bytes (four
// steps), so no kernel below checks a bound along a row: codes of padding are zero, and scales
// past the padded codes are loaded with their 16 bytes but never used.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "hip_common.hpp"

namespace vcsrmc {

enum : int { kMxFp4 = 4, kMxFp8 = 8 };                // bits of a code
enum : int { kTypeF32 = 0, kTypeF16 = 1, kTypeBf16 = 2 };

constexpr int kMxBlock = 32;
constexpr int kMxStep = 128;   // values of a row in one 16x16x128 matrix instruction

__host__ __device__ inline long long mx_padded(long long cols) { return (cols + 127) / 128 * 128; }
__host__ __device__ inline long long mx_code_bytes(long long cols, int fmt) {
    return mx_padded(cols) * fmt / 8;
}
__host__ __device__ inline long long mx_scale_bytes(long long cols) {
    return (cols + 511) / 512 * 16;
}

typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef float mx_v4f __attribute__((ext_vector_type(4)));
typedef float mx_v2f __attribute__((ext_vector_type(2)));
typedef short mx_v2s __attribute__((ext_vector_type(2)));

// ---- element types --------------------------------------------------------------------------
struct F32 {
    using Raw = float;
    static __device__ __forceinline__ float get(Raw v) { return v; }
    static __device__ __forceinline__ Raw put(float v) { return v; }
};
struct F16 {
    using Raw = _Float16;
    static __device__ __forceinline__ float get(Raw v) { return (float)v; }
    static __device__ __forceinline__ Raw put(float v) { return (_Float16)v; }
};
struct BF16 {
    using Raw = __bf16;
    static __device__ __forceinline__ float get(Raw v) { return (float)v; }
    static __device__ __forceinline__ Raw put(float v) { return (__bf16)v; }
};

// Eight consecutive values; `vec` says that p is 16-byte aligned, `n` how many of them exist.
template <typename T>
__device__ __forceinline__ void load8(const typename T::Raw* p, bool vec, int n, float (&v)[8]) {
    using Raw = typename T::Raw;
    if (vec && n >= 8) {
        constexpr int kPer = 16 / sizeof(Raw);
        Raw raw[8];
#pragma unroll
        for (int i = 0; i < 8; i += kPer) *(uint4*)(raw + i) = *(const uint4*)(p + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = T::get(raw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? T::get(p[i]) : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(typename T::Raw* p, bool vec, int n, const float (&v)[8]) {
    using Raw = typename T::Raw;
    if (vec && n >= 8) {
        constexpr int kPer = 16 / sizeof(Raw);
        Raw raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = T::put(v[i]);
#pragma unroll
        for (int i = 0; i < 8; i += kPer) *(uint4*)(p + i) = *(const uint4*)(raw + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = T::put(v[i]);
    }
}

// ---- quantisation ---------------------------------------------------------------------------
// Biased exponent of a block's scale from the bits of its largest magnitude: the format's largest
// binade (2^8 for E4M3, 2^2 for E2M1) is put at the block's.  Values above the format's largest
// number inside that binade saturate, which is what the formats' standard does.  255 where the
// block holds an infinity or a NaN (as integers their magnitudes exceed every finite one).
__device__ __forceinline__ int mx_scale_of(unsigned amax_bits, int fmt) {
    const int field = (int)(amax_bits >> 23);
    const int e = field - (fmt == kMxFp8 ? 8 : 2);
    return field == 255 ? 255 : (e < 0 ? 0 : e);
}

__device__ __forceinline__ float mx_scale_value(int e) {  // e < 255
    return __uint_as_float(e ? (unsigned)e << 23 : 0x00400000u);
}

// Eight codes under scale byte e: 8 bytes (FP8) or the low 4 (FP4).  The conversion instructions
// divide by the scale exactly and round to nearest even; the FP8 one makes NaN of what rounds past
// 448, so values are cut to it first.
__device__ __forceinline__ uint2 mx_codes8(const float (&v)[8], int e, int fmt) {
    uint2 out = make_uint2(0u, 0u);
    if (e == 255) return out;
    const float s = mx_scale_value(e);
    if (fmt == kMxFp8) {
        const float top = 448.f * s;
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_fmed3f(v[i], -top, top);
        mx_v2s lo = {0, 0}, hi = {0, 0};
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, c[0], c[1], s, false);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, c[2], c[3], s, true);
        hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, c[4], c[5], s, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, c[6], c[7], s, true);
        out.x = __builtin_bit_cast(unsigned, lo);
        out.y = __builtin_bit_cast(unsigned, hi);
    } else {
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
        out.x = w;
    }
    return out;
}

// Largest magnitude of eight values, as bits (so that a NaN is larger than all else).
__device__ __forceinline__ unsigned absmax8(const float (&v)[8]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}

// Maximum over each aligned group of four lanes (DPP quad_perm).
__device__ __forceinline__ unsigned max_of_quad(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));
    return m;
}

// ---- matrix steps ---------------------------------------------------------------------------
// v_mfma_scale_f32_16x16x128_f8f6f4: A is 16 weight rows in FP4, B 16 tokens in FP8 or FP4, and
// lane (n = lane % 16, q = lane / 16) gives for its row or token
//   FP4: values 32 q .. 32 q + 31 of the 128 (16 bytes);
//   FP8: values 16 q .. 16 q + 15 and 64 + 16 q .. 64 + 16 q + 15 (twice 16 bytes);
//   the scale byte of values 32 q .. 32 q + 31;
// and holds rows 4 q .. 4 q + 3 of token n of the result.
template <int FX> struct MxFrag {
    uint4 lo, hi;
    __device__ __forceinline__ void load(const unsigned char* p) {  // p: this lane's, at the step
        lo = *(const uint4*)p;
        if constexpr (FX == kMxFp8) hi = *(const uint4*)(p + 64);
    }
    __device__ __forceinline__ mx_v8i reg() const {
        if constexpr (FX == kMxFp8)
            return mx_v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w,
                          (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
        else
            return mx_v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, 0, 0, 0, 0};
    }
};

template <int FX>
__device__ __forceinline__ mx_v4f mx_step(const MxFrag<kMxFp4>& w, int ws, const MxFrag<FX>& x,
                                          int xs, mx_v4f acc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.reg(), x.reg(), acc, 4,
                                                            FX == kMxFp8 ? 0 : 4, 0, ws, 0, xs);
}

__device__ __forceinline__ unsigned word_of(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Bytes of a step's codes in a row.
template <int FX> constexpr int kMxStepBytes = FX == kMxFp8 ? 128 : 64;

// ---- matrix steps with nothing lost -----------------------------------------------------------
// The same products through bfloat16 on v_mfma_f32_16x16x32_bf16: products exact, sums in 32 bits,
// where the FP8 path cuts the smaller products of 8 neighbours (2^-13 of the largest).  bfloat16 holds
// every value of FP8 under scale bytes 3 to 246 and of FP4 under 0 to 252; quantisation writes none
// above these.  Under 0 to 2 FP8 values lose what lies below 2^-133 (the least are 2^-136); above 246
// and 252 values past 2^128 become infinities, where the scaled instructions go on.  For sums that are rounded to 8 bits again:
// there the cut moves values across rounding boundaries, a step of 2^-4 each.  The conversions
// cost 16 vector instructions per operand and step, hidden where the weights come from memory.
// Lane (n, q) holds block q of the step on both sides; instruction j takes its values 8 j .. + 7.
typedef __bf16 mx_v2b __attribute__((ext_vector_type(2)));
typedef __bf16 mx_v8b __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float mx_scale_or_nan(unsigned e) {
    return e == 255 ? __uint_as_float(0x7fc00000u) : mx_scale_value((int)e);
}

// Values 8 j .. 8 j + 7 of a block in FP4 (word j of its 16 bytes).
__device__ __forceinline__ mx_v8b mx_bf16_of_fp4(unsigned w, float s) {
    const mx_v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0);
    const mx_v2b b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
    const mx_v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2);
    const mx_v2b d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
    return mx_v8b{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The same of a block in FP8 (two words of its 32 bytes).
__device__ __forceinline__ mx_v8b mx_bf16_of_fp8(unsigned lo, unsigned hi, float s) {
    const mx_v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
    const mx_v2b b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    const mx_v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
    const mx_v2b d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return mx_v8b{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---- weights from memory through LDS ------------------------------------------------------------
// 16 bytes a lane from `base` (the same for all) + the lane's offset to LDS, at `to` + 16 * lane.  The
// copy has no register to wait for, and its reader waits with wait_copies or arrive_but.  It is not
// the builtin, because the compiler then adds waits of its own before reads of LDS, and with more
// than a few arrays these wait for every copy on its way.  Waits that it adds for other loads count
// these copies too, which only makes them longer.  m0 carries the LDS address, one instruction ahead
// of its use; it is named as written, so that no use of the compiler's own of m0 is torn apart (the
// warning is that the compiler would not save a reserved register, of which it never keeps a value).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16_to_lds(const unsigned char* base, unsigned offset,
                                              unsigned char* to) {
    const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)to;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset),
                 "s"(base)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// Where chunks of 16 bytes of a row lie in LDS: chunk c of row r at place c ^ place(r) of its row, so
// that the 16 lanes that read together (rows 0-3, 12-15, 20-23, 24-27 and the like, or 0-15) touch all
// 64 banks: rows of 64 bytes fill them four at a time, of 128 two, longer ones alone.
template <int ROW> __device__ __forceinline__ int place(int row) {
    static_assert(ROW == 64 || ROW == 128 || ROW % 256 == 0, "rows of 4 or 8 chunks, or of whole 16");
    return ROW == 64 ? row >> 2 & 3 : ROW == 128 ? row >> 1 & 7 : row & 15;
}

// Waits until at most N of this wave's copies are on their way, then for the other waves.  (The
// fence of __syncthreads would wait for all of them.)
template <int N> __device__ __forceinline__ void arrive_but() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The same where this wave's reads of LDS need no wait: their values have been used.
template <int N> __device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A product of few tokens, bound by reading the weights: a work-group of WR x WK waves has 16 WR weight
// rows and TOK tokens and goes along the rows in stages of 128 SPS WK values, NS of them in LDS, wave
// (r, k) multiplying the k-th 128 SPS of each with row tile r.  Why through LDS: a matrix instruction's
// operand is 16 rows by 64 bytes, and loaded straight to registers it took the address path 92 cycles,
// 79% of a kernel that did so.  Copies to LDS take whole lines of a row, and stages on their way take
// no registers.  What it reaches: 5.1 to 5.2 TB/s where the weights are 285 MB and more, 3.7 for 36 MB
// in one launch.
//
// Rows and tokens past the end are copies of the last; past the end of a row its last chunk is
// repeated, and its steps are not multiplied.  Lanes of a tile's 16 tokens past TOK read the last
// one's row too.
template <int FX_, int WR_, int WK_, int TOK_, int SPS_, int NS_> struct MxStream {
    static constexpr int FX = FX_, WR = WR_, WK = WK_, TOK = TOK_, SPS = SPS_, NS = NS_;
    static constexpr int W = WR * WK, R = 16 * WR, MT = (TOK + 15) / 16;
    static constexpr int kRowW = 64 * SPS * WK, kRowX = 16 * FX * SPS * WK;
    static constexpr int P = (SPS * WK + 3) / 4;  // 16-byte pieces of a row's scales in a stage
    static constexpr int kShare = P * 4 / (SPS * WK);  // stages that share them
    static_assert(SPS * WK % 4 == 0 || 4 % (SPS * WK) == 0, "a stage in one piece, or whole ones");
    static constexpr int kBytesW = R * kRowW, kAllX = (TOK * kRowX + 1023) / 1024;  // copies of X
    static constexpr int kStage = kBytesW + 1024 * kAllX;
    static constexpr int kScaleCallsW = (R * P * 16 + 1023) / 1024,
                         kScaleCalls = kScaleCallsW + (TOK * P * 16 + 1023) / 1024;
    static constexpr int kScales = 1024 * kScaleCalls, kSlots = kShare > 1 ? 2 : NS;
    static constexpr int kLds = NS * kStage + kSlots * kScales;
    static constexpr int kCallsW = kBytesW / 1024 / W, kCallsX = (kAllX + W - 1) / W;
    static_assert(kBytesW % (1024 * W) == 0, "whole copies a wave");
    static_assert(kScaleCalls <= W, "at most one copy of scales a wave");
    // Copies of a wave and stage.  With more than two stages, waits count those of later ones, so
    // waves that have none left make the last one again.
    static constexpr int kCalls = kCallsW + kCallsX + 1;
    static constexpr bool kEven = NS > 2;
    static_assert(NS >= 2 && (NS - 2) * kCalls < 64 && (kShare == 1 || NS <= 3), "a wait's count; slots");

    const unsigned char *w, *x, *s;  // codes of W and X, this wave's scales
    unsigned row_w[kCallsW], row_x[kCallsX], row_s;
    int chunk_w[kCallsW], chunk_x[kCallsX], chunk_s, last_w, last_x, last_s;
    int wave, lane;

    // row_of(r): offset in rows of tile row r from `w0`; token_of(m): of token m from `x0`.
    template <typename RowOf, typename TokenOf>
    __device__ __forceinline__ void init(const unsigned char* w0, const unsigned char* ws0,
                                         const unsigned char* x0, const unsigned char* xs0,
                                         long long cols, int wave_, RowOf row_of, TokenOf token_of) {
        wave = wave_;
        lane = lane_id();
        w = w0;
        x = x0;
        const unsigned wb = (unsigned)mx_code_bytes(cols, kMxFp4), xb = (unsigned)mx_code_bytes(cols, FX),
                       sb = (unsigned)mx_scale_bytes(cols);
        last_w = (int)wb / 16 - 1;
        last_x = (int)xb / 16 - 1;
        last_s = (int)sb / 16 - 1;
#pragma unroll
        for (int i = 0; i < kCallsW; ++i) {
            const int slot = (wave * kCallsW + i) * 64 + lane, r = slot / (kRowW / 16);
            row_w[i] = row_of(r) * wb;
            chunk_w[i] = slot % (kRowW / 16) ^ place<kRowW>(r);
        }
#pragma unroll
        for (int i = 0; i < kCallsX; ++i) {
            const int slot = call_x(i) * 64 + lane, r = min(slot / (kRowX / 16), TOK - 1);
            row_x[i] = token_of(r) * xb;
            chunk_x[i] = slot % (kRowX / 16) ^ place<kRowX>(r);
        }
        const int call = min(wave, kScaleCalls - 1);
        const bool of_w = call < kScaleCallsW;
        const int slot = (call - (of_w ? 0 : kScaleCallsW)) * 64 + lane, r = slot / P;
        s = of_w ? ws0 : xs0;
        row_s = (of_w ? row_of(min(r, R - 1)) : token_of(min(r, TOK - 1))) * sb;
        chunk_s = slot % P;
    }

    __device__ __forceinline__ int call_x(int i) const { return min(wave * kCallsX + i, kAllX - 1); }

    // Sends for stage t, to place t % NS; past the end for the last one again.
    __device__ __forceinline__ void issue(unsigned char* lds, int t, int place, int stages) const {
        const int from = min(t, stages - 1);
        unsigned char* to = lds + place * kStage;
#pragma unroll
        for (int i = 0; i < kCallsW; ++i)
            copy16_to_lds(w, row_w[i] + 16 * min(chunk_w[i] + from * (kRowW / 16), last_w),
                          to + (wave * kCallsW + i) * 1024);
#pragma unroll
        for (int i = 0; i < kCallsX; ++i)
            if (kEven || wave * kCallsX + i < kAllX)
                copy16_to_lds(x, row_x[i] + 16 * min(chunk_x[i] + from * (kRowX / 16), last_x),
                              to + kBytesW + call_x(i) * 1024);
        if (kEven || (wave < kScaleCalls && t % kShare == 0))
            copy16_to_lds(s, row_s + 16 * min(chunk_s + SPS * WK * from / 4, last_s),
                          scales(lds, t, place) + min(wave, kScaleCalls - 1) * 1024);
    }
    static __device__ __forceinline__ unsigned char* scales(unsigned char* lds, int t, int place) {
        return lds + NS * kStage + (kShare > 1 ? t / kShare & 1 : place) * kScales;
    }

    __device__ __forceinline__ int row_tile() const { return wave % WR; }
    __device__ __forceinline__ int part() const { return wave / WR; }

    template <int ROW>
    static __device__ __forceinline__ uint4 chunk(const unsigned char* rows, int row, int c) {
        return *(const uint4*)(rows + row * ROW + 16 * (c ^ place<ROW>(row)));
    }

    // Step s of this wave's part of a stage; even and odd steps have sums of their own, or the
    // matrix instructions of one token tile would all wait for each other.
    template <bool EXACT>
    __device__ __forceinline__ void step(mx_v4f (&acc)[2][MT], const unsigned char* lds, int s,
                                         const unsigned (&sw)[SPS], const unsigned (&sx)[MT][SPS]) const {
        const int r16 = lane & 15, q = lane >> 4, k = part(), row = 16 * row_tile() + r16;
        const unsigned char* xl = lds + kBytesW;
        const uint4 a = chunk<kRowW>(lds, row, 4 * (SPS * k + s) + q);
        const unsigned es = sw[s] >> (8 * q);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int tok = min(16 * m + r16, TOK - 1);
            const unsigned xe = sx[m][s] >> (8 * q);
            mx_v4f& sum = acc[s & 1][m];
            if constexpr (EXACT) {
                const int c = 8 * (SPS * k + s) + 2 * q;
                const uint4 lo = chunk<kRowX>(xl, tok, c), hi = chunk<kRowX>(xl, tok, c + 1);
                const float fw = mx_scale_or_nan(es & 255), fx = mx_scale_or_nan(xe & 255);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4& h = j < 2 ? lo : hi;
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        mx_bf16_of_fp4(word_of(a, j), fw),
                        mx_bf16_of_fp8(word_of(h, 2 * (j & 1)), word_of(h, 2 * (j & 1) + 1), fx), sum,
                        0, 0, 0);
                }
            } else {
                MxFrag<kMxFp4> fw;
                MxFrag<FX> fx;
                fw.lo = a;
                if constexpr (FX == kMxFp8) {
                    const int c = 8 * (SPS * k + s) + q;
                    fx.lo = chunk<kRowX>(xl, tok, c);
                    fx.hi = chunk<kRowX>(xl, tok, c + 4);
                } else {
                    fx.lo = chunk<kRowX>(xl, tok, 4 * (SPS * k + s) + q);
                }
                sum = mx_step<FX>(fw, es, fx, xe, sum);
            }
        }
    }

    // Adds this wave's part of stage t, of `steps` in all.
    template <bool EXACT>
    __device__ __forceinline__ void multiply(mx_v4f (&acc)[2][MT], unsigned char* lds, int t, int place,
                                             int steps) const {
        const int r16 = lane & 15, first = SPS * (WK * t + part()), n = steps - first;
        const unsigned char* stage = lds + place * kStage;
        const unsigned char* sc = scales(lds, t, place) + 4 * (first % (4 * P));
        unsigned sw[SPS], sx[MT][SPS];
#pragma unroll
        for (int s = 0; s < SPS; ++s)
            sw[s] = *(const unsigned*)(sc + (16 * row_tile() + r16) * (16 * P) + 4 * s);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int s = 0; s < SPS; ++s)
                sx[m][s] = *(const unsigned*)(sc + 1024 * kScaleCallsW +
                                              min(16 * m + r16, TOK - 1) * (16 * P) + 4 * s);
        if (n >= SPS) {
#pragma unroll
            for (int s = 0; s < SPS; ++s) step<EXACT>(acc, stage, s, sw, sx);
        } else {
#pragma unroll
            for (int s = 0; s < SPS - 1; ++s)
                if (s < n) step<EXACT>(acc, stage, s, sw, sx);
        }
    }

    // All of it, through kLds bytes.  Leaves no copy on its way, and the bytes free for all.
    template <bool EXACT>
    __device__ __forceinline__ void run(mx_v4f (&sum)[MT], unsigned char* lds, int steps) const {
        mx_v4f acc[2][MT] = {};
        const int stages = (steps + SPS * WK - 1) / (SPS * WK);
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) issue(lds, i, i, stages);
        for (int t = 0, now = 0; t < stages; ++t) {
            arrive_but<(NS - 2) * kCalls>();
            issue(lds, t + NS - 1, now ? now - 1 : NS - 1, stages);
            multiply<EXACT>(acc, lds, t, now, steps);
            now = now + 1 < NS ? now + 1 : 0;
        }
        arrive_but<0>();
#pragma unroll
        for (int m = 0; m < MT; ++m) sum[m] = acc[0][m] + acc[1][m];
    }
};

// ---- host entry points (checked by the C ABI) -------------------------------------------------
struct MxOperand {  // rows x cols values
    const unsigned char* codes;
    const unsigned char* scales;
    long long rows;
    long long cols;
    int fmt;
};

void mx_quantise(const void* x, int type, long long rows, long long cols, long long ldx, int fmt,
                 unsigned char* codes, unsigned char* scales, hipStream_t st);
void mx_dequantise(const MxOperand& q, void* out, int type, long long ldo, hipStream_t st);

struct RmsNormArgs {
    const void *x, *residual, *weight;
    void* residual_out;
    unsigned char *codes, *scales;
    long long rows, cols, ldx, ldr, ldro;
    int type, weight_type, fmt;
    float eps;
};
void rms_norm_mx(const RmsNormArgs& a, hipStream_t st);

void mx_matmul(const MxOperand& x, const MxOperand& w, void* out, int type, long long ldo,
               hipStream_t st);

constexpr int kMoeExperts = 1024, kMoeTopK = 64;  // most experts of a layer, and of a token

struct MoeArgs {
    MxOperand x;       // T x D, FP8
    const void* router;  // E x D
    int router_type;
    MxOperand w13;     // E 2F x D: gate rows, then up rows, of each expert
    MxOperand w2;      // E D x F
    int experts, top_k, renormalise;
    void* out;
    int type;
    long long ldo;
    void* workspace;
};
long long mx_moe_workspace(long long T, long long D, long long F, int experts, int top_k);
void mx_moe(const MoeArgs& a, hipStream_t st);

}  // namespace vcsrmc
