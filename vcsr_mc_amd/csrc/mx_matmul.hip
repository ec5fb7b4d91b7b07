// mx_matmul.hip -- Y = X.W^T with W in MXFP4 and X in MXFP8 or MXFP4, on gfx950's scaled matrix
// instructions: Y[m, n] = sum over blocks b of 2^(ex + ew - 254) * sum over i of X[m, i] W[n, i],
// products and block sums inside v_mfma_scale_f32_16x16x128_f8f6f4, sums of steps in FP32.
#include "internal.hpp"
#include "mx.hpp"

#include "../../include/vcsrmc.h"

namespace vcsrmc {
namespace {

// ---- few tokens -------------------------------------------------------------------------------
// Work-groups of 16 WR rows and 16 MT tokens as MxStream describes; the sums of the WK parts of a
// row tile meet in LDS, in order.
template <typename T, typename S>
__global__ void __launch_bounds__(64 * S::W)
k_mx_rows(MxOperand x, MxOperand wt, typename T::Raw* out, long long ldo) {
    __shared__ __attribute__((aligned(256))) unsigned char lds[S::kLds];
    const int lane = lane_id(), n = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const long long row0 = group_index() * S::R;
    if (row0 >= wt.rows) return;  // the whole work-group
    const int rows = (int)min(wt.rows - row0, (long long)S::R), tokens = (int)x.rows;
    S stream;
    stream.init(wt.codes + row0 * mx_code_bytes(x.cols, kMxFp4), wt.scales + row0 * mx_scale_bytes(x.cols),
                x.codes, x.scales, x.cols, wave, [&](int r) { return (unsigned)min(r, rows - 1); },
                [&](int m) { return (unsigned)min(m, tokens - 1); });
    mx_v4f acc[S::MT] = {};
    stream.template run<false>(acc, lds, (int)(mx_padded(x.cols) / kMxStep));
    mx_v4f(*const part)[S::MT][64] = (mx_v4f(*)[S::MT][64])lds;  // [k * WR + r]
    if constexpr (S::WK > 1) {
#pragma unroll
        for (int m = 0; m < S::MT; ++m) part[wave][m][lane] = acc[m];
        __syncthreads();
    }
    for (int t = wave; t < S::WR * S::MT; t += S::W) {
        const int r = S::WK > 1 ? t % S::WR : wave, m = t / S::WR;
        mx_v4f sum = {0, 0, 0, 0};
        if constexpr (S::WK > 1) {
            sum = part[r][m][lane];
#pragma unroll
            for (int k = 1; k < S::WK; ++k) sum += part[k * S::WR + r][m][lane];
        } else {
#pragma unroll
            for (int i = 0; i < S::MT; ++i) sum = i == m ? acc[i] : sum;
        }
        const int tok = 16 * m + n, row = 16 * r + 4 * q;
        if (tok >= tokens) continue;
        typename T::Raw* p = out + tok * ldo + row0 + row;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (row + i < rows) p[i] = T::put(sum[i]);
    }
}

template <typename T, typename S>
void launch_rows(const MxOperand& x, const MxOperand& w, void* out, long long ldo, hipStream_t st) {
    k_mx_rows<T, S><<<grid_of((w.rows + S::R - 1) / S::R), 64 * S::W, 0, st>>>(
        x, w, (typename T::Raw*)out, ldo);
    VCSRMC_HIP(hipGetLastError());
}

// As many rows a work-group as leave one for every CU, since each work-group reads all of X; waves and
// steps such that a stage brings 16 KB of weights (32 tokens: 8 KB, or X would not fit LDS three
// times).  Deeper rings changed nothing.  Times in us of 16, 32 and 64 rows a work-group, weights from
// memory, FP8, 1 token and 32:
//   4096 x 16384   9.5 15.7   12.6 19.7   17.5 27.1   (reading the weights at 6.25 TB/s: 5.7)
//   8192 x 8192   10.2 18.2    9.9 13.8   12.4 16.8   (5.7)
//   16384 x 8192  17.3 34.8   17.0 25.6   16.9 20.8   (11.4)
//   32768 x 4096  20.1 43.4   16.3 29.8   15.2 21.5   (11.4)
// About 3 us of each is the start and end of a launch.  32 tokens bring 4, 2 or 1 bytes of X into LDS for
// each of weights.
template <typename T, int FX, int TOK>
void rows_of(const MxOperand& x, const MxOperand& w, void* out, long long ldo, hipStream_t st) {
    constexpr int kCus = 256;
    constexpr bool kMany = TOK > 16;
    if (w.rows >= 64 * kCus)
        launch_rows<T, MxStream<FX, 4, kMany ? 2 : 1, TOK, 4, kMany ? 2 : 3>>(x, w, out, ldo, st);
    else if (w.rows >= 32 * kCus) launch_rows<T, MxStream<FX, 2, 4, TOK, 2, 3>>(x, w, out, ldo, st);
    else launch_rows<T, MxStream<FX, 1, 8, TOK, kMany ? 1 : 2, 3>>(x, w, out, ldo, st);
}

// ---- many tokens ------------------------------------------------------------------------------
// Work-groups of BN weight rows x BM tokens go along the rows in stages of 128 or 256 values, NS of them
// in LDS: while stage t is multiplied, t + 1 has arrived (its first operands are read in advance, so the
// matrix cores do not wait at the barrier), those up to t + NS - 2 are on their way and t + NS - 1 is
// sent for, all without passing registers.
//
// 128 values' 4 blocks are taken as steps s = 0, 1 of v_mfma_scale_f32_32x32x64_f8f6f4, step s
// multiplying blocks s and 2 + s: lane (n = lane % 32, b = lane / 32) then needs the scales of blocks
// 2 b and 2 b + 1 of its row, a half word, of which step s selects byte s.
//   FP4: lane (n, b) gives block s + 2 b (16 bytes);
//   FP8: half b of block s, then half b of block 2 + s (16 bytes each).
typedef float mx_v16f __attribute__((ext_vector_type(16)));

// SV: values of a row in a stage; NS: stages in LDS.  Scales come for 512 values, kQuad stages, at a
// time (16 bytes a row), kSlots times of them in LDS.
template <int FX, int NT_, int MT_, int WN_, int WM_, int SV_, int NS_> struct MxTile {
    static constexpr int NT = NT_, MT = MT_, WN = WN_, WM = WM_, SV = SV_, NS = NS_;
    static constexpr int BN = 32 * NT * WN, BM = 32 * MT * WM, W = WN * WM, kThreads = 64 * W;
    static constexpr int kRowW = SV / 2, kRowX = SV * FX / 8;
    static constexpr int kBytesW = BN * kRowW, kBytesX = BM * kRowX;
    static constexpr int kStageBytes = kBytesW + kBytesX;
    static constexpr int kCalls = kStageBytes / 1024 / W;  // copies of a wave and stage
    static constexpr int kScaleBytes = (BN + BM) * 16;
    static constexpr int kScaleCalls = (kScaleBytes / 1024 + W - 1) / W;  // of a wave
    static constexpr int kQuad = 512 / SV, kSlots = (NS - 3 + kQuad) / kQuad;
    static constexpr int kLds = NS * kStageBytes + kSlots * kScaleBytes;
    // Stages after which places and scales are as before.
    static constexpr int kRound = NS % kQuad == 0 ? NS : NS * kQuad;
    static_assert(SV == 128 || SV == 256, "one or two whole steps of the format's padding");
    static_assert(NS >= 3 && (NS - 2) * kCalls < 64 && kLds <= 160 * 1024, "a wait's count; LDS");
    // Scales are sent for in a quad's second stage, kSlots quads ahead: the copies that follow before
    // they are read outnumber those that a wait leaves.
    static_assert(kSlots >= 1 && kQuad * kSlots - 1 >= NS - 3 && kRound / kQuad % kSlots == 0, "scales");
};

// One operand's loads of stages, ROWS rows of ROW bytes in LDS; a wave's instruction brings 1024
// consecutive bytes of them.  A stage that a row's end cuts in half brings its first half twice.
template <int ROW, int ROWS, int W> struct StageLoads {
    static constexpr int kPerRow = ROW / 16, kCalls = ROWS * kPerRow / 64;
    static_assert(kCalls % W == 0, "whole instructions a wave");
    static constexpr int kMine = kCalls / W;
    const unsigned char* base;  // the tile's first row
    unsigned offset[kMine];     // this lane's row and chunk from there
    unsigned second;            // bit i: the chunk is of a stage's second half

    __device__ __forceinline__ void init(const unsigned char* codes, long long row_bytes,
                                         long long row0, long long rows, int wave, int lane) {
        base = codes + row0 * row_bytes;
        const int last = (int)min(rows - 1 - row0, (long long)ROWS - 1);
        second = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int slot = (wave * kMine + i) * 64 + lane, r = slot / kPerRow;
            const int chunk = slot % kPerRow ^ place<ROW>(r);
            offset[i] = (unsigned)(min(r, last) * (int)row_bytes + 16 * chunk);
            second |= (unsigned)(chunk >= kPerRow / 2) << i;
        }
    }
    __device__ __forceinline__ void issue(unsigned char* lds, int t, bool cut, int wave, int i) const {
        const unsigned back = cut ? (second >> i & 1) * (ROW / 2) : 0;
        copy16_to_lds(base + (long long)t * ROW, offset[i] - back, lds + (wave * kMine + i) * 1024);
    }
};

template <typename C> struct Frags {
    mx_v8i w[C::NT], x[C::MT];
};

template <typename C, int FX>
__device__ __forceinline__ void read_frags(Frags<C>& f, const unsigned char* lds, int s, int n0, int m0,
                                           int n, int b) {
    const int w0 = 4 * (s / 2) + (s & 1);
#pragma unroll
    for (int i = 0; i < C::NT; ++i) {
        const int row = n0 + 32 * i + n;
        const uint4 v = *(const uint4*)(lds + row * C::kRowW + 16 * ((w0 + 2 * b) ^ place<C::kRowW>(row)));
        f.w[i] = mx_v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < C::MT; ++j) {
        const int row = m0 + 32 * j + n;
        const unsigned char* p = lds + C::kBytesW + row * C::kRowX;
        if constexpr (FX == kMxFp4) {
            const uint4 v = *(const uint4*)(p + 16 * ((w0 + 2 * b) ^ place<C::kRowX>(row)));
            f.x[j] = mx_v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
        } else {
            const int at = (8 * (s / 2) + 2 * (s & 1) + b) ^ place<C::kRowX>(row);
            const uint4 v = *(const uint4*)(p + 16 * at), u = *(const uint4*)(p + 16 * (at ^ 4));
            f.x[j] = mx_v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w,
                            (int)u.x, (int)u.y, (int)u.z, (int)u.w};
        }
    }
}

// Step S's products; after the k-th, between(k).  What stands between is sent while the matrix cores
// work: a stage's copies one after the other would hold the wave up at the address path.
template <typename C, int FX, int S, typename Between>
__device__ __forceinline__ void use_frags(mx_v16f (&acc)[C::NT][C::MT], const Frags<C>& f,
                                          const int (&ws)[C::NT], const int (&xs)[C::MT],
                                          Between between) {
#pragma unroll
    for (int i = 0; i < C::NT; ++i)
#pragma unroll
        for (int j = 0; j < C::MT; ++j) {
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                f.w[i], f.x[j], acc[i][j], 4, FX == kMxFp8 ? 0 : 4, S, ws[i], S, xs[j]);
            __builtin_amdgcn_sched_barrier(0);
            between(i * C::MT + j);
        }
    __builtin_amdgcn_sched_barrier(0);
}

// Tile of work-group `id`: work-groups go to the 8 XCDs in turn, so XCD x takes the x-th eighth of
// the tiles, in columns of 8 tiles of weight rows, whose operands its L2 holds together.
__device__ __forceinline__ void tile_of(unsigned id, unsigned total, unsigned tn, unsigned tm,
                                        unsigned& bn, unsigned& bm) {
    const unsigned x = id % 8, each = total / 8, more = total % 8;
    const unsigned t = x * each + min(x, more) + id / 8;
    const unsigned band = 8 * tm, g = t / band, in = t % band;
    const unsigned wide = min(8u, tn - 8 * g);
    bn = 8 * g + in % wide;
    bm = in / wide;
}

template <typename T, int FX, typename C>
__global__ void __launch_bounds__(C::kThreads)
k_mx_tiles(MxOperand x, MxOperand wt, typename T::Raw* out, long long ldo, unsigned tn, unsigned tm) {
    __shared__ __attribute__((aligned(256))) unsigned char lds[C::kLds];
    unsigned char* const scales = lds + C::NS * C::kStageBytes;
    const int lane = lane_id(), n = lane & 31, b = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n0 = (wave % C::WN) * 32 * C::NT, m0 = (wave / C::WN) * 32 * C::MT;
    const unsigned id = (unsigned)group_index();
    if (id >= tn * tm) return;  // the whole work-group
    unsigned bn, bm;
    tile_of(id, tn * tm, tn, tm, bn, bm);
    const long long row0 = (long long)bn * C::BN, tok0 = (long long)bm * C::BM;
    const int steps = (int)(mx_padded(x.cols) / kMxStep), quads = (steps + 3) / 4;
    constexpr int kSteps = C::SV / kMxStep;  // of the format's padding, in a stage
    const int stages = (steps + kSteps - 1) / kSteps;
    const bool odd = steps % kSteps;  // the last stage is cut
    StageLoads<C::kRowW, C::BN, C::W> lw;
    StageLoads<C::kRowX, C::BM, C::W> lx;
    lw.init(wt.codes, mx_code_bytes(x.cols, kMxFp4), row0, wt.rows, wave, lane);
    lx.init(x.codes, mx_code_bytes(x.cols, FX), tok0, x.rows, wave, lane);
    // stages past the end are the last again: every wave always has the same number of copies
    auto load_part = [&](unsigned char* to, int t, int i) {
        const int at = min(t, stages - 1);
        const bool cut = kSteps > 1 && odd && at == stages - 1;
        if (i < lw.kMine) lw.issue(to, at, cut, wave, i);
        else lx.issue(to + C::kBytesW, at, cut, wave, i - lw.kMine);
    };
    auto load_stage = [&](unsigned char* to, int t) {
#pragma unroll
        for (int i = 0; i < C::kCalls; ++i) load_part(to, t, i);
    };
    // scales: the rows of W, then the rows of X
    const long long sb = mx_scale_bytes(x.cols);
    static_assert(C::BN % 64 == 0 && C::BM % 64 == 0, "a copy of scales is of W or of X");
    const unsigned char* scale_base[C::kScaleCalls];
    unsigned scale_row[C::kScaleCalls];
    int scale_call[C::kScaleCalls];
#pragma unroll
    for (int i = 0; i < C::kScaleCalls; ++i) {
        scale_call[i] = min(wave * C::kScaleCalls + i, C::kScaleBytes / 1024 - 1);
        const bool of_w = 64 * scale_call[i] < C::BN;
        const long long first = of_w ? row0 + 64 * scale_call[i] : tok0 + 64 * scale_call[i] - C::BN;
        const long long last = (of_w ? wt.rows : x.rows) - 1;
        scale_base[i] = (of_w ? wt.scales : x.scales) + min(first, last) * sb;
        scale_row[i] = (unsigned)((int)min((long long)lane, max(last - first, 0ll)) * (int)sb);
    }
    auto load_scales = [&](int quad, int slot) {
#pragma unroll
        for (int i = 0; i < C::kScaleCalls; ++i)
            copy16_to_lds(scale_base[i], scale_row[i] + 16u * min(quad, quads - 1),
                          scales + slot * C::kScaleBytes + scale_call[i] * 1024);
    };
    mx_v16f acc[C::NT][C::MT] = {};
    uint4 ws[C::NT], xs[C::MT];
    Frags<C> f, g;
#pragma unroll
    for (int i = 0; i < C::kSlots; ++i) load_scales(i, i);
#pragma unroll
    for (int i = 0; i < C::NS - 1; ++i) load_stage(lds + i * C::kStageBytes, i);
    wait_copies<(C::NS - 2) * C::kCalls>();
    read_frags<C, FX>(f, lds, 0, n0, m0, n, b);
    for (int t0 = 0;; t0 += C::kRound) {
        bool more = true;
#pragma unroll
        for (int u = 0; u < C::kRound; ++u) {
            if (!more) break;
            const int t = t0 + u;
            unsigned char* const stage = lds + u % C::NS * C::kStageBytes;
            wait_copies<(C::NS - 3) * C::kCalls>();  // stage t + 1 is here; all are done with t - 1
            // scales go to registers for all their stages, so later ones can take their place at once
            constexpr int Q = C::kQuad;
            const unsigned char* const quad = scales + u / Q % C::kSlots * C::kScaleBytes;
            if (u % Q == 0) {
#pragma unroll
                for (int i = 0; i < C::NT; ++i) ws[i] = *(const uint4*)(quad + 16 * (n0 + 32 * i + n));
#pragma unroll
                for (int j = 0; j < C::MT; ++j)
                    xs[j] = *(const uint4*)(quad + 16 * (C::BN + m0 + 32 * j + n));
            }
            if (u % Q == 1) load_scales(t / Q + C::kSlots, u / Q % C::kSlots);
            int sw[C::NT], sx[C::MT];
#pragma unroll
            for (int s = 0; s < 2 * kSteps; ++s) {
                if (s == 2 && odd && t + 1 == stages) break;
                Frags<C>&now = s & 1 ? g : f, &next = s & 1 ? f : g;
                if (s % 2 == 0) {
#pragma unroll
                    for (int i = 0; i < C::NT; ++i)
                        sw[i] = (int)(word_of(ws[i], u % Q * kSteps + s / 2) >> (16 * b));
#pragma unroll
                    for (int j = 0; j < C::MT; ++j)
                        sx[j] = (int)(word_of(xs[j], u % Q * kSteps + s / 2) >> (16 * b));
                }
                if (s + 1 < 2 * kSteps) read_frags<C, FX>(next, stage, s + 1, n0, m0, n, b);
                else read_frags<C, FX>(next, lds + (u + 1) % C::NS * C::kStageBytes, 0, n0, m0, n, b);
                __builtin_amdgcn_sched_barrier(0);  // reads first: the products then cover their time
                // copies among the products of the first half of the steps
                constexpr int kSpots = C::NT * C::MT * kSteps, kEach = (C::kCalls + kSpots - 1) / kSpots;
                constexpr int kGap = kSpots / ((C::kCalls + kEach - 1) / kEach);  // products to a copy
                auto send = [&](int k) {
                    const int spot = s * C::NT * C::MT + k;
                    if (s >= kSteps) return;
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        const int call = spot / kGap * kEach + i;
                        if (spot % kGap == 0 && call < C::kCalls)
                            load_part(lds + (u + C::NS - 1) % C::NS * C::kStageBytes, t + C::NS - 1, call);
                    }
                };
                if (s & 1) use_frags<C, FX, 1>(acc, now, sw, sx, send);
                else use_frags<C, FX, 0>(acc, now, sw, sx, send);
            }
            more = t + 1 < stages;
        }
        if (!more) break;
    }
    // Lane (n, b) holds weight rows 8 g + 4 b + i, g, i = 0 .. 3, of token n of each 32 x 32 tile.
    // Through LDS, 32 tokens at a time, so that a token's rows leave 16 bytes a lane, whole lines.
    arrive_but<0>();
    using Raw = typename T::Raw;
    constexpr int kPass = sizeof(Raw) == 4 && C::NT > 2 ? C::NT / 2 : C::NT;  // tiles at a time
    constexpr int kRows = 32 * kPass, kPitch = kRows * (int)sizeof(Raw) + 16, kPer = 16 / sizeof(Raw);
    constexpr int kLanes = kRows / kPer;  // of a token
    static_assert(32 * kPitch * C::W <= sizeof lds, "every wave has room");
    unsigned char* const mine = lds + wave * (32 * kPitch);
    const bool vec = ((uintptr_t)out | (uintptr_t)(ldo * sizeof(Raw))) % 16 == 0;
#pragma unroll
    for (int ij = 0; ij < C::MT * (C::NT / kPass); ++ij) {
        const int j = ij % C::MT, i0 = ij / C::MT * kPass;
#pragma unroll
        for (int i = 0; i < kPass; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                Raw v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = T::put(acc[i0 + i][j][4 * g + k]);
                __builtin_memcpy(mine + n * kPitch + (32 * i + 8 * g + 4 * b) * sizeof(Raw), v, sizeof v);
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll 4
        for (int u = lane; u < 32 * kLanes; u += 64) {
            const int tk = u / kLanes, r = u % kLanes * kPer;
            const uint4 v = *(const uint4*)(mine + tk * kPitch + r * sizeof(Raw));
            const long long tok = tok0 + m0 + 32 * j + tk, row = row0 + n0 + 32 * i0 + r;
            if (tok >= x.rows) continue;
            Raw* p = out + tok * ldo + row;
            if (vec && row + kPer <= wt.rows) {
                *(uint4*)p = v;
            } else {
                Raw e[kPer];
                __builtin_memcpy(e, &v, 16);
#pragma unroll
                for (int k = 0; k < kPer; ++k)
                    if (row + k < wt.rows) p[k] = e[k];
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, int FX, typename C>
void launch_tiles(const MxOperand& x, const MxOperand& w, void* out, long long ldo, hipStream_t st) {
    const long long tn = (w.rows + C::BN - 1) / C::BN, tm = (x.rows + C::BM - 1) / C::BM;
    // more than any memory holds the result of: tiles are counted in 32 bits
    if (tn * tm >= 1ll << 31) throw Error(VCSRMC_ERR_OVERFLOW, "product too large for one launch");
    k_mx_tiles<T, FX, C><<<grid_of(tn * tm), C::kThreads, 0, st>>>(
        x, w, (typename T::Raw*)out, ldo, (unsigned)tn, (unsigned)tm);
    VCSRMC_HIP(hipGetLastError());
}

// The largest tiles that still give three quarters of the CUs one: a larger tile loads less for each
// product, an idle CU multiplies nothing.  Times in us of 256 x 256 (FP4 alone: its stages fit LDS four
// times), 256 x 128, 128 x 128, 128 x 64 and 64 x 64 (rows x tokens), each with four stages of 128
// values: 8192^3 FP4 295, 362, 408, 557, 717; 1024 x 8192 x 8192 FP8 -, 60, 74, 84, 102; 2048^3 FP4 19,
// 13, 10.5, 12, 14; 333 x 5000 x 4100 FP8 -, 28, 21, 14, 16; 64 x 8192 x 8192 FP4 52, 36, 23, 19, 17.
//
// The smaller tiles' stages: an FP4 row of 128 values is half a line, and lines are what L2 counts, so
// where tiles fill the CUs, FP4 takes 256; where a CU has one tile, the way of a copy bounds it, and
// eight stages of 128 keep more of them going.  Four of 128, eight of 128 and four of 256:
//   128 x 128  333 x 8192 x 8192 FP4 30.9  30.4  26.4   FP8 35.4  34.8  -  (three of 256 fit: 39.5)
//   128 x 64   333 x 5000 x 4100 FP4 13.4  12.9  12.3   FP8 14.5  14.1 14.2; 320 tiles FP8 23.2  25.6  25.6
//   64 x 64    64 x 8192 x 8192 FP4  23.7  17.4  17.7   FP8 24.9  21.3 20.0
//              64 x 4096 x 4096 FP4   9.1   7.5   7.9   FP8 10.0   9.1  8.8
//              700 x 2048 x 16384 (352 tiles) FP4 40.9  39.2  32.3   FP8 43.0  48.8  50.6
template <typename T, int FX>
void tiles_of(const MxOperand& x, const MxOperand& w, void* out, long long ldo, hipStream_t st) {
    constexpr long long kCus = 256;
    constexpr int kWide = FX == kMxFp4 ? 256 : 128;  // values of a stage
    auto tiles = [&](long long bn, long long bm) {
        return ((w.rows + bn - 1) / bn) * ((x.rows + bm - 1) / bm);
    };
    auto enough = [&](long long bn, long long bm) { return tiles(bn, bm) >= kCus * 3 / 4; };
    if constexpr (FX == kMxFp4)
        if (enough(256, 256)) return launch_tiles<T, FX, MxTile<FX, 2, 4, 4, 2, 128, 4>>(x, w, out, ldo, st);
    if (enough(256, 128)) return launch_tiles<T, FX, MxTile<FX, 2, 2, 4, 2, 128, 4>>(x, w, out, ldo, st);
    if (enough(128, 128)) return launch_tiles<T, FX, MxTile<FX, 2, 2, 2, 2, kWide, 4>>(x, w, out, ldo, st);
    if (enough(128, 64)) {
        if constexpr (FX == kMxFp8)
            if (tiles(128, 64) <= kCus)
                return launch_tiles<T, FX, MxTile<FX, 2, 1, 2, 2, 128, 8>>(x, w, out, ldo, st);
        return launch_tiles<T, FX, MxTile<FX, 2, 1, 2, 2, kWide, 4>>(x, w, out, ldo, st);
    }
    if (tiles(64, 64) <= kCus) launch_tiles<T, FX, MxTile<FX, 1, 1, 2, 2, 128, 8>>(x, w, out, ldo, st);
    else launch_tiles<T, FX, MxTile<FX, 1, 1, 2, 2, kWide, 4>>(x, w, out, ldo, st);
}

template <typename T, int FX>
void launch(const MxOperand& x, const MxOperand& w, void* out, long long ldo, hipStream_t st) {
    if (x.rows <= 1) rows_of<T, FX, 1>(x, w, out, ldo, st);
    else if (x.rows <= 4) rows_of<T, FX, 4>(x, w, out, ldo, st);
    else if (x.rows <= 16) rows_of<T, FX, 16>(x, w, out, ldo, st);
    else if (x.rows <= 32) rows_of<T, FX, 32>(x, w, out, ldo, st);
    else tiles_of<T, FX>(x, w, out, ldo, st);
}

template <typename T>
void launch(const MxOperand& x, const MxOperand& w, void* out, long long ldo, hipStream_t st) {
    if (x.fmt == kMxFp8) launch<T, kMxFp8>(x, w, out, ldo, st);
    else launch<T, kMxFp4>(x, w, out, ldo, st);
}

}  // namespace

void mx_matmul(const MxOperand& x, const MxOperand& w, void* out, int type, long long ldo,
               hipStream_t st) {
    if (x.rows == 0 || w.rows == 0) return;
    if (type == kTypeF32) launch<F32>(x, w, out, ldo, st);
    else if (type == kTypeF16) launch<F16>(x, w, out, ldo, st);
    else launch<BF16>(x, w, out, ldo, st);
}

}  // namespace vcsrmc
