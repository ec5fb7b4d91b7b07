// mx_moe.hip -- a mixture-of-experts layer for a few tokens, experts in MXFP4, activations in
// MXFP8: l = x R^T; the top k experts of a token by l (ties to the lowest index) under
// p = softmax(l); h = MX8(silu(x G^T) * (x U^T)) for each of them; y = sum p (h D^T).
//
// Launches for up to kMoeTokens tokens: the router's logits; the choice of experts and their lists of
// tokens (a single token's in the next launch); gate and up rows of the chosen experts, ending in MX
// blocks of h; down rows of the chosen experts, and the sum over a token's experts in the same launch or
// one more.  Each weight of a chosen expert is read once for 16, 32 or 64 of its tokens.  Between the
// launches lie the logits (T x E), the lists (T k), h (T k x F bytes) and the down rows' sums; nothing
// is added by floating atomics, so results do not depend on the order of work-groups.
#include <type_traits>

#include "internal.hpp"
#include "mx.hpp"

#include "../../include/vcsrmc.h"

namespace vcsrmc {
namespace {

constexpr int kMoeTokens = 64;     // of one set of launches; more tokens take several sets

// A token in an expert's list, and an expert among a token's: the slot where they meet.  Slots are
// those of the first chosen expert, then of the second, and so on; h has a row for each.
struct Slot {
    int token;
    float weight;
};
struct Pair {
    int slot;
    float weight;
};

// Where the parts of a workspace begin.
struct MoePlan {
    long long logits, active, start, slots, pairs, hcodes, hscales, sums, bytes;
};

long long up256(long long n) { return (n + 255) / 256 * 256; }
__host__ __device__ long long up64(long long n) { return (n + 63) / 64 * 64; }

// Parts that the router's rows are cut into, and are added from: no more than there are steps for the
// waves of a work-group.
constexpr int kLogitWaves = 16, kLogitStep = 64, kMaxParts = 4;
int logit_parts(long long D) {
    const long long most = (D + kLogitWaves * kLogitStep - 1) / (kLogitWaves * kLogitStep);
    return (int)(most < kMaxParts ? most : kMaxParts);
}

// Down rows an expert at a time, or of all experts together: see k_moe_down.
constexpr int kFewPairs = 16;
bool by_expert(long long T, int k) { return T * k > kFewPairs; }

MoePlan moe_plan(long long T, long long D, long long F, int E, int k) {
    MoePlan p;
    p.logits = 0;
    p.active = p.logits + up256(4 * T * E * logit_parts(D));
    p.start = p.active + up256(4ll * E);
    p.slots = p.start + up256(4ll * E + 8);
    p.pairs = p.slots + up256((long long)sizeof(Slot) * T * k);
    p.hcodes = p.pairs + up256((long long)sizeof(Pair) * T * k);
    p.hscales = p.hcodes + up256(T * k * mx_code_bytes(F, kMxFp8));
    p.sums = p.hscales + up256(T * k * mx_scale_bytes(F));
    p.bytes = p.sums + (by_expert(T, k) ? 4 * T * k * up64(D) : 0);
    return p;
}

struct MoeDevice {
    const unsigned char *xc, *xs, *w13c, *w13s, *w2c, *w2s;
    const void* router;
    float* logits;  // [parts][T][E]
    int* active;    // the chosen experts, in order
    int* start;     // where their tokens begin in slots; then their number; start[E + 1]: of experts
    Slot* slots;    // T k in all
    Pair* pairs;    // [T][k]
    unsigned char *hc, *hs;
    float* sums;    // of an expert's down rows for a slot: [T k][D rounded up to 64]
    void* out;
    long long ldo;
    int T, D, F, E, k, renormalise;
    int parts;
};

// ---- router -----------------------------------------------------------------------------------
// 16 experts x 16 tokens a work-group on v_mfma_f32_16x16x4_f32 (every product and sum in 32
// bits), its part of the row cut over the waves in steps of 64 values: lane (n, q) takes values
// 16 q .. 16 q + 15 of a step, four matrix instructions' worth each of 4.  Four steps are loaded
// at a time: the launch is one round trip to memory long, 5 us for 1 and for 64 tokens of 64 experts of
// 4096 bfloat16 values (0.5 MB).  With the rows uncut 64 tokens took 14 us.
template <typename R>
__device__ __forceinline__ void load16(const typename R::Raw* p, bool vec, int n, float (&v)[16]) {
    float a[8], b[8];
    load8<R>(p, vec, n, a);
    load8<R>(p + 8, vec, n - 8, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = a[i], v[8 + i] = b[i];
}

template <typename R>
__global__ void __launch_bounds__(64 * kLogitWaves) k_moe_logits(MoeDevice d, bool vec) {
    constexpr int W = kLogitWaves;
    __shared__ mx_v4f part[W][64];
    const int lane = lane_id(), n = lane & 15, q = lane >> 4, wave = threadIdx.x / kWave;
    const int e = min((int)blockIdx.x * 16 + n, d.E - 1), t = min((int)blockIdx.y * 16 + n, d.T - 1);
    const typename R::Raw* r = (const typename R::Raw*)d.router + (long long)e * d.D;
    const unsigned char* xc = d.xc + t * mx_code_bytes(d.D, kMxFp8);
    const unsigned char* xs = d.xs + t * mx_scale_bytes(d.D);
    const int steps = (d.D + 63) / 64, each = (steps + d.parts - 1) / d.parts;
    const int first = blockIdx.z * each, last = min(first + each, steps);
    mx_v4f acc = {0, 0, 0, 0};
    for (int s0 = first + wave; s0 < last; s0 += 4 * W) {
        float a[4][16];
        uint4 c[4];
        int sc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int s = s0 + u * W, at = 64 * s + 16 * q;
            if (s < last) {
                load16<R>(r + at, vec, d.D - at, a[u]);
                c[u] = *(const uint4*)(xc + at);  // padded to 128: inside the row
                sc[u] = xs[at / 32];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (s0 + u * W >= last) break;
            const float f = mx_scale_or_nan(sc[u]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned w = word_of(c[u], i / 2);
                const mx_v2f v = (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.f, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.f, false);
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u][2 * i], v[0] * f, acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u][2 * i + 1], v[1] * f, acc, 0, 0, 0);
            }
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < W; ++w) acc += part[w][lane];
    const int token = blockIdx.y * 16 + n;
    if (token >= d.T) return;
    float* out = d.logits + (long long)blockIdx.z * d.T * d.E;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = blockIdx.x * 16 + 4 * q + i;
        if (row < d.E) out[token * d.E + row] = acc[i];
    }
}

// ---- choice of experts ------------------------------------------------------------------------
// Order of a token's experts: larger logit first, equal ones by index, NaN last.  Logits are compared
// as whole numbers of the same order, at least 1; NaN is 1, an expert already taken 0.
__device__ __forceinline__ unsigned key_of(float v) {
    const unsigned u = __float_as_uint(v + 0.f);  // -0 is 0
    return v != v ? 1u : u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key == 1 ? 0x7fc00000u : key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}
// Over the L lanes of a group, 16 (a DPP row) or 64; every lane gets it.
template <int L> __device__ __forceinline__ unsigned group_max(unsigned v) {
    static_assert(L == 16 || L == 64);
    auto turned = [](unsigned u, auto by) {
        return (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, 0x120 + by.value, 0xf, 0xf, true);
    };
    v = max(v, turned(v, std::integral_constant<int, 8>{}));
    v = max(v, turned(v, std::integral_constant<int, 4>{}));
    v = max(v, turned(v, std::integral_constant<int, 2>{}));
    v = max(v, turned(v, std::integral_constant<int, 1>{}));
    if (L == 64) {
        v = max(v, (unsigned)__shfl_xor((int)v, 16));
        v = max(v, (unsigned)__shfl_xor((int)v, 32));
    }
    return v;
}
template <int L> __device__ __forceinline__ float group_add(float v) {
#pragma unroll
    for (int i = 1; i < L; i *= 2) v += __shfl_xor(v, i);
    return v;
}

// L lanes' work on token t, lane l with the KE experts l, L + l and so on: picks the largest key top_k
// times and calls put(rank, expert, exp(l - the largest l)) in one of the lanes.  Returns what the
// weights are to be divided by.  16 lanes take 8 of 64 experts with a quarter of the instructions that
// a wave would need: on one CU, 64 tokens are bound by those.
template <int L, int KE, typename Put>
__device__ __forceinline__ float choose(const MoeDevice& d, int t, Put put) {
    const int lane = lane_id() % L;
    unsigned key[KE], left[KE];
#pragma unroll
    for (int i = 0; i < KE; ++i) {
        const int e = L * i + lane;
        const float* p = d.logits + t * d.E + min(e, d.E - 1);
        float v[kMaxParts], sum = 0.f;
#pragma unroll
        for (int s = 0; s < kMaxParts; ++s) v[s] = p[min(s, d.parts - 1) * d.T * d.E];
#pragma unroll
        for (int s = 0; s < kMaxParts; ++s) sum = s == 0 ? v[0] : s < d.parts ? sum + v[s] : sum;
        key[i] = left[i] = e < d.E ? key_of(sum) : 0u;
    }
    float first = 0.f, z = 0.f;
    for (int r = 0; r < d.k; ++r) {
        unsigned best = 0, e = ~0u;
#pragma unroll
        for (int i = 0; i < KE; ++i) best = max(best, left[i]);
        best = group_max<L>(best);
#pragma unroll
        for (int i = KE - 1; i >= 0; --i) e = left[i] == best ? (unsigned)(L * i + lane) : e;
        e = ~group_max<L>(~e);  // the lowest
#pragma unroll
        for (int i = 0; i < KE; ++i) left[i] = e == (unsigned)(L * i + lane) ? 0u : left[i];
        if (r == 0) first = value_of(best);
        const float w = expf(value_of(best) - first);
        if (lane == r % L) put(r, (int)e, w);
        z += w;
    }
    if (d.renormalise) return z;
    z = 0.f;
#pragma unroll
    for (int i = 0; i < KE; ++i) z += key[i] ? expf(value_of(key[i]) - first) : 0.f;
    return group_add<L>(z);
}

// One work-group, for 2 tokens and more; a single one's experts are chosen by the next launch.  A set of
// tokens for every expert gives the lists: where a token stands in one is how many earlier tokens are in
// the set.  Bound by latency: 4 us for 7 tokens, 6 of 60 experts, and 6.8 us for 64 tokens, 8 of 64 (12.4
// with a wave a token).  Every work-group of the next launch choosing anew for 64 tokens took 10 us more.
template <int L, int KE>
__global__ void __launch_bounds__(1024) k_moe_choose(MoeDevice d) {
    constexpr int W = 16, kAtOnce = W * 64 / L;  // tokens
    static_assert(64 * W >= kMoeExperts && kMoeTokens <= 64, "a thread an expert, a bit a token");
    __shared__ unsigned long long tokens_of[kMoeExperts];
    __shared__ int list_of[kMoeExperts], wave_on[W], wave_tokens[W];
    __shared__ unsigned short ids[kMoeTokens * kMoeTopK];
    __shared__ float weights[kMoeTokens * kMoeTopK], over[kMoeTokens];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    tokens_of[threadIdx.x] = 0;
    __syncthreads();
    for (int t0 = wave * (64 / L); t0 < d.T; t0 += kAtOnce) {
        const int t = t0 + lane / L;  // groups past the last token work on it and keep quiet
        const float z = choose<L, KE>(d, min(t, d.T - 1), [&](int r, int e, float w) {
            if (t >= d.T) return;
            ids[t * d.k + r] = (unsigned short)e;
            weights[t * d.k + r] = w;
            atomicOr(&tokens_of[e], 1ull << t);
        });
        if (lane % L == 0 && t < d.T) over[t] = z;
    }
    __syncthreads();
    // chosen experts in order, and where their tokens begin
    const int count = __popcll(tokens_of[threadIdx.x]);
    const unsigned long long on = __ballot(count > 0);
    const int upto = wave_scan(count, OpAdd{}, 0);  // of this wave's experts, this one included
    if (lane == 63) wave_tokens[wave] = upto;
    if (lane == 0) wave_on[wave] = __popcll(on);
    __syncthreads();
    int before_on = 0, before_tokens = 0;
    for (int w = 0; w < wave; ++w) before_on += wave_on[w], before_tokens += wave_tokens[w];
    const int at = before_on + __popcll(on & ((1ull << lane) - 1)), first = before_tokens + upto - count;
    if (count > 0) {
        d.active[at] = threadIdx.x;
        d.start[at] = first;
        list_of[threadIdx.x] = first;
    }
    if (threadIdx.x == 64 * W - 1) {
        const int all = before_on + __popcll(on);
        d.start[all] = before_tokens + upto;
        d.start[d.E + 1] = all;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < d.T * d.k; i += 64 * W) {
        const int e = ids[i], t = i / d.k;
        const int slot = list_of[e] + __popcll(tokens_of[e] & ((1ull << t) - 1));
        const float w = weights[i] / over[t];
        d.slots[slot] = Slot{t, w};
        d.pairs[i] = Pair{slot, w};
    }
}

// ---- gate and up rows -------------------------------------------------------------------------
// Work-group (f, a): rows 32 f .. 32 f + 31 of gate and up of the a-th chosen expert.  A wave has 16 of
// the rows; their sums meet in LDS, where one wave forms h and its MX block, whose 32 values are the
// work-group's rows.  The products are taken in bfloat16, which holds every FP4 and FP8 value
// but at the ends of their scales' range, on instructions that add them in 32 bits: the FP8 ones cut small products, which would show in h's
// rounding.  Bound by reading the weights: 64 experts of 2 x 2048 x 4096 (570 MB) in 110 us, 5.2 TB/s.
// Stages are small (two, 28 KB) so that five work-groups share a CU: three stages took 124 us.
// For up to 4 tokens, whose work-groups are few, twice the waves; 35 MB in 11 us.
// With KE the work-groups choose a single token's experts first: 22 us a layer, with a launch for it 25.
// TOK: tokens of an expert that are worked on at a time.
template <int TOK, int WK, int L, int KE>
__global__ void __launch_bounds__(256 * WK) k_moe_up(MoeDevice d) {
    using UpStream = MxStream<kMxFp8, 4, WK, TOK, 2, 2>;
    __shared__ __attribute__((aligned(256))) unsigned char lds[UpStream::kLds];
    const int lane = lane_id(), n = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int f0 = blockIdx.x * 32, a = blockIdx.y;
    int e, count = 1, slot0 = a;
    if constexpr (KE > 0) {
        static_assert(TOK == 1, "a single token");
        __shared__ int chosen;
        if (wave == 0) {
            int mine = 0;
            float w = 0.f;
            const float z = choose<L, KE>(d, 0, [&](int r, int e, float v) {
                if (r != a || lane >= L) return;
                chosen = mine = e;
                w = v;
            });
            if (f0 == 0 && lane == a % L) {  // the lists, experts in the order of their ranks
                d.active[a] = mine;
                d.start[a] = a;
                d.start[d.k] = d.start[d.E + 1] = d.k;
                d.slots[a] = Slot{0, w / z};
                d.pairs[a] = Pair{a, w / z};
            }
        }
        __syncthreads();
        e = __builtin_amdgcn_readfirstlane(chosen);
    } else {
        if (a >= d.start[d.E + 1]) return;
        e = d.active[a];
        slot0 = d.start[a];
        count = d.start[a + 1] - slot0;
    }
    const Slot* const slots = d.slots + slot0;
    const int steps = (int)(mx_padded(d.D) / kMxStep);
    const long long first = (long long)e * 2 * d.F, wb = mx_code_bytes(d.D, kMxFp4);
    const long long hb = mx_code_bytes(d.F, kMxFp8), hsb = mx_scale_bytes(d.F);
    for (int t0 = 0; t0 < count; t0 += TOK) {
        UpStream up;  // row tiles: gate rows 0..15, 16..31, up rows 0..15, 16..31
        up.init(d.w13c + first * wb, d.w13s + first * mx_scale_bytes(d.D), d.xc, d.xs, d.D, wave,
                [&](int r) { return (unsigned)((r >> 5) * d.F + min(f0 + (r & 31), d.F - 1)); },
                [&](int m) { return KE ? 0u : (unsigned)slots[min(t0 + m, count - 1)].token; });
        constexpr int MT = UpStream::MT;
        static_assert(4 * WK * MT * 1024 <= UpStream::kLds && MT <= 4 * WK, "sums fit, a wave a tile");
        mx_v4f acc[MT] = {};
        up.template run<true>(acc, lds, steps);
        mx_v4f(*const part)[MT][64] = (mx_v4f(*)[MT][64])lds;
#pragma unroll
        for (int m = 0; m < MT; ++m) part[wave][m][lane] = acc[m];
        __syncthreads();
        if (wave < MT) {  // tokens 16 wave .. 16 wave + 15
            mx_v4f g[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                g[r] = part[r][wave][lane];
#pragma unroll
                for (int k = 1; k < WK; ++k) g[r] += part[4 * k + r][wave][lane];
            }
            // lane (n, q) holds h of values 4 q .. 4 q + 3 and 16 + 4 q .. 16 + 4 q + 3
            float h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float gate = g[i / 4][i % 4], up = g[2 + i / 4][i % 4];
                h[i] = f0 + 16 * (i / 4) + 4 * q + i % 4 < d.F ? gate / (1.f + expf(-gate)) * up : 0.f;
            }
            unsigned m = absmax8(h);
            m = max(m, (unsigned)__shfl_xor((int)m, 16));
            m = max(m, (unsigned)__shfl_xor((int)m, 32));
            const int sc = mx_scale_of(m, kMxFp8);
            const uint2 c = mx_codes8(h, sc, kMxFp8);
            const int token = 16 * wave + n;
            if (token < TOK && t0 + token < count) {
                const long long row = slot0 + t0 + token;
                unsigned char* p = d.hc + row * hb + f0 + 4 * q;
                *(unsigned*)p = c.x;
                *(unsigned*)(p + 16) = c.y;
                if (q == 0) d.hs[row * hsb + f0 / 32] = (unsigned char)sc;
            }
        }
        __syncthreads();
    }
}

// ---- down rows --------------------------------------------------------------------------------
// Few pairs: a work-group has 16 rows of D of every chosen expert.  Each of its waves has a part of one
// expert's rows (as many parts as there are waves for); the parts' 16 x 16 products, under the tokens'
// weights, meet in LDS and are added in wave order, so that no launch has to follow.  Bound by the
// latency of one chain of loads: 6 us for 4 experts of 4096 x 2048 (17 MB).  More pairs would send the
// waves from expert to expert, and their loads, 64 bytes of each of 16 rows, then take 80 us for 64
// experts against 56 + 5 of the kernels below; at 32 pairs both are equal.
struct DownChunk {  // 512 values of 16 rows of weights
    uint4 w[4], scale;
};

template <typename O>
__global__ void __launch_bounds__(64 * kFewPairs) k_moe_down(MoeDevice d) {
    constexpr int W = kFewPairs;  // waves, and most experts and tokens
    __shared__ float sums[W][W * 16];
    const int lane = lane_id(), n = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int steps = (int)(mx_padded(d.F) / kMxStep), chunks = (steps + 3) / 4;
    const int nactive = d.start[d.E + 1], parts = min(chunks, W / nactive), a = wave / parts;
    const int row0 = blockIdx.x * 16;
    for (int i = lane; i < d.T * 16; i += 64) sums[wave][i] = 0.f;
    if (a < nactive) {
        const long long wb = mx_code_bytes(d.F, kMxFp4), hb = mx_code_bytes(d.F, kMxFp8),
                        sb = mx_scale_bytes(d.F);
        const long long row = (long long)d.active[a] * d.D + min(row0 + n, d.D - 1);
        const int count = d.start[a + 1] - d.start[a], at = d.start[a] + min(n, count - 1);
        const unsigned char *wc = d.w2c + row * wb + 16 * q, *ws = d.w2s + row * sb,
                            *hc = d.hc + at * hb + 16 * q, *hs = d.hs + at * sb;
        const Slot slot = d.slots[at];
        auto load = [&](DownChunk& to, int c) {
            to.scale = *(const uint4*)(ws + 16ll * c);
#pragma unroll
            for (int s = 0; s < 4; ++s)  // past the end: the last step's codes, not used
                to.w[s] = *(const uint4*)(wc + 64ll * min(4 * c + s, steps - 1));
        };
        int c = wave % parts;
        DownChunk now;
        load(now, c);
        mx_v4f acc = {0, 0, 0, 0};
        while (c < chunks) {
            const uint4 scale = *(const uint4*)(hs + 16ll * c);
            MxFrag<kMxFp8> h[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) h[s].load(hc + 128ll * min(4 * c + s, steps - 1));
            DownChunk next = now;
            if (c + parts < chunks) load(next, c + parts);
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (4 * c + s < steps) {
                    MxFrag<kMxFp4> w;
                    w.lo = now.w[s];
                    acc = mx_step<kMxFp8>(w, word_of(now.scale, s) >> (8 * q), h[s],
                                          word_of(scale, s) >> (8 * q), acc);
                }
            c += parts;
            now = next;
        }
        if (n < count) *(mx_v4f*)(sums[wave] + slot.token * 16 + 4 * q) = acc * slot.weight;
    }
    __syncthreads();
    const int t = threadIdx.x / 16, r = threadIdx.x % 16;
    if (t >= d.T || row0 + r >= d.D) return;
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) y += sums[w][threadIdx.x];
    ((typename O::Raw*)d.out)[t * d.ldo + row0 + r] = O::put(y);
}

// More pairs: work-group (r, a) has rows 64 r .. 64 r + 63 of the a-th chosen expert, and streams them
// through LDS; its sums go to memory (8 MB for 64 tokens of 8 experts and 4096 rows) for k_moe_join.
// Bound by reading the weights: 64 experts of 4096 x 2048 (285 MB) in 56 us, 5.1 TB/s.
template <int TOK>
__global__ void __launch_bounds__(256) k_moe_down_rows(MoeDevice d) {
    using Stream = MxStream<kMxFp8, 4, 1, TOK, 2, 2>;
    __shared__ __attribute__((aligned(256))) unsigned char lds[Stream::kLds];
    const int lane = lane_id(), n = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int row0 = blockIdx.x * 64, a = blockIdx.y;
    if (a >= d.start[d.E + 1]) return;
    const long long first = (long long)d.active[a] * d.D, slot0 = d.start[a], Dp = up64(d.D);
    const int count = d.start[a + 1] - d.start[a], steps = (int)(mx_padded(d.F) / kMxStep);
    const long long wb = mx_code_bytes(d.F, kMxFp4), hb = mx_code_bytes(d.F, kMxFp8),
                    sb = mx_scale_bytes(d.F);
    for (int t0 = 0; t0 < count; t0 += TOK) {
        Stream down;
        down.init(d.w2c + first * wb, d.w2s + first * sb, d.hc + slot0 * hb, d.hs + slot0 * sb, d.F, wave,
                  [&](int r) { return (unsigned)min(row0 + r, d.D - 1); },
                  [&](int m) { return (unsigned)min(t0 + m, count - 1); });
        mx_v4f acc[Stream::MT] = {};
        down.template run<false>(acc, lds, steps);
#pragma unroll
        for (int m = 0; m < Stream::MT; ++m) {
            const int token = t0 + 16 * m + n;
            if (token < count) *(mx_v4f*)(d.sums + (slot0 + token) * Dp + row0 + 16 * wave + 4 * q) = acc[m];
        }
    }
}

// Adds a token's rows under their weights, the largest first: 64 tokens x 8 x 4096 in 4.8 us.
template <typename O>
__global__ void __launch_bounds__(256) k_moe_join(MoeDevice d) {
    const int c = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
    const long long Dp = up64(d.D);
    if (c >= d.D) return;
    const Pair* const pairs = d.pairs + t * d.k;
    float y = 0.f;
    for (int r0 = 0; r0 < d.k; r0 += 8) {
        float v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = d.sums[pairs[min(r0 + r, d.k - 1)].slot * Dp + c];
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r0 + r < d.k) y += pairs[r0 + r].weight * v[r];
    }
    ((typename O::Raw*)d.out)[t * d.ldo + c] = O::put(y);
}

template <typename R>
void launch_logits(const MoeDevice& d, hipStream_t st) {
    const bool vec = (uintptr_t)d.router % 16 == 0 &&
                     (long long)d.D * sizeof(typename R::Raw) % 16 == 0;
    const dim3 grid((d.E + 15) / 16, (d.T + 15) / 16, d.parts);
    k_moe_logits<R><<<grid, 64 * kLogitWaves, 0, st>>>(d, vec);
}

// Tokens of an expert that gate, up and down rows are multiplied with at a time, by the mean list: a
// longer list reads the expert's weights once more for each, places past its end are multiplied for
// nothing and take LDS.  us of a layer of 4096 x 2048 with 16, 32 and 64 at a time: 64 tokens, 8 of 64
// experts (mean 8) 183, 214, -; 8 of 40 (12.8) 145, 149, -; 8 of 32 (16) 142, 123, 170; 48 tokens, 8 of
// 16 (24) 94, 72, 100; 64 tokens, 8 of 16 (32) 117, 101, 101; 4 of 8 (32) 75, 69, 60; 8 of 8 (64) 100,
// 78, 66.
int tokens_at_once(const MoeDevice& d) {
    const int all = d.T * d.k;
    return all >= 32 * d.E ? 64 : all >= 14 * d.E ? 32 : 16;
}

template <int L, int KE>
void launch_up(const MoeDevice& d, dim3 grid, hipStream_t st) {
    if (d.T == 1) {
        k_moe_up<1, 2, L, KE><<<grid, 512, 0, st>>>(d);
        return;
    }
    k_moe_choose<L, KE><<<1, 1024, 0, st>>>(d);
    VCSRMC_HIP(hipGetLastError());
    if (d.T <= 4) k_moe_up<4, 2, 0, 0><<<grid, 512, 0, st>>>(d);
    else if (tokens_at_once(d) == 16) k_moe_up<16, 1, 0, 0><<<grid, 256, 0, st>>>(d);
    else if (tokens_at_once(d) == 32) k_moe_up<32, 1, 0, 0><<<grid, 256, 0, st>>>(d);
    else k_moe_up<64, 1, 0, 0><<<grid, 256, 0, st>>>(d);
}

template <typename O>
void launch_down(const MoeDevice& d, long long experts, hipStream_t st) {
    if (by_expert(d.T, d.k)) {
        const dim3 grid((d.D + 63) / 64, (unsigned)experts);
        if (tokens_at_once(d) == 16) k_moe_down_rows<16><<<grid, 256, 0, st>>>(d);
        else if (tokens_at_once(d) == 32) k_moe_down_rows<32><<<grid, 256, 0, st>>>(d);
        else k_moe_down_rows<64><<<grid, 256, 0, st>>>(d);
        VCSRMC_HIP(hipGetLastError());
        k_moe_join<O><<<dim3((d.D + 255) / 256, d.T), 256, 0, st>>>(d);
        return;
    }
    k_moe_down<O><<<(d.D + 15) / 16, 64 * kFewPairs, 0, st>>>(d);
}

}  // namespace

long long mx_moe_workspace(long long T, long long D, long long F, int experts, int top_k) {
    long long most = 0;  // of a whole set of tokens and of the last one
    for (const long long n : {T < kMoeTokens ? T : (long long)kMoeTokens, T % kMoeTokens})
        if (n > 0 && moe_plan(n, D, F, experts, top_k).bytes > most)
            most = moe_plan(n, D, F, experts, top_k).bytes;
    return most;
}

void mx_moe(const MoeArgs& a, hipStream_t st) {
    const long long T = a.x.rows, D = a.x.cols, F = a.w2.cols;
    char* ws = (char*)a.workspace;
    for (long long t0 = 0; t0 < T; t0 += kMoeTokens) {
        const long long n = T - t0 < kMoeTokens ? T - t0 : kMoeTokens;
        const MoePlan p = moe_plan(n, D, F, a.experts, a.top_k);
        MoeDevice d;
        d.xc = a.x.codes + t0 * mx_code_bytes(D, kMxFp8);
        d.xs = a.x.scales + t0 * mx_scale_bytes(D);
        d.w13c = a.w13.codes;
        d.w13s = a.w13.scales;
        d.w2c = a.w2.codes;
        d.w2s = a.w2.scales;
        d.router = a.router;
        d.logits = (float*)(ws + p.logits);
        d.active = (int*)(ws + p.active);
        d.start = (int*)(ws + p.start);
        d.slots = (Slot*)(ws + p.slots);
        d.pairs = (Pair*)(ws + p.pairs);
        d.hc = (unsigned char*)ws + p.hcodes;
        d.hs = (unsigned char*)ws + p.hscales;
        d.sums = (float*)(ws + p.sums);
        d.out = (char*)a.out + t0 * a.ldo * (a.type == kTypeF32 ? 4 : 2);
        d.ldo = a.ldo;
        d.T = (int)n;
        d.D = (int)D;
        d.F = (int)F;
        d.E = a.experts;
        d.k = a.top_k;
        d.renormalise = a.renormalise;
        d.parts = logit_parts(D);
        if (a.router_type == kTypeF32) launch_logits<F32>(d, st);
        else if (a.router_type == kTypeF16) launch_logits<F16>(d, st);
        else launch_logits<BF16>(d, st);
        VCSRMC_HIP(hipGetLastError());
        const long long most = n * a.top_k < a.experts ? n * a.top_k : a.experts;  // chosen experts
        const dim3 grid((unsigned)(mx_padded(F) / 32), (unsigned)most);
        if (d.E <= 64) launch_up<16, 4>(d, grid, st);
        else if (d.E <= 256) launch_up<16, 16>(d, grid, st);
        else launch_up<64, 16>(d, grid, st);
        VCSRMC_HIP(hipGetLastError());
        if (a.type == kTypeF32) launch_down<F32>(d, most, st);
        else if (a.type == kTypeF16) launch_down<F16>(d, most, st);
        else launch_down<BF16>(d, most, st);
        VCSRMC_HIP(hipGetLastError());
    }
}

}  // namespace vcsrmc
