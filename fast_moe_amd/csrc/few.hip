// fmoe_few_tokens: a whole mixture-of-experts layer for a few tokens (a decode step) in two launches.
//
//   l[t, :] = x[t] . G[e] + bg[e];   the k largest l of a token are its experts, g = softmax of l over them (or over all)
//   h[t, j] = g[t, j] * silu(x[t] . W[e] + b[e]) (* (x[t] . Wp[e] + bp[e]))             e = the token's j-th expert
//   y[t]    = sum_j h[t, j] . Wo[e] + g[t, j] * bo[e]
//
// What bounds it are the bytes of the experts hit, each to be read once: 2 * T flops a byte leave the matrix cores idle.  So the
// weights go from memory to the MFMAs' registers with nothing in between (no LDS, no other wave reads them), and everything else
// is kept out of their way:
//   few_up    every block computes the whole router for itself (the same sums in the same order, so the same selection everywhere:
//             a launch of its own would cost more than the gate's few hundred KB from the L2), then takes (expert, 16 hidden columns)
//             items; its waves share the contraction and meet in LDS.  An expert's tokens are gathered into the MFMAs' columns.
//   few_down  a block owns 16 output columns for all tokens; its waves share the experts and their contraction.  The gate is folded into h, so
//             the experts' products add up in one accumulator, no partial sum leaves the block and no atomics are needed.
// Weights are the MFMAs' A operand (rows = output columns), tokens its B operand (16 columns).
#include "common.h"

namespace fmoe {
namespace {

constexpr int kFewMostTokens = 64, kFewMostExperts = 256, kFewMostK = 16, kFewMostWidth = 1 << 16, kFewMostStride = 1 << 20;
constexpr int kWaves = 16;             // of a block: one to a CU, so that the router is computed once per CU
constexpr int kLogitWaves = 8;
constexpr int kRouterRow = 64 + 4;      // floats of a token's sums over 64 experts (the 4: other banks for the next token)

struct FewParams {
    fmoe_few_desc d;
    void* lists;            // who goes where (FewLists)
    void* h;                // hidden rows [T * k][H]
    const float* logits;    // [stretches][T][E]
    int stretches;          // of the router's own launch, 0: the router is few_up's
};

enum { kWF32 = 0, kWBF16 = 1, kWE4M3 = 2 };

// Elements of a 16-byte chunk, bytes of an element, and chunks of x that go with one of weights
template <int WT> struct Wt;
template <> struct Wt<kWF32> { static constexpr int CE = 4, ES = 4, XES = 4, XC = 1; };
template <> struct Wt<kWBF16> { static constexpr int CE = 8, ES = 2, XES = 2, XC = 1; };
template <> struct Wt<kWE4M3> { static constexpr int CE = 16, ES = 1, XES = 2, XC = 2; };

// 16 bytes of a row of n elements of ES bytes from element k on, zeros behind its end.  VEC: rows are whole chunks at 16-byte boundaries.
template <int ES, bool VEC>
__device__ __forceinline__ u32x4 chunk(const uint8_t* row, int k, int n) {
    u32x4 v = {0, 0, 0, 0};
    if constexpr (VEC) {
        if (k < n) v = *reinterpret_cast<const u32x4*>(row + (int64_t)k * ES);
    } else {
#pragma unroll
        for (int i = 0; i < 16 / ES; ++i) {
            if (k + i >= n) continue;
            const uint8_t* p = row + (int64_t)(k + i) * ES;
            if constexpr (ES == 4) v[i] = *reinterpret_cast<const uint32_t*>(p);
            else if constexpr (ES == 2) v[i / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p) << (16 * (i & 1));
            else v[i / 4] |= (uint32_t)*p << (8 * (i & 3));
        }
    }
    return v;
}
// Rows behind a base address that is the same in all lanes, each at a byte offset of its own (below 2^31: few_check).  Whole chunks come through a
// buffer descriptor: an offset beyond its range reads as zeros, which makes the end of a row one select in the place of a branch around every load.
template <int ES, bool VEC>
struct Rows {
    const uint8_t* base;
    __amdgpu_buffer_rsrc_t buffer;
    __device__ __forceinline__ void at(const void* p) {
        base = (const uint8_t*)p;
        if constexpr (VEC) buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, 0x7ffffff0, 0x00027000);
    }
    __device__ __forceinline__ u32x4 chunk(uint32_t row, int k, int n) const {
        if constexpr (VEC) return __builtin_amdgcn_raw_buffer_load_b128(buffer, k < n ? (int)(row + (uint32_t)k * ES) : -1, 0, 0);
        else return fmoe::chunk<ES, false>(base + row, k, n);
    }
};

// Eight e4m3 values as bf16, which holds them exactly.
__device__ __forceinline__ bf16x8 e4m3_to_bf16(uint32_t lo, uint32_t hi) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int w = (int)(i ? hi : lo);
        const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        r[2 * i] = cvt_pk_bf16(a[0], a[1]);
        r[2 * i + 1] = cvt_pk_bf16(b[0], b[1]);
    }
    return __builtin_bit_cast(bf16x8, r);
}

// acc += weights chunk (A) x tokens chunk (B); the order of k inside a chunk is the same on both sides and so does not matter
template <int WT>
__device__ __forceinline__ void mma(f32x4& acc, const u32x4& w, const u32x4* x) {
    if constexpr (WT == kWF32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[j]), __uint_as_float(x[0][j]), acc, 0, 0, 0);
    } else if constexpr (WT == kWBF16) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x[0]), acc, 0, 0, 0);
    } else {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3_to_bf16(w[0], w[1]), __builtin_bit_cast(bf16x8, x[0]), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3_to_bf16(w[2], w[3]), __builtin_bit_cast(bf16x8, x[1]), acc, 0, 0, 0);
    }
}

// (what the compiler cannot know to be the same in all lanes of a wave)
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <bool F32>
__device__ __forceinline__ float element(const void* p, int64_t i) {
    if constexpr (F32) return reinterpret_cast<const float*>(p)[i];
    else return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}
template <bool F32>
__device__ __forceinline__ void put_element(void* p, int64_t i, float v) {
    if constexpr (F32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16_bits(v);
}

// The largest key of the wave: inside a row of 16 lanes on the DPP network, the four rows on the scalar unit.
__device__ __forceinline__ uint32_t wave_max_key(uint32_t v) {
#define FMOE_DPP_MAX(ctrl) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, ctrl, 0xF, 0xF, false))
    FMOE_DPP_MAX(0xB1);      // quad_perm [1,0,3,2]
    FMOE_DPP_MAX(0x4E);      // quad_perm [2,3,0,1]
    FMOE_DPP_MAX(0x141);     // row_half_mirror
    FMOE_DPP_MAX(0x140);     // row_mirror
#undef FMOE_DPP_MAX
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) m = max(m, (uint32_t)__builtin_amdgcn_readlane((int)v, 16 * r));
    return m;
}
// Order of floats as unsigned integers: NaN above all, -0 beside +0; 0 is below every value.
__device__ __forceinline__ uint32_t order_key(float f) {
    if (f != f) return 0xffffffffu;
    const uint32_t u = __float_as_uint(f + 0.0f);
    return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

struct FewLists {           // in LDS
    int16_t* sel;           // [T * k] expert, -1: none
    float* gate;            // [T * k]
    unsigned long long* mask;   // [E] tokens
    int16_t* rank;          // [E]
    int16_t* act;           // [E]
    int16_t* base;          // [E + 1] first of an active expert's slots
    int16_t* slots;         // [T * k] t * k + j, by expert and token
    int16_t* item;          // [2 E] active expert | 0x4000 for its tokens 32 .. 63 (16 .. where NT = 1: cannot be)
    int* counts;            // [2] active experts, items
};
__host__ __device__ constexpr int few_align(int bytes) { return (bytes + 15) & ~15; }
__host__ __device__ inline int few_lists_bytes(int T, int E, int k) {
    return 2 * few_align(T * k * 2) + few_align(T * k * 4) + few_align(E * 8) + 2 * few_align(E * 2) + few_align(E * 2 + 2) + few_align(E * 4) + 16;
}
__device__ __forceinline__ FewLists few_lists(uint8_t* p, int T, int E, int k) {
    FewLists l;
    auto take = [&](int bytes) {
        uint8_t* at = p;
        p += few_align(bytes);
        return at;
    };
    l.mask = (unsigned long long*)take(E * 8);
    l.gate = (float*)take(T * k * 4);
    l.sel = (int16_t*)take(T * k * 2);
    l.slots = (int16_t*)take(T * k * 2);
    l.rank = (int16_t*)take(E * 2);
    l.act = (int16_t*)take(E * 2);
    l.base = (int16_t*)take(E * 2 + 2);
    l.item = (int16_t*)take(E * 4);
    l.counts = (int*)take(8);
    return l;
}
// Sums that meet: of 8 shares of the router, or of 16 waves' two accumulators
constexpr int kRedBytes = kWaves / 2 * 16 * kRouterRow * 4;
static_assert(kRedBytes >= kWaves * 2 * kWave * 16, "the waves' accumulators lie in the router's buffer");

// Logits of tokens t0 .. t0 + 15 into LDS [16][E], 64 experts at a time: the waves' halves have 32 each and share the contraction in pieces of
// 128 bytes per row (whole cache lines); their sums are added in wave order.
template <bool F32, bool VEC>
__device__ __forceinline__ void router_logits(const fmoe_few_desc& d, int t0, float* red, float* logits) {
    constexpr int WT = F32 ? kWF32 : kWBF16, CE = Wt<WT>::CE, ES = Wt<WT>::ES, STEP = 4 * CE, U = 4, SHARES = kWaves / 2;
    const int lane = lane_id(), wave = uniform(threadIdx.x / kWave), share = wave % SHARES, half = wave / SHARES, r16 = lane & 15, quarter = lane >> 4;
    const int t = t0 + r16 < d.T ? t0 + r16 : d.T - 1;
    const uint32_t xrow = (uint32_t)(t * (int)d.x_stride_row * ES);
    Rows<ES, VEC> x, g;
    x.at(d.x);
    g.at(d.gate_weight);
    const int steps = (d.D + STEP - 1) / STEP;
    for (int e0 = 0; e0 < d.E; e0 += 64) {
        const int first = e0 + 32 * half, tiles = first < d.E ? min(2, (d.E - first + 15) / 16) : 0;
        uint32_t wrow[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) wrow[f] = (uint32_t)(min(first + 16 * f + r16, d.E - 1) * (int)d.gate_stride_row * ES);
        f32x4 acc[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s0 = 2 * share; tiles && s0 < steps; s0 += SHARES * U) {
            u32x4 xv[U], wv[U][2];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (s0 + (u / 2) * 2 * SHARES + (u & 1)) * STEP + quarter * CE;
                xv[u] = x.chunk(xrow, k, d.D);
#pragma unroll
                for (int f = 0; f < 2; ++f) wv[u][f] = g.chunk(wrow[f], k, f < tiles ? d.D : 0);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int f = 0; f < 2; ++f) mma<WT>(acc[f], wv[u][f], &xv[u]);
        }
#pragma unroll
        for (int f = 0; f < 2; ++f)
            *reinterpret_cast<f32x4*>(red + (share * 16 + r16) * kRouterRow + 32 * half + 16 * f + 4 * quarter) = acc[f];
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * 64; i += kWaves * kWave) {
            const int row = i >> 6, e = e0 + (i & 63);
            if (e < d.E) {
                float s = red[row * kRouterRow + (i & 63)];
#pragma unroll
                for (int w = 1; w < SHARES; ++w) s += red[(w * 16 + row) * kRouterRow + (i & 63)];
                if (d.gate_bias) s += element<F32>(d.gate_bias, e);
                logits[row * d.E + e] = s;
            }
        }
        __syncthreads();
    }
}

// The router in a launch of its own: 16 experts and 16 tokens a block, a stretch of the contraction (blockIdx.z), sums [stretch][T][E].
template <bool F32, bool VEC>
__global__ __launch_bounds__(kLogitWaves* kWave) void few_logits_kernel(fmoe_few_desc d, float* part) {
    constexpr int WT = F32 ? kWF32 : kWBF16, CE = Wt<WT>::CE, ES = Wt<WT>::ES, STEP = 4 * CE, U = 4;
    __shared__ f32x4 red[kLogitWaves][kWave];
    const int lane = lane_id(), wave = uniform(threadIdx.x / kWave), r16 = lane & 15, quarter = lane >> 4, e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
    const int steps = (d.D + STEP - 1) / STEP, all = kLogitWaves * gridDim.z, share = blockIdx.z * kLogitWaves + wave;
    const uint32_t xrow = (uint32_t)(min(t0 + r16, d.T - 1) * (int)d.x_stride_row * ES), wrow = (uint32_t)(min(e0 + r16, d.E - 1) * (int)d.gate_stride_row * ES);
    Rows<ES, VEC> x, g;
    x.at(d.x);
    g.at(d.gate_weight);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 2 * share; s0 < steps; s0 += U * all) {
        u32x4 xv[U], wv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (s0 + (u / 2) * 2 * all + (u & 1)) * STEP + quarter * CE;
            xv[u] = x.chunk(xrow, k, d.D);
            wv[u] = g.chunk(wrow, k, d.D);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) mma<WT>(acc, wv[u], &xv[u]);
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && t0 + r16 < d.T) {
#pragma unroll
        for (int w = 1; w < kLogitWaves; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += red[w][lane][i];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = e0 + 4 * quarter + i;
            if (e < d.E) part[((int64_t)blockIdx.z * d.T + t0 + r16) * d.E + e] = acc[i] + (d.gate_bias && blockIdx.z == 0 ? element<F32>(d.gate_bias, e) : 0.0f);
        }
    }
}

// The k experts of one token by one wave, from its logits: descending, equal ones by ascending id.
template <typename Logit>
__device__ __forceinline__ void select_token(const fmoe_few_desc& d, int t, Logit&& logit, const FewLists& l) {
    const int lane = lane_id();
    if (d.token_mask && !d.token_mask[t]) {
        if (lane < d.k) {
            l.sel[t * d.k + lane] = -1;
            l.gate[t * d.k + lane] = 0.0f;
        }
        return;
    }
    constexpr int R = kFewMostExperts / kWave;
    float v[R];
    uint32_t key[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int e = i * kWave + lane;
        v[i] = e < d.E ? logit(e) : 0.0f;
        key[i] = e < d.E ? order_key(v[i]) : 0u;
    }
    float top = 0.0f, mine = -__builtin_inff();
    int expert = 0;
    for (int j = 0; j < d.k; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < R; ++i) best = max(best, key[i]);
        best = wave_max_key(best);
        bool found = false;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (found) continue;
            const unsigned long long hit = __ballot(key[i] == best);
            if (!hit) continue;
            found = true;
            const int at = __builtin_ctzll(hit);
            const float value = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v[i]), at));
            if (lane == at) key[i] = 0u;
            if (j == 0) top = value;
            if (lane == j) {
                expert = i * kWave + at;
                mine = value;
            }
        }
    }
    const float p = lane < d.k ? expf(mine - top) : 0.0f;
    float sum = 0.0f;
    if (d.renorm) {
        sum = p;
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, kWave);      // (k <= 16 lanes hold something)
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i * kWave + lane < d.E) sum += expf(v[i] - top);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    }
    if (lane < d.k) {
        l.sel[t * d.k + lane] = (int16_t)expert;
        l.gate[t * d.k + lane] = p / sum;
    }
}

// Who goes where, from every token's selection: per expert its tokens, the experts that have any, and the items (an expert, up to 16 * NT tokens).
template <int NT>
__device__ __forceinline__ void build_lists(const fmoe_few_desc& d, const FewLists& l) {
    const int lane = lane_id();
    for (int i = threadIdx.x; i < d.T * d.k; i += kWaves * kWave)
        if (l.sel[i] >= 0) atomicOr(&l.mask[l.sel[i]], 1ull << (i / d.k));
    __syncthreads();
    if (threadIdx.x < kWave) {
        int active = 0, rows = 0, items = 0;
        for (int e0 = 0; e0 < d.E; e0 += kWave) {
            const int e = e0 + lane;
            const int n = e < d.E ? __popcll(l.mask[e]) : 0, groups = (n + 16 * NT - 1) / (16 * NT);
            const unsigned long long any = __ballot(n > 0);
            const int a = active + __popcll(any & ((1ull << lane) - 1));
            const int upto = wave_inclusive_scan(n), item = wave_inclusive_scan(groups);
            if (n > 0) {
                l.rank[e] = (int16_t)a;
                l.act[a] = (int16_t)e;
                l.base[a] = (int16_t)(rows + upto - n);
                for (int i = 0; i < groups; ++i) l.item[items + item - groups + i] = (int16_t)(a | i << 14);
            }
            active += __popcll(any);
            rows += __shfl(upto, kWave - 1, kWave);
            items += __shfl(item, kWave - 1, kWave);
        }
        if (lane == 0) {
            l.counts[0] = active;
            l.counts[1] = items;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < d.T * d.k; i += kWaves * kWave)
        if (l.sel[i] >= 0) {
            const int e = l.sel[i];
            l.slots[l.base[l.rank[e]] + __popcll(l.mask[e] & ((1ull << (i / d.k)) - 1))] = (int16_t)i;
        }
    __syncthreads();
}

template <int WT, bool VEC, int NT, bool GATED>
__global__ __launch_bounds__(kWaves* kWave) void few_up_kernel(FewParams p, int share_bits) {
    constexpr bool F32 = WT == kWF32;
    constexpr int CE = Wt<WT>::CE, ES = Wt<WT>::ES, XES = Wt<WT>::XES, XC = Wt<WT>::XC, STEP = 4 * CE, MATS = GATED ? 2 : 1;
    constexpr int AHEAD = !VEC || NT * XC * MATS > 2 ? 2 : 3;    // batches of loads in flight
    constexpr int ROUND = NT == 1 ? MATS : 1;           // matrices whose sums are in LDS at a time
    extern __shared__ uint8_t lds[];
    const fmoe_few_desc& d = p.d;
    const int lane = lane_id(), wave = uniform(threadIdx.x / kWave), r16 = lane & 15, quarter = lane >> 4;
    float* const red = (float*)lds;
    float* const logits = (float*)(lds + kRedBytes);
    uint8_t* const listed = lds + kRedBytes + (p.stretches ? 0 : few_align(16 * d.E * 4));
    const FewLists l = few_lists(listed, d.T, d.E, d.k);
    for (int e = threadIdx.x; e < d.E; e += kWaves * kWave) l.mask[e] = 0;
    if (p.stretches) {          // few_logits has run
        __syncthreads();
        for (int t = wave; t < d.T; t += kWaves)
            select_token(d, t, [&](int e) {
                float v = p.logits[(int64_t)t * d.E + e];
                for (int z = 1; z < p.stretches; ++z) v += p.logits[((int64_t)z * d.T + t) * d.E + e];
                return v;
            }, l);
        __syncthreads();
    } else {
        for (int t0 = 0; t0 < d.T; t0 += 16) {
            router_logits<F32, VEC>(d, t0, red, logits);
            for (int t = wave; t < 16 && t0 + t < d.T; t += kWaves) select_token(d, t0 + t, [&](int e) { return logits[t * d.E + e]; }, l);
            __syncthreads();
        }
    }
    build_lists<NT>(d, l);
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < few_lists_bytes(d.T, d.E, d.k) / 16; i += kWaves * kWave)
            reinterpret_cast<u32x4*>(p.lists)[i] = reinterpret_cast<const u32x4*>(listed)[i];
    // Groups of `shares` waves have an item each and share its contraction in pieces of two steps.
    const int shares = 1 << share_bits, group = wave >> share_bits, share = wave & (shares - 1), groups = kWaves >> share_bits;
    const int tiles = (d.H + 15) / 16, items = uniform(l.counts[1]) * tiles, steps = (d.D + STEP - 1) / STEP;
    const int batches = (steps + 2 * shares - 1) / (2 * shares);       // of two steps a wave
    struct Item {
        int e, n, h0;
        const int16_t* slots;
    };
    auto item = [&](int it) {
        Item at = {0, 0, 0, l.slots};
        if (it < items) {
            const int entry = uniform(l.item[it / tiles]), a = entry & 0x3fff, first = (entry >> 14) * 16 * NT;
            at.h0 = it % tiles * 16;
            at.e = uniform(l.act[a]);
            at.n = uniform(min(16 * NT, (int)__popcll(l.mask[at.e]) - first));
            at.slots = l.slots + uniform(l.base[a]) + first;
        }
        return at;
    };
    const int step = gridDim.x * groups;
    int base = blockIdx.x * groups;         // (the same in all waves: the groups of a block go through the barriers together)
    // What is loaded runs AHEAD batches before what is multiplied, over the ends of items.
    Rows<ES, VEC> w[MATS];
    Rows<XES, VEC> x;
    x.at(d.x);
    uint32_t wrow = 0, xrow[NT];
    int wcols = 0, xcols[NT], load_it = base + group, load_s = 0;
    auto take = [&] {
        const Item at = item(load_it);
        const int64_t from = ((int64_t)at.e * d.w_stride_e + (int64_t)at.h0 * d.w_stride_n) * ES;
        wrow = (uint32_t)(min(r16, d.H - 1 - at.h0) * (int)d.w_stride_n * ES);
        wcols = at.n ? d.D : 0;
        w[0].at((const uint8_t*)d.w + from);
        if constexpr (GATED) w[1].at((const uint8_t*)d.wp + from);
#pragma unroll
        for (int f = 0; f < NT; ++f) {
            const bool live = 16 * f + r16 < at.n;
            xrow[f] = live ? (uint32_t)(at.slots[16 * f + r16] / d.k * (int)d.x_stride_row * XES) : 0u;
            xcols[f] = live ? d.D : 0;
        }
    };
    u32x4 wv[AHEAD][2][MATS], xv[AHEAD][2][NT][XC];
    auto load = [&](u32x4 (&wb)[2][MATS], u32x4 (&xb)[2][NT][XC]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int k = (load_s + 2 * share + u) * STEP + quarter * CE;
#pragma unroll
            for (int m = 0; m < MATS; ++m) wb[u][m] = w[m].chunk(wrow, k, wcols);
#pragma unroll
            for (int f = 0; f < NT; ++f)
#pragma unroll
                for (int c = 0; c < XC; ++c) xb[u][f][c] = x.chunk(xrow[f], k + c * (16 / XES), xcols[f]);
        }
        load_s += 2 * shares;
        if (load_s >= steps) {
            load_s = 0;
            load_it += step;
            take();
        }
    };
    f32x4 acc[MATS][NT];
    auto clear = [&] {
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int f = 0; f < NT; ++f) acc[m][f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };
    take();
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(wv[i], xv[i]);
    clear();
    Item done = item(base + group);
    auto finish = [&] {
        f32x4 sum[MATS][NT];
#pragma unroll
        for (int m0 = 0; m0 < MATS; m0 += ROUND) {
            if (m0 > 0) __syncthreads();
#pragma unroll
            for (int m = 0; m < ROUND; ++m)
#pragma unroll
                for (int f = 0; f < NT; ++f) reinterpret_cast<f32x4*>(red)[((wave * ROUND + m) * NT + f) * kWave + lane] = acc[m0 + m][f];
            __syncthreads();
#pragma unroll
            for (int f = 0; f < NT; ++f)
                if ((f & (shares - 1)) == share && 16 * f < done.n)
#pragma unroll
                    for (int m = 0; m < ROUND; ++m) {
                        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                        for (int w = 0; w < shares; ++w) {
                            const f32x4 part = reinterpret_cast<f32x4*>(red)[(((group * shares + w) * ROUND + m) * NT + f) * kWave + lane];
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] += part[i];
                        }
                        sum[m0 + m][f] = v;
                    }
        }
#pragma unroll
        for (int f = 0; f < NT; ++f) {
            if ((f & (shares - 1)) != share || 16 * f + r16 >= done.n) continue;
            const int slot = done.slots[16 * f + r16];
            const float g = l.gate[slot];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = done.h0 + 4 * quarter + i;
                if (col >= d.H) break;
                float v = sum[0][f][i];
                if constexpr (WT == kWE4M3) v /= d.w_scale[(int64_t)done.e * d.H + col];
                if (d.bias) v += element<F32>(d.bias, (int64_t)done.e * d.bias_stride_e + col);
                v = silu_f32(v);
                if constexpr (GATED) {
                    float u = sum[1][f][i];
                    if constexpr (WT == kWE4M3) u /= d.wp_scale[(int64_t)done.e * d.H + col];
                    if (d.bias_p) u += element<F32>(d.bias_p, (int64_t)done.e * d.bias_stride_e + col);
                    v *= u;
                }
                // bf16: the one rounding between the two products, of the gated value (half a step of bf16, as of the layer's own hidden rows)
                put_element<F32>(p.h, (int64_t)slot * d.H + col, g * v);
            }
        }
        clear();
        base += step;
        done = item(base + group);
        __syncthreads();
    };
    for (int left = batches; base < items;) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (base >= items) break;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int f = 0; f < NT; ++f)
                    if (f == 0 || 16 * f < done.n) {
#pragma unroll
                        for (int m = 0; m < MATS; ++m) mma<WT>(acc[m][f], wv[i][u][m], xv[i][u][f]);
                    }
            load(wv[i], xv[i]);
            if (--left == 0) {
                finish();
                left = batches;
            }
        }
    }
}

// PARTS: a tile has 16 / PARTS output columns, and the MFMAs' rows (and columns: up to 16 / PARTS tokens) hold that many stretches of the
// contraction side by side, of whose products the diagonal blocks count: more, smaller tiles where 16 columns each would leave CUs without one.
template <int WT, bool VEC, int NT, int PARTS>
__global__ __launch_bounds__(kWaves* kWave) void few_down_kernel(FewParams p) {
    constexpr bool F32 = WT == kWF32;
    constexpr int CE = Wt<WT>::CE, ES = Wt<WT>::ES, XES = Wt<WT>::XES, XC = Wt<WT>::XC, STEP = 4 * CE, COLS = 16 / PARTS;
    constexpr int AHEAD = !VEC ? 1 : NT * XC == 1 ? 4 : NT * XC == 2 ? 3 : 2;      // pieces whose loads are in flight
    extern __shared__ uint8_t lds[];
    const fmoe_few_desc& d = p.d;
    const int lane = lane_id(), wave = threadIdx.x / kWave, waves = blockDim.x / kWave, r16 = lane & 15, quarter = lane >> 4;
    float* const sums = (float*)lds;                                        // [waves][T][16]
    uint8_t* const listed = lds + (size_t)waves * d.T * 64;
    const FewLists l = few_lists(listed, d.T, d.E, d.k);
    for (int i = threadIdx.x; i < few_lists_bytes(d.T, d.E, d.k) / 16; i += blockDim.x)
        reinterpret_cast<u32x4*>(listed)[i] = reinterpret_cast<const u32x4*>(p.lists)[i];
    for (int i = threadIdx.x; i < waves * d.T * 4; i += blockDim.x) reinterpret_cast<f32x4*>(sums)[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();
    const int part = r16 / COLS, n0 = blockIdx.x * COLS, row = min(n0 + r16 % COLS, d.O - 1);
    const int steps = (d.H + STEP - 1) / STEP, pieces = (steps + 1) / 2, total = l.counts[1] * pieces;
    // every stretch (a wave's, or a part of its) takes as many pieces of two steps, experts after one another
    const int per = (total + waves * PARTS - 1) / (waves * PARTS), from = (wave * PARTS + part) * per;
    const int until = min(total, from + per);
    struct Entry {
        int index, e, n;
        const int16_t* slots;
    };
    auto entry_of = [&](int index) {
        const int item = l.item[index], a = item & 0x3fff, first = (item >> 14) * 16 * NT;
        Entry en;
        en.index = index;
        en.e = l.act[a];
        en.n = min(16 * NT, (int)__popcll(l.mask[en.e]) - first);
        en.slots = l.slots + l.base[a] + first;
        return en;
    };
    Entry next = {-1, 0, 0, l.slots}, cur = next;       // the expert whose loads are on their way, and whose products add up
    int next_of[AHEAD];
    const uint8_t *wrow = nullptr, *xrow[NT] = {};
    u32x4 wv[AHEAD][2], xv[AHEAD][2][NT][XC];
    int q = from, index = total ? from / pieces : 0, piece = from - index * pieces;
    auto load = [&](int& of, u32x4 (&wb)[2], u32x4 (&xb)[2][NT][XC]) {
        const bool any = q < until;
        of = any ? index : next.index;
        if (any && index != next.index) {
            next = entry_of(index);
            wrow = (const uint8_t*)d.wo + ((int64_t)next.e * d.wo_stride_e + (int64_t)row * d.wo_stride_n) * ES;
#pragma unroll
            for (int f = 0; f < NT; ++f) {
                const int c = 16 * f + r16 % COLS;
                xrow[f] = c < next.n ? (const uint8_t*)p.h + (int64_t)next.slots[c] * d.H * XES : nullptr;
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int k = (2 * piece + s) * STEP + quarter * CE;
            wb[s] = chunk<ES, VEC>(wrow, k, any ? d.H : 0);
#pragma unroll
            for (int f = 0; f < NT; ++f)
#pragma unroll
                for (int c = 0; c < XC; ++c) xb[s][f][c] = chunk<XES, VEC>(xrow[f], k + c * (16 / XES), any && xrow[f] ? d.H : 0);
        }
        ++q;
        if (++piece == pieces) {
            piece = 0;
            ++index;
        }
    };
    f32x4 acc[NT];
#pragma unroll
    for (int f = 0; f < NT; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // An expert's products go to its own tokens' sums, and only there (a column without a token holds zeros, which an infinity among the weights
    // turns into NaN).
    auto flush = [&] {
        if (cur.index >= 0) {
            f32x4 inv = {1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (WT == kWE4M3) {
#pragma unroll
                for (int i = 0; i < 4; ++i) inv[i] = 1.0f / d.wo_scale[(int64_t)cur.e * d.O + min(n0 + (4 * quarter + i) % COLS, d.O - 1)];
            }
#pragma unroll
            for (int f = 0; f < NT; ++f) {
                const int c = 16 * f + r16 % COLS;
                if (c < cur.n && quarter * 4 / COLS == part) {
                    f32x4* const to = reinterpret_cast<f32x4*>(sums + ((size_t)wave * d.T + cur.slots[c] / d.k) * 16 + 4 * quarter);
                    f32x4 v = *to;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] += acc[f][i] * inv[i];
                    *to = v;
                }
            }
        }
#pragma unroll
        for (int f = 0; f < NT; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(next_of[i], wv[i], xv[i]);
    for (int done = 0; done < per; done += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {       // (behind a stretch's last piece come zeros)
            if (__any(next_of[i] != cur.index)) {
                flush();
                if (next_of[i] >= 0) cur = entry_of(next_of[i]);
            }
#pragma unroll
            for (int f = 0; f < NT; ++f)
                if (f == 0 || 16 * f < cur.n) {
                    mma<WT>(acc[f], wv[i][0], xv[i][0][f]);
                    mma<WT>(acc[f], wv[i][1], xv[i][1][f]);
                }
            load(next_of[i], wv[i], xv[i]);
        }
    }
    flush();
    __syncthreads();
    for (int i = threadIdx.x; i < d.T * COLS; i += blockDim.x) {
        const int t = i / COLS, c = i % COLS, col = n0 + c;
        if (col >= d.O) continue;
        float v = 0.0f;
        for (int w = 0; w < waves; ++w)
#pragma unroll
            for (int q2 = 0; q2 < PARTS; ++q2) v += sums[((size_t)w * d.T + t) * 16 + q2 * COLS + c];
        if (d.bias_out)
            for (int j = 0; j < d.k; ++j) {
                const int e = l.sel[t * d.k + j];
                if (e >= 0) v += l.gate[t * d.k + j] * element<F32>(d.bias_out, (int64_t)e * d.bias_out_stride_e + col);
            }
        put_element<F32>(d.out, (int64_t)t * d.out_stride_row + col, v);
    }
}

// The workspace: the lists as few_up's first block leaves them, and the hidden rows.
size_t few_hidden_at(const fmoe_few_desc& d) { return ((size_t)few_lists_bytes(d.T, d.E, d.k) + 255) & ~(size_t)255; }
size_t few_logits_at(const fmoe_few_desc& d) { return (few_hidden_at(d) + (size_t)d.T * d.k * d.H * (d.dtype == FMOE_F32 ? 4 : 2) + 255) & ~(size_t)255; }
// Stretches of the router's own launch, 0 where few_up computes the router.
int few_stretches(const fmoe_few_desc& d) {
    if ((int64_t)d.E * d.D * (d.dtype == FMOE_F32 ? 4 : 2) * ((d.T + 15) / 16) <= 32 * 1024) return 0;
    return d.T <= 16 ? 4 : 1;
}
size_t few_bytes(const fmoe_few_desc& d) { return few_logits_at(d) + (size_t)few_stretches(d) * d.T * d.E * 4; }

int few_check(const fmoe_few_desc* d) {
    FMOE_REQUIRE(d, "fmoe_few_tokens: desc is NULL");
    FMOE_REQUIRE(d->T >= 0 && d->T <= kFewMostTokens, "fmoe_few_tokens: up to %d tokens, got T=%d", kFewMostTokens, d->T);
    FMOE_REQUIRE(d->E >= 1 && d->E <= kFewMostExperts && d->k >= 1 && d->k <= kFewMostK && d->k <= d->E,
                 "fmoe_few_tokens: need 1 <= k <= E, k <= %d, E <= %d, got k=%d E=%d", kFewMostK, kFewMostExperts, d->k, d->E);
    FMOE_REQUIRE(d->D >= 1 && d->H >= 1 && d->O >= 1 && d->D <= kFewMostWidth && d->H <= kFewMostWidth && d->O <= kFewMostWidth,
                 "fmoe_few_tokens: widths of 1 to %d expected", kFewMostWidth);
    FMOE_REQUIRE(d->dtype == FMOE_F32 || d->dtype == FMOE_BF16, "fmoe_few_tokens: tokens must be bf16 or fp32");
    FMOE_REQUIRE(d->weight_dtype == d->dtype || (d->weight_dtype == FMOE_E4M3 && d->dtype == FMOE_BF16),
                 "fmoe_few_tokens: weights must have the tokens' type, or be e4m3 with bf16 tokens");
    if (d->T == 0) return FMOE_OK;
    FMOE_REQUIRE(d->x && d->gate_weight && d->w && d->wo && d->out, "fmoe_few_tokens: NULL tensor pointer");
    FMOE_REQUIRE(d->weight_dtype != FMOE_E4M3 || (d->w_scale && d->wo_scale && (!d->wp || d->wp_scale)), "fmoe_few_tokens: e4m3 weights need their scales");
    FMOE_REQUIRE(d->wp || !d->bias_p, "fmoe_few_tokens: bias_p goes with wp");
    FMOE_REQUIRE(d->x_stride_row >= (d->T > 1 ? d->D : 0) && d->gate_stride_row >= (d->E > 1 ? d->D : 0) && d->out_stride_row >= (d->T > 1 ? d->O : 0) &&
                     d->w_stride_n >= (d->H > 1 ? d->D : 0) && d->wo_stride_n >= (d->O > 1 ? d->H : 0) && d->w_stride_e >= 0 && d->wo_stride_e >= 0,
                 "fmoe_few_tokens: rows overlap");
    // (offsets of rows from their tile's first are 31 bits of bytes)
    FMOE_REQUIRE(d->x_stride_row <= kFewMostStride && d->gate_stride_row <= kFewMostStride && d->w_stride_n <= kFewMostStride &&
                     d->wo_stride_n <= kFewMostStride,
                 "fmoe_few_tokens: row strides of up to %d elements expected", kFewMostStride);
    return FMOE_OK;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" size_t fmoe_few_tokens_workspace_bytes(const fmoe_few_desc* d) {
    if (few_check(d) != FMOE_OK || d->T == 0) return 0;
    return few_bytes(*d);
}

extern "C" int fmoe_few_tokens(const fmoe_few_desc* desc, void* workspace, size_t workspace_bytes, fmoe_stream_t stream_) {
    const int rc = few_check(desc);
    if (rc != FMOE_OK || desc->T == 0) return rc;
    const fmoe_few_desc& d = *desc;
    const size_t need = few_bytes(d);
    if (!workspace || workspace_bytes < need)
        return fail(FMOE_ERR_WORKSPACE, "fmoe_few_tokens: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    FMOE_REQUIRE(aligned16(workspace), "fmoe_few_tokens: the workspace must be 16-byte aligned");
    const FewParams p{d, workspace, (uint8_t*)workspace + few_hidden_at(d), (const float*)((uint8_t*)workspace + few_logits_at(d)), few_stretches(d)};
    const int es = d.dtype == FMOE_F32 ? 4 : 2, wes = d.weight_dtype == FMOE_E4M3 ? 1 : es;
    // whole 16-byte chunks at 16-byte boundaries wherever rows are read
    auto whole = [](const void* q, int64_t elements, int size) { return aligned16(q) && elements * size % 16 == 0; };
    const bool vec = whole(d.x, d.D, es) && whole(d.x, d.x_stride_row, es) && whole(d.gate_weight, d.gate_stride_row, es) && whole(d.w, d.D, wes) &&
                     whole(d.w, d.w_stride_n, wes) && whole(d.w, d.w_stride_e, wes) && whole(d.wp, d.D, wes) && whole(d.wo, d.H, wes) &&
                     whole(d.wo, d.wo_stride_n, wes) && whole(d.wo, d.wo_stride_e, wes) && d.H * es % 16 == 0;
    const bool gated = d.wp != nullptr;
    const int most_active = d.T * d.k < d.E ? d.T * d.k : d.E;
    hipStream_t stream = (hipStream_t)stream_;
    const int lists = few_lists_bytes(d.T, d.E, d.k), step = wes == 1 ? 64 : 64 / wes;
    // waves to an item: four steps each where the rows are that long
    int share_bits = 0;
    while (share_bits < 4 && (4 << share_bits) * step < d.D) ++share_bits;
    auto up = [&](auto kern, int nt) {
        const int64_t items = (int64_t)most_active * ((d.H + 15) / 16) * (nt == 2 && d.T > 32 ? 2 : 1), blocks = (items + (kWaves >> share_bits) - 1) / (kWaves >> share_bits);
        kern<<<(unsigned)(blocks < 256 ? blocks : 256), kWaves * kWave, kRedBytes + (p.stretches ? 0 : few_align(16 * d.E * 4)) + lists, stream>>>(p, share_bits);
    };
    auto down = [&](auto kern, int parts) {
        const int cols = 16 / parts, waves = d.T > 32 ? kWaves / 2 : kWaves;        // (their sums for 64 tokens in 64 KB of LDS)
        kern<<<(unsigned)((d.O + cols - 1) / cols), waves * kWave, waves * d.T * 64 + lists, stream>>>(p);
    };
    const int parts = d.O >= 16 * 256 || d.T > 8 ? 1 : d.O >= 8 * 256 || d.T > 4 ? 2 : 4;
#define FMOE_FEW_UP(WT, VEC, NT) (gated ? up(few_up_kernel<WT, VEC, NT, true>, NT) : up(few_up_kernel<WT, VEC, NT, false>, NT))
#define FMOE_FEW(WT, VEC)                                                   \
    do {                                                                    \
        if (p.stretches) {                                                  \
            few_logits_kernel<WT == kWF32, VEC><<<dim3((d.E + 15) / 16, (d.T + 15) / 16, p.stretches), kLogitWaves * kWave, 0, stream>>>(d, const_cast<float*>(p.logits)); \
            const int first = check_launch("fmoe_few_tokens");              \
            if (first != FMOE_OK) return first;                             \
        }                                                                   \
        if (d.T <= 16) FMOE_FEW_UP(WT, VEC, 1); else FMOE_FEW_UP(WT, VEC, 2); \
        const int launched = check_launch("fmoe_few_tokens");               \
        if (launched != FMOE_OK) return launched;                           \
        if (d.T > 16) down(few_down_kernel<WT, VEC, 2, 1>, 1);              \
        else if (parts == 1) down(few_down_kernel<WT, VEC, 1, 1>, 1);       \
        else if (parts == 2) down(few_down_kernel<WT, VEC, 1, 2>, 2);       \
        else down(few_down_kernel<WT, VEC, 1, 4>, 4);                       \
    } while (0)
    if (d.weight_dtype == FMOE_F32) {
        if (vec) FMOE_FEW(kWF32, true); else FMOE_FEW(kWF32, false);
    } else if (d.weight_dtype == FMOE_BF16) {
        if (vec) FMOE_FEW(kWBF16, true); else FMOE_FEW(kWBF16, false);
    } else {
        if (vec) FMOE_FEW(kWE4M3, true); else FMOE_FEW(kWE4M3, false);
    }
#undef FMOE_FEW
#undef FMOE_FEW_UP
    return check_launch("fmoe_few_tokens");
}
