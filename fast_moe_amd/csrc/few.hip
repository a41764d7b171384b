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

constexpr int kFewMostTokens = 64, kFewMostExperts = 256, kFewMostK = 16;
constexpr int kUpWaves = 8, kDownWaves = 16;
constexpr int kRouterRow = 64 + 4;      // floats of a token's sums over 64 experts (the 4: other banks for the next token)

struct FewParams {
    fmoe_few_desc d;
    // the workspace: routing as few_up's first block leaves it, and the hidden rows [T * k][H]
    int32_t* count;         // experts with a token
    int32_t* act;           // [E] their ids, ascending
    uint64_t* mask;         // [E] their tokens
    int32_t* sel;           // [T * k] rank of the expert, -1: none
    float* gate;            // [T * k]
    void* h;
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
__host__ __device__ constexpr int few_router_floats() { return kUpWaves * 16 * kRouterRow; }
__host__ __device__ constexpr int few_up_floats(int mats, int nt) { return kUpWaves * mats * nt * 256; }

// Logits of tokens t0 .. t0 + 15 into LDS [16][E]: 64 experts at a time, the waves share the contraction in pieces of 128 bytes per row
// (whole cache lines) and their sums are added in wave order.
template <bool F32, bool VEC>
__device__ __forceinline__ void router_logits(const fmoe_few_desc& d, int t0, float* red, float* logits) {
    constexpr int WT = F32 ? kWF32 : kWBF16, CE = Wt<WT>::CE, ES = Wt<WT>::ES, STEP = 4 * CE, U = 4;
    const int lane = lane_id(), wave = threadIdx.x / kWave, r16 = lane & 15, quarter = lane >> 4;
    const int t = t0 + r16 < d.T ? t0 + r16 : d.T - 1;
    const uint8_t* const xrow = (const uint8_t*)d.x + (int64_t)t * d.x_stride_row * ES;
    const int steps = (d.D + STEP - 1) / STEP;
    for (int e0 = 0; e0 < d.E; e0 += 64) {
        const int tiles = min(4, (d.E - e0 + 15) / 16);
        const uint8_t* wrow[4];
#pragma unroll
        for (int f = 0; f < 4; ++f)
            wrow[f] = (const uint8_t*)d.gate_weight + (int64_t)min(e0 + 16 * f + r16, d.E - 1) * d.gate_stride_row * ES;
        f32x4 acc[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s0 = 2 * wave; s0 < steps; s0 += 2 * kUpWaves * (U / 2)) {
            u32x4 xv[U], wv[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (s0 + (u / 2) * 2 * kUpWaves + (u & 1)) * STEP + quarter * CE;
                xv[u] = chunk<ES, VEC>(xrow, k, d.D);
#pragma unroll
                for (int f = 0; f < 4; ++f)
                    if (f < tiles) wv[u][f] = chunk<ES, VEC>(wrow[f], k, d.D);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int f = 0; f < 4; ++f)
                    if (f < tiles) mma<WT>(acc[f], wv[u][f], &xv[u]);
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) *reinterpret_cast<f32x4*>(red + (wave * 16 + r16) * kRouterRow + 16 * f + 4 * quarter) = acc[f];
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * 64; i += kUpWaves * kWave) {
            const int row = i >> 6, e = e0 + (i & 63);
            if (e < d.E) {
                float s = red[row * kRouterRow + (i & 63)];
#pragma unroll
                for (int w = 1; w < kUpWaves; ++w) s += red[(w * 16 + row) * kRouterRow + (i & 63)];
                if (d.gate_bias) s += element<F32>(d.gate_bias, e);
                logits[row * d.E + e] = s;
            }
        }
        __syncthreads();
    }
}

// The k experts of one token by one wave: descending logit, equal ones by ascending id.
__device__ __forceinline__ void select_token(const fmoe_few_desc& d, int t, const float* logits, const FewLists& l) {
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
        v[i] = e < d.E ? logits[e] : 0.0f;
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
    for (int i = threadIdx.x; i < d.T * d.k; i += kUpWaves * kWave)
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
    for (int i = threadIdx.x; i < d.T * d.k; i += kUpWaves * kWave)
        if (l.sel[i] >= 0) {
            const int e = l.sel[i];
            l.slots[l.base[l.rank[e]] + __popcll(l.mask[e] & ((1ull << (i / d.k)) - 1))] = (int16_t)i;
        }
    __syncthreads();
}

template <int WT, bool VEC, int NT, bool GATED>
__global__ __launch_bounds__(kUpWaves* kWave) __attribute__((amdgpu_waves_per_eu(4))) void few_up_kernel(FewParams p) {
    constexpr bool F32 = WT == kWF32;
    constexpr int CE = Wt<WT>::CE, ES = Wt<WT>::ES, XES = Wt<WT>::XES, XC = Wt<WT>::XC, STEP = 4 * CE, MATS = GATED ? 2 : 1;
    constexpr int U = NT == 1 ? 4 : 2;      // steps whose loads are in flight
    extern __shared__ uint8_t lds[];
    const fmoe_few_desc& d = p.d;
    const int lane = lane_id(), wave = threadIdx.x / kWave, r16 = lane & 15, quarter = lane >> 4;
    float* const red = (float*)lds;
    constexpr int kRed = (few_router_floats() > few_up_floats(MATS, NT) ? few_router_floats() : few_up_floats(MATS, NT)) * 4;
    float* const logits = (float*)(lds + kRed);
    const FewLists l = few_lists(lds + kRed + few_align(16 * d.E * 4), d.T, d.E, d.k);
    for (int e = threadIdx.x; e < d.E; e += kUpWaves * kWave) l.mask[e] = 0;
    for (int t0 = 0; t0 < d.T; t0 += 16) {
        router_logits<F32, VEC>(d, t0, red, logits);
        for (int t = wave; t < 16 && t0 + t < d.T; t += kUpWaves) select_token(d, t0 + t, logits + t * d.E, l);
        __syncthreads();
    }
    build_lists<NT>(d, l);
    const int active = l.counts[0];
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < d.T * d.k; i += kUpWaves * kWave) {
            p.sel[i] = l.sel[i] >= 0 ? l.rank[l.sel[i]] : -1;
            p.gate[i] = l.gate[i];
        }
        for (int a = threadIdx.x; a < active; a += kUpWaves * kWave) {
            p.act[a] = l.act[a];
            p.mask[a] = l.mask[l.act[a]];
        }
        if (threadIdx.x == 0) *p.count = active;
    }
    const int tiles = (d.H + 15) / 16, items = l.counts[1] * tiles, steps = (d.D + STEP - 1) / STEP;
    for (int it = blockIdx.x; it < items; it += gridDim.x) {
        const int entry = l.item[it / tiles], a = entry & 0x3fff, first = (entry >> 14) * 16 * NT, h0 = it % tiles * 16;
        const int e = l.act[a], n = min(16 * NT, (int)__popcll(l.mask[e]) - first);
        const int16_t* const slots = l.slots + l.base[a] + first;
        const int row = min(h0 + r16, d.H - 1);
        const uint8_t* wrow[MATS];
        wrow[0] = (const uint8_t*)d.w + ((int64_t)e * d.w_stride_e + (int64_t)row * d.w_stride_n) * ES;
        if constexpr (GATED) wrow[1] = (const uint8_t*)d.wp + ((int64_t)e * d.w_stride_e + (int64_t)row * d.w_stride_n) * ES;
        const uint8_t* xrow[NT];
        int xn[NT];
#pragma unroll
        for (int f = 0; f < NT; ++f) {
            const bool in = 16 * f + r16 < n;
            xn[f] = in ? d.D : 0;
            xrow[f] = (const uint8_t*)d.x + (in ? (int64_t)(slots[16 * f + r16] / d.k) * d.x_stride_row * XES : 0);
        }
        f32x4 acc[MATS][NT];
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int f = 0; f < NT; ++f) acc[m][f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s0 = 2 * wave; s0 < steps; s0 += kUpWaves * U) {
            u32x4 wv[U][MATS], xv[U][NT][XC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (s0 + (u / 2) * 2 * kUpWaves + (u & 1)) * STEP + quarter * CE;
#pragma unroll
                for (int m = 0; m < MATS; ++m) wv[u][m] = chunk<ES, VEC>(wrow[m], k, d.D);
#pragma unroll
                for (int f = 0; f < NT; ++f)
#pragma unroll
                    for (int c = 0; c < XC; ++c) xv[u][f][c] = chunk<XES, VEC>(xrow[f], k + c * (16 / XES), xn[f]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int f = 0; f < NT; ++f)
                    if (f == 0 || 16 * f < n) {
#pragma unroll
                        for (int m = 0; m < MATS; ++m) mma<WT>(acc[m][f], wv[u][m], xv[u][f]);
                    }
        }
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int f = 0; f < NT; ++f) reinterpret_cast<f32x4*>(red)[((wave * MATS + m) * NT + f) * kWave + lane] = acc[m][f];
        __syncthreads();
        if (wave < NT && 16 * wave + r16 < n) {
            f32x4 sum[MATS];
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                sum[m] = reinterpret_cast<f32x4*>(red)[(m * NT + wave) * kWave + lane];
#pragma unroll
                for (int w = 1; w < kUpWaves; ++w) {
                    const f32x4 v = reinterpret_cast<f32x4*>(red)[((w * MATS + m) * NT + wave) * kWave + lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[m][i] += v[i];
                }
            }
            const int slot = slots[16 * wave + r16];
            const float g = l.gate[slot];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = h0 + 4 * quarter + i;
                if (col >= d.H) break;
                float v = sum[0][i];
                if constexpr (WT == kWE4M3) v /= d.w_scale[(int64_t)e * d.H + col];
                if (d.bias) v += element<F32>(d.bias, (int64_t)e * d.bias_stride_e + col);
                v = silu_f32(v);
                if constexpr (GATED) {
                    float u = sum[1][i];
                    if constexpr (WT == kWE4M3) u /= d.wp_scale[(int64_t)e * d.H + col];
                    if (d.bias_p) u += element<F32>(d.bias_p, (int64_t)e * d.bias_stride_e + col);
                    v *= u;
                }
                // bf16: the one rounding between the two products, of the gated value (half a step of bf16, as of the layer's own hidden rows)
                put_element<F32>(p.h, (int64_t)slot * d.H + col, g * v);
            }
        }
        __syncthreads();
    }
}

template <int WT, bool VEC, int NT>
__global__ __launch_bounds__(kDownWaves* kWave) void few_down_kernel(FewParams p) {
    constexpr bool F32 = WT == kWF32;
    constexpr int CE = Wt<WT>::CE, ES = Wt<WT>::ES, XES = Wt<WT>::XES, XC = Wt<WT>::XC, STEP = 4 * CE, U = NT == 4 ? 2 : 4;
    extern __shared__ uint8_t lds[];
    const fmoe_few_desc& d = p.d;
    const int lane = lane_id(), wave = threadIdx.x / kWave, r16 = lane & 15, quarter = lane >> 4;
    f32x4* const red = (f32x4*)lds;                                 // [waves][lanes]
    int16_t* const slot_of = (int16_t*)(lds + kDownWaves * kWave * 16);        // [active][16 * NT] slot of a token at an expert, -1: none
    const int active = *p.count;
    for (int i = threadIdx.x; i < active * 16 * NT; i += kDownWaves * kWave) slot_of[i] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < d.T * d.k; i += kDownWaves * kWave) {
        const int a = p.sel[i];
        if (a >= 0) slot_of[a * 16 * NT + i / d.k] = (int16_t)i;
    }
    __syncthreads();
    const int n0 = blockIdx.x * 16, row = min(n0 + r16, d.O - 1);
    const int steps = (d.H + STEP - 1) / STEP, pieces = (steps + 1) / 2, total = active * pieces;
    f32x4 acc[NT];
#pragma unroll
    for (int f = 0; f < NT; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int q0 = wave; q0 < total; q0 += kDownWaves * (U / 2)) {
        u32x4 wv[U], xv[U][NT][XC];
        uint64_t mask[U / 2];
        f32x4 inv[U / 2];
#pragma unroll
        for (int u = 0; u < U / 2; ++u) {
            const int q = q0 + u * kDownWaves;
            mask[u] = 0;
            if (q >= total) continue;
            const int a = q / pieces, piece = q - a * pieces;
            const int e = p.act[a];
            mask[u] = p.mask[a];
            const uint8_t* const wrow = (const uint8_t*)d.wo + ((int64_t)e * d.wo_stride_e + (int64_t)row * d.wo_stride_n) * ES;
            if constexpr (WT == kWE4M3) {
#pragma unroll
                for (int i = 0; i < 4; ++i) inv[u][i] = 1.0f / d.wo_scale[(int64_t)e * d.O + min(n0 + 4 * quarter + i, d.O - 1)];
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k = (2 * piece + s) * STEP + quarter * CE;
                wv[2 * u + s] = chunk<ES, VEC>(wrow, k, d.H);
#pragma unroll
                for (int f = 0; f < NT; ++f) {
                    const int slot = slot_of[a * 16 * NT + 16 * f + r16];
                    const uint8_t* const hrow = (const uint8_t*)p.h + (slot < 0 ? 0 : (int64_t)slot * d.H * XES);
#pragma unroll
                    for (int c = 0; c < XC; ++c) xv[2 * u + s][f][c] = chunk<XES, VEC>(hrow, k + c * (16 / XES), slot < 0 ? 0 : d.H);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U / 2; ++u)
#pragma unroll
            for (int f = 0; f < NT; ++f) {
                const uint32_t here = (uint32_t)(mask[u] >> (16 * f)) & 0xffff;
                if (!here) continue;
                f32x4 part = {0.0f, 0.0f, 0.0f, 0.0f};
                mma<WT>(part, wv[2 * u], xv[2 * u][f]);
                mma<WT>(part, wv[2 * u + 1], xv[2 * u + 1][f]);
                // (a token that is not the expert's has zeros in its column, which an infinity among the weights would make a NaN)
                const bool routed = here >> r16 & 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (WT == kWE4M3) part[i] *= inv[u][i];
                    acc[f][i] += routed ? part[i] : 0.0f;
                }
            }
    }
#pragma unroll
    for (int f = 0; f < NT; ++f) {
        if (f > 0) __syncthreads();
        red[wave * kWave + lane] = acc[f];
        __syncthreads();
        const int t = 16 * f + r16;
        if (wave == 0 && t < d.T) {
            f32x4 sum = red[lane];
#pragma unroll
            for (int w = 1; w < kDownWaves; ++w) {
                const f32x4 v = red[w * kWave + lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] += v[i];
            }
            if (d.bias_out)
                for (int j = 0; j < d.k; ++j) {
                    const int a = p.sel[t * d.k + j];
                    if (a < 0) continue;
                    const float g = p.gate[t * d.k + j];
                    for (int i = 0; i < 4; ++i) {
                        const int col = n0 + 4 * quarter + i;
                        if (col < d.O) sum[i] += g * element<F32>(d.bias_out, (int64_t)p.act[a] * d.bias_out_stride_e + col);
                    }
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = n0 + 4 * quarter + i;
                if (col < d.O) put_element<F32>(d.out, (int64_t)t * d.out_stride_row + col, sum[i]);
            }
        }
    }
}

struct FewLayout {
    size_t act, mask, sel, gate, h, end;
};
FewLayout few_layout(const fmoe_few_desc& d) {
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    FewLayout l;
    l.mask = 256;                                                   // (the count first)
    l.act = up(l.mask + (size_t)d.E * 8);
    l.sel = up(l.act + (size_t)d.E * 4);
    l.gate = up(l.sel + (size_t)d.T * d.k * 4);
    l.h = up(l.gate + (size_t)d.T * d.k * 4);
    l.end = up(l.h + (size_t)d.T * d.k * d.H * (d.dtype == FMOE_F32 ? 4 : 2));
    return l;
}

int few_check(const fmoe_few_desc* d) {
    FMOE_REQUIRE(d, "fmoe_few_tokens: desc is NULL");
    FMOE_REQUIRE(d->T >= 0 && d->T <= kFewMostTokens, "fmoe_few_tokens: up to %d tokens, got T=%d", kFewMostTokens, d->T);
    FMOE_REQUIRE(d->E >= 1 && d->E <= kFewMostExperts && d->k >= 1 && d->k <= kFewMostK && d->k <= d->E,
                 "fmoe_few_tokens: need 1 <= k <= E, k <= %d, E <= %d, got k=%d E=%d", kFewMostK, kFewMostExperts, d->k, d->E);
    FMOE_REQUIRE(d->D >= 1 && d->H >= 1 && d->O >= 1 && d->D <= (1 << 24) && d->H <= (1 << 24) && d->O <= (1 << 24),
                 "fmoe_few_tokens: widths of 1 to 2^24 expected");
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
    return FMOE_OK;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" size_t fmoe_few_tokens_workspace_bytes(const fmoe_few_desc* d) {
    if (few_check(d) != FMOE_OK || d->T == 0) return 0;
    return few_layout(*d).end;
}

extern "C" int fmoe_few_tokens(const fmoe_few_desc* desc, void* workspace, size_t workspace_bytes, fmoe_stream_t stream_) {
    const int rc = few_check(desc);
    if (rc != FMOE_OK || desc->T == 0) return rc;
    const fmoe_few_desc& d = *desc;
    const FewLayout at = few_layout(d);
    if (!workspace || workspace_bytes < at.end)
        return fail(FMOE_ERR_WORKSPACE, "fmoe_few_tokens: workspace of %zu bytes, %zu needed", workspace_bytes, at.end);
    FMOE_REQUIRE(aligned16(workspace), "fmoe_few_tokens: the workspace must be 16-byte aligned");
    uint8_t* const ws = (uint8_t*)workspace;
    FewParams p{d, (int32_t*)ws, (int32_t*)(ws + at.act), (uint64_t*)(ws + at.mask), (int32_t*)(ws + at.sel), (float*)(ws + at.gate), ws + at.h};
    const int es = d.dtype == FMOE_F32 ? 4 : 2, wes = d.weight_dtype == FMOE_E4M3 ? 1 : es;
    // whole 16-byte chunks at 16-byte boundaries wherever rows are read
    auto whole = [](const void* q, int64_t elements, int size) { return aligned16(q) && elements * size % 16 == 0; };
    const bool vec = whole(d.x, d.D, es) && whole(d.x, d.x_stride_row, es) && whole(d.gate_weight, d.gate_stride_row, es) && whole(d.w, d.D, wes) &&
                     whole(d.w, d.w_stride_n, wes) && whole(d.w, d.w_stride_e, wes) && whole(d.wp, d.D, wes) && whole(d.wo, d.H, wes) &&
                     whole(d.wo, d.wo_stride_n, wes) && whole(d.wo, d.wo_stride_e, wes) && d.H * es % 16 == 0;
    const bool gated = d.wp != nullptr;
    const int most_active = d.T * d.k < d.E ? d.T * d.k : d.E;
    hipStream_t stream = (hipStream_t)stream_;
    auto up = [&](auto kern, int mats, int nt) {
        const int floats = few_router_floats() > few_up_floats(mats, nt) ? few_router_floats() : few_up_floats(mats, nt);
        const int64_t items = (int64_t)most_active * ((d.H + 15) / 16) * (nt == 2 && d.T > 32 ? 2 : 1);
        const unsigned grid = (unsigned)(items < 512 ? items : 512);
        kern<<<grid, kUpWaves * kWave, floats * 4 + few_align(16 * d.E * 4) + few_lists_bytes(d.T, d.E, d.k), stream>>>(p);
    };
    auto down = [&](auto kern, int nt) {
        kern<<<(unsigned)((d.O + 15) / 16), kDownWaves * kWave, kDownWaves * kWave * 16 + few_align(most_active * 16 * nt * 2), stream>>>(p);
    };
#define FMOE_FEW_UP(WT, VEC, NT) (gated ? up(few_up_kernel<WT, VEC, NT, true>, 2, NT) : up(few_up_kernel<WT, VEC, NT, false>, 1, NT))
#define FMOE_FEW(WT, VEC)                                                   \
    do {                                                                    \
        if (d.T <= 16) FMOE_FEW_UP(WT, VEC, 1); else FMOE_FEW_UP(WT, VEC, 2); \
        const int launched = check_launch("fmoe_few_tokens");               \
        if (launched != FMOE_OK) return launched;                           \
        if (d.T <= 16) down(few_down_kernel<WT, VEC, 1>, 1);                \
        else if (d.T <= 32) down(few_down_kernel<WT, VEC, 2>, 2);           \
        else down(few_down_kernel<WT, VEC, 4>, 4);                          \
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
