// fmoe_few_tokens: a whole mixture-of-experts layer for a few tokens (a decode step) in two launches, three where the gate is large.
//
//   l[t, :] = x[t] . G[e] + bg[e];   the k largest l of a token are its experts, g = softmax of l over them (or over all)
//   h[t, j] = g[t, j] * silu(x[t] . W[e] + b[e]) (* (x[t] . Wp[e] + bp[e]))             e = the token's j-th expert
//   y[t]    = sum_j h[t, j] . Wo[e] + g[t, j] * bo[e]
//
// What bounds it are the bytes of the experts hit, each to be read once: 2 * T flops a byte leave the matrix cores idle.  So the
// weights go from memory to the MFMAs' registers with nothing in between (no LDS, no other wave reads them), and everything else
// is kept out of their way:
//   few_logits  the router's products, where the gate is more than what every CU reads for itself in the time of a launch
//   few_up      every block selects for itself (the same logits, so the same experts everywhere), then takes (expert, 16 hidden columns)
//               items; its waves share the contraction and meet in LDS.  An expert's tokens are gathered into the MFMAs' columns.
//   few_down    a block owns 16 output columns for all tokens; its waves share the experts and their contraction.  The gate is folded into h, so
//               the experts' products add up in one sum.  Where there are few output columns several blocks share them, and the last one
//               to arrive adds their sums in block order: the same bits every time.
// Measured, whole passes: 16 tokens (12 of them live), 128 experts of 4096 x 1536 bf16, 2.6 GB 437 us, 6.0 TB/s; 4 tokens, the same in e4m3, 0.55 GB 117 us,
// 4.7 TB/s; 1 token, 64 experts of 2048 x 1408 bf16, 0.14 GB 40 us, 3.5 TB/s; 37 tokens, 12 experts of 1000 x 2600 fp32, 0.25 GB 89 us, 2.8 TB/s;
// 1 token, 128 x 256, 14 us.  (A 1 GiB copy: 5.2 TB/s.)  Some 12 us of each are the launches, the selection, a first load's way to memory, twice, and the last sums.
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
    void* h;                // hidden rows [T * k][H]; of bf16 two planes of them, whose sum they are
    const float* logits;    // [stretches][T][E]
    int stretches;          // of the router's own launch, 0: the router is few_up's
    int tiles;              // of few_down that several blocks share, or 0
    int32_t* arrivals;      // [tiles of few_down] blocks of a tile that have left their sums
    float* partial;
};

enum { kWF32 = 0, kWBF16 = 1, kWE4M3 = 2, kWE4M3Half = 3 };       // Half: rows of e4m3 that are whole chunks of 8 bytes only

// Elements of a lane's chunk (16 bytes, 8 for Half), bytes of an element, and 16-byte chunks of x that go with one of weights
template <int WT> struct Wt;
template <> struct Wt<kWF32> { static constexpr int CE = 4, ES = 4, XES = 4, XC = 1; };
template <> struct Wt<kWBF16> { static constexpr int CE = 8, ES = 2, XES = 2, XC = 1; };
template <> struct Wt<kWE4M3> { static constexpr int CE = 16, ES = 1, XES = 2, XC = 2; };
template <> struct Wt<kWE4M3Half> { static constexpr int CE = 8, ES = 1, XES = 2, XC = 1; };

// A chunk (BYTES: 16 or 8) of a row of n elements of ES bytes from element k on, zeros behind its end.  VEC: rows are whole chunks at its boundaries.
template <int ES, bool VEC, int BYTES = 16>
__device__ __forceinline__ u32x4 chunk(const uint8_t* row, int k, int n) {
    u32x4 v = {0, 0, 0, 0};
    if constexpr (VEC && BYTES == 8) {
        if (k < n) {
            const u32x2 h = *reinterpret_cast<const u32x2*>(row + (int64_t)k * ES);
            v = u32x4{h[0], h[1], 0, 0};
        }
    } else if constexpr (VEC) {
        if (k < n) v = *reinterpret_cast<const u32x4*>(row + (int64_t)k * ES);
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / ES; ++i) {
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
template <int ES, bool VEC, int BYTES = 16>
struct Rows {
    const uint8_t* base;
    __amdgpu_buffer_rsrc_t buffer;
    __device__ __forceinline__ void at(const void* p) {
        base = (const uint8_t*)p;
        if constexpr (VEC) buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, 0x7ffffff0, 0x00027000);
    }
    __device__ __forceinline__ u32x4 chunk(uint32_t row, int k, int n) const {
        if constexpr (VEC && BYTES == 8) {
            const u32x2 h = __builtin_amdgcn_raw_buffer_load_b64(buffer, k < n ? (int)(row + (uint32_t)k * ES) : -1, 0, 0);
            return u32x4{h[0], h[1], 0, 0};
        } else if constexpr (VEC) {
            return __builtin_amdgcn_raw_buffer_load_b128(buffer, k < n ? (int)(row + (uint32_t)k * ES) : -1, 0, 0);
        } else {
            return fmoe::chunk<ES, false, BYTES>(base + row, k, n);
        }
    }
};

// Eight e4m3 values as bf16, which holds them exactly.
__device__ __forceinline__ bf16x8 e4m3_to_bf16(uint32_t lo, uint32_t hi) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t w = i ? hi : lo;
        r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
        r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
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
    } else if constexpr (WT == kWE4M3Half) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3_to_bf16(w[0], w[1]), __builtin_bit_cast(bf16x8, x[0]), acc, 0, 0, 0);
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

struct FewLists {           // in LDS, and as few_up's first block leaves them in the workspace
    unsigned long long* mask;   // [E] tokens
    uint2* entry;           // [2 E] an expert and up to 16 * NT tokens of its: x = id | tokens << 16, y = first of their slots
    float* gate;            // [T * k]
    int16_t* sel;           // [T * k] expert, -1: none
    int16_t* slots;         // [T * k] t * k + j, by expert and token
    int16_t* first;         // [E] first of an expert's slots
    int* entries;           // how many
};
__host__ __device__ constexpr int few_align(int bytes) { return (bytes + 15) & ~15; }
__host__ __device__ inline int few_lists_bytes(int T, int E, int k) {
    return few_align(E * 8) + E * 16 + few_align(T * k * 4) + 2 * few_align(T * k * 2) + few_align(E * 2) + 16;
}
__device__ __forceinline__ FewLists few_lists(uint8_t* p, int T, int E, int k) {
    FewLists l;
    auto take = [&](int bytes) {
        uint8_t* at = p;
        p += few_align(bytes);
        return at;
    };
    l.mask = (unsigned long long*)take(E * 8);
    l.entry = (uint2*)take(E * 16);
    l.gate = (float*)take(T * k * 4);
    l.sel = (int16_t*)take(T * k * 2);
    l.slots = (int16_t*)take(T * k * 2);
    l.first = (int16_t*)take(E * 2);
    l.entries = (int*)take(16);
    return l;
}
// One of the entries, the same in all lanes (PARTS > 1 of few_down: in a part of them).
struct Entry {
    int e, n, first;
};
template <bool UNIFORM>
__device__ __forceinline__ Entry few_entry(const FewLists& l, int i) {
    const uint2 v = l.entry[i];
    const int x = UNIFORM ? uniform((int)v.x) : (int)v.x, y = UNIFORM ? uniform((int)v.y) : (int)v.y;
    return Entry{x & 0xffff, x >> 16, y};
}
// Elements of a plane of hidden rows
__host__ __device__ inline int64_t few_plane(const fmoe_few_desc& d) { return (int64_t)d.T * d.k * d.H; }

// Sums that meet in few_up: two buffers of the 16 waves' accumulators, or 8 shares of the router
__host__ __device__ constexpr int few_red_bytes(int nt, int mats) { return 2 * kWaves * nt * mats * kWave * 16 > kWaves / 2 * 16 * kRouterRow * 4 ? 2 * kWaves * nt * mats * kWave * 16 : kWaves / 2 * 16 * kRouterRow * 4; }

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
template <int R, typename Logit>
__device__ __forceinline__ void select_token_of(const fmoe_few_desc& d, int t, Logit&& logit, const FewLists& l) {
    const int lane = lane_id();
    if (d.token_mask && !d.token_mask[t]) {
        if (lane < d.k) {
            l.sel[t * d.k + lane] = -1;
            l.gate[t * d.k + lane] = 0.0f;
        }
        return;
    }
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

template <typename Logit>
__device__ __forceinline__ void select_token(const fmoe_few_desc& d, int t, Logit&& logit, const FewLists& l) {
    static_assert(kFewMostExperts == 4 * kWave, "a lane holds up to four experts");
    if (d.E <= kWave) select_token_of<1>(d, t, logit, l);
    else if (d.E <= 2 * kWave) select_token_of<2>(d, t, logit, l);
    else select_token_of<4>(d, t, logit, l);
}

// Who goes where, from every token's selection.
template <int NT>
__device__ __forceinline__ void build_lists(const fmoe_few_desc& d, const FewLists& l) {
    const int lane = lane_id();
    if (d.T == 1) {             // every slot is an entry (1.1 us less than the general way)
        const bool any = l.sel[0] >= 0;
        if ((int)threadIdx.x < d.k && any) {
            l.entry[lane] = uint2{(uint32_t)(l.sel[lane] | 1 << 16), (uint32_t)lane};
            l.slots[lane] = (int16_t)lane;
        }
        if (threadIdx.x == 0) *l.entries = any ? d.k : 0;
        __syncthreads();
        return;
    }
    for (int i = threadIdx.x; i < d.T * d.k; i += kWaves * kWave)
        if (l.sel[i] >= 0) atomicOr(&l.mask[l.sel[i]], 1ull << (i / d.k));
    __syncthreads();
    if (threadIdx.x < kWave) {
        int sofar = 0;          // rows in the low half, entries in the high one
        for (int e0 = 0; e0 < d.E; e0 += kWave) {
            const int e = e0 + lane;
            const int n = e < d.E ? __popcll(l.mask[e]) : 0, groups = (n + 16 * NT - 1) / (16 * NT);
            const int upto = sofar + wave_inclusive_scan(n | groups << 16);
            if (n > 0) {
                const int first = (upto & 0xffff) - n, at = (upto >> 16) - groups;
                l.first[e] = (int16_t)first;
                for (int i = 0; i < groups; ++i)
                    l.entry[at + i] = uint2{(uint32_t)(e | min(16 * NT, n - i * 16 * NT) << 16), (uint32_t)(first + i * 16 * NT)};
            }
            sofar = __builtin_amdgcn_readlane(upto, kWave - 1);
        }
        if (lane == 0) *l.entries = sofar >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < d.T * d.k; i += kWaves * kWave)
        if (l.sel[i] >= 0) {
            const int e = l.sel[i];
            l.slots[l.first[e] + __popcll(l.mask[e] & ((1ull << (i / d.k)) - 1))] = (int16_t)i;
        }
    __syncthreads();
}

template <int WT, bool VEC, int NT, bool GATED>
__global__ __launch_bounds__(kWaves* kWave) void few_up_kernel(FewParams p, int share_bits) {
    constexpr bool F32 = WT == kWF32, E4M3 = WT == kWE4M3 || WT == kWE4M3Half;
    constexpr int CE = Wt<WT>::CE, ES = Wt<WT>::ES, XES = Wt<WT>::XES, XC = Wt<WT>::XC, STEP = 4 * CE, MATS = GATED ? 2 : 1;
    constexpr int AHEAD = !VEC || NT * XC * MATS > 2 ? 2 : 3;    // batches of loads in flight
    constexpr int RED = few_red_bytes(NT, MATS) / 8;     // floats of the waves' sums, of which there are two buffers
    extern __shared__ uint8_t lds[];
    const fmoe_few_desc& d = p.d;
    const int lane = lane_id(), wave = uniform(threadIdx.x / kWave), r16 = lane & 15, quarter = lane >> 4;
    float* const red = (float*)lds;
    float* const logits = (float*)(lds + few_red_bytes(NT, MATS));
    uint8_t* const listed = lds + few_red_bytes(NT, MATS) + (p.stretches ? 0 : few_align(16 * d.E * 4));
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
        for (int i = threadIdx.x; i < p.tiles; i += kWaves * kWave) p.arrivals[i] = 0;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < few_lists_bytes(d.T, d.E, d.k) / 16; i += kWaves * kWave)
            reinterpret_cast<u32x4*>(p.lists)[i] = reinterpret_cast<const u32x4*>(listed)[i];
    // Groups of `shares` waves have an item each and share its contraction in pieces of two steps.
    const int shares = 1 << share_bits, group = wave >> share_bits, share = wave & (shares - 1), groups = kWaves >> share_bits;
    const int tiles = (d.H + 15) / 16, entries = uniform(*l.entries), steps = (d.D + STEP - 1) / STEP;
    const int batches = (steps + 2 * shares - 1) / (2 * shares);       // of two steps a wave
    // An item is an entry's tile of 16 hidden columns; a group takes every `stride`th.  The groups of a block go through the barriers
    // together, those behind the last item with nothing to do.
    const int stride = gridDim.x * groups, over = stride / tiles, rest = stride - over * tiles;
    struct Item {
        int entry, tile;
    };
    auto step = [&](Item& it) {
        it.entry += over;
        it.tile += rest;
        if (it.tile >= tiles) {
            it.tile -= tiles;
            ++it.entry;
        }
    };
    const int start = blockIdx.x * groups;
    Item loading = {(start + group) / tiles, (start + group) % tiles}, adding = loading;
    const int total = entries * tiles, rounds = start < total ? (total - start + stride - 1) / stride : 0;
    // What is loaded runs AHEAD batches before what is multiplied, over the ends of items.
    Rows<ES, VEC, CE * ES> w[MATS];
    Rows<XES, VEC> x;
    x.at(d.x);
    uint32_t wrow = 0, xrow[NT];
    int wcols = 0, xcols[NT], load_s = 0;
    auto take = [&] {
        const bool any = loading.entry < entries;
        const Entry at = any ? few_entry<true>(l, loading.entry) : Entry{0, 0, 0};
        const int h0 = any ? 16 * loading.tile : 0;
        const int64_t from = ((int64_t)at.e * d.w_stride_e + (int64_t)h0 * d.w_stride_n) * ES;
        wrow = (uint32_t)(min(r16, d.H - 1 - h0) * (int)d.w_stride_n * ES);
        wcols = any ? d.D : 0;
        w[0].at((const uint8_t*)d.w + from);
        if constexpr (GATED) w[1].at((const uint8_t*)d.wp + from);
#pragma unroll
        for (int f = 0; f < NT; ++f) {
            const bool live = 16 * f + r16 < at.n;
            xrow[f] = live ? (uint32_t)(l.slots[at.first + 16 * f + r16] / d.k * (int)d.x_stride_row * XES) : 0u;
            xcols[f] = live ? d.D : 0;
        }
    };
    u32x4 wv[AHEAD][2][MATS], xv[AHEAD][2][NT][XC];
    auto load = [&](u32x4 (&wb)[2][MATS], u32x4 (&xb)[2][NT][XC]) {
        // (the two halves of a row's 128-byte line behind one another, so that the L1 asks the L2 for the line once)
        const int k = (load_s + 2 * share) * STEP + quarter * CE;
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int u = 0; u < 2; ++u) wb[u][m] = w[m].chunk(wrow, k + u * STEP, wcols);
#pragma unroll
        for (int f = 0; f < NT; ++f)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int c = 0; c < XC; ++c) xb[u][f][c] = x.chunk(xrow[f], k + u * STEP + c * (16 / XES), xcols[f]);
        load_s += 2 * shares;
        if (load_s >= steps) {
            load_s = 0;
            step(loading);
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
    int turn = 0, n = NT > 1 && adding.entry < entries ? few_entry<true>(l, adding.entry).n : 0;
    // An item's sums: a wave adds one of a lane's four columns (of one of the NT halves of the tokens) over the group's waves, others of the group each
    // time; the rest goes on to the next item at once (the buffers take turns, so that it has read one before that is written again: in between is a
    // barrier that it has to reach).  So few instructions on purpose: they come from memory the first time, 64 bytes after one another.
    auto finish = [&](int round) {
        float* const buf = red + turn * RED;
        turn ^= 1;
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int f = 0; f < NT; ++f) *reinterpret_cast<f32x4*>(buf + (((wave * MATS + m) * NT + f) * kWave + lane) * 4) = acc[m][f];
        __syncthreads();
        if (adding.entry < entries) {
            const Entry at = few_entry<true>(l, adding.entry);
#pragma unroll 1
            for (int j = (share - 4 * NT * round) & (shares - 1); j < 4 * NT; j += shares) {
                const int c = 16 * (j / 4) + r16, col = 16 * adding.tile + 4 * quarter + j % 4;
                if (c >= at.n || col >= d.H) continue;
                const float* from = buf + ((group * shares * MATS * NT + j / 4) * kWave + lane) * 4 + j % 4;
                float v[MATS] = {};
#pragma unroll 4
                for (int w = 0; w < shares; ++w, from += MATS * NT * kWave * 4)
#pragma unroll
                    for (int m = 0; m < MATS; ++m) v[m] += from[m * NT * kWave * 4];
                const int slot = l.slots[at.first + c];
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    const void* const b = m ? d.bias_p : d.bias;
                    if constexpr (E4M3) v[m] /= (m ? d.wp_scale : d.w_scale)[(int64_t)at.e * d.H + col];
                    if (b) v[m] += element<F32>(b, (int64_t)at.e * d.bias_stride_e + col);
                }
                float h = silu_f32(v[0]);
                if constexpr (GATED) h *= v[1];
                h *= l.gate[slot];
                const int64_t to = (int64_t)slot * d.H + col;
                put_element<F32>(p.h, to, h);
                if constexpr (!F32) {       // what the rounding leaves
                    const float hi = bf16_bits_to_f32(f32_to_bf16_bits(h));
                    put_element<false>(p.h, few_plane(d) + to, __builtin_isinf(hi) ? 0.0f : h - hi);
                }
            }
        }
        clear();
        step(adding);
        if constexpr (NT > 1) n = adding.entry < entries ? few_entry<true>(l, adding.entry).n : 0;
    };
    for (int round = 0, left = batches; round < rounds;) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (round >= rounds) break;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int f = 0; f < NT; ++f)
                    if (f == 0 || 16 * f < n) {
#pragma unroll
                        for (int m = 0; m < MATS; ++m) mma<WT>(acc[m][f], wv[i][u][m], xv[i][u][f]);
                    }
            load(wv[i], xv[i]);
            if (--left == 0) {
                finish(round);
                ++round;
                left = batches;
            }
        }
    }
}

// PARTS: a tile has 16 / PARTS output columns, and the MFMAs' rows (and columns: up to 16 / PARTS tokens) hold that many stretches of the
// contraction side by side, of whose products the diagonal blocks count: more, smaller tiles where 16 columns each would leave CUs without one.
// bf16: a hidden row is the sum of two, its rounding to bf16 and what that leaves.  The second ones take columns that an expert's tokens leave free, at no more
// loads or products; an expert with more than half as many tokens as a tile has columns does without them (half a step of bf16 for each hidden value, which
// makes the output's error 1.4 times that of its own rounding; columns of their own for all of them took 10 to 30 % of this kernel's time).
// gridDim.y > 1: so many blocks share a tile's contraction; their sums go through memory, and the one that arrives last adds them in block order.
template <int WT, bool VEC, int NT, int PARTS>
__global__ __launch_bounds__(kWaves* kWave) void few_down_kernel(FewParams p, bool spread) {
    constexpr bool F32 = WT == kWF32, E4M3 = WT == kWE4M3 || WT == kWE4M3Half, ONE = PARTS == 1;
    constexpr int CE = Wt<WT>::CE, ES = Wt<WT>::ES, XES = Wt<WT>::XES, XC = Wt<WT>::XC, STEP = 4 * CE, COLS = 16 / PARTS;
    constexpr int AHEAD = !VEC ? 1 : NT * XC == 1 ? 4 : NT * XC == 2 ? 3 : 2;      // pieces whose loads are in flight
    extern __shared__ uint8_t lds[];
    const fmoe_few_desc& d = p.d;
    const int lane = lane_id(), wave = uniform(threadIdx.x / kWave), waves = blockDim.x / kWave, r16 = lane & 15, quarter = lane >> 4;
    float* const sums = (float*)lds;                                        // [waves][T][16]
    uint8_t* const listed = lds + (size_t)waves * d.T * 64;
    const FewLists l = few_lists(listed, d.T, d.E, d.k);
    for (int i = threadIdx.x; i < few_lists_bytes(d.T, d.E, d.k) / 16; i += blockDim.x)
        reinterpret_cast<u32x4*>(listed)[i] = reinterpret_cast<const u32x4*>(p.lists)[i];
    for (int i = threadIdx.x; i < waves * d.T * 4; i += blockDim.x) reinterpret_cast<f32x4*>(sums)[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();
    const int part = ONE ? 0 : r16 / COLS, n0 = blockIdx.x * COLS, row = min(n0 + r16 % COLS, d.O - 1);
    const int steps = (d.H + STEP - 1) / STEP, pieces = (steps + 1) / 2, total = uniform(*l.entries) * pieces;
    // Every stretch (a wave's, or a part of its) takes as many pieces of two steps, experts after one another: all of its in a row, or (spread) every
    // stretches-th, so that all of them work on the same rows at a time and an expert with more tokens costs each as much.
    const int stretches = waves * PARTS * gridDim.y, per = (total + stretches - 1) / stretches, unit = spread ? 1 : per;
    const int from = ((blockIdx.y * waves + wave) * PARTS + part) * unit, until = spread ? total : min(total, from + per);
    const int skip = spread ? stretches - 1 : 0, over = skip / pieces, rest = skip - over * pieces;
    Entry next = {0, 0, 0}, cur = {0, 0, 0};            // whose loads are on their way, and whose products add up
    int next_index = -1, cur_index = -1, of[AHEAD];
    const uint8_t *wrow = nullptr, *xrow[NT] = {};
    Rows<ES, VEC, CE * ES> w;
    Rows<XES, VEC> x;
    uint32_t xoff[NT] = {};
    w.at(d.wo);
    x.at(p.h);
    const uint32_t second = F32 ? 0u : (uint32_t)(few_plane(d) * XES);      // of a row's two (the workspace is shorter than 2^31 bytes)
    auto both = [&](const Entry& at) { return !F32 && 2 * at.n <= COLS; };
    const uint32_t woff = (uint32_t)((row - n0) * (int)d.wo_stride_n * ES);
    u32x4 wv[AHEAD][2], xv[AHEAD][2][NT][XC];
    int q = from, index = total ? from / pieces : 0, piece = from - index * pieces;
    auto load = [&](int& of, u32x4 (&wb)[2], u32x4 (&xb)[2][NT][XC]) {
        const bool any = q < until;
        of = any ? index : next_index;
        if (any && index != next_index) {
            next = few_entry<ONE>(l, index);
            next_index = index;
            if constexpr (ONE) w.at((const uint8_t*)d.wo + ((int64_t)next.e * d.wo_stride_e + (int64_t)n0 * d.wo_stride_n) * ES);
            else wrow = (const uint8_t*)d.wo + ((int64_t)next.e * d.wo_stride_e + (int64_t)row * d.wo_stride_n) * ES;
#pragma unroll
            for (int f = 0; f < NT; ++f) {
                int c = 16 * f + r16 % COLS;
                uint32_t at = 0;
                if (f == 0 && both(next) && c >= COLS / 2) {
                    c -= COLS / 2;
                    at = second;
                }
                at = c < next.n ? at + (uint32_t)(l.slots[next.first + c] * d.H * XES) : ~0u;
                if constexpr (ONE) xoff[f] = at;
                else xrow[f] = at != ~0u ? (const uint8_t*)p.h + at : nullptr;
            }
        }
        const int k = 2 * piece * STEP + quarter * CE;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if constexpr (ONE) wb[s] = w.chunk(woff, k + s * STEP, any ? d.H : 0);
            else wb[s] = chunk<ES, VEC, CE * ES>(wrow, k + s * STEP, any ? d.H : 0);
        }
#pragma unroll
        for (int f = 0; f < NT; ++f)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int c = 0; c < XC; ++c) {
                    const int at = k + s * STEP + c * (16 / XES);
                    if constexpr (ONE) xb[s][f][c] = x.chunk(xoff[f], at, any && xoff[f] != ~0u ? d.H : 0);
                    else xb[s][f][c] = chunk<XES, VEC>(xrow[f], at, any && xrow[f] ? d.H : 0);
                }
        q += 1 + skip;
        index += over;
        piece += 1 + rest;
        if (piece >= pieces) {
            piece -= pieces;
            ++index;
        }
    };
    f32x4 acc[NT], inv = {1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
    for (int f = 0; f < NT; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // An expert's products go to its own tokens' sums, and only there (a column without a token holds zeros, which an infinity among the weights
    // turns into NaN).
    auto flush = [&] {
        if (cur_index >= 0) {
#pragma unroll
            for (int f = 0; f < NT; ++f) {
                const int c = 16 * f + r16 % COLS;
                f32x4 own = acc[f];
                if (f == 0 && both(cur)) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) own[i] += __shfl_xor(acc[0][i], COLS / 2, kWave);
                }
                if (c < cur.n && (ONE || quarter * 4 / COLS == part)) {
                    f32x4* const to = reinterpret_cast<f32x4*>(sums + ((size_t)wave * d.T + l.slots[cur.first + c] / d.k) * 16 + 4 * quarter);
                    f32x4 v = *to;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] += E4M3 ? own[i] / inv[i] : own[i];
                    *to = v;
                }
            }
        }
#pragma unroll
        for (int f = 0; f < NT; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(of[i], wv[i], xv[i]);
    for (int done = 0; done < per; done += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {       // (behind a stretch's last piece come zeros)
            if (ONE ? of[i] != cur_index : __any(of[i] != cur_index)) {
                flush();
                if (of[i] >= 0) {
                    cur = few_entry<ONE>(l, of[i]);
                    cur_index = of[i];
                    if constexpr (E4M3)
#pragma unroll
                        for (int j = 0; j < 4; ++j) inv[j] = d.wo_scale[(int64_t)cur.e * d.O + min(n0 + (4 * quarter + j) % COLS, d.O - 1)];
                }
            }
#pragma unroll
            for (int f = 0; f < NT; ++f)
                if (f == 0 || 16 * f < cur.n) {
                    mma<WT>(acc[f], wv[i][0], xv[i][0][f]);
                    mma<WT>(acc[f], wv[i][1], xv[i][1][f]);
                }
            load(of[i], wv[i], xv[i]);
        }
    }
    flush();
    __syncthreads();
    float* const partial = p.partial + (int64_t)blockIdx.x * gridDim.y * d.T * COLS;        // [tile][block][T][COLS]
    bool last = true;
    auto own = [&](int t, int c) {
        float v = 0.0f;
        for (int w0 = 0; w0 < waves; w0 += 8)       // (8 or 16)
#pragma unroll
            for (int w = 0; w < 8; ++w)
#pragma unroll
                for (int q2 = 0; q2 < PARTS; ++q2) v += sums[((w0 + w) * d.T + t) * 16 + q2 * COLS + c];
        return v;
    };
    if (gridDim.y > 1) {
        for (int i = threadIdx.x; i < d.T * COLS; i += blockDim.x) partial[(int64_t)blockIdx.y * d.T * COLS + i] = own(i / COLS, i % COLS);
        __syncthreads();
        int* const arrived = (int*)lds;         // (the sums have been read)
        // (one wave's release and acquire, behind and before a barrier, stand for the block's; a fence of every wave took 50 us)
        if (threadIdx.x == 0) *arrived = __hip_atomic_fetch_add(p.arrivals + blockIdx.x, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        last = *arrived == (int)gridDim.y - 1;
    }
    if (!last) return;
    for (int i = threadIdx.x; i < d.T * COLS; i += blockDim.x) {
        const int t = i / COLS, c = i % COLS, col = n0 + c;
        if (col >= d.O) continue;
        float v = 0.0f;
        if (gridDim.y > 1)
            for (unsigned y = 0; y < gridDim.y; ++y) v += __hip_atomic_load(partial + (int64_t)y * d.T * COLS + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        else v = own(t, c);
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
size_t few_logits_at(const fmoe_few_desc& d) { return (few_hidden_at(d) + (size_t)few_plane(d) * 4 + 255) & ~(size_t)255; }
// Stretches of the router's own launch, 0 where few_up computes the router: 256 CUs reading 256 KB of gate each take 9 us, a launch and its reading back 5.
// Up to 16 tokens are one block per 16 experts and stretch (4 of them: 4.5 us for 128 experts of 4096); more have blocks of their own, and every stretch is
// read back for every token: 32 tokens, 128 experts of 4096 11.2 us as one stretch, 7.0 as two, 5.3 as four, which cost the selection 3.
int few_stretches(const fmoe_few_desc& d) {
    if ((int64_t)d.E * d.D * (d.dtype == FMOE_F32 ? 4 : 2) * ((d.T + 15) / 16) <= 32 * 1024) return 0;
    return d.T <= 16 ? 4 : 2;
}
size_t few_arrivals_at(const fmoe_few_desc& d) { return (few_logits_at(d) + (size_t)few_stretches(d) * d.T * d.E * 4 + 255) & ~(size_t)255; }
// few_down's tiles: parts of an MFMA's rows (up to 16 / parts tokens) so that there are 256 of them, else blocks to a tile.  Parts against tiles of 16:
// 1 token, 1408 x 2048 12.8 us and 18.7, 1408 x 512 7.9 and 13.5, 5 tokens, 256 x 128 5.4 and 8.5.  Blocks against one to a tile: 64 tokens, 64 experts of
// 1408 x 1024 bf16 54 us and 147, 37 tokens, 2600 x 1000 fp32 45 and 110.
struct DownPlan {
    int parts, tiles, blocks;
};
DownPlan few_down_plan(const fmoe_few_desc& d) {
    DownPlan p;
    p.parts = d.O >= 16 * 256 || d.T > 8 ? 1 : d.O >= 8 * 256 || d.T > 4 ? 2 : 4;
    p.tiles = (d.O + 16 / p.parts - 1) / (16 / p.parts);
    p.blocks = p.parts > 1 || p.tiles > 128 ? 1 : 256 / p.tiles < 8 ? 256 / p.tiles : 8;
    return p;
}
size_t few_bytes(const fmoe_few_desc& d) {
    const DownPlan p = few_down_plan(d);
    return few_arrivals_at(d) + (p.blocks > 1 ? (((size_t)p.tiles * 4 + 255) & ~(size_t)255) + (size_t)p.tiles * p.blocks * d.T * (16 / p.parts) * 4 : 0);
}

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
    const DownPlan plan = few_down_plan(d);
    const FewParams p{d, workspace, (uint8_t*)workspace + few_hidden_at(d), (const float*)((uint8_t*)workspace + few_logits_at(d)), few_stretches(d), plan.blocks > 1 ? plan.tiles : 0,
                      (int32_t*)((uint8_t*)workspace + few_arrivals_at(d)),
                      (float*)((uint8_t*)workspace + few_arrivals_at(d) + (((size_t)plan.tiles * 4 + 255) & ~(size_t)255))};
    const int es = d.dtype == FMOE_F32 ? 4 : 2, wes = d.weight_dtype == FMOE_E4M3 ? 1 : es;
    // whole chunks at their boundaries wherever rows are read: 16 bytes, 8 of e4m3 weights where it comes to that
    auto whole = [](const void* q, int64_t elements, int size, int chunk) { return ((uintptr_t)q & (chunk - 1)) == 0 && elements * size % chunk == 0; };
    auto weights = [&](int chunk) {
        return whole(d.w, d.D, wes, chunk) && whole(d.w, d.w_stride_n, wes, chunk) && whole(d.w, d.w_stride_e, wes, chunk) && whole(d.wp, d.D, wes, chunk) &&
               whole(d.wo, d.H, wes, chunk) && whole(d.wo, d.wo_stride_n, wes, chunk) && whole(d.wo, d.wo_stride_e, wes, chunk);
    };
    const bool rows = whole(d.x, d.D, es, 16) && whole(d.x, d.x_stride_row, es, 16) && whole(d.gate_weight, d.gate_stride_row, es, 16) && d.H * es % 16 == 0;
    const bool vec = rows && weights(16), half = rows && wes == 1 && weights(8);
    const bool gated = d.wp != nullptr;
    const int most_active = d.T * d.k < d.E ? d.T * d.k : d.E;
    hipStream_t stream = (hipStream_t)stream_;
    const int lists = few_lists_bytes(d.T, d.E, d.k), step = wes == 1 ? 64 : 64 / wes;
    const int64_t items = (int64_t)most_active * ((d.H + 15) / 16) * (d.T > 32 ? 2 : 1);
    // waves to an item: so that each has four steps, and no CU is without an item for want of blocks.  (16 to every item: 16 tokens, 128 experts of 512 x 1536
    // bf16 76 us in place of 58, a wave's two steps at a time being more than its share.)
    int share_bits = 0;
    while (share_bits < 4 && ((4 << share_bits) * step < d.D || (items << share_bits) < 256 * kWaves)) ++share_bits;
    auto up = [&](auto kern, bool& reserved, int red) {
        const int bytes = red + (p.stretches ? 0 : few_align(16 * d.E * 4)) + lists;
        if (!reserved) {        // (more than 64 KB; the most that any call of this kernel asks for)
            const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                       red + few_align(16 * kFewMostExperts * 4) + few_lists_bytes(kFewMostTokens, kFewMostExperts, kFewMostK));
            if (err != hipSuccess) return fail(FMOE_ERR_LAUNCH, "fmoe_few_tokens: cannot reserve %d B of LDS: %s", bytes, hipGetErrorString(err));
            reserved = true;
        }
        const int64_t blocks = (items + (kWaves >> share_bits) - 1) / (kWaves >> share_bits);
        kern<<<(unsigned)(blocks < 256 ? blocks : 256), kWaves * kWave, bytes, stream>>>(p, share_bits);
        return check_launch("fmoe_few_tokens");
    };
    auto down = [&](auto kern) {
        const int waves = d.T > 32 ? kWaves / 2 : kWaves;        // (their sums for 64 tokens in 32 KB of LDS)
        // Spread where an expert has two pieces for every stretch: 37 tokens, 12 experts, 2600 x 1000 fp32 48.9 us in a row, 44.6 spread, 1 token, 14336 x
        // 4096 bf16 47.0 and 44.1.  With fewer, a stretch changes experts at nearly every piece: 16 tokens, 128 experts, 1536 x 4096 bf16 150 and 155 us,
        // 1 token, 1408 x 2048 13.2 and 14.3, 4 tokens, 1536 x 4096 e4m3 43 and 48.
        const int down_step = half && !vec ? 32 : step, pieces = ((d.H + down_step - 1) / down_step + 1) / 2;
        kern<<<dim3(plan.tiles, plan.blocks), waves * kWave, waves * d.T * 64 + lists, stream>>>(p, pieces >= 2 * waves * plan.parts * plan.blocks);
    };
#define FMOE_FEW_UP(WT, VEC, NT, GATED)                                     \
    ([&] {                                                                  \
        static bool reserved = false;                                       \
        return up(few_up_kernel<WT, VEC, NT, GATED>, reserved, few_red_bytes(NT, GATED ? 2 : 1)); \
    })()
#define FMOE_FEW(WT, VEC)                                                   \
    do {                                                                    \
        if (p.stretches) {                                                  \
            few_logits_kernel<WT == kWF32, VEC><<<dim3((d.E + 15) / 16, (d.T + 15) / 16, p.stretches), kLogitWaves * kWave, 0, stream>>>(d, const_cast<float*>(p.logits)); \
            const int first = check_launch("fmoe_few_tokens");              \
            if (first != FMOE_OK) return first;                             \
        }                                                                   \
        const int second = d.T <= 16 ? (gated ? FMOE_FEW_UP(WT, VEC, 1, true) : FMOE_FEW_UP(WT, VEC, 1, false)) \
                                     : (gated ? FMOE_FEW_UP(WT, VEC, 2, true) : FMOE_FEW_UP(WT, VEC, 2, false)); \
        if (second != FMOE_OK) return second;                               \
        if (d.T > 16) down(few_down_kernel<WT, VEC, 2, 1>);                 \
        else if (plan.parts == 1) down(few_down_kernel<WT, VEC, 1, 1>);     \
        else if (plan.parts == 2) down(few_down_kernel<WT, VEC, 1, 2>);     \
        else down(few_down_kernel<WT, VEC, 1, 4>);                          \
    } while (0)
    if (d.weight_dtype == FMOE_F32) {
        if (vec) FMOE_FEW(kWF32, true); else FMOE_FEW(kWF32, false);
    } else if (d.weight_dtype == FMOE_BF16) {
        if (vec) FMOE_FEW(kWBF16, true); else FMOE_FEW(kWBF16, false);
    } else {
        if (vec) FMOE_FEW(kWE4M3, true); else if (half) FMOE_FEW(kWE4M3Half, true); else FMOE_FEW(kWE4M3, false);
    }
#undef FMOE_FEW
#undef FMOE_FEW_UP
    return check_launch("fmoe_few_tokens");
}
