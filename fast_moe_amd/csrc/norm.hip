// The norms before and after an expert block with its gate and residual scale (fmoe_norm_add and its backward):
//
//   y    given [T, D], or the merge of the K expert rows of every token (sum_j w_j * value[r_j], fmoe_combine's arguments)
//   a    = (y - m) * r            m the row's mean (layer norm; rms norm: 0), r = 1 / sqrt(mean((y - m)^2) + eps)
//   z    = a * weight + bias      (y itself without a weight)
//   out  = residual + scale * gate * z
//   b    = (out - m') * r',       next = b * next_weight + next_bias
//
// backward, with d the whole gradient of out and <.> the mean over a row (the terms in <d..> of a mean only for layer norm):
//   db   = d_next * next_weight,  d = d_out + r' * (db - b * <db * b> - <db>)            = d_residual
//   dz   = d * scale * gate,      da = dz * weight,   d_y = r * (da - a * <da * a> - <da>)
//   d_gate = sum of d * scale * z (per token, or as it is), times gate * (1 - gate) behind a sigmoid
//   d_scale = sum over rows of d * gate * z, d_weight of dz * a, d_bias of dz, d_next_weight of d_next * b, d_next_bias of d_next
//
// Bound by the bytes: every input once, every output once.  A row lies in the registers of as many waves as it has 16-byte chunks for their
// lanes (one wave: no barriers at all), in fp32 from its load to its last use; the sums over rows stay in registers while a block walks its rows and
// leave once per block, added up by a second launch in block order.  The two means and reciprocals of a row are kept by the forward pass (16 bytes
// a row), which leaves the backward pass two exchanges between waves per row in place of four.
#include "common.h"

#include <type_traits>

namespace fmoe {
namespace {

constexpr int kNormMostWaves = 16;

template <typename E> struct NE;
template <> struct NE<float> { static constexpr int V = 4; };
template <> struct NE<uint16_t> { static constexpr int V = 8; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(uint16_t v) { return bf16_bits_to_f32(v); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(uint16_t* p, float v) { *p = (uint16_t)f32_to_bf16_bits(v); }

// 16 bytes at any address an element may have (the hardware takes them at every alignment)
__device__ __forceinline__ u32x4 load16(const void* p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
__device__ __forceinline__ void store16(void* p, const u32x4& v) { __builtin_memcpy(p, &v, 16); }

// Which columns a lane holds: chunks of V neighbours, 16 bytes.  WHOLE: rows are whole chunks; otherwise bf16's last one is read and written by elements, and
// fp32 goes by elements altogether, neighbours in neighbouring lanes (16 bytes at addresses between the chunks' are slower: 3063 x 1001, forward and
// backward 64 us against 49; in bf16, where an element is 2 bytes, faster: 12975 x 1822 forward 74 us against 102).
template <typename E, bool WHOLE, int CH>
struct Row {
    static constexpr int V = NE<E>::V, N = V * CH;
    static constexpr bool ELEMENTS = !WHOLE && V == 4;
    struct Raw {            // what has been loaded and not been looked at
        u32x4 v[CH];
    };
    int tid, threads, cols;
    __device__ __forceinline__ int col(int i) const { return ELEMENTS ? i * threads + tid : ((i / V) * threads + tid) * V + i % V; }
    __device__ __forceinline__ bool in(int i) const { return col(WHOLE ? i / V * V : i) < cols; }
    __device__ __forceinline__ bool whole(int c) const { return WHOLE ? in(c * V) : !ELEMENTS && col(c * V) + V <= cols; }
    __device__ __forceinline__ void fetch(const E* p, Raw& r) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if constexpr (ELEMENTS) {
#pragma unroll
                for (int i = 0; i < V; ++i) r.v[c][i] = in(c * V + i) ? __float_as_uint(p[col(c * V + i)]) : 0u;
                continue;
            }
            r.v[c] = u32x4{0, 0, 0, 0};
            if (whole(c)) {
                r.v[c] = load16(p + col(c * V));
            } else if (!WHOLE && in(c * V)) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (in(c * V + i)) r.v[c][i / 2] |= (uint32_t)p[col(c * V + i)] << (16 * (i & 1));
            }
        }
    }
    __device__ __forceinline__ void take(const Raw& r, float (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (V == 4) f[i] = __uint_as_float(r.v[i / V][i % V]);
            else f[i] = i & 1 ? __uint_as_float(r.v[i / V][i % V / 2] & 0xffff0000u) : __uint_as_float(r.v[i / V][i % V / 2] << 16);
        }
    }
    __device__ __forceinline__ void take_chunk(const Raw& r, int c, float (&f)[V]) const {
        float all[N];
        take(r, all);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = all[c * V + i];
    }
    __device__ __forceinline__ void store(E* p, const float (&f)[N]) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (whole(c)) {
                u32x4 v;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (V == 4) v[i] = __float_as_uint(f[c * V + i]);
                    else v[i] = cvt_pk_bf16(f[c * V + 2 * i], f[c * V + 2 * i + 1]);
                }
                store16(p + col(c * V), v);
            } else if (!WHOLE) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (in(c * V + i)) from_f32(p + col(c * V + i), f[c * V + i]);
            }
        }
    }
    // a parameter of the columns of chunk c, in fp32 or bf16 whatever the rows are
    __device__ __forceinline__ void param(const void* p, int dtype, int c, float (&f)[V], float none) const {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = none;
        if (!p) return;
        if (whole(c)) {
            if (dtype == FMOE_F32) {
                __builtin_memcpy(f, (const float*)p + col(c * V), sizeof(f));
            } else {
                uint16_t h[V];
                __builtin_memcpy(h, (const uint16_t*)p + col(c * V), sizeof(h));
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = bf16_bits_to_f32(h[i]);
            }
        } else if (!WHOLE) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int at = col(c * V + i);
                if (at < cols) f[i] = dtype == FMOE_F32 ? reinterpret_cast<const float*>(p)[at] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[at]);
            }
        }
    }
    // rows of fp32 at the same columns, whatever E is
    struct Raw32 {
        u32x4 v[N / 4];
    };
    __device__ __forceinline__ void fetch_f32(const float* p, Raw32& r) const {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int q = 0; q < V / 4; ++q) {
                u32x4& v = r.v[c * (V / 4) + q];
                v = u32x4{0, 0, 0, 0};
                if (whole(c)) {
                    v = load16(p + col(c * V) + 4 * q);
                } else if (!WHOLE) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = in(c * V + 4 * q + i) ? __float_as_uint(p[col(c * V + 4 * q + i)]) : 0u;
                }
            }
    }
    __device__ __forceinline__ void take_f32(const Raw32& r, float (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __uint_as_float(r.v[i / 4][i % 4]);
    }
    __device__ __forceinline__ void store_f32(float* p, const float (&f)[N]) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (whole(c)) {
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    u32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[c * V + 4 * q + i]);
                    store16(p + col(c * V) + 4 * q, v);
                }
            } else if (!WHOLE) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (in(c * V + i)) p[col(c * V + i)] = f[c * V + i];
            }
        }
    }
};

// The sum over a wave in every lane: a row of 16 lanes on the DPP network, the four rows in order.
__device__ __forceinline__ float wave_sum(float v) {
#define FMOE_DPP_ADD(ctrl) v += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), ctrl, 0xF, 0xF, false))
    FMOE_DPP_ADD(0xB1);      // quad_perm [1,0,3,2]
    FMOE_DPP_ADD(0x4E);      // quad_perm [2,3,0,1]
    FMOE_DPP_ADD(0x141);     // row_half_mirror
    FMOE_DPP_ADD(0x140);     // row_mirror
#undef FMOE_DPP_ADD
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) s += __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 16 * r));
    return s;
}

// Sums over the waves of a row; two buffers in turn, so that one barrier a call is enough.
struct Exchange {
    float (*buf)[kNormMostWaves][4];    // [2]
    int waves, wave, turn;
    template <int NV>
    __device__ __forceinline__ void sum(float (&v)[NV]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = wave_sum(v[i]);
        if (waves == 1) return;
        if (lane_id() == 0)
#pragma unroll
            for (int i = 0; i < NV; ++i) buf[turn][wave][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = buf[turn][0][i];
            for (int w = 1; w < waves; ++w) v[i] += buf[turn][w][i];
        }
        turn ^= 1;
    }
};

// Mean (0 for rms norm) and 1 / sqrt(mean square + eps) of a row; the squares are those of the centred values.
template <typename R, int N>
__device__ __forceinline__ void row_stats(const R& row, const float (&f)[N], bool layer, float eps, Exchange& x, float& mean, float& rstd) {
    mean = 0.0f;
    if (layer) {
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < N; ++i) s[0] += f[i];       // (0 behind the last column)
        x.sum(s);
        mean = s[0] / (float)row.cols;
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float c = f[i] - mean;
        if (!layer || row.in(i)) q[0] += c * c;
    }
    x.sum(q);
    rstd = 1.0f / sqrtf(q[0] / (float)row.cols + eps);
}

__device__ __forceinline__ float sigmoid_f32(float v) { return 1.0f / (1.0f + expf(-v)); }

// A parameter where it is used: kept in registers over the rows where a lane has one chunk, asked for again (from the L1) where it has more.
template <typename R, bool KEPT>
struct Param {
    static constexpr int V = R::V;
    const void* p;
    int dtype;
    float none, kept[KEPT ? V : 1];
    __device__ __forceinline__ Param(const R& row, const void* p, int dtype, float none) : p(p), dtype(dtype), none(none) {
        if constexpr (KEPT) row.param(p, dtype, 0, kept, none);
    }
    __device__ __forceinline__ void get(const R& row, int c, float (&f)[V]) const {
        if constexpr (KEPT) {
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = kept[i];
        } else {
            row.param(p, dtype, c, f, none);
        }
    }
};

// y given, or none (only the next norm).  16384 x 2048 bf16, a sigmoid gate for each token: 53 us, 5.1 TB/s; 8 x 2048 4.6 us, a launch and two ways to memory.
template <typename E, bool WHOLE, int CH>
__global__ __launch_bounds__(kNormMostWaves* kWave) void norm_add_kernel(fmoe_norm_desc d, int waves) {
    using R = Row<E, WHOLE, CH>;
    using P = Param<R, CH == 1>;
    constexpr int N = R::N, V = R::V;
    __shared__ float buf[2][kNormMostWaves][4];
    const int per = waves == 1 ? blockDim.x / kWave : 1, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);       // rows of a block at a time
    const R row{waves == 1 ? (int)threadIdx.x % kWave : (int)threadIdx.x, waves * kWave, d.cols};
    Exchange x{buf, waves, wave, 0};
    const bool layer = d.norm == FMOE_NORM_LAYER;
    const P scale(row, d.scale, d.param_dtype, d.scale_value), weight(row, d.weight, d.param_dtype, 1.0f), bias(row, d.bias, d.param_dtype, 0.0f),
        next_weight(row, d.next_weight, d.param_dtype, 0.0f), next_bias(row, d.next_bias, d.param_dtype, 0.0f);
    // The next row's loads are issued before this row's sums are exchanged.
    const int64_t first = (int64_t)blockIdx.x * per + (waves == 1 ? wave : 0), step = (int64_t)gridDim.x * per;
    typename R::Raw ro, rg, ry;
    const bool element = d.gate_mode == FMOE_GATE_ELEMENT;
    E token_gate = E(0);
    auto fetch = [&](int64_t t) {
        if (t >= d.rows) return;
        row.fetch((const E*)d.residual + t * d.residual_stride, ro);
        if (element) row.fetch((const E*)d.gate + t * d.gate_stride, rg);
        else if (d.gate_mode) token_gate = ((const E*)d.gate)[t * d.gate_stride];
        if (d.y) row.fetch((const E*)d.y + t * d.y_stride, ry);
    };
    fetch(first);
    for (int64_t t = first; t < d.rows; t += step) {
        float o[N], mean = 0.0f, rstd = 1.0f, mean2 = 0.0f, rstd2 = 1.0f;
        row.take(ro, o);
        const typename R::Raw gates = rg;
        float token = d.gate_mode == FMOE_GATE_TOKEN ? to_f32(token_gate) : 1.0f;
        if (d.gate_mode == FMOE_GATE_TOKEN && d.gate_sigmoid) token = sigmoid_f32(token);
        if (d.y) {
            float y[N];
            row.take(ry, y);
            fetch(t + step);
            if (d.weight) row_stats(row, y, layer, d.eps, x, mean, rstd);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float s[V], w[V], b[V], g[V];
                scale.get(row, c, s);
                weight.get(row, c, w);
                bias.get(row, c, b);
                if (element) {
                    row.take_chunk(gates, c, g);
                    if (d.gate_sigmoid)
#pragma unroll
                        for (int i = 0; i < V; ++i) g[i] = sigmoid_f32(g[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) g[i] = token;
                }
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (row.in(c * V + i)) o[c * V + i] += s[i] * g[i] * ((y[c * V + i] - mean) * rstd * w[i] + b[i]);
            }
            if (d.out) row.store((E*)d.out + t * d.cols, o);
        } else {
            fetch(t + step);
        }
        if (d.next) {
            row_stats(row, o, layer, d.eps, x, mean2, rstd2);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float w[V], b[V];
                next_weight.get(row, c, w);
                next_bias.get(row, c, b);
#pragma unroll
                for (int i = 0; i < V; ++i) o[c * V + i] = (o[c * V + i] - mean2) * rstd2 * w[i] + b[i];
            }
            row.store((E*)d.next + t * d.cols, o);
        }
        if (d.stats && row.tid == 0) *reinterpret_cast<f32x4*>(d.stats + 4 * t) = f32x4{mean, rstd, mean2, rstd2};
    }
}

// The merge of expert rows and what follows it.  A row's waves take BATCH rows of the merge at a time, the first of them while the row before is normed; the
// rows' numbers and weights come a lane each, another row ahead.  16384 x 2048 bf16, 8 rows a token: 156 us, 4.7 TB/s (164 with the gate's kind looked up in
// the kernel, whose chunk then takes registers in any case).
struct MergeParams {
    int64_t rows, value_rows, y_stride, residual_stride, gate_stride;
    int32_t cols, K, merge_f32, gate_mode, gate_sigmoid;
    float eps, scale_value;
    const void *y, *residual, *gate, *merge, *scale, *weight, *bias, *next_weight, *next_bias;
    const int64_t *reverse_index, *merge_index;
    void *out, *next;
    float *y_out, *stats;
};
template <typename E, bool WHOLE, int CH, bool LAYER, bool P32, int BATCH, bool ELEMENT>
__global__ __launch_bounds__(kNormMostWaves* kWave) void norm_merge_kernel(MergeParams p, int waves) {
    using R = Row<E, WHOLE, CH>;
    constexpr int V = R::V, N = R::N;
    __shared__ float buf[2][kNormMostWaves][4];
    const int per = waves == 1 ? blockDim.x / kWave : 1, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const R row{waves == 1 ? lane : (int)threadIdx.x, waves * kWave, p.cols};
    Exchange x{buf, waves, wave, 0};
    auto param = [&](const void* q, int c, float (&f)[V], float none) { row.param(q, P32 ? FMOE_F32 : FMOE_BF16, c, f, none); };
    const int64_t first = (int64_t)blockIdx.x * per + (waves == 1 ? wave : 0), step = (int64_t)gridDim.x * per;
    int64_t from = -1;
    float share = 0.0f;
    auto number = [&](int64_t t) {
        from = lane < p.K && t < p.rows ? p.reverse_index[t * p.K + lane] : -1;
        if ((uint64_t)from >= (uint64_t)p.value_rows) from = -1;
        share = 1.0f;
        if (from >= 0 && p.merge) {
            const int64_t at = p.merge_index ? p.merge_index[from] : from;
            if ((uint64_t)at >= (uint64_t)p.value_rows) from = -1;
            else share = p.merge_f32 ? reinterpret_cast<const float*>(p.merge)[at] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p.merge)[at]);
        }
    };
    int lo = -1, hi = -1, share_bits = 0;
    typename R::Raw ro, rg, ry[BATCH];
    E token_gate = E(0);
    auto rows = [&](int j0) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {       // (a row that is not there: row 0, and left out of the sum)
            const int at = min(j0 + j, p.K - 1), h = __builtin_amdgcn_readlane(hi, at);
            const int64_t r = h < 0 ? 0 : (int64_t)h << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, at);
            row.fetch((const E*)p.y + r * p.y_stride, ry[j]);
        }
    };
    auto fetch = [&](int64_t t) {
        lo = (int)(uint32_t)from, hi = (int)(from >> 32), share_bits = (int)__float_as_uint(share);
        number(t + step);
        if (t >= p.rows) return;
        row.fetch((const E*)p.residual + t * p.residual_stride, ro);
        if constexpr (ELEMENT) row.fetch((const E*)p.gate + t * p.gate_stride, rg);
        else if (p.gate_mode) token_gate = ((const E*)p.gate)[t * p.gate_stride];
        rows(0);
    };
    number(first);
    fetch(first);
    for (int64_t t = first; t < p.rows; t += step) {
        float y[N], o[N], mean = 0.0f, rstd = 1.0f, mean2 = 0.0f, rstd2 = 1.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = 0.0f;
        for (int j0 = 0; j0 < p.K; j0 += BATCH) {
            if (j0 > 0) rows(j0);
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                if (j0 + j >= p.K || __builtin_amdgcn_readlane(hi, min(j0 + j, p.K - 1)) < 0) continue;
                const float w = __uint_as_float((uint32_t)__builtin_amdgcn_readlane(share_bits, min(j0 + j, p.K - 1)));
                float f[N];
                row.take(ry[j], f);
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = __builtin_fmaf(w, f[i], y[i]);
            }
        }
        row.take(ro, o);
        const typename R::Raw gates = rg;
        float token = p.gate_mode && !ELEMENT ? to_f32(token_gate) : 1.0f;
        if (p.gate_sigmoid && !ELEMENT) token = sigmoid_f32(token);
        fetch(t + step);
        if (p.y_out) row.store_f32(p.y_out + t * p.cols, y);
        if (p.weight) row_stats(row, y, LAYER, p.eps, x, mean, rstd);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float f[V], g[V];
            param(p.weight, c, f, 1.0f);
            param(p.bias, c, g, 0.0f);
#pragma unroll
            for (int i = 0; i < V; ++i) y[c * V + i] = (y[c * V + i] - mean) * rstd * f[i] + g[i];
            param(p.scale, c, f, p.scale_value);
            if constexpr (ELEMENT) {
                row.take_chunk(gates, c, g);
                if (p.gate_sigmoid)
#pragma unroll
                    for (int i = 0; i < V; ++i) g[i] = sigmoid_f32(g[i]);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = token;
            }
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (row.in(c * V + i)) o[c * V + i] += f[i] * g[i] * y[c * V + i];
        }
        if (p.out) row.store((E*)p.out + t * p.cols, o);
        if (p.next) {
            row_stats(row, o, LAYER, p.eps, x, mean2, rstd2);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float f[V], g[V];
                param(p.next_weight, c, f, 0.0f);
                param(p.next_bias, c, g, 0.0f);
#pragma unroll
                for (int i = 0; i < V; ++i) o[c * V + i] = (o[c * V + i] - mean2) * rstd2 * f[i] + g[i];
            }
            row.store((E*)p.next + t * p.cols, o);
        }
        if (p.stats && row.tid == 0) *reinterpret_cast<f32x4*>(p.stats + 4 * t) = f32x4{mean, rstd, mean2, rstd2};
    }
}

// Which of the five sums over rows are asked for, in the order of their partial sums [blocks][5][cols].
enum { kDScale = 0, kDWeight, kDNextWeight, kDBias, kDNextBias, kSums };

// The next row's loads are issued before this row's sums are exchanged.  16384 x 2048 bf16 90 us, 4.5 TB/s, and 5 us for the sums; 3063 x 1001 fp32 layer norms
// with a gate for each element 26 us, 3.8 TB/s, and 6.
// MERGED: y is the merged rows in fp32, and so is d_y (a sum of expert rows against its gradient takes what two roundings would leave out).
template <typename E, bool WHOLE, int CH, bool LAYER, bool ELEMENT, bool MERGED, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_add_bwd_kernel(fmoe_norm_desc d, int waves, float* partial) {
    using R = Row<E, WHOLE, CH>;
    using P = Param<R, CH == 1>;
    constexpr int N = R::N, V = R::V, SUMS = LAYER ? kSums : 3;       // LAYER: a layer norm, or an rms norm with biases
    __shared__ float buf[2][kNormMostWaves][4];
    const int per = waves == 1 ? blockDim.x / kWave : 1, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const R row{waves == 1 ? (int)threadIdx.x % kWave : (int)threadIdx.x, waves * kWave, d.cols};
    Exchange x{buf, waves, wave, 0};
    const float inv = 1.0f / (float)d.cols;
    const bool centred = d.norm == FMOE_NORM_LAYER;
    auto mean_of = [&](float s) { return LAYER && centred ? s * inv : 0.0f; };
    const P scale(row, d.scale, d.param_dtype, d.scale_value), weight(row, d.weight, d.param_dtype, 1.0f), bias(row, LAYER ? d.bias : nullptr, d.param_dtype, 0.0f),
        next_weight(row, d.next_weight, d.param_dtype, 0.0f);
    float sums[SUMS][N];
#pragma unroll
    for (int s = 0; s < SUMS; ++s)
#pragma unroll
        for (int i = 0; i < N; ++i) sums[s][i] = 0.0f;
    const int first = blockIdx.x * per + (waves == 1 ? wave : 0);
    const int64_t step = (int64_t)gridDim.x * per;
    typename R::Raw ry, ro, rn, rt, rg;
    typename R::Raw32 rm;
    f32x4 st;
    E token_gate = E(0);
    auto fetch = [&](int64_t t) {
        if (t >= d.rows) return;
        st = *reinterpret_cast<const f32x4*>(d.stats + 4 * t);
        row.fetch((const E*)d.residual + t * d.residual_stride, ro);
        if constexpr (MERGED) row.fetch_f32((const float*)d.y + t * d.cols, rm);
        else if (d.y) row.fetch((const E*)d.y + t * d.y_stride, ry);
        if (d.d_next) row.fetch((const E*)d.d_next + t * d.cols, rn);
        if (d.d_out) row.fetch((const E*)d.d_out + t * d.cols, rt);
        if constexpr (ELEMENT) row.fetch((const E*)d.gate + t * d.gate_stride, rg);
        else if (d.gate_mode) token_gate = ((const E*)d.gate)[t * d.gate_stride];
    };
    fetch(first);
    for (int64_t t = first; t < d.rows; t += step) {
        const float m = st[0], r = st[1], m2 = st[2], r2 = st[3];
        float a[N], o[N], dn[N], dt[N], gates[ELEMENT ? N : 1];
        row.take(ro, o);
        if constexpr (MERGED) row.take_f32(rm, a);
        else if (d.y) row.take(ry, a);
        if (d.d_next) row.take(rn, dn);
        if (d.d_out) row.take(rt, dt);
        else
#pragma unroll
            for (int i = 0; i < N; ++i) dt[i] = 0.0f;
        if constexpr (ELEMENT) {
            row.take(rg, gates);
            if (d.gate_sigmoid)
#pragma unroll
                for (int i = 0; i < N; ++i) gates[i] = sigmoid_f32(gates[i]);
        } else {
            gates[0] = d.gate_mode ? to_f32(token_gate) : 1.0f;
            if (d.gate_mode && d.gate_sigmoid) gates[0] = sigmoid_f32(gates[0]);
        }
        fetch(t + step);
        auto gate = [&](int i) { return gates[ELEMENT ? i : 0]; };
        if (d.y) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float s[V], w[V], b[V];
                scale.get(row, c, s);
                weight.get(row, c, w);
                if constexpr (LAYER) bias.get(row, c, b);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int i = c * V + j;
                    a[i] = row.in(i) ? (a[i] - m) * r : 0.0f;
                    if (row.in(i)) o[i] += s[j] * gate(i) * (a[i] * w[j] + (LAYER ? b[j] : 0.0f));
                }
            }
        }
        if (d.d_next) {
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float w[V];
                next_weight.get(row, c, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int i = c * V + j;
                    o[i] = row.in(i) ? (o[i] - m2) * r2 : 0.0f;
                    sums[kDNextWeight][i] += dn[i] * o[i];
                    if constexpr (LAYER) sums[kDNextBias][i] += dn[i];
                    dn[i] *= w[j];
                    s[0] += dn[i] * o[i];
                    if constexpr (LAYER) s[1] += dn[i];
                }
            }
            x.sum(s);
#pragma unroll
            for (int i = 0; i < N; ++i) dt[i] += r2 * (dn[i] - o[i] * (s[0] * inv) - mean_of(s[1]));
        }
        if (d.d_residual) row.store((E*)d.d_residual + t * d.cols, dt);
        if (d.y) {
            float q[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float s[V], w[V], b[V];
                scale.get(row, c, s);
                weight.get(row, c, w);
                if constexpr (LAYER) bias.get(row, c, b);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int i = c * V + j;
                    const float z = a[i] * w[j] + (LAYER ? b[j] : 0.0f), g = gate(i), dsz = dt[i] * s[j], dz = dsz * g, da = dz * w[j];
                    sums[kDScale][i] += dt[i] * g * z;
                    sums[kDWeight][i] += dz * a[i];
                    if constexpr (LAYER) sums[kDBias][i] += dz;
                    float dg = dsz * z;
                    if (d.gate_sigmoid) dg *= g * (1.0f - g);
                    if (row.in(i)) {
                        q[0] += da * a[i];
                        if constexpr (LAYER) q[1] += da;
                        if constexpr (!ELEMENT) q[2] += dg;
                    }
                    dt[i] = da;
                    if constexpr (ELEMENT) gates[i] = dg;
                }
            }
            if (d.weight || d.gate_mode == FMOE_GATE_TOKEN) x.sum(q);
            if (d.d_gate) {
                if constexpr (ELEMENT) row.store((E*)d.d_gate + t * d.cols, gates);
                else if (row.tid == 0) from_f32((E*)d.d_gate + t, q[2]);
            }
            if (d.d_y) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (d.weight) dt[i] = r * (dt[i] - a[i] * (q[0] * inv) - mean_of(q[1]));
                if constexpr (MERGED) row.store_f32((float*)d.d_y + t * d.cols, dt);
                else row.store((E*)d.d_y + t * d.cols, dt);
            }
        }
    }
    if (partial) {      // a group without a row leaves zeros
        float* const at = partial + (int64_t)first * kSums * d.cols;
        void* const want[kSums] = {d.d_scale, d.d_weight, d.d_next_weight, d.d_bias, d.d_next_bias};
#pragma unroll
        for (int s = 0; s < SUMS; ++s)
            if (want[s]) row.store_f32(at + (int64_t)s * d.cols, sums[s]);
    }
}

// What d_y [rows, cols] of the merged rows (fp32) gives the routed rows, a wave to each: d_value[r] = w_r * d_y[token], and <value[r], d_y[token]> for its weight.
struct MergeBwdParams {
    const float* d_y;
    const void* value;
    int64_t rows, value_rows, value_stride;
    const int64_t *token_index, *merge_index;
    const void* merge;
    int32_t cols, merge_f32;
    void* d_value;
    float* d_merge;
};
template <typename E, bool WHOLE>
__global__ __launch_bounds__(256) void norm_merge_bwd_kernel(MergeBwdParams p) {
    using R = Row<E, WHOLE, 1>;
    constexpr int N = R::N, STEP = kWave * N;
    const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (r >= p.value_rows) return;
    const int64_t t = p.token_index[r], flat = p.merge_index ? p.merge_index[r] : r;
    const bool named = (uint64_t)t < (uint64_t)p.rows, weighted = (uint64_t)flat < (uint64_t)p.value_rows;
    float w = 1.0f, dot = 0.0f;
    if (p.merge) w = !weighted ? 0.0f : p.merge_f32 ? reinterpret_cast<const float*>(p.merge)[flat] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p.merge)[flat]);
    for (int c = 0; c < p.cols; c += STEP) {
        const R row{lane_id(), kWave, p.cols - c};
        typename R::Raw32 raw;
        typename R::Raw rv;
        float d[N], v[N];
        if (p.d_merge) row.fetch((const E*)p.value + r * p.value_stride + c, rv);
        row.fetch_f32(p.d_y + (named ? t : 0) * p.cols + c, raw);
        row.take_f32(raw, d);
        if (p.d_merge) {
            row.take(rv, v);
#pragma unroll
            for (int i = 0; i < N; ++i) dot = __builtin_fmaf(v[i], d[i], dot);
        }
        if (p.d_value) {
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = named ? w * d[i] : 0.0f;
            row.store((E*)p.d_value + r * p.cols + c, d);
        }
    }
    if (p.d_merge) {
        dot = wave_sum(dot);
        if (lane_id() == 0 && weighted) p.d_merge[flat] = named ? dot : 0.0f;
    }
}

// The groups' partial sums added in order: 32 columns a block, its 32 half waves share the groups.
constexpr int kSumWaves = 16, kSumCols = 32;
__global__ __launch_bounds__(kSumWaves* kWave) void norm_sums_kernel(fmoe_norm_desc d, const float* partial, int groups) {
    __shared__ float part[2 * kSumWaves][kSumCols];
    const int lane = threadIdx.x % kSumCols, share = threadIdx.x / kSumCols, which = blockIdx.y, col = blockIdx.x * kSumCols + lane;
    void* const to[kSums] = {d.d_scale, d.d_weight, d.d_next_weight, d.d_bias, d.d_next_bias};
    void* out = nullptr;
#pragma unroll
    for (int s = 0; s < kSums; ++s)
        if (which == s) out = to[s];
    if (!out) return;
    const int per = (groups + 2 * kSumWaves - 1) / (2 * kSumWaves), from = share * per, until = min(groups, from + per);
    float v = 0.0f;
    if (col < d.cols) {
        const float* const at = partial + (int64_t)which * d.cols + col;
        int g = from;
        for (; g + 8 <= until; g += 8) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = at[(int64_t)(g + i) * kSums * d.cols];
#pragma unroll
            for (int i = 0; i < 8; ++i) v += p[i];
        }
        for (; g < until; ++g) v += at[(int64_t)g * kSums * d.cols];
    }
    part[share][lane] = v;
    __syncthreads();
    if (share == 0 && col < d.cols) {
#pragma unroll
        for (int w = 1; w < 2 * kSumWaves; ++w) v += part[w][lane];
        if (d.param_dtype == FMOE_F32) reinterpret_cast<float*>(out)[col] = v;
        else reinterpret_cast<uint16_t*>(out)[col] = (uint16_t)f32_to_bf16_bits(v);
    }
}

constexpr int kNormMostCols = 8192, kNormBwdWaves = 8;

struct NormPlan {
    bool whole;
    int chunks, waves, per, threads;
};
// Chunks of a lane and waves of a row: one chunk, the row spread over as many lanes as it has chunks, as far as 16 waves (8 in the backward pass, whose
// sums over rows take registers) go.  A row per wave of four chunks each, with no barrier, was slower: 16384 x 2048 bf16 forward 97 us against 67 (the
// parameters are asked for again for every row, and 245 registers leave two waves to a SIMD).
NormPlan norm_plan(const fmoe_norm_desc& d, bool backward) {
    const int v = d.dtype == FMOE_F32 ? 4 : 8;
    NormPlan p;
    p.whole = d.cols % v == 0;
    const int lanes = (d.cols + v - 1) / v;                      // one chunk each
    auto waves = [&](int chunks) { return (lanes + chunks * kWave - 1) / (chunks * kWave); };
    p.chunks = 1;
    if (backward) {
        while (waves(p.chunks) > (p.whole ? kNormBwdWaves : kNormMostWaves)) p.chunks *= 2;
    } else if (waves(1) > kNormMostWaves) {
        p.chunks = 2;
    }
    p.waves = waves(p.chunks);
    p.per = p.waves == 1 ? 4 : 1;
    p.threads = (p.waves == 1 ? 4 : p.waves) * kWave;
    return p;
}
// Groups (blocks, or waves where a wave has a row) of the backward pass: as many as the chip holds at once
int norm_groups(const fmoe_norm_desc& d, const NormPlan& p) {
    const int64_t most = 256 * 12 / p.waves;
    return (int)(d.rows < most ? d.rows : most);
}

int norm_check(const fmoe_norm_desc* d, bool backward) {
    const char* const name = backward ? "fmoe_norm_add_bwd" : "fmoe_norm_add";
    FMOE_REQUIRE(d, "%s: desc is NULL", name);
    FMOE_REQUIRE(d->rows >= 0 && d->cols >= 1 && d->cols <= kNormMostCols, "%s: rows >= 0 and 1 to %d columns expected, got %lld, %d", name, kNormMostCols,
                 (long long)d->rows, d->cols);
    FMOE_REQUIRE(d->dtype == FMOE_F32 || d->dtype == FMOE_BF16, "%s: bf16 or fp32 expected", name);
    FMOE_REQUIRE(d->param_dtype == FMOE_F32 || d->param_dtype == FMOE_BF16, "%s: parameters must be bf16 or fp32", name);
    FMOE_REQUIRE(d->norm == FMOE_NORM_RMS || d->norm == FMOE_NORM_LAYER, "%s: unknown norm %d", name, d->norm);
    FMOE_REQUIRE(d->gate_mode >= FMOE_GATE_NONE && d->gate_mode <= FMOE_GATE_ELEMENT, "%s: unknown gate mode %d", name, d->gate_mode);
    FMOE_REQUIRE(d->weight || !d->bias, "%s: bias goes with weight", name);
    FMOE_REQUIRE(d->next_weight || !d->next_bias, "%s: next_bias goes with next_weight", name);
    if (d->rows == 0) return FMOE_OK;
    FMOE_REQUIRE(d->residual && d->residual_stride >= 0, "%s: residual is missing", name);
    FMOE_REQUIRE(!d->gate_mode || (d->gate && d->y), "%s: a gate needs its tensor and y", name);
    FMOE_REQUIRE(d->K >= 0 && d->K <= 64 && (!d->K || (d->y && (backward || d->reverse_index) && d->value_rows == d->rows * d->K)),
                 "%s: a merge needs y [rows * K, cols] and reverse_index, K <= 64", name);
    FMOE_REQUIRE(!d->merge || d->merge_dtype == FMOE_F32 || d->merge_dtype == FMOE_BF16, "%s: merge weights must be bf16 or fp32", name);
    FMOE_REQUIRE(!d->stats || aligned16(d->stats), "%s: stats must be 16-byte aligned", name);
    if (!backward) {
        FMOE_REQUIRE(d->next ? d->next_weight != nullptr : d->out != nullptr, "%s: nothing to write", name);
        FMOE_REQUIRE(d->y || !d->out, "%s: out without y is the residual", name);
    } else {
        FMOE_REQUIRE(!d->K || (d->y_out && d->token_index), "%s: a merge needs the merged rows of the forward pass and token_index", name);
        FMOE_REQUIRE((d->K && d->merge) || !d->d_merge, "%s: the gradient of an operand that is not there", name);
        FMOE_REQUIRE(d->stats && (d->d_next || d->d_out), "%s: needs the forward pass's stats and a gradient", name);
        FMOE_REQUIRE(!d->d_next || d->next_weight, "%s: d_next needs next_weight", name);
        FMOE_REQUIRE((d->y || !(d->d_y || d->d_gate || d->d_scale || d->d_weight || d->d_bias)) && (d->gate_mode || !d->d_gate) && (d->scale || !d->d_scale) &&
                         (d->weight || !d->d_weight) && (d->bias || !d->d_bias) && (d->next_weight || !d->d_next_weight) && (d->next_bias || !d->d_next_bias),
                     "%s: the gradient of an operand that is not there", name);
    }
    return FMOE_OK;
}

template <typename F>
void with_bool(bool b, F&& f) {
    if (b) f(std::true_type());
    else f(std::false_type());
}

bool norm_wants_sums(const fmoe_norm_desc& d) { return d.d_scale || d.d_weight || d.d_bias || d.d_next_weight || d.d_next_bias; }

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_norm_add(const fmoe_norm_desc* desc, fmoe_stream_t stream) {
    const int rc = norm_check(desc, false);
    if (rc != FMOE_OK || desc->rows == 0) return rc;
    const fmoe_norm_desc& d = *desc;
    const NormPlan p = norm_plan(d, false);
    const int64_t blocks = (d.rows + p.per - 1) / p.per, most = 256 * 16 / (p.threads / kWave);
    auto go = [&](auto kern) { kern<<<(unsigned)(blocks < most ? blocks : most), p.threads, 0, (hipStream_t)stream>>>(d, p.waves); };
    if (d.K) {
        const MergeParams m{d.rows, d.value_rows, d.y_stride, d.residual_stride, d.gate_stride, d.cols, d.K, d.merge_dtype == FMOE_F32, d.gate_mode,
                            d.gate_mode && d.gate_sigmoid, d.eps, d.scale_value, d.y, d.residual, d.gate, d.merge, d.scale, d.weight, d.bias, d.next_weight, d.next_bias,
                            d.reverse_index, d.merge_index, d.out, d.next, d.y_out, d.stats};
        auto run = [&](auto kern) { kern<<<(unsigned)(blocks < most ? blocks : most), p.threads, 0, (hipStream_t)stream>>>(m, p.waves); };
        auto of = [&](auto value, auto whole, auto layer, auto p32, auto element) {
            using E = decltype(value);
            constexpr bool WHOLE = decltype(whole)::value, LAYER = decltype(layer)::value, P32 = decltype(p32)::value, ELEMENT = decltype(element)::value;
            if constexpr (sizeof(E) == 4) {
                if (p.chunks == 2) return run(norm_merge_kernel<E, WHOLE, 2, LAYER, P32, 2, ELEMENT>);
            }
            if constexpr (WHOLE) {
                if (d.K <= 2) return run(norm_merge_kernel<E, WHOLE, 1, LAYER, P32, 2, ELEMENT>);
                if (d.K > 4) return run(norm_merge_kernel<E, WHOLE, 1, LAYER, P32, 8, ELEMENT>);
            }
            // (a row read element by element takes a register for every one)
            run(norm_merge_kernel<E, WHOLE, 1, LAYER, P32, WHOLE || sizeof(E) == 4 ? 4 : 2, ELEMENT>);
        };
        with_bool(p.whole, [&](auto whole) {
            with_bool(d.norm == FMOE_NORM_LAYER, [&](auto layer) {
                with_bool(d.param_dtype == FMOE_F32, [&](auto p32) {
                    with_bool(d.gate_mode == FMOE_GATE_ELEMENT, [&](auto element) {
                        if (d.dtype == FMOE_F32) of(float(), whole, layer, p32, element);
                        else of(uint16_t(), whole, layer, p32, element);
                    });
                });
            });
        });
        return check_launch("fmoe_norm_add");
    }
    with_bool(p.whole, [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        if (d.dtype == FMOE_BF16) go(norm_add_kernel<uint16_t, WHOLE, 1>);
        else if (p.chunks == 1) go(norm_add_kernel<float, WHOLE, 1>);
        else go(norm_add_kernel<float, WHOLE, 2>);
    });
    return check_launch("fmoe_norm_add");
}

// The workspace of the backward pass: the sums' partial ones, and d_y of the merged rows.
static size_t norm_partial_bytes(const fmoe_norm_desc& d) {
    if (!norm_wants_sums(d)) return 0;
    const NormPlan p = norm_plan(d, true);
    const int64_t groups = norm_groups(d, p), all = (groups + p.per - 1) / p.per * p.per;
    return ((size_t)all * kSums * d.cols * sizeof(float) + 255) & ~(size_t)255;
}

extern "C" size_t fmoe_norm_add_bwd_workspace_bytes(const fmoe_norm_desc* desc) {
    if (norm_check(desc, true) != FMOE_OK || desc->rows == 0) return 0;
    return norm_partial_bytes(*desc) + (desc->K && (desc->d_y || desc->d_merge) ? (size_t)desc->rows * desc->cols * sizeof(float) : 0);
}

extern "C" int fmoe_norm_add_bwd(const fmoe_norm_desc* desc, void* workspace, size_t workspace_bytes, fmoe_stream_t stream) {
    const int rc = norm_check(desc, true);
    if (rc != FMOE_OK || desc->rows == 0) return rc;
    const size_t need = fmoe_norm_add_bwd_workspace_bytes(desc), sums = norm_partial_bytes(*desc);
    if (need && (!workspace || workspace_bytes < need))
        return fail(FMOE_ERR_WORKSPACE, "fmoe_norm_add_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    FMOE_REQUIRE(!need || aligned16(workspace), "fmoe_norm_add_bwd: the workspace must be 16-byte aligned");
    fmoe_norm_desc d = *desc;
    const NormPlan p = norm_plan(d, true);
    float* const partial = sums ? (float*)workspace : nullptr;
    if (d.K) {
        d.y = d.y_out;
        d.d_y = d.d_y || d.d_merge ? (uint8_t*)workspace + sums : nullptr;
    }
    const int blocks = (norm_groups(d, p) + p.per - 1) / p.per;
    auto go = [&](auto kern) { kern<<<blocks, p.threads, 0, (hipStream_t)stream>>>(d, p.waves, partial); };
    with_bool(p.whole, [&](auto whole) {
        with_bool(d.norm == FMOE_NORM_LAYER || d.bias || d.next_bias, [&](auto layer) {
            with_bool(d.gate_mode == FMOE_GATE_ELEMENT, [&](auto element) {
                with_bool(d.K > 0, [&](auto merged) {
                    constexpr bool WHOLE = decltype(whole)::value, LAYER = decltype(layer)::value, ELEMENT = decltype(element)::value, MERGED = decltype(merged)::value;
                    constexpr int THREADS = WHOLE ? kNormBwdWaves * kWave : kNormMostWaves * kWave;
                    if (d.dtype == FMOE_F32) {
                        if (p.chunks == 1) go(norm_add_bwd_kernel<float, WHOLE, 1, LAYER, ELEMENT, MERGED, THREADS>);
                        else if (p.chunks == 2) go(norm_add_bwd_kernel<float, WHOLE, 2, LAYER, ELEMENT, MERGED, THREADS>);
                        else if constexpr (WHOLE) go(norm_add_bwd_kernel<float, WHOLE, 4, LAYER, ELEMENT, MERGED, THREADS>);
                    } else {
                        if (p.chunks == 1 && p.waves <= kNormBwdWaves) go(norm_add_bwd_kernel<uint16_t, WHOLE, 1, LAYER, ELEMENT, MERGED, kNormBwdWaves * kWave>);
                        else if (p.chunks == 1) go(norm_add_bwd_kernel<uint16_t, WHOLE, 1, LAYER, ELEMENT, MERGED, THREADS>);
                        else if constexpr (WHOLE) go(norm_add_bwd_kernel<uint16_t, WHOLE, 2, LAYER, ELEMENT, MERGED, THREADS>);
                    }
                });
            });
        });
    });
    int launched = check_launch("fmoe_norm_add_bwd");
    if (launched == FMOE_OK && d.K && d.d_y) {
        const MergeBwdParams m{(const float*)d.d_y, desc->y, d.rows, d.value_rows, d.y_stride, d.token_index, d.merge_index, d.merge, d.cols, d.merge_dtype == FMOE_F32,
                               desc->d_y, d.d_merge};
        const unsigned rows = (unsigned)((d.value_rows + 3) / 4);
        with_bool(p.whole, [&](auto whole) {
            if (d.dtype == FMOE_F32) norm_merge_bwd_kernel<float, decltype(whole)::value><<<rows, 256, 0, (hipStream_t)stream>>>(m);
            else norm_merge_bwd_kernel<uint16_t, decltype(whole)::value><<<rows, 256, 0, (hipStream_t)stream>>>(m);
        });
        launched = check_launch("fmoe_norm_add_bwd");
    }
    if (launched != FMOE_OK || !partial) return launched;
    norm_sums_kernel<<<dim3((d.cols + kSumCols - 1) / kSumCols, kSums), kSumWaves * kWave, 0, (hipStream_t)stream>>>(d, partial, blocks * p.per);
    return check_launch("fmoe_norm_add_bwd");
}
