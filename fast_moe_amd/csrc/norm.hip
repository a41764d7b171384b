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

// Which columns a lane holds: VEC: chunks of V neighbours, 16 bytes; otherwise single ones, neighbours in neighbouring lanes.
template <typename E, bool VEC, int CH>
struct Row {
    static constexpr int V = NE<E>::V, N = V * CH;
    int tid, threads, cols;
    __device__ __forceinline__ int col(int i) const {
        return VEC ? ((i / V) * threads + tid) * V + i % V : i * threads + tid;
    }
    __device__ __forceinline__ bool in(int i) const { return col(i) < cols; }       // (VEC: all of a chunk or none)
    __device__ __forceinline__ void load(const E* p, float (&f)[N]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                u32x4 v = {0, 0, 0, 0};
                if (in(c * V)) v = *reinterpret_cast<const u32x4*>(p + col(c * V));
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if constexpr (V == 4) f[c * V + i] = __uint_as_float(v[i]);
                    else f[c * V + i] = i & 1 ? __uint_as_float(v[i / 2] & 0xffff0000u) : __uint_as_float(v[i / 2] << 16);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = in(i) ? to_f32(p[col(i)]) : 0.0f;
        }
    }
    __device__ __forceinline__ void store(E* p, const float (&f)[N]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (!in(c * V)) continue;
                u32x4 v;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (V == 4) v[i] = __float_as_uint(f[c * V + i]);
                    else v[i] = cvt_pk_bf16(f[c * V + 2 * i], f[c * V + 2 * i + 1]);
                }
                *reinterpret_cast<u32x4*>(p + col(c * V)) = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (in(i)) from_f32(p + col(i), f[i]);
        }
    }
    // a parameter of the columns, in fp32 or bf16 whatever the rows are
    __device__ __forceinline__ void param(const void* p, int dtype, float (&f)[N], float none) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            f[i] = none;
            if (p && in(i)) f[i] = dtype == FMOE_F32 ? reinterpret_cast<const float*>(p)[col(i)] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[col(i)]);
        }
    }
    __device__ __forceinline__ void store_f32(float* p, const float (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (in(i)) p[col(i)] = f[i];
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

template <typename E, bool VEC, int CH>
__global__ __launch_bounds__(kNormMostWaves* kWave) void norm_add_kernel(fmoe_norm_desc d, int waves) {
    using R = Row<E, VEC, CH>;
    constexpr int N = R::N;
    __shared__ float buf[2][kNormMostWaves][4];
    const int per = waves == 1 ? blockDim.x / kWave : 1, wave = threadIdx.x / kWave;       // rows of a block at a time
    const R row{waves == 1 ? (int)threadIdx.x % kWave : (int)threadIdx.x, waves * kWave, d.cols};
    Exchange x{buf, waves, wave, 0};
    const bool layer = d.norm == FMOE_NORM_LAYER;
    float scale[N], weight[N], bias[N], next_w[N], next_b[N];
    row.param(d.scale, d.param_dtype, scale, d.scale_value);
    row.param(d.weight, d.param_dtype, weight, 1.0f);
    row.param(d.bias, d.param_dtype, bias, 0.0f);
    row.param(d.next_weight, d.param_dtype, next_w, 0.0f);
    row.param(d.next_bias, d.param_dtype, next_b, 0.0f);
    for (int64_t t = (int64_t)blockIdx.x * per + (waves == 1 ? wave : 0); t < d.rows; t += (int64_t)gridDim.x * per) {
        float o[N], y[N], mean = 0.0f, rstd = 1.0f, mean2 = 0.0f, rstd2 = 1.0f;
        row.load((const E*)d.residual + t * d.residual_stride, o);
        if (d.y) {
            if (d.K) {
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = 0.0f;
                for (int j = 0; j < d.K; ++j) {
                    const int64_t r = d.reverse_index[t * d.K + j];
                    if ((uint64_t)r >= (uint64_t)d.value_rows) continue;
                    float w = 1.0f;
                    if (d.merge) {
                        const int64_t at = d.merge_index ? d.merge_index[r] : r;
                        if ((uint64_t)at >= (uint64_t)d.value_rows) continue;
                        w = d.merge_dtype == FMOE_F32 ? reinterpret_cast<const float*>(d.merge)[at]
                                                      : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(d.merge)[at]);
                    }
                    float v[N];
                    row.load((const E*)d.y + r * d.y_stride, v);
#pragma unroll
                    for (int i = 0; i < N; ++i) y[i] = __builtin_fmaf(w, v[i], y[i]);
                }
                if (d.y_out) row.store((E*)d.y_out + t * d.cols, y);
            } else {
                row.load((const E*)d.y + t * d.y_stride, y);
            }
            if (d.weight) row_stats(row, y, layer, d.eps, x, mean, rstd);
            float gate[N];
            if (d.gate_mode == FMOE_GATE_ELEMENT) {
                row.load((const E*)d.gate + t * d.gate_stride, gate);
            } else {
                const float g = d.gate_mode == FMOE_GATE_TOKEN ? to_f32(((const E*)d.gate)[t * d.gate_stride]) : 1.0f;
#pragma unroll
                for (int i = 0; i < N; ++i) gate[i] = g;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float g = d.gate_mode && d.gate_sigmoid ? sigmoid_f32(gate[i]) : gate[i];
                const float z = (y[i] - mean) * rstd * weight[i] + bias[i];
                if (row.in(i)) o[i] += scale[i] * g * z;
            }
            if (d.out) row.store((E*)d.out + t * d.cols, o);
        }
        if (d.next) {
            row_stats(row, o, layer, d.eps, x, mean2, rstd2);
            float n[N];
#pragma unroll
            for (int i = 0; i < N; ++i) n[i] = (o[i] - mean2) * rstd2 * next_w[i] + next_b[i];
            row.store((E*)d.next + t * d.cols, n);
        }
        if (d.stats && row.tid == 0) *reinterpret_cast<f32x4*>(d.stats + 4 * t) = f32x4{mean, rstd, mean2, rstd2};
    }
}

// Which of the five sums over rows are asked for, in the order of their partial sums [blocks][5][cols].
enum { kDScale = 0, kDWeight, kDBias, kDNextWeight, kDNextBias, kSums };

template <typename E, bool VEC, int CH>
__global__ __launch_bounds__(kNormMostWaves* kWave) void norm_add_bwd_kernel(fmoe_norm_desc d, int waves, float* partial) {
    using R = Row<E, VEC, CH>;
    constexpr int N = R::N;
    __shared__ float buf[2][kNormMostWaves][4];
    const int per = waves == 1 ? blockDim.x / kWave : 1, wave = threadIdx.x / kWave;
    const R row{waves == 1 ? (int)threadIdx.x % kWave : (int)threadIdx.x, waves * kWave, d.cols};
    Exchange x{buf, waves, wave, 0};
    const bool layer = d.norm == FMOE_NORM_LAYER;
    const float inv = 1.0f / (float)d.cols;
    float scale[N], weight[N], bias[N], next_w[N], sums[kSums][N];
    row.param(d.scale, d.param_dtype, scale, d.scale_value);
    row.param(d.weight, d.param_dtype, weight, 1.0f);
    row.param(d.bias, d.param_dtype, bias, 0.0f);
    row.param(d.next_weight, d.param_dtype, next_w, 0.0f);
#pragma unroll
    for (int s = 0; s < kSums; ++s)
#pragma unroll
        for (int i = 0; i < N; ++i) sums[s][i] = 0.0f;
    const int first = blockIdx.x * per + (waves == 1 ? wave : 0);
    for (int64_t t = first; t < d.rows; t += (int64_t)gridDim.x * per) {
        const f32x4 st = *reinterpret_cast<const f32x4*>(d.stats + 4 * t);
        float a[N], o[N], gate[N], dn[N], dt[N];
        row.load((const E*)d.residual + t * d.residual_stride, o);
        if (d.y) row.load((const E*)d.y + t * d.y_stride, a);
        if (d.d_next) row.load((const E*)d.d_next + t * d.cols, dn);
        if (d.d_out) row.load((const E*)d.d_out + t * d.cols, dt);
        if (!d.d_out)
#pragma unroll
            for (int i = 0; i < N; ++i) dt[i] = 0.0f;
        if (d.y) {
            if (d.gate_mode == FMOE_GATE_ELEMENT) {
                row.load((const E*)d.gate + t * d.gate_stride, gate);
            } else {
                const float g = d.gate_mode == FMOE_GATE_TOKEN ? to_f32(((const E*)d.gate)[t * d.gate_stride]) : 1.0f;
#pragma unroll
                for (int i = 0; i < N; ++i) gate[i] = g;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (d.gate_mode && d.gate_sigmoid) gate[i] = sigmoid_f32(gate[i]);
                a[i] = row.in(i) ? (a[i] - st[0]) * st[1] : 0.0f;
                if (row.in(i)) o[i] += scale[i] * gate[i] * (a[i] * weight[i] + bias[i]);
            }
        }
        if (d.d_next) {
            float s[2] = {0.0f, 0.0f}, b[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                b[i] = row.in(i) ? (o[i] - st[2]) * st[3] : 0.0f;
                sums[kDNextWeight][i] += dn[i] * b[i];
                sums[kDNextBias][i] += dn[i];
                dn[i] *= next_w[i];
                s[0] += dn[i] * b[i];
                s[1] += dn[i];
            }
            x.sum(s);
#pragma unroll
            for (int i = 0; i < N; ++i) dt[i] += st[3] * (dn[i] - b[i] * (s[0] * inv) - (layer ? s[1] * inv : 0.0f));
        }
        if (d.d_residual) row.store((E*)d.d_residual + t * d.cols, dt);
        if (d.y) {
            float s[3] = {0.0f, 0.0f, 0.0f}, dz[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float z = a[i] * weight[i] + bias[i], dsz = dt[i] * scale[i];
                dz[i] = dsz * gate[i];
                sums[kDScale][i] += dt[i] * gate[i] * z;
                sums[kDWeight][i] += dz[i] * a[i];
                sums[kDBias][i] += dz[i];
                const float da = dz[i] * weight[i];
                float dg = dsz * z;
                if (d.gate_sigmoid) dg *= gate[i] * (1.0f - gate[i]);
                if (row.in(i)) {
                    s[0] += da * a[i];
                    s[1] += da;
                    s[2] += dg;
                }
                dz[i] = da;
                gate[i] = dg;
            }
            if (d.weight || d.gate_mode == FMOE_GATE_TOKEN) x.sum(s);
            if (d.d_gate) {
                if (d.gate_mode == FMOE_GATE_ELEMENT) row.store((E*)d.d_gate + t * d.cols, gate);
                else if (row.tid == 0) from_f32((E*)d.d_gate + t, s[2]);
            }
            if (d.d_y) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (d.weight) dz[i] = st[1] * (dz[i] - a[i] * (s[0] * inv) - (layer ? s[1] * inv : 0.0f));
                row.store((E*)d.d_y + t * d.cols, dz);
            }
        }
    }
    if (partial) {      // a group without a row leaves zeros
        float* const at = partial + (int64_t)first * kSums * d.cols;
        void* const want[kSums] = {d.d_scale, d.d_weight, d.d_bias, d.d_next_weight, d.d_next_bias};
#pragma unroll
        for (int s = 0; s < kSums; ++s)
            if (want[s]) row.store_f32(at + (int64_t)s * d.cols, sums[s]);
    }
}

// The groups' partial sums added in order: 64 columns a block, its waves share the groups.
constexpr int kSumWaves = 8;
__global__ __launch_bounds__(kSumWaves* kWave) void norm_sums_kernel(fmoe_norm_desc d, const float* partial, int groups) {
    __shared__ float part[kSumWaves][kWave];
    const int lane = lane_id(), wave = threadIdx.x / kWave, which = blockIdx.y, col = blockIdx.x * kWave + lane;
    void* const to[kSums] = {d.d_scale, d.d_weight, d.d_bias, d.d_next_weight, d.d_next_bias};
    void* out = nullptr;
#pragma unroll
    for (int s = 0; s < kSums; ++s)
        if (which == s) out = to[s];
    if (!out) return;
    const int per = (groups + kSumWaves - 1) / kSumWaves, from = wave * per, until = min(groups, from + per);
    float v = 0.0f;
    if (col < d.cols)
        for (int g = from; g < until; ++g) v += partial[((int64_t)g * kSums + which) * d.cols + col];
    part[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && col < d.cols) {
#pragma unroll
        for (int w = 1; w < kSumWaves; ++w) v += part[w][lane];
        if (d.param_dtype == FMOE_F32) reinterpret_cast<float*>(out)[col] = v;
        else reinterpret_cast<uint16_t*>(out)[col] = (uint16_t)f32_to_bf16_bits(v);
    }
}

constexpr int kNormMostCols = 8192;

struct NormPlan {
    bool vec;
    int chunks, waves, per, threads;
};
NormPlan norm_plan(const fmoe_norm_desc& d) {
    const int v = d.dtype == FMOE_F32 ? 4 : 8, es = d.dtype == FMOE_F32 ? 4 : 2;
    auto whole = [&](const void* p, int64_t stride) { return aligned16(p) && stride * es % 16 == 0; };
    NormPlan p;
    p.vec = d.cols % v == 0 && whole(d.y, d.y_stride) && whole(d.residual, d.residual_stride) && whole(d.out, 0) && whole(d.next, 0) && whole(d.y_out, 0) &&
            (d.gate_mode != FMOE_GATE_ELEMENT || whole(d.gate, d.gate_stride)) && whole(d.d_out, 0) && whole(d.d_next, 0) && whole(d.d_y, 0) &&
            whole(d.d_residual, 0) && (d.gate_mode != FMOE_GATE_ELEMENT || whole(d.d_gate, 0));
    const int lanes = (d.cols + v - 1) / v;                      // one chunk each
    p.chunks = lanes <= kNormMostWaves * kWave ? 1 : 2;
    p.waves = (lanes + p.chunks * kWave - 1) / (p.chunks * kWave);
    p.per = p.waves == 1 ? 4 : 1;
    p.threads = (p.waves == 1 ? 4 : p.waves) * kWave;
    return p;
}
// Groups (blocks, or waves where a wave has a row) of the backward pass: as many as the chip holds at once, fewer where that is many partial sums to a row
int norm_groups(const fmoe_norm_desc& d, const NormPlan& p) {
    const int64_t most = p.waves == 1 ? 2048 : 1024;
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
    FMOE_REQUIRE(d->K >= 0 && d->K <= 64 && (!d->K || (d->y && d->reverse_index && d->value_rows == d->rows * d->K)),
                 "%s: a merge needs y [rows * K, cols] and reverse_index, K <= 64", name);
    FMOE_REQUIRE(!d->merge || d->merge_dtype == FMOE_F32 || d->merge_dtype == FMOE_BF16, "%s: merge weights must be bf16 or fp32", name);
    FMOE_REQUIRE(!d->stats || aligned16(d->stats), "%s: stats must be 16-byte aligned", name);
    if (!backward) {
        FMOE_REQUIRE(d->next ? d->next_weight != nullptr : d->out != nullptr, "%s: nothing to write", name);
        FMOE_REQUIRE(d->y || !d->out, "%s: out without y is the residual", name);
    } else {
        FMOE_REQUIRE(!d->K, "%s: takes the merged y", name);
        FMOE_REQUIRE(d->stats && (d->d_next || d->d_out), "%s: needs the forward pass's stats and a gradient", name);
        FMOE_REQUIRE(!d->d_next || d->next_weight, "%s: d_next needs next_weight", name);
        FMOE_REQUIRE((d->y || !(d->d_y || d->d_gate || d->d_scale || d->d_weight || d->d_bias)) && (d->gate_mode || !d->d_gate) && (d->scale || !d->d_scale) &&
                         (d->weight || !d->d_weight) && (d->bias || !d->d_bias) && (d->next_weight || !d->d_next_weight) && (d->next_bias || !d->d_next_bias),
                     "%s: the gradient of an operand that is not there", name);
    }
    return FMOE_OK;
}

bool norm_wants_sums(const fmoe_norm_desc& d) { return d.d_scale || d.d_weight || d.d_bias || d.d_next_weight || d.d_next_bias; }

}  // namespace
}  // namespace fmoe

using namespace fmoe;

#define FMOE_NORM(kern, ...)                                                                                             \
    do {                                                                                                                 \
        if (d.dtype == FMOE_F32) {                                                                                       \
            if (p.vec) { if (p.chunks == 1) kern<float, true, 1> __VA_ARGS__; else kern<float, true, 2> __VA_ARGS__; }   \
            else { if (p.chunks == 1) kern<float, false, 1> __VA_ARGS__; else kern<float, false, 2> __VA_ARGS__; }       \
        } else {                                                                                                         \
            if (p.vec) kern<uint16_t, true, 1> __VA_ARGS__; else kern<uint16_t, false, 1> __VA_ARGS__;                   \
        }                                                                                                                \
    } while (0)

extern "C" int fmoe_norm_add(const fmoe_norm_desc* desc, fmoe_stream_t stream) {
    const int rc = norm_check(desc, false);
    if (rc != FMOE_OK || desc->rows == 0) return rc;
    const fmoe_norm_desc& d = *desc;
    const NormPlan p = norm_plan(d);
    const int64_t blocks = (d.rows + p.per - 1) / p.per, most = 256 * 32 / (p.threads / kWave);
    FMOE_NORM(norm_add_kernel, <<<(unsigned)(blocks < most ? blocks : most), p.threads, 0, (hipStream_t)stream>>>(d, p.waves));
    return check_launch("fmoe_norm_add");
}

extern "C" size_t fmoe_norm_add_bwd_workspace_bytes(const fmoe_norm_desc* desc) {
    if (norm_check(desc, true) != FMOE_OK || desc->rows == 0 || !norm_wants_sums(*desc)) return 0;
    const NormPlan p = norm_plan(*desc);
    const int64_t groups = norm_groups(*desc, p), all = (groups + p.per - 1) / p.per * p.per;
    return (size_t)all * kSums * desc->cols * sizeof(float);
}

extern "C" int fmoe_norm_add_bwd(const fmoe_norm_desc* desc, void* workspace, size_t workspace_bytes, fmoe_stream_t stream) {
    const int rc = norm_check(desc, true);
    if (rc != FMOE_OK || desc->rows == 0) return rc;
    const fmoe_norm_desc& d = *desc;
    const NormPlan p = norm_plan(d);
    const size_t need = fmoe_norm_add_bwd_workspace_bytes(desc);
    if (need && (!workspace || workspace_bytes < need))
        return fail(FMOE_ERR_WORKSPACE, "fmoe_norm_add_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    float* const partial = need ? (float*)workspace : nullptr;
    const int blocks = (norm_groups(d, p) + p.per - 1) / p.per;
    FMOE_NORM(norm_add_bwd_kernel, <<<blocks, p.threads, 0, (hipStream_t)stream>>>(d, p.waves, partial));
    const int launched = check_launch("fmoe_norm_add_bwd");
    if (launched != FMOE_OK || !need) return launched;
    norm_sums_kernel<<<dim3((d.cols + kWave - 1) / kWave, kSums), kSumWaves * kWave, 0, (hipStream_t)stream>>>(d, partial, blocks * p.per);
    return check_launch("fmoe_norm_add_bwd");
}
