// The two pre-activations of a SwiGLU expert block in 8 bits between forward and backward (fmoe_swiglu_checkpoint and what reads it):
//
//   a block of 32 neighbours of a row shares the power of two X = 2^floor(log2(largest magnitude)), kept as its biased exponent in a byte;
//   code = round(v / X * 64) to nearest even, held to +-127;  v' = code * X / 64            (the MXINT8 format of the OCP microscaling spec)
//   backward on g', u':  s = sigmoid(g'),  h = g' s u',  dh = w d,  dg = dh u' s (1 + g' (1 - s)),  du = dh g' s,
//   and, for the weight gradient behind it and the rows' own weights w: w h and the row sums of h d
//
// 33 / 32 bytes for a value of 2 or 4, error at most half a step of 1 / 64 (3 % of the blocks' largest, rounded down to +-127: a whole step at the
// very top); every v' is exact in bf16.  A zero block has exponent 0; one with an infinity or NaN has 255 and reads as NaN.
// All of it is bound by the bytes; a lane has 16 values to write and 8 to read with (a row's sum wants its lanes in one wave, and 1408 columns leave
// a third of the lanes of 16 idle, 8 % of those of 8).
#include "common.h"

#include <type_traits>

namespace fmoe {
namespace {

template <typename E> struct CE;
template <> struct CE<float> { static constexpr int V = 4; };
template <> struct CE<uint16_t> { static constexpr int V = 8; };

// N values (whole 16-byte chunks) at any address an element may have; those from `left` on are zeros, or not written.  WHOLE: `left` is whole chunks;
// otherwise the last one goes by elements.
template <typename E, bool WHOLE, int N>
__device__ __forceinline__ void load_values(const E* p, int left, float (&f)[N]) {
    constexpr int V = CE<E>::V;
#pragma unroll
    for (int c = 0; c < N / V; ++c) {
        u32x4 v = {0, 0, 0, 0};
        if (WHOLE ? c * V < left : (c + 1) * V <= left) {
            __builtin_memcpy(&v, p + c * V, 16);
        } else if (!WHOLE && c * V < left) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c * V + i < left) {
                    if constexpr (V == 4) v[i] = __float_as_uint(p[c * V + i]);
                    else v[i / 2] |= (uint32_t)p[c * V + i] << (16 * (i & 1));
                }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (V == 4) f[c * V + i] = __uint_as_float(v[i]);
            else f[c * V + i] = i & 1 ? __uint_as_float(v[i / 2] & 0xffff0000u) : __uint_as_float(v[i / 2] << 16);
        }
    }
}
template <typename E, bool WHOLE, int N>
__device__ __forceinline__ void store_values(E* p, int left, const float (&f)[N]) {
    constexpr int V = CE<E>::V;
#pragma unroll
    for (int c = 0; c < N / V; ++c) {
        if (WHOLE ? c * V < left : (c + 1) * V <= left) {
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (V == 4) v[i] = __float_as_uint(f[c * V + i]);
                else v[i] = cvt_pk_bf16(f[c * V + 2 * i], f[c * V + 2 * i + 1]);
            }
            __builtin_memcpy(p + c * V, &v, 16);
        } else if (!WHOLE && c * V < left) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c * V + i < left) {
                    if constexpr (sizeof(E) == 4) p[c * V + i] = f[c * V + i];
                    else p[c * V + i] = (uint16_t)f32_to_bf16_bits(f[c * V + i]);
                }
        }
    }
}

struct CkptRows {
    const void *g, *u;
    int64_t g_stride, u_stride, rows;
    int32_t cols, padded;       // padded: cols in whole blocks of 32
    int8_t* q;                  // [rows][2][padded]
    uint8_t* e;                 // [rows][2][padded / 32]
};

// 16 values a lane, two lanes a block; the lanes of a grid go over (row, matrix, half block) in memory order.  131072 x 1408 bf16: 233 us, 4.8 TB/s.
template <typename E, bool WHOLE>
__global__ __launch_bounds__(256) void swiglu_checkpoint_kernel(CkptRows p) {
    const int halves = p.padded / 16, per_row = 2 * halves;
    const int64_t first = (int64_t)blockIdx.x * 256, row0 = first / per_row;        // (once per wave, on the scalar unit)
    const uint32_t at = (uint32_t)(first - row0 * per_row) + threadIdx.x;
    const int64_t r = row0 + at / (uint32_t)per_row;
    if (r >= p.rows) return;            // (whole blocks of 32: both lanes of one)
    const int in_row = at % (uint32_t)per_row, m = in_row >= halves, c = 16 * (in_row - m * halves);
    float f[16];
    load_values<E, WHOLE>((const E*)(m ? p.u : p.g) + r * (m ? p.u_stride : p.g_stride) + c, p.cols - c, f);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp((int)top, (int)top, 0xB1, 0xF, 0xF, false));      // quad_perm [1,0,3,2]: the other half
    const int biased = (int)(top >> 23);        // 255: not finite
    u32x4 out;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = fminf(fmaxf(rintf(__builtin_amdgcn_ldexpf(f[4 * w + i], 133 - biased)), -127.0f), 127.0f);
            word |= ((uint32_t)(int)v & 0xffu) << (8 * i);
        }
        out[w] = biased == 255 ? 0u : word;
    }
    const int64_t base = (2 * r + m) * p.padded + c;
    *reinterpret_cast<u32x4*>(p.q + base) = out;
    if (!(threadIdx.x & 1)) p.e[base / 32] = (uint8_t)biased;
}

// The scale of a block's codes, X / 64 (NaN for one that is not finite)
__device__ __forceinline__ float code_scale(int biased) { return biased == 255 ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(1.0f, biased - 133); }

// Eight codes
__device__ __forceinline__ void decode(u32x2 q, float scale, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)(int)(int8_t)(q[i / 4] >> (8 * (i & 3))) * scale;
}

// The same, 8 values a lane.  131072 x 1408 bf16: 200 us, 5.6 TB/s.
template <typename E, bool WHOLE>
__global__ __launch_bounds__(256) void swiglu_checkpoint_read_kernel(CkptRows p) {
    const int eighths = p.padded / 8, per_row = 2 * eighths;
    const int64_t first = (int64_t)blockIdx.x * 256, row0 = first / per_row;
    const uint32_t at = (uint32_t)(first - row0 * per_row) + threadIdx.x;
    const int64_t r = row0 + at / (uint32_t)per_row;
    if (r >= p.rows) return;
    const int in_row = at % (uint32_t)per_row, m = in_row >= eighths, c = 8 * (in_row - m * eighths);
    const int64_t base = (2 * r + m) * p.padded + c;
    float f[8];
    decode(*reinterpret_cast<const u32x2*>(p.q + base), code_scale(p.e[base / 32]), f);
    store_values<E, WHOLE>((E*)(m ? p.u : p.g) + r * (m ? p.u_stride : p.g_stride) + c, p.cols - c, f);
}

struct CkptBwd {
    const int8_t* q;
    const uint8_t* e;
    int64_t rows;
    int32_t cols, padded;
    const void* d;
    int64_t d_stride;
    const void* weight;
    int32_t weight_f32;
    void *dg, *du, *h;
    int64_t dg_stride, h_stride;        // of dg and du, of h
    float* dots;
};

// Eight values a lane; LANES of a wave to a row (all of them, or as many as a shorter row has eighths, rounded up to 2, 8 or 32): 200000 x 40 bf16 17 us against
// 85 with a wave to every row, 100000 x 200 36 against 47.  9189 x 2600 bf16: 44 us, 5.5 TB/s.
template <typename E, bool WHOLE, int LANES>
__global__ __launch_bounds__(256) void swiglu_checkpoint_bwd_kernel(CkptBwd p) {
    constexpr int ROWS = kWave / LANES;
    const int lane = lane_id() % LANES;
    const int64_t step = (int64_t)gridDim.x * 4 * ROWS;
    for (int64_t r = ((int64_t)blockIdx.x * 4 + threadIdx.x / kWave) * ROWS + lane_id() / LANES; r < p.rows; r += step) {
        const float w = !p.weight ? 1.0f : p.weight_f32 ? reinterpret_cast<const float*>(p.weight)[r] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p.weight)[r]);
        const int8_t* const q = p.q + 2 * r * p.padded;
        const uint8_t* const e = p.e + 2 * r * (p.padded / 32);
        float dot = 0.0f;
        for (int c = 8 * lane; c < p.cols; c += 8 * LANES) {
            float g[8], u[8], d[8], dg[8], du[8], h[8];
            const u32x2 qg = *reinterpret_cast<const u32x2*>(q + c), qu = *reinterpret_cast<const u32x2*>(q + p.padded + c);
            const int eg = e[c / 32], eu = e[p.padded / 32 + c / 32];
            load_values<E, WHOLE>((const E*)p.d + r * p.d_stride + c, p.cols - c, d);
            decode(qg, code_scale(eg), g);
            decode(qu, code_scale(eu), u);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float s;
                if constexpr (sizeof(E) == 4) s = 1.0f / (1.0f + expf(-g[i]));
                else s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g[i] * -1.44269504088896341f));     // (rounded to bf16 behind it)
                const float gs = g[i] * s, dh = w * d[i], hi = gs * u[i];
                dg[i] = dh * u[i] * (s + gs * (1.0f - s));
                du[i] = dh * gs;
                h[i] = w * hi;
                if (WHOLE || c + i < p.cols) dot = __builtin_fmaf(hi, d[i], dot);
            }
            store_values<E, WHOLE>((E*)p.dg + r * p.dg_stride + c, p.cols - c, dg);
            store_values<E, WHOLE>((E*)p.du + r * p.dg_stride + c, p.cols - c, du);
            if (p.h) store_values<E, WHOLE>((E*)p.h + r * p.h_stride + c, p.cols - c, h);
        }
        if (p.dots) {           // (the lanes of a row stay together: they have the same r)
#pragma unroll
            for (int o = LANES / 2; o >= 1; o >>= 1) dot += __shfl_xor(dot, o, kWave);
            if (lane == 0) p.dots[r] = dot;
        }
    }
}

int ckpt_check(const char* name, int dtype, int64_t rows, int64_t cols, const void* q, const void* e) {
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16, "%s: bf16 or fp32 expected", name);
    FMOE_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 24), "%s: rows >= 0 and 1 to 2^24 columns expected", name);
    FMOE_REQUIRE(rows == 0 || (q && e), "%s: NULL tensor pointer", name);
    FMOE_REQUIRE(aligned16(q), "%s: codes must be 16-byte aligned", name);
    return FMOE_OK;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int64_t fmoe_swiglu_checkpoint_cols(int64_t cols) { return (cols + 31) / 32 * 32; }

static int ckpt_both(bool write, const char* name, void* g, void* u, int dtype, int64_t rows, int64_t cols, int64_t g_stride, int64_t u_stride, int8_t* q,
                     uint8_t* e, fmoe_stream_t stream_) {
    if (int rc = ckpt_check(name, dtype, rows, cols, q, e)) return rc;
    if (rows == 0) return FMOE_OK;
    FMOE_REQUIRE(g && u, "%s: NULL tensor pointer", name);
    FMOE_REQUIRE(rows == 1 || (g_stride >= cols && u_stride >= cols), "%s: rows overlap", name);
    const CkptRows p{g, u, g_stride, u_stride, rows, (int32_t)cols, (int32_t)fmoe_swiglu_checkpoint_cols(cols), q, e};
    const bool whole = cols % 8 == 0;
    const int64_t n = (rows * (2 * p.padded / (write ? 16 : 8)) + 255) / 256;
    FMOE_REQUIRE(n < ((int64_t)1 << 24), "%s: too many values for one call", name);      // (2^32 lanes are a grid)
    const unsigned blocks = (unsigned)n;
    hipStream_t stream = (hipStream_t)stream_;
#define FMOE_CKPT(kern)                                                                                                    \
    do {                                                                                                                   \
        if (dtype == FMOE_F32) { if (whole) kern<float, true><<<blocks, 256, 0, stream>>>(p); else kern<float, false><<<blocks, 256, 0, stream>>>(p); } \
        else { if (whole) kern<uint16_t, true><<<blocks, 256, 0, stream>>>(p); else kern<uint16_t, false><<<blocks, 256, 0, stream>>>(p); }           \
    } while (0)
    if (write) FMOE_CKPT(swiglu_checkpoint_kernel);
    else FMOE_CKPT(swiglu_checkpoint_read_kernel);
#undef FMOE_CKPT
    return check_launch(name);
}

extern "C" int fmoe_swiglu_checkpoint(const void* g, const void* u, int dtype, int64_t rows, int64_t cols, int64_t g_stride_row, int64_t u_stride_row,
                                      int8_t* q, uint8_t* e, fmoe_stream_t stream) {
    return ckpt_both(true, "fmoe_swiglu_checkpoint", const_cast<void*>(g), const_cast<void*>(u), dtype, rows, cols, g_stride_row, u_stride_row, q, e, stream);
}

extern "C" int fmoe_swiglu_checkpoint_read(const int8_t* q, const uint8_t* e, void* g, void* u, int dtype, int64_t rows, int64_t cols,
                                           int64_t g_stride_row, int64_t u_stride_row, fmoe_stream_t stream) {
    return ckpt_both(false, "fmoe_swiglu_checkpoint_read", g, u, dtype, rows, cols, g_stride_row, u_stride_row, const_cast<int8_t*>(q),
                     const_cast<uint8_t*>(e), stream);
}

extern "C" int fmoe_swiglu_checkpoint_bwd(const int8_t* q, const uint8_t* e, const void* d, int dtype, int64_t rows, int64_t cols, int64_t d_stride_row,
                                          const void* weight, int weight_dtype, void* dg, void* du, int64_t dg_stride_row, void* h, int64_t h_stride_row,
                                          float* dots, fmoe_stream_t stream_) {
    const char* const name = "fmoe_swiglu_checkpoint_bwd";
    if (int rc = ckpt_check(name, dtype, rows, cols, q, e)) return rc;
    FMOE_REQUIRE(!weight || weight_dtype == FMOE_F32 || weight_dtype == FMOE_BF16, "%s: row weights must be bf16 or fp32", name);
    if (rows == 0) return FMOE_OK;
    FMOE_REQUIRE(d && dg && du, "%s: NULL tensor pointer", name);
    FMOE_REQUIRE(rows == 1 || (d_stride_row >= cols && dg_stride_row >= cols && (!h || h_stride_row >= cols)), "%s: rows overlap", name);
    const CkptBwd p{q, e, rows, (int32_t)cols, (int32_t)fmoe_swiglu_checkpoint_cols(cols), d, d_stride_row, weight, weight_dtype == FMOE_F32, dg, du, h,
                    dg_stride_row, h_stride_row, dots};
    const bool whole = cols % 8 == 0;
    const int lanes = cols > 256 ? 64 : cols > 64 ? 32 : cols > 16 ? 8 : 2;
    const int64_t per = 4 * (kWave / lanes), n = (rows + per - 1) / per;
    auto go = [&](auto kern) { kern<<<(unsigned)(n < 256 * 8 ? n : 256 * 8), 256, 0, (hipStream_t)stream_>>>(p); };
    auto of = [&](auto value, auto w) {
        using E = decltype(value);
        constexpr bool WHOLE = decltype(w)::value;
        if (lanes == 64) go(swiglu_checkpoint_bwd_kernel<E, WHOLE, 64>);
        else if (lanes == 32) go(swiglu_checkpoint_bwd_kernel<E, WHOLE, 32>);
        else if (lanes == 8) go(swiglu_checkpoint_bwd_kernel<E, WHOLE, 8>);
        else go(swiglu_checkpoint_bwd_kernel<E, WHOLE, 2>);
    };
    if (dtype == FMOE_F32) whole ? of(float(), std::true_type()) : of(float(), std::false_type());
    else whole ? of(uint16_t(), std::true_type()) : of(uint16_t(), std::false_type());
    return check_launch(name);
}
