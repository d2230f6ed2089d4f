// Rows in registers: eight values of a row at a time from 16 or 32 bits to fp32 and back, sums and maxima over a row's waves, and
// a row's form in 8-bit integers (q8.hip, norm.hip).
//
// A row v of K values as whole numbers up to 127 and one scale: top = max |v|, code = v 127 / top to the nearest, ties to even, scale =
// top / 127. The values that the codes stand for are at most half a scale off. A row of zeros, or of nothing above TOP_LEAST
// (its 127 / top would leave fp32), is codes 0 with scale 0; one with an infinity or a NaN is codes 0 with scale NaN, so that all
// its products are NaN.
#pragma once
#include "gemm16.hpp"

namespace bmx {

constexpr float TOP_LEAST = 0x1p-110f;

// Where a row's values lie: 16 bits of either type, or fp32
enum RowType { ROW_F16 = BMX_DT_FP16, ROW_BF16 = BMX_DT_BF16, ROW_F32 = BMX_DT_FP32 };

inline size_t row_type_bytes(int t) { return t == ROW_F32 ? 4 : 2; }

// 8 values as they lie in memory: the second half for fp32 alone
struct Raw8 { u32x4 a, b; };
typedef float f32x2 __attribute__((ext_vector_type(2)));

// values i .. i + 7 of p (16-byte aligned)
__device__ __forceinline__ Raw8 load_raw8(const void* p, int type, int64_t i)
{
    Raw8 r;
    if (type == ROW_F32)
    {
        r.a = ldg4(static_cast<const float*>(p) + i);
        r.b = ldg4(static_cast<const float*>(p) + i + 4);
    }
    else r.a = r.b = ldg4(static_cast<const uint16_t*>(p) + i);
    return r;
}

__device__ __forceinline__ float value16(int type, uint32_t bits)
{
    return type == ROW_F16 ? from16<f16>((uint16_t)bits) : __builtin_bit_cast(float, bits << 16);
}

__device__ __forceinline__ void to_f32(const Raw8& r, int type, float (&v)[8])
{
    if (type == ROW_F32)
    {
        const f32x4 a = __builtin_bit_cast(f32x4, r.a), b = __builtin_bit_cast(f32x4, r.b);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[i + 4] = b[i]; }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        v[2 * i] = value16(type, r.a[i] & 0xffffu);
        v[2 * i + 1] = value16(type, r.a[i] >> 16);
    }
}

// (of an fp32 value, as f2h_r: fused with the product before it into one instruction with one rounding, fp16 results would differ
// between kernels)
__device__ __forceinline__ uint32_t bits16(int type, float v) { return type == ROW_F16 ? f2h_r(v) : to16<bf16>(v); }

// v to 8 values at i of p; rounds v to what is stored
__device__ __forceinline__ void store8(void* p, int type, int64_t i, float (&v)[8])
{
    if (type == ROW_F32)
    {
        f32x4* q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + i);
        q[0] = f32x4{v[0], v[1], v[2], v[3]};
        q[1] = f32x4{v[4], v[5], v[6], v[7]};
        return;
    }
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k)
    {
        const uint32_t lo = bits16(type, v[2 * k]), hi = bits16(type, v[2 * k + 1]);
        w[k] = lo | hi << 16;
        v[2 * k] = value16(type, lo);
        v[2 * k + 1] = value16(type, hi);
    }
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) = w;
}

// |v| as bits: ordered as the magnitudes, NaN above infinity above all numbers
__device__ __forceinline__ uint32_t mag(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// Sum and maximum over the wave, uniform: exchanges within quads, half rows and rows of 16 lanes, then row 0 into 1 and 2 into 3, rows 0 and 1
// into 2 and 3; lane 63 holds the result. (DPP moves: through LDS, as __shfl_xor, the six steps take half a microsecond.)
template <class Op> __device__ __forceinline__ uint32_t wave_all(uint32_t v, Op op)
{
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_sum(float v)
{
    return __builtin_bit_cast(float, wave_all(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) { return wave_all(v, [](uint32_t a, uint32_t b) { return max(a, b); }); }

// What a row's largest magnitude makes of it: codes are v inv to the nearest whole number, the scale is top / 127
struct Top8 { float inv, scale, part; };    // part: top / 128
__device__ __forceinline__ Top8 top8(uint32_t top)
{
    const float t = __builtin_bit_cast(float, top);
    if (top >= 0x7f800000u) return {0.0f, __builtin_nanf(""), 0.0f};
    if (t < TOP_LEAST) return {0.0f, 0.0f, 0.0f};
    return {__fdiv_rn(127.0f, t), __fdiv_rn(t, 127.0f), t * 0x1p-7f};
}

// Four codes: adding 1.5 * 2^23 leaves the whole number n nearest to v inv in the low bits, as a two's complement byte. Rows of
// 16-bit values hold true ties, v = top / 2 first of all (63.5, about one in each row), which inv's rounding would send up or down;
// 127 v - n top, scaled by 2^-7 and exact for them, says so, and the even neighbour is taken. The codes of their other values are those
// of the exact quotients too: with v = a 2^-d and top = b, significands as whole numbers below 2^11, 127 v / top is |254 a - m b 2^d|
// / (b 2^(d + 1)) from the border m / 2 (m odd), where the upper part is 1 at least, and 2 for d > 0: 2^-12 or 2^-(11 + d). v inv is below
// 2^(8 - d) (127 for d = 0) and off by half a step of inv, less than 2^-17 or 2^-(16 + d). (Another code here and there in x
// moves one h in a hundred to its neighbour behind the next quantization: a block's error against 64 bits was 0.0053 of the norm for
// it, 0.0017 without.) inv 0 stands for rows of zeros, and for rows that hold a NaN or an infinity: codes 0 whatever they hold.
__device__ __forceinline__ uint32_t codes4(const float* v, const Top8& o)
{
    if (o.inv == 0.0f) return 0;
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const float f = __builtin_fmaf(v[i], o.inv, 12582912.0f), n = f - 12582912.0f;
        const float r = __builtin_fmaf(-n, o.part, v[i] * (127.0f / 128.0f));
        b[i] = __builtin_bit_cast(uint32_t, f);
        if (fabsf(r) == 0.5f * o.part && (b[i] & 1)) b[i] += r > 0.0f ? 1 : -1;
    }
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    return lo | hi;
}

// Codes in blocks of 16 rows x 64 columns (bmx_q8): 1 KB, in the order in which v_mfma_i32_16x16x64_i8's lanes hold it (or two halves of
// one of 32x32x32): chunk c of 16 columns of row r at c * 256 + r * 16, so that a wave's load is one contiguous piece whatever the row's
// length. (Row by row a wave's load is 64 bytes of each of 16 rows, for K = 4096 all in one memory channel: 4,096 x 4,096 x 11,008 187 us,
// in blocks 175. In blocks of rows of 64 bytes a compute unit takes fragments in at 74 bytes a nanosecond, this way at 115 to 140, since
// its L1 gives 64 neighbouring bytes to four lanes at a time.)
constexpr int Q8_ROWS = 16, Q8_COLS = 64, Q8_BLOCK = Q8_ROWS * Q8_COLS, Q8_CHUNK = Q8_ROWS * 16;
__host__ __device__ constexpr int q8_blocks(int K) { return (K + Q8_COLS - 1) / Q8_COLS; }     // of a row of blocks
__host__ __device__ constexpr int64_t q8_at(int64_t row, int k, int blocks)
{
    return (row / Q8_ROWS * blocks + k / Q8_COLS) * Q8_BLOCK + (k % Q8_COLS >> 4) * Q8_CHUNK + (row % Q8_ROWS) * 16 + k % 16;
}
inline size_t q8_bytes(int N, int K) { return (size_t)round_up(N, Q8_ROWS) * q8_blocks(K) * Q8_COLS; }

// Rows x of a row type into out's codes and scales (norm.hip)
int launch_quantize(const void* x, int type, const bmx_q8* out, hipStream_t s);
// q8.hip: refuses what is no matrix of codes; rows: ... of T rows of K codes
int check_q8(const bmx_q8* q, const char* who);
int check_rows8(const bmx_q8* rows, int T, int K, const char* who);
// ffn.hip: out[t] = sigmoid(x[t] . v), x and v of dtype
int launch_row_gate(const void* x, const void* v, int dtype, int n, int H, float* out, hipStream_t s);

}  // namespace bmx
