// Products of few tokens with a weight matrix: y[t][n] = sum_k x[t][k] W[n][k], bound by the bytes of W. Each wave takes 16
// rows of W (RT tiles of 16) at every W-th 128 columns, straight from HBM to MFMA operands, so that a lane's loads are its
// fragment and no LDS stands between; x comes through the caches in the same layout. The waves' sums are joined through LDS
// in the waves' order (the result does not depend on timing).
//
// v_mfma_f32_16x16x32: A = 16 tokens, B = 16 rows of W: lane l holds token / row l % 16 and columns (l / 16) * 8 .. + 7; of
// the result column (row of W) l % 16 and tokens (l / 16) * 4 .. + 3. Fewer than 16 tokens load a token again: those
// results are not stored.
#pragma once
#include "gemm16.hpp"

namespace bmx {

constexpr int SK_W = 8;             // waves of a workgroup
constexpr int SK_K = 128;           // columns of a wave's step

// 4-bit weights in fragment order (bmx_q4): per tile of 16 rows x 128 columns, lane l's 32 codes are 16 bytes: word j holds
// row l % 16, columns j * 32 + (l / 16) * 8 + e, code e = 2 p in bits 4 p, e = 2 p + 1 in bits 4 p + 16, so that a mask
// leaves the two codes of a packed pair in its halves. scale and zero: [tile of 16 rows][group][16].
struct Q4View {
    const u32x4* codes;
    const uint16_t* scale;
    const uint8_t* zero;            // null: 8
    int scale_bf16;
};

struct SkinnyArgs {
    const void* w[2];               // 16-bit weights [N][K]; second: up
    Q4View q[2];
    const uint16_t* x;
    int T, N, K, group;
    void* out;
    int ldo;
    const float* scale;             // EPI_ADD: [T] or null
    ActPar act;
    uint16_t *g, *u;                // EPI_GU: saved when not null
};

// q4.hip
Q4View q4_view(const bmx_q4* q);
int check_q4(const bmx_q4* q, const char* who);
int launch_q4_dequant(const bmx_q4* q, int dtype, void* out, hipStream_t s);
// skinny_k on a's weights (a.group 0: 16-bit) with one matrix (EPI_STORE, EPI_ADD) or two (EPI_GU)
int launch_skinny(const SkinnyArgs& a, int dtype, int epi, hipStream_t s);
// the most tokens that skinny_k takes
int skinny_tokens_max(int group);
// ffn.hip: y [T][N] = x w^T with 16-bit weights on gemm16_k; part: product_part_bytes bytes
int launch_product(const void* w, const void* x, int T, int N, int K, int dtype, void* y, void* part, hipStream_t s);
size_t product_part_bytes(int N, int T, int K);

// One decoded word: 8 weights. fp16: 1024 + c is 0x6400 | c, 1024 + 16 c is 0x6400 | c << 4; subtracting the offset and the
// zero point is exact. bf16 has no packed arithmetic here: 128 + c is 0x4300 | c, and the 128 + z comes off the sum, as
// (128 + z) times the group's sum of x.
template <class T> struct Q4Dec;
template <> struct Q4Dec<f16>
{
    static constexpr bool OFFSET = false;
    f16x2 c0, c1;
    __device__ __forceinline__ void zero(float z)
    {
        c0 = f16x2{(f16)(-1024.0f - z), (f16)(-1024.0f - z)};
        c1 = f16x2{(f16)(-64.0f - z), (f16)(-64.0f - z)};
    }
    __device__ __forceinline__ f16x8 operator()(uint32_t v) const
    {
        const f16x2 s = f16x2{(f16)0.0625f, (f16)0.0625f};
        uint32_t r[4];
#pragma unroll
        for (int h = 0; h < 2; ++h, v >>= 8)
        {
            r[2 * h] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, (v & 0x000f000fu) | 0x64006400u) + c0);
            r[2 * h + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(
                __builtin_bit_cast(f16x2, (v & 0x00f000f0u) | 0x64006400u), s, c1));
        }
        return __builtin_bit_cast(f16x8, u32x4{r[0], r[1], r[2], r[3]});
    }
};
template <> struct Q4Dec<bf16>
{
    static constexpr bool OFFSET = true;
    __device__ __forceinline__ void zero(float) {}
    __device__ __forceinline__ bf16x8 operator()(uint32_t v) const
    {
        u32x4 r;
#pragma unroll
        for (int p = 0; p < 4; ++p, v >>= 4) r[p] = (v & 0x000f000fu) | 0x43004300u;
        return __builtin_bit_cast(bf16x8, r);
    }
};

// NM: matrices (2: gate and up), RT: tiles of 16 rows a wave takes of each, TT: tiles of 16 tokens, G: group size (0: 16-bit
// weights)
template <class T, int NM, int RT, int TT, int G, int EPI>
__global__ __launch_bounds__(SK_W * 64) void skinny_k(const SkinnyArgs p)
{
    typedef typename Elem<T>::v8 v8;
    constexpr bool Q4 = G != 0;
    constexpr int NG = Q4 ? SK_K / G : 1, JG = 4 / NG;             // groups of a step, words of a group
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * (RT * 16), t0 = blockIdx.y * (TT * 16);
    const int KT = (p.K + SK_K - 1) / SK_K, NT = (p.N + 15) / 16;

    f32x4 acc[NM][RT][TT];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[m][i][t] = f32x4{0, 0, 0, 0};

    const uint16_t* xr[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) xr[t] = p.x + (int64_t)min(t0 + t * 16 + r, p.T - 1) * p.K + q * 8;

    for (int kt = wave; kt < KT; kt += SK_W)
    {
        const int k0 = kt * SK_K;
        u32x4 xv[4][TT];
        // weights, then x; past K both are 0
        u32x4 wv[NM][RT][Q4 ? 1 : 4];
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int i = 0; i < RT; ++i)
            {
                if (Q4)
                {
                    const int tile = min(blockIdx.x * RT + i, (unsigned)NT - 1);
                    wv[m][i][0] = ldg4(p.q[m].codes + ((int64_t)tile * KT + kt) * 64 + lane);
                }
                else
                {
                    const uint16_t* w = static_cast<const uint16_t*>(p.w[m]) + (int64_t)min(n0 + i * 16 + r, p.N - 1) * p.K + q * 8;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                    {
                        const int k = k0 + j * 32;
                        const bool in = k + q * 8 < p.K;
                        wv[m][i][j] = in ? ldg4(w + k) : u32x4{0, 0, 0, 0};
                    }
                }
            }
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                const int k = k0 + j * 32;
                xv[j][t] = k + q * 8 < p.K ? ldg4(xr[t] + k) : u32x4{0, 0, 0, 0};
            }
        if (Q4)
        {
            const int groups = KT * NG;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi)
            {
                f32x4 xs[TT];                                      // the group's sums of x (bf16)
                v8 ones;
#pragma unroll
                for (int e = 0; e < 8; ++e) ones[e] = (T)1.0f;
#pragma unroll
                for (int t = 0; t < TT; ++t)
                {
                    xs[t] = f32x4{0, 0, 0, 0};
                    if (Q4Dec<T>::OFFSET)
#pragma unroll
                        for (int j = 0; j < JG; ++j)
                            xs[t] = Elem<T>::mfma16(__builtin_bit_cast(v8, xv[gi * JG + j][t]), ones, xs[t]);
                }
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int i = 0; i < RT; ++i)
                    {
                        const int tile = min(blockIdx.x * RT + i, (unsigned)NT - 1);
                        const int64_t at = ((int64_t)tile * groups + kt * NG + gi) * 16 + r;
                        const uint16_t sb = p.q[m].scale[at];
                        const float s = p.q[m].scale_bf16 ? from16<bf16>(sb) : from16<f16>(sb);
                        const float z = p.q[m].zero ? (float)p.q[m].zero[at] : 8.0f;
                        Q4Dec<T> dec;
                        dec.zero(z);
                        f32x4 part[TT];
#pragma unroll
                        for (int t = 0; t < TT; ++t) part[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < JG; ++j)
                        {
                            const v8 w = dec(wv[m][i][0][gi * JG + j]);
#pragma unroll
                            for (int t = 0; t < TT; ++t)
                                part[t] = Elem<T>::mfma16(__builtin_bit_cast(v8, xv[gi * JG + j][t]), w, part[t]);
                        }
#pragma unroll
                        for (int t = 0; t < TT; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                            {
                                const float v = Q4Dec<T>::OFFSET ? __builtin_fmaf(-128.0f - z, xs[t][e], part[t][e]) : part[t][e];
                                acc[m][i][t][e] = __builtin_fmaf(s, v, acc[m][i][t][e]);
                            }
                    }
            }
        }
        else
        {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int i = 0; i < RT; ++i)
#pragma unroll
                        for (int t = 0; t < TT; ++t)
                            acc[m][i][t] = Elem<T>::mfma16(__builtin_bit_cast(v8, xv[j][t]), __builtin_bit_cast(v8, wv[m][i][j]),
                                                           acc[m][i][t]);
        }
    }

    // join the waves: value v of a matrix = (row tile, token tile, element, lane)
    constexpr int V = RT * TT * 256;
    __shared__ float part[SK_W][NM * V];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[wave][m * V + ((i * TT + t) * 4 + e) * 64 + lane] = acc[m][i][t][e];
    __syncthreads();
    for (int v = threadIdx.x; v < V; v += SK_W * 64)
    {
        const int l = v & 63, e = (v >> 6) & 3, t = t0 + (v >> 8) % TT * 16 + (l >> 4) * 4 + e, n = n0 + (v >> 8) / TT * 16 + (l & 15);
        if (t >= p.T || n >= p.N) continue;
        float s[NM];
#pragma unroll
        for (int m = 0; m < NM; ++m)
        {
            s[m] = part[0][m * V + v];
#pragma unroll
            for (int w = 1; w < SK_W; ++w) s[m] += part[w][m * V + v];
        }
        const int64_t o = (int64_t)t * p.ldo + n;
        if (EPI == EPI_GU)
        {
            static_cast<uint16_t*>(p.out)[o] = to16<T>(act_h(p.act, s[0], s[NM - 1]));
            if (p.g) save_gu<T>(p.act, s[0], s[NM - 1], p.g[o], p.u[o]);
        }
        else if (EPI == EPI_ADD)
        {
            float* y = static_cast<float*>(p.out) + o;
            *y = __builtin_fmaf(p.scale ? p.scale[t] : 1.0f, s[0], *y);
        }
        else static_cast<uint16_t*>(p.out)[o] = to16<T>(s[0]);
    }
}

}  // namespace bmx
