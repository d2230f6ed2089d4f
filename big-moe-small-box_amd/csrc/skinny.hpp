// Products of few tokens with a weight matrix: y[t][n] = sum_k x[t][k] W[n][k], bound by the bytes of W. A workgroup has 16
// tokens and 16, 32 or 64 rows of W (half of gate and half of up in the gated product); each of its waves takes every
// SK_W-th 128 columns of them straight from HBM to MFMA operands, so that a lane's loads are its fragment and no LDS stands
// between, several steps ahead of the products; x comes through the caches in the same layout. The waves' sums are joined
// through LDS in the waves' order (the result does not depend on timing).
//
// v_mfma_f32_16x16x32: A = 16 tokens, B = 16 rows of W: lane l holds token / row l % 16 and columns (l / 16) * 8 .. + 7; of
// the result column (row of W) l % 16 and tokens (l / 16) * 4 .. + 3. Fewer than 16 tokens load a token again: those
// results are not stored.
#pragma once
#include "gemm16.hpp"

namespace bmx {

constexpr int SK_W = 8;             // waves of a workgroup

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
    bool keep;                      // 4-bit weights are not to be rounded to 16 bits (q4_keep)
    void* out;
    int ldo;
    const float* scale;             // EPI_ADD: [T] or null
    ActPar act;
    float *g, *u;                   // EPI_GU: kept when not null
};

// q4.hip
Q4View q4_view(const bmx_q4* q);
int check_q4(const bmx_q4* q, const char* who);
// Whether fp16 may not hold the weights: bf16 scales reach past both ends of its range
inline bool q4_keep(const bmx_q4* q, int dtype) { return dtype == BMX_DT_FP16 && q->scale_dtype == BMX_DT_BF16; }
int launch_q4_dequant(const bmx_q4* q, int dtype, void* out, hipStream_t s);
// A product on skinny_k or slice_k, on a's weights (a.group 0: 16-bit) with one matrix (EPI_STORE, EPI_ADD) or two (EPI_GU);
// part: skinny_part_bytes bytes
int launch_skinny(const SkinnyArgs& a, int dtype, int epi, float* part, hipStream_t s);
// A product of more tokens on 4-bit weights q[0] (and q[1]: EPI_GU); ws: q4_many_bytes bytes
int launch_q4_many(const SkinnyArgs& a, const bmx_q4* const* q, int dtype, int epi, char* ws, hipStream_t s);
// ffn.hip: a product of 16-bit weights on gemm16_k (EPI_STORE, EPI_ADD, EPI_GU with two matrices); g.part:
// product_part_bytes bytes
int launch_product(const GemmArgs& g, int dtype, int epi, hipStream_t s);

// (v & mask) | magic in one v_and_or_b32, which takes one scalar register and no literals: the constants are put into
// registers, or the compiler would make two instructions of two literals. (The instruction itself is the compiler's: a matrix
// instruction may read its result only two wait states later, which it would not know of one in inline asm.)
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t magic)
{
    asm("" : "+s"(mask));
    asm("" : "+v"(magic));
    return (v & mask) | magic;
}

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
            r[2 * h] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, and_or(v, 0x000f000fu, 0x64006400u)) + c0);
            r[2 * h + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(
                __builtin_bit_cast(f16x2, and_or(v, 0x00f000f0u, 0x64006400u)), s, c1));
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
        for (int p = 0; p < 4; ++p, v >>= 4) r[p] = and_or(v, 0x000f000fu, 0x43004300u);
        return __builtin_bit_cast(bf16x8, r);
    }
};

// RT: tiles of 16 rows of W (each 8 of gate and 8 of up in the gated product), G: group size (0: 16-bit weights), D: steps of
// 128 columns in flight per wave, XL: x in LDS (dynamic, p.T rows of K values and 16 bytes): where x is small, a fragment read
// from there costs a sixteenth of the cache lines that one from HBM asks for, which 4-bit weights notice (one token 4096 ->
// 14336: 8.6 -> 8.0 us) and 16-bit weights do not
template <class T, int RT, int G, int D, int EPI, bool XL>
__global__ __launch_bounds__(SK_W * 64) void skinny_k(const SkinnyArgs p)
{
    typedef typename Elem<T>::v8 v8;
    constexpr bool Q4 = G != 0, GU = EPI == EPI_GU;
    constexpr int NG = Q4 ? SK_K / (G ? G : 1) : 1, JG = 4 / NG;             // groups of a step, words of a group
    constexpr int ROWS = GU ? 8 : 16;                              // result columns of a tile
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    // 16 tokens a workgroup; those of one block of rows follow one another on one XCD (workgroups are dealt to the 8 in turn), so
    // that all but the first find W in its L2
    int row = blockIdx.x, t0 = 0;
    if (p.T > 16)
    {
        const int tt = (p.T + 15) >> 4, rest = row >> 3;
        t0 = rest % tt * 16;
        row = rest / tt * 8 + (row & 7);
    }
    const int n0 = row * (ROWS * RT);
    if (n0 >= p.N) return;
    const int KT = (p.K + SK_K - 1) / SK_K;
    // this lane's rows of W, and whose (rows past the last load it again)
    const int mat = GU ? r >> 3 : 0;
    const Q4View v = p.q[mat];
    const u32x4* codes[RT];
    int64_t sg[RT];
    const uint16_t* w16[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        const int n = min(n0 + i * ROWS + (GU ? r & 7 : r), p.N - 1);
        codes[i] = v.codes + (int64_t)(n >> 4) * KT * 64 + q * 16 + (n & 15);
        sg[i] = (int64_t)(n >> 4) * (KT * NG) * 16 + (n & 15);
        w16[i] = static_cast<const uint16_t*>(p.w[mat]) + (int64_t)n * p.K + q * 8;
    }
    const uint16_t* xr = p.x + (int64_t)min(t0 + r, p.T - 1) * p.K + q * 8;
    extern __shared__ __attribute__((aligned(16))) char xl[];
    const int xrow = p.K * 2 + 16;

    struct Step {
        u32x4 w[RT][Q4 ? 1 : 4], x[XL ? 1 : 4];
        uint16_t s[RT][NG];
        uint8_t z[RT][NG];
    } st[D];
    auto load = [&](Step& b, int kt) {
        const int k0 = kt * SK_K;
        if (Q4)
        {
#pragma unroll
            for (int i = 0; i < RT; ++i)
            {
                b.w[i][0] = ldg4(codes[i] + (int64_t)kt * 64);
#pragma unroll
                for (int g = 0; g < NG; ++g)
                {
                    b.s[i][g] = v.scale[sg[i] + (kt * NG + g) * 16];
                    b.z[i][g] = v.zero ? v.zero[sg[i] + (kt * NG + g) * 16] : 8;
                }
            }
        }
        if (k0 + SK_K <= p.K)
        {
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                if (!Q4)
#pragma unroll
                    for (int i = 0; i < RT; ++i) b.w[i][Q4 ? 0 : j] = ldg4(w16[i] + k0 + j * 32);
                if (!XL) b.x[XL ? 0 : j] = ldg4(xr + k0 + j * 32);
            }
        }
        else
        {
            // the last columns: x and 16-bit weights past K are 0
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                const bool in = k0 + j * 32 + q * 8 < p.K;
                if (!Q4)
#pragma unroll
                    for (int i = 0; i < RT; ++i) b.w[i][Q4 ? 0 : j] = in ? ldg4(w16[i] + k0 + j * 32) : u32x4{0, 0, 0, 0};
                if (!XL) b.x[XL ? 0 : j] = in ? ldg4(xr + k0 + j * 32) : u32x4{0, 0, 0, 0};
            }
        }
    };

    f32x4 acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = f32x4{0, 0, 0, 0};
    auto multiply = [&](const Step& b, int kt) {
        auto x = [&](int j) {
            if (!XL) return __builtin_bit_cast(v8, b.x[XL ? 0 : j]);
            const int k = kt * SK_K + j * 32 + q * 8;
            const u32x4 v = *reinterpret_cast<const u32x4*>(xl + min(r, p.T - 1) * xrow + (k < p.K ? k : p.K) * 2);
            return __builtin_bit_cast(v8, v);
        };
        if (!Q4)
        {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < RT; ++i) acc[i] = Elem<T>::mfma16(x(j), __builtin_bit_cast(v8, b.w[i][Q4 ? 0 : j]), acc[i]);
            return;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
        {
            v8 xv[JG], ones;
#pragma unroll
            for (int j = 0; j < JG; ++j) xv[j] = x(g * JG + j);
#pragma unroll
            for (int e = 0; e < 8; ++e) ones[e] = (T)1.0f;
            f32x4 xs = {0, 0, 0, 0};                               // the group's sums of x (bf16)
            if (Q4Dec<T>::OFFSET)
#pragma unroll
                for (int j = 0; j < JG; ++j) xs = Elem<T>::mfma16(xv[j], ones, xs);
#pragma unroll
            for (int i = 0; i < RT; ++i)
            {
                const float s = v.scale_bf16 ? from16<bf16>(b.s[i][g]) : from16<f16>(b.s[i][g]), z = (float)b.z[i][g];
                Q4Dec<T> dec;
                dec.zero(z);
                f32x4 part = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < JG; ++j) part = Elem<T>::mfma16(xv[j], dec(b.w[i][0][g * JG + j]), part);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[i][e] = __builtin_fmaf(s, Q4Dec<T>::OFFSET ? __builtin_fmaf(-128.0f - z, xs[e], part[e]) : part[e], acc[i][e]);
            }
        }
    };

    int kt = wave;                                                 // the next step to multiply; D are in flight
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (kt + d * SK_W < KT) load(st[d], kt + d * SK_W);
    if (XL)
    {
        // the rows, each with 16 bytes of zeros behind it for the columns past K
        for (int t = 0; t < p.T; ++t)
            for (int c = threadIdx.x; c <= p.K / 8; c += SK_W * 64)
                *reinterpret_cast<u32x4*>(xl + t * xrow + c * 16) = c < p.K / 8 ? ldg4(p.x + (int64_t)t * p.K + c * 8) : u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    while (kt < KT)
    {
#pragma unroll
        for (int d = 0; d < D; ++d)
        {
            if (kt >= KT) break;
            multiply(st[d], kt);
            if (kt + D * SK_W < KT) load(st[d], kt + D * SK_W);
            kt += SK_W;
        }
    }

    // join the waves
    constexpr int V = RT * 256;                                    // (row tile, element, lane)
    __shared__ float part[SK_W][V];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[wave][(i * 4 + e) * 64 + lane] = acc[i][e];
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += SK_W * 64)
    {
        const int c = i & 15, t = t0 + ((i >> 4) & 3) * 4 + ((i >> 6) & 3), n = n0 + (i >> 8) * ROWS + c;
        if (t >= p.T || c >= ROWS || n >= p.N) continue;
        auto sum = [&](int at) {
            float s = part[0][at];
#pragma unroll
            for (int w = 1; w < SK_W; ++w) s += part[w][at];
            return s;
        };
        const float s = sum(i);
        const int64_t o = (int64_t)t * p.ldo + n;
        if (EPI == EPI_GU)
        {
            const float u = sum(i + 8);
            static_cast<uint16_t*>(p.out)[o] = to16<T>(act_h(p.act, s, u));            // (16 bits: put_gu)
            if (p.g) { p.g[o] = s; p.u[o] = u; }
        }
        else if (EPI == EPI_ADD)
        {
            float* y = static_cast<float*>(p.out) + o;
            *y = __builtin_fmaf(p.scale ? p.scale[t] : 1.0f, s, *y);
        }
        else static_cast<uint16_t*>(p.out)[o] = to16<T>(s);
    }
}

// ---- 4-bit weights, more tokens: slices of K ---------------------------------------------------------------------------------------------
// skinny_k decodes W again for every 16 tokens. Here a workgroup keeps 512 columns of x in LDS and streams rows of W past them, a
// tile of 16 rows x 512 columns per wave at a time; every slice's sums go to part (as EPI_PART), gemm_finish_k joins them.
// waves of a workgroup: few, so that small matrices still spread evenly; more where x leaves room for one or two workgroups
template <int TT> constexpr int SL_W = TT <= 3 ? 4 : 8;

struct SliceArgs {
    SkinnyArgs a;
    int products, slices, ldp, tiles;   // tiles of 16 rows of all products, one after the other
    int per;                            // tiles of a workgroup
    float* part;
};

template <class T, int TT, int G>
__global__ __launch_bounds__(SL_W<TT> * 64) void slice_k(const SliceArgs sp)
{
    typedef typename Elem<T>::v8 v8;
    constexpr bool OFFSET = Q4Dec<T>::OFFSET;
    constexpr int NG = SK_K / G, JG = 4 / NG, U = SL_K / SK_K;     // groups of a step, words of a group, steps of a tile
    constexpr int SG = SL_K / G;                                   // groups of a slice
    const SkinnyArgs& p = sp.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int slice = blockIdx.y, k0 = slice * SL_K, KT = (p.K + SK_K - 1) / SK_K, NT = (p.N + 15) / 16;
    const int end = min((int)(blockIdx.x + 1) * sp.per, sp.tiles);

    // x: row t, 16-byte chunk c at position c ^ (t & 15): 16 tokens at one chunk (a fragment read) on different banks
    __shared__ __attribute__((aligned(16))) char xl[TT * 16 * SL_K * 2];
    __shared__ __attribute__((aligned(16))) float xs[OFFSET ? SG * TT * 16 : 4];   // [group][token]: sums of x (bf16)

    struct Step {
        u32x4 w;
        uint16_t s[NG];
        uint8_t z[NG];
    } st[U];
    auto load = [&](int tile) {
        const int m = tile >= NT ? 1 : 0, nt = tile - m * NT;
        const Q4View v = p.q[m];
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int kt = k0 / SK_K + u;
            if (kt >= KT) return;
            Step& b = st[u];
            b.w = ldg4(v.codes + ((int64_t)nt * KT + kt) * 64 + lane);
#pragma unroll
            for (int g = 0; g < NG; ++g)
            {
                const int64_t at = ((int64_t)nt * (KT * NG) + kt * NG + g) * 16 + r;
                b.s[g] = v.scale[at];
                b.z[g] = v.zero ? v.zero[at] : 8;
            }
        }
    };

    int tile = blockIdx.x * sp.per + wave;
    if (tile < end) load(tile);
    // x in loads of up to 8 at a time: one after the other they would each wait for L2
    constexpr int CH = SL_K / 8, LOADS = TT * 16 * CH / (SL_W<TT> * 64), B = LOADS % 8 == 0 ? 8 : LOADS % 5 == 0 ? 5 : 4;
    static_assert(LOADS % B == 0, "whole batches");
#pragma unroll
    for (int l0 = 0; l0 < LOADS; l0 += B)
    {
        u32x4 v[B];
#pragma unroll
        for (int l = 0; l < B; ++l)
        {
            const int i = (l0 + l) * (SL_W<TT> * 64) + threadIdx.x, t = i / CH, k = k0 + i % CH * 8;
            v[l] = t < p.T && k < p.K ? ldg4(p.x + (int64_t)t * p.K + k) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int l = 0; l < B; ++l)
        {
            const int i = (l0 + l) * (SL_W<TT> * 64) + threadIdx.x, t = i / CH, c = i % CH;
            *reinterpret_cast<u32x4*>(xl + t * (SL_K * 2) + ((c ^ (t & 15)) << 4)) = v[l];
            if (OFFSET)
            {
                // the lanes of a group are neighbours
                constexpr int LG = G / 8;
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += from16<T>((uint16_t)v[l][e]) + from16<T>((uint16_t)(v[l][e] >> 16));
#pragma unroll
                for (int o = 1; o < LG; o <<= 1) sum += __shfl_xor(sum, o);
                if (c % LG == 0) xs[c / LG * (TT * 16) + t] = sum;
            }
        }
    }
    __syncthreads();

    for (; tile < end; tile += SL_W<TT>)
    {
        f32x4 acc[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[t] = f32x4{0, 0, 0, 0};
        const int m = tile >= NT ? 1 : 0, nt = tile - m * NT;
        const Q4View v = p.q[m];
        auto x = [&](int u, int j, int t) {
            const int row = t * 16 + r, c = u * (SK_K / 8) + j * 4 + q;
            return *reinterpret_cast<const v8*>(xl + row * (SL_K * 2) + ((c ^ r) << 4));
        };
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            if (k0 / SK_K + u >= KT) break;
            const Step b = st[u];
#pragma unroll
            for (int g = 0; g < NG; ++g)
            {
                const float s = v.scale_bf16 ? from16<bf16>(b.s[g]) : from16<f16>(b.s[g]), z = (float)b.z[g];
                Q4Dec<T> dec;
                dec.zero(z);
                f32x4 part[TT];
#pragma unroll
                for (int t = 0; t < TT; ++t) part[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = g * JG; j < (g + 1) * JG; ++j)
                {
                    const v8 w = dec(b.w[j]);
#pragma unroll
                    for (int t = 0; t < TT; ++t) part[t] = Elem<T>::mfma16(x(u, j, t), w, part[t]);
                }
#pragma unroll
                for (int t = 0; t < TT; ++t)
                {
                    f32x4 o = {0, 0, 0, 0};
                    if (OFFSET) o = *reinterpret_cast<const f32x4*>(xs + (u * NG + g) * (TT * 16) + t * 16 + q * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[t][e] = __builtin_fmaf(s, OFFSET ? __builtin_fmaf(-128.0f - z, o[e], part[t][e]) : part[t][e], acc[t][e]);
                }
            }
        }
        if (tile + SL_W<TT> < end) load(tile + SL_W<TT>);
        const int n = nt * 16 + r;
        float* out = sp.part + (int64_t)(m * sp.slices + slice) * p.T * sp.ldp + n;
        if (n < p.N)
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (t * 16 + q * 4 + e < p.T) out[(int64_t)(t * 16 + q * 4 + e) * sp.ldp] = acc[t][e];
    }
}

}  // namespace bmx
