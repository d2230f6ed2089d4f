// Products of 8-bit integers: y[t][n] = sx[t] sw[n] sum_k a[t][k] c[n][k], the sum exact in int32 (K <= 131,071), so that a result
// does not depend on tiles, splits or the tokens beside it. Both factors lie in blocks of 16 rows x 64 columns (rows8.hpp).
//
// skinny8_k: to 128 tokens, bound by the bytes of W and by what a compute unit takes in. A workgroup has 16 or 32 rows of W (half of
// gate and half of up in the gated product) and all tokens; its eight waves take every eighth block of columns straight from HBM to
// matrix operands, several blocks ahead, with the tokens' blocks of the same columns from the caches. Few tokens' rows are quantized
// by each workgroup itself while its first loads of W are on their way, into LDS: one launch instead of two.
// v_mfma_i32_16x16x64_i8: A = 16 tokens, B = 16 rows of W: lane l holds token / row l % 16 and columns (l / 16) * 16 .. + 15; of the
// result column (row of W) l % 16 and tokens (l / 16) * 4 .. + 3.
//
// gemm8_k: many tokens, gemm16_k's tiles with v_mfma_i32_32x32x32_i8, in stages of 64 columns: as many bytes as half of gemm16_k's K
// tile, for as many products. gemm8_big_k: its largest tile, a workgroup one after the other.
#pragma once
#include "rows8.hpp"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

namespace bmx {

struct Q8Args {
    const int8_t* w[2];             // second: up
    const float* sw[2];
    const void* x;                  // rows to quantize (skinny8_k), of row type xt, K values each
    int xt;
    const int8_t* xc;               // or codes
    const float* sx;
    int T, N, K;                    // N: rows of W (of each of the two matrices)
    int from;                       // W's first row, a multiple of 16: the rows before are another launch's
    void* out;                      // EPI_STORE: 16 bits of type ot; EPI_ADD: fp32 +=; EPI_GU: h fp32
    int ot, ldo;
    const float* scale;             // EPI_ADD: [T] or null
    ActPar act;
    int* part;                      // EPI_PART
    int tm, tn, splits, ldp;
};

// ---- few tokens ---------------------------------------------------------------------------------------------------------

inline size_t skinny8_lds(int T, int K) { return (size_t)T * (q8_blocks(K) * Q8_COLS + 16); }

// TT: tiles of 16 tokens; RT: tiles of 16 rows of W. In the gated product RT 1 is eight rows of gate and eight of up, RT 2 16 of each.
// IN: the tokens are codes, or 16-bit or fp32 rows to be quantized by pieces of 512 values, NS a wave (with the other type's and three
// more pieces' code in the kernel a token's call took 0.7 us longer: instructions are fetched from L2 too).
enum Skinny8In { IN_CODES, IN_16, IN_32 };
template <int IN, int NS, int TT, int RT, int EPI>
__global__ __launch_bounds__(S8_W * 64) void skinny8_k(const Q8Args p)
{
    constexpr bool FUSED = IN != IN_CODES;
    const int xt = IN == IN_32 ? (int)ROW_F32 : p.xt == ROW_BF16 ? (int)ROW_BF16 : (int)ROW_F16;
    constexpr bool GU = EPI == EPI_GU, HALF = GU && RT == 1;
    constexpr int ROWS = GU ? 8 * RT : 16 * RT, D = TT + RT == 2 ? 8 : TT + RT <= 5 ? 4 : 3;     // result columns, blocks in flight
    static_assert(!FUSED || TT == 1, "one tile of tokens quantized here");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * ROWS, KB = q8_blocks(p.K);

    extern __shared__ __attribute__((aligned(16))) char xl[];
    __shared__ uint32_t tops[S8_SLOTS];
    __shared__ float lsx[16];
    const int xrow = KB * Q8_COLS + 16, spt = (p.K + 511) / 512;   // (rows an odd number of 16 bytes apart: 16 of them on all banks)
    Raw8 raw[NS];
    if (FUSED)
#pragma unroll
        for (int n = 0; n < NS; ++n)
        {
            const int s = wave + n * S8_W, t = s / spt, h = s % spt * 512 + lane * 8;
            if (t < p.T && h < p.K) raw[n] = load_raw8(p.x, xt, (int64_t)t * p.K + h);
        }

    // this lane's rows of W, and whose (rows past the last load it again)
    const int8_t* w[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        const int mat = HALF ? r >> 3 : GU ? i : 0, n = min(n0 + (HALF ? r & 7 : GU ? r : i * 16 + r), p.N - 1);
        w[i] = p.w[mat] + q8_at(n, q * 16, KB);
    }
    const int8_t* xr = FUSED ? nullptr : p.xc + q8_at(r, q * 16, KB);
    struct Step { u32x4 w[RT], x[FUSED ? 1 : TT]; } st[D];
    auto load = [&](Step& b, int kb) {
#pragma unroll
        for (int i = 0; i < RT; ++i) b.w[i] = ldg4(w[i] + (int64_t)kb * Q8_BLOCK);
        if (!FUSED)
#pragma unroll
            for (int i = 0; i < TT; ++i) b.x[FUSED ? 0 : i] = ldg4(xr + ((int64_t)i * KB + kb) * Q8_BLOCK);
    };
    i32x4 acc[RT][TT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    auto multiply = [&](const Step& b, int kb) {
#pragma unroll
        for (int j = 0; j < TT; ++j)
        {
            const u32x4 x = FUSED ? *reinterpret_cast<const u32x4*>(xl + min(r, p.T - 1) * xrow + kb * Q8_COLS + q * 16) : b.x[FUSED ? 0 : j];
#pragma unroll
            for (int i = 0; i < RT; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x), __builtin_bit_cast(i32x4, b.w[i]), acc[i][j], 0, 0, 0);
        }
    };

    int kb = wave;                                                 // the next block to multiply; D are in flight
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (kb + d * S8_W < KB) load(st[d], kb + d * S8_W);
    if (FUSED)
    {
        float v[NS][8];
#pragma unroll
        for (int n = 0; n < NS; ++n)
        {
            const int s = wave + n * S8_W, t = s / spt, h = s % spt * 512 + lane * 8;
            if (t >= p.T) break;
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[n][i] = 0.0f;
            if (h < p.K) to_f32(raw[n], xt, v[n]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, mag(v[n][i]));
            top = wave_max(top);
            if (lane == 0) tops[s] = top;
        }
        lds_barrier();
#pragma unroll
        for (int n = 0; n < NS; ++n)
        {
            const int s = wave + n * S8_W, t = s / spt, h = s % spt * 512 + lane * 8;
            if (t >= p.T) break;
            const Top8 o = top8(wave_max(lane < spt ? tops[t * spt + lane] : 0u));
            if (h < KB * Q8_COLS) *reinterpret_cast<u32x2*>(xl + t * xrow + h) = u32x2{codes4(v[n], o), codes4(v[n] + 4, o)};
            if (s % spt == 0 && lane == 0) lsx[t] = o.scale;
        }
        lds_barrier();
    }
    while (kb < KB)
    {
#pragma unroll
        for (int d = 0; d < D; ++d)
        {
            if (kb >= KB) break;
            multiply(st[d], kb);
            if (kb + D * S8_W < KB) load(st[d], kb + D * S8_W);
            kb += S8_W;
        }
    }

    // join the waves
    constexpr int V = RT * TT * 256;                               // (row tile, token tile, element, lane)
    __shared__ int part[S8_W][V];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[wave][((i * TT + j) * 4 + e) * 64 + lane] = acc[i][j][e];
    __syncthreads();
    constexpr int OUT = GU && RT == 2 ? V / 2 : V;                 // (up's sums lie TT tiles behind gate's)
    for (int i = threadIdx.x; i < OUT; i += S8_W * 64)
    {
        const int c = i & 15, tile = i >> 8, t = tile % TT * 16 + ((i >> 4) & 3) * 4 + ((i >> 6) & 3), n = n0 + tile / TT * 16 + c;
        if (t >= p.T || (HALF && c >= 8) || n >= p.N) continue;
        auto sum = [&](int at) {
            int s = part[0][at];
#pragma unroll
            for (int w = 1; w < S8_W; ++w) s += part[w][at];
            return (float)s;
        };
        const float sx = FUSED ? lsx[t] : p.sx[t], s = sum(i) * sx * p.sw[0][n];
        const int64_t o = (int64_t)t * p.ldo + n;
        if (GU) static_cast<float*>(p.out)[o] = act_h(p.act, s, sum(HALF ? i + 8 : i + TT * 256) * sx * p.sw[1][n]);
        else if (EPI == EPI_ADD)
        {
            float* y = static_cast<float*>(p.out) + o;
            *y = __builtin_fmaf(p.scale ? p.scale[t] : 1.0f, s, *y);
        }
        else static_cast<uint16_t*>(p.out)[o] = (uint16_t)bits16(p.ot, s);
    }
}

// ---- many tokens --------------------------------------------------------------------------------------------------------

// The scales of 8 neighbouring rows of W from row m of p.N (0 behind the last)
__device__ __forceinline__ void scales8(const Q8Args& p, int mat, int m, float (&w)[8])
{
    const float* sw = p.sw[mat] + p.from + m;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = m + i < p.N ? sw[i] : 0.0f;
}

// What becomes of 8 neighbouring sums (rows m .. m + 7 of W, of scales w; u: up's) of token n, of scale sx; k: its factor (EPI_ADD).
// OT: EPI_STORE's type, or ANY_OT: p.ot, what a launch says (known to the kernel, 4,096 x 4,096 x 11,008 175 -> 167 us)
constexpr int ANY_OT = -1;
template <int EPI, int OT>
__device__ __forceinline__ void put8(const Q8Args& p, int n, int m, const int (&s)[8], const int (&u)[8], float sx, float k,
                                     const float (&w)[8], const float (&wu)[8])
{
    const int ot = OT == ANY_OT ? p.ot : OT;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)s[i] * sx * w[i];
    const int64_t o = (int64_t)n * p.ldo + p.from + m;
    if (EPI == EPI_GU)
    {
        if (is_silu(p.act))                                
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = silu_h(v[i], (float)u[i] * sx * wu[i]);
        else
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_h(p.act, v[i], (float)u[i] * sx * wu[i]);
        store8(p.out, ROW_F32, o, v);
    }
    else if (EPI == EPI_ADD)
    {
        float* y = static_cast<float*>(p.out) + o;
        const Vals<8> c = load32<8>(y);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(k, v[i], c.v[i]);
        store8(y, ROW_F32, 0, v);
    }
    else if (!(p.ldo & 7)) store8(p.out, ot, o, v);
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (m + i < p.N) static_cast<uint16_t*>(p.out)[o + i] = (uint16_t)bits16(ot, v[i]);
    }
}

// BM rows of W x BN tokens by WK groups of WM x WN waves, NB buffers of a stage of 64 columns each; every group has every WK-th stage.
// A stage's loads go out NB - 1 stages ahead (two or three microseconds), each a contiguous block; as gemm16_tile otherwise, whose
// comments say why.
template <int BM, int BN, int WM, int WN, int WK, int NB> constexpr int gemm8_lds()
{
    constexpr int TILES = WK * NB * (BM + BN) * Q8_COLS, TURN = WM * WN * WK * 32 * (BM / WM + 4) * 4;
    return TILES > TURN ? TILES : TURN;
}

template <int BM, int BN, int WM, int WN, int WK, int NB, int EPI, int OT>
__global__ __launch_bounds__(WM * WN * WK * 64) void gemm8_k(const Q8Args p)
{
    __shared__ __attribute__((aligned(1024))) char lds_all[gemm8_lds<BM, BN, WM, WN, WK, NB>()];
    constexpr int NW = WM * WN;                                    // waves of a group
    constexpr int MF = BM / WM / 32, NF = BN / WN / 32;            // 32 x 32 fragments of a wave
    constexpr int ABYTES = BM * Q8_COLS, BUF = (BM + BN) * Q8_COLS, AL = BM / 16 / NW, BL = BN / 16 / NW;    // blocks a wave loads
    static_assert(AL * NW * 16 == BM && BL * NW * 16 == BN, "whole blocks");
    const int z = blockIdx.z;
    const int lane = threadIdx.x & 63, any = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = any / NW, wave = any % NW;
    const lds_ptr lds = (lds_ptr)lds_all + group * (NB * BUF);
    const int wm = wave / WN, wn = wave % WN;

    // an XCD on neighbouring tiles (gemm16_tile)
    const int nwg = p.tm * p.tn;
    int id = blockIdx.x;
    {
        const int q = nwg / 8, r = nwg % 8, x = id & 7;
        id = x * q + (x < r ? x : r) + (id >> 3);
    }
    constexpr int GRP = 8;
    const int per = GRP * p.tn, g0 = id / per * GRP, gn = min(GRP, p.tm - g0);
    const int tm = g0 + (id % per) % gn, tn = (id % per) / gn;
    const int m0 = EPI == EPI_GU ? tm * (BM / 2) : tm * BM, n0 = tn * BN;
    const int KB = q8_blocks(p.K);
    int kt = 0, kt_end = KB;
    const int prod = EPI == EPI_PART ? z / p.splits : 0;
    if (EPI == EPI_PART)
    {
        const int q = kt_end / p.splits, r = kt_end % p.splits, sp = z - prod * p.splits;
        kt = sp * q + min(sp, r);
        kt_end = kt + q + (sp < r);
    }

    // this wave's blocks of a stage: NW apart, rows of blocks past the last load it again. EPI_GU: two of gate, two of up in turn
    const char *ap[AL], *bp[BL];
    int loaded = kt + group;                                       // this group's next stage to load
    auto block = [&](const int8_t* m, int rb, int rows) {
        return reinterpret_cast<const char*>(m) + ((int64_t)min(rb, (rows - 1) / Q8_ROWS) * KB + loaded) * Q8_BLOCK;
    };
#pragma unroll
    for (int j = 0; j < AL; ++j)
    {
        const int i = wave + j * NW;
        ap[j] = EPI == EPI_GU ? block(i & 2 ? p.w[1] : p.w[0], (p.from + m0) / Q8_ROWS + (i >> 2) * 2 + (i & 1), p.from + p.N)
                              : block(p.w[prod], (p.from + m0) / Q8_ROWS + i, p.from + p.N);
    }
#pragma unroll
    for (int j = 0; j < BL; ++j) bp[j] = block(p.xc, n0 / Q8_ROWS + wave + j * NW, p.T);
    auto load = [&](lds_ptr to, const char*& from, int place) {
        // (past the last stage zeros: an empty range, so that the count of loads holds)
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(from), 0, loaded < kt_end ? Q8_BLOCK : 0, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + place * Q8_BLOCK), 16, lane * 16, 0, 0, 0);
        from += WK * Q8_BLOCK;
    };
    auto load_a = [&](lds_ptr to) {
#pragma unroll
        for (int j = 0; j < AL; ++j) load(to, ap[j], wave + j * NW);
    };
    auto load_b = [&](lds_ptr to) {
#pragma unroll
        for (int j = 0; j < BL; ++j) load(to + ABYTES, bp[j], wave + j * NW);
        loaded += WK;
    };
    // 32 rows from row0, 32 columns from ks * 32: lane l holds row l % 32, columns (l / 32) * 16 .. + 15
    const int frag_at = (lane >> 4 & 1) * Q8_BLOCK + (lane >> 5) * Q8_CHUNK + (lane & 15) * 16;
    auto frag = [&](lds_ptr at, int row0, int ks) -> i32x4 {
        return *(__attribute__((address_space(3))) i32x4*)(at + row0 * Q8_COLS + ks * 2 * Q8_CHUNK + frag_at);
    };
    i32x16 acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    i32x4 a[2][MF], b[2][NF];
    auto read = [&](int ks, lds_ptr at) {
#pragma unroll
        for (int i = 0; i < MF; ++i) a[ks][i] = frag(at, wm * (BM / WM) + i * 32, ks);
#pragma unroll
        for (int j = 0; j < NF; ++j) b[ks][j] = frag(at + ABYTES, wn * (BN / WN) + j * 32, ks);
    };
    auto products = [&](int ks, int from, int to) {
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                if (i >= from && i < to) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[ks][i], b[ks][j], acc[i][j], 0, 0, 0);
    };
    constexpr int BEHIND = (AL + BL) * (NB - 2);
    static_assert(BEHIND < 64, "vmcnt has 6 bits");
    auto landed = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_s_waitcnt(0x0070 | (BEHIND & 15) | (BEHIND >> 4) << 14);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    // One stage: the second half of the stage before's products first, so that the wait has products on both sides
    auto stage = [&](lds_ptr __restrict__ at, lds_ptr __restrict__ to) __attribute__((always_inline)) {
        read(0, at);
        products(1, 0, MF);
        __builtin_amdgcn_sched_barrier(0);
        load_a(to);
        products(0, 0, MF / 2);
        __builtin_amdgcn_sched_barrier(0);
        load_b(to);
        read(1, at);
        products(0, MF / 2, MF);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < NB - 1; ++i)
    {
        load_a(lds + i * BUF);
        load_b(lds + i * BUF);
    }
    // the first stage follows products with zeros
#pragma unroll
    for (int i = 0; i < MF; ++i) a[1][i] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NF; ++j) b[1][j] = i32x4{0, 0, 0, 0};
    int buf = 0, before = NB - 1;
    for (; kt < kt_end; kt += WK)                                  // group 0's stage; the others' may lie past the end: zeros
    {
        landed();
        stage(lds + buf * BUF, lds + before * BUF);
        before = buf;
        buf = buf + 1 == NB ? 0 : buf + 1;
    }
    products(1, 0, MF);

    // results, 32 tokens at a time turned over in LDS (gemm16_tile). A lane's pieces are the same 8 rows of W of different tokens: their
    // scales are loaded once, all tokens' before the pieces (loaded for each piece, the epilogue took 25 us of 4,096 x 4,096 x 11,008's
    // 187)
    constexpr int WROW = BM / WM, LROW = WROW + 4, AREA = WM * WN * 32 * LROW;
    constexpr int PIECES = (EPI == EPI_GU ? WROW / 2 : WROW) / 8, MINE = 32 * PIECES / WK, EACH = MINE / 64;
    static_assert(MINE % 64 == 0 && 64 % PIECES == 0, "whole steps, a lane's pieces in one column");
    int* turn = reinterpret_cast<int*>(lds_all) + wave * (32 * LROW);
    const int c = lane % PIECES * 8, m = (EPI == EPI_GU ? m0 + wm * (WROW / 2) : m0 + wm * WROW) + c;
    const int nb0 = n0 + wn * (BN / WN) + (group * MINE + lane) / PIECES;     // the lane's first token
    float w0[8], w1[8], sx[NF][EACH], add[NF][EACH];
    if (EPI != EPI_PART)
    {
        scales8(p, 0, m, w0);
        if (EPI == EPI_GU) scales8(p, 1, m, w1);
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int e = 0; e < EACH; ++e)
            {
                const int n = min(nb0 + j * 32 + e * (64 / PIECES), p.T - 1);
                sx[j][e] = p.sx[n];
                add[j][e] = EPI == EPI_ADD && p.scale ? p.scale[n] : 1.0f;
            }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NF; ++j)
    {
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<i32x4*>(turn + group * AREA + (lane & 31) * LROW + i * 32 + e * 2 + (lane >> 5) * 4) =
                    i32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
        if (WK > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
        for (int e = 0; e < EACH; ++e)
        {
            const int rr = (group * MINE + lane) / PIECES + e * (64 / PIECES), n = nb0 + j * 32 + e * (64 / PIECES);
            if (n >= p.T || m >= p.N) continue;
            auto piece = [&](int col, int (&v)[8]) {
#pragma unroll
                for (int w = 0; w < WK; ++w)
                {
                    const i32x4 lo = *reinterpret_cast<const i32x4*>(turn + w * AREA + rr * LROW + col);
                    const i32x4 hi = *reinterpret_cast<const i32x4*>(turn + w * AREA + rr * LROW + col + 4);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                    {
                        v[t] = w ? v[t] + lo[t] : lo[t];
                        v[t + 4] = w ? v[t + 4] + hi[t] : hi[t];
                    }
                }
            };
            int s[8], u[8];
            if (EPI == EPI_GU)
            {
                const int col = (c >> 5) * 64 + (c & 31);          // gate and up rows in turn by 32
                piece(col, s);
                piece(col + 32, u);
            }
            else piece(c, s);
            if (EPI == EPI_PART)
            {
                i32x4* to = reinterpret_cast<i32x4*>(p.part + ((int64_t)z * p.T + n) * p.ldp + m);
                to[0] = i32x4{s[0], s[1], s[2], s[3]};
                to[1] = i32x4{s[4], s[5], s[6], s[7]};
            }
            else put8<EPI, OT>(p, n, m, s, u, sx[j][e], add[j][e], w0, w1);
        }
        if (WK > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    }
}

// 256 x 256 results by 8 waves, a workgroup one tile after the other (every gridDim.x-th): the stages of its next tile are on their way
// while a tile's results are turned over and written, in LDS of their own (4 KB a wave). In a launch per tile the chip waits at each
// tile's two ends, 12 us for a tile of 65 at K 4096 (4,096 x 4,096 x 11,008 174 us, this way 162: 2.28 POP/s).
constexpr int BIG8 = 256, BIG8_NB = 4, BIG8_RING = BIG8_NB * 2 * BIG8 * Q8_COLS;

template <int EPI, int OT>
__global__ __launch_bounds__(512) void gemm8_big_k(const Q8Args p)
{
    constexpr int WN = 4, MF = 4, NF = 2, NB = BIG8_NB, ABYTES = BIG8 * Q8_COLS, BUF = 2 * ABYTES;
    constexpr bool GU = EPI == EPI_GU;
    constexpr int ROWS = GU ? BIG8 / 2 : BIG8;                     // rows of W (of each matrix) of a tile
    __shared__ __attribute__((aligned(1024))) char lds_all[BIG8_RING + 8 * 4096];
    const lds_ptr lds = (lds_ptr)lds_all;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    const int KB = q8_blocks(p.K), nwg = p.tm * p.tn;

    // tile `index` of the launch: an XCD on neighbouring tiles (gemm16_tile)
    struct At { int m0, n0; };
    auto place = [&](int index) {
        const int q = nwg / 8, r = nwg % 8, x = index & 7, id = x * q + (x < r ? x : r) + (index >> 3);
        constexpr int GRP = 8;
        const int per = GRP * p.tn, g0 = id / per * GRP, gn = min(GRP, p.tm - g0);
        return At{(g0 + (id % per) % gn) * ROWS, (id % per) / gn * BIG8};
    };

    // this wave's two blocks of each operand of a stage, and the stages: `left` of the tile whose loads go out, then the next tile's
    const char *ap[2], *bp[2];
    int loading = blockIdx.x, left = 0;
    auto seek = [&]() {
        if (loading >= nwg) return;
        const At t = place(loading);
        auto block = [&](const int8_t* m, int rb, int rows) {
            return reinterpret_cast<const char*>(m) + (int64_t)min(rb, (rows - 1) / Q8_ROWS) * KB * Q8_BLOCK;
        };
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            const int i = wave + j * 8, rb = (p.from + t.m0) / Q8_ROWS;
            ap[j] = GU ? block(i & 2 ? p.w[1] : p.w[0], rb + (i >> 2) * 2 + (i & 1), p.from + p.N) : block(p.w[0], rb + i, p.from + p.N);
            bp[j] = block(p.xc, t.n0 / Q8_ROWS + i, p.T);
        }
        left = KB;
    };
    auto load = [&](lds_ptr to, const char*& from, int at) {
        // (behind the last tile zeros: an empty range, so that the count of loads holds)
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(from), 0, left ? Q8_BLOCK : 0, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + at * Q8_BLOCK), 16, lane * 16, 0, 0, 0);
        from += Q8_BLOCK;
    };
    auto load_a = [&](lds_ptr to) {
        load(to, ap[0], wave);
        load(to, ap[1], wave + 8);
    };
    auto load_b = [&](lds_ptr to) {
        load(to + ABYTES, bp[0], wave);
        load(to + ABYTES, bp[1], wave + 8);
        if (left && --left == 0)
        {
            loading += gridDim.x;
            seek();
        }
    };
    const int frag_at = (lane >> 4 & 1) * Q8_BLOCK + (lane >> 5) * Q8_CHUNK + (lane & 15) * 16;
    auto frag = [&](lds_ptr at, int row0, int ks) -> i32x4 {
        return *(__attribute__((address_space(3))) i32x4*)(at + row0 * Q8_COLS + ks * 2 * Q8_CHUNK + frag_at);
    };
    i32x16 acc[MF][NF];
    i32x4 a[2][MF], b[2][NF];
    auto read = [&](int ks, lds_ptr at) {
#pragma unroll
        for (int i = 0; i < MF; ++i) a[ks][i] = frag(at, wm * 128 + i * 32, ks);
#pragma unroll
        for (int j = 0; j < NF; ++j) b[ks][j] = frag(at + ABYTES, wn * 64 + j * 32, ks);
    };
    auto products = [&](int ks, int from, int to) {
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                if (i >= from && i < to) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[ks][i], b[ks][j], acc[i][j], 0, 0, 0);
    };
    // (the epilogue's loads and stores are counted too: behind one the wait is for more than the stage's loads, never for fewer)
    constexpr int BEHIND = 4 * (NB - 2);
    auto landed = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_s_waitcnt(0x0070 | (BEHIND & 15) | (BEHIND >> 4) << 14);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    auto stage = [&](lds_ptr __restrict__ at, lds_ptr __restrict__ to) __attribute__((always_inline)) {
        read(0, at);
        products(1, 0, MF);
        __builtin_amdgcn_sched_barrier(0);
        load_a(to);
        products(0, 0, MF / 2);
        __builtin_amdgcn_sched_barrier(0);
        load_b(to);
        read(1, at);
        products(0, MF / 2, MF);
        __builtin_amdgcn_sched_barrier(0);
    };

    seek();
#pragma unroll
    for (int i = 0; i < NB - 1; ++i)
    {
        load_a(lds + i * BUF);
        load_b(lds + i * BUF);
    }
    int buf = 0, before = NB - 1;
    char* turn = lds_all + BIG8_RING + wave * 4096;                // 32 tokens x 128 bytes, chunk c of 16 at c ^ (token / 2 % 8)
    for (int tile = blockIdx.x; tile < nwg; tile += gridDim.x)
    {
#pragma unroll
        for (int i = 0; i < MF; ++i)
        {
            a[1][i] = i32x4{0, 0, 0, 0};                           // the first stage follows products with zeros
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
        }
#pragma unroll
        for (int j = 0; j < NF; ++j) b[1][j] = i32x4{0, 0, 0, 0};
        for (int k = 0; k < KB; ++k)
        {
            landed();
            stage(lds + buf * BUF, lds + before * BUF);
            before = buf;
            buf = buf + 1 == NB ? 0 : buf + 1;
        }
        products(1, 0, MF);

        // A lane's sums are token l % 32 and rows g * 8 + (l / 32) * 4 .. + 3 of a fragment: scaled where they are, then turned over 128
        // bytes of 32 tokens at a time, so that whole pieces of rows are written
        const At t = place(tile);
        const int half = lane >> 5, mw = t.m0 + wm * (ROWS / 2), nw = t.n0 + wn * 64;
        const bool whole = t.m0 + ROWS <= p.N, silu = is_silu(p.act);
        auto scales = [&](int mat, int m, f32x4 (&w)[4]) {         // of a fragment's rows from m
            const float* sw = p.sw[mat] + p.from;
#pragma unroll
            for (int g = 0; g < 4; ++g)
            {
                const int at = m + g * 8 + half * 4;
                if (whole) w[g] = f32x4{sw[at], sw[at + 1], sw[at + 2], sw[at + 3]};
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[g][e] = at + e < p.N ? sw[at + e] : 0.0f;
            }
        };
        float sx[NF];
#pragma unroll
        for (int j = 0; j < NF; ++j) sx[j] = p.sx[min(nw + j * 32 + (lane & 31), p.T - 1)];
        auto value = [&](const i32x16& s, int g, int e, float x, const f32x4 (&w)[4]) { return (float)s[g * 4 + e] * x * w[g][e]; };
        constexpr int FR = EPI == EPI_ADD ? 1 : 2;                 // fragments turned over together
#pragma unroll
        for (int i = 0; i < MF; i += FR)
        {
            f32x4 w[FR][4];
            const int m = mw + (GU ? i / 2 : i) * 32;
#pragma unroll
            for (int f = 0; f < FR; ++f) scales(GU ? f : 0, GU ? m : m + f * 32, w[f]);
#pragma unroll
            for (int j = 0; j < NF; ++j)
            {
                const int row = lane & 31, swz = (row >> 1) & 7;
                char* to = turn + row * 128;
#pragma unroll
                for (int g = 0; g < 4; ++g)
                {
                    if (EPI == EPI_STORE)
                    {
#pragma unroll
                        for (int f = 0; f < FR; ++f)
                        {
                            uint32_t h[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) h[e] = bits16(OT, value(acc[i + f][j], g, e, sx[j], w[f]));
                            *reinterpret_cast<u32x2*>(to + (((f * 4 + g) ^ swz) << 4) + half * 8) = u32x2{h[0] | h[1] << 16, h[2] | h[3] << 16};
                        }
                    }
                    else
                    {
                        f32x4 v;
                        auto gate = [&](int e) { return value(acc[i][j], g, e, sx[j], w[0]); };
                        auto up = [&](int e) { return value(acc[GU ? i + 1 : i][j], g, e, sx[j], w[FR - 1]); };
                        if (GU && silu)
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = silu_h(gate(e), up(e));
                        else
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = GU ? act_h(p.act, gate(e), up(e)) : gate(e);
                        *reinterpret_cast<f32x4*>(to + (((g * 2 + half) ^ swz) << 4)) = v;
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    const int rr = e * 8 + (lane >> 3), c = lane & 7, n = nw + j * 32 + rr;
                    const u32x4 v = *reinterpret_cast<const u32x4*>(turn + rr * 128 + ((c ^ ((rr >> 1) & 7)) << 4));
                    const int at = m + c * (EPI == EPI_STORE ? 8 : 4);
                    if (n >= p.T || at >= p.N) continue;
                    const int64_t o = (int64_t)n * p.ldo + p.from + at;
                    if (EPI == EPI_STORE)
                    {
                        uint16_t* y = static_cast<uint16_t*>(p.out) + o;
                        if (!(p.ldo & 7)) *reinterpret_cast<u32x4*>(y) = v;
                        else
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (at + k < p.N) y[k] = (uint16_t)(v[k / 2] >> (16 * (k & 1)));
                    }
                    else
                    {
                        f32x4* y = reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + o);
                        if (GU) *y = __builtin_bit_cast(f32x4, v);
                        else
                        {
                            const f32x4 d = __builtin_bit_cast(f32x4, v), c0 = ldg4f(reinterpret_cast<const float*>(y));
                            const float k = p.scale ? p.scale[n] : 1.0f;
                            *y = f32x4{__builtin_fmaf(k, d[0], c0[0]), __builtin_fmaf(k, d[1], c0[1]), __builtin_fmaf(k, d[2], c0[2]),
                                       __builtin_fmaf(k, d[3], c0[3])};
                        }
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
    }
}

// The sums over the splits (EPI_PART) and what EPI does with them: 8 values a thread
template <int EPI>
__global__ __launch_bounds__(64) void finish8_k(const Q8Args p)
{
    constexpr int PRODS = EPI == EPI_GU ? 2 : 1, B = 8 / PRODS;
    const int64_t plane = (int64_t)p.T * p.ldp, at = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 8;
    if (at >= plane) return;
    const int n = (int)(at / p.ldp), m = (int)(at % p.ldp);
    int sum[2][8] = {};
    float w0[8], w1[8];
    scales8(p, 0, m, w0);
    if (EPI == EPI_GU) scales8(p, 1, m, w1);
    const float sx = p.sx[n], add = EPI == EPI_ADD && p.scale ? p.scale[n] : 1.0f;
    for (int s0 = 0; s0 < p.splits; s0 += B)
    {
        i32x4 v[PRODS][B][2];
#pragma unroll
        for (int s = 0; s < B; ++s)
#pragma unroll
            for (int k = 0; k < PRODS; ++k)
                if (s0 + s < p.splits)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        v[k][s][h] = __builtin_bit_cast(i32x4, ldg4(p.part + (k * p.splits + s0 + s) * plane + at + h * 4));
#pragma unroll
        for (int s = 0; s < B; ++s)
#pragma unroll
            for (int k = 0; k < PRODS; ++k)
                if (s0 + s < p.splits)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[k][i] += v[k][s][i / 4][i % 4];
    }
    put8<EPI, ANY_OT>(p, n, m, sum[0], sum[1], sx, add, w0, w1);
}

}  // namespace bmx
