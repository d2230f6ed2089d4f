// Products of 8-bit integers: y[t][n] = sx[t] sw[n] sum_k a[t][k] c[n][k], the sum exact in int32 (K <= 131,071), so that a result
// does not depend on tiles, splits or the tokens beside it. Rows of codes are whole 16-byte chunks with zeros past K.
//
// skinny8_k: few tokens, bound by the bytes of W. A workgroup has 16 RT rows of W (half of gate and half of up in the gated product);
// its eight waves take every eighth 128 columns of them straight from HBM to matrix operands, several steps ahead. Up to four
// tokens' rows are quantized by each workgroup itself while its first loads of W are on their way, into LDS: one launch instead of two.
// v_mfma_i32_16x16x64_i8: A = 16 tokens, B = 16 rows of W: lane l holds token / row l % 16 and columns (l / 16) * 16 .. + 15; of the
// result column (row of W) l % 16 and tokens (l / 16) * 4 .. + 3.
//
// gemm8_k: many tokens, gemm16_k's tiles: an 8-bit row of 128 columns is the 128 bytes of a 16-bit row of 64, and
// v_mfma_i32_32x32x32_i8 takes the same 16 bytes a lane in the same places as v_mfma_f32_32x32x16, for twice the products.
#pragma once
#include "rows8.hpp"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

namespace bmx {

constexpr int G8_K = 2 * GK;        // columns of a K tile
constexpr int S8_K = 128;           // columns of a step (skinny8_k)
constexpr int S8_W = 8;             // waves of a workgroup
constexpr int S8_SLOTS = 32;        // pieces of 512 values that a workgroup quantizes: 4 a wave

struct Q8Args {
    const int8_t* w[2];             // second: up
    const float* sw[2];
    int64_t ldw;
    const void* x;                  // rows to quantize (skinny8_k<true>), of row type xt, K values each
    int xt;
    const int8_t* xc;               // or codes
    const float* sx;
    int64_t ldx;
    int T, N, K;                    // N: rows of W (of each of the two matrices)
    int from;                       // W's first row: the rows before are another launch's
    void* out;                      // EPI_STORE: 16 bits of type ot; EPI_ADD: fp32 +=; EPI_GU: h fp32
    int ot, ldo;
    const float* scale;             // EPI_ADD: [T] or null
    ActPar act;
    int* part;                      // EPI_PART
    int tm, tn, splits, ldp;
};

// ---- few tokens ---------------------------------------------------------------------------------------------------------

inline bool skinny8_fused(int T, int K) { return K % 8 == 0 && (int64_t)T * ((K + 511) / 512) <= S8_SLOTS; }
inline size_t skinny8_lds(int T, int K) { return (size_t)T * (round_up(K, S8_K) + 16); }

template <bool FUSED, int RT, int EPI>
__global__ __launch_bounds__(S8_W * 64) void skinny8_k(const Q8Args p)
{
    constexpr bool GU = EPI == EPI_GU;
    constexpr int ROWS = GU ? 8 : 16, D = RT == 1 ? 4 : 2;         // result columns of a tile, steps in flight
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    // 16 tokens a workgroup; those of one block of rows follow one another on one XCD, so that all but the first find W in its L2
    int row = blockIdx.x, t0 = 0;
    if (p.T > 16)
    {
        const int tt = (p.T + 15) >> 4, rest = row >> 3;
        t0 = rest % tt * 16;
        row = rest / tt * 8 + (row & 7);
    }
    const int n0 = row * (ROWS * RT);
    if (n0 >= p.N) return;
    const int KP = (p.K + 15) & ~15, KT = (KP + S8_K - 1) / S8_K;

    extern __shared__ __attribute__((aligned(16))) char xl[];
    __shared__ uint32_t tops[S8_SLOTS];
    __shared__ float lsx[16];
    const int xrow = KT * S8_K + 16, spt = (p.K + 511) / 512;      // (rows an odd number of 16 bytes apart: 16 of them on all banks)
    Raw8 raw[4];
    if (FUSED)
#pragma unroll
        for (int n = 0; n < 4; ++n)
        {
            const int s = wave + n * S8_W, t = s / spt, h = s % spt * 512 + lane * 8;
            if (t < p.T && h < p.K) raw[n] = load_raw8(p.x, p.xt, (int64_t)t * p.K + h);
        }

    // this lane's rows of W, and whose (rows past the last load it again)
    const int mat = GU ? r >> 3 : 0;
    const int8_t* w[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) w[i] = p.w[mat] + (int64_t)min(n0 + i * ROWS + (GU ? r & 7 : r), p.N - 1) * p.ldw;
    const int8_t* xr = FUSED ? nullptr : p.xc + (int64_t)min(t0 + r, p.T - 1) * p.ldx;
    struct Step { u32x4 w[RT][2], x[FUSED ? 1 : 2]; } st[D];
    auto load = [&](Step& b, int kt) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            // past the last column the last again, beside zeros of x
            const int k = kt * S8_K + j * 64 + q * 16, at = min(k, KP - 16);
#pragma unroll
            for (int i = 0; i < RT; ++i) b.w[i][j] = ldg4(w[i] + at);
            if (FUSED) continue;
            const u32x4 x = ldg4(xr + at);
            b.x[FUSED ? 0 : j] = k < KP ? x : u32x4{0, 0, 0, 0};
        }
    };
    i32x4 acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = i32x4{0, 0, 0, 0};
    auto multiply = [&](const Step& b, int kt) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            const u32x4 x = FUSED ? *reinterpret_cast<const u32x4*>(xl + min(r, p.T - 1) * xrow + kt * S8_K + j * 64 + q * 16)
                                  : b.x[FUSED ? 0 : j];
#pragma unroll
            for (int i = 0; i < RT; ++i)
                acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x), __builtin_bit_cast(i32x4, b.w[i][j]), acc[i], 0, 0, 0);
        }
    };

    int kt = wave;                                                 // the next step to multiply; D are in flight
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (kt + d * S8_W < KT) load(st[d], kt + d * S8_W);
    if (FUSED)
    {
        float v[4][8];
#pragma unroll
        for (int n = 0; n < 4; ++n)
        {
            const int s = wave + n * S8_W, t = s / spt, h = s % spt * 512 + lane * 8;
            if (t >= p.T) break;
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[n][i] = 0.0f;
            if (h < p.K) to_f32(raw[n], p.xt, v[n]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, mag(v[n][i]));
            top = wave_max(top);
            if (lane == 0) tops[s] = top;
        }
        lds_barrier();
#pragma unroll
        for (int n = 0; n < 4; ++n)
        {
            const int s = wave + n * S8_W, t = s / spt, h = s % spt * 512 + lane * 8;
            if (t >= p.T) break;
            const Top8 o = top8(wave_max(lane < spt ? tops[t * spt + lane] : 0u));
            if (h < KT * S8_K)
                *reinterpret_cast<u32x2*>(xl + t * xrow + h) = u32x2{codes4(v[n], o), codes4(v[n] + 4, o)};
            if (s % spt == 0 && lane == 0) lsx[t] = o.scale;
        }
        lds_barrier();
    }
    while (kt < KT)
    {
#pragma unroll
        for (int d = 0; d < D; ++d)
        {
            if (kt >= KT) break;
            multiply(st[d], kt);
            if (kt + D * S8_W < KT) load(st[d], kt + D * S8_W);
            kt += S8_W;
        }
    }

    // join the waves
    constexpr int V = RT * 256;                                    // (row tile, element, lane)
    __shared__ int part[S8_W][V];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[wave][(i * 4 + e) * 64 + lane] = acc[i][e];
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += S8_W * 64)
    {
        const int c = i & 15, tl = ((i >> 4) & 3) * 4 + ((i >> 6) & 3), t = t0 + tl, n = n0 + (i >> 8) * ROWS + c;
        if (t >= p.T || c >= ROWS || n >= p.N) continue;
        auto sum = [&](int at) {
            int s = part[0][at];
#pragma unroll
            for (int w = 1; w < S8_W; ++w) s += part[w][at];
            return (float)s;
        };
        const float sx = FUSED ? lsx[tl] : p.sx[t], s = sum(i) * sx * p.sw[0][n];
        const int64_t o = (int64_t)t * p.ldo + n;
        if (GU) static_cast<float*>(p.out)[o] = act_h(p.act, s, sum(i + 8) * sx * p.sw[1][n]);
        else if (EPI == EPI_ADD)
        {
            float* y = static_cast<float*>(p.out) + o;
            *y = __builtin_fmaf(p.scale ? p.scale[t] : 1.0f, s, *y);
        }
        else static_cast<uint16_t*>(p.out)[o] = (uint16_t)bits16(p.ot, s);
    }
}

// ---- many tokens --------------------------------------------------------------------------------------------------------

// What becomes of 8 neighbouring sums (rows m .. m + 7 of W) of token n
__device__ __forceinline__ void times8(const Q8Args& p, int mat, int n, int m, const int (&s)[8], float (&v)[8])
{
    const float sx = p.sx[n];
    const float* sw = p.sw[mat] + p.from + m;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)s[i] * sx * (m + i < p.N ? sw[i] : 0.0f);
}

template <int EPI> __device__ __forceinline__ void put8(const Q8Args& p, int n, int m, const int (&s)[8], const int (&u)[8])
{
    float v[8];
    times8(p, 0, n, m, s, v);
    const int64_t o = (int64_t)n * p.ldo + p.from + m;
    if (EPI == EPI_GU)
    {
        float b[8];
        times8(p, 1, n, m, u, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_h(p.act, v[i], b[i]);
        store8(p.out, ROW_F32, o, v);
    }
    else if (EPI == EPI_ADD)
    {
        const float k = p.scale ? p.scale[n] : 1.0f;
        float* y = static_cast<float*>(p.out) + o;
        const Vals<8> c = load32<8>(y);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(k, v[i], c.v[i]);
        store8(y, ROW_F32, 0, v);
    }
    else if (!(p.ldo & 7)) store8(p.out, p.ot, o, v);
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (m + i < p.N) static_cast<uint16_t*>(p.out)[o + i] = (uint16_t)bits16(p.ot, v[i]);
    }
}

// BM rows of W x BN tokens by WK groups of WM x WN waves, NB buffers of a K tile each; as gemm16_tile, whose comments say why
template <int BM, int BN, int WM, int WN, int WK, int NB, int EPI>
__global__ __launch_bounds__(WM * WN * WK * 64) void gemm8_k(const Q8Args p)
{
    __shared__ __attribute__((aligned(1024))) char lds_all[gemm16_lds<BM, BN, WM, WN, WK, NB>()];
    constexpr int NT = WM * WN * 64;                               // threads of a group
    constexpr int MF = BM / WM / 32, NF = BN / WN / 32;            // 32 x 32 fragments of a wave
    constexpr int ABYTES = BM * G8_K, BBYTES = BN * G8_K;
    const int z = blockIdx.z;
    const int lane = threadIdx.x & 63, any = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = any / (WM * WN), wave = any % (WM * WN);
    char* lds = lds_all + group * (NB * (ABYTES + BBYTES));
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
    const int KP = (p.K + 15) & ~15;
    int kt = 0, kt_end = (KP + G8_K - 1) / G8_K;
    const int prod = EPI == EPI_PART ? z / p.splits : 0;
    if (EPI == EPI_PART)
    {
        const int q = kt_end / p.splits, r = kt_end % p.splits, sp = z - prod * p.splits;
        kt = sp * q + min(sp, r);
        kt_end = kt + q + (sp < r);
    }

    // the loaders count in 16-bit values: two codes
    TileLoader<BM, NT, WK, false, EPI == EPI_GU> la;
    TileLoader<BN, NT, WK, false, false> lb;
    la.init((int)(p.ldw / 2), wave);
    lb.init((int)(p.ldx / 2), wave);
    int loaded = kt + group;                                       // this group's next tile to load
    la.seek(p.w[prod], p.w[1], p.from + m0, loaded * GK, p.from + p.N, KP / 2, wave);
    lb.seek(p.xc, nullptr, n0, loaded * GK, p.T, KP / 2, wave);
    auto tail = [&]() { return KP / 2 - loaded * GK; };
    auto load_a = [&](lds_ptr to) { la.load(to, wave, tail(), loaded < kt_end); };
    auto load_b = [&](lds_ptr to) {
        lb.load(to + ABYTES, wave, tail(), loaded < kt_end);
        la.next();
        lb.next();
        loaded += WK;
    };
    // 32 rows from row0, 32 columns from ks * 32: lane l holds row l % 32, columns (l / 32) * 16 .. + 15
    auto frag = [&](lds_ptr tile, int row0, int ks) -> i32x4 {
        const int r = row0 + (lane & 31), c = ks * 2 + (lane >> 5);
        return *(__attribute__((address_space(3))) i32x4*)(tile + r * G8_K + ((c ^ swz_along(r)) << 4));
    };
    i32x16 acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    constexpr int KS = G8_K / 32;
    i32x4 a[2][MF], b[2][NF];
    auto read = [&](int set, lds_ptr at, int ks) {
#pragma unroll
        for (int i = 0; i < MF; ++i) a[set][i] = frag(at, wm * (BM / WM) + i * 32, ks);
#pragma unroll
        for (int j = 0; j < NF; ++j) b[set][j] = frag(at + ABYTES, wn * (BN / WN) + j * 32, ks);
    };
    auto products = [&](int set, int from, int to) {
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                if (i >= from && i < to) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[set][i], b[set][j], acc[i][j], 0, 0, 0);
    };
    constexpr int BEHIND = (la.INSTR + lb.INSTR) * (NB - 2);
    static_assert(BEHIND < 64, "vmcnt has 6 bits");
    auto landed = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_s_waitcnt(0x0070 | (BEHIND & 15) | (BEHIND >> 4) << 14);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    constexpr bool SPREAD = MF * NF >= 8, IN_STEPS = MF * NF >= 4;
    static_assert(!SPREAD || NB == 2, "spread loads end early: only a wait for all of them fits");
    auto tile = [&](lds_ptr __restrict__ at, lds_ptr __restrict__ to) __attribute__((always_inline)) {
        if (!SPREAD) { load_a(to); load_b(to); }
        read(0, at, 0);
        products((KS - 1) & 1, 0, MF);
        if (IN_STEPS) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS - 1; ++ks)
        {
            if (SPREAD)
            {
                if (loaded < kt_end)
                {
                    if (ks == 0) load_a(to);
                    if (ks == 1) load_b(to);
                }
                products(ks & 1, 0, MF / 2);
                __builtin_amdgcn_sched_barrier(0);
            }
            read((ks + 1) & 1, at, ks + 1);
            products(ks & 1, SPREAD ? MF / 2 : 0, MF);
            if (IN_STEPS) __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr int BUF = ABYTES + BBYTES;
#pragma unroll
    for (int i = 0; i < NB - 1; ++i)
    {
        load_a((lds_ptr)lds + i * BUF);
        load_b((lds_ptr)lds + i * BUF);
    }
    // the first tile follows products with zeros
#pragma unroll
    for (int i = 0; i < MF; ++i) a[(KS - 1) & 1][i] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NF; ++j) b[(KS - 1) & 1][j] = i32x4{0, 0, 0, 0};
    int buf = 0, before = NB - 1;
    for (; kt < kt_end; kt += WK)
    {
        landed();
        tile((lds_ptr)lds + buf * BUF, (lds_ptr)lds + before * BUF);
        before = buf;
        buf = buf + 1 == NB ? 0 : buf + 1;
    }
    products((KS - 1) & 1, 0, MF);

    // results, 32 tokens at a time turned over in LDS (gemm16_tile)
    constexpr int WROW = BM / WM, LROW = WROW + 4, AREA = WM * WN * 32 * LROW;
    int* turn = reinterpret_cast<int*>(lds_all) + wave * (32 * LROW);
    const int wm0 = EPI == EPI_GU ? m0 + wm * (WROW / 2) : m0 + wm * WROW;
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NF; ++j)
    {
        const int nb = n0 + wn * (BN / WN) + j * 32;
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<i32x4*>(turn + group * AREA + (lane & 31) * LROW + i * 32 + e * 2 + (lane >> 5) * 4) =
                    i32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
        if (WK > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        constexpr int PIECES = (EPI == EPI_GU ? WROW / 2 : WROW) / 8, MINE = 32 * PIECES / WK;
        static_assert(MINE % 64 == 0, "whole steps");
        for (int q = group * MINE + lane; q < (group + 1) * MINE; q += 64)
        {
            const int rr = q / PIECES, c = q % PIECES * 8, n = nb + rr, m = wm0 + c;
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
            else put8<EPI>(p, n, m, s, u);
        }
        if (WK > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
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
    put8<EPI>(p, n, m, sum[0], sum[1]);
}

}  // namespace bmx
