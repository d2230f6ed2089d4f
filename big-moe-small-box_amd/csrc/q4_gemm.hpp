// Many tokens times a 4-bit matrix: y[t][n] = sum_k x[t][k] scale (code - zero), 128 tokens x 128 rows of W a workgroup. The
// codes stay codes until they are operands: a step's 8 KB of them lie in LDS beside 32 KB of x, a lane reads its 32 rows' 64
// codes of 128 columns with two loads and decodes eight at a time for one matrix instruction (skinny.hpp, Q4Dec). Scales and
// zero points go onto each group's sums, so the weights are never rounded. Against decoding the matrix to 16 bits first (the
// bytes written and read again: 4096 -> 11008 23 us beside a product of 57 for 517 tokens, 80) this wins, 71 us, until the tokens
// are so many that the larger tiles of gemm16_k pay for it (q4_whole_most; 4,096 tokens 437 against 317 us). A wave's step is 32
// matrix instructions (1,024 cycles, 1,280 with the bf16 correction) and about 240 others.
//
// v_mfma_f32_32x32x16: A = 32 tokens, B = 32 rows of W; the result's column is the row of W, its rows the tokens.
#pragma once
#include "skinny.hpp"

namespace bmx {

struct Q4GemmArgs {
    GemmArgs g;             // M: rows of W (EPI_GU: of each matrix), N: tokens, K; outputs and epilogue as gemm16_k's
    Q4View q[2];
    const uint16_t* x;
    const float* xs;        // bf16: [groups][padded tokens] sums of x over each group
    int xs_ld;
};

// xs[g][t] = sum of x[t] over group g, 0 for the groups between K and its next multiple of 128; 8 values a lane, the G / 8
// lanes of a group are neighbours
template <class T, int G>
__global__ __launch_bounds__(256) void group_sums_k(const uint16_t* __restrict__ x, int n, int K, float* __restrict__ xs, int ld)
{
    const int chunks = (K + SK_K - 1) / SK_K * (SK_K / 8);
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, t = i / chunks;
    const int c = (int)(i % chunks);
    float sum = 0.0f;
    if (t < n && c * 8 < K)
    {
        const u32x4 v = ldg4(x + t * K + c * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += from16<T>((uint16_t)v[e]) + from16<T>((uint16_t)(v[e] >> 16));
    }
#pragma unroll
    for (int o = 1; o < G / 8; o <<= 1) sum += __shfl_xor(sum, o);
    if (t < n && c % (G / 8) == 0) xs[(int64_t)(c / (G / 8)) * ld + t] = sum;
}

template <class T, int G, int EPI>
__global__ __launch_bounds__(256, 2) void gemm_q4_k(const Q4GemmArgs qp)
{
    typedef typename Elem<T>::v8 v8;
    constexpr bool OFFSET = Q4Dec<T>::OFFSET, GATED = EPI == EPI_GU;
    constexpr int NG = SK_K / G, MT = 2, NW = 2;                   // groups of a step; a wave's 32-token and 32-row fragments
    constexpr int XB = QG_T * GK * 2, CB = QG_N * SK_K / 2, STEP = 2 * XB + CB;
    const GemmArgs& p = qp.g;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STEP];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, r = lane & 15, half = (lane >> 4) & 1, h = lane >> 5;
    const int nwg = p.tm * p.tn;
    int id = blockIdx.x;
    {
        const int q = nwg / 8, m = nwg % 8, x = id & 7;             // an XCD takes a contiguous run of tiles
        id = x * q + (x < m ? x : m) + (id >> 3);
    }
    // a run walks the tokens within one tile of rows: W is read once, x stays in the XCD's L2
    const int n0 = id / p.tn * (GATED ? QG_N / 2 : QG_N), t0 = id % p.tn * QG_T, z = blockIdx.z;
    const int KT = (p.K + SK_K - 1) / SK_K, NT = (p.M + 15) / 16;
    const int prod = EPI == EPI_PART ? z / p.splits : 0;
    int kt = 0, kt_end = KT;
    if (EPI == EPI_PART)
    {
        const int q = KT / p.splits, m = KT % p.splits, sp = z - prod * p.splits;
        kt = sp * q + min(sp, m);
        kt_end = kt + q + (sp < m);
    }

    TileLoader<QG_T, 256, 1, false, false> lx;
    lx.init(p.K, wave);
    lx.seek(qp.x, nullptr, t0, kt * SK_K, p.N, p.K, wave);
    // the 8 tiles of 16 rows of a workgroup: slot = (wave column, fragment, half); gated, fragment 0 is of gate, 1 of up
    auto tile_of = [&](int slot, int& mat) {
        mat = GATED ? (slot >> 1) & 1 : prod;
        const int nt = n0 / 16 + (GATED ? (slot >> 2) * 2 + (slot & 1) : slot);
        return min(nt, NT - 1);                                    // past the last row: that tile again, never stored
    };
    int loaded = kt;
    auto load = [&](int buf) {
        lds_ptr to = (lds_ptr)lds + buf * STEP;
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            lx.load(to + i * XB, wave, p.K - loaded * SK_K - i * GK, true);
            lx.next();
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            int mat;
            const int nt = tile_of(wave + i * 4, mat);
            const u32x4* c = (mat ? qp.q[1] : qp.q[0]).codes + ((int64_t)nt * KT + loaded) * 64;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                __builtin_amdgcn_make_buffer_rsrc(const_cast<u32x4*>(c), 0, 1024, 0x00020000),
                (__attribute__((address_space(3))) void*)(to + 2 * XB + (wave + i * 4) * 1024), 16, lane * 16, 0, 0, 0);
        }
        ++loaded;
    };
    // Scales and zero points of this lane's rows of W, and (bf16) the sums of x of its tokens, a step ahead. The 128 + zero
    // that bf16 codes carry too much come off as one more product over the groups, sums of x times -scale (128 + zero), on
    // the fp32 matrix instruction of two columns: lanes 0 .. 31 hold the even group of a pair, 32 .. 63 the odd (or nothing).
    constexpr int NP = (NG + 1) / 2;
    struct Scales { uint16_t s[NW][NG]; uint8_t z[NW][NG]; float xs[MT][NP]; } sc, sn;
    auto load_scales = [&](Scales& v, int at) {
#pragma unroll
        for (int i = 0; i < NW; ++i)
        {
            int mat;
            const int nt = tile_of((wn * 2 + i) * 2 + half, mat);
            const uint16_t* s = mat ? qp.q[1].scale : qp.q[0].scale;
            const uint8_t* zp = mat ? qp.q[1].zero : qp.q[0].zero;
#pragma unroll
            for (int g = 0; g < NG; ++g)
            {
                const int64_t o = ((int64_t)nt * (KT * NG) + at * NG + g) * 16 + r;
                v.s[i][g] = s[o];
                v.z[i][g] = zp ? zp[o] : 8;
            }
        }
        if (OFFSET)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                {
                    const int g = q * 2 + (NG > 1 ? h : 0);
                    const float xs = qp.xs[(int64_t)(at * NG + g) * qp.xs_ld + t0 + wm * 64 + m * 32 + (lane & 31)];
                    v.xs[m][q] = NG == 1 && h ? 0.0f : xs;
                }
    };
    const bool sbf[2] = {(GATED ? qp.q[0] : qp.q[prod]).scale_bf16 != 0, (GATED ? qp.q[1] : qp.q[prod]).scale_bf16 != 0};

    f32x16 acc[MT][NW];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][i][e] = 0.0f;

    load(0);
    load_scales(sc, kt);
    for (int buf = 0; kt < kt_end; ++kt, buf ^= 1)
    {
        // vmcnt 0: the step is in LDS; lgkmcnt 0: the one before is read
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_s_waitcnt(0x0070);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (kt + 1 < kt_end)
        {
            load(buf ^ 1);
            load_scales(sn, kt + 1);
        }
        lds_ptr at = (lds_ptr)lds + buf * STEP;
        u32x4 code[NW][2];
#pragma unroll
        for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int o = 0; o < 2; ++o)
                code[i][o] = *(__attribute__((address_space(3))) u32x4*)(at + 2 * XB + ((wn * 2 + i) * 2 + half) * 1024 +
                                                                         ((o * 2 + h) * 16 + r) * 16);
        // x fragments one product ahead
        v8 x[2][MT];
        auto read = [&](int kk) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
            {
                const int row = wm * 64 + m * 32 + (lane & 31), c = (kk & 3) * 2 + h;
                x[kk & 1][m] = *(__attribute__((address_space(3))) v8*)(at + (kk >> 2) * XB + row * (GK * 2) + ((c ^ swz_along(row)) << 4));
            }
        };
        read(0);
#pragma unroll
        for (int g = 0; g < NG; ++g)
        {
            Q4Dec<T> dec[NW];
#pragma unroll
            for (int i = 0; i < NW; ++i) dec[i].zero((float)sc.z[i][g]);
            f32x16 part[MT][NW];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < NW; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) part[m][i][e] = 0.0f;
#pragma unroll
            for (int kk = g * (G / 16); kk < (g + 1) * (G / 16); ++kk)
            {
                v8 w[NW];
                if (kk < 7) read(kk + 1);
#pragma unroll
                for (int i = 0; i < NW; ++i) w[i] = dec[i](code[i][kk & 1][kk >> 1]);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < NW; ++i) part[m][i] = Elem<T>::mfma32(x[kk & 1][m], w[i], part[m][i]);
            }
            float s[NW], off[NW];
#pragma unroll
            for (int i = 0; i < NW; ++i)
            {
                s[i] = sbf[i] ? from16<bf16>(sc.s[i][g]) : from16<f16>(sc.s[i][g]);
                off[i] = s[i] * (-128.0f - (float)sc.z[i][g]);
                if (NG > 1 && (g & 1))
                {
                    const float even = (sbf[i] ? from16<bf16>(sc.s[i][g & ~1]) : from16<f16>(sc.s[i][g & ~1])) *
                                       (-128.0f - (float)sc.z[i][g & ~1]);
                    off[i] = h ? off[i] : even;
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < NW; ++i)
                {
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[m][i][e] = __builtin_fmaf(s[i], part[m][i][e], acc[m][i][e]);
                    if (OFFSET && (NG == 1 || (g & 1)))
                        acc[m][i] = __builtin_amdgcn_mfma_f32_32x32x2f32(sc.xs[m][g / 2], off[i], acc[m][i], 0, 0, 0);
                }
        }
        sc = sn;
    }

    // results: lane l holds row l % 32 of W and tokens (e / 4) * 8 + (l / 32) * 4 + e % 4 of a fragment; turned over in LDS
    constexpr int WROW = NW * 32, LROW = WROW + 4;
    float* turn = reinterpret_cast<float*>(lds) + wave * (32 * LROW);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m)
    {
#pragma unroll
        for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) turn[((e >> 2) * 8 + h * 4 + (e & 3)) * LROW + i * 32 + (lane & 31)] = acc[m][i][e];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        store_turned<T, EPI, WROW, 1>(p, turn, 0, lane, 0, t0 + wm * 64 + m * 32, n0 + wn * (GATED ? 32 : 64), z, prod);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    }
}

}  // namespace bmx
