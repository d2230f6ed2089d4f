// Tiled 16-bit matrix product for gfx950: D[n][m] = sum_k A(m, k) B(n, k), the products of the gated feed-forward block and
// of its gradients (many tokens). A is the side whose index m is contiguous in the result's rows, so that a lane's four
// neighbouring accumulators are four neighbouring values of one row.
//
// An operand is stored [rows][K] ("along K": weights of a forward product, activations) or [K][rows] ("across K": weights of
// a product with their transpose, both sides of a weight gradient). Either way its tile goes from HBM to LDS by 16-byte
// direct loads in the order in which it lies in memory; operands across K are transposed on the way to registers by
// ds_read_b64_tr_b16. Rows and columns outside the matrices come from the buffer range check as zeros (last rows) or hold
// neighbouring data whose results are never stored.
#pragma once
#include "ffn_act.hpp"
#include "bmx_internal.hpp"
#include "product_plan.hpp"

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

namespace bmx {

template <class T> struct Elem;
template <> struct Elem<f16>
{
    typedef f16x8 v8;
    static __device__ __forceinline__ f32x16 mfma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mfma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<bf16>
{
    typedef bf16x8 v8;
    static __device__ __forceinline__ f32x16 mfma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mfma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// 16-bit value of an fp32 one (round to nearest even) and back, as bits
template <class T> __device__ __forceinline__ uint16_t to16(float v) { return __builtin_bit_cast(uint16_t, (T)v); }
template <class T> __device__ __forceinline__ float from16(uint16_t b) { return (float)__builtin_bit_cast(T, b); }

// What a product does with its sums
enum GemmEpi {
    EPI_STORE = 0,   // out[n][m], 16 bits
    EPI_ADD = 1,     // out32[n][m] += scale[n] * sum
    EPI_PART = 2,    // part[matrix * splits + split][n][m] fp32: K in several splits, joined by gemm_finish_k
    EPI_GU = 3,      // the rows of A are gate and up rows in turn by 32: h = act(g, u) (and g, u for a backward pass)
    EPI_DGU = 4,     // the sum is dh: dg = dh dh/dg, du = dh dh/du from the saved g, u
};

struct GemmArgs {
    const void* a[2];       // second: the up matrix (EPI_GU), or the second product of a chain or batch
    const void* b[2];
    void* out[2];
    int M, N, K;            // M: rows of A (EPI_GU: of each of its two matrices), N: rows of B
    int from;               // A's first row: the rows before are another launch's; out, g and u start at it
    int lda, ldb, ldo;      // elements
    int ldp;                // EPI_PART: row of the partial sums, a multiple of 8
    int chain;              // 2: the two products are summed
    int batch;              // 2: two products side by side (grid z)
    int splits;             // of K (EPI_PART; grid z = product * splits + split)
    int tm, tn;             // tiles along M and N
    float* part;
    const float* scale;     // EPI_ADD: [N] or null
    ActPar act;
    float *g, *u;           // EPI_GU: kept when not null; EPI_DGU: read. fp32: a backward pass from g and u of 16 bits is off
                            // by as much again as its results' own rounding (both, and dg's: 1.8 times; this way 1.4)
};

typedef __attribute__((address_space(3))) char* lds_ptr;

// W (4 or 8) neighbouring values of a result row: 8 or 16 bytes of 16-bit values
template <int W> struct Vals { float v[W]; };

template <class T, int W> __device__ __forceinline__ void store16(uint16_t* q, const Vals<W>& v)
{
    uint32_t w[W / 2];
#pragma unroll
    for (int i = 0; i < W / 2; ++i) w[i] = (uint32_t)to16<T>(v.v[2 * i]) | (uint32_t)to16<T>(v.v[2 * i + 1]) << 16;
    if constexpr (W == 8) *reinterpret_cast<u32x4*>(q) = u32x4{w[0], w[1], w[2], w[3]};
    else *reinterpret_cast<u32x2*>(q) = u32x2{w[0], w[1]};
}
template <int W> __device__ __forceinline__ void store32(float* q, const Vals<W>& v)
{
#pragma unroll
    for (int i = 0; i < W; i += 4) *reinterpret_cast<f32x4*>(q + i) = f32x4{v.v[i], v.v[i + 1], v.v[i + 2], v.v[i + 3]};
}
template <int W> __device__ __forceinline__ Vals<W> load32(const float* q)
{
    Vals<W> v;
#pragma unroll
    for (int i = 0; i < W; i += 4)
    {
        const f32x4 a = ldg4f(q + i);
#pragma unroll
        for (int t = 0; t < 4; ++t) v.v[i + t] = a[t];
    }
    return v;
}

// What becomes of W neighbouring sums of a result row (columns m .. m + W - 1), at element o of the outputs. Rows are
// multiples of 8 values except in put (4-bit matrices of any N), where the last ones are stored one by one.
template <class T, int W> __device__ __forceinline__ void put(const GemmArgs& p, void* out, int64_t o, int m, const Vals<W>& v)
{
    uint16_t* q = static_cast<uint16_t*>(out) + o;
    if (!(p.ldo & 7)) { store16<T>(q, v); return; }
#pragma unroll
    for (int t = 0; t < W; ++t)
        if (m + t < p.M) q[t] = to16<T>(v.v[t]);
}

template <int W> __device__ __forceinline__ void put_add(const GemmArgs& p, int64_t o, int n, const Vals<W>& v)
{
    const float sc = p.scale ? p.scale[n] : 1.0f;
    float* q = static_cast<float*>(p.out[0]) + o;
    Vals<W> c = load32<W>(q);
#pragma unroll
    for (int t = 0; t < W; ++t) c.v[t] = __builtin_fmaf(sc, v.v[t], c.v[t]);
    store32(q, c);
}

// h goes to 16 bits: down's matrix instructions take factors of 16, and a second product for what the rounding leaves would be a
// third of the block's work again. y's error against 64 bits is 1.4 times that of the formulas in fp32 for it (bf16, one token to
// 4,096: 0.0023 against 0.0017 of the norm, the rounding of y itself; fp16 0.00028 / 0.00021).
template <class T, int W> __device__ __forceinline__ void put_gu(const GemmArgs& p, int64_t o, const Vals<W>& g, const Vals<W>& u)
{
    Vals<W> h;
#pragma unroll
    for (int t = 0; t < W; ++t) h.v[t] = act_h(p.act, g.v[t], u.v[t]);
    store16<T>(static_cast<uint16_t*>(p.out[0]) + o, h);
    if (p.g)
    {
        store32(p.g + o, g);
        store32(p.u + o, u);
    }
}

// g and u, loaded ahead of their use
template <int W> struct GU { Vals<W> g, u; };
template <int W> __device__ __forceinline__ GU<W> load_gu(const GemmArgs& p, int64_t o) { return {load32<W>(p.g + o), load32<W>(p.u + o)}; }

// dg and du go to 16 bits, factors of the next products as h is: the gradients' errors are 1.4 times the fp32 formulas' too
template <class T, int W> __device__ __forceinline__ void put_dgu(const GemmArgs& p, int64_t o, const Vals<W>& dh, const GU<W>& s)
{
    Vals<W> dg, du;
#pragma unroll
    for (int t = 0; t < W; ++t)
    {
        float hg, hu;
        act_grad(p.act, s.g.v[t], s.u.v[t], hg, hu);
        dg.v[t] = dh.v[t] * hg;
        du.v[t] = dh.v[t] * hu;
    }
    store16<T>(static_cast<uint16_t*>(p.out[0]) + o, dg);
    store16<T>(static_cast<uint16_t*>(p.out[1]) + o, du);
}

// ---- tiles --------------------------------------------------------------------------------------------------------------
// LDS position of 16-byte chunk c of row r. Along K: a row is 64 values = 8 chunks; 16 rows at one chunk (a fragment read)
// fall on 16 different 16-byte columns of the 64 banks. Across K: a row is the tile's rows; the 4 rows x 64 bytes that 32 lanes
// read for a transposition fall on four different quarters of the banks (with 32 bytes as the unit the reads took twice the
// cycles: 256 bytes go out at a time).
__device__ __forceinline__ int swz_along(int r) { return (r >> 1) & 7; }
// Rows of 64 values are half the banks: two of the four lie apart by themselves.
template <int ROWS> __device__ __forceinline__ int swz_across(int r) { return ROWS == 64 ? (r & 2) << 1 : (r & 3) << 2; }

// One operand's tiles of ROWS rows x GK, loaded by the NT threads of a group in INSTR loads of 16 bytes each, every
// WK-th one. ACROSS: stored [K][rows].
// GU: the rows are 32 of one matrix and 32 of a second in turn.
template <int ROWS, int NT, int WK, bool ACROSS, bool GU>
struct TileLoader {
    static constexpr int INSTR = ROWS * GK * 2 / (NT * 16);
    static constexpr int CPR = ACROSS ? ROWS / 8 : GK / 8;         // chunks of an LDS row
    static constexpr int RPI = NT / CPR;                           // LDS rows of one load of all threads
    static_assert(RPI % (ACROSS ? 4 : 16) == 0 && (!GU || RPI == 32 || RPI == 64), "later loads' rows are swizzled as the first's, and of one matrix per wave");
    const char *base0, *base1;      // the tile's first element, in the matrix of the even and of the odd loads
    int64_t left;       // bytes from there to the matrix's last
    int64_t step;       // bytes to the group's next tile along K
    int rows_ld;        // bytes of a matrix row
    uint32_t voff;      // of this lane's chunk in the first load (bytes from the tile's base)
    int chunk;          // ... its column chunk in the matrix
    __device__ __forceinline__ void init(int ld, int wave)
    {
        const int id = threadIdx.x % NT, r = GU ? (wave * 8 & 31) + (id & 63) / 8 : id / CPR, p = id % CPR;
        chunk = p ^ (ACROSS ? swz_across<ROWS>(r) : swz_along(r));
        voff = (uint32_t)r * ld * 2 + chunk * 16;
        rows_ld = ld * 2;
        step = (ACROSS ? (int64_t)GK * ld * 2 : GK * 2) * WK;
    }
    // the tile at row r0 (of the result's side) and column k0, of matrices with `rows` rows and K columns
    __device__ __forceinline__ void seek(const void* m0, const void* m1, int r0, int k0, int rows, int K, int wave)
    {
        const OperandSpan at = operand_span(ACROSS, rows_ld / 2, rows, K, r0, k0);
        base0 = static_cast<const char*>(m0) + at.first;
        base1 = GU ? static_cast<const char*>(m1) + at.first : base0;
        if (GU && RPI == 64) base0 = base1 = wave & 4 ? base1 : base0;     // one matrix for all of a wave's loads
        left = at.left;
    }
    // Offsets past the range load zeros: the bytes left, at most 1 GiB (a tile spans half of that at the widest rows the
    // entries take); none without `on`. tail: columns of K left; what lies past them in the last tile along K is moved out
    // of the range.
    __device__ __forceinline__ void load(lds_ptr to, int wave, int tail, bool on)
    {
        const int range = (int)(!on || left < 0 ? 0 : left > 0x40000000 ? 0x40000000 : left);
        uint32_t v0 = voff;
        if (!ACROSS && tail < GK) v0 = chunk * 8 < tail ? v0 : 0x7ff00000u;
#pragma unroll
        for (int j = 0; j < INSTR; ++j)
        {
            const __amdgpu_buffer_rsrc_t r =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(j & 1 ? base1 : base0), 0, range, 0x00020000);
            // rows of one matrix that the loads before have taken
            const uint32_t at = (uint32_t)(GU ? (j * RPI >> 6) * 32 : j * RPI) * rows_ld;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + wave * 1024 + j * NT * 16), 16,
                                                     v0 + at, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void next()
    {
        base0 += step;
        base1 += step;
        left -= step;
    }
};

// 32 result rows from nb, turned over in LDS: turn [32][WROW + 4] of a wave, one of each of WK groups WM * WN * 32 rows apart,
// whose sums belong together. The columns are those of the result from wm0 (EPI_GU: gate and up in turn by 32).
template <class T, int EPI, int WROW, int WK>
__device__ __forceinline__ void store_turned(const GemmArgs& p, const float* turn, int area, int lane, int group, int nb, int wm0, int z,
                                             int prod)
{
    constexpr int LROW = WROW + 4, PIECES = (EPI == EPI_GU ? WROW / 2 : WROW) / 8;   // 8-value pieces of a row
    // four pieces at a time, so that what they read from HBM (g and u) is on its way together
    constexpr int MINE = 32 * PIECES / WK, AHEAD = MINE / 64 < 4 ? MINE / 64 : 4;
    static_assert(MINE % (64 * AHEAD) == 0, "whole steps");
    for (int q0 = group * MINE + lane; q0 < (group + 1) * MINE; q0 += 64 * AHEAD)
    {
        GU<8> saved[EPI == EPI_DGU ? AHEAD : 1];
        if (EPI == EPI_DGU)
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
            {
                const int q = q0 + k * 64, n = nb + q / PIECES, m = wm0 + q % PIECES * 8;
                if (n < p.N && m < p.M) saved[EPI == EPI_DGU ? k : 0] = load_gu<8>(p, (int64_t)n * p.ldo + m);
            }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
        {
            const int q = q0 + k * 64, rr = q / PIECES, c = q % PIECES * 8, n = nb + rr, m = wm0 + c;
            if (n >= p.N || m >= p.M) continue;
            const int64_t o = (int64_t)n * p.ldo + m;
            auto piece = [&](int col) {
                Vals<8> v;
#pragma unroll
                for (int w = 0; w < WK; ++w)
                {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(turn + w * area + rr * LROW + col);
                    const f32x4 b = *reinterpret_cast<const f32x4*>(turn + w * area + rr * LROW + col + 4);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                    {
                        v.v[t] = w ? v.v[t] + a[t] : a[t];
                        v.v[t + 4] = w ? v.v[t + 4] + b[t] : b[t];
                    }
                }
                return v;
            };
            if (EPI == EPI_GU)
            {
                // gate and up rows in turn by 32
                const int col = (c >> 5) * 64 + (c & 31);
                put_gu<T>(p, o, piece(col), piece(col + 32));
            }
            else if (EPI == EPI_PART) store32(p.part + ((int64_t)z * p.N + n) * p.ldp + m, piece(c));
            else if (EPI == EPI_ADD) put_add(p, o, n, piece(c));
            else if (EPI == EPI_DGU) put_dgu<T>(p, o, piece(c), saved[EPI == EPI_DGU ? k : 0]);
            else put<T>(p, p.out[prod], o, m, piece(c));
        }
    }
}

// BM x BN results by WK groups of WM x WN waves, NB buffers of a K tile each. Every group has K tiles of its own (the WK-th
// ones, loaded by itself into its own part of LDS); their sums are added at the end, in the groups' order.
template <int BM, int BN, int WM, int WN, int WK, int NB> constexpr int gemm16_lds()
{
    constexpr int TILES = WK * NB * (BM + BN) * GK * 2, TURN = WM * WN * WK * 32 * (BM / WM + 4) * 4;
    return TILES > TURN ? TILES : TURN;
}

// tile `block` (of p.tm * p.tn) of product or split z; lds_all: gemm16_lds bytes
template <class T, int BM, int BN, int WM, int WN, int WK, int NB, bool AX, bool BX, int EPI>
__device__ __forceinline__ void gemm16_tile(const GemmArgs& p, char* lds_all, int block, int z)
{
    constexpr int NT = WM * WN * 64;                               // threads of a group
    constexpr int MF = BM / WM / 32, NF = BN / WN / 32;            // 32 x 32 fragments of a wave
    constexpr int ABYTES = BM * GK * 2, BBYTES = BN * GK * 2;
    typedef typename Elem<T>::v8 v8;

    const int lane = threadIdx.x & 63, any = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = any / (WM * WN), wave = any % (WM * WN);
    char* lds = lds_all + group * (NB * (ABYTES + BBYTES));
    const int wm = wave / WN, wn = wave % WN;

    // Tiles in an order that keeps an XCD (workgroups are dealt to the 8 XCDs in turn) on neighbouring tiles: each XCD takes
    // one contiguous run, and a run walks N within groups of 8 or 4 tiles of M, so that its L2 holds the rows it shares
    // (without the first, products across K take a sixth longer)
    const int nwg = p.tm * p.tn;
    int id = block;
    {
        const int q = nwg / 8, r = nwg % 8, x = id & 7;
        id = x * q + (x < r ? x : r) + (id >> 3);
    }
    constexpr int GRP = AX ? 4 : 8;                                 // (A across K: dh of 8,192 x 2,048 168 us with 8, 156)
    const int per = GRP * p.tn, g0 = id / per * GRP, gn = min(GRP, p.tm - g0);
    const int tm = g0 + (id % per) % gn, tn = (id % per) / gn;
    const int m0 = EPI == EPI_GU ? tm * (BM / 2) : tm * BM, n0 = tn * BN;
    const int nk1 = (p.K + GK - 1) / GK;                           // K tiles of one product
    int kt = 0, kt_end = nk1 * p.chain;
    const int prod = EPI == EPI_PART ? z / p.splits : z;           // which of the products side by side
    if (EPI == EPI_PART)
    {
        const int q = kt_end / p.splits, r = kt_end % p.splits, sp = z - prod * p.splits;
        kt = sp * q + min(sp, r);
        kt_end = kt + q + (sp < r);
    }

    TileLoader<BM, NT, WK, AX, EPI == EPI_GU> la;
    TileLoader<BN, NT, WK, BX, false> lb;
    la.init(p.lda, wave);
    lb.init(p.ldb, wave);
    int loaded = kt + group;                                       // this group's next tile to load
    bool second = loaded >= nk1;                                   // of a chain
    auto seek = [&](int pi, int k0) {
        la.seek(p.a[pi], p.a[1], p.from + m0, k0, p.from + p.M, p.K, wave);
        lb.seek(p.b[pi], nullptr, n0, k0, p.N, p.K, wave);
    };
    seek(second ? 1 : prod, (second ? loaded - nk1 : loaded) * GK);
    auto tail = [&]() { return p.K - (second ? loaded - nk1 : loaded) * GK; };
    auto load_a = [&](lds_ptr to) {
        if (p.chain > 1 && !second && loaded >= nk1)
        {
            second = true;
            seek(1, (loaded - nk1) * GK);
        }
        la.load(to, wave, tail(), loaded < kt_end);
    };
    auto load_b = [&](lds_ptr to) {
        lb.load(to + ABYTES, wave, tail(), loaded < kt_end);
        la.next();
        lb.next();
        loaded += WK;
    };

    // A fragment (32 rows from row0, 16 of K from ks * 16): lane l holds row l % 32, K (l / 32) * 8 .. + 7
    auto frag = [&](lds_ptr tile, int row0, int ks, bool across, int rows) -> v8 {
        if (!across)
        {
            const int r = row0 + (lane & 31), c = ks * 2 + (lane >> 5);
            return *(__attribute__((address_space(3))) v8*)(tile + r * (GK * 2) + ((c ^ swz_along(r)) << 4));
        }
        s16x8 v;
        const int m = lane & 15, c = (row0 + ((lane >> 4) & 1) * 16 + (m & 3) * 4) >> 3;
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            const int k = ks * 16 + (lane >> 5) * 8 + i * 4 + (m >> 2);
            const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(tile + k * (rows * 2) + ((c ^ (rows == 64 ? swz_across<64>(k) : swz_across<128>(k))) << 4) + (m & 1) * 8));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i * 4 + e] = t[e];
        }
        return __builtin_bit_cast(v8, v);
    };

    f32x16 acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    constexpr int KS = GK / 16;
    v8 a[2][MF], b[2][NF];
    auto read = [&](int set, lds_ptr at, int ks) {
#pragma unroll
        for (int i = 0; i < MF; ++i) a[set][i] = frag(at, wm * (BM / WM) + i * 32, ks, AX, BM);
#pragma unroll
        for (int j = 0; j < NF; ++j) b[set][j] = frag(at + ABYTES, wn * (BN / WN) + j * 32, ks, BX, BN);
    };
    auto products = [&](int set, int from, int to) {
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                if (i >= from && i < to) acc[i][j] = Elem<T>::mfma32(a[set][i], b[set][j], acc[i][j]);
    };
    // NB buffers. At the wait for tile kt + 1 the loads of the NB - 2 tiles behind it stay in flight. (Past the last tile
    // they go on with an empty range, so that the count holds; the results wait for all of them.)
    constexpr int BEHIND = (la.INSTR + lb.INSTR) * (NB - 2);
    static_assert(BEHIND < 64, "vmcnt has 6 bits");
    auto landed = [&]() {
        // this wave's loads up to the tile's are in LDS (vmcnt) and its fragment reads done (lgkmcnt 0), then everyone's. The
        // waits are written out because a workgroup fence would wait for every load; the wavefront fences only keep the
        // compiler from moving LDS accesses across.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_s_waitcnt(0x0070 | (BEHIND & 15) | (BEHIND >> 4) << 14);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    // 256-row tiles: the loads of the next tile go out in two parts, ahead of the products of the first two steps: all at once,
    // or right behind the wait, they hold the products up (286 -> 301 us on 4,096 x 4,096 x 11,008), later they land too late
    // (298 us), and dealt out one by one between the products they stall each of them (274 -> 317 us). The next step's
    // fragments are read between the two halves of a step's products (282 -> 274 us; gate and up of 2,048 x 8,192 x 4,096 222 ->
    // 217). Smaller tiles have fewer products to wait behind: loads right behind the wait (128 rows, 390 -> 342 us on the
    // same). (The branch around the last tile's loads also keeps the compiler from moving them: without it 289 -> 299 us.)
    constexpr bool SPREAD = MF * NF >= 8;
    // the compiler keeps to this order of reads and products, but where a step is only two products (128 x 64; 4,096 -> 4,096
    // for 128 tokens on 128 x 128 50 -> 44 us, dx of 517 x 2,048 on 128 x 64 12.4 -> 11.8 without)
    constexpr bool IN_STEPS = MF * NF >= 4;
    static_assert(!SPREAD || NB == 2, "spread loads end early: only a wait for all of them fits");
    // One tile: its products, but for the last step's, behind the last step's of the tile before. Fragments are read one step
    // of 16 ahead of their products, across tiles too, so that the only wait of all waves for each other (this tile has
    // landed, and the one before is read to the end) has products on both sides.
    // The loads that go out meanwhile fill the buffer of the tile before: `to` is not `at`, and the compiler has to know it.
    // Without __restrict__ it holds every transposing read back until all loads out have landed, those just sent too
    // (2 x 2,048 x 4,096 x 8,192, both operands across K: 246 us, this way 208).
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
    for (int i = 0; i < MF; ++i) a[(KS - 1) & 1][i] = v8{};
#pragma unroll
    for (int j = 0; j < NF; ++j) b[(KS - 1) & 1][j] = v8{};
    int buf = 0, before = NB - 1;
    for (; kt < kt_end; kt += WK)                                  // group 0's tile; the others' may lie past the end: zeros
    {
        landed();
        tile((lds_ptr)lds + buf * BUF, (lds_ptr)lds + before * BUF);
        before = buf;
        buf = buf + 1 == NB ? 0 : buf + 1;
    }
    products((KS - 1) & 1, 0, MF);

    // ---- results ----
    // A lane's accumulators are column n = l % 32 and rows m = (e / 4) * 8 + (l / 32) * 4 + e % 4 of a fragment: four
    // neighbouring values of 32 different result rows. Each wave turns 32 result rows at a time over in its own part of
    // the tiles' LDS (rows padded by 4 floats: 16 lanes at one m fall on different banks), so that what is read and written
    // in HBM is whole 16-byte pieces of whole rows. (Straight from the accumulators, 8 bytes at a time, the gradient
    // epilogue of 8,192 x 2,048 values cost 100 us beside a product of 120; this way about 25.)
    constexpr int WROW = BM / WM, LROW = WROW + 4;                  // a wave's columns m, and an LDS row of them
    constexpr int AREA = WM * WN * 32 * LROW;                       // of a group
    float* turn = reinterpret_cast<float*>(lds_all) + wave * (32 * LROW);
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
                *reinterpret_cast<f32x4*>(turn + group * AREA + (lane & 31) * LROW + i * 32 + e * 2 + (lane >> 5) * 4) =
                    f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
        // one group: the wave's own rows only, its LDS writes and reads are in order
        if (WK > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        store_turned<T, EPI, WROW, WK>(p, turn, AREA, lane, group, nb, wm0, z, prod);
        if (WK > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    }
}

template <class T, int BM, int BN, int WM, int WN, int WK, int NB, bool AX, bool BX, int EPI>
__global__ __launch_bounds__(WM * WN * WK * 64) void gemm16_k(const GemmArgs p)
{
    __shared__ __attribute__((aligned(1024))) char lds[gemm16_lds<BM, BN, WM, WN, WK, NB>()];
    gemm16_tile<T, BM, BN, WM, WN, WK, NB, AX, BX, EPI>(p, lds, blockIdx.x, blockIdx.z);
}

// Two independent products of a backward pass in one grid of 256 x 256 tiles: down's gradient (long sums over the tokens),
// then dh with the activation's gradient behind it. Neither fills the chip in whole rounds by itself, and one's products run
// beside the other's epilogue, which by itself waits for HBM (8,192 tokens' forward and backward of 4096 x 2048 1,104 us,
// in a launch each 1,129).
template <class T>
__global__ __launch_bounds__(512) void gemm16_two_k(const GemmArgs dd, const GemmArgs dh)
{
    __shared__ __attribute__((aligned(1024))) char lds[gemm16_lds<256, 256, 2, 4, 1, 2>()];
    const int first = dd.tm * dd.tn;
    if ((int)blockIdx.x < first) gemm16_tile<T, 256, 256, 2, 4, 1, 2, true, true, EPI_STORE>(dd, lds, blockIdx.x, 0);
    else gemm16_tile<T, 256, 256, 2, 4, 1, 2, true, false, EPI_DGU>(dh, lds, blockIdx.x - first, 0);
}

// The sums over the splits of a product (EPI_PART), in the splits' order, and what EPI does with them. Four values per thread
// and up to 16 splits' loads at a time: the kernel is a few waves, each load round of which waits for HBM once.
template <class T, int EPI>
__global__ __launch_bounds__(64) void gemm_finish_k(const GemmArgs p)
{
    constexpr int W = 4, PRODS = EPI == EPI_GU ? 2 : 1, B = 16 / PRODS;
    const int64_t plane = (int64_t)p.N * p.ldp, at = ((int64_t)blockIdx.x * 64 + threadIdx.x) * W;
    if (at >= plane) return;
    const int n = (int)(at / p.ldp), m = (int)(at % p.ldp);
    const int64_t o = (int64_t)n * p.ldo + m;
    GU<W> saved;
    if (EPI == EPI_DGU) saved = load_gu<W>(p, o);
    Vals<W> sum[PRODS];
#pragma unroll
    for (int k = 0; k < PRODS; ++k)
#pragma unroll
        for (int t = 0; t < W; ++t) sum[k].v[t] = 0.0f;
    for (int s0 = 0; s0 < p.splits; s0 += B)
    {
        Vals<W> part[PRODS][B];
#pragma unroll
        for (int s = 0; s < B; ++s)
#pragma unroll
            for (int k = 0; k < PRODS; ++k)
                if (s0 + s < p.splits) part[k][s] = load32<W>(p.part + (k * p.splits + s0 + s) * plane + at);
#pragma unroll
        for (int s = 0; s < B; ++s)
#pragma unroll
            for (int k = 0; k < PRODS; ++k)
                if (s0 + s < p.splits)
#pragma unroll
                    for (int t = 0; t < W; ++t) sum[k].v[t] += part[k][s].v[t];
    }
    if (EPI == EPI_GU) put_gu<T>(p, o, sum[0], sum[PRODS - 1]);
    else if (EPI == EPI_ADD) put_add(p, o, n, sum[0]);
    else if (EPI == EPI_DGU) put_dgu<T>(p, o, sum[0], saved);
    else put<T>(p, p.out[0], o, m, sum[0]);
}

}  // namespace bmx
