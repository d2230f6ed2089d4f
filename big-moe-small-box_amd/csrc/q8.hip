// 8-bit matrices: decoding, the launches of their products (skinny8_k, gemm8_k, planned in product_plan.hpp), single products and the
// gated feed-forward block on them.
#include <algorithm>

#include "q8_gemm.hpp"

namespace bmx {

static bool odd16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; }
static bool is16(int t) { return t == BMX_DT_FP16 || t == BMX_DT_BF16; }

int check_q8(const bmx_q8* q, const char* who)
{
    if (!q) return set_error(BMX_ERR_ARG, "%s: null matrix", who);
    if (q->N <= 0 || q->N > (1 << 24) || q->K <= 0 || q->K > 131071)
        return set_error(BMX_ERR_ARG, "%s: N (%d) must be in [1, 2^24], K (%d) in [1, 131071]", who, q->N, q->K);
    if (!q->codes || !q->scale) return set_error(BMX_ERR_ARG, "%s: null codes or scale", who);
    if (odd16(q->codes) || reinterpret_cast<uintptr_t>(q->scale) % 4)
        return set_error(BMX_ERR_ARG, "%s: codes must be 16-byte, scale 4-byte aligned", who);
    return BMX_OK;
}

int check_rows8(const bmx_q8* rows, int T, int K, const char* who)
{
    if (T == 0 && rows) return BMX_OK;
    if (const int rc = check_q8(rows, who)) return rc;
    if (rows->N != T || rows->K != K)
        return set_error(BMX_ERR_ARG, "%s: rows must be %d of %d codes, got %d of %d", who, T, K, rows->N, rows->K);
    return BMX_OK;
}

// Piece i of the blocks' 16 codes each: of row n, columns k .. k + 15. A wave has a block: one piece of the codes, 64 columns of 16 rows
struct Piece8 { int64_t n; int k; };
__device__ __forceinline__ Piece8 piece8(int64_t i, int blocks)
{
    const int64_t b = i >> 6;
    const int j = (int)i & 63;
    return {b / blocks * Q8_ROWS + (j & 15), (int)(b % blocks) * Q8_COLS + (j >> 4) * 16};
}

// v = scale code (scale null: the codes themselves); 16 codes a thread, of one row. For checks and conversions, in no model's call: each
// value is a store of its own (4096 x 11008 to fp16 111 us, 1.2 TB/s; the codes 89)
__global__ __launch_bounds__(256) void q8_dequant_k(const int8_t* __restrict__ codes, const float* __restrict__ scale, int N, int K, int type,
                                                    void* __restrict__ out, int64_t pieces)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const Piece8 at = piece8(i, q8_blocks(K));
    const int64_t n = at.n;
    const int k = at.k;
    if (n >= N || k >= K) return;
    const u32x4 c = ldg4(codes + i * 16);
    const float s = scale ? scale[n] : 1.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e)
    {
        const int8_t code = (int8_t)(c[e / 4] >> (8 * (e % 4)));
        const int64_t o = n * K + k + e;
        if (k + e >= K) continue;
        if (!scale) static_cast<int8_t*>(out)[o] = code;
        else if (type == ROW_F32) static_cast<float*>(out)[o] = s * (float)code;
        else static_cast<uint16_t*>(out)[o] = (uint16_t)bits16(type, s * (float)code);
    }
}

// Row-major codes into blocks: 16 a thread, zeros past K
__global__ __launch_bounds__(256) void q8_pack_k(const int8_t* __restrict__ in, int N, int K, bool whole, int8_t* __restrict__ codes,
                                                 int64_t pieces)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const Piece8 at = piece8(i, q8_blocks(K));
    const int64_t n = at.n;
    const int k = at.k;
    if (n >= N) return;
    u32x4 c = {0, 0, 0, 0};
    if (whole)                                                     // rows of whole aligned pieces (54 -> 15 us for 4096 x 11008)
    {
        if (k < K) c = ldg4(in + n * K + k);
    }
    else
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (k + e < K) c[e / 4] |= (uint32_t)(uint8_t)in[n * K + k + e] << (8 * (e % 4));
    *reinterpret_cast<u32x4*>(codes + i * 16) = c;
}

static int q8_whole(const char* fn, const bmx_q8* q, int64_t* pieces)
{
    *pieces = (int64_t)(q8_bytes(q->N, q->K) / 16);
    if (*pieces > (int64_t)1 << 31) return set_error(BMX_ERR_ARG, "%s: %d x %d values are too many for one call", fn, q->N, q->K);
    return BMX_OK;
}

// ---- launches -----------------------------------------------------------------------------------------------------------

template <int IN, int NS, int TT, int RT, int EPI> static int skinny8_launch(const Q8Args& a, hipStream_t s)
{
    constexpr int ROWS = (EPI == EPI_GU ? 8 : 16) * RT;
    hipLaunchKernelGGL((skinny8_k<IN, NS, TT, RT, EPI>), dim3((unsigned)((a.N + ROWS - 1) / ROWS)), dim3(S8_W * 64),
                       IN != IN_CODES ? skinny8_lds(a.T, a.K) : 0, s, a);
    return check_launch("skinny8");
}

template <int TT, int EPI> static int skinny8_codes(const Q8Args& a, hipStream_t s)
{
    if constexpr (TT <= 5)
        if (q8_few_rows(a.N, a.K, a.T, EPI == EPI_GU ? 2 : 1).rt == 2) return skinny8_launch<IN_CODES, 1, TT, 2, EPI>(a, s);
    return skinny8_launch<IN_CODES, 1, TT, 1, EPI>(a, s);
}

// (the workgroups that quantize take 16 rows of W: what they read of the tokens is little)
template <int IN, int EPI> static int skinny8_values(const Q8Args& a, hipStream_t s)
{
    return skinny8_pieces(a.T, a.K) <= S8_W ? skinny8_launch<IN, 1, 1, 1, EPI>(a, s) : skinny8_launch<IN, 4, 1, 1, EPI>(a, s);
}

template <int EPI> static int skinny8_tokens(const Q8Args& a, hipStream_t s)
{
    if (!a.xc)
    {
        // (a block's x has 16 bits, its h 32)
        if constexpr (EPI != EPI_GU)
            if (a.xt == ROW_F32) return skinny8_values<IN_32, EPI>(a, s);
        if constexpr (EPI != EPI_ADD) return skinny8_values<IN_16, EPI>(a, s);
    }
    switch ((a.T + 15) / 16)
    {
        case 1: return skinny8_codes<1, EPI>(a, s);
        case 2: return skinny8_codes<2, EPI>(a, s);
        case 3: return skinny8_codes<3, EPI>(a, s);
        case 4: return skinny8_codes<4, EPI>(a, s);
        case 5: return skinny8_codes<5, EPI>(a, s);
        case 6: return skinny8_codes<6, EPI>(a, s);
        case 7: return skinny8_codes<7, EPI>(a, s);
        default: return skinny8_codes<8, EPI>(a, s);
    }
}

template <int EPI, int OT> static int gemm8_tiles(Q8Args a, int tile, hipStream_t s)
{
    const int bm = EPI == EPI_GU ? TILES8[tile].M / 2 : TILES8[tile].M;
    a.tm = (a.N + bm - 1) / bm;
    a.tn = (a.T + TILES8[tile].N - 1) / TILES8[tile].N;
    const dim3 grid((unsigned)(a.tm * a.tn), 1, (unsigned)(EPI == EPI_PART ? a.splits * (a.w[1] ? 2 : 1) : 1));
    if constexpr (EPI != EPI_PART)
    {
        if (tile == 0)
            hipLaunchKernelGGL((gemm8_big_k<EPI, OT>), dim3(std::min(grid.x, (unsigned)TILES8[0].slots)), dim3(512), 0, s, a);
        else if (tile == 1)
            hipLaunchKernelGGL((gemm8_k<128, 128, 2, 2, 1, 4, EPI, OT>), grid, dim3(256), 0, s, a);
        else if (tile == 2)
            hipLaunchKernelGGL((gemm8_k<128, 64, 2, 2, 2, 4, EPI, OT>), grid, dim3(512), 0, s, a);
        else if (tile == 3)
            hipLaunchKernelGGL((gemm8_k<128, 128, 2, 2, 2, 4, EPI, OT>), grid, dim3(512), 0, s, a);
        else if (tile == 4)
            hipLaunchKernelGGL((gemm8_k<256, 128, 4, 2, 1, 4, EPI, OT>), grid, dim3(512), 0, s, a);
    }
    if (tile == Q8_SPLIT) hipLaunchKernelGGL((gemm8_k<64, 64, 1, 2, 2, 4, EPI, OT>), grid, dim3(256), 0, s, a);
    return check_launch("gemm8");
}

// A product with one matrix (EPI_STORE, EPI_ADD) or two (EPI_GU, a.w[1]); a.part: q8_part_bytes
template <int EPI> static int product8(const Q8Args& base, hipStream_t s)
{
    Q8Args a = base;
    if (q8_few(a.N, a.K, a.T, EPI == EPI_GU ? 2 : 1)) return skinny8_tokens<EPI>(a, s);
    const TilePlan tp = q8_plan(a.N, a.K, a.T, EPI == EPI_GU ? 2 : 1);
    if (tp.splits == 1)
    {
        ProductPart part[2];
        const int n = product_parts(tp, a.N, EPI == EPI_GU ? 2 : 1, part);
        for (int i = 0; i < n; ++i)
        {
            Q8Args g = a;
            g.from = part[i].from;
            g.N = part[i].rows;
            const int rc = EPI != EPI_STORE || a.ot == ROW_F16 ? gemm8_tiles<EPI, ROW_F16>(g, part[i].tile, s)
                                                               : gemm8_tiles<EPI, EPI == EPI_STORE ? ROW_BF16 : ROW_F16>(g, part[i].tile, s);
            if (rc) return rc;
        }
        return BMX_OK;
    }
    a.splits = tp.splits;
    a.ldp = padded(a.N);
    if (const int rc = gemm8_tiles<EPI_PART, ROW_F16>(a, tp.tile, s)) return rc;
    const int64_t pieces = (int64_t)a.ldp / 8 * a.T;
    hipLaunchKernelGGL((finish8_k<EPI>), dim3((unsigned)((pieces + 63) / 64)), dim3(64), 0, s, a);
    return check_launch("finish8");
}

// Tokens of a product: codes already (rows), or to be quantized by the product's workgroups themselves, or into ws first
struct Tokens {
    const void* x;
    int type;
    const bmx_q8* rows;
};

static bool fused8(const Tokens& in, int T, int K) { return !in.rows && skinny8_fused(T, K); }
static size_t rows8_bytes(int T, int K) { return align_up(q8_bytes(T, K), 256) + align_up((size_t)T * 4, 256); }

static int take_tokens(const Tokens& in, int T, int K, char* ws, Q8Args& a, hipStream_t s)
{
    a.T = T;
    a.K = K;
    a.x = nullptr;
    a.xc = nullptr;
    if (fused8(in, T, K))
    {
        a.x = in.x;
        a.xt = in.type;
        return BMX_OK;
    }
    bmx_q8 q = {T, K, ws, reinterpret_cast<float*>(ws + align_up(q8_bytes(T, K), 256))};
    if (in.rows) q = *in.rows;
    a.xc = static_cast<const int8_t*>(q.codes);
    a.sx = q.scale;
    return in.rows ? BMX_OK : launch_quantize(in.x, in.type, &q, s);
}

static void put_matrix(Q8Args& a, int m, const bmx_q8* w)
{
    a.w[m] = static_cast<const int8_t*>(w->codes);
    a.sw[m] = w->scale;
}

static size_t linear8_ws(const bmx_q8* w, int T, bool rows)
{
    const size_t r = rows || skinny8_fused(T, w->K) ? 0 : rows8_bytes(T, w->K), p = q8_part_bytes(w->N, w->K, T, 1);
    return r + p;
}

static int check_ws(const void* ws, size_t have, size_t need, const char* who)
{
    if (need && (!ws || odd16(ws))) return set_error(BMX_ERR_ARG, "%s: workspace null or not 16-byte aligned", who);
    if (have < need) return set_error(BMX_ERR_WORKSPACE, "%s: workspace %zu < %zu", who, have, need);
    return BMX_OK;
}

// ---- the block ----------------------------------------------------------------------------------------------------------

struct Ffn8Plan { size_t h, gate, rows, part, total; };

static Ffn8Plan ffn8_plan(const bmx_ffn8_desc* d, int T)
{
    Ffn8Plan p;
    size_t o = 0;
    auto take = [&](size_t b) { const size_t at = o; o += align_up(b, 256); return at; };
    const int H = d->gate->K, I = d->gate->N;
    p.h = take((size_t)T * I * 4);
    p.gate = take((size_t)T * 4);
    p.rows = take(std::max(rows8_bytes(T, H), rows8_bytes(T, I)));       // x's, then h's
    p.part = take(std::max(q8_part_bytes(I, H, T, 2), q8_part_bytes(H, I, T, 1)));
    p.total = o + 256;
    return p;
}

static int ffn8_call(const bmx_ffn8_desc* d, const void* x, const bmx_q8* rows, int T, void* y, float* add, const void* gate_vec,
                     char* ws, hipStream_t s)
{
    const Ffn8Plan p = ffn8_plan(d, T);
    const int H = d->gate->K, I = d->gate->N;
    Q8Args a = {};
    a.act = act_par(d->act, d->act_limit);
    a.part = reinterpret_cast<int*>(ws + p.part);
    int rc = take_tokens({x, d->dtype, rows}, T, H, ws + p.rows, a, s);
    if (rc) return rc;
    put_matrix(a, 0, d->gate);
    a.w[1] = static_cast<const int8_t*>(d->up->codes);
    a.sw[1] = d->up->scale;
    a.N = a.ldo = I;
    a.out = ws + p.h;
    if ((rc = product8<EPI_GU>(a, s))) return rc;
    if (gate_vec)
    {
        a.scale = reinterpret_cast<float*>(ws + p.gate);
        if ((rc = launch_row_gate(x, gate_vec, d->dtype, T, H, reinterpret_cast<float*>(ws + p.gate), s))) return rc;
    }
    if ((rc = take_tokens({ws + p.h, BMX_DT_FP32, nullptr}, T, I, ws + p.rows, a, s))) return rc;
    put_matrix(a, 0, d->down);
    a.w[1] = nullptr;
    a.N = a.ldo = H;
    a.ot = d->dtype;
    a.out = add ? static_cast<void*>(add) : y;
    return add ? product8<EPI_ADD>(a, s) : product8<EPI_STORE>(a, s);
}

static int check_ffn8(const bmx_ffn8_desc* d, int T, const char* who)
{
    if (!d) return set_error(BMX_ERR_ARG, "%s: null descriptor", who);
    for (const bmx_q8* q : {d->gate, d->up, d->down})
        if (const int rc = check_q8(q, who)) return rc;
    const int H = d->gate->K, I = d->gate->N;
    if (d->up->K != H || d->up->N != I || d->down->K != I || d->down->N != H)
        return set_error(BMX_ERR_ARG, "%s: gate and up must be [I, H], down [H, I]", who);
    if (H % 8 || I % 8) return set_error(BMX_ERR_ARG, "%s: H (%d) and I (%d) must be multiples of 8", who, H, I);
    if (!is16(d->dtype)) return set_error(BMX_ERR_ARG, "%s: unknown dtype %d", who, d->dtype);
    if (d->act < BMX_ACT_SILU || d->act > BMX_ACT_SILU_OAI) return set_error(BMX_ERR_ARG, "%s: unknown activation %d", who, d->act);
    if (!(d->act_limit >= 0.0f)) return set_error(BMX_ERR_ARG, "%s: act_limit must be 0 (off) or positive", who);
    if (T < 0 || T > (1 << 24)) return set_error(BMX_ERR_ARG, "%s: T (%d) outside [0, 2^24]", who, T);
    return BMX_OK;
}

static int ffn8_entry(const char* fn, const bmx_ffn8_desc* d, const void* x, const bmx_q8* rows, int T, void* y, float* add,
                      const void* gate_vec, void* workspace, size_t workspace_bytes, bmx_stream_t stream)
{
    int rc = check_ffn8(d, T, fn);
    if (rc) return rc;
    if (rows && (rc = check_rows8(rows, T, d->gate->K, fn))) return rc;
    if (T == 0) return BMX_OK;
    const void* out = add ? static_cast<const void*>(add) : y;
    if (!out || odd16(out) || odd16(x) || odd16(gate_vec))
        return set_error(BMX_ERR_ARG, "%s: output null, or it, x or gate_vec not 16-byte aligned", fn);
    if (!x && (!rows || gate_vec)) return set_error(BMX_ERR_ARG, "%s: x is null, and needed without rows and for gate_vec", fn);
    if ((rc = check_ws(workspace, workspace_bytes, ffn8_plan(d, T).total, fn))) return rc;
    return ffn8_call(d, x, rows, T, y, add, gate_vec, static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
}

}  // namespace bmx

using namespace bmx;

extern "C" {

int bmx_q8_quantize(const void* x, int dtype, const bmx_q8* out, bmx_stream_t stream)
{
    const char* fn = "bmx_q8_quantize";
    if (const int rc = check_q8(out, fn)) return rc;
    if (!is16(dtype) && dtype != BMX_DT_FP32) return set_error(BMX_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (!x || reinterpret_cast<uintptr_t>(x) % row_type_bytes(dtype)) return set_error(BMX_ERR_ARG, "%s: x null or not aligned", fn);
    return launch_quantize(x, dtype, out, static_cast<hipStream_t>(stream));
}

size_t bmx_q8_code_bytes(int N, int K) { return N <= 0 || K <= 0 ? 0 : q8_bytes(N, K); }

int bmx_q8_pack(const bmx_q8* q, const void* codes, bmx_stream_t stream)
{
    const char* fn = "bmx_q8_pack";
    int64_t pieces = 0;
    if (const int rc = check_q8(q, fn)) return rc;
    if (!codes) return set_error(BMX_ERR_ARG, "%s: codes are null", fn);
    if (const int rc = q8_whole(fn, q, &pieces)) return rc;
    hipLaunchKernelGGL(q8_pack_k, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const int8_t*>(codes), q->N, q->K, q->K % 16 == 0 && !odd16(codes), static_cast<int8_t*>(const_cast<void*>(q->codes)), pieces);
    return check_launch(fn);
}

static int dequant_call(const char* fn, const bmx_q8* q, const float* scale, int dtype, void* out, bmx_stream_t stream)
{
    int64_t pieces = 0;
    if (const int rc = q8_whole(fn, q, &pieces)) return rc;
    hipLaunchKernelGGL(q8_dequant_k, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const int8_t*>(q->codes), scale, q->N, q->K, dtype, out, pieces);
    return check_launch(fn);
}

int bmx_q8_unpack(const bmx_q8* q, void* codes, bmx_stream_t stream)
{
    const char* fn = "bmx_q8_unpack";
    if (const int rc = check_q8(q, fn)) return rc;
    if (!codes) return set_error(BMX_ERR_ARG, "%s: codes are null", fn);
    return dequant_call(fn, q, nullptr, 0, codes, stream);
}

int bmx_q8_dequant(const bmx_q8* q, int dtype, void* out, bmx_stream_t stream)
{
    const char* fn = "bmx_q8_dequant";
    if (const int rc = check_q8(q, fn)) return rc;
    if (!is16(dtype) && dtype != BMX_DT_FP32) return set_error(BMX_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (!out || odd16(out)) return set_error(BMX_ERR_ARG, "%s: out null or not 16-byte aligned", fn);
    return dequant_call(fn, q, q->scale, dtype, out, stream);
}

size_t bmx_q8_linear_workspace(const bmx_q8* w, int T)
{
    if (check_q8(w, "bmx_q8_linear_workspace") || T < 0 || T > (1 << 24)) return 0;
    return linear8_ws(w, T, false);
}

int bmx_q8_linear(const bmx_q8* w, int dtype, const void* x, const bmx_q8* rows, int T, void* y, void* workspace,
                  size_t workspace_bytes, bmx_stream_t stream)
{
    const char* fn = "bmx_q8_linear";
    int rc = check_q8(w, fn);
    if (rc) return rc;
    if (!is16(dtype)) return set_error(BMX_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (T < 0 || T > (1 << 24)) return set_error(BMX_ERR_ARG, "%s: T (%d) outside [0, 2^24]", fn, T);
    if (rows && (rc = check_rows8(rows, T, w->K, fn))) return rc;
    if (T == 0) return BMX_OK;
    if (!x == !rows) return set_error(BMX_ERR_ARG, "%s: x or rows, one of them", fn);
    if (!y || odd16(y) || odd16(x)) return set_error(BMX_ERR_ARG, "%s: y null, or x or y not 16-byte aligned", fn);
    if ((rc = check_ws(workspace, workspace_bytes, linear8_ws(w, T, rows), fn))) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    Q8Args a = {};
    if ((rc = take_tokens({x, dtype, rows}, T, w->K, ws, a, s))) return rc;
    put_matrix(a, 0, w);
    a.N = a.ldo = w->N;
    a.out = y;
    a.ot = dtype;
    a.part = reinterpret_cast<int*>(ws + (a.xc && !rows ? rows8_bytes(T, w->K) : 0));
    return product8<EPI_STORE>(a, s);
}

size_t bmx_ffn8_workspace(const bmx_ffn8_desc* desc, int T)
{
    return check_ffn8(desc, T, "bmx_ffn8_workspace") ? 0 : ffn8_plan(desc, T).total;
}

int bmx_ffn8_forward(const bmx_ffn8_desc* desc, const void* x, const bmx_q8* rows, int T, void* y, void* workspace,
                     size_t workspace_bytes, bmx_stream_t stream)
{
    return ffn8_entry("bmx_ffn8_forward", desc, x, rows, T, y, nullptr, nullptr, workspace, workspace_bytes, stream);
}

int bmx_ffn8_add(const bmx_ffn8_desc* desc, const void* x, const bmx_q8* rows, int T, const void* gate_vec, float* out,
                 void* workspace, size_t workspace_bytes, bmx_stream_t stream)
{
    const char* fn = "bmx_ffn8_add";
    if (T > 0 && !out) return set_error(BMX_ERR_ARG, "%s: out is null", fn);
    return ffn8_entry(fn, desc, x, rows, T, nullptr, out, gate_vec, workspace, workspace_bytes, stream);
}

}  // extern "C"
