// 4-bit matrices with group scales: packing into fragment order, decoding to 16 bits, and the launches of their products (skinny_k,
// slice_k, gemm_q4_k, gemm16_k behind a decoding); skinny_k also for 16-bit weights.
#include <algorithm>

#include "q4_gemm.hpp"

namespace bmx {

// ---- packing and decoding -----------------------------------------------------------------------------------------------

// Packing: a thread takes every PACK_BLOCKS * 256-th value, since a launch has to stay below 2^32 threads and a matrix of 2^20 rows
// has more words
constexpr int PACK_BLOCKS = 1 << 20;

// Checkpoint codes [N][K / 2] (the even column in a byte's low half) -> fragment order; one word (8 codes) at a time
__global__ __launch_bounds__(256) void q4_pack_codes_k(const uint8_t* __restrict__ in, int N, int K, uint32_t* __restrict__ out,
                                                       int64_t words)
{
    const int KT = (K + SK_K - 1) / SK_K;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256)
    {
        const int j = (int)(i & 3), lane = (int)(i >> 2) & 63;
        const int64_t tile = i >> 8;
        const int n = (int)(tile / KT) * 16 + (lane & 15), k = (int)(tile % KT) * SK_K + j * 32 + (lane >> 4) * 8;
        uint32_t w = 0;
        if (n < N && k < K)
        {
            const uint8_t* b = in + (int64_t)n * (K / 2) + k / 2;
#pragma unroll
            for (int p = 0; p < 4; ++p) w |= (uint32_t)(b[p] & 15) << (4 * p) | (uint32_t)(b[p] >> 4) << (4 * p + 16);
        }
        out[i] = w;
    }
}

// Scales and zero points [N][K / group] -> [tile of 16 rows][group][16]; outside the matrix scale 0
__global__ __launch_bounds__(256) void q4_pack_scales_k(const uint16_t* __restrict__ scale, const uint8_t* __restrict__ zero, int N,
                                                        int groups, int padded, uint16_t* __restrict__ so, uint8_t* __restrict__ zo,
                                                        int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    {
        const int64_t row = i / 16 / padded * 16 + (i & 15);
        const int g = (int)(i / 16 % padded);
        const bool in = row < N && g < groups;
        so[i] = in ? scale[row * groups + g] : 0;
        if (zo) zo[i] = in ? zero[row * groups + g] : 0;
    }
}

// w = scale (code - zero), exact in fp32 (5 and 11 bits), rounded once to 16 bits; one lane's 32 codes per thread
template <class T>
__global__ __launch_bounds__(256) void q4_dequant_k(const Q4View q, int N, int K, int group, uint16_t* __restrict__ out,
                                                    int64_t lanes)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= lanes) return;
    const int KT = (K + SK_K - 1) / SK_K, lane = (int)i & 63;
    const int64_t tile = i >> 6, nt = tile / KT;
    const int64_t n = nt * 16 + (lane & 15);
    const int kt = (int)(tile % KT), per = SK_K / group;
    if (n >= N) return;
    const u32x4 c = ldg4(q.codes + i);
#pragma unroll
    for (int j = 0; j < 4; ++j)
    {
        const int k = kt * SK_K + j * 32 + (lane >> 4) * 8;
        if (k >= K) return;
        const int64_t at = (nt * KT * per + k / group) * 16 + (lane & 15);
        const float s = q.scale_bf16 ? from16<bf16>(q.scale[at]) : from16<f16>(q.scale[at]);
        const float z = q.zero ? (float)q.zero[at] : 8.0f;
        u32x4 w;
#pragma unroll
        for (int p = 0; p < 4; ++p)
            w[p] = (uint32_t)to16<T>(s * ((float)(c[j] >> (4 * p) & 15) - z)) |
                   (uint32_t)to16<T>(s * ((float)(c[j] >> (4 * p + 16) & 15) - z)) << 16;
        *reinterpret_cast<u32x4*>(out + n * K + k) = w;
    }
}

static int64_t ceil_to(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

int check_q4(const bmx_q4* q, const char* who)
{
    if (!q) return set_error(BMX_ERR_ARG, "%s: null matrix", who);
    if (q->group != 32 && q->group != 64 && q->group != 128)
        return set_error(BMX_ERR_ARG, "%s: group (%d) must be 32, 64 or 128", who, q->group);
    if (q->N <= 0 || q->K <= 0 || q->K % q->group || q->N > (1 << 20) || q->K > (1 << 20))
        return set_error(BMX_ERR_ARG, "%s: N (%d) and K (%d) must be positive, at most 2^20, K a multiple of the group (%d)", who,
                         q->N, q->K, q->group);
    if (q->scale_dtype != BMX_DT_FP16 && q->scale_dtype != BMX_DT_BF16)
        return set_error(BMX_ERR_ARG, "%s: unknown scale dtype %d", who, q->scale_dtype);
    if (!q->codes || !q->scale) return set_error(BMX_ERR_ARG, "%s: null codes or scale", who);
    if (reinterpret_cast<uintptr_t>(q->codes) % 16 || reinterpret_cast<uintptr_t>(q->scale) % 16 ||
        reinterpret_cast<uintptr_t>(q->zero) % 16)
        return set_error(BMX_ERR_ARG, "%s: codes, scale and zero must be 16-byte aligned", who);
    return BMX_OK;
}

Q4View q4_view(const bmx_q4* q)
{
    return {static_cast<const u32x4*>(q->codes), static_cast<const uint16_t*>(q->scale), static_cast<const uint8_t*>(q->zero),
            q->scale_dtype == BMX_DT_BF16};
}

int launch_q4_dequant(const bmx_q4* q, int dtype, void* out, hipStream_t s)
{
    const int64_t lanes = ceil_to(q->N, 16) / 16 * (ceil_to(q->K, SK_K) / SK_K) * 64;
    const dim3 grid((unsigned)((lanes + 255) / 256));
    if (dtype == BMX_DT_FP16)
        hipLaunchKernelGGL((q4_dequant_k<f16>), grid, dim3(256), 0, s, q4_view(q), q->N, q->K, q->group, static_cast<uint16_t*>(out), lanes);
    else
        hipLaunchKernelGGL((q4_dequant_k<bf16>), grid, dim3(256), 0, s, q4_view(q), q->N, q->K, q->group, static_cast<uint16_t*>(out), lanes);
    return check_launch("q4_dequant");
}

// ---- products of few tokens ---------------------------------------------------------------------------------------------

template <class T, int TT, int G> static int slice_launch(const SliceArgs& a, dim3 grid, hipStream_t s)
{
    hipLaunchKernelGGL((slice_k<T, TT, G>), grid, dim3(SL_W<TT> * 64), 0, s, a);
    return check_launch("slice");
}

template <class T, int G> static int slice_tokens(const SliceArgs& a, dim3 grid, hipStream_t s)
{
    switch ((a.a.T + 15) / 16)
    {
        case 2: return slice_launch<T, 2, G>(a, grid, s);
        case 3: return slice_launch<T, 3, G>(a, grid, s);
        case 4: return slice_launch<T, 4, G>(a, grid, s);
        default: return slice_launch<T, 5, G>(a, grid, s);
    }
}

template <class T, int EPI> static int slice_product(const SkinnyArgs& k, float* part, hipStream_t s)
{
    SliceArgs a;
    a.a = k;
    a.products = EPI == EPI_GU ? 2 : 1;
    a.slices = slices_of(k.K);
    a.ldp = padded(k.N);
    a.tiles = (k.N + 15) / 16 * a.products;
    a.part = part;
    // up to 768 workgroups of 4 waves or 512 of 8 (what the compute units hold at 48 and 64 tokens), of at least a tile per wave
    const int waves = k.T <= 48 ? SL_W<3> : SL_W<4>, most = k.T <= 48 ? 768 : 512;
    const int blocks = most / a.slices > 0 ? most / a.slices : 1;
    a.per = ((a.tiles + blocks - 1) / blocks + waves - 1) / waves * waves;
    const dim3 grid((unsigned)((a.tiles + a.per - 1) / a.per), (unsigned)a.slices);
    int rc;
    switch (k.group)
    {
        case 32: rc = slice_tokens<T, 32>(a, grid, s); break;
        case 64: rc = slice_tokens<T, 64>(a, grid, s); break;
        default: rc = slice_tokens<T, 128>(a, grid, s);
    }
    if (rc) return rc;
    GemmArgs g = {};
    g.M = k.N; g.N = k.T; g.ldp = a.ldp; g.splits = a.slices; g.part = part;
    g.out[0] = k.out; g.ldo = k.ldo; g.scale = k.scale; g.act = k.act; g.g = k.g; g.u = k.u;
    const int64_t pieces = (int64_t)a.ldp / 4 * k.T;
    hipLaunchKernelGGL((gemm_finish_k<T, EPI>), dim3((unsigned)((pieces + 63) / 64)), dim3(64), 0, s, g);
    return check_launch("gemm_finish");
}

template <class T, int RT, int G, int EPI, bool XL> static int direct_rows(const SkinnyArgs& a, hipStream_t s)
{
    constexpr int ROWS = (EPI == EPI_GU ? 8 : 16) * RT;
    constexpr int D = RT == 4 && G == 32 ? 1 : 2;                  // (two steps of four tiles and 16 groups spill)
    const int64_t rows = (a.N + ROWS - 1) / ROWS, blocks = a.T <= 16 ? rows : (rows + 7) / 8 * 8 * ((a.T + 15) / 16);
    hipLaunchKernelGGL((skinny_k<T, RT, G, D, EPI, XL>), dim3((unsigned)blocks), dim3(SK_W * 64),
                       XL ? (size_t)a.T * (a.K * 2 + 16) : 0, s, a);
    return check_launch("skinny");
}

template <class T, int G, int EPI> static int direct_launch(const SkinnyArgs& a, hipStream_t s)
{
    const FewForm f = few_form(a.N, a.K, a.T, EPI == EPI_GU ? 2 : 1, G);
    if constexpr (G != 0)
    {
        if (f.xl) return direct_rows<T, 1, G, EPI, true>(a, s);
        if (f.rt == 4) return direct_rows<T, 4, G, EPI, false>(a, s);
    }
    return f.rt == 2 ? direct_rows<T, 2, G, EPI, false>(a, s) : direct_rows<T, 1, G, EPI, false>(a, s);
}

template <class T, int EPI> static int few_tokens(const SkinnyArgs& a, float* part, hipStream_t s)
{
    if (a.T > 16 && product_path(a.N, a.K, a.T, EPI == EPI_GU ? 2 : 1, a.group, a.keep) == FEW_SLICES) return slice_product<T, EPI>(a, part, s);
    switch (a.group)
    {
        case 0: return direct_launch<T, 0, EPI>(a, s);
        case 32: return direct_launch<T, 32, EPI>(a, s);
        case 64: return direct_launch<T, 64, EPI>(a, s);
        default: return direct_launch<T, 128, EPI>(a, s);
    }
}

int launch_skinny(const SkinnyArgs& a, int dtype, int epi, float* part, hipStream_t s)
{
    const bool h = dtype == BMX_DT_FP16;
    if (epi == EPI_GU) return h ? few_tokens<f16, EPI_GU>(a, part, s) : few_tokens<bf16, EPI_GU>(a, part, s);
    if (epi == EPI_ADD) return h ? few_tokens<f16, EPI_ADD>(a, part, s) : few_tokens<bf16, EPI_ADD>(a, part, s);
    return h ? few_tokens<f16, EPI_STORE>(a, part, s) : few_tokens<bf16, EPI_STORE>(a, part, s);
}

// ---- products of many tokens ----------------------------------------------------------------------------------------------

template <class T, int G, int EPI> static int gemm_q4_launch(Q4GemmArgs a, int splits, hipStream_t s)
{
    constexpr int PRODS = EPI == EPI_GU ? 2 : 1;
    if (Q4Dec<T>::OFFSET)
    {
        const int64_t n = (int64_t)a.g.N * (ceil_to(a.g.K, SK_K) / 8);
        hipLaunchKernelGGL((group_sums_k<T, G>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a.x, a.g.N, a.g.K,
                           const_cast<float*>(a.xs), a.xs_ld);
        const int rc = check_launch("group_sums");
        if (rc) return rc;
    }
    a.g.tn = (a.g.N + QG_T - 1) / QG_T;
    a.g.splits = splits;
    if (splits == 1)
    {
        const int rows = EPI == EPI_GU ? QG_N / 2 : QG_N;
        a.g.tm = (a.g.M + rows - 1) / rows;
        hipLaunchKernelGGL((gemm_q4_k<T, G, EPI>), dim3((unsigned)(a.g.tm * a.g.tn)), dim3(256), 0, s, a);
        return check_launch("gemm_q4");
    }
    a.g.tm = (a.g.M + QG_N - 1) / QG_N;
    hipLaunchKernelGGL((gemm_q4_k<T, G, EPI_PART>), dim3((unsigned)(a.g.tm * a.g.tn), 1, (unsigned)(splits * PRODS)), dim3(256), 0, s, a);
    const int rc = check_launch("gemm_q4");
    if (rc) return rc;
    const int64_t pieces = (int64_t)a.g.ldp / 4 * a.g.N;
    hipLaunchKernelGGL((gemm_finish_k<T, EPI>), dim3((unsigned)((pieces + 63) / 64)), dim3(64), 0, s, a.g);
    return check_launch("gemm_finish");
}

template <class T, int EPI> static int q4_many(const SkinnyArgs& k, const bmx_q4* const* q, int dtype, char* ws, hipStream_t s)
{
    constexpr int PRODS = EPI == EPI_GU ? 2 : 1;
    const Q4Plan plan = q4_plan(k.N, k.K, k.T, PRODS, k.group, k.keep);
    Q4GemmArgs a = {};
    a.g.chain = a.g.batch = a.g.splits = 1;
    a.g.M = k.N; a.g.N = k.T; a.g.K = k.K; a.g.ldo = k.ldo; a.g.ldp = padded(k.N);
    a.g.out[0] = k.out; a.g.scale = k.scale; a.g.act = k.act;
    if (!plan.direct)
    {
        const size_t one = (size_t)k.N * k.K * 2;
        for (int m = 0; m < PRODS; ++m)
            if (const int rc = launch_q4_dequant(q[m], dtype, ws + m * one, s)) return rc;
        a.g.a[0] = ws; a.g.a[1] = ws + one; a.g.b[0] = k.x;
        a.g.lda = a.g.ldb = k.K;
        a.g.part = reinterpret_cast<float*>(ws + align_up(PRODS * one, 256));
        return launch_product(a.g, dtype, EPI, s);
    }
    a.q[0] = k.q[0]; a.q[1] = k.q[1];
    a.x = k.x;
    a.xs = reinterpret_cast<float*>(ws);
    a.xs_ld = (int)ceil_to(k.T, QG_T);
    a.g.part = reinterpret_cast<float*>(ws + group_sums_bytes(k.K, k.T, k.group));
    switch (k.group)
    {
        case 32: return gemm_q4_launch<T, 32, EPI>(a, plan.splits, s);
        case 64: return gemm_q4_launch<T, 64, EPI>(a, plan.splits, s);
        default: return gemm_q4_launch<T, 128, EPI>(a, plan.splits, s);
    }
}

int launch_q4_many(const SkinnyArgs& k, const bmx_q4* const* q, int dtype, int epi, char* ws, hipStream_t s)
{
    const bool h = dtype == BMX_DT_FP16;
    if (epi == EPI_GU) return h ? q4_many<f16, EPI_GU>(k, q, dtype, ws, s) : q4_many<bf16, EPI_GU>(k, q, dtype, ws, s);
    if (epi == EPI_ADD) return h ? q4_many<f16, EPI_ADD>(k, q, dtype, ws, s) : q4_many<bf16, EPI_ADD>(k, q, dtype, ws, s);
    return h ? q4_many<f16, EPI_STORE>(k, q, dtype, ws, s) : q4_many<bf16, EPI_STORE>(k, q, dtype, ws, s);
}

// ---- y = x W^T ----------------------------------------------------------------------------------------------------------

static size_t q4_linear_ws(const bmx_q4* q, int T, bool keep) { return product_bytes(q->N, q->K, T, 1, q->group, keep); }

}  // namespace bmx

using namespace bmx;

extern "C" {

size_t bmx_q4_code_bytes(int N, int K)
{
    return N <= 0 || K <= 0 ? 0 : (size_t)ceil_to(N, 16) * ceil_to(K, SK_K) / 2;
}

size_t bmx_q4_group_count(int N, int K, int group)
{
    return N <= 0 || K <= 0 || (group != 32 && group != 64 && group != 128) ? 0 : (size_t)ceil_to(N, 16) * (ceil_to(K, SK_K) / group);
}

int bmx_q4_pack(const bmx_q4* q, const void* codes, const void* scale, const void* zero, bmx_stream_t stream)
{
    const char* fn = "bmx_q4_pack";
    int rc = check_q4(q, fn);
    if (rc) return rc;
    if (!codes || !scale || !zero != !q->zero) return set_error(BMX_ERR_ARG, "%s: null pointer, or zero points on one side only", fn);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t words = (int64_t)bmx_q4_code_bytes(q->N, q->K) / 4, n = (int64_t)bmx_q4_group_count(q->N, q->K, q->group);
    const auto blocks = [](int64_t v) { return dim3((unsigned)std::min<int64_t>((v + 255) / 256, PACK_BLOCKS)); };
    hipLaunchKernelGGL(q4_pack_codes_k, blocks(words), dim3(256), 0, s, static_cast<const uint8_t*>(codes),
                       q->N, q->K, static_cast<uint32_t*>(const_cast<void*>(q->codes)), words);
    if ((rc = check_launch(fn))) return rc;
    hipLaunchKernelGGL(q4_pack_scales_k, blocks(n), dim3(256), 0, s, static_cast<const uint16_t*>(scale),
                       static_cast<const uint8_t*>(zero), q->N, q->K / q->group, (int)(ceil_to(q->K, SK_K) / q->group),
                       static_cast<uint16_t*>(const_cast<void*>(q->scale)), static_cast<uint8_t*>(const_cast<void*>(q->zero)), n);
    return check_launch(fn);
}

int bmx_q4_dequant(const bmx_q4* q, int dtype, void* out, bmx_stream_t stream)
{
    const int rc = check_q4(q, "bmx_q4_dequant");
    if (rc) return rc;
    if (dtype != BMX_DT_FP16 && dtype != BMX_DT_BF16) return set_error(BMX_ERR_ARG, "bmx_q4_dequant: unknown dtype %d", dtype);
    if (!out || reinterpret_cast<uintptr_t>(out) % 16) return set_error(BMX_ERR_ARG, "bmx_q4_dequant: out null or not 16-byte aligned");
    return launch_q4_dequant(q, dtype, out, static_cast<hipStream_t>(stream));
}

size_t bmx_q4_linear_workspace(const bmx_q4* q, int T)
{
    if (check_q4(q, "bmx_q4_linear_workspace") || T < 0 || T > (1 << 24)) return 0;
    // of either type of x
    return std::max(q4_linear_ws(q, T, q4_keep(q, BMX_DT_FP16)), q4_linear_ws(q, T, q4_keep(q, BMX_DT_BF16)));
}

int bmx_q4_linear(const bmx_q4* q, int dtype, const void* x, int T, void* y, void* workspace, size_t workspace_bytes,
                  bmx_stream_t stream)
{
    const char* fn = "bmx_q4_linear";
    int rc = check_q4(q, fn);
    if (rc) return rc;
    if (dtype != BMX_DT_FP16 && dtype != BMX_DT_BF16) return set_error(BMX_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (T < 0 || T > (1 << 24)) return set_error(BMX_ERR_ARG, "%s: T (%d) outside [0, 2^24]", fn, T);
    if (T == 0) return BMX_OK;
    if (!x || !y || reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(y) % 16)
        return set_error(BMX_ERR_ARG, "%s: x or y null or not 16-byte aligned", fn);
    const bool keep = q4_keep(q, dtype);
    const size_t need = q4_linear_ws(q, T, keep);
    if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
        return set_error(BMX_ERR_ARG, "%s: workspace null or not 16-byte aligned", fn);
    if (workspace_bytes < need) return set_error(BMX_ERR_WORKSPACE, "%s: workspace %zu < %zu", fn, workspace_bytes, need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    SkinnyArgs a = {};
    a.q[0] = q4_view(q);
    a.x = static_cast<const uint16_t*>(x);
    a.T = T; a.N = q->N; a.K = q->K; a.group = q->group; a.keep = keep;
    a.out = y; a.ldo = q->N;
    if (product_path(q->N, q->K, T, 1, q->group, keep) == MANY) return launch_q4_many(a, &q, dtype, EPI_STORE, static_cast<char*>(workspace), s);
    return launch_skinny(a, dtype, EPI_STORE, static_cast<float*>(workspace), s);
}

}  // extern "C"
