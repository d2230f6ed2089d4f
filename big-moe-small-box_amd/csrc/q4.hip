// 4-bit matrices with group scales: packing into fragment order, decoding to 16 bits, and products of few tokens (skinny_k).
#include "skinny.hpp"

namespace bmx {

// ---- packing and decoding -----------------------------------------------------------------------------------------------

// Checkpoint codes [N][K / 2] (the even column in a byte's low half) -> fragment order; one word (8 codes) per thread
__global__ __launch_bounds__(256) void q4_pack_codes_k(const uint8_t* __restrict__ in, int N, int K, uint32_t* __restrict__ out,
                                                       int64_t words)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= words) return;
    const int KT = (K + SK_K - 1) / SK_K;
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

// Scales and zero points [N][K / group] -> [tile of 16 rows][group][16]; outside the matrix scale 0
__global__ __launch_bounds__(256) void q4_pack_scales_k(const uint16_t* __restrict__ scale, const uint8_t* __restrict__ zero, int N,
                                                        int groups, int padded, uint16_t* __restrict__ so, uint8_t* __restrict__ zo,
                                                        int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t row = i / 16 / padded * 16 + (i & 15);
    const int g = (int)(i / 16 % padded);
    const bool in = row < N && g < groups;
    so[i] = in ? scale[row * groups + g] : 0;
    if (zo) zo[i] = in ? zero[row * groups + g] : 0;
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

template <class T, int NM, int TT, int G, int EPI> static int skinny_launch(const SkinnyArgs& a, hipStream_t s)
{
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.T + TT * 16 - 1) / (TT * 16)));
    hipLaunchKernelGGL((skinny_k<T, NM, 1, TT, G, EPI>), grid, dim3(SK_W * 64), 0, s, a);
    return check_launch("skinny");
}

template <class T, int NM, int G, int EPI> static int skinny_tokens(const SkinnyArgs& a, hipStream_t s)
{
    if (a.T <= 16) return skinny_launch<T, NM, 1, G, EPI>(a, s);
    if (a.T <= 32) return skinny_launch<T, NM, 2, G, EPI>(a, s);
    return skinny_launch<T, NM, 4, G, EPI>(a, s);
}

template <class T, int NM, int EPI> static int skinny_group(const SkinnyArgs& a, hipStream_t s)
{
    switch (a.group)
    {
        case 0: return skinny_tokens<T, NM, 0, EPI>(a, s);
        case 32: return skinny_tokens<T, NM, 32, EPI>(a, s);
        case 64: return skinny_tokens<T, NM, 64, EPI>(a, s);
        default: return skinny_tokens<T, NM, 128, EPI>(a, s);
    }
}

int skinny_tokens_max(int group) { return 64; }

int launch_skinny(const SkinnyArgs& a, int dtype, int epi, hipStream_t s)
{
    const bool h = dtype == BMX_DT_FP16;
    if (epi == EPI_GU) return h ? skinny_group<f16, 2, EPI_GU>(a, s) : skinny_group<bf16, 2, EPI_GU>(a, s);
    if (epi == EPI_ADD) return h ? skinny_group<f16, 1, EPI_ADD>(a, s) : skinny_group<bf16, 1, EPI_ADD>(a, s);
    return h ? skinny_group<f16, 1, EPI_STORE>(a, s) : skinny_group<bf16, 1, EPI_STORE>(a, s);
}

// ---- y = x W^T ----------------------------------------------------------------------------------------------------------

static size_t q4_linear_ws(const bmx_q4* q, int T)
{
    return skinny_tokens_max(q->group) >= T ? 0 : align_up((size_t)q->N * q->K * 2, 256) + product_part_bytes(q->N, T, q->K);
}

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
    hipLaunchKernelGGL(q4_pack_codes_k, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, s, static_cast<const uint8_t*>(codes),
                       q->N, q->K, static_cast<uint32_t*>(const_cast<void*>(q->codes)), words);
    if ((rc = check_launch(fn))) return rc;
    hipLaunchKernelGGL(q4_pack_scales_k, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, static_cast<const uint16_t*>(scale),
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
    return q4_linear_ws(q, T);
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
    const size_t need = q4_linear_ws(q, T);
    if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
        return set_error(BMX_ERR_ARG, "%s: workspace null or not 16-byte aligned", fn);
    if (workspace_bytes < need) return set_error(BMX_ERR_WORKSPACE, "%s: workspace %zu < %zu", fn, workspace_bytes, need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (need)
    {
        // many tokens: the weights once to 16 bits, then the tiled product
        if ((rc = launch_q4_dequant(q, dtype, workspace, s))) return rc;
        return launch_product(workspace, x, T, q->N, q->K, dtype, y, static_cast<char*>(workspace) + align_up((size_t)q->N * q->K * 2, 256), s);
    }
    SkinnyArgs a = {};
    a.q[0] = q4_view(q);
    a.x = static_cast<const uint16_t*>(x);
    a.T = T; a.N = q->N; a.K = q->K; a.group = q->group;
    a.out = y; a.ldo = q->N;
    return launch_skinny(a, dtype, EPI_STORE, s);
}

}  // extern "C"
