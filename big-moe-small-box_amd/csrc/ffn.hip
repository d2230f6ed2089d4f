// Gated feed-forward block: forward and the form that adds to a layer's output (16-bit and 4-bit weights), gradients (16-bit).
// The products are skinny_k's for few tokens and gemm16_k's for many (4-bit weights: slice_k's and gemm_q4_k's between), planned
// in product_plan.hpp; this file launches gemm16_k, lays out the workspace and checks arguments.
#include <algorithm>

#include "skinny.hpp"

namespace bmx {

// ---- launches -----------------------------------------------------------------------------------------------------------

static bool dtype_ok(int d) { return d == BMX_DT_FP16 || d == BMX_DT_BF16; }

template <class T, bool AX, bool BX, int EPI>
static int run_gemm(const GemmArgs& a, int tile, hipStream_t s)
{
    GemmArgs p = a;
    // EPI_GU: a tile's rows are half gate, half up
    const int bm = EPI == EPI_GU ? TILES[tile].M / 2 : TILES[tile].M;
    p.tm = (a.M + bm - 1) / bm;
    p.tn = (a.N + TILES[tile].N - 1) / TILES[tile].N;
    const dim3 grid((unsigned)(p.tm * p.tn), 1, (unsigned)(EPI == EPI_PART ? a.splits * a.batch : a.batch));
    switch (tile)
    {
        case 0: hipLaunchKernelGGL((gemm16_k<T, 256, 256, 2, 4, 1, 2, AX, BX, EPI>), grid, dim3(512), 0, s, p); break;
        case 1: hipLaunchKernelGGL((gemm16_k<T, 128, 128, 2, 2, 1, 2, AX, BX, EPI>), grid, dim3(256), 0, s, p); break;
        case 2: hipLaunchKernelGGL((gemm16_k<T, 128, 64, 2, 2, 2, 3, AX, BX, EPI>), grid, dim3(512), 0, s, p); break;
        default: hipLaunchKernelGGL((gemm16_k<T, 128, 128, 2, 2, 2, 2, AX, BX, EPI>), grid, dim3(512), 0, s, p);
    }
    return check_launch("gemm16");
}

// One product, split or in two parts or not; EPI: what becomes of the sums
template <class T, bool AX, bool BX, int EPI>
static int product(GemmArgs a, const TilePlan& tp, hipStream_t s)
{
    if (tp.splits == 1)
    {
        ProductPart part[2];
        const int n = product_parts(tp, a.M, EPI == EPI_GU ? 2 : 1, part);
        for (int i = 0; i < n; ++i)
        {
            GemmArgs g = a;
            g.from = part[i].from;
            g.M = part[i].rows;
            for (void*& o : g.out)
                if (o) o = static_cast<char*>(o) + (int64_t)g.from * (EPI == EPI_ADD ? 4 : 2);
            if (g.g) { g.g += g.from; g.u += g.from; }
            if (const int rc = run_gemm<T, AX, BX, EPI>(g, part[i].tile, s)) return rc;
        }
        return BMX_OK;
    }
    a.splits = tp.splits;
    a.ldp = (a.M + 7) / 8 * 8;
    GemmArgs g = a;
    g.batch = EPI == EPI_GU ? 2 : 1;
    if (EPI == EPI_GU) g.b[1] = g.b[0];
    int rc = run_gemm<T, AX, BX, EPI_PART>(g, tp.tile, s);
    if (rc) return rc;
    const int64_t pieces = (int64_t)a.ldp / 4 * a.N;
    hipLaunchKernelGGL((gemm_finish_k<T, EPI>), dim3((unsigned)((pieces + 63) / 64)), dim3(64), 0, s, a);
    return check_launch("gemm_finish");
}

// s_t = sigmoid(x[t] . v): one wave per token, fp32 sums
template <class T>
__global__ __launch_bounds__(256) void row_gate_k(const uint16_t* __restrict__ x, const uint16_t* __restrict__ v, int n, int H,
                                                  float* __restrict__ out)
{
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= n) return;
    float sum = 0.0f;
    for (int k = lane * 8; k < H; k += 512)
    {
        const u32x4 a = ldg4(x + (int64_t)t * H + k), b = ldg4(v + k);
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            sum = __builtin_fmaf(from16<T>((uint16_t)a[i]), from16<T>((uint16_t)b[i]), sum);
            sum = __builtin_fmaf(from16<T>((uint16_t)(a[i] >> 16)), from16<T>((uint16_t)(b[i] >> 16)), sum);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) out[t] = sigmoid_fixed(sum);
}

int launch_product(const GemmArgs& g, int dtype, int epi, hipStream_t s)
{
    const TilePlan p = plan_for(g.M, g.N, g.K, epi == EPI_GU ? 2 : 1);
    const bool h = dtype == BMX_DT_FP16;
    if (epi == EPI_GU) return h ? product<f16, false, false, EPI_GU>(g, p, s) : product<bf16, false, false, EPI_GU>(g, p, s);
    if (epi == EPI_ADD) return h ? product<f16, false, false, EPI_ADD>(g, p, s) : product<bf16, false, false, EPI_ADD>(g, p, s);
    return h ? product<f16, false, false, EPI_STORE>(g, p, s) : product<bf16, false, false, EPI_STORE>(g, p, s);
}

// A forward pass's weights: 16-bit, or q[3] (4-bit)
struct FfnIn {
    int H, I, dtype;
    ActPar act;
    const void* w[3];
    const bmx_q4* q[3];
    int group(int m) const { return q[0] ? q[m]->group : 0; }
    // of the product whose first matrix is m
    bool keep(int m) const { return q[0] && (q4_keep(q[m], dtype) || (m == 0 && q4_keep(q[1], dtype))); }
};

static FfnIn ffn_in(const bmx_ffn_desc* d)
{
    return {d->H, d->I, d->dtype, act_par(d->act, d->act_limit), {d->gate, d->up, d->down}, {nullptr, nullptr, nullptr}};
}

static FfnIn ffn_in(const bmx_ffn4_desc* d)
{
    return {d->gate->K, d->gate->N, d->dtype, act_par(d->act, d->act_limit), {nullptr, nullptr, nullptr}, {d->gate, d->up, d->down}};
}

struct FfnPlan { size_t h, gate, part, total; };       // workspace offsets; part: what the larger of the products needs

static FfnPlan ffn_plan(const FfnIn& d, int T)
{
    FfnPlan p;
    size_t o = 0;
    auto take = [&](size_t b) { const size_t at = o; o += align_up(b, 256); return at; };
    p.h = take((size_t)T * d.I * 2);
    p.gate = take((size_t)T * 4);
    const size_t gu = product_bytes(d.I, d.H, T, 2, d.group(0), d.keep(0)),
                 down = product_bytes(d.H, d.I, T, 1, d.group(2), d.keep(2));
    p.part = take(gu > down ? gu : down);
    p.total = o + 256;
    return p;
}

// One of the block's products on the kernel for its tokens and weights. first: 0 gate and up (EPI_GU), 2 down
static int block_product(const FfnIn& d, const SkinnyArgs& base, int first, int epi, char* part, hipStream_t s)
{
    SkinnyArgs k = base;
    const int n = epi == EPI_GU ? 2 : 1;
    for (int m = 0; m < n; ++m)
    {
        k.w[m] = d.w[first + m];
        if (d.q[0]) k.q[m] = q4_view(d.q[first + m]);
    }
    k.group = d.group(first);
    k.keep = d.keep(first);
    if (product_path(k.N, k.K, k.T, n, k.group, k.keep) != MANY) return launch_skinny(k, d.dtype, epi, reinterpret_cast<float*>(part), s);
    if (k.group) return launch_q4_many(k, d.q + first, d.dtype, epi, part, s);
    GemmArgs a = {};
    a.chain = a.batch = a.splits = 1;
    a.part = reinterpret_cast<float*>(part);
    a.act = k.act; a.scale = k.scale; a.g = k.g; a.u = k.u;
    a.a[0] = k.w[0]; a.a[1] = k.w[1]; a.b[0] = k.x; a.out[0] = k.out;
    a.M = k.N; a.N = k.T; a.K = k.K; a.lda = a.ldb = k.K; a.ldo = k.ldo;
    return launch_product(a, d.dtype, epi, s);
}

template <class T>
static int ffn_forward(const FfnIn& d, const void* x, int n, void* y, float* add, const void* gate_vec, const bmx_ffn_saved* sv,
                       char* ws, hipStream_t s)
{
    const FfnPlan p = ffn_plan(d, n);
    void* h = sv ? sv->h : ws + p.h;
    SkinnyArgs k = {};
    k.T = n;
    k.act = d.act;
    // h = act(x Wg^T, x Wu^T)
    k.x = static_cast<const uint16_t*>(x);
    k.N = k.ldo = d.I; k.K = d.H; k.out = h;
    if (sv) { k.g = sv->g; k.u = sv->u; }
    int rc = block_product(d, k, 0, EPI_GU, ws + p.part, s);
    if (rc) return rc;
    if (gate_vec)
    {
        float* scale = reinterpret_cast<float*>(ws + p.gate);
        hipLaunchKernelGGL((row_gate_k<T>), dim3((n + 3) / 4), dim3(256), 0, s, static_cast<const uint16_t*>(x),
                           static_cast<const uint16_t*>(gate_vec), n, d.H, scale);
        if ((rc = check_launch("row_gate"))) return rc;
        k.scale = scale;
    }
    // y = h Wd^T
    k.x = static_cast<const uint16_t*>(h);
    k.N = k.ldo = d.H; k.K = d.I; k.out = add ? static_cast<void*>(add) : y;
    return block_product(d, k, 2, add ? EPI_ADD : EPI_STORE, ws + p.part, s);
}

struct FfnBackPlan {
    BackTiles t;
    size_t dg, du, part, total;
};

static FfnBackPlan ffn_back_plan(const bmx_ffn_desc* d, int T)
{
    FfnBackPlan p;
    p.t = back_tiles(d->H, d->I, T);
    size_t o = 0;
    auto take = [&](size_t b) { const size_t at = o; o += align_up(b, 256); return at; };
    p.dg = take((size_t)T * d->I * 2);
    p.du = take((size_t)T * d->I * 2);
    const size_t ph = p.t.dh.splits > 1 ? (size_t)p.t.dh.splits * T * d->I * 4 : 0;
    const size_t px = p.t.dx.splits > 1 ? (size_t)p.t.dx.splits * T * d->H * 4 : 0;
    p.part = take(ph > px ? ph : px);
    p.total = o + 256;
    return p;
}

template <class T>
static int ffn_backward(const bmx_ffn_desc* d, const void* x, int n, const bmx_ffn_saved* sv, const void* dy, void* dx,
                        void* dgate, void* dup, void* ddown, char* ws, hipStream_t s)
{
    const FfnBackPlan p = ffn_back_plan(d, n);
    const int H = d->H, I = d->I;
    GemmArgs z = {};
    z.chain = z.batch = z.splits = 1;
    z.part = reinterpret_cast<float*>(ws + p.part);
    z.act = act_par(d->act, d->act_limit);
    int rc = BMX_OK;
    GemmArgs h = z;                                                // dh = dy Wd, then dg, du
    h.a[0] = d->down; h.b[0] = dy; h.out[0] = ws + p.dg; h.out[1] = ws + p.du;
    h.g = sv->g; h.u = sv->u;
    h.M = I; h.N = n; h.K = H; h.lda = I; h.ldb = H; h.ldo = I;
    GemmArgs w = z;                                                // dWd = dy^T h
    w.a[0] = sv->h; w.b[0] = dy; w.out[0] = ddown;
    w.M = I; w.N = H; w.K = n; w.lda = I; w.ldb = H; w.ldo = I;
    const bool need_dh = dx || dgate || dup;
    if (need_dh && ddown && p.t.two)
    {
        h.tm = w.tm = (I + 255) / 256;
        h.tn = (n + 255) / 256;
        w.tn = (H + 255) / 256;
        hipLaunchKernelGGL((gemm16_two_k<T>), dim3((unsigned)(w.tm * w.tn + h.tm * h.tn)), dim3(512), 0, s, w, h);
        rc = check_launch("gemm16_two");
    }
    else
    {
        if (need_dh) rc = product<T, true, false, EPI_DGU>(h, p.t.dh, s);
        if (!rc && ddown) rc = product<T, true, true, EPI_STORE>(w, p.t.dd, s);
    }
    if (!rc && dx)
    {
        GemmArgs a = z;                                            // dx = dg Wg + du Wu
        a.a[0] = d->gate; a.a[1] = d->up; a.b[0] = ws + p.dg; a.b[1] = ws + p.du; a.out[0] = dx;
        a.chain = 2;
        a.M = H; a.N = n; a.K = I; a.lda = H; a.ldb = I; a.ldo = H;
        rc = product<T, true, false, EPI_STORE>(a, p.t.dx, s);
    }
    if (!rc && (dgate || dup))
    {
        GemmArgs a = z;                                            // dWg = dg^T x, dWu = du^T x
        a.batch = dgate && dup ? 2 : 1;
        a.a[0] = a.a[1] = x;
        a.b[0] = dgate ? ws + p.dg : ws + p.du; a.out[0] = dgate ? dgate : dup;
        a.b[1] = ws + p.du; a.out[1] = dup;
        a.M = H; a.N = I; a.K = n; a.lda = H; a.ldb = I; a.ldo = H;
        rc = product<T, true, true, EPI_STORE>(a, p.t.dw, s);
    }
    return rc;
}

// ---- argument checks ----------------------------------------------------------------------------------------------------

static bool odd16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; }

static int check_ffn(const bmx_ffn_desc* d, int T, const char* who)
{
    if (!d) return set_error(BMX_ERR_ARG, "%s: null descriptor", who);
    if (d->H <= 0 || d->I <= 0 || d->H % 8 || d->I % 8 || d->H > (1 << 20) || d->I > (1 << 20))
        return set_error(BMX_ERR_ARG, "%s: H (%d) and I (%d) must be positive multiples of 8, at most 2^20", who, d->H, d->I);
    if (!dtype_ok(d->dtype)) return set_error(BMX_ERR_ARG, "%s: unknown dtype %d", who, d->dtype);
    if (d->act < BMX_ACT_SILU || d->act > BMX_ACT_SILU_OAI) return set_error(BMX_ERR_ARG, "%s: unknown activation %d", who, d->act);
    if (!(d->act_limit >= 0.0f)) return set_error(BMX_ERR_ARG, "%s: act_limit must be 0 (off) or positive", who);
    if (!d->gate || !d->up || !d->down) return set_error(BMX_ERR_ARG, "%s: null weight pointer", who);
    if (odd16(d->gate) || odd16(d->up) || odd16(d->down)) return set_error(BMX_ERR_ARG, "%s: weights must be 16-byte aligned", who);
    // launch sizes: the tiles of a product are one grid dimension
    if (T < 0 || T > (1 << 24)) return set_error(BMX_ERR_ARG, "%s: T (%d) outside [0, 2^24]", who, T);
    return BMX_OK;
}

static int check_ffn(const bmx_ffn4_desc* d, int T, const char* who)
{
    if (!d) return set_error(BMX_ERR_ARG, "%s: null descriptor", who);
    for (const bmx_q4* q : {d->gate, d->up, d->down})
        if (const int rc = check_q4(q, who)) return rc;
    const int H = d->gate->K, I = d->gate->N;
    if (d->up->K != H || d->up->N != I || d->down->K != I || d->down->N != H)
        return set_error(BMX_ERR_ARG, "%s: gate and up must be [I, H], down [H, I]", who);
    if (d->gate->group != d->up->group) return set_error(BMX_ERR_ARG, "%s: gate and up must have groups of one size", who);
    if (!dtype_ok(d->dtype)) return set_error(BMX_ERR_ARG, "%s: unknown dtype %d", who, d->dtype);
    if (d->act < BMX_ACT_SILU || d->act > BMX_ACT_SILU_OAI) return set_error(BMX_ERR_ARG, "%s: unknown activation %d", who, d->act);
    if (!(d->act_limit >= 0.0f)) return set_error(BMX_ERR_ARG, "%s: act_limit must be 0 (off) or positive", who);
    if (T < 0 || T > (1 << 24)) return set_error(BMX_ERR_ARG, "%s: T (%d) outside [0, 2^24]", who, T);
    return BMX_OK;
}

static int check_saved(const bmx_ffn_saved* sv, const char* who)
{
    if (!sv->g || !sv->u || !sv->h || odd16(sv->g) || odd16(sv->u) || odd16(sv->h))
        return set_error(BMX_ERR_ARG, "%s: g, u and h must be 16-byte aligned device arrays", who);
    return BMX_OK;
}

static int check_ws(const void* ws, size_t have, size_t need, const char* who)
{
    if (!ws || odd16(ws)) return set_error(BMX_ERR_ARG, "%s: workspace null or not 16-byte aligned", who);
    if (have < need) return set_error(BMX_ERR_WORKSPACE, "%s: workspace %zu < %zu", who, have, need);
    return BMX_OK;
}

template <class Desc>
static int forward_call(const char* fn, const Desc* desc, const void* x, int T, void* y, const bmx_ffn_saved* saved, void* workspace,
                        size_t workspace_bytes, bmx_stream_t stream)
{
    int rc = check_ffn(desc, T, fn);
    if (rc || T == 0) return rc;
    if (!x || !y || odd16(x) || odd16(y)) return set_error(BMX_ERR_ARG, "%s: x or y null or not 16-byte aligned", fn);
    if (saved && (rc = check_saved(saved, fn))) return rc;
    const FfnIn d = ffn_in(desc);
    if ((rc = check_ws(workspace, workspace_bytes, ffn_plan(d, T).total, fn))) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    return d.dtype == BMX_DT_FP16 ? ffn_forward<f16>(d, x, T, y, nullptr, nullptr, saved, ws, s)
                                  : ffn_forward<bf16>(d, x, T, y, nullptr, nullptr, saved, ws, s);
}

template <class Desc>
static int add_call(const char* fn, const Desc* desc, const void* x, int T, const void* gate_vec, float* out, void* workspace,
                    size_t workspace_bytes, bmx_stream_t stream)
{
    int rc = check_ffn(desc, T, fn);
    if (rc || T == 0) return rc;
    if (!x || !out || odd16(x) || odd16(out)) return set_error(BMX_ERR_ARG, "%s: x or out null or not 16-byte aligned", fn);
    if (odd16(gate_vec)) return set_error(BMX_ERR_ARG, "%s: gate_vec not 16-byte aligned", fn);
    const FfnIn d = ffn_in(desc);
    if ((rc = check_ws(workspace, workspace_bytes, ffn_plan(d, T).total, fn))) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    return d.dtype == BMX_DT_FP16 ? ffn_forward<f16>(d, x, T, nullptr, out, gate_vec, nullptr, ws, s)
                                  : ffn_forward<bf16>(d, x, T, nullptr, out, gate_vec, nullptr, ws, s);
}

__global__ __launch_bounds__(256) void zero16_k(u32x4* p, int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = u32x4{0, 0, 0, 0};
}

}  // namespace bmx

using namespace bmx;

extern "C" {

size_t bmx_ffn_workspace(const bmx_ffn_desc* desc, int T)
{
    return check_ffn(desc, T, "bmx_ffn_workspace") ? 0 : ffn_plan(ffn_in(desc), T).total;
}

size_t bmx_ffn4_workspace(const bmx_ffn4_desc* desc, int T)
{
    return check_ffn(desc, T, "bmx_ffn4_workspace") ? 0 : ffn_plan(ffn_in(desc), T).total;
}

size_t bmx_ffn_backward_workspace(const bmx_ffn_desc* desc, int T)
{
    if (check_ffn(desc, T, "bmx_ffn_backward_workspace")) return 0;
    return ffn_back_plan(desc, T).total;
}

int bmx_ffn_forward(const bmx_ffn_desc* desc, const void* x, int T, void* y, const bmx_ffn_saved* saved, void* workspace,
                    size_t workspace_bytes, bmx_stream_t stream)
{
    return forward_call("bmx_ffn_forward", desc, x, T, y, saved, workspace, workspace_bytes, stream);
}

int bmx_ffn4_forward(const bmx_ffn4_desc* desc, const void* x, int T, void* y, void* workspace, size_t workspace_bytes,
                     bmx_stream_t stream)
{
    return forward_call("bmx_ffn4_forward", desc, x, T, y, nullptr, workspace, workspace_bytes, stream);
}

int bmx_ffn_add(const bmx_ffn_desc* desc, const void* x, int T, const void* gate_vec, float* out, void* workspace,
                size_t workspace_bytes, bmx_stream_t stream)
{
    return add_call("bmx_ffn_add", desc, x, T, gate_vec, out, workspace, workspace_bytes, stream);
}

int bmx_ffn4_add(const bmx_ffn4_desc* desc, const void* x, int T, const void* gate_vec, float* out, void* workspace,
                 size_t workspace_bytes, bmx_stream_t stream)
{
    return add_call("bmx_ffn4_add", desc, x, T, gate_vec, out, workspace, workspace_bytes, stream);
}

int bmx_ffn_backward(const bmx_ffn_desc* desc, const void* x, int T, const bmx_ffn_saved* saved, const void* dy, void* dx,
                     void* dgate, void* dup, void* ddown, void* workspace, size_t workspace_bytes, bmx_stream_t stream)
{
    const char* fn = "bmx_ffn_backward";
    int rc = check_ffn(desc, T, fn);
    if (rc) return rc;
    if (odd16(dx) || odd16(dgate) || odd16(dup) || odd16(ddown)) return set_error(BMX_ERR_ARG, "%s: gradients must be 16-byte aligned", fn);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (T == 0)
    {
        const int64_t n = (int64_t)desc->H * desc->I / 8;
        for (void* w : {dgate, dup, ddown})
            if (w)
            {
                hipLaunchKernelGGL(zero16_k, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, static_cast<u32x4*>(w), n);
                if ((rc = check_launch(fn))) return rc;
            }
        return BMX_OK;
    }
    if (!x || !dy || odd16(x) || odd16(dy)) return set_error(BMX_ERR_ARG, "%s: x or dy null or not 16-byte aligned", fn);
    if (!saved) return set_error(BMX_ERR_ARG, "%s: needs the forward pass's saved values", fn);
    if ((rc = check_saved(saved, fn))) return rc;
    if ((rc = check_ws(workspace, workspace_bytes, ffn_back_plan(desc, T).total, fn))) return rc;
    char* ws = static_cast<char*>(workspace);
    return desc->dtype == BMX_DT_FP16 ? ffn_backward<f16>(desc, x, T, saved, dy, dx, dgate, dup, ddown, ws, s)
                                      : ffn_backward<bf16>(desc, x, T, saved, dy, dx, dgate, dup, ddown, ws, s);
}

}  // extern "C"
