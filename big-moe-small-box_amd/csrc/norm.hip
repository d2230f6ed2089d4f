// Root-mean-square norm with the residual's addition: forward into 16 bits, 8-bit rows or both, and its gradients. With
//   s = x + residual (fp32), r = s rounded to the stream's type, v = r (no residual: v = x),
//   rstd = 1 / sqrt(mean(v^2) + eps), y = v w rstd
// the norm is of the sum as the stream holds it, since that is what the next layers add to; y is rounded once. In 8 bits rstd drops
// out of the codes: code = round(v w 127 / top), scale = top rstd / 127, top = max |v w| (rows8.hpp). Gradients from dy of y and
// dr of r, g = dy w, c = mean(g v) rstd^2:
//   dv = rstd (g - v c) + dr,  dx = dresidual = dv,  dw = sum over the rows of dy v rstd
// (the rounding of s to r passes a gradient as it is). Everything is bound by the bytes of the rows: each is read once and kept in
// registers, and rstd is computed again from them in the backward pass, which has to read v anyhow.
#include <algorithm>
#include <cfloat>

#include "rows8.hpp"

namespace bmx {

struct NormArgs {
    const void *x, *res, *w;        // w null: the rows as they are in 8 bits (quantize_rows), neither weight nor norm
    void *r, *y;
    int8_t* codes;
    float* scale;
    int blocks;                     // q8_blocks(H)
    int T, H;
    int xt, rt, wt, yt;             // row types
    float eps;
};

// A launch's axis holds fewer than 2^32 threads: rows past 2^20 on the second. Of whole 128 rows an XCD has 16 neighbours (workgroups go to
// the XCDs in turn), whose codes share lines of memory: written on eight XCDs a line goes out in eight parts (4,096 rows of 11,008 62 us,
// this way 44).
constexpr int ROW_BITS = 20;
static dim3 row_grid(int T) { return dim3((unsigned)std::min(T, 1 << ROW_BITS), (unsigned)(((int64_t)T + (1 << ROW_BITS) - 1) >> ROW_BITS)); }
__device__ __forceinline__ int64_t row_here(int T)
{
    const int64_t i = (int64_t)blockIdx.y << ROW_BITS | blockIdx.x, g = i & ~(int64_t)127;
    return g + 128 <= T ? g + (i & 7) * 16 + (i >> 3 & 15) : i;
}

// A workgroup a row, CH chunks of 8 values a lane: one to 4,096 values, two past them (8,192 rows of 5,120: ten waves of one chunk 72 us,
// five of two 62). NORM false: the rows as they are in 8 bits alone. WIDE: some tensor is fp32, and a chunk's registers hold any type;
// 16 bits alone need half of them (8,192 rows of 4,096, two tensors in and two out: 44 us, 6.0 TB/s; with any type's 50, of 16,384 190
// and 271), and the quantizing form no sums and weight (4,096 x 4,096 a fourth less: 13.0 us). fp32
// rows into a stream of 16 bits: 8,192 of 5,120 78 us, 5.4 TB/s.
template <int CH, bool NORM, bool WIDE>
__global__ __launch_bounds__(1024) void norm_k(const NormArgs p)
{
    auto type = [](int t) { return !WIDE ? t == ROW_BF16 ? (int)ROW_BF16 : (int)ROW_F16 : NORM ? t : (int)ROW_F32; };
    const int xt = type(p.xt), rt = type(p.rt), wt = type(p.wt), yt = p.yt == ROW_BF16 ? (int)ROW_BF16 : (int)ROW_F16;
    __shared__ float ssum[16];
    __shared__ uint32_t smax[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t t = row_here(p.T), row = t * p.H;
    if (t >= p.T) return;
    float v[CH][8];                                                // the row, then v w
    Raw8 x[CH], res[CH], w;
    auto at = [&](int c) { return (int)(threadIdx.x + c * blockDim.x) * 8; };
#pragma unroll
    for (int c = 0; c < CH; ++c)
    {
        const int h = at(c);
        if (h >= p.H) continue;
        x[c] = load_raw8(p.x, xt, row + h);
        if (NORM && p.res) res[c] = load_raw8(p.res, rt, row + h);
        if (NORM && CH == 1) w = load_raw8(p.w, wt, h);
    }
    float ssq = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
    {
        const int h = at(c);
        if (h >= p.H) continue;
        to_f32(x[c], xt, v[c]);
        if (NORM && p.res)
        {
            float a[8];
            to_f32(res[c], rt, a);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] += a[i];
            store8(p.r, rt, row + h, v[c]);
        }
        float b[8];
        if (NORM)
        {
            if (CH > 1) w = load_raw8(p.w, wt, h);
            to_f32(w, wt, b);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            if (NORM)
            {
                ssq = __builtin_fmaf(v[c][i], v[c][i], ssq);
                v[c][i] *= b[i];
            }
            top = max(top, mag(v[c][i]));
        }
        if (NORM && CH > 1) __builtin_amdgcn_sched_barrier(0);     // (else all chunks' weights are loaded at once: 74 registers)
    }
    const bool codes = !NORM || p.codes;
    if (NORM) ssq = wave_sum(ssq);
    if (codes) top = wave_max(top);
    if (waves > 1)
    {
        if (lane == 0) { ssum[wave] = ssq; smax[wave] = top; }
        lds_barrier();
        // (a lane each: one after the other their LDS reads are as long as the row's loads)
        if (NORM) ssq = wave_sum(lane < waves ? ssum[lane] : 0.0f);
        if (codes) top = wave_max(lane < waves ? smax[lane] : 0u);
    }
    const float rstd = NORM ? __fdiv_rn(1.0f, __builtin_sqrtf(__fdiv_rn(ssq, (float)p.H) + p.eps)) : 1.0f;
    const Top8 q = top8(top);
#pragma unroll
    for (int c = 0; c < CH; ++c)
    {
        const int h = at(c);
        if (codes && h < p.blocks * Q8_COLS)
            *reinterpret_cast<u32x2*>(p.codes + q8_at(t, h, p.blocks)) =
                h < p.H ? u32x2{codes4(v[c], q), codes4(v[c] + 4, q)} : u32x2{0, 0};
        if (NORM && p.y && h < p.H)
        {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = v[c][i] * rstd;
            store8(p.y, yt, row + h, y);
        }
    }
    if (codes && threadIdx.x == 0) p.scale[t] = NORM ? q.scale * rstd : q.scale;
}

static int launch_norm(const NormArgs& a, hipStream_t s)                  // H <= BMX_NORM_MAX_H
{
    const int chunks = (a.H + 511) / 512;                          // of a wave
    const bool wide = a.xt == ROW_F32 || a.rt == ROW_F32 || a.wt == ROW_F32;
    const dim3 grid = row_grid(a.T), one(chunks * 64), two((chunks + 1) / 2 * 64);
    if (!a.w)
    {
        if (wide) hipLaunchKernelGGL((norm_k<2, false, true>), grid, two, 0, s, a);
        else hipLaunchKernelGGL((norm_k<2, false, false>), grid, two, 0, s, a);
    }
    else if (chunks <= 8)
    {
        if (wide) hipLaunchKernelGGL((norm_k<1, true, true>), grid, one, 0, s, a);
        else hipLaunchKernelGGL((norm_k<1, true, false>), grid, one, 0, s, a);
    }
    else if (wide) hipLaunchKernelGGL((norm_k<2, true, true>), grid, two, 0, s, a);
    else hipLaunchKernelGGL((norm_k<2, true, false>), grid, two, 0, s, a);
    return check_launch("rms_norm");
}

// The same for any K and rows at any 2-byte boundary: a workgroup per row, read twice, a value a lane at a time: loads issued, not bytes,
// bound it (4,096 rows of 18,432 in fp32 152 us, in bf16 148; of 16,384 norm_k takes 65 for fp32's)
__global__ __launch_bounds__(512) void quantize_any_k(const NormArgs p)
{
    __shared__ uint32_t smax[8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = row_here(p.T), row = t * p.H;
    if (t >= p.T) return;
    auto value = [&](int h) {
        if (h >= p.H) return 0.0f;
        return p.xt == ROW_F32 ? static_cast<const float*>(p.x)[row + h] : value16(p.xt, static_cast<const uint16_t*>(p.x)[row + h]);
    };
    uint32_t top = 0;
    for (int h = threadIdx.x; h < p.H; h += 512) top = max(top, mag(value(h)));
    top = wave_max(top);
    if (lane == 0) smax[wave] = top;
    __syncthreads();
    for (int i = 0; i < 8; ++i) top = max(top, smax[i]);
    const Top8 q = top8(top);
    for (int h = threadIdx.x * 4; h < p.blocks * Q8_COLS; h += 2048)
    {
        const float v[4] = {value(h), value(h + 1), value(h + 2), value(h + 3)};
        *reinterpret_cast<uint32_t*>(p.codes + q8_at(t, h, p.blocks)) = codes4(v, q);
    }
    if (threadIdx.x == 0) p.scale[t] = q.scale;
}

int launch_quantize(const void* x, int type, const bmx_q8* out, hipStream_t s)
{
    NormArgs a = {};
    a.x = x; a.xt = type; a.T = out->N; a.H = out->K;
    a.codes = static_cast<int8_t*>(const_cast<void*>(out->codes));
    a.scale = const_cast<float*>(out->scale);
    a.blocks = q8_blocks(out->K);
    if (a.H % 8 == 0 && a.H <= BMX_NORM_MAX_H && reinterpret_cast<uintptr_t>(x) % 16 == 0) return launch_norm(a, s);
    hipLaunchKernelGGL(quantize_any_k, row_grid(a.T), dim3(512), 0, s, a);
    return check_launch("quantize");
}

// ---- gradients ----------------------------------------------------------------------------------------------------------

struct NormBackArgs {
    const void *v, *w, *dy, *dr;    // dr null: no gradient of r
    void *dx, *dres;                // null: not wanted
    float* part;                    // [workgroup][H], null: the weight's gradient is not wanted
    int T, H;
    int vt, wt, yt, xt;             // row types: v, dr and dres (of a sum v the residual's), w, dy, dx
    float eps;
};

// A workgroup takes every gridDim.x-th row and keeps its rows' sums for the weight's gradient in registers, and for rows of one chunk a
// lane the weight; the next row's loads are on their way while one is summed up. WIDE: some tensor is fp32. (Of 16 bits alone a chunk
// takes half the registers, and 24 waves of one chunk fit a compute unit: 8,192 rows of 4,096 with the forward pass 100 us, with an fp32
// weight and so WIDE 114; 4,096 of 16,384 223 and 264.) Two chunks of any type leave no registers for loads ahead and for what the first
// pass made of a row: AHEAD false makes it again.
template <int CH, bool WIDE>
__global__ __launch_bounds__(1024) void norm_back_k(const NormBackArgs p)
{
    constexpr bool AHEAD = CH == 1 || !WIDE;
    const int yt = p.yt == ROW_BF16 ? (int)ROW_BF16 : (int)ROW_F16, vt = WIDE ? p.vt : yt, wt = WIDE ? p.wt : yt, xt = WIDE ? p.xt : yt;
    __shared__ f32x2 red[2][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    float w[8], dw[CH][8];
    Raw8 v[CH], dy[CH], dr[CH];
    auto at = [&](int c) { return (int)(threadIdx.x + c * blockDim.x) * 8; };
    auto load = [&](int t) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
        {
            const int64_t i = (int64_t)t * p.H + at(c);
            if (at(c) >= p.H) continue;
            v[c] = load_raw8(p.v, vt, i);
            dy[c] = load_raw8(p.dy, yt, i);
            if (AHEAD && p.dr) dr[c] = load_raw8(p.dr, vt, i);
        }
    };
    auto weight = [&](int c) { to_f32(load_raw8(p.w, wt, at(c)), wt, w); };
    int t = blockIdx.x;
    load(t);
    if (CH == 1 && at(0) < p.H) weight(0);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[c][i] = 0.0f;
    for (int set = 0; t < p.T; t += gridDim.x, set ^= 1)
    {
        float a[CH][8], d[CH][8], more[CH][8];
        float ssq = 0.0f, dot = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
        {
            if (at(c) >= p.H) continue;
            to_f32(v[c], vt, a[c]);
            to_f32(dy[c], yt, d[c]);
            if (AHEAD && p.dr) to_f32(dr[c], vt, more[c]);
            if (CH > 1) weight(c);
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                ssq = __builtin_fmaf(a[c][i], a[c][i], ssq);
                dot = __builtin_fmaf(d[c][i] * w[i], a[c][i], dot);
            }
            if (CH > 1) __builtin_amdgcn_sched_barrier(0);
        }
        if (AHEAD && t + (int)gridDim.x < p.T) load(t + gridDim.x);
        ssq = wave_sum(ssq);
        dot = wave_sum(dot);
        if (lane == 0) red[set][wave] = f32x2{ssq, dot};
        lds_barrier();
        const f32x2 one = lane < waves ? red[set][lane] : f32x2{0.0f, 0.0f};
        ssq = wave_sum(one[0]);
        dot = wave_sum(one[1]);
        const float rstd = __fdiv_rn(1.0f, __builtin_sqrtf(__fdiv_rn(ssq, (float)p.H) + p.eps));
        const float k = __fdiv_rn(dot, (float)p.H) * rstd * rstd;
#pragma unroll
        for (int c = 0; c < CH; ++c)
        {
            if (at(c) >= p.H) continue;
            const int64_t at_row = (int64_t)t * p.H + at(c);
            float o[8], q[8];
            if (CH > 1) weight(c);
            if (!AHEAD)
            {
                asm volatile("" : "+v"(v[c].a), "+v"(v[c].b), "+v"(dy[c].a));     // (not to be kept from the first pass)
                dy[c].b = dy[c].a;
                to_f32(v[c], vt, a[c]);
                to_f32(dy[c], yt, d[c]);
                if (p.dr) to_f32(load_raw8(p.dr, vt, at_row), vt, more[c]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                o[i] = rstd * (d[c][i] * w[i] - a[c][i] * k);
                if (p.dr) o[i] += more[c][i];
                q[i] = o[i];
                dw[c][i] = __builtin_fmaf(d[c][i], a[c][i] * rstd, dw[c][i]);
            }
            if (p.dx) store8(p.dx, xt, at_row, o);
            if (p.dres) store8(p.dres, vt, at_row, q);
            if (CH > 1) __builtin_amdgcn_sched_barrier(0);
        }
        if (!AHEAD && t + (int)gridDim.x < p.T) load(t + gridDim.x);
    }
    if (!p.part) return;
#pragma unroll
    for (int c = 0; c < CH; ++c)
        if (at(c) < p.H) store8(p.part + (int64_t)blockIdx.x * p.H, ROW_F32, at(c), dw[c]);
}

// dw: the workgroups' sums of 32 columns, every 64th by a group of 8 lanes, then the groups' in their order
__global__ __launch_bounds__(512) void norm_weight_k(const float* __restrict__ part, int groups, int H, void* __restrict__ dw, int wt)
{
    __shared__ f32x4 red[64][8];
    const int q = threadIdx.x & 7, g = threadIdx.x >> 3, h = blockIdx.x * 32 + q * 4;
    f32x4 s = {0, 0, 0, 0};
    if (h < H)
#pragma unroll 4
        for (int i = g; i < groups; i += 64)
        {
            const f32x4 v = ldg4f(part + (int64_t)i * H + h);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[e];
        }
    red[g][q] = s;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const int c = blockIdx.x * 32 + threadIdx.x;
    if (c >= H) return;
    float sum = 0.0f;
#pragma unroll 8
    for (int i = 0; i < 64; ++i) sum += red[i][threadIdx.x >> 2][threadIdx.x & 3];
    if (wt == ROW_F32) static_cast<float*>(dw)[c] = sum;
    else static_cast<uint16_t*>(dw)[c] = (uint16_t)bits16(wt, sum);
}

// Waves of a row and workgroups of a backward pass: as many as the compute units hold at once (8,192 rows of 4,096: 16 waves a unit
// 98 us with the forward pass, 24 94, 32 96)
static int norm_back_waves(int H) { return H <= 8192 ? (H + 511) / 512 : (H + 1023) / 1024; }
static int norm_back_groups(int T, int H, bool wide) { return std::min(T, 256 * ((H <= 8192 && !wide ? 24 : 16) / norm_back_waves(H))); }

static int launch_norm_back(const NormBackArgs& a, int groups, bool wide, hipStream_t s)
{
    const dim3 grid(groups), block(norm_back_waves(a.H) * 64);
    if (a.H <= 8192)
    {
        if (wide) hipLaunchKernelGGL((norm_back_k<1, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((norm_back_k<1, false>), grid, block, 0, s, a);
    }
    else if (wide) hipLaunchKernelGGL((norm_back_k<2, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((norm_back_k<2, false>), grid, block, 0, s, a);
    return check_launch("rms_norm_backward");
}

// ---- argument checks ----------------------------------------------------------------------------------------------------

static bool odd16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; }
static bool is16(int t) { return t == BMX_DT_FP16 || t == BMX_DT_BF16; }

static int check_norm(const bmx_norm_desc* d, int T, const char* who)
{
    if (!d) return set_error(BMX_ERR_ARG, "%s: null descriptor", who);
    if (d->H <= 0 || d->H % 8 || d->H > BMX_NORM_MAX_H)
        return set_error(BMX_ERR_ARG, "%s: H (%d) must be a positive multiple of 8, at most %d", who, d->H, BMX_NORM_MAX_H);
    if (!is16(d->dtype)) return set_error(BMX_ERR_ARG, "%s: unknown dtype %d", who, d->dtype);
    for (int t : {d->x_dtype, d->residual_dtype, d->weight_dtype})
        if (t != d->dtype && t != BMX_DT_FP32)
            return set_error(BMX_ERR_ARG, "%s: x, residual and weight must be of dtype or fp32, got %d beside %d", who, t, d->dtype);
    if (!(d->eps > 0.0f && d->eps <= FLT_MAX)) return set_error(BMX_ERR_ARG, "%s: eps must be positive and finite", who);
    if (!d->weight || odd16(d->weight)) return set_error(BMX_ERR_ARG, "%s: weight null or not 16-byte aligned", who);
    if (T < 0 || T > (1 << 24)) return set_error(BMX_ERR_ARG, "%s: T (%d) outside [0, 2^24]", who, T);
    return BMX_OK;
}

// Outputs on inputs or on each other. A row's workgroup reads it whole before it writes: an output of the same type may lie where
// the input lies, but for another type, or rows further on, it would be on rows that other workgroups have yet to read.
struct Place { const void* at; size_t bytes; };
static bool meet(const Place& a, const Place& b)
{
    const uintptr_t p = reinterpret_cast<uintptr_t>(a.at), q = reinterpret_cast<uintptr_t>(b.at);
    return p && q && p < q + b.bytes && q < p + a.bytes;
}
static bool norm_overlaps(const NormArgs& a)
{
    const size_t n = (size_t)a.T * a.H, r = n * row_type_bytes(a.rt);
    const Place x = {a.x, n * row_type_bytes(a.xt)}, res = {a.res, r}, w = {a.w, a.H * row_type_bytes(a.wt)}, sum = {a.r, r},
                y = {a.y, n * row_type_bytes(a.yt)}, codes = {a.codes, q8_bytes(a.T, a.H)}, scale = {a.scale, (size_t)a.T * 4};
    if (meet(sum, x) && !(sum.at == x.at && a.rt == a.xt)) return true;
    if (meet(sum, res) && sum.at != res.at) return true;
    if (meet(y, x) && !(y.at == x.at && a.yt == a.xt)) return true;
    if (meet(y, res) || meet(y, sum) || meet(codes, scale)) return true;
    for (const Place& o : {sum, y})
        if (meet(o, w) || meet(o, codes) || meet(o, scale)) return true;
    for (const Place& i : {x, res, w})
        if (meet(i, codes) || meet(i, scale)) return true;
    return false;
}

// zeros for the weight's gradient of no rows
__global__ __launch_bounds__(256) void norm_zero_k(uint32_t* p, int n)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

}  // namespace bmx

using namespace bmx;

extern "C" {

int bmx_rms_norm(const bmx_norm_desc* desc, const void* x, const void* residual, int T, void* sum, void* y, const bmx_q8* rows,
                 bmx_stream_t stream)
{
    const char* fn = "bmx_rms_norm";
    int rc = check_norm(desc, T, fn);
    if (rc) return rc;
    if (rows && (rc = check_rows8(rows, T, desc->H, fn))) return rc;
    if (T == 0) return BMX_OK;
    if (!x || odd16(x) || odd16(residual) || odd16(sum) || odd16(y))
        return set_error(BMX_ERR_ARG, "%s: x null, or x, residual, sum or y not 16-byte aligned", fn);
    if (!residual != !sum) return set_error(BMX_ERR_ARG, "%s: a residual and its sum go together", fn);
    if (!y && !rows) return set_error(BMX_ERR_ARG, "%s: neither y nor rows is wanted", fn);
    NormArgs a = {};
    a.x = x; a.res = residual; a.w = desc->weight; a.r = sum; a.y = y;
    if (rows)
    {
        a.codes = static_cast<int8_t*>(const_cast<void*>(rows->codes));
        a.scale = const_cast<float*>(rows->scale);
        a.blocks = q8_blocks(rows->K);
    }
    a.T = T; a.H = desc->H;
    a.xt = desc->x_dtype; a.rt = desc->residual_dtype; a.wt = desc->weight_dtype; a.yt = desc->dtype;
    a.eps = desc->eps;
    if (norm_overlaps(a)) return set_error(BMX_ERR_ARG, "%s: sum, y or rows overlap an input or each other", fn);
    return launch_norm(a, static_cast<hipStream_t>(stream));
}

size_t bmx_rms_norm_backward_workspace(const bmx_norm_desc* desc, int T)
{
    if (check_norm(desc, T, "bmx_rms_norm_backward_workspace")) return 0;
    return align_up((size_t)(T ? norm_back_groups(T, desc->H, false) : 1) * desc->H * 4, 256);
}

int bmx_rms_norm_backward(const bmx_norm_desc* desc, const void* v, int summed, int T, const void* dy, const void* dr, void* dx,
                          void* dresidual, void* dweight, void* workspace, size_t workspace_bytes, bmx_stream_t stream)
{
    const char* fn = "bmx_rms_norm_backward";
    int rc = check_norm(desc, T, fn);
    if (rc) return rc;
    if (odd16(dweight) || odd16(dx) || odd16(dresidual)) return set_error(BMX_ERR_ARG, "%s: gradients must be 16-byte aligned", fn);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (T == 0)
    {
        if (!dweight) return BMX_OK;
        const int n = desc->weight_dtype == BMX_DT_FP32 ? desc->H : desc->H / 2;
        hipLaunchKernelGGL(norm_zero_k, dim3((n + 255) / 256), dim3(256), 0, s, static_cast<uint32_t*>(dweight), n);
        return check_launch(fn);
    }
    if (!v || !dy || odd16(v) || odd16(dy) || odd16(dr)) return set_error(BMX_ERR_ARG, "%s: v or dy null, or v, dy or dr not 16-byte aligned", fn);
    if (!summed && (dr || dresidual)) return set_error(BMX_ERR_ARG, "%s: gradients of a residual that was not there", fn);
    if (!dx && !dresidual && !dweight) return BMX_OK;
    if (dweight)
    {
        const size_t need = bmx_rms_norm_backward_workspace(desc, T);
        if (!workspace || odd16(workspace)) return set_error(BMX_ERR_ARG, "%s: workspace null or not 16-byte aligned", fn);
        if (workspace_bytes < need) return set_error(BMX_ERR_WORKSPACE, "%s: workspace %zu < %zu", fn, workspace_bytes, need);
    }
    NormBackArgs a = {};
    a.v = v; a.w = desc->weight; a.dy = dy; a.dr = dr; a.dx = dx; a.dres = dresidual;
    a.part = dweight ? static_cast<float*>(workspace) : nullptr;
    a.T = T; a.H = desc->H;
    a.vt = summed ? desc->residual_dtype : desc->x_dtype;
    a.wt = desc->weight_dtype; a.yt = desc->dtype; a.xt = desc->x_dtype;
    a.eps = desc->eps;
    const bool wide = a.vt == ROW_F32 || a.wt == ROW_F32 || a.xt == ROW_F32;
    const int groups = norm_back_groups(T, desc->H, wide);
    if ((rc = launch_norm_back(a, groups, wide, s)) || !dweight) return rc;
    hipLaunchKernelGGL(norm_weight_k, dim3((desc->H + 31) / 32), dim3(512), 0, s, a.part, groups, desc->H, dweight, desc->weight_dtype);
    return check_launch("norm_weight");
}

}  // extern "C"
