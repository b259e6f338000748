// The end of a residual block in one pass over the rows, and its gradient in another:
//
//     ry = (mean_f y^2 + eps)^-1/2                          norm after the block (with a post weight)
//     s  = x + scale sigmoid(gate) (y ry post)              residual scale and gate
//     rs = (mean_f s^2 + eps)^-1/2,   h = s rs w            norm before the next block
//
// Without y this is the first norm of a network: s = x.  Every array may be float or bfloat16;
// everything between the loads and the stores is fp32, h is taken from s before s is rounded.
//
// Backward, with t = ds + rs (dh w), q = scale sigmoid(gate) and means over f:
//     dx = t - s rs^3 mean(dh w s)                          (= the whole gradient of s)
//     dy = ry dx q post - y ry^3 mean(dx q post y),  dgate = dx q (y ry post) (1 - sigmoid(gate))
//     dw = sum_r dh s rs,   dpost = sum_r dx q y ry,   dscale = sum_r dx sigmoid(gate) y ry post
// The second mean needs dx, which needs the first; written out, mean(dx q post y) =
// mean(t q post y) - rs^3 mean(dh w s) mean(s q post y), so that one reduction of three sums over
// the row serves both.  s is recomputed from x, y, gate (read anyway) with the two inverse norms
// that the forward leaves (8 bytes a row), not from its rounded copy.
//
// Bound by memory.  L lanes share a row (L the power of two that covers it with 16 bytes a lane, up
// to a whole workgroup), the row stays in registers between the reduction and the stores.  A
// workgroup of the backward pass walks rows gridDim apart and keeps its share of the three column
// sums in registers; the workgroups' sums are added in order by a second kernel: no atomics.
#include <algorithm>
#include <type_traits>

#include "tile_product.h"

namespace jg {

constexpr int kNormBlocks = 1024;      // workgroups of the backward pass, at most
constexpr int kNormMaxWidth = 8192;

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);      // elements of a 16-byte access

// V consecutive elements as floats; `n` of them exist (the rest read as zero, are not written)
__device__ __forceinline__ void load_vec(const bf16 *p, int n, float (&v)[8])
{
    Eight<bf16> e;
    if (n >= 8) e.load(p);
    else e.load_some(p, n);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = bf16_lo(e.v[i]);
        v[2 * i + 1] = bf16_hi(e.v[i]);
    }
}
__device__ __forceinline__ void load_vec(const float *p, int n, float (&v)[4])
{
    if (n >= 4) {
        const f32x4 e = *reinterpret_cast<const f32x4_at4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = e[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = i < n ? p[i] : 0.f;
    }
}
__device__ __forceinline__ void store_vec(bf16 *p, int n, const float (&v)[8])
{
    if (n >= 8) {
        *reinterpret_cast<u32x4_at2 *>(p) =
            u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < n) p[i] = from_float<bf16>(v[i]);
}
__device__ __forceinline__ void store_vec(float *p, int n, const float (&v)[4])
{
    if (n >= 4) {
        *reinterpret_cast<f32x4_at4 *>(p) = f32x4{v[0], v[1], v[2], v[3]};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) p[i] = v[i];
}

// sums of `v[0..N-1]` over the L lanes of a row, in every one of them.  L > 64: the row's lanes are
// the workgroup, which calls this together; `scratch` holds N * L / 64 floats.
template <int L, int N> __device__ __forceinline__ void row_sum(float (&v)[N], float *scratch)
{
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int o = (L < kWave ? L : kWave) / 2; o > 0; o >>= 1) v[i] += __shfl_xor(v[i], o, kWave);
    if (L > kWave) {
        constexpr int waves = L / kWave;
        __syncthreads();
        if (lane_id() == 0)
#pragma unroll
            for (int i = 0; i < N; i++) scratch[i * waves + wave_in_block()] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = 0.f;
            for (int w = 0; w < waves; w++) v[i] += scratch[i * waves + w];
        }
    }
}

struct NormArgs {
    const void *x, *y, *gate, *scale, *post, *w;
    void *s, *h;
    float *ry, *rs;
    int64_t R;
    int F;
    float eps;
};

__device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + __expf(-g)); }

template <int L> constexpr int norm_threads() { return L > 256 ? L : 256; }

// L lanes a row, C vectors a lane; grid: rows / (threads / L)
template <typename T, int L, int C> __global__ __launch_bounds__(norm_threads<L>()) void norm_fwd(NormArgs a)
{
    constexpr int V = kVec<T>;
    __shared__ float scratch[2 * (L > kWave ? L / kWave : 1)];
    const int lane = threadIdx.x % L;
    const int64_t row = (int64_t)blockIdx.x * (norm_threads<L>() / L) + threadIdx.x / L;
    const bool mine = row < a.R;      // rows past the last are computed from nothing and not stored
    const int64_t base = row * a.F;
    const T *x = static_cast<const T *>(a.x), *y = static_cast<const T *>(a.y), *gate = static_cast<const T *>(a.gate);
    const T *scale = static_cast<const T *>(a.scale), *post = static_cast<const T *>(a.post), *w = static_cast<const T *>(a.w);
    float s[C][V], b[C][V], q[C][V];
    int left[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int f = (c * L + lane) * V;
        left[c] = mine ? a.F - f : 0;
        load_vec(x + base + f, left[c], s[c]);
        if (y) load_vec(y + base + f, left[c], b[c]);
        if (gate) load_vec(gate + base + f, left[c], q[c]);
    }
    if (y) {
        float ry = 1.f;
        if (post) {
            float sum[1] = {0.f};
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < V; i++) sum[0] += b[c][i] * b[c][i];
            row_sum<L>(sum, scratch);
            ry = rsqrtf(sum[0] / (float)a.F + a.eps);
            if (a.ry && lane == 0 && mine) a.ry[row] = ry;
        }
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int f = (c * L + lane) * V;
            float v[V];
            if (post) {
                load_vec(post + f, left[c], v);
#pragma unroll
                for (int i = 0; i < V; i++) b[c][i] *= ry * v[i];
            }
            if (gate) {
#pragma unroll
                for (int i = 0; i < V; i++) b[c][i] *= sigmoid(q[c][i]);
            }
            if (scale) {
                load_vec(scale + f, left[c], v);
#pragma unroll
                for (int i = 0; i < V; i++) b[c][i] *= v[i];
            }
#pragma unroll
            for (int i = 0; i < V; i++) s[c][i] += i < left[c] ? b[c][i] : 0.f;
            if (a.s) store_vec(static_cast<T *>(a.s) + base + f, left[c], s[c]);
        }
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < V; i++) sum[0] += s[c][i] * s[c][i];
    row_sum<L>(sum, scratch + (L > kWave ? L / kWave : 1));
    const float rs = rsqrtf(sum[0] / (float)a.F + a.eps);
    if (a.rs && lane == 0 && mine) a.rs[row] = rs;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int f = (c * L + lane) * V;
        float v[V];
        load_vec(w + f, left[c], v);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] *= s[c][i] * rs;
        store_vec(static_cast<T *>(a.h) + base + f, left[c], v);
    }
}

struct NormGradArgs {
    const void *x, *y, *gate, *scale, *post, *w;
    const float *ry, *rs;
    const void *ds, *dh;
    void *dx, *dy, *dgate, *dscale, *dpost, *dw;
    float *part;      // [3][blocks][F]: the workgroups' sums for dw, dpost, dscale
    int64_t R;
    int F;
};

template <typename T, int L, int C> __global__ __launch_bounds__(norm_threads<L>()) void norm_bwd(NormGradArgs a)
{
    constexpr int V = kVec<T>;
    constexpr int groups = norm_threads<L>() / L;      // rows of a workgroup at a time
    __shared__ float scratch[3 * (L > kWave ? L / kWave : 1)];
    __shared__ float joined[groups > 1 ? norm_threads<L>() * C * V : 1];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const T *x = static_cast<const T *>(a.x), *y = static_cast<const T *>(a.y), *gate = static_cast<const T *>(a.gate);
    const T *scale = static_cast<const T *>(a.scale), *post = static_cast<const T *>(a.post), *w = static_cast<const T *>(a.w);
    const T *ds = static_cast<const T *>(a.ds), *dh = static_cast<const T *>(a.dh);
    float sum_w[C][V] = {}, sum_p[C][V] = {}, sum_s[C][V] = {};
    const float over_f = 1.f / (float)a.F;
    // every wavefront takes the same number of turns: the reductions of wide rows have barriers
    for (int64_t row0 = (int64_t)blockIdx.x * groups; row0 < a.R; row0 += (int64_t)gridDim.x * groups) {
        const int64_t row = row0 + group;
        const bool mine = row < a.R;
        const int64_t base = row * a.F;
        const float rs = mine ? a.rs[row] : 0.f, ry = mine && y && post ? a.ry[row] : 1.f;
        float s[C][V], b[C][V], t[C][V], g[C][V], e[C][V];
        int left[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int f = (c * L + lane) * V;
            left[c] = mine ? a.F - f : 0;
            load_vec(x + base + f, left[c], s[c]);
            if (y) load_vec(y + base + f, left[c], b[c]);
            if (gate) load_vec(gate + base + f, left[c], g[c]);
            if (dh) load_vec(dh + base + f, left[c], e[c]);
            if (ds) load_vec(ds + base + f, left[c], t[c]);
        }
        float sums[3] = {0.f, 0.f, 0.f};      // dh w s, t q post y, s q post y
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int f = (c * L + lane) * V;
            float wv[V], pv[V], sv[V];
            load_vec(w + f, left[c], wv);
            if (post) load_vec(post + f, left[c], pv);
            if (scale) load_vec(scale + f, left[c], sv);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const bool in = i < left[c];
                if (y) {
                    const float p = post ? pv[i] : 1.f, k = scale ? sv[i] : 1.f;
                    g[c][i] = gate ? sigmoid(g[c][i]) : 1.f;
                    s[c][i] += in ? k * g[c][i] * (b[c][i] * ry * p) : 0.f;
                }
                if (!dh) e[c][i] = 0.f;
                if (!ds) t[c][i] = 0.f;
                const float hw = e[c][i] * wv[i];
                t[c][i] += rs * hw;
                sums[0] += hw * s[c][i];
                if (dh) sum_w[c][i] += e[c][i] * (s[c][i] * rs);
                if (y && post) {
                    const float z = (scale ? sv[i] : 1.f) * g[c][i] * pv[i] * b[c][i];
                    sums[1] += in ? t[c][i] * z : 0.f;
                    sums[2] += in ? s[c][i] * z : 0.f;
                }
            }
        }
        row_sum<L>(sums, scratch);
        const float back = rs * rs * rs * (sums[0] * over_f);
        const float back_y = ry * ry * ry * ((sums[1] - back * sums[2]) * over_f);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int f = (c * L + lane) * V;
            float pv[V], sv[V], dy[V], dg[V];
            if (post) load_vec(post + f, left[c], pv);
            if (scale) load_vec(scale + f, left[c], sv);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float dx = t[c][i] - s[c][i] * back;
                t[c][i] = dx;
                if (y) {
                    const float k = scale ? sv[i] : 1.f, p = post ? pv[i] : 1.f;
                    const float u = b[c][i] * ry, dv = dx * k * g[c][i];
                    dy[i] = post ? ry * (dv * p) - b[c][i] * back_y : dv;
                    dg[i] = dv * (u * p) * (1.f - g[c][i]);
                    if (post) sum_p[c][i] += dv * u;
                    if (scale) sum_s[c][i] += dx * g[c][i] * (u * p);
                }
            }
            if (a.dx) store_vec(static_cast<T *>(a.dx) + base + f, left[c], t[c]);
            if (a.dy) store_vec(static_cast<T *>(a.dy) + base + f, left[c], dy);
            if (a.dgate) store_vec(static_cast<T *>(a.dgate) + base + f, left[c], dg);
        }
    }
    // the workgroup's column sums: its row groups in order
    auto join = [&](float (&v)[C][V], int which) {
        float *out = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * a.F;
        if (groups > 1) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < V; i++) joined[group * (L * C * V) + (c * L + lane) * V + i] = v[c][i];
            __syncthreads();
            for (int f = threadIdx.x; f < a.F; f += norm_threads<L>()) {
                float sum = 0.f;
                for (int k = 0; k < groups; k++) sum += joined[k * (L * C * V) + f];
                out[f] = sum;
            }
        } else {
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < V; i++)
                    if ((c * L + lane) * V + i < a.F) out[(c * L + lane) * V + i] = v[c][i];
        }
    };
    if (a.dw) join(sum_w, 0);
    if (a.dpost) join(sum_p, 1);
    if (a.dscale) join(sum_s, 2);
}

// The workgroups' sums in order: a workgroup adds 32 columns, 8 strands of workgroups each.
// grid: x = columns / 32, y = the three sums
template <typename T> __global__ __launch_bounds__(256) void norm_bwd_columns(NormGradArgs a, int blocks)
{
    __shared__ float strands[8][32];
    void *out = blockIdx.y == 0 ? a.dw : blockIdx.y == 1 ? a.dpost : a.dscale;
    if (!out) return;
    const int f = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
    float v = 0.f;
    if (f < a.F)
        for (int b = strand; b < blocks; b += 8) v += a.part[((int64_t)blockIdx.y * blocks + b) * a.F + f];
    strands[strand][threadIdx.x & 31] = v;
    __syncthreads();
    if (strand == 0 && f < a.F) {
#pragma unroll
        for (int k = 1; k < 8; k++) v += strands[k][threadIdx.x];
        static_cast<T *>(out)[f] = from_float<T>(v);
    }
}

// calls body(L, C) as compile-time constants: the narrowest lanes and vectors that cover a row
template <typename T, typename Body> static void norm_shape(int F, Body &&body)
{
    const int v = (int)ceil_div(F, kVec<T>);      // vectors of a row
    if (v <= 8) body(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    else if (v <= 16) body(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    else if (v <= 32) body(std::integral_constant<int, 32>(), std::integral_constant<int, 1>());
    else if (v <= 64) body(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    else if (v <= 128) body(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    else if (v <= 256) body(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
    else if (v <= 512) body(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    else if (v <= 1024) body(std::integral_constant<int, 512>(), std::integral_constant<int, 2>());
    else if constexpr (kNormMaxWidth / kVec<T> > 1024)
        body(std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
}
static int norm_lanes(int32_t dtype, int F)
{
    int lanes = 0;
    auto take = [&](auto l, auto) { lanes = l; };
    if (dtype == JGAMD_F32) norm_shape<float>(F, take);
    else norm_shape<bf16>(F, take);
    return lanes;
}
static int norm_blocks(int64_t R, int lanes)
{
    const int groups = lanes > 256 ? 1 : 256 / lanes;
    return (int)std::min<int64_t>(ceil_div(R, groups), kNormBlocks);
}

static int32_t norm_check(const char *who, int64_t R, int32_t F, int32_t dtype)
{
    if (R < 0 || F <= 0 || F > kNormMaxWidth)
        return fail(JGAMD_ERR_SIZE, "%s: R=%lld F=%d (R >= 0, 0 < F <= %d)", who, (long long)R, F, kNormMaxWidth);
    if (R > 0x7fffffffLL) return fail(JGAMD_ERR_SIZE, "%s: R=%lld too large", who, (long long)R);
    if (dtype != JGAMD_F32 && dtype != JGAMD_BF16) return fail(JGAMD_ERR_UNSUPPORTED, "%s: unknown dtype %d", who, dtype);
    return 0;
}

}  // namespace jg

using namespace jg;
#define JG_EXPORT extern "C" __attribute__((visibility("default")))

JG_EXPORT int32_t jgamd_residual_norm_fwd(const void *x, const void *y, const void *gate, const void *scale,
                                          const void *post, const void *w, void *s, void *h, float *ry, float *rs,
                                          int64_t R, int32_t F, float eps, int32_t dtype, void *stream)
{
    if (int32_t rc = norm_check("residual_norm_fwd", R, F, dtype)) return rc;
    if (R == 0) return 0;
    if (!y && (gate || scale || post))
        return fail(JGAMD_ERR_NULL, "residual_norm_fwd: gate, scale and post need y");
    if (!x || !w || !h) return fail(JGAMD_ERR_NULL, "residual_norm_fwd: x / w / h is NULL");
    const uintptr_t any = (uintptr_t)x | (uintptr_t)y | (uintptr_t)gate | (uintptr_t)scale | (uintptr_t)post |
                          (uintptr_t)w | (uintptr_t)s | (uintptr_t)h;
    if ((any & (dtype == JGAMD_F32 ? 3 : 1)) || (((uintptr_t)ry | (uintptr_t)rs) & 3))
        return fail(JGAMD_ERR_ALIGN, "residual_norm_fwd: an array does not start at a multiple of its element's size");
    const NormArgs a{x, y, gate, scale, post, w, s, h, ry, rs, R, F, eps};
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto launch = [&](auto type, auto l, auto c) {
        using T = decltype(type);
        constexpr int L = decltype(l)::value, C = decltype(c)::value, threads = norm_threads<L>();
        hipLaunchKernelGGL((norm_fwd<T, L, C>), dim3((unsigned)ceil_div(R, threads / L)), dim3(threads), 0, st, a);
    };
    if (dtype == JGAMD_F32) norm_shape<float>(F, [&](auto l, auto c) { launch(float(), l, c); });
    else norm_shape<bf16>(F, [&](auto l, auto c) { launch(bf16(), l, c); });
    return launch_status("residual_norm_fwd");
}

JG_EXPORT int32_t jgamd_residual_norm_bwd_workspace(int64_t R, int32_t F, size_t *bytes)
{
    if (!bytes) return fail(JGAMD_ERR_NULL, "residual_norm_bwd_workspace: bytes is NULL");
    if (int32_t rc = norm_check("residual_norm_bwd_workspace", R, F, JGAMD_F32)) return rc;
    *bytes = carve_bytes((size_t)3 * std::min<int64_t>(R, kNormBlocks) * F, 4);
    return 0;
}

JG_EXPORT int32_t jgamd_residual_norm_bwd(const void *x, const void *y, const void *gate, const void *scale,
                                          const void *post, const void *w, const float *ry, const float *rs,
                                          const void *ds, const void *dh, void *dx, void *dy, void *dgate, void *dscale,
                                          void *dpost, void *dw, int64_t R, int32_t F, int32_t dtype, void *ws,
                                          size_t ws_bytes, void *stream)
{
    if (int32_t rc = norm_check("residual_norm_bwd", R, F, dtype)) return rc;
    if (R > 0 && !y && (gate || scale || post || dy))
        return fail(JGAMD_ERR_NULL, "residual_norm_bwd: gate, scale, post and dy need y");
    if ((dgate && !gate) || (dscale && !scale) || (dpost && !post))
        return fail(JGAMD_ERR_NULL, "residual_norm_bwd: a gradient of an input that is NULL");
    if (R > 0 && (!x || !w || !rs || (post && !ry))) return fail(JGAMD_ERR_NULL, "residual_norm_bwd: x / w / rs / ry is NULL");
    const uintptr_t any = (uintptr_t)x | (uintptr_t)y | (uintptr_t)gate | (uintptr_t)scale | (uintptr_t)post |
                          (uintptr_t)w | (uintptr_t)ds | (uintptr_t)dh | (uintptr_t)dx | (uintptr_t)dy |
                          (uintptr_t)dgate | (uintptr_t)dscale | (uintptr_t)dpost | (uintptr_t)dw;
    if ((any & (dtype == JGAMD_F32 ? 3 : 1)) || (((uintptr_t)ry | (uintptr_t)rs) & 3))
        return fail(JGAMD_ERR_ALIGN, "residual_norm_bwd: an array does not start at a multiple of its element's size");
    const bool columns = dw || dpost || dscale;
    const size_t need = columns ? carve_bytes((size_t)3 * std::min<int64_t>(R, kNormBlocks) * F, 4) : 0;
    if (need > 0 && (!ws || ws_bytes < need))
        return fail(JGAMD_ERR_WORKSPACE, "residual_norm_bwd: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
    if (need > 0 && ((uintptr_t)ws & 255) != 0)
        return fail(JGAMD_ERR_ALIGN, "residual_norm_bwd: workspace not 256-byte aligned");
    const NormGradArgs a{x, y, gate, scale, post, w, ry, rs, ds, dh, dx, dy, dgate, dscale, dpost, dw,
                         static_cast<float *>(ws), R, F};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int blocks = norm_blocks(R, norm_lanes(dtype, F));
    auto launch = [&](auto type, auto l, auto c) {
        using T = decltype(type);
        constexpr int L = decltype(l)::value, C = decltype(c)::value;
        hipLaunchKernelGGL((norm_bwd<T, L, C>), dim3((unsigned)blocks), dim3(norm_threads<L>()), 0, st, a);
    };
    if (blocks > 0) {
        if (dtype == JGAMD_F32) norm_shape<float>(F, [&](auto l, auto c) { launch(float(), l, c); });
        else norm_shape<bf16>(F, [&](auto l, auto c) { launch(bf16(), l, c); });
        if (int32_t rc = launch_status("residual_norm_bwd")) return rc;
    }
    if (!columns) return 0;
    const dim3 grid((unsigned)ceil_div(F, 32), 3);
    if (dtype == JGAMD_F32) hipLaunchKernelGGL((norm_bwd_columns<float>), grid, dim3(256), 0, st, a, blocks);
    else hipLaunchKernelGGL((norm_bwd_columns<bf16>), grid, dim3(256), 0, st, a, blocks);
    return launch_status("residual_norm_bwd");
}
