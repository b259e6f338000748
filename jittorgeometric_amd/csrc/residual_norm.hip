// The end of a residual block in one pass over the rows, and its gradient in another:
//
//     ry = (mean_f y^2 + eps)^-1/2                          norm after the block (with a post weight)
//     s  = x + scale sigmoid(gate) (y ry post)              residual scale and gate
//     rs = (mean_f s^2 + eps)^-1/2,   h = s rs w            norm before the next block
//
// Without y this is the first norm of a network: s = x.  Every array may be float or bfloat16;
// everything between the loads and the stores is fp32, h is taken from s before s is rounded.
//
// Backward, with t = ds + rs (dh w), z = q post (y ry), q = scale sigmoid(gate) and means over f:
//     dx = t - (s rs) rs m,   m = mean(dh w s) rs           (= the whole gradient of s)
//     dy = ry dx q post - (y ry) ry mean(dx z),   dgate = dx q (y ry post) sigmoid(-gate)
//     dw = sum_r dh s rs,   dpost = sum_r dx q y ry,   dscale = sum_r dx sigmoid(gate) y ry post
// The second mean needs dx, which needs the first; written out, mean(dx z) = mean(t z) - rs m rs mean(s z),
// so that one reduction of three sums over the row serves both.  Every inverse norm stands at a factor
// of its row's size: rs^3 by itself leaves float32 for rows of 1e13 and of 1e-13.  s is recomputed from x, y,
// gate (read anyway) with the two inverse norms that the forward leaves (8 bytes a row), not from its rounded copy.
//
// Bound by memory.  L lanes share a row (L the power of two that covers it with 16 bytes a lane, up
// to a whole workgroup), the row stays in registers between the reduction and the stores.  A
// workgroup of the backward pass walks rows gridDim apart and keeps its share of the three column
// sums in registers; the workgroups' sums are added in order by a second kernel: no atomics.
#include <algorithm>
#include <type_traits>

#include "tile_product.h"

namespace jg {

// Workgroups of the backward pass, at most: those resident at once (100 registers, 60 without a block).
// 30011 rows of 1001 floats without a block: 92 us with 1024, 72 with 2048; 262144 rows of 1024 bfloat16
// with one: 890 with 1024, 1040 with 2048.
constexpr int kNormBlocks = 1024, kNormBlocksAlone = 2048;
constexpr int kNormMaxWidth = 8192;

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);      // elements of a 16-byte access
// of the backward pass: eight arrays of a row in registers leave no room for more (262144 rows of 1024 bfloat16:
// 887 us, 1012 with 8)
constexpr int kGradVec = 4;

// V consecutive elements as floats; `n` of them exist (the rest read as zero, are not written).
// WHOLE: rows are whole vectors, n is at least V or nothing exists.
template <bool WHOLE> __device__ __forceinline__ void load_vec(const bf16 *p, int n, float (&v)[8])
{
    Eight<bf16> e;
    if (WHOLE) {
        e.clear();
        if (n > 0) e.load(p);
    } else if (n >= 8) e.load(p);
    else e.load_some(p, n);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = bf16_lo(e.v[i]);
        v[2 * i + 1] = bf16_hi(e.v[i]);
    }
}
typedef uint32_t u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));

// four elements as they lie in memory, on their way to four floats
template <typename T> struct Four;
template <> struct Four<bf16> {
    u32x2 v;
    __device__ __forceinline__ void clear() { v = u32x2{0, 0}; }
    __device__ __forceinline__ void load(const bf16 *p) { v = *reinterpret_cast<const u32x2_at2 *>(p); }
    __device__ __forceinline__ void load_some(const bf16 *p, int n)
    {
        uint32_t e[4];
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = i < n ? p[i].u : 0;
        v = u32x2{e[0] | e[1] << 16, e[2] | e[3] << 16};
    }
    __device__ __forceinline__ void get(float (&f)[4]) const
    {
        f[0] = bf16_lo(v[0]), f[1] = bf16_hi(v[0]), f[2] = bf16_lo(v[1]), f[3] = bf16_hi(v[1]);
    }
};
template <> struct Four<float> {
    f32x4 v;
    __device__ __forceinline__ void clear() { v = f32x4{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ void load(const float *p) { v = *reinterpret_cast<const f32x4_at4 *>(p); }
    __device__ __forceinline__ void load_some(const float *p, int n)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = i < n ? p[i] : 0.f;
    }
    __device__ __forceinline__ void get(float (&f)[4]) const
    {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = v[i];
    }
};
template <bool WHOLE, typename T> __device__ __forceinline__ Four<T> load_four(const T *p, int n)
{
    Four<T> e;
    if (WHOLE) {
        e.clear();
        if (n > 0) e.load(p);
    } else if (n >= 4) e.load(p);
    else e.load_some(p, n);
    return e;
}
template <bool WHOLE, typename T> __device__ __forceinline__ void load_vec(const T *p, int n, float (&v)[4])
{
    load_four<WHOLE>(p, n).get(v);
}
template <bool WHOLE> __device__ __forceinline__ void store_vec(bf16 *p, int n, const float (&v)[4])
{
    if (WHOLE ? n > 0 : n >= 4) {
        *reinterpret_cast<u32x2_at2 *>(p) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        return;
    }
    if (WHOLE) return;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) p[i] = from_float<bf16>(v[i]);
}
template <bool WHOLE> __device__ __forceinline__ void store_vec(bf16 *p, int n, const float (&v)[8])
{
    if (WHOLE ? n > 0 : n >= 8) {
        *reinterpret_cast<u32x4_at2 *>(p) =
            u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
        return;
    }
    if (WHOLE) return;
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < n) p[i] = from_float<bf16>(v[i]);
}
template <bool WHOLE> __device__ __forceinline__ void store_vec(float *p, int n, const float (&v)[4])
{
    if (WHOLE ? n > 0 : n >= 4) {
        *reinterpret_cast<f32x4_at4 *>(p) = f32x4{v[0], v[1], v[2], v[3]};
        return;
    }
    if (WHOLE) return;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) p[i] = v[i];
}

// sums of `v[0..N-1]` over the L lanes of a row, in every one of them.  L > 64: the workgroup calls this
// together; `scratch` holds N floats a wavefront.
template <int L, int N> __device__ __forceinline__ void row_sum(float (&v)[N], float *scratch)
{
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int o = (L < kWave ? L : kWave) / 2; o > 0; o >>= 1) v[i] += __shfl_xor(v[i], o, kWave);
    if (L > kWave) {
        constexpr int waves = L / kWave;
        const int first = wave_in_block() / waves * waves;
        __syncthreads();
        if (lane_id() == 0)
#pragma unroll
            for (int i = 0; i < N; i++) scratch[wave_in_block() * N + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < waves; w++) v[i] += scratch[(first + w) * N + i];
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

// hardware exponential and reciprocal: within a few units of the last place
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

// The smaller of sigmoid(g) and sigmoid(-g), negative where it is the first: one register for both.  1 - sigmoid(g)
// of a rounded sigmoid is off by 1 % at g = 12 and zero from 17 on.
__device__ __forceinline__ float sigmoids(float g)
{
    const float e = __expf(-fabsf(g));
    return copysignf(e * __builtin_amdgcn_rcpf(1.f + e), g);
}
__device__ __forceinline__ float open_of(float v) { return signbit(v) ? -v : 1.f - v; }      // sigmoid(g)
__device__ __forceinline__ float shut_of(float v) { return signbit(v) ? 1.f + v : v; }       // sigmoid(-g)

template <int L> constexpr int norm_threads() { return L > 256 ? L : 256; }

// L lanes a row, C vectors a lane; grid: rows / (threads / L) workgroups by block_number
template <typename T, int L, int C, bool WHOLE>
__global__ __launch_bounds__(norm_threads<L>()) void norm_fwd(NormArgs a)
{
    constexpr int V = kVec<T>;
    __shared__ float scratch[2 * norm_threads<L>() / kWave];
    const int lane = threadIdx.x % L;
    const int64_t row = block_number() * (norm_threads<L>() / L) + threadIdx.x / L;
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
        load_vec<WHOLE>(x + base + f, left[c], s[c]);
        if (y) load_vec<WHOLE>(y + base + f, left[c], b[c]);
        if (gate) load_vec<WHOLE>(gate + base + f, left[c], q[c]);
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
                load_vec<WHOLE>(post + f, left[c], v);
#pragma unroll
                for (int i = 0; i < V; i++) b[c][i] *= ry * v[i];
            }
            if (gate) {
#pragma unroll
                for (int i = 0; i < V; i++) b[c][i] *= sigmoid(q[c][i]);
            }
            if (scale) {
                load_vec<WHOLE>(scale + f, left[c], v);
#pragma unroll
                for (int i = 0; i < V; i++) b[c][i] *= v[i];
            }
#pragma unroll
            for (int i = 0; i < V; i++) s[c][i] += i < left[c] ? b[c][i] : 0.f;
            if (a.s) store_vec<WHOLE>(static_cast<T *>(a.s) + base + f, left[c], s[c]);
        }
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < V; i++) sum[0] += s[c][i] * s[c][i];
    row_sum<L>(sum, scratch + norm_threads<L>() / kWave);
    const float rs = rsqrtf(sum[0] / (float)a.F + a.eps);
    if (a.rs && lane == 0 && mine) a.rs[row] = rs;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int f = (c * L + lane) * V;
        float v[V];
        load_vec<WHOLE>(w + f, left[c], v);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] *= s[c][i] * rs;
        store_vec<WHOLE>(static_cast<T *>(a.h) + base + f, left[c], v);
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

// BLOCK: there is a y.  grid: x = workgroups, each with every gridDim.x-th group of rows
template <typename T, int L, int C, bool WHOLE, bool BLOCK>
__global__ __launch_bounds__(norm_threads<L>(), C == 1 ? 4 : 2) void norm_bwd(NormGradArgs a)
{
    constexpr int V = kGradVec;
    constexpr int groups = norm_threads<L>() / L;      // rows of a workgroup at a time
    __shared__ float scratch[3 * norm_threads<L>() / kWave];
    __shared__ float joined[groups > 1 ? norm_threads<L>() * C * V : 1];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const T *x = static_cast<const T *>(a.x), *y = BLOCK ? static_cast<const T *>(a.y) : nullptr;
    const T *gate = BLOCK ? static_cast<const T *>(a.gate) : nullptr;
    const T *scale = BLOCK ? static_cast<const T *>(a.scale) : nullptr, *post = BLOCK ? static_cast<const T *>(a.post) : nullptr;
    const T *w = static_cast<const T *>(a.w);
    const T *ds = static_cast<const T *>(a.ds), *dh = static_cast<const T *>(a.dh);
    float sum_w[C][V] = {}, sum_p[C][V] = {}, sum_s[C][V] = {};
    // the three small rows; a part that is left out counts as 1: no branch in the arithmetic
    constexpr bool kKeep = C < 4;      // in registers, or read again for every row
    struct Small {
        float w[V], post[V], scale[V];
    };
    auto small = [&](int c) {
        Small v;
        const int f = (c * L + lane) * V, n = a.F - f;
        load_vec<WHOLE>(w + f, n, v.w);
        if (post) load_vec<WHOLE>(post + f, n, v.post);
        if (scale) load_vec<WHOLE>(scale + f, n, v.scale);
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (!post) v.post[i] = 1.f;
            if (!scale) v.scale[i] = 1.f;
        }
        return v;
    };
    Small kept[kKeep ? C : 1];
    if (kKeep)
#pragma unroll
        for (int c = 0; c < C; c++) kept[c] = small(c);
    const float over_f = 1.f / (float)a.F;
    struct Row {
        Four<T> x[C], y[C], gate[C], dh[C], ds[C];
        float rs, ry;
    };
    // whether no lane of this wavefront holds the row's ragged end
    bool even[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int n = a.F - (c * L + lane) * V;
        even[c] = __all(n >= V || n <= 0);
    }
    auto read = [&](int64_t row) {
        Row r;
        const bool mine = row < a.R;
        const int64_t base = row * a.F;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int f = (c * L + lane) * V, left = mine ? a.F - f : 0;
            r.y[c].clear();
            r.gate[c].clear();
            r.dh[c].clear();
            r.ds[c].clear();
            auto load = [&](auto whole) {
                constexpr bool W = decltype(whole)::value;
                r.x[c] = load_four<W>(x + base + f, left);
                if (y) r.y[c] = load_four<W>(y + base + f, left);
                if (gate) r.gate[c] = load_four<W>(gate + base + f, left);
                if (dh) r.dh[c] = load_four<W>(dh + base + f, left);
                if (ds) r.ds[c] = load_four<W>(ds + base + f, left);
            };
            if (WHOLE || even[c]) load(std::true_type());
            else load(std::false_type());
        }
        r.rs = mine ? a.rs[row] : 0.f;
        r.ry = mine && post ? a.ry[row] : 1.f;
        return r;
    };
    // every wavefront takes the same number of turns: the reductions of wide rows have barriers.  What a
    // lane holds past the row's end, or past the last row, is zero and adds zero.  The next row is read
    // while this one is worked on (rows of 1024 bfloat16: 1192 -> 896 us for 262144 of them), but not
    // in the widest, whose registers would spill more.
    constexpr bool kAhead = C < 4;
    const int64_t stride = (int64_t)gridDim.x * groups;
    Row next = read((int64_t)blockIdx.x * groups + group);
    for (int64_t row0 = (int64_t)blockIdx.x * groups; row0 < a.R; row0 += stride) {
        const int64_t row = row0 + group;
        const int64_t base = row * a.F;
        const float rs = next.rs, ry = next.ry;
        float s[C][V], b[C][V], t[C][V], g[C][V], e[C][V];
        int left[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
            left[c] = row < a.R ? a.F - (c * L + lane) * V : 0;
            next.x[c].get(s[c]);
            next.y[c].get(b[c]);
            next.gate[c].get(g[c]);
            next.dh[c].get(e[c]);
            next.ds[c].get(t[c]);
        }
        if (kAhead && row0 + stride < a.R) next = read(row + stride);
        float sums[3] = {0.f, 0.f, 0.f};      // dh w s, t z, s z
#pragma unroll
        for (int c = 0; c < C; c++) {
            const Small k = kKeep ? kept[c] : small(c);
            if (gate) {      // never without a block
#pragma unroll
                for (int i = 0; i < V; i++) g[c][i] = sigmoids(g[c][i]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) g[c][i] = 0.f;      // open: 1
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float z = BLOCK ? k.scale[i] * open_of(g[c][i]) * k.post[i] * (b[c][i] * ry) : 0.f;
                if (BLOCK) s[c][i] += z;
                const float hw = e[c][i] * k.w[i];
                t[c][i] += rs * hw;
                sums[0] += hw * s[c][i];
                if (BLOCK) {
                    sums[1] += t[c][i] * z;
                    sums[2] += s[c][i] * z;
                }
                sum_w[c][i] += e[c][i] * (s[c][i] * rs);
            }
        }
        if (BLOCK) row_sum<L>(sums, scratch);
        else row_sum<L>(reinterpret_cast<float(&)[1]>(sums), scratch);
        const float back = rs * (sums[0] * rs * over_f);
        const float back_y = post ? ry * ((sums[1] - back * (rs * sums[2])) * over_f) : 0.f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const Small k = kKeep ? kept[c] : small(c);
            const int f = (c * L + lane) * V;
            float dy[V], dg[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float dx = t[c][i] - (s[c][i] * rs) * back;
                t[c][i] = dx;
                if (!BLOCK) continue;
                const float u = b[c][i] * ry, xg = dx * open_of(g[c][i]), dv = xg * k.scale[i], up = u * k.post[i];
                dy[i] = ry * (dv * k.post[i]) - u * back_y;
                dg[i] = dv * up * shut_of(g[c][i]);
                sum_p[c][i] += dv * u;
                sum_s[c][i] += xg * up;
            }
            auto store = [&](auto whole) {
                constexpr bool W = decltype(whole)::value;
                if (a.dx) store_vec<W>(static_cast<T *>(a.dx) + base + f, left[c], t[c]);
                if (BLOCK && a.dy) store_vec<W>(static_cast<T *>(a.dy) + base + f, left[c], dy);
                if (BLOCK && a.dgate) store_vec<W>(static_cast<T *>(a.dgate) + base + f, left[c], dg);
            };
            if (WHOLE || even[c]) store(std::true_type());
            else store(std::false_type());
        }
        if (!kAhead && row0 + stride < a.R) next = read(row + stride);
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
    if (BLOCK && a.dpost) join(sum_p, 1);
    if (BLOCK && a.dscale) join(sum_s, 2);
}

// The workgroups' sums in order: a workgroup adds 32 columns, 32 strands of workgroups each.
// grid: x = columns / 32, y = the three sums
template <typename T> __global__ __launch_bounds__(1024) void norm_bwd_columns(NormGradArgs a, int blocks)
{
    __shared__ float strands[32][33];
    void *out = blockIdx.y == 0 ? a.dw : blockIdx.y == 1 ? a.dpost : a.dscale;
    if (!out) return;
    const int column = threadIdx.x & 31, strand = threadIdx.x >> 5;
    const int f = blockIdx.x * 32 + column;
    const float *part = a.part + (int64_t)blockIdx.y * blocks * a.F + f;
    float v = 0.f;
    if (f < a.F) {
#pragma unroll 8
        for (int b = strand; b < blocks; b += 32) v += part[(int64_t)b * a.F];
    }
    strands[strand][column] = v;
    __syncthreads();
    if (strand == 0 && f < a.F) {
#pragma unroll
        for (int k = 1; k < 32; k++) v += strands[k][column];
        static_cast<T *>(out)[f] = from_float<T>(v);
    }
}

// calls body(L, C) as compile-time constants: the narrowest lanes and vectors that cover a row
template <int V, typename Body> static void norm_shape(int F, Body &&body)
{
    const int v = (int)ceil_div(F, V);      // vectors of a row
    if (v <= 8) body(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    else if (v <= 16) body(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    else if (v <= 32) body(std::integral_constant<int, 32>(), std::integral_constant<int, 1>());
    else if (v <= 64) body(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    else if (v <= 128) body(std::integral_constant<int, 128>(), std::integral_constant<int, 1>());
    else if (v <= 256) body(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
    else if (v <= 512) body(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    else if (v <= 1024) body(std::integral_constant<int, 512>(), std::integral_constant<int, 2>());
    else if constexpr (kNormMaxWidth / V > 1024)
        body(std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
}
static int norm_grad_lanes(int F)
{
    int lanes = 0;
    norm_shape<kGradVec>(F, [&](auto l, auto) { lanes = l; });
    return lanes;
}
static int norm_blocks(int64_t R, int lanes, bool block)
{
    const int groups = lanes > 256 ? 1 : 256 / lanes;
    return (int)std::min<int64_t>(ceil_div(R, groups), block ? kNormBlocks : kNormBlocksAlone);
}

// three sums of kNormBlocks workgroups, or one (and two unused) of kNormBlocksAlone
static size_t norm_part_floats(int64_t R, int F) { return (size_t)3 * std::min<int64_t>(R, kNormBlocks) * F; }

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
        const dim3 grid = grid_of_blocks(ceil_div(R, threads / L));
        if (F % kVec<T> == 0) hipLaunchKernelGGL((norm_fwd<T, L, C, true>), grid, dim3(threads), 0, st, a);
        else hipLaunchKernelGGL((norm_fwd<T, L, C, false>), grid, dim3(threads), 0, st, a);
    };
    if (dtype == JGAMD_F32) norm_shape<kVec<float>>(F, [&](auto l, auto c) { launch(float(), l, c); });
    else norm_shape<kVec<bf16>>(F, [&](auto l, auto c) { launch(bf16(), l, c); });
    return launch_status("residual_norm_fwd");
}

JG_EXPORT int32_t jgamd_residual_norm_bwd_workspace(int64_t R, int32_t F, size_t *bytes)
{
    if (!bytes) return fail(JGAMD_ERR_NULL, "residual_norm_bwd_workspace: bytes is NULL");
    if (int32_t rc = norm_check("residual_norm_bwd_workspace", R, F, JGAMD_F32)) return rc;
    *bytes = carve_bytes(norm_part_floats(R, F), 4);
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
    const size_t need = columns ? carve_bytes(norm_part_floats(R, F), 4) : 0;
    if (need > 0 && (!ws || ws_bytes < need))
        return fail(JGAMD_ERR_WORKSPACE, "residual_norm_bwd: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
    if (need > 0 && ((uintptr_t)ws & 255) != 0)
        return fail(JGAMD_ERR_ALIGN, "residual_norm_bwd: workspace not 256-byte aligned");
    const NormGradArgs a{x, y, gate, scale, post, w, ry, rs, ds, dh, dx, dy, dgate, dscale, dpost, dw,
                         static_cast<float *>(ws), R, F};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int blocks = norm_blocks(R, norm_grad_lanes(F), y != nullptr);
    auto launch = [&](auto type, auto l, auto c) {
        using T = decltype(type);
        constexpr int L = decltype(l)::value, C = decltype(c)::value;
        const dim3 grid((unsigned)blocks), threads(norm_threads<L>());
        if (F % kGradVec == 0) {
            if (y) hipLaunchKernelGGL((norm_bwd<T, L, C, true, true>), grid, threads, 0, st, a);
            else hipLaunchKernelGGL((norm_bwd<T, L, C, true, false>), grid, threads, 0, st, a);
        } else {
            if (y) hipLaunchKernelGGL((norm_bwd<T, L, C, false, true>), grid, threads, 0, st, a);
            else hipLaunchKernelGGL((norm_bwd<T, L, C, false, false>), grid, threads, 0, st, a);
        }
    };
    if (blocks > 0) {
        if (dtype == JGAMD_F32) norm_shape<kGradVec>(F, [&](auto l, auto c) { launch(float(), l, c); });
        else norm_shape<kGradVec>(F, [&](auto l, auto c) { launch(bf16(), l, c); });
        if (int32_t rc = launch_status("residual_norm_bwd")) return rc;
    }
    if (!columns) return 0;
    const dim3 grid((unsigned)ceil_div(F, 32), 3);
    if (dtype == JGAMD_F32) hipLaunchKernelGGL((norm_bwd_columns<float>), grid, dim3(1024), 0, st, a, blocks);
    else hipLaunchKernelGGL((norm_bwd_columns<bf16>), grid, dim3(1024), 0, st, a, blocks);
    return launch_status("residual_norm_bwd");
}
