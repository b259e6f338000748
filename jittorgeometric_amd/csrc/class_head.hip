// Softmax cross entropy of z = x w^T + b over many classes, and its gradients, without the [V,C]
// matrix of logits:
//
//     lse[i] = log sum_c exp(z[i,c]),   loss[i] = lse[i] - z[i,label[i]]     (0 without a label in [0,C))
//     d[i,c] = g[i] (exp(z[i,c] - lse[i]) - [c == label[i]]),   dx = d w,   dw = d^T x,   db = sum_i d
//
// Forward: a workgroup keeps BM rows and walks a range of class tiles.  A lane holds four
// consecutive classes of one row, so the running maximum and sum of exponentials of a row are two
// registers of a lane; lanes, wavefronts and ranges are joined at the end, in a fixed order.
//
// Backward: z is computed again, tile by tile, and d is written for a block of rows and a piece of
// the classes (at most kPieceElements numbers, in the type of x); two products take it from there.
// dx sums over the pieces and dw over the blocks of rows in fp32 (a workspace where several take
// part), rounded once at the end.  Four products instead of the three of a loss that keeps its
// logits.  d in bfloat16 is off by 2^-9 of itself, like any gradient of logits of that type.
//
// Bound by the matrix units from some hundred rows on, by reading w below that.
#include <algorithm>

#include "tile_product.h"

namespace jg {

constexpr int kHeadMaxFeatures = 1 << 20;
constexpr int64_t kPieceElements = (int64_t)1 << 27;
constexpr int kBlockRows = 16384;      // rows of a block of the backward pass
constexpr int kJoinThreads = 256;

struct HeadArgs {
    const void *x, *w, *bias;
    const int32_t *y32;
    const int64_t *y64;
    int64_t V;
    int F, C;
};

__device__ __forceinline__ int64_t head_label(const HeadArgs &a, int64_t row)
{
    const int64_t y = a.y64 ? a.y64[row] : (int64_t)a.y32[row];
    return y >= 0 && y < a.C ? y : -1;
}

// (m, s): s exponentials relative to m.  An m of -inf holds nothing (s = 0).
__device__ __forceinline__ void join_stats(float &m, float &s, float m2, float s2)
{
    const float top = fmaxf(m, m2);
    const float ref = top == -INFINITY ? 0.f : top;
    s = s * __expf(m - ref) + s2 * __expf(m2 - ref);
    m = top;
}

// bias of classes n .. n + 3, zero past the last
template <typename T> __device__ __forceinline__ f32x4 bias4(const void *bias, int n, int C)
{
    f32x4 b = {0.f, 0.f, 0.f, 0.f};
    if (bias) {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (n + r < C) b[r] = to_float(static_cast<const T *>(bias)[n + r]);
    }
    return b;
}

// grid: x = blocks of BM rows x ranges of class tiles, ranges fastest.  stats [ranges][V]
template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void head_stats(HeadArgs a, int ranges, int tiles_per_range,
                                                          float2 *__restrict__ stats, float *__restrict__ at_label)
{
    using Product = TileProduct<T, S, kAlongK, kAlongK>;
    __shared__ __align__(16) char lds[Product::kLds];
    __shared__ float2 joined[S::WN][S::BM];
    const int range = blockIdx.x % ranges;
    const int64_t row0 = (int64_t)(blockIdx.x / ranges) * S::BM;
    const int rows = (int)min((int64_t)S::BM, a.V - row0);
    const Operand<T> q{static_cast<const T *>(a.x) + row0 * a.F, a.F, rows};
    float m[S::FM], s[S::FM];
    int label[S::FM];
#pragma unroll
    for (int j = 0; j < S::FM; j++) {
        m[j] = -INFINITY;
        s[j] = 0.f;
        label[j] = m_of<S>(j) < rows ? (int)head_label(a, row0 + m_of<S>(j)) : -1;
    }
    const int tiles = (a.C + S::BN - 1) / S::BN;
    const int last = min(tiles, (range + 1) * tiles_per_range);
    for (int tile = range * tiles_per_range; tile < last; tile++) {
        const int c0 = tile * S::BN;
        f32x4 acc[S::FN][S::FM];
#pragma unroll
        for (int i = 0; i < S::FN; i++) {
            const f32x4 b = bias4<T>(a.bias, c0 + n_of<S>(i), a.C);
#pragma unroll
            for (int j = 0; j < S::FM; j++) acc[i][j] = b;
        }
        const Operand<T> p{static_cast<const T *>(a.w) + (int64_t)c0 * a.F, a.F, a.C - c0};
        Product::run(acc, p, q, 0, a.F, lds);
        if (c0 + S::BN > a.C) {      // classes past the last count as -inf
#pragma unroll
            for (int i = 0; i < S::FN; i++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (c0 + n_of<S>(i) + r >= a.C)
#pragma unroll
                        for (int j = 0; j < S::FM; j++) acc[i][j][r] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < S::FM; j++) {
            float top = m[j];
#pragma unroll
            for (int i = 0; i < S::FN; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) top = fmaxf(top, acc[i][j][r]);
            const float ref = top == -INFINITY ? 0.f : top;
            float sum = s[j] * __expf(m[j] - ref);
#pragma unroll
            for (int i = 0; i < S::FN; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) sum += __expf(acc[i][j][r] - ref);
            m[j] = top;
            s[j] = sum;
            // the one lane that holds the label's logit hands it on
            const int at = label[j] - c0;
#pragma unroll
            for (int i = 0; i < S::FN; i++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (at == n_of<S>(i) + r) at_label[row0 + m_of<S>(j)] = acc[i][j][r];
        }
    }
    // the four lanes of a row, then the wavefronts beside each other
#pragma unroll
    for (int j = 0; j < S::FM; j++) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m[j], o, kWave), s2 = __shfl_xor(s[j], o, kWave);
            join_stats(m[j], s[j], m2, s2);
        }
        if (lane_id() < 16) joined[wave_in_block() / S::WM][m_of<S>(j)] = float2{m[j], s[j]};
    }
    __syncthreads();
    for (int r = threadIdx.x; r < rows; r += S::kThreads) {
        float2 v = joined[0][r];
#pragma unroll
        for (int k = 1; k < S::WN; k++) join_stats(v.x, v.y, joined[k][r].x, joined[k][r].y);
        stats[(int64_t)range * a.V + row0 + r] = v;
    }
}

// a row's ranges joined: lse, loss; and the workgroup's sum of losses and number of labels
__global__ __launch_bounds__(kJoinThreads) void head_rows(HeadArgs a, int ranges, const float2 *__restrict__ stats,
                                                          const float *__restrict__ at_label, float *__restrict__ lse,
                                                          float *__restrict__ row_loss, double *__restrict__ block_sum,
                                                          int32_t *__restrict__ block_count)
{
    __shared__ double s_sum[kJoinThreads / kWave];
    __shared__ int s_count[kJoinThreads / kWave];
    const int64_t row = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x;
    double loss = 0.0;
    int count = 0;
    if (row < a.V) {
        float m = -INFINITY, s = 0.f;
        for (int k = 0; k < ranges; k++) {
            const float2 v = stats[(int64_t)k * a.V + row];
            join_stats(m, s, v.x, v.y);
        }
        const float l = m + logf(s);
        lse[row] = l;
        const bool counted = head_label(a, row) >= 0;
        const float v = counted ? l - at_label[row] : 0.f;
        if (row_loss) row_loss[row] = v;
        loss = (double)v;
        count = counted ? 1 : 0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        loss += __shfl_xor(loss, o, kWave);
        count += __shfl_xor(count, o, kWave);
    }
    if (lane_id() == 0) {
        s_sum[wave_in_block()] = loss;
        s_count[wave_in_block()] = count;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kJoinThreads / kWave; k++) {
            loss += s_sum[k];
            count += s_count[k];
        }
        block_sum[blockIdx.x] = loss;
        block_count[blockIdx.x] = count;
    }
}

// loss[0] = sum (/ count), count[0] = rows with a label; one workgroup, fixed order
__global__ __launch_bounds__(kJoinThreads) void head_total(const double *__restrict__ block_sum,
                                                           const int32_t *__restrict__ block_count, int blocks, int mean,
                                                           float *__restrict__ loss, int32_t *__restrict__ count)
{
    __shared__ double s_sum[kJoinThreads];
    __shared__ long long s_count[kJoinThreads];
    double t = 0.0;
    long long n = 0;
    for (int b = threadIdx.x; b < blocks; b += kJoinThreads) {
        t += block_sum[b];
        n += block_count[b];
    }
    s_sum[threadIdx.x] = t;
    s_count[threadIdx.x] = n;
    __syncthreads();
    for (int half = kJoinThreads / 2; half > 0; half >>= 1) {
        if ((int)threadIdx.x < half) {
            s_sum[threadIdx.x] += s_sum[threadIdx.x + half];
            s_count[threadIdx.x] += s_count[threadIdx.x + half];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (loss) loss[0] = (float)(mean ? s_sum[0] / (double)s_count[0] : s_sum[0]);
        count[0] = (int32_t)min(s_count[0], 0x7fffffffLL);
    }
}

struct PieceArgs {
    HeadArgs head;             // of the whole problem
    const float *lse, *grad;   // [V]; [1], or [V] with per_row
    const int32_t *count;      // NULL: not a mean
    int per_row;
    int64_t row0;              // the block of rows and the piece of classes
    int rows, c0, classes;
    void *d;                   // [rows][ld]
    int64_t ld;
};

// d for a block of rows and a piece of classes.  grid: x = tiles, those of one block of rows together
template <typename T, typename S> __global__ __launch_bounds__(S::kThreads) void head_piece(PieceArgs a)
{
    using Product = TileProduct<T, S, kAlongK, kAlongK>;
    __shared__ __align__(16) char lds[Product::kLds];
    const int ctiles = (a.classes + S::BN - 1) / S::BN;
    const int n0 = (blockIdx.x % ctiles) * S::BN, m0 = (blockIdx.x / ctiles) * S::BM;
    const int F = a.head.F;
    f32x4 acc[S::FN][S::FM];
#pragma unroll
    for (int i = 0; i < S::FN; i++) {
        const f32x4 b = bias4<T>(a.head.bias, a.c0 + n0 + n_of<S>(i), a.head.C);
#pragma unroll
        for (int j = 0; j < S::FM; j++) acc[i][j] = b;
    }
    const Operand<T> p{static_cast<const T *>(a.head.w) + (int64_t)(a.c0 + n0) * F, F, a.classes - n0};
    const Operand<T> q{static_cast<const T *>(a.head.x) + (a.row0 + m0) * F, F, a.rows - m0};
    Product::run(acc, p, q, 0, F, lds);
    const float all = a.per_row ? 0.f : a.grad[0] / (a.count ? (float)a.count[0] : 1.f);
#pragma unroll
    for (int j = 0; j < S::FM; j++) {
        const int m = m0 + m_of<S>(j);
        if (m >= a.rows) continue;
        const int64_t row = a.row0 + m;
        const int64_t label = head_label(a.head, row);
        const float g = a.per_row ? a.grad[row] : all, l = a.lse[row];
#pragma unroll
        for (int i = 0; i < S::FN; i++) {
            const int n = n0 + n_of<S>(i);
            if (n >= a.classes) continue;
            f32x4 d;
#pragma unroll
            for (int r = 0; r < 4; r++)
                d[r] = label < 0 ? 0.f : g * (__expf(acc[i][j][r] - l) - (a.c0 + n + r == label ? 1.f : 0.f));
            store4<T>(static_cast<T *>(a.d) + m * a.ld + n, d, a.classes - n, true);
        }
    }
}

// out[m][n] = (first ? 0 : acc[m][n]) + sum_k P[n][k] Q[m][k], to `out` when `last`, else to `acc`; with
// several splits of k every split leaves its sum in part and head_join finishes.
struct SumArgs {
    const void *p, *q;
    int64_t ldp, ldq;
    int N, M, K, splits, k_split;
    void *out;          // [M][N]
    float *acc, *part;  // [M][N], [splits][M][N]
    void *out_b;        // sums of Q over k, [M]; the same three arrays for them, NULL: not wanted
    float *acc_b, *part_b;
    int first, last;
    int whole;          // four neighbouring values lie on an address that one access can take
};

template <typename T> __device__ __forceinline__ void finish4(const SumArgs &a, void *out, float *acc, int64_t at, f32x4 v, int n)
{
    if (!a.first) {
        if (a.whole && n >= 4) v += *reinterpret_cast<const f32x4 *>(acc + at);
        else {
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (r < n) v[r] += acc[at + r];
        }
    }
    if (a.last) store4<T>(static_cast<T *>(out) + at, v, n, a.whole);
    else store4<float>(acc + at, v, n, a.whole);
}

// grid: x = tiles x splits, the tiles of one split together
template <typename T, typename S, Layout PL, Layout QL> __global__ __launch_bounds__(S::kThreads) void head_sum(SumArgs a)
{
    using Product = TileProduct<T, S, PL, QL>;
    __shared__ __align__(16) char lds[Product::kLds];
    const int ntiles = (a.N + S::BN - 1) / S::BN, mtiles = (a.M + S::BM - 1) / S::BM;
    const int tile = blockIdx.x % (ntiles * mtiles), split = blockIdx.x / (ntiles * mtiles);
    const int n0 = (tile % ntiles) * S::BN, m0 = (tile / ntiles) * S::BM;
    f32x4 acc[S::FN][S::FM], sums[S::FM];
#pragma unroll
    for (int j = 0; j < S::FM; j++) {
        sums[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < S::FN; i++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const T *pb = static_cast<const T *>(a.p), *qb = static_cast<const T *>(a.q);
    const Operand<T> p{PL == kAlongK ? pb + n0 * a.ldp : pb + n0, a.ldp, a.N - n0};
    const Operand<T> q{QL == kAlongK ? qb + m0 * a.ldq : qb + m0, a.ldq, a.M - m0};
    const int k0 = split * a.k_split, k1 = min(a.K, k0 + a.k_split);
    const bool with_sums = a.out_b && n0 == 0;
    if (with_sums) Product::template run<kSumQ>(acc, p, q, k0, k1, lds, sums);
    else Product::run(acc, p, q, k0, k1, lds);
#pragma unroll
    for (int j = 0; j < S::FM; j++) {
        const int m = m0 + m_of<S>(j);
        if (m >= a.M) continue;
        if (with_sums && n_of<S>(0) == 0) {
            if (a.splits > 1) a.part_b[(int64_t)split * a.M + m] = sums[j][0];
            else finish4<T>(a, a.out_b, a.acc_b, m, sums[j], 1);
        }
#pragma unroll
        for (int i = 0; i < S::FN; i++) {
            const int n = n0 + n_of<S>(i);
            if (n >= a.N) continue;
            const int64_t at = (int64_t)m * a.N + n;
            if (a.splits > 1) store4<float>(a.part + (int64_t)split * a.M * a.N + at, acc[i][j], a.N - n, a.whole);
            else finish4<T>(a, a.out, a.acc, at, acc[i][j], a.N - n);
        }
    }
}

// grid: x = results / 1024 (of [M][N], then of [M])
template <typename T> __global__ __launch_bounds__(256) void head_join(SumArgs a)
{
    const int64_t size = (int64_t)a.M * a.N, all = size + (a.out_b ? a.M : 0);
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int64_t e = (int64_t)blockIdx.x * 1024 + u * 256 + threadIdx.x;
        if (e >= all) return;
        const bool b = e >= size;
        const int64_t at = b ? e - size : e, stride = b ? a.M : size;
        const float *part = b ? a.part_b : a.part;
        float *acc = b ? a.acc_b : a.acc;
        float v = a.first ? 0.f : acc[at];
        for (int k = 0; k < a.splits; k++) v += part[k * stride + at];
        if (a.last) static_cast<T *>(b ? a.out_b : a.out)[at] = from_float<T>(v);
        else acc[at] = v;
    }
}

template <typename T> using HeadShape = Shape<T, 128, 128, 2, 2>;
constexpr int kHeadTile = 128;

// ranges of class tiles: enough workgroups for the chip, several tiles each where there are many
static int head_ranges(int64_t V, int C)
{
    const int64_t tiles = ceil_div(C, kHeadTile), blocks = std::max<int64_t>(1, ceil_div(V, kHeadTile));
    const int64_t ranges = std::min<int64_t>(tiles, std::max<int64_t>(1, ceil_div(1024, blocks)));
    return (int)ceil_div(tiles, ceil_div(tiles, ranges));
}

// splits of a sum over K for an [M][N] result: about four workgroups a compute unit, at least 512 steps each
static int sum_splits(int64_t M, int64_t N, int64_t K)
{
    const int64_t tiles = ceil_div(M, kHeadTile) * ceil_div(N, kHeadTile);
    return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(768, tiles), K / 512));
}

struct Pieces {
    int64_t rows, blocks;      // rows of a block, blocks
    int64_t classes, pieces;   // classes of a piece (whole tiles), pieces
};
static Pieces head_pieces(int64_t V, int C)
{
    Pieces s;
    s.rows = std::min<int64_t>(std::max<int64_t>(V, 1), kBlockRows);
    s.blocks = std::max<int64_t>(1, ceil_div(V, s.rows));
    s.classes = std::max<int64_t>(kHeadTile, kPieceElements / s.rows / kHeadTile * kHeadTile);
    s.classes = std::min<int64_t>(s.classes, ceil_div(C, kHeadTile) * kHeadTile);
    s.pieces = ceil_div(C, s.classes);
    return s;
}

// the workspace of the backward pass, in the order it is carved
struct HeadScratch {
    size_t d, part, part_b, acc_x, acc_w, acc_b;      // floats (d: bytes)
    size_t bytes() const
    {
        return carve_bytes(d, 1) + carve_bytes(part, 4) + carve_bytes(part_b, 4) + carve_bytes(acc_x, 4) +
               carve_bytes(acc_w, 4) + carve_bytes(acc_b, 4);
    }
};
static HeadScratch head_scratch(int64_t V, int F, int C, int32_t dtype)
{
    const Pieces s = head_pieces(V, C);
    HeadScratch n{};
    n.d = (size_t)(s.rows * s.classes) * (dtype == JGAMD_F32 ? 4 : 2);
    const int64_t sx = sum_splits(s.rows, F, s.classes), sw = sum_splits(s.classes, F, s.rows);
    n.part = (size_t)std::max(sx > 1 ? sx * s.rows * F : 0, sw > 1 ? sw * s.classes * F : 0);
    n.part_b = (size_t)(sw > 1 ? sw * s.classes : 0);
    n.acc_x = s.pieces > 1 ? (size_t)s.rows * F : 0;
    n.acc_w = s.blocks > 1 ? (size_t)C * F : 0;
    n.acc_b = s.blocks > 1 ? (size_t)C : 0;
    return n;
}

static int32_t head_check(const char *who, int64_t V, int32_t F, int32_t C, int32_t dtype, int32_t reduction)
{
    if (V < 0 || F <= 0 || C <= 0)
        return fail(JGAMD_ERR_SIZE, "%s: V=%lld F=%d C=%d (V >= 0, the others positive)", who, (long long)V, F, C);
    if (V > 0x7fffffffLL || F > kHeadMaxFeatures || C > 0x7fffff00)
        return fail(JGAMD_ERR_SIZE, "%s: V=%lld F=%d C=%d is too large", who, (long long)V, F, C);
    if (dtype != JGAMD_F32 && dtype != JGAMD_BF16) return fail(JGAMD_ERR_UNSUPPORTED, "%s: unknown dtype %d", who, dtype);
    if (reduction < 0 || reduction > JGAMD_LOSS_SUM) return fail(JGAMD_ERR_SIZE, "%s: unknown reduction %d", who, reduction);
    return 0;
}
static bool head_off_element(int32_t dtype, const void *a, const void *b, const void *c)
{
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & (dtype == JGAMD_F32 ? 3 : 1)) != 0;
}

template <typename T, Layout PL, Layout QL> static int32_t launch_sum(SumArgs a, hipStream_t s)
{
    using S = HeadShape<T>;
    const int64_t blocks = ceil_div(a.N, S::BN) * ceil_div(a.M, S::BM) * a.splits;
    if (blocks > 0x7fffffffLL) return fail(JGAMD_ERR_SIZE, "linear_cross_entropy: F=%d is too large", a.N);
    hipLaunchKernelGGL((head_sum<T, S, PL, QL>), dim3((unsigned)blocks), dim3(S::kThreads), 0, s, a);
    if (a.splits > 1) {
        const int64_t all = (int64_t)a.M * a.N + (a.out_b ? a.M : 0);
        hipLaunchKernelGGL((head_join<T>), dim3((unsigned)ceil_div(all, 1024)), dim3(256), 0, s, a);
    }
    return launch_status("linear_cross_entropy_bwd");
}

template <typename T>
static int32_t head_backward(const HeadArgs &h, const float *lse, const int32_t *count, const float *grad, int32_t reduction,
                             T *dx, T *dw, T *db, void *ws, int32_t dtype, hipStream_t st)
{
    using S = HeadShape<T>;
    const Pieces s = head_pieces(h.V, h.C);
    const HeadScratch n = head_scratch(h.V, h.F, h.C, dtype);
    Carver carve(ws);
    T *d = reinterpret_cast<T *>(carve.take<char>(n.d));
    float *part = carve.take<float>(n.part), *part_b = carve.take<float>(n.part_b);
    float *acc_x = carve.take<float>(n.acc_x), *acc_w = carve.take<float>(n.acc_w), *acc_b = carve.take<float>(n.acc_b);
    auto whole = [](int N, const void *p) { return N % 4 == 0 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0; };
    for (int64_t b = 0; b < s.blocks; b++) {
        const int64_t row0 = b * s.rows;
        const int rows = (int)std::min<int64_t>(s.rows, h.V - row0);
        const T *x = static_cast<const T *>(h.x) + row0 * h.F;
        for (int64_t c = 0; c < s.pieces; c++) {
            const int c0 = (int)(c * s.classes), classes = (int)std::min<int64_t>(s.classes, h.C - c0);
            if (rows > 0) {
                const PieceArgs a{h, lse, grad, reduction == JGAMD_LOSS_MEAN ? count : nullptr,
                                  reduction == JGAMD_LOSS_NONE, row0, rows, c0, classes, d, s.classes};
                const int64_t blocks = ceil_div(classes, S::BN) * ceil_div(rows, S::BM);
                hipLaunchKernelGGL((head_piece<T, S>), dim3((unsigned)blocks), dim3(S::kThreads), 0, st, a);
                if (int32_t rc = launch_status("linear_cross_entropy_bwd")) return rc;
            }
            const T *w = static_cast<const T *>(h.w) + (int64_t)c0 * h.F;
            if (dx && rows > 0) {
                SumArgs a{};
                a.p = w, a.ldp = h.F, a.q = d, a.ldq = s.classes;
                a.N = h.F, a.M = rows, a.K = classes;
                a.splits = sum_splits(s.rows, h.F, s.classes);
                a.k_split = (int)(ceil_div(ceil_div(s.classes, a.splits), 64) * 64);
                a.out = dx + row0 * h.F, a.acc = acc_x, a.part = part;
                a.first = c == 0, a.last = c == s.pieces - 1, a.whole = whole(h.F, a.out);
                if (int32_t rc = launch_sum<T, kAcrossK, kAlongK>(a, st)) return rc;
            }
            if (dw || db) {
                SumArgs a{};
                a.p = x, a.ldp = h.F, a.q = d, a.ldq = s.classes;
                a.N = h.F, a.M = classes, a.K = rows;
                a.splits = sum_splits(s.classes, h.F, s.rows);
                a.k_split = (int)(ceil_div(ceil_div(s.rows, a.splits), 64) * 64);
                a.out = dw + (int64_t)c0 * h.F, a.acc = acc_w + (s.blocks > 1 ? (int64_t)c0 * h.F : 0), a.part = part;
                a.out_b = db ? db + c0 : nullptr, a.acc_b = acc_b + (s.blocks > 1 ? c0 : 0), a.part_b = part_b;
                a.first = b == 0, a.last = b == s.blocks - 1, a.whole = whole(h.F, a.out);
                if (int32_t rc = launch_sum<T, kAcrossK, kAcrossK>(a, st)) return rc;
            }
        }
    }
    return 0;
}

}  // namespace jg

using namespace jg;
#define JG_EXPORT extern "C" __attribute__((visibility("default")))

static size_t head_fwd_bytes(int64_t V, int32_t C)
{
    const size_t blocks = (size_t)ceil_div(V, kJoinThreads);
    return carve_bytes((size_t)head_ranges(V, C) * V, 8) + carve_bytes((size_t)V, 4) + carve_bytes(blocks, 8) +
           carve_bytes(blocks, 4);
}

JG_EXPORT int32_t jgamd_linear_cross_entropy_workspace(int64_t V, int32_t F, int32_t C, int32_t dtype, int32_t backward,
                                                       size_t *bytes)
{
    if (!bytes) return fail(JGAMD_ERR_NULL, "linear_cross_entropy_workspace: bytes is NULL");
    if (int32_t rc = head_check("linear_cross_entropy_workspace", V, F, C, dtype, 0)) return rc;
    *bytes = backward ? head_scratch(V, F, C, dtype).bytes() : head_fwd_bytes(V, C);
    return 0;
}

JG_EXPORT int32_t jgamd_linear_cross_entropy_fwd(const void *x, const void *w, const void *bias, const void *labels,
                                                 int32_t labels_are_i64, int64_t V, int32_t F, int32_t C, int32_t dtype,
                                                 int32_t reduction, float *loss, int32_t *count, float *lse, void *ws,
                                                 size_t ws_bytes, void *stream)
{
    if (int32_t rc = head_check("linear_cross_entropy_fwd", V, F, C, dtype, reduction)) return rc;
    if (!count || (reduction != JGAMD_LOSS_NONE && !loss))
        return fail(JGAMD_ERR_NULL, "linear_cross_entropy_fwd: loss / count is NULL");
    if (V > 0 && (!x || !w || !labels || !lse || !loss)) return fail(JGAMD_ERR_NULL, "linear_cross_entropy_fwd: NULL array");
    if (head_off_element(dtype, x, w, bias) || ((uintptr_t)labels & (labels_are_i64 ? 7 : 3)) != 0 ||
        (((uintptr_t)loss | (uintptr_t)count | (uintptr_t)lse) & 3) != 0)
        return fail(JGAMD_ERR_ALIGN, "linear_cross_entropy_fwd: an array does not start at a multiple of its element's size");
    const size_t need = head_fwd_bytes(V, C);
    if (need > 0 && (!ws || ws_bytes < need))
        return fail(JGAMD_ERR_WORKSPACE, "linear_cross_entropy_fwd: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
    if (need > 0 && ((uintptr_t)ws & 255) != 0)
        return fail(JGAMD_ERR_ALIGN, "linear_cross_entropy_fwd: workspace not 256-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int ranges = head_ranges(V, C), blocks = (int)ceil_div(V, kJoinThreads);
    const int per_range = (int)ceil_div(ceil_div(C, kHeadTile), ranges);
    Carver carve(ws);
    float2 *stats = carve.take<float2>((size_t)ranges * V);
    float *at_label = carve.take<float>((size_t)V);
    double *block_sum = carve.take<double>((size_t)blocks);
    int32_t *block_count = carve.take<int32_t>((size_t)blocks);
    const HeadArgs a{x, w, bias, labels_are_i64 ? nullptr : static_cast<const int32_t *>(labels),
                     labels_are_i64 ? static_cast<const int64_t *>(labels) : nullptr, V, F, C};
    if (V > 0) {
        const int64_t grid = ceil_div(V, kHeadTile) * ranges;
        if (grid > 0x7fffffffLL) return fail(JGAMD_ERR_SIZE, "linear_cross_entropy_fwd: V=%lld is too large", (long long)V);
        if (dtype == JGAMD_F32)
            hipLaunchKernelGGL((head_stats<float, HeadShape<float>>), dim3((unsigned)grid), dim3(HeadShape<float>::kThreads),
                               0, st, a, ranges, per_range, stats, at_label);
        else
            hipLaunchKernelGGL((head_stats<bf16, HeadShape<bf16>>), dim3((unsigned)grid), dim3(HeadShape<bf16>::kThreads), 0,
                               st, a, ranges, per_range, stats, at_label);
        hipLaunchKernelGGL(head_rows, dim3((unsigned)blocks), dim3(kJoinThreads), 0, st, a, ranges, stats, at_label, lse,
                           reduction == JGAMD_LOSS_NONE ? loss : nullptr, block_sum, block_count);
    }
    if (reduction != JGAMD_LOSS_NONE)
        hipLaunchKernelGGL(head_total, dim3(1), dim3(kJoinThreads), 0, st, block_sum, block_count, blocks,
                           reduction == JGAMD_LOSS_MEAN ? 1 : 0, loss, count);
    return launch_status("linear_cross_entropy_fwd");
}

JG_EXPORT int32_t jgamd_linear_cross_entropy_bwd(const void *x, const void *w, const void *bias, const void *labels,
                                                 int32_t labels_are_i64, const float *lse, const int32_t *count,
                                                 const float *grad, int64_t V, int32_t F, int32_t C, int32_t dtype,
                                                 int32_t reduction, void *dx, void *dw, void *db, void *ws,
                                                 size_t ws_bytes, void *stream)
{
    if (int32_t rc = head_check("linear_cross_entropy_bwd", V, F, C, dtype, reduction)) return rc;
    if (db && !dw) return fail(JGAMD_ERR_NULL, "linear_cross_entropy_bwd: db without dw");
    if (V > 0 && (!x || !w || !labels || !lse || !grad || (reduction == JGAMD_LOSS_MEAN && !count)))
        return fail(JGAMD_ERR_NULL, "linear_cross_entropy_bwd: NULL array");
    if (head_off_element(dtype, x, w, bias) || head_off_element(dtype, dx, dw, db) ||
        ((uintptr_t)labels & (labels_are_i64 ? 7 : 3)) != 0 || (((uintptr_t)lse | (uintptr_t)count | (uintptr_t)grad) & 3) != 0)
        return fail(JGAMD_ERR_ALIGN, "linear_cross_entropy_bwd: an array does not start at a multiple of its element's size");
    if (!dx && !dw) return 0;
    const size_t need = head_scratch(V, F, C, dtype).bytes();
    if (!ws || ws_bytes < need)
        return fail(JGAMD_ERR_WORKSPACE, "linear_cross_entropy_bwd: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
    if (((uintptr_t)ws & 255) != 0) return fail(JGAMD_ERR_ALIGN, "linear_cross_entropy_bwd: workspace not 256-byte aligned");
    const HeadArgs h{x, w, bias, labels_are_i64 ? nullptr : static_cast<const int32_t *>(labels),
                     labels_are_i64 ? static_cast<const int64_t *>(labels) : nullptr, V, F, C};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == JGAMD_F32)
        return head_backward<float>(h, lse, count, grad, reduction, static_cast<float *>(dx), static_cast<float *>(dw),
                                    static_cast<float *>(db), ws, dtype, st);
    return head_backward<bf16>(h, lse, count, grad, reduction, static_cast<bf16 *>(dx), static_cast<bf16 *>(dw),
                               static_cast<bf16 *>(db), ws, dtype, st);
}
