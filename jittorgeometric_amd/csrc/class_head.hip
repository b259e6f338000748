// Softmax cross entropy of z = x w^T + b over many classes, and its gradients, without the [V,C]
// matrix of logits:
//
//     lse[i] = log sum_c exp(z[i,c]),   loss[i] = lse[i] - z[i,label[i]]     (0 without a label in [0,C))
//     d[i,c] = exp(z[i,c] - lse[i]) - [c == label[i]]                        (0 without a label)
//     dx[i] = g[i] d[i] w,   dw = d^T (g x),   db = sum_i g[i] d[i]
//
// Forward: a workgroup keeps BM rows and walks a range of class tiles.  A lane holds four
// consecutive classes of one row in a fragment (32 of a tile of 256 x 256, in eights), so the running maximum
// and sum of exponentials of a row are two registers of a lane; lanes, wavefronts and ranges are joined at the
// end, in a fixed order.
//
// Backward: z is computed again, tile by tile, and d is written for a block of rows and a piece of
// the classes (at most kPieceBytes, in the type of x); two products take it from there.
// dx sums over the pieces and dw over the blocks of rows in fp32 (a workspace where several take
// part), rounded once at the end.  Four products instead of the three of a loss that keeps its
// logits.  d in bfloat16 is off by 2^-8 of itself, like any gradient of logits of that type; it is kept
// without g, since -1 is exact but g (1 / rows) rounded once for all rows would shift every result alike
// (16384 rows of 131072 classes: dw off by 3.1e-3 with g in d, 1.7e-3 without).  g multiplies the fp32
// sums where it is one number, and dx's rows and a copy of x where it is one a row (rounded to bfloat16 once
// more there: its roundings are as many as the entries and independent of each other).
//
// Bound by the matrix units from some hundred rows on, by reading w below that.
#include <algorithm>

#include "lds_size.h"
#include "stream_product.h"

namespace jg {

constexpr int kHeadMaxFeatures = 1 << 20;
// of d.  16384 rows, 512 features, 131072 classes, bfloat16: 9.7 ms with pieces of 512 MB, 9.4 with 1 GB
constexpr int64_t kPieceBytes = (int64_t)1 << 30;
constexpr int kBlockRows = 16384;      // rows of a block of the backward pass
constexpr int kJoinThreads = 256;
constexpr int kCus = 256;
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kPad = 128;      // classes between the rows of d: rows a power of two apart meet in one channel of the L2

// 256 x 256 results, eight wavefronts of 128 x 64, two stages of 64 KB: steps of 64.  Two workgroups a compute
// unit, one of which could multiply while the other takes exponentials, need narrower tiles and steps of 32,
// whose loads ask for 64 bytes of a row.  The statistics of 16384 rows, 512 features, 131072 classes in
// bfloat16: 2.43 ms; 256 x 256 with four stages of 32: 2.61; two workgroups of 256 x 128: 2.77, of 128 x 256:
// 2.52.  Floats in three parts: 256 x 128, two stages of 72 KB, steps of 32.
template <typename T> struct HeadShapeOf;
template <> struct HeadShapeOf<bf16> {
    using S = StreamShape<1, 256, 256, 2, 4, 64, 2>;
};
template <> struct HeadShapeOf<float> {
    using S = StreamShape<3, 256, 128, 4, 2, 32, 2>;
};
template <typename T> using HeadShape = typename HeadShapeOf<T>::S;
// tiles of a few rows, two workgroups a compute unit
template <typename T> struct HeadFewOf;
template <> struct HeadFewOf<bf16> {
    using S = StreamShape<1, 128, 32, 4, 1, 64, 4>;
};
template <> struct HeadFewOf<float> {
    using S = StreamShape<3, 128, 64, 4, 1, 32, 2>;
};
template <typename T> using HeadFew = typename HeadFewOf<T>::S;

// Floats enter as the three bfloat16 parts of tile_product.h, six products of them: every entry keeps its own
// 24 bits, and so does every entry of d, whatever the others of its row, its class or its array are.  Two
// float16 parts under one exponent an array take half the products (4099 rows, 256 features, 32003 classes,
// training: 1.05 instead of 1.61 ms) and lose them: a row 1e8 times the others moved the others' losses by 1e-3,
// and the gradients of classes of probability 1e-12 were off by 0.4 of themselves.
struct HeadArgs {
    const bf16 *x, *w;           // [V][ld], [C][ld] as parts (stream_product.h)
    int64_t part_x, part_w;
    int ld;                      // F rounded up to 8
    const void *bias;            // [C] of T, or NULL
    const int32_t *y32;
    const int64_t *y64;
    int64_t V;
    int F, C;
};

// the label of a row, -1 where it names no class
__device__ __forceinline__ int64_t label_in(const int32_t *y32, const int64_t *y64, int C, int64_t row)
{
    const int64_t y = y64 ? y64[row] : (int64_t)y32[row];
    return y >= 0 && y < C ? y : -1;
}
__device__ __forceinline__ int64_t head_label(const HeadArgs &a, int64_t row) { return label_in(a.y32, a.y64, a.C, row); }

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

// Order of the tiles of an M x N grid of tiles: runs of consecutive numbers cover blocks of up to 8 x 4
// tiles, and the workgroups of one XCD (every eighth) work on one run, so that the operands of a run
// are read into one L2 once.  `step` counts the tiles of workgroup blockIdx.x.
__device__ __forceinline__ void tile_at(int step, int mtiles, int ntiles, int *m, int *n, bool *exists)
{
    const int g = gridDim.x, b = blockIdx.x;
    const int64_t id = (int64_t)step * g + (g % 8 == 0 ? (b % 8) * (g / 8) + b / 8 : b);
    *exists = id < (int64_t)mtiles * ntiles;
    const int64_t group = id / ((int64_t)8 * ntiles);
    const int height = min(8, mtiles - (int)group * 8);
    const int in = (int)(id - group * 8 * ntiles);
    *m = (int)group * 8 + in % max(height, 1);
    *n = in / max(height, 1);
}
// how many tiles workgroup blockIdx.x has
__device__ __forceinline__ int tiles_of(int mtiles, int ntiles)
{
    const int g = gridDim.x, b = blockIdx.x;
    const int64_t all = (int64_t)mtiles * ntiles;
    const int64_t first = g % 8 == 0 ? (b % 8) * (g / 8) + b / 8 : b;
    return first < all ? (int)((all - 1 - first) / g + 1) : 0;
}

// eight neighbouring values as one or three bfloat16 parts, kept where `keep` has ones
template <int PARTS> __device__ __forceinline__ void store_parts8(bf16 *out, int64_t part, float (&v)[8], uint32_t keep)
{
#pragma unroll
    for (int s = 0; s < PARTS; s++) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            if (s + 1 < PARTS) {
                v[2 * i] -= bf16_lo(w[i]);
                v[2 * i + 1] -= bf16_hi(w[i]);
            }
            w[i] &= keep;
        }
        *reinterpret_cast<u32x4 *>(out + s * part) = w;
    }
}

// One array to be laid out as parts: [R][F] of T to [R][ld], zero behind F; rows times scale[R] unless
// that is NULL (a row times zero is zero whatever it holds), or, with `labelled`, zero without a label:
// what a padded row holds does not enter dW as 0 x NaN.
struct Copy {
    const void *src;
    const float *scale;
    int labelled;
    int64_t R;
    bf16 *dst;
    int64_t part;            // elements between the parts
};
struct Copies {
    Copy of[2];
    const int32_t *y32;
    const int64_t *y64;
    int blocks0, blocks;     // workgroups of the first; of both: the others have the second
    int F, ld, C;
};

// piece `id` of 8 entries of an array
template <typename T> __device__ __forceinline__ Eight<T> copy_piece(const Copies &a, const Copy &c, int64_t id)
{
    const int across = a.ld / 8;
    const int64_t row = id / across;
    const int at = (int)(id - row * across) * 8;
    Eight<T> e;
    const T *src = static_cast<const T *>(c.src) + row * a.F + at;
    if (at + 8 <= a.F) e.load(src);
    else e.load_some(src, a.F - at);
    if (c.scale) e.scale(c.scale[row]);
    if (c.labelled && label_in(a.y32, a.y64, a.C, row) < 0) e.clear();
    return e;
}

// grid: blocks0 + the second array's workgroups by block_number, 256 pieces of 8 each
template <typename T> __global__ __launch_bounds__(256) void head_parts(Copies a)
{
    const int64_t number = block_number();
    if (number >= a.blocks) return;
    const bool second = number >= a.blocks0;
    const Copy &c = a.of[second];
    const int64_t id = (number - (second ? a.blocks0 : 0)) * 256 + threadIdx.x;
    if (id >= c.R * (a.ld / 8)) return;
    const Eight<T> e = copy_piece<T>(a, c, id);
    if constexpr (sizeof(T) == 4) {
        float rest[8] = {e.a[0], e.a[1], e.a[2], e.a[3], e.b[0], e.b[1], e.b[2], e.b[3]};
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[i] = pack_bf16(finite(rest[2 * i]), finite(rest[2 * i + 1]));
            rest[2 * i] -= bf16_lo(w[i]);
            rest[2 * i + 1] -= bf16_hi(w[i]);
        }
        *reinterpret_cast<u32x4 *>(c.dst + id * 8) = w;
        store_parts8<2>(c.dst + id * 8 + c.part, c.part, rest, 0xffffffffu);
    } else *reinterpret_cast<u32x4 *>(c.dst + id * 8) = e.v;
}

// a tile's sums, of classes c0 and up, to logits
template <typename T, typename Product, typename S>
__device__ __forceinline__ void logits(f32x4 (&acc)[S::FN][S::FM], const HeadArgs &h, int c0)
{
    if (!h.bias) return;
#pragma unroll
    for (int i = 0; i < S::FN; i++) {
        const f32x4 b = bias4<T>(h.bias, c0 + Product::n_of(i), h.C);
#pragma unroll
        for (int j = 0; j < S::FM; j++) acc[i][j] += b;
    }
}

// grid: x = blocks of BM rows x ranges of class tiles.  stats [ranges][V]
template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads, 2) void head_stats(HeadArgs a, int ranges, int tiles_per_range,
                                                          float2 *__restrict__ stats, float *__restrict__ at_label)
{
    using Product = StreamProduct<S, kAlongK, kAlongK>;
    extern __shared__ __align__(16) char lds[];
    const int blocks = (int)((a.V + S::BM - 1) / S::BM);
    int block, range;
    bool exists;
    tile_at(0, blocks, ranges, &block, &range, &exists);
    if (!exists) return;
    const int64_t row0 = (int64_t)block * S::BM;
    const int rows = (int)min((int64_t)S::BM, a.V - row0);
    float m[S::FM], s[S::FM];
    int label[S::FM];
#pragma unroll
    for (int j = 0; j < S::FM; j++) {
        m[j] = -INFINITY;
        s[j] = 0.f;
        label[j] = Product::m_of(j) < rows ? (int)head_label(a, row0 + Product::m_of(j)) : -1;
    }
    const int tiles = (a.C + S::BN - 1) / S::BN;
    const int first = range * tiles_per_range;
    const bf16 *x = a.x + row0 * a.ld;
    Product::template run<kNoSums>(
        min(tiles, first + tiles_per_range) - first, lds,
        [&](int t) {
            const int c0 = (first + t) * S::BN;
            return StreamTile{a.w + (int64_t)c0 * a.ld, x, a.part_w, a.part_x, a.ld, a.ld, a.C - c0, rows, a.F};
        },
        [&](int t, f32x4(&acc)[S::FN][S::FM], f32x4 *) {
            const int c0 = (first + t) * S::BN;
            logits<T, Product, S>(acc, a, c0);
            if (c0 + S::BN > a.C) {      // classes past the last count as -inf
#pragma unroll
                for (int i = 0; i < S::FN; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (c0 + Product::n_of(i) + r >= a.C)
#pragma unroll
                            for (int j = 0; j < S::FM; j++) acc[i][j][r] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < S::FM; j++) {
                float top = m[j];
#pragma unroll
                for (int i = 0; i < S::FN; i++)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) top = fmaxf(fmaxf(top, acc[i][j][r]), acc[i][j][r + 1]);
                const float ref = top == -INFINITY ? 0.f : top;
                float sum = s[j] * __expf(m[j] - ref);
#pragma unroll
                for (int i = 0; i < S::FN; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) sum += __builtin_amdgcn_exp2f((acc[i][j][r] - ref) * kLog2e);
                m[j] = top;
                s[j] = sum;
                // the one lane that holds the label's logit hands it on
                const int at = label[j] - c0;
                if (at >= 0 && at < S::BN) {
#pragma unroll
                    for (int i = 0; i < S::FN; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (at == Product::n_of(i) + r) at_label[row0 + Product::m_of(j)] = acc[i][j][r];
                }
            }
        });
    // the four lanes of a row, then the wavefronts beside each other
    float2 *joined = reinterpret_cast<float2 *>(lds);      // [WN][BM]
#pragma unroll
    for (int j = 0; j < S::FM; j++) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m[j], o, kWave), s2 = __shfl_xor(s[j], o, kWave);
            join_stats(m[j], s[j], m2, s2);
        }
        if (lane_id() < 16) joined[(wave_in_block() / S::WM) * S::BM + Product::m_of(j)] = float2{m[j], s[j]};
    }
    __syncthreads();
    for (int r = threadIdx.x; r < rows; r += S::kThreads) {
        float2 v = joined[r];
#pragma unroll
        for (int k = 1; k < S::WN; k++) join_stats(v.x, v.y, joined[k * S::BM + r].x, joined[k * S::BM + r].y);
        stats[(int64_t)range * a.V + row0 + r] = v;
    }
}

// The statistics of a few rows of floats: w is read once, as it is, and multiplied on the vector unit, instead of
// being laid out as parts for it.  kThinRows rows of x stand in LDS; sixteen lanes share four classes, 4 k a lane
// and step.  The 32 sums of a group meet in a transposing reduction (16 + 8 + 4 + 2 shuffles) that leaves each
// lane one class of two rows, whose running maximum and sum it keeps.  Bound by reading w for up to kThinRows
// rows, by the vector unit beyond.  Whole calls, with parts and like this: 4 rows, 387 features, 48749 classes 66
// and 26 us; 256 features, 50021 classes: 7 rows 48 and 24, 24 rows 47 and 45, 32 rows 48 and 46, 48 rows 49 and 65;
// 2000 features, 20000 classes, 32 rows: 193 and 157.  (bfloat16 of odd widths, copied once: 8 rows 23 and 27, 32 rows
// 23 and 46.)
// grid: x = blocks of kThinRows rows x ranges of tiles of 64 classes
constexpr int kThinRows = 8;
constexpr int kThinMost = 32;            // rows of a call, at most
constexpr int kThinFeatures = 2048;      // 64 KB of x
constexpr int kThinClasses = 64;

// the first n (at most four, at least none) of p, zero behind them
__device__ __forceinline__ f32x4 four(const float *p, int n)
{
    if (n >= 4) return *reinterpret_cast<const f32x4_at4 *>(p);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 3; i++)
        if (i < n) v[i] = p[i];
    return v;
}

__global__ __launch_bounds__(256, 3) void head_thin(HeadArgs a, const float *__restrict__ x, const float *__restrict__ w,
                                                    int ranges, int tiles_per_range, float2 *__restrict__ stats,
                                                    float *__restrict__ at_label)
{
    extern __shared__ __align__(16) float xs[];      // [kThinRows][across]
    __shared__ float2 joined[4][kThinRows];
    const int across = (a.F + 63) / 64 * 64;
    const int64_t row0 = (int64_t)(blockIdx.x / ranges) * kThinRows;
    const int range = blockIdx.x % ranges, rows = (int)min((int64_t)kThinRows, a.V - row0);
    for (int i = threadIdx.x; i < kThinRows * across; i += 256) {
        const int r = i / across, k = i - r * across;
        xs[i] = r < rows && k < a.F ? x[(row0 + r) * a.F + k] : 0.f;
    }
    __syncthreads();
    const int lane = lane_id() & 15, group = wave_in_block() * 4 + (lane_id() >> 4);
    const int r0 = ((lane >> 1) & 1) * 4 + (lane & 1) * 2;      // this lane's rows, r0 and r0 + 1
    int label[2];
    float m[2] = {-INFINITY, -INFINITY}, s[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; u++) label[u] = r0 + u < rows ? (int)head_label(a, row0 + r0 + u) : -1;
    const int tiles = (a.C + kThinClasses - 1) / kThinClasses;
    const int last = min(tiles, (range + 1) * tiles_per_range);
    for (int t = range * tiles_per_range; t < last; t++) {
        const int c0 = t * kThinClasses + group * 4;
        const float *from[4];
#pragma unroll
        for (int c = 0; c < 4; c++) from[c] = w + (int64_t)min(c0 + c, a.C - 1) * a.F;
        float acc[4 * kThinRows] = {};
#pragma unroll 2
        for (int k = lane * 4; k < across; k += 64) {
            f32x4 wv[4];
#pragma unroll
            for (int c = 0; c < 4; c++) wv[c] = four(from[c] + k, a.F - k);
#pragma unroll
            for (int r = 0; r < kThinRows; r++) {
                const f32x4 xv = *reinterpret_cast<const f32x4 *>(xs + r * across + k);
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[c * kThinRows + r] = fmaf(wv[c][i], xv[i], acc[c * kThinRows + r]);
            }
        }
        // class bits 1 and 0, row bits 2 and 1 go to lane bits 3, 2, 1, 0
        auto fold = [&](auto lane_bit) {
            constexpr int bit = decltype(lane_bit)::value, half = bit * kThinRows / 4;
            const bool high = (lane & bit) != 0;
#pragma unroll
            for (int i = 0; i < half; i++) {
                const float give = high ? acc[i] : acc[i + half], keep = high ? acc[i + half] : acc[i];
                acc[i] = keep + __shfl_xor(give, bit, kWave);
            }
        };
        fold(std::integral_constant<int, 8>());
        fold(std::integral_constant<int, 4>());
        fold(std::integral_constant<int, 2>());
        fold(std::integral_constant<int, 1>());
        const int cls = c0 + (lane >> 2);
        const float b = a.bias && cls < a.C ? static_cast<const float *>(a.bias)[cls] : 0.f;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const float z = cls < a.C ? acc[u] + b : -INFINITY;
            if (label[u] == cls) at_label[row0 + r0 + u] = z;
            join_stats(m[u], s[u], z, cls < a.C ? 1.f : 0.f);
        }
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int o = 4; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m[u], o, kWave), s2 = __shfl_xor(s[u], o, kWave);
            join_stats(m[u], s[u], m2, s2);
        }
        if (lane_id() < 4) joined[wave_in_block()][r0 + u] = float2{m[u], s[u]};
    }
    __syncthreads();
    if ((int)threadIdx.x < rows) {
        float2 v = joined[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < 4; k++) join_stats(v.x, v.y, joined[k][threadIdx.x].x, joined[k][threadIdx.x].y);
        stats[(int64_t)range * a.V + row0 + threadIdx.x] = v;
    }
}

// Joins a row's ranges to lse and loss, `lanes` lanes a row (a power of two up to 64), and adds the
// workgroup's losses and labels in a fixed order; with one workgroup that is the result.
// grid: x = rows / (kJoinThreads / lanes)
__global__ __launch_bounds__(kJoinThreads) void head_rows(HeadArgs a, int ranges, int lanes, int mean,
                                                          const float2 *__restrict__ stats,
                                                          const float *__restrict__ at_label, float *__restrict__ lse,
                                                          float *__restrict__ row_loss, double *__restrict__ block_sum,
                                                          int32_t *__restrict__ block_count, float *__restrict__ total,
                                                          int32_t *__restrict__ total_count)
{
    __shared__ double s_sum[kJoinThreads / kWave];
    __shared__ int s_count[kJoinThreads / kWave];
    const int64_t row = (int64_t)blockIdx.x * (kJoinThreads / lanes) + threadIdx.x / lanes;
    const int lane = threadIdx.x % lanes;
    float m = -INFINITY, s = 0.f;
    if (row < a.V) {
#pragma unroll 4
        for (int k = lane; k < ranges; k += lanes) {
            const float2 v = stats[(int64_t)k * a.V + row];
            join_stats(m, s, v.x, v.y);
        }
    }
    for (int o = lanes / 2; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(m, o, kWave), s2 = __shfl_xor(s, o, kWave);
        join_stats(m, s, m2, s2);
    }
    double loss = 0.0;
    int count = 0;
    if (row < a.V && lane == 0) {
        const float l = m + logf(s);
        lse[row] = l;
        const bool counted = head_label(a, row) >= 0;
        const float v = counted ? l - at_label[row] : 0.f;
        if (row_loss) row_loss[row] = v;
        loss = (double)v;
        count = counted ? 1 : 0;
    }
    if (row_loss) return;
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
        if (gridDim.x == 1) {
            total[0] = (float)(mean ? loss / (double)count : loss);
            total_count[0] = count;
        } else {
            block_sum[blockIdx.x] = loss;
            block_count[blockIdx.x] = count;
        }
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
    const float *lse;          // [V]
    int64_t row0;              // the block of rows and the piece of classes
    int rows, c0, classes;
    bf16 *d;                   // [rows][ld] as parts
    int64_t part;
    int ld;
};

// d for a block of rows and a piece of classes.  Classes between the last and ld are written as zero.
// grid: x = workgroups, each with every gridDim.x-th tile
template <typename T, typename S> __global__ __launch_bounds__(S::kThreads, 2) void head_piece(PieceArgs a)
{
    using Product = StreamProduct<S, kAlongK, kAlongK>;
    extern __shared__ __align__(16) char lds[];
    const int ntiles = (a.classes + S::BN - 1) / S::BN, mtiles = (a.rows + S::BM - 1) / S::BM;
    const HeadArgs &h = a.head;
    auto corner = [&](int t, int *m0, int *n0) {
        int m, n;
        bool exists;
        tile_at(t, mtiles, ntiles, &m, &n, &exists);
        *m0 = m * S::BM;
        *n0 = n * S::BN;
    };
    Product::template run<kNoSums>(
        tiles_of(mtiles, ntiles), lds,
        [&](int t) {
            int m0, n0;
            corner(t, &m0, &n0);
            return StreamTile{h.w + (int64_t)(a.c0 + n0) * h.ld, h.x + (a.row0 + m0) * h.ld, h.part_w, h.part_x,
                              h.ld, h.ld, a.classes - n0, a.rows - m0, h.F};
        },
        [&](int t, f32x4(&acc)[S::FN][S::FM], f32x4 *) {
            int m0, n0;
            corner(t, &m0, &n0);
            logits<T, Product, S>(acc, h, a.c0 + n0);
            const bool edge = n0 + S::BN > a.classes;
#pragma unroll
            for (int j = 0; j < S::FM; j++) {
                const int m = m0 + Product::m_of(j);
                if (m >= a.rows) continue;
                const int64_t row = a.row0 + m;
                const int64_t label = head_label(h, row);
                const float l = a.lse[row];
                const uint32_t keep = label < 0 ? 0u : 0xffffffffu;
                const int at = label < 0 ? -1 : (int)(label - a.c0 - n0);
                bf16 *out = a.d + m * (int64_t)a.ld + n0;
#pragma unroll
                for (int i = 0; i < S::FN; i += 2) {
                    const int n = Product::n_of(i);
                    float d[8];
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        float t = acc[i + r / 4][j][r % 4] - l;
                        // bfloat16: the z of the statistics to the bit, so z <= l.  The z of a few rows of floats was
                        // summed in another order, which shows where logits have no bits behind the point (4e6: t = 2)
                        if (S::kParts > 1) t = t > 0.f ? 0.f : t;      // NaN stays
                        d[r] = __builtin_amdgcn_exp2f(t * kLog2e);
                    }
                    if (at >= n && at < n + 8) {
#pragma unroll
                        for (int r = 0; r < 8; r++)
                            if (n + r == at) d[r] -= 1.f;
                    }
                    if (edge) {
                        if (n0 + n >= a.ld) continue;
#pragma unroll
                        for (int r = 0; r < 8; r++)
                            if (n0 + n + r >= a.classes) d[r] = 0.f;
                    }
                    store_parts8<S::kParts>(out + n, a.part, d, keep);
                }
            }
        });
}

// out[m][n] = g ((first ? 0 : acc[m][n]) + sum_k P[n][k] Q[m][k]) when `last`, else the sum alone to
// `acc`; with several splits of k every split leaves its sum in part and head_join finishes.
struct SumArgs {
    const bf16 *p, *q;
    int64_t part_p, part_q;
    int ldp, ldq;
    int N, M, K, splits, k_split;
    void *out;          // [M][N]
    float *acc, *part;  // [M][N], [splits][M][N]
    void *out_b;        // sums of Q over k, [M]; the same three arrays for them, NULL: not wanted
    float *acc_b, *part_b;
    const float *row_scale;      // g of m, or NULL:
    const float *grad;           // g = grad[0] (/ count[0]); both NULL: 1
    const int32_t *count;
    int first, last;
    int whole;          // four neighbouring values lie on an address that one access can take
};

// what a sum is multiplied by
__device__ __forceinline__ float sum_scale(const SumArgs &a, int m)
{
    if (a.row_scale) return a.row_scale[m];
    if (!a.grad) return 1.f;
    if (!a.count) return a.grad[0];
    return a.count[0] > 0 ? a.grad[0] / (float)a.count[0] : 0.f;      // no row counts: every sum is zero
}

template <typename T>
__device__ __forceinline__ void finish4(const SumArgs &a, void *out, float *acc, int64_t at, f32x4 v, int n, float g)
{
    if (!a.first) {
        if (a.whole && n >= 4) v += *reinterpret_cast<const f32x4 *>(acc + at);
        else {
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (r < n) v[r] += acc[at + r];
        }
    }
    if (a.last) store4<T>(static_cast<T *>(out) + at, v * g, n, a.whole);
    else store4<float>(acc + at, v, n, a.whole);
}

// grid: x = workgroups, each with every gridDim.x-th tile of a split after the other
template <typename T, typename S, Layout QL, Sums SUMS> __global__ __launch_bounds__(S::kThreads, 2) void head_sum(SumArgs a)
{
    using Product = StreamProduct<S, kAcrossK, QL>;
    extern __shared__ __align__(16) char lds[];
    const int ntiles = (a.N + S::BN - 1) / S::BN, mtiles = (a.M + S::BM - 1) / S::BM;
    // the splits of a tile are tiles of their own, `mtiles` apart
    auto corner = [&](int t, int *m0, int *n0, int *split) {
        int m, n;
        bool exists;
        tile_at(t, mtiles * a.splits, ntiles, &m, &n, &exists);
        *split = m / mtiles;
        *m0 = (m % mtiles) * S::BM;
        *n0 = n * S::BN;
    };
    Product::template run<SUMS>(
        tiles_of(mtiles * a.splits, ntiles), lds,
        [&](int t) {
            int m0, n0, split;
            corner(t, &m0, &n0, &split);
            const int k0 = split * a.k_split, K = max(0, min(a.K - k0, a.k_split));
            return StreamTile{a.p + (int64_t)k0 * a.ldp + n0,
                              QL == kAlongK ? a.q + (int64_t)m0 * a.ldq + k0 : a.q + (int64_t)k0 * a.ldq + m0,
                              a.part_p, a.part_q, a.ldp, a.ldq, a.ldp - n0,
                              QL == kAlongK ? a.M - m0 : a.ldq - m0, K};
        },
        [&](int t, f32x4(&acc)[S::FN][S::FM], f32x4 *sums) {
            int m0, n0, split;
            corner(t, &m0, &n0, &split);
#pragma unroll
            for (int j = 0; j < S::FM; j++) {
                const int m = m0 + Product::m_of(j);
                if (m >= a.M) continue;
                const float g = a.splits > 1 ? 1.f : sum_scale(a, m);
                if (SUMS == kSumQ && n0 == 0 && Product::n_of(0) == 0) {
                    if (a.splits > 1) a.part_b[(int64_t)split * a.M + m] = sums[j][0];
                    else finish4<T>(a, a.out_b, a.acc_b, m, sums[j], 1, g);
                }
#pragma unroll
                for (int i = 0; i < S::FN; i++) {
                    const int n = n0 + Product::n_of(i);
                    if (n >= a.N) continue;
                    const int64_t at = (int64_t)m * a.N + n;
                    if (a.splits > 1) store4<float>(a.part + (int64_t)split * a.M * a.N + at, acc[i][j], a.N - n, a.whole);
                    else finish4<T>(a, a.out, a.acc, at, acc[i][j], a.N - n, g);
                }
            }
        });
}

// grid: x = results / 256 (of [M][N], then of [M])
template <typename T> __global__ __launch_bounds__(256) void head_join(SumArgs a)
{
    const int64_t size = (int64_t)a.M * a.N, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= size + (a.out_b ? a.M : 0)) return;
    const bool b = e >= size;
    const int64_t at = b ? e - size : e, stride = b ? a.M : size;
    const float *part = (b ? a.part_b : a.part) + at;
    float *acc = b ? a.acc_b : a.acc;
    float v = a.first ? 0.f : acc[at];
#pragma unroll 8
    for (int k = 0; k < a.splits; k++) v += part[k * stride];
    if (a.last)
        static_cast<T *>(b ? a.out_b : a.out)[at] = from_float<T>(v * sum_scale(a, a.row_scale ? (int)(at / a.N) : 0));
    else acc[at] = v;
}

// g of every row: grad where the row has a label, else zero.  grid: x = rows / 256
__global__ __launch_bounds__(256) void head_row_scale(HeadArgs a, const float *__restrict__ grad, float *__restrict__ scale)
{
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row < a.V) scale[row] = head_label(a, row) >= 0 ? grad[row] : 0.f;
}

// db of a piece with one g a row: acc[c] (+)= sum_m scale[m] d[m][c] over the block's rows, rounded to out
// when `last`.  A workgroup has 64 classes, 32 strands of rows.  grid: x = classes / 64
template <typename T>
__global__ __launch_bounds__(256) void head_bias(const bf16 *__restrict__ d, int64_t part, int ld, int rows, int classes,
                                                 const float *__restrict__ scale, float *__restrict__ acc, T *__restrict__ out,
                                                 int first, int last)
{
    __shared__ float strands[32][65];
    const int c = blockIdx.x * 64 + (threadIdx.x & 7) * 8, strand = threadIdx.x >> 3;
    float v[8] = {};
    if (c < classes) {      // ld is a multiple of 8 and holds zeros behind the last class
#pragma unroll 4
        for (int m = strand; m < rows; m += 32) {
            const float g = scale[m];
#pragma unroll
            for (int s = 0; s < HeadShape<T>::kParts; s++) {
                const u32x4 w = *reinterpret_cast<const u32x4 *>(d + s * part + (int64_t)m * ld + c);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[2 * i] = fmaf(g, bf16_lo(w[i]), v[2 * i]);
                    v[2 * i + 1] = fmaf(g, bf16_hi(w[i]), v[2 * i + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) strands[strand][(threadIdx.x & 7) * 8 + i] = v[i];
    __syncthreads();
    const int n = blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x < 64 && n < classes) {
        float sum = first ? 0.f : acc[n];
        for (int k = 0; k < 32; k++) sum += strands[k][threadIdx.x];
        if (last) out[n] = from_float<T>(sum);
        else acc[n] = sum;
    }
}

// workgroups of a launch: as many as are resident at once
template <typename S> constexpr int head_resident() { return kCus * (int)(160 * 1024 / S::kLds); }
template <typename S> static unsigned head_grid(int64_t tiles) { return (unsigned)std::min<int64_t>(tiles, head_resident<S>()); }

// ranges of class tiles: as many as fill the chip once
template <typename S> static int ranges_of(int64_t V, int C)
{
    const int64_t tiles = ceil_div(C, S::BN), blocks = std::max<int64_t>(1, ceil_div(V, S::BM));
    const int64_t ranges = std::min<int64_t>(tiles, std::max<int64_t>(1, head_resident<S>() / blocks));
    return (int)ceil_div(tiles, ceil_div(tiles, ranges));
}
template <typename T> static bool head_thin_takes(int64_t V, int F)
{
    return sizeof(T) == 4 && V <= kThinMost && F <= kThinFeatures;
}
// Small tiles for the logits where large ones would leave half of the chip without one.  Forward, large and small:
// floats, 100 rows, 1000 features, 16000 classes, 63 tiles: 112 and 77 us; 500, 256, 2000, 32 tiles: 34 and 22;
// 300, 256, 16000, 189 tiles: 42 and 49.  bfloat16, 100, 1000, 16000: 41 and 28; 2000, 256, 4000, 128 tiles: 22
// and 18; 200, 200, 40000, 157 tiles: 21 and 28.
template <typename T> static bool head_few(int64_t V, int C)
{
    return V <= HeadFew<T>::BM || ceil_div(V, HeadShape<T>::BM) * ceil_div(C, HeadShape<T>::BN) <= kCus / 2;
}
template <typename T> static int head_ranges(int64_t V, int F, int C)
{
    if (head_thin_takes<T>(V, F)) {      // about four workgroups a compute unit
        const int64_t tiles = ceil_div(C, kThinClasses), blocks = std::max<int64_t>(1, ceil_div(V, kThinRows));
        return (int)ceil_div(tiles, ceil_div(tiles, std::min<int64_t>(tiles, 1024 / blocks)));
    }
    return head_few<T>(V, C) ? ranges_of<HeadFew<T>>(V, C) : ranges_of<HeadShape<T>>(V, C);
}

// calls body(S()) with the shape of the tiles of a sum with N columns
template <typename T, typename Body> static auto with_sum_shape(int64_t N, Body &&body)
{
    using Full = HeadShape<T>;
    const int width = stream_width(N);
    if (width == 64) return body(typename StreamOfWidth<Full::kParts, 64, Full::kStep>::S());
    if (width == 128) return body(typename StreamOfWidth<Full::kParts, 128, Full::kStep>::S());
    return body(Full());
}

// splits of a sum over K for an [M][N] result: the fewest (of at least 512 steps each, up to 32) that
// leave under an eighth of the workgroups' turns empty, or the best there is
template <typename T> static int sum_splits(int64_t M, int64_t N, int64_t K)
{
    return with_sum_shape<T>(N, [&](auto shape) {
        using S = decltype(shape);
        const int64_t tiles = ceil_div(M, S::BM) * ceil_div(N, S::BN), resident = head_resident<S>();
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(std::max<int64_t>(32, resident / tiles), K / 512));
        int64_t best = 1;
        double best_used = 0.0;
        for (int64_t n = 1; n <= most; n++) {
            const double used = (double)(tiles * n) / (double)(ceil_div(tiles * n, resident) * resident);
            if (used > best_used + 0.02) best = n, best_used = used;
            if (used >= 0.875) break;
        }
        return (int)best;
    });
}

struct Pieces {
    int64_t rows, blocks;      // rows of a block, blocks
    int64_t classes, pieces;   // classes of a piece (whole tiles), pieces
};
template <typename T> static Pieces head_pieces(int64_t V, int C)
{
    constexpr int tile = HeadShape<T>::BN;
    Pieces s;
    s.rows = std::min<int64_t>(std::max<int64_t>(V, 1), kBlockRows);
    s.blocks = std::max<int64_t>(1, ceil_div(V, s.rows));
    s.classes = std::max<int64_t>(tile, kPieceBytes / (2 * HeadShape<T>::kParts) / s.rows / tile * tile);
    s.classes = std::min<int64_t>(s.classes, ceil_div(C, 8) * 8);
    s.pieces = ceil_div(C, s.classes);
    return s;
}

// where the parts of x and w come from: the arrays themselves, or copies in the workspace
template <typename T> static bool parts_in_place(int F) { return sizeof(T) == 2 && F % 8 == 0; }
static int64_t parts_ld(int F) { return ceil_div(F, 8) * 8; }
template <typename T> static size_t parts_elements(int64_t R, int F)
{
    return parts_in_place<T>(F) ? 0 : (size_t)(R * parts_ld(F) * HeadShape<T>::kParts);
}

template <typename T> struct HeadScratch {      // of the forward pass, then of the backward pass
    size_t x = 0, w = 0, gx = 0;                                      // bfloat16
    size_t scale = 0;                                                 // float
    size_t stats = 0, at_label = 0, blocks = 0;                       // float2, float, double + int
    size_t d = 0;                                                     // bfloat16
    size_t part = 0, part_b = 0, acc_x = 0, acc_w = 0, acc_b = 0;     // float
    HeadScratch(int64_t V, int F, int C, bool backward)
    {
        if (backward || !head_thin_takes<T>(V, F)) {
            x = parts_elements<T>(V, F);
            w = parts_elements<T>(C, F);
        }
        if (!backward) {
            stats = (size_t)head_ranges<T>(V, F, C) * V;
            at_label = (size_t)V;
            blocks = (size_t)ceil_div(V, kJoinThreads / kWave);
            return;
        }
        const Pieces s = head_pieces<T>(V, C);
        gx = (size_t)(V * parts_ld(F) * HeadShape<T>::kParts);
        scale = (size_t)V;
        d = (size_t)(s.rows * (s.classes + kPad) * HeadShape<T>::kParts);
        const int64_t sx = sum_splits<T>(s.rows, F, s.classes), sw = sum_splits<T>(s.classes, F, s.rows);
        part = (size_t)std::max(sx > 1 ? sx * s.rows * F : 0, sw > 1 ? sw * s.classes * F : 0);
        part_b = (size_t)(sw > 1 ? sw * s.classes : 0);
        acc_x = s.pieces > 1 ? (size_t)s.rows * F : 0;
        acc_w = s.blocks > 1 ? (size_t)C * F : 0;
        acc_b = s.blocks > 1 ? (size_t)C : 0;
    }
    size_t bytes() const
    {
        return carve_bytes(x, 2) + carve_bytes(w, 2) + carve_bytes(gx, 2) + carve_bytes(scale, 4) + carve_bytes(stats, 8) +
               carve_bytes(at_label, 4) +
               carve_bytes(blocks, 8) + carve_bytes(blocks, 4) + carve_bytes(d, 2) + carve_bytes(part, 4) +
               carve_bytes(part_b, 4) + carve_bytes(acc_x, 4) + carve_bytes(acc_w, 4) + carve_bytes(acc_b, 4);
    }
};

static int32_t head_check(const char *who, int64_t V, int32_t F, int32_t C, int32_t dtype, int32_t reduction)
{
    if (V < 0 || F <= 0 || C <= 0)
        return fail(JGAMD_ERR_SIZE, "%s: V=%lld F=%d C=%d (V >= 0, the others positive)", who, (long long)V, F, C);
    // V: blocks of 256 rows, 512 threads each, stay under 2^32 threads
    if (V > 0x7fffff00LL || F > kHeadMaxFeatures || C > 0x7fffff00)
        return fail(JGAMD_ERR_SIZE, "%s: V=%lld F=%d C=%d is too large", who, (long long)V, F, C);
    if (dtype != JGAMD_F32 && dtype != JGAMD_BF16) return fail(JGAMD_ERR_UNSUPPORTED, "%s: unknown dtype %d", who, dtype);
    if (reduction < 0 || reduction > JGAMD_LOSS_SUM) return fail(JGAMD_ERR_SIZE, "%s: unknown reduction %d", who, reduction);
    return 0;
}
// lays out one or two arrays as parts
template <typename T> static void head_copies(const Copy *of, int n, const HeadArgs &h, hipStream_t s)
{
    const int64_t first = ceil_div(of[0].R * (h.ld / 8), 256), second = n == 2 ? ceil_div(of[1].R * (h.ld / 8), 256) : 0;
    const Copies a{{of[0], of[n - 1]}, h.y32, h.y64, (int)first, (int)(first + second), h.F, h.ld, h.C};
    hipLaunchKernelGGL((head_parts<T>), grid_of_blocks(first + second), dim3(256), 0, s, a);
}

// x and w as parts: copies into the workspace, or the arrays themselves
template <typename T>
static int32_t head_operands(HeadArgs *h, const void *x, const void *w, bf16 *xs, bf16 *ws, hipStream_t s)
{
    h->ld = (int)parts_ld(h->F);
    h->part_x = h->V * h->ld;
    h->part_w = (int64_t)h->C * h->ld;
    if (parts_in_place<T>(h->F)) {
        h->x = static_cast<const bf16 *>(x);
        h->w = static_cast<const bf16 *>(w);
        return 0;
    }
    h->x = xs;
    h->w = ws;
    const int64_t blocks = ceil_div(h->part_x / 8, 256) + ceil_div(h->part_w / 8, 256);
    if (blocks > 0x7fffffffLL)
        return fail(JGAMD_ERR_SIZE, "linear_cross_entropy: V=%lld F=%d C=%d is too large", (long long)h->V, h->F, h->C);
    const Copy of[2] = {{x, nullptr, 1, h->V, xs, h->part_x}, {w, nullptr, 0, h->C, ws, h->part_w}};
    head_copies<T>(of, 2, *h, s);
    return launch_status("linear_cross_entropy");
}

template <typename T, Layout QL, Sums SUMS> static int32_t launch_sum(const SumArgs &a, hipStream_t s)
{
    with_sum_shape<T>(a.N, [&](auto shape) {
        using S = decltype(shape);
        raise_lds<&head_sum<T, S, QL, SUMS>>(S::kLds);
        const unsigned grid = head_grid<S>(ceil_div(a.N, S::BN) * ceil_div(a.M, S::BM) * a.splits);
        hipLaunchKernelGGL((head_sum<T, S, QL, SUMS>), dim3(grid), dim3(S::kThreads), S::kLds, s, a);
        return 0;
    });
    if (a.splits > 1) {
        const int64_t all = (int64_t)a.M * a.N + (a.out_b ? a.M : 0);
        hipLaunchKernelGGL((head_join<T>), dim3((unsigned)ceil_div(all, 256)), dim3(256), 0, s, a);
    }
    return launch_status("linear_cross_entropy_bwd");
}

template <typename T, typename S> static void launch_piece(const PieceArgs &a, hipStream_t st)
{
    raise_lds<&head_piece<T, S>>(S::kLds);
    hipLaunchKernelGGL((head_piece<T, S>), dim3(head_grid<S>(ceil_div(a.classes, S::BN) * ceil_div(a.rows, S::BM))),
                       dim3(S::kThreads), S::kLds, st, a);
}

template <typename T, typename S>
static void launch_stats(const HeadArgs &h, int ranges, float2 *stats, float *at_label, hipStream_t st)
{
    raise_lds<&head_stats<T, S>>(S::kLds);
    hipLaunchKernelGGL((head_stats<T, S>), dim3((unsigned)(ceil_div(h.V, S::BM) * ranges)), dim3(S::kThreads), S::kLds, st, h,
                       ranges, (int)ceil_div(ceil_div(h.C, S::BN), ranges), stats, at_label);
}

template <typename T>
static int32_t head_forward(HeadArgs h, const void *x, const void *w, int32_t reduction, float *loss, int32_t *count,
                            float *lse, void *ws, hipStream_t st)
{
    const HeadScratch<T> n(h.V, h.F, h.C, false);
    Carver carve(ws);
    bf16 *xs = carve.take<bf16>(n.x), *wp = carve.take<bf16>(n.w);
    float2 *stats = carve.take<float2>(n.stats);
    float *at_label = carve.take<float>(n.at_label);
    double *block_sum = carve.take<double>(n.blocks);
    int32_t *block_count = carve.take<int32_t>(n.blocks);
    const int mean = reduction == JGAMD_LOSS_MEAN ? 1 : 0;
    int blocks = 0;
    if (h.V > 0) {
        const int ranges = head_ranges<T>(h.V, h.F, h.C);
        const bool thin = head_thin_takes<T>(h.V, h.F);
        if (!thin)
            if (int32_t rc = head_operands<T>(&h, x, w, xs, wp, st)) return rc;
        if (thin) {
            const size_t lds = sizeof(float) * kThinRows * (size_t)(ceil_div(h.F, 64) * 64);
            raise_lds<&head_thin>(sizeof(float) * kThinRows * kThinFeatures);
            hipLaunchKernelGGL(head_thin, dim3((unsigned)(ceil_div(h.V, kThinRows) * ranges)), dim3(256), lds, st, h,
                               static_cast<const float *>(x), static_cast<const float *>(w), ranges,
                               (int)ceil_div(ceil_div(h.C, kThinClasses), ranges), stats, at_label);
        } else if (head_few<T>(h.V, h.C)) launch_stats<T, HeadFew<T>>(h, ranges, stats, at_label, st);
        else launch_stats<T, HeadShape<T>>(h, ranges, stats, at_label, st);
        int lanes = 1;      // four ranges a lane
        while (lanes < kWave && lanes * 4 < ranges) lanes *= 2;
        blocks = (int)ceil_div(h.V, kJoinThreads / lanes);
        hipLaunchKernelGGL(head_rows, dim3((unsigned)blocks), dim3(kJoinThreads), 0, st, h, ranges, lanes, mean, stats,
                           at_label, lse, reduction == JGAMD_LOSS_NONE ? loss : nullptr, block_sum, block_count, loss, count);
    }
    if (reduction != JGAMD_LOSS_NONE && blocks != 1)
        hipLaunchKernelGGL(head_total, dim3(1), dim3(kJoinThreads), 0, st, block_sum, block_count, blocks, mean, loss, count);
    return launch_status("linear_cross_entropy_fwd");
}

template <typename T>
static int32_t head_backward(HeadArgs h, const void *x, const void *w, const float *lse, const int32_t *count,
                             const float *grad, int32_t reduction, T *dx, T *dw, T *db, void *ws, hipStream_t st)
{
    const Pieces s = head_pieces<T>(h.V, h.C);
    const HeadScratch<T> n(h.V, h.F, h.C, true);
    Carver carve(ws);
    bf16 *xs = carve.take<bf16>(n.x), *wp = carve.take<bf16>(n.w), *gx = carve.take<bf16>(n.gx);
    float *scale = carve.take<float>(n.scale);
    bf16 *d = carve.take<bf16>(n.d);
    float *part = carve.take<float>(n.part), *part_b = carve.take<float>(n.part_b);
    float *acc_x = carve.take<float>(n.acc_x), *acc_w = carve.take<float>(n.acc_w), *acc_b = carve.take<float>(n.acc_b);
    if (h.V > 0)
        if (int32_t rc = head_operands<T>(&h, x, w, xs, wp, st)) return rc;
    if (h.V == 0) h.ld = (int)parts_ld(h.F);
    const bool per_row = reduction == JGAMD_LOSS_NONE;
    if (per_row && h.V > 0) hipLaunchKernelGGL(head_row_scale, dim3((unsigned)ceil_div(h.V, 256)), dim3(256), 0, st, h, grad, scale);
    // what dW sums: x, times one g a row if there is one, rows without a label zero (7 us of 9 ms for bf16)
    const bool own_copy = per_row || parts_in_place<T>(h.F);
    if (dw && own_copy && h.V > 0) {
        const Copy of{x, per_row ? scale : nullptr, !per_row, h.V, gx, h.V * h.ld};
        head_copies<T>(&of, 1, h, st);
    }
    const int ldd = (int)s.classes + kPad;
    const int64_t part_d = s.rows * ldd;
    auto whole = [](int N, const void *p) { return N % 4 == 0 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0; };
    for (int64_t b = 0; b < s.blocks; b++) {
        const int64_t row0 = b * s.rows;
        const int rows = (int)std::min<int64_t>(s.rows, h.V - row0);
        for (int64_t c = 0; c < s.pieces; c++) {
            const int c0 = (int)(c * s.classes), classes = (int)std::min<int64_t>(s.classes, h.C - c0);
            if (rows > 0) {
                const PieceArgs a{h, lse, row0, rows, c0, classes, d, part_d, ldd};
                if (head_few<T>(rows, classes)) launch_piece<T, HeadFew<T>>(a, st);
                else launch_piece<T, HeadShape<T>>(a, st);
                if (int32_t rc = launch_status("linear_cross_entropy_bwd")) return rc;
            }
            SumArgs a{};
            a.q = d, a.part_q = part_d, a.ldq = ldd, a.ldp = h.ld, a.N = h.F, a.part = part;
            a.grad = per_row ? nullptr : grad, a.count = reduction == JGAMD_LOSS_MEAN ? count : nullptr;
            if (dx && rows > 0) {
                a.row_scale = per_row ? scale + row0 : nullptr;
                a.p = h.w + (int64_t)c0 * h.ld, a.part_p = h.part_w;
                a.M = rows, a.K = classes;
                a.splits = sum_splits<T>(s.rows, h.F, s.classes);
                a.k_split = (int)(ceil_div(ceil_div(s.classes, a.splits), 64) * 64);
                a.out = dx + row0 * h.F, a.acc = acc_x;
                a.first = c == 0, a.last = c == s.pieces - 1, a.whole = whole(h.F, a.out);
                if (int32_t rc = launch_sum<T, kAlongK, kNoSums>(a, st)) return rc;
            }
            if (dw) {
                a.p = (own_copy ? gx : h.x) + row0 * h.ld, a.part_p = own_copy ? h.V * h.ld : h.part_x;
                a.row_scale = nullptr;
                a.M = classes, a.K = rows;
                a.splits = sum_splits<T>(s.classes, h.F, s.rows);
                a.k_split = (int)(ceil_div(ceil_div(s.rows, a.splits), 64) * 64);
                a.out = dw + (int64_t)c0 * h.F, a.acc = s.blocks > 1 ? acc_w + (int64_t)c0 * h.F : nullptr;
                const bool sums = db && !per_row;      // db beside dw
                a.out_b = sums ? db + c0 : nullptr, a.acc_b = s.blocks > 1 ? acc_b + c0 : nullptr, a.part_b = part_b;
                a.first = b == 0, a.last = b == s.blocks - 1, a.whole = whole(h.F, a.out);
                if (db && per_row)
                    hipLaunchKernelGGL((head_bias<T>), dim3((unsigned)ceil_div(classes, 64)), dim3(256), 0, st, d, part_d, ldd,
                                       rows, classes, scale + row0, a.acc_b, db + c0, a.first, a.last);
                const int32_t rc = sums ? launch_sum<T, kAcrossK, kSumQ>(a, st) : launch_sum<T, kAcrossK, kNoSums>(a, st);
                if (rc) return rc;
            }
        }
    }
    return 0;
}

}  // namespace jg

using namespace jg;
#define JG_EXPORT extern "C" __attribute__((visibility("default")))

static size_t head_bytes(int64_t V, int32_t F, int32_t C, int32_t dtype, bool backward)
{
    return dtype == JGAMD_F32 ? HeadScratch<float>(V, F, C, backward).bytes() : HeadScratch<bf16>(V, F, C, backward).bytes();
}

// what the two entry points ask of their arrays
static int32_t head_arrays(const char *who, int32_t dtype, const void *x, const void *w, const void *bias, const void *labels,
                           int32_t i64, int32_t F, const void *ws, size_t ws_bytes, size_t need)
{
    const uintptr_t element = dtype == JGAMD_F32 ? 3 : F % 8 == 0 ? 15 : 1;
    if ((((uintptr_t)x | (uintptr_t)w) & element) != 0)
        return fail(JGAMD_ERR_ALIGN, "%s: x / w not aligned to %d bytes", who, (int)element + 1);
    if (((uintptr_t)bias & (dtype == JGAMD_F32 ? 3 : 1)) != 0 || ((uintptr_t)labels & (i64 ? 7 : 3)) != 0)
        return fail(JGAMD_ERR_ALIGN, "%s: bias / labels do not start at a multiple of their element's size", who);
    if (need > 0 && (!ws || ws_bytes < need))
        return fail(JGAMD_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, ws ? ws_bytes : (size_t)0, need);
    if (need > 0 && ((uintptr_t)ws & 255) != 0) return fail(JGAMD_ERR_ALIGN, "%s: workspace not 256-byte aligned", who);
    return 0;
}

static HeadArgs head_args(const void *bias, const void *labels, int32_t i64, int64_t V, int32_t F, int32_t C)
{
    HeadArgs h{};
    h.bias = bias;
    h.y32 = i64 ? nullptr : static_cast<const int32_t *>(labels);
    h.y64 = i64 ? static_cast<const int64_t *>(labels) : nullptr;
    h.V = V, h.F = F, h.C = C;
    return h;
}

JG_EXPORT int32_t jgamd_linear_cross_entropy_workspace(int64_t V, int32_t F, int32_t C, int32_t dtype, int32_t backward,
                                                       size_t *bytes)
{
    if (!bytes) return fail(JGAMD_ERR_NULL, "linear_cross_entropy_workspace: bytes is NULL");
    if (int32_t rc = head_check("linear_cross_entropy_workspace", V, F, C, dtype, 0)) return rc;
    *bytes = head_bytes(V, F, C, dtype, backward != 0);
    return 0;
}

JG_EXPORT int32_t jgamd_linear_cross_entropy_fwd(const void *x, const void *w, const void *bias, const void *labels,
                                                 int32_t labels_are_i64, int64_t V, int32_t F, int32_t C, int32_t dtype,
                                                 int32_t reduction, float *loss, int32_t *count, float *lse, void *ws,
                                                 size_t ws_bytes, void *stream)
{
    const char *who = "linear_cross_entropy_fwd";
    if (int32_t rc = head_check(who, V, F, C, dtype, reduction)) return rc;
    if (reduction != JGAMD_LOSS_NONE && (!loss || !count)) return fail(JGAMD_ERR_NULL, "%s: loss / count is NULL", who);
    if (V > 0 && (!x || !w || !labels || !lse || !loss)) return fail(JGAMD_ERR_NULL, "%s: NULL array", who);
    if ((((uintptr_t)loss | (uintptr_t)count | (uintptr_t)lse) & 3) != 0)
        return fail(JGAMD_ERR_ALIGN, "%s: loss / count / lse not 4-byte aligned", who);
    const size_t need = head_bytes(V, F, C, dtype, false);
    if (int32_t rc = head_arrays(who, dtype, x, w, bias, labels, labels_are_i64, F, ws, ws_bytes, need)) return rc;
    const HeadArgs h = head_args(bias, labels, labels_are_i64, V, F, C);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == JGAMD_F32 ? head_forward<float>(h, x, w, reduction, loss, count, lse, ws, st)
                              : head_forward<bf16>(h, x, w, reduction, loss, count, lse, ws, st);
}

JG_EXPORT int32_t jgamd_linear_cross_entropy_bwd(const void *x, const void *w, const void *bias, const void *labels,
                                                 int32_t labels_are_i64, const float *lse, const int32_t *count,
                                                 const float *grad, int64_t V, int32_t F, int32_t C, int32_t dtype,
                                                 int32_t reduction, void *dx, void *dw, void *db, void *ws,
                                                 size_t ws_bytes, void *stream)
{
    const char *who = "linear_cross_entropy_bwd";
    if (int32_t rc = head_check(who, V, F, C, dtype, reduction)) return rc;
    if (db && !dw) return fail(JGAMD_ERR_NULL, "%s: db without dw", who);
    if (V > 0 && (!x || !w || !labels || !lse || !grad || (reduction == JGAMD_LOSS_MEAN && !count)))
        return fail(JGAMD_ERR_NULL, "%s: NULL array", who);
    const uintptr_t outs = (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)db;
    if ((outs & (dtype == JGAMD_F32 ? 3 : 1)) != 0 || (((uintptr_t)lse | (uintptr_t)count | (uintptr_t)grad) & 3) != 0)
        return fail(JGAMD_ERR_ALIGN, "%s: an array does not start at a multiple of its element's size", who);
    if (!dx && !dw) return 0;
    const size_t need = head_bytes(V, F, C, dtype, true);
    if (int32_t rc = head_arrays(who, dtype, x, w, bias, labels, labels_are_i64, F, ws, ws_bytes, need)) return rc;
    const HeadArgs h = head_args(bias, labels, labels_are_i64, V, F, C);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == JGAMD_F32)
        return head_backward<float>(h, x, w, lse, count, grad, reduction, static_cast<float *>(dx), static_cast<float *>(dw),
                                    static_cast<float *>(db), ws, st);
    return head_backward<bf16>(h, x, w, lse, count, grad, reduction, static_cast<bf16 *>(dx), static_cast<bf16 *>(dw),
                               static_cast<bf16 *>(db), ws, st);
}
