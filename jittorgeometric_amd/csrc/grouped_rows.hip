// Product of rows with the weight of their type, and its weight gradient:
//
//     out[r,:] = x[r,:] W[g] + b[g]        for off[g] <= r < off[g+1], rows of no type zero
//     dW[g]    = sum over those r of x[r,:]^T dout[r,:],   db[g] = sum of dout[r,:]
//
// W is [G][K][N], or [G][N][K] (the same weight, transposed: the input gradient dx = dout W^T).
// The offsets stay on the device.  Every workgroup finds the type its tile of rows belongs to by
// scanning them: a tile never holds rows of two types, so there are at most M / BM + min(G, M) + 2
// tiles (one more run of rows before the first type and one behind the last) and the workgroups
// past the actual number leave at once.  Offsets that fall or leave [0, M] are read as their
// running maximum clamped to [0, M], so that no offset can lead a kernel out of its arrays.
//
// The weight gradient's sum over the rows of a type is cut into pieces of `piece` rows when a type
// has more; a type of several pieces leaves fp32 tiles in the workspace, added in order by a second
// kernel: no atomics, the same bits every time.
#include <algorithm>

#include "lds_size.h"
#include "stream_product.h"

namespace jg {

constexpr int kMaxTypes = 65535;      // the summing kernel's grid.y
constexpr int kMaxWidth = 1 << 20;
constexpr int kSumBlocks = 4096;      // of the summing kernel

// exclusive prefix over the workgroup of `v`, combined by max (MAX) or by addition; the total in *total
template <int THREADS, bool MAX> __device__ __forceinline__ int block_exclusive(int v, int *wave_totals, int *total)
{
    auto join = [](int a, int b) { return MAX ? max(a, b) : a + b; };
    int inc = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(inc, d, kWave);
        if (lane_id() >= d) inc = join(inc, o);
    }
    const int wave = wave_in_block();
    __syncthreads();      // the totals of a previous call have been read
    if (lane_id() == kWave - 1) wave_totals[wave] = inc;
    __syncthreads();
    int before = 0, all = 0;      // both kinds of value are non-negative: 0 joins as nothing
#pragma unroll
    for (int w = 0; w < THREADS / kWave; w++) {
        if (w < wave) before = join(before, wave_totals[w]);
        all = join(all, wave_totals[w]);
    }
    const int left = __shfl_up(inc, 1, kWave);
    *total = all;
    return lane_id() == 0 ? before : join(before, left);
}

struct Run {
    int type;      // -1 before the first type, G behind the last, otherwise the type
    int row, rows; // first row of the piece and how many it has
    int piece;     // number of the piece within its type
    int pieces;    // pieces of the type
    int slot;      // pieces of earlier types that have more than one
};

// Pieces of at most `step` rows, counted over the types in order.  Looks up `count` of them: the i-th is
// number wanted(i); runs[i].pieces is 0 where there is no such piece.  With `typed` false the rows
// before the first and behind the last type are runs of their own; with it true only types count, and
// a type without rows has one (empty) piece.  The workgroup calls it; runs[] lies in LDS.
template <int THREADS, typename Wanted>
__device__ __forceinline__ void find_runs(const int32_t *__restrict__ off, int G, int M, int step, bool typed, int count,
                                          Wanted &&wanted, Run *runs)
{
    __shared__ int wave_totals[THREADS / kWave];
    // thread t reads `per` neighbouring offsets: 0 .. G + 1 with off[G + 1] taken as M
    const int n = G + 2;
    const int per = (n + THREADS - 1) / THREADS;
    const int first = min((int)threadIdx.x * per, n), last = min(first + per, n);
    auto clean = [&](int i) { return i > G ? M : min(max(off[i], 0), M); };
    int top = 0;
    for (int i = first; i < last; i++) top = max(top, clean(i));
    int total;
    const int before = block_exclusive<THREADS, true>(top, wave_totals, &total);
    // run i lies between offset i - 1 and offset i: run 0 before the first type, run G + 1 behind the last
    int pieces = 0, slots = 0;
    auto each = [&](auto &&body) {
        int begin = before, high = before;
        for (int i = first; i < last; i++) {
            high = max(high, clean(i));
            const int rows = high - begin;
            const bool counted = !typed || (i >= 1 && i <= G);
            int np = counted && rows > 0 ? (rows - 1) / step + 1 : 0;
            if (typed && counted && np == 0) np = 1;
            if (np > 0) body(i - 1, begin, rows, np);
            begin = high;
        }
    };
    each([&](int, int, int, int np) {
        pieces += np;
        slots += np > 1 ? np : 0;
    });
    int all, ignored;
    const int at0 = block_exclusive<THREADS, false>(pieces, wave_totals, &all);
    const int slot0 = block_exclusive<THREADS, false>(slots, wave_totals, &ignored);
    for (int k = 0; k < count; k++) {
        const int want = wanted(k);
        if (want >= at0 && want < at0 + pieces) {
            int at = at0, slot = slot0;
            each([&](int type, int begin, int rows, int np) {
                if (want >= at && want < at + np) {
                    const int piece = want - at;
                    runs[k] = Run{type, begin + piece * step, min(step, rows - piece * step), piece, np, slot};
                }
                at += np;
                slot += np > 1 ? np : 0;
            });
        }
        if (threadIdx.x == 0 && want >= all) runs[k].pieces = 0;
    }
    __syncthreads();
}

// one of them, for workgroup blockIdx.x's single tile; false where there is none
template <int THREADS>
__device__ __forceinline__ bool find_run(const int32_t *__restrict__ off, int G, int M, int step, int wanted, bool typed,
                                         Run *run)
{
    __shared__ Run found;
    find_runs<THREADS>(off, G, M, step, typed, 1, [&](int) { return wanted; }, &found);
    *run = found;
    return found.pieces != 0;
}

struct GroupedArgs {
    const void *x, *w, *bias;
    const int32_t *off;
    void *out;
    int M, K, N, G;
    int whole;      // four neighbouring results always lie on an address that one store can take
};

// This workgroup's place among `each` workgroups that read the same rows: group and place in it.  The
// groups go round the XCDs (every eighth workgroup runs on one), a group stays on one, one L2.  169343 rows,
// 129 -> 200 floats, forward, dx and dW: 124, 140, 154 us with neighbours on different XCDs, 120, 128, 143 like this.
__device__ __forceinline__ void group_of(int each, int *group, int *place)
{
    const int64_t b = block_number();
    const int i = (int)(b / 8);
    *group = i / each * 8 + (int)(b % 8);
    *place = i % each;
}
static int64_t grid_of_groups(int64_t groups, int64_t each) { return ceil_div(groups, 8) * 8 * each; }

// grid: x = tiles of rows x tiles of columns, by group_of
template <typename T, typename S, Layout WL> __global__ __launch_bounds__(S::kThreads) void grouped_rows(GroupedArgs a)
{
    using Product = TileProduct<T, S, WL, kAlongK>;
    __shared__ __align__(16) char lds[Product::kLds];
    const int ntiles = (a.N + S::BN - 1) / S::BN;
    Run run;
    int group, place;
    group_of(ntiles, &group, &place);
    if (!find_run<S::kThreads>(a.off, a.G, a.M, S::BM, group, false, &run)) return;
    const int type = uniform(run.type), row0 = uniform(run.row), rows = uniform(run.rows);
    const int n0 = place * S::BN;
    const bool typed = type >= 0 && type < a.G;
    f32x4 acc[S::FN][S::FM];
#pragma unroll
    for (int i = 0; i < S::FN; i++)
#pragma unroll
        for (int j = 0; j < S::FM; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (typed) {
        const T *w = static_cast<const T *>(a.w) + (int64_t)type * a.K * a.N;
        const Operand<T> p = WL == kAlongK ? Operand<T>{w + (int64_t)n0 * a.K, a.K, a.N - n0}
                                           : Operand<T>{w + n0, a.N, a.N - n0};
        const Operand<T> q{static_cast<const T *>(a.x) + (int64_t)row0 * a.K, a.K, rows};
        Product::run(acc, p, q, 0, a.K, lds);
    }
#pragma unroll
    for (int i = 0; i < S::FN; i++) {
        const int n = n0 + n_of<S>(i);
        if (n >= a.N) continue;
        f32x4 b = {0.f, 0.f, 0.f, 0.f};
        if (a.bias && typed) {
            const T *src = static_cast<const T *>(a.bias) + (int64_t)type * a.N + n;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (n + r < a.N) b[r] = to_float(src[r]);
        }
#pragma unroll
        for (int j = 0; j < S::FM; j++) {
            const int m = m_of<S>(j);
            if (m < rows)
                store4<T>(static_cast<T *>(a.out) + (int64_t)(row0 + m) * a.N + n, acc[i][j] + b, a.N - n, a.whole);
        }
    }
}

// The same with operands that stream into LDS (bfloat16, K and N multiples of 8, whole addresses).
// Workgroup b has tiles first(b), first(b) + gridDim.x, ...: at most kRunsKept.  The tiles of a run's
// columns are neighbours, and the workgroups of one XCD (every eighth) take neighbouring tiles: they
// share rows of x and the weight of a type in one L2.
constexpr int kRunsKept = 64;

__device__ __forceinline__ int first_tile()
{
    const int g = gridDim.x, b = blockIdx.x;
    return g % 8 == 0 ? (b % 8) * (g / 8) + b / 8 : b;
}

template <typename S, Layout WL> __global__ __launch_bounds__(S::kThreads, 2) void grouped_rows_stream(GroupedArgs a, int mtiles)
{
    using Product = StreamProduct<S, WL, kAlongK, true>;      // results in pairs: 16-byte stores
    extern __shared__ __align__(16) char lds[];
    __shared__ Run runs[kRunsKept];
    const int ntiles = (a.N + S::BN - 1) / S::BN;
    const int first = first_tile(), tiles = mtiles * ntiles;
    const int mine = first < tiles ? (tiles - 1 - first) / (int)gridDim.x + 1 : 0;
    auto number = [&](int t) { return first + t * (int)gridDim.x; };
    find_runs<S::kThreads>(a.off, a.G, a.M, S::BM, false, mine, [&](int t) { return number(t) / ntiles; }, runs);
    int count = 0;      // pieces are numbered without gaps: those that exist come first
    while (count < mine && uniform(runs[count].pieces) != 0) count++;
    const bf16 *x = static_cast<const bf16 *>(a.x), *w = static_cast<const bf16 *>(a.w);
    auto typed = [&](int type) { return type >= 0 && type < a.G; };
    Product::template run<kNoSums>(
        count, lds,
        [&](int t) {
            const int type = uniform(runs[t].type), row0 = uniform(runs[t].row), rows = uniform(runs[t].rows);
            const int n0 = (number(t) % ntiles) * S::BN;
            const bf16 *wt = w + (int64_t)(typed(type) ? type : 0) * a.K * a.N;
            return StreamTile{WL == kAlongK ? wt + (int64_t)n0 * a.K : wt + n0, x + (int64_t)row0 * a.K, 0, 0,
                              WL == kAlongK ? a.K : a.N, a.K, a.N - n0, rows, typed(type) ? a.K : 0};
        },
        [&](int t, f32x4(&acc)[S::FN][S::FM], f32x4 *) {
            const int type = uniform(runs[t].type), row0 = uniform(runs[t].row), rows = uniform(runs[t].rows);
            const int n0 = (number(t) % ntiles) * S::BN;
            bf16 *out = static_cast<bf16 *>(a.out) + (int64_t)row0 * a.N;
            Eight<bf16> b[S::FN / 2];      // asked for before the first store: loads and stores end in order
#pragma unroll
            for (int i = 0; i < S::FN / 2; i++) b[i].clear();
            if (a.bias && typed(type)) {
#pragma unroll
                for (int i = 0; i < S::FN / 2; i++) {
                    const int n = n0 + Product::n_of(2 * i);
                    b[i].load(static_cast<const bf16 *>(a.bias) + (int64_t)type * a.N + (n < a.N ? n : 0));
                }
            }
#pragma unroll
            for (int i = 0; i < S::FN; i += 2) {
                const int n = n0 + Product::n_of(i);
                const u32x4 e = b[i / 2].v;
                const f32x4 b0 = {bf16_lo(e[0]), bf16_hi(e[0]), bf16_lo(e[1]), bf16_hi(e[1])};
                const f32x4 b1 = {bf16_lo(e[2]), bf16_hi(e[2]), bf16_lo(e[3]), bf16_hi(e[3])};
#pragma unroll
                for (int j = 0; j < S::FM; j++) {
                    const int m = Product::m_of(j);
                    const f32x4 v = acc[i][j] + b0, v2 = acc[i + 1][j] + b1;
                    Product::store(out, ((uint32_t)m * (uint32_t)a.N + (uint32_t)n) * 2, m < rows && n < a.N,
                                   u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v2[0], v2[1]),
                                         pack_bf16(v2[2], v2[3])});
                }
            }
        });
}

// Few rows: the weights are read once and multiplied on the vector unit.  A tile of 128 rows holds a
// handful, its steps follow one another a memory latency each, and reading the weights is all there is
// to do: here every wavefront asks for its share of them at once.  kThinRows rows of x stand in LDS as
// floats.  48 rows of 16 types, 256 x 256 floats: 20.6 us with tiles, 7.9 like this.
constexpr int kThinRows = 8;
constexpr int kThinMost = 128;       // rows of a call, at most
constexpr int kThinSteps = 512;      // of k in LDS at a time
constexpr int kThinThreads = 512;

// rows row0 .. row0 + rows - 1 of x, steps k0 .. k0 + kThinSteps - 1, zero where there is none
template <typename T>
__device__ __forceinline__ void thin_stage(const T *x, int row0, int rows, int K, int k0, float (*xs)[kThinSteps])
{
#pragma unroll
    for (int r = 0; r < kThinRows; r++) {
        const int k = k0 + threadIdx.x;
        xs[r][threadIdx.x] = r < rows && k < K ? to_float(x[(int64_t)(row0 + r) * K + k]) : 0.f;
    }
}
static_assert(kThinSteps == kThinThreads, "a thread stages one step of every row");

// W [K][N]: two neighbouring columns a lane, CW columns a workgroup; wavefronts and the lanes that
// columns leave over share k.  grid: x = runs x blocks of CW columns
template <typename T, int CW> __global__ __launch_bounds__(kThinThreads) void grouped_thin_across(GroupedArgs a)
{
    constexpr int kLanes = CW / 2, kShares = kThinThreads / kLanes;      // lanes of a step, steps at a time
    __shared__ float xs[kThinRows][kThinSteps];
    __shared__ float part[kShares / 2][kThinRows][CW];
    const int blocks = (a.N + CW - 1) / CW;
    Run run;
    if (!find_run<kThinThreads>(a.off, a.G, a.M, kThinRows, blockIdx.x / blocks, false, &run)) return;
    const int type = uniform(run.type), row0 = uniform(run.row), rows = uniform(run.rows);
    const bool typed = type >= 0 && type < a.G;
    const int col = (blockIdx.x % blocks) * CW + (threadIdx.x % kLanes) * 2, share = threadIdx.x / kLanes;
    const int n = a.N - col;      // columns from here on
    float acc[kThinRows][2] = {};
    if (typed) {
        const T *w = static_cast<const T *>(a.w) + (int64_t)type * a.K * a.N + (n > 0 ? col : 0);
        for (int k0 = 0; k0 < a.K; k0 += kThinSteps) {
            __syncthreads();
            thin_stage(static_cast<const T *>(a.x), row0, rows, a.K, k0, xs);
            __syncthreads();
            const int steps = min(kThinSteps, a.K - k0);
#pragma unroll 8
            for (int k = share; k < steps; k += kShares) {
                const T *src = w + (int64_t)(k0 + k) * a.N;
                const float w0 = to_float(src[0]), w1 = to_float(src[n > 1 ? 1 : 0]);
#pragma unroll
                for (int r = 0; r < kThinRows; r++) {
                    const float xv = xs[r][k];
                    acc[r][0] = fmaf(xv, w0, acc[r][0]);
                    acc[r][1] = fmaf(xv, w1, acc[r][1]);
                }
            }
        }
    }
    // the shares in order, the upper half onto the lower first
    const int c = (threadIdx.x % kLanes) * 2;
    if (share >= kShares / 2)
#pragma unroll
        for (int r = 0; r < kThinRows; r++) {
            part[share - kShares / 2][r][c] = acc[r][0];
            part[share - kShares / 2][r][c + 1] = acc[r][1];
        }
    __syncthreads();
    if (share < kShares / 2)
#pragma unroll
        for (int r = 0; r < kThinRows; r++) {
            part[share][r][c] += acc[r][0];
            part[share][r][c + 1] += acc[r][1];
        }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * CW; e += kThinThreads) {
        const int r = e / CW, column = (blockIdx.x % blocks) * CW + e % CW;
        if (column >= a.N) continue;
        float v = a.bias && typed ? to_float(static_cast<const T *>(a.bias)[(int64_t)type * a.N + column]) : 0.f;
#pragma unroll
        for (int s = 0; s < kShares / 2; s++) v += part[s][r][e % CW];
        static_cast<T *>(a.out)[(int64_t)(row0 + r) * a.N + column] = from_float<T>(v);
    }
}

// W [N][K]: sixteen lanes a row of W, 16 bytes each, whose sums meet in shuffles.
// grid: x = runs x blocks of 32 columns
template <typename T> __global__ __launch_bounds__(kThinThreads) void grouped_thin_along(GroupedArgs a)
{
    constexpr int V = 8, kColumns = kThinThreads / 16;
    __shared__ __align__(16) float xs[kThinRows][kThinSteps];
    const int blocks = (a.N + kColumns - 1) / kColumns;
    Run run;
    if (!find_run<kThinThreads>(a.off, a.G, a.M, kThinRows, blockIdx.x / blocks, false, &run)) return;
    const int type = uniform(run.type), row0 = uniform(run.row), rows = uniform(run.rows);
    const bool typed = type >= 0 && type < a.G;
    const int lane = threadIdx.x % 16, col = (blockIdx.x % blocks) * kColumns + threadIdx.x / 16;
    float acc[kThinRows] = {};
    if (typed) {
        const T *w = static_cast<const T *>(a.w) + ((int64_t)type * a.N + min(col, a.N - 1)) * a.K;
        for (int k0 = 0; k0 < a.K; k0 += kThinSteps) {
            __syncthreads();
            thin_stage(static_cast<const T *>(a.x), row0, rows, a.K, k0, xs);
            __syncthreads();
            const int steps = min(kThinSteps, a.K - k0);
#pragma unroll
            for (int u = 0; u < kThinSteps / (16 * V); u++) {
                const int k = (u * 16 + lane) * V, left = steps - k;
                if (left <= 0) continue;
                float wv[V];
                if (left >= V) {
#pragma unroll
                    for (int i = 0; i < V; i++) wv[i] = to_float(w[k0 + k + i]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; i++) wv[i] = i < left ? to_float(w[k0 + k + i]) : 0.f;
                }
#pragma unroll
                for (int r = 0; r < kThinRows; r++)
#pragma unroll
                    for (int i = 0; i < V; i++) acc[r] = fmaf(xs[r][k + i], wv[i], acc[r]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kThinRows; r++)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) acc[r] += __shfl_xor(acc[r], o, 16);
    if (lane != 0 || col >= a.N) return;
    const float b = a.bias && typed ? to_float(static_cast<const T *>(a.bias)[(int64_t)type * a.N + col]) : 0.f;
#pragma unroll
    for (int r = 0; r < kThinRows; r++)
        if (r < rows) static_cast<T *>(a.out)[(int64_t)(row0 + r) * a.N + col] = from_float<T>(acc[r] + b);
}

struct GradArgs {
    const void *x, *dout;
    const int32_t *off;
    void *dw, *db;
    float *part, *part_b;      // [slots][K][N], [slots][N]: pieces of types that have several
    int M, K, N, G, piece;
    int whole;
};

// grid: x = pieces x tiles of dW, by group_of
template <typename T, typename S> __global__ __launch_bounds__(S::kThreads) void grouped_weight_grad(GradArgs a)
{
    using Product = TileProduct<T, S, kAcrossK, kAcrossK>;
    __shared__ __align__(16) char lds[Product::kLds];
    const int ntiles = (a.N + S::BN - 1) / S::BN, ktiles = (a.K + S::BM - 1) / S::BM;
    Run run;
    int group, tile;
    group_of(ntiles * ktiles, &group, &tile);
    if (!find_run<S::kThreads>(a.off, a.G, a.M, a.piece, group, true, &run)) return;
    const int type = uniform(run.type), row0 = uniform(run.row), rows = uniform(run.rows);
    const int n0 = (tile % ntiles) * S::BN, k0 = (tile / ntiles) * S::BM;
    f32x4 acc[S::FN][S::FM], sums[S::FN];
#pragma unroll
    for (int i = 0; i < S::FN; i++) {
        sums[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < S::FM; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const Operand<T> p{static_cast<const T *>(a.dout) + (int64_t)row0 * a.N + n0, a.N, a.N - n0};
    const Operand<T> q{static_cast<const T *>(a.x) + (int64_t)row0 * a.K + k0, a.K, a.K - k0};
    const bool with_bias = a.db && k0 == 0;
    if (with_bias) Product::template run<kSumP>(acc, p, q, 0, rows, lds, sums);
    else Product::run(acc, p, q, 0, rows, lds);

    const bool direct = run.pieces == 1;
    const int64_t slot = (int64_t)run.slot + run.piece;
#pragma unroll
    for (int i = 0; i < S::FN; i++) {
        const int n = n0 + n_of<S>(i);
        if (n >= a.N) continue;
        if (with_bias && m_of<S>(0) == 0) {
            if (direct) store4<T>(static_cast<T *>(a.db) + (int64_t)type * a.N + n, sums[i], a.N - n, a.whole);
            else store4<float>(a.part_b + slot * a.N + n, sums[i], a.N - n, a.whole);
        }
#pragma unroll
        for (int j = 0; j < S::FM; j++) {
            const int k = k0 + m_of<S>(j);
            if (k >= a.K) continue;
            if (direct)
                store4<T>(static_cast<T *>(a.dw) + ((int64_t)type * a.K + k) * a.N + n, acc[i][j], a.N - n, a.whole);
            else store4<float>(a.part + (slot * a.K + k) * a.N + n, acc[i][j], a.N - n, a.whole);
        }
    }
}

// The same, streaming
template <typename S, Sums SUMS> __global__ __launch_bounds__(S::kThreads, 2) void grouped_weight_grad_stream(GradArgs a, int pieces)
{
    using Product = StreamProduct<S, kAcrossK, kAcrossK>;
    extern __shared__ __align__(16) char lds[];
    __shared__ Run runs[kRunsKept];
    const int ntiles = (a.N + S::BN - 1) / S::BN, ktiles = (a.K + S::BM - 1) / S::BM, each = ntiles * ktiles;
    const int first = first_tile(), tiles = pieces * each;
    const int mine = first < tiles ? (tiles - 1 - first) / (int)gridDim.x + 1 : 0;
    auto number = [&](int t) { return first + t * (int)gridDim.x; };
    find_runs<S::kThreads>(a.off, a.G, a.M, a.piece, true, mine, [&](int t) { return number(t) / each; }, runs);
    int count = 0;
    while (count < mine && uniform(runs[count].pieces) != 0) count++;
    const bf16 *x = static_cast<const bf16 *>(a.x), *dout = static_cast<const bf16 *>(a.dout);
    auto corner = [&](int t, int *n0, int *k0) {
        const int tile = number(t) % each;
        *n0 = (tile % ntiles) * S::BN;
        *k0 = (tile / ntiles) * S::BM;
    };
    Product::template run<SUMS>(
        count, lds,
        [&](int t) {
            int n0, k0;
            corner(t, &n0, &k0);
            const int row0 = uniform(runs[t].row), rows = uniform(runs[t].rows);
            return StreamTile{dout + (int64_t)row0 * a.N + n0, x + (int64_t)row0 * a.K + k0, 0, 0,
                              a.N, a.K, a.N - n0, a.K - k0, rows};
        },
        [&](int t, f32x4(&acc)[S::FN][S::FM], f32x4 *sums) {
            int n0, k0;
            corner(t, &n0, &k0);
            const int type = uniform(runs[t].type);
            const bool direct = uniform(runs[t].pieces) == 1;
            const int64_t slot = (int64_t)uniform(runs[t].slot) + uniform(runs[t].piece);
#pragma unroll
            for (int i = 0; i < S::FN; i++) {
                const int n = n0 + Product::n_of(i);
                if (n >= a.N) continue;
                if (SUMS == kSumP && k0 == 0 && Product::m_of(0) == 0) {
                    if (direct) store4<bf16>(static_cast<bf16 *>(a.db) + (int64_t)type * a.N + n, sums[i], 4, a.whole);
                    else store4<float>(a.part_b + slot * a.N + n, sums[i], 4, true);
                }
#pragma unroll
                for (int j = 0; j < S::FM; j++) {
                    const int k = k0 + Product::m_of(j);
                    if (k >= a.K) continue;
                    if (direct)
                        store4<bf16>(static_cast<bf16 *>(a.dw) + ((int64_t)type * a.K + k) * a.N + n, acc[i][j], 4, a.whole);
                    else store4<float>(a.part + (slot * a.K + k) * a.N + n, acc[i][j], 4, true);
                }
            }
        });
}

// Adds the pieces of the types that have several, in order: workgroup y takes the y-th such type.
// grid: x = blocks of 256 results (all, or kSumBlocks over y, each with every gridDim.x-th), y = as many such
// types as there can be: most may not exist, as when every type fits a piece.  45 pieces of 256 x 256 results on
// average, up to 100: 15 us with four results a thread and one strand
template <typename T> __global__ __launch_bounds__(256) void grouped_weight_grad_sum(GradArgs a)
{
    __shared__ int wave_totals[4];
    __shared__ int s_type, s_slot, s_pieces;
    const int n = a.G + 1;
    const int per = (n + 255) / 256;
    const int first = min((int)threadIdx.x * per, n), last = min(first + per, n);
    auto clean = [&](int i) { return min(max(a.off[i], 0), a.M); };
    int top = 0, ignored;
    for (int i = first; i < last; i++) top = max(top, clean(i));
    const int before = block_exclusive<256, true>(top, wave_totals, &ignored);
    // type i - 1 has the rows between offset i - 1 and offset i
    auto each = [&](auto &&body) {
        int begin = before, high = before;
        for (int i = first; i < last; i++) {
            high = max(high, clean(i));
            const int np = i >= 1 && high > begin ? (high - begin - 1) / a.piece + 1 : 0;
            if (np > 1) body(i - 1, np);
            begin = high;
        }
    };
    int types = 0, slots = 0;
    each([&](int, int np) {
        types++;
        slots += np;
    });
    int at = block_exclusive<256, false>(types, wave_totals, &ignored);
    int slot_at = block_exclusive<256, false>(slots, wave_totals, &ignored);
    if (threadIdx.x == 0) s_pieces = 0;
    __syncthreads();
    each([&](int type, int np) {
        if (at++ == (int)blockIdx.y) {
            s_type = type;
            s_slot = slot_at;
            s_pieces = np;
        }
        slot_at += np;
    });
    __syncthreads();
    const int pieces = uniform(s_pieces);
    if (pieces == 0) return;
    const int64_t type = uniform(s_type), slot = uniform(s_slot), size = (int64_t)a.K * a.N;
    // Four neighbouring results a lane, eight pieces under way at a time; wavefront s takes pieces s, s + 4, ...
    // and the four sums are added in order.
    __shared__ f32x4 strands[3][kWave];
    const int strand = wave_in_block(), lane = lane_id();
    auto add = [&](const float *part, int64_t stride, int64_t block, T *out) {
        const int64_t e = (block * kWave + lane) * 4;
        const int n = (int)min((int64_t)4, stride - e);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (n == 4 && stride % 4 == 0) {
            const f32x4 *src = reinterpret_cast<const f32x4 *>(part + slot * stride + e);
#pragma unroll 8
            for (int p = strand; p < pieces; p += 4) v += src[p * (stride / 4)];
        } else {
            for (int r = 0; r < 4 && r < n; r++)
                for (int p = strand; p < pieces; p += 4) v[r] += part[(slot + p) * stride + e + r];
        }
        __syncthreads();
        if (strand > 0) strands[strand - 1][lane] = v;
        __syncthreads();
        if (strand > 0 || n <= 0) return;
        for (int s = 0; s < 3; s++) v += strands[s][lane];
        store4<T>(out + e, v, n, a.whole && stride % 4 == 0);
    };
    for (int64_t block = blockIdx.x; block * kWave * 4 < size; block += gridDim.x) {
        add(a.part, size, block, static_cast<T *>(a.dw) + type * size);
        if (a.db && block * kWave * 4 < a.N) add(a.part_b, a.N, block, static_cast<T *>(a.db) + type * a.N);
    }
}

// Rows a piece of the weight gradient sums: so many that about three workgroups per compute unit
// result, but whole steps of the product and at least 256
static int grad_piece(int32_t M, int32_t K, int32_t N)
{
    const int64_t tiles = ceil_div(K, 128) * ceil_div(N, 128);
    const int64_t pieces = std::max<int64_t>(1, 768 / tiles);
    const int64_t rows = ceil_div(ceil_div(M, pieces), 256) * 256;
    return (int)std::min<int64_t>(std::max<int64_t>(256, rows), 0x7fffff00);
}
static int64_t grad_slots(int32_t M, int32_t G, int piece)
{
    // a type with several pieces has more than `piece` rows: there are at most M / piece of them
    const int64_t whole = M / piece;
    return whole + std::min<int64_t>(G, whole);
}

static int32_t grouped_check(const char *who, int32_t M, int32_t K, int32_t N, int32_t G, int32_t dtype)
{
    if (M < 0 || K <= 0 || N <= 0 || G <= 0)
        return fail(JGAMD_ERR_SIZE, "%s: M=%d K=%d N=%d G=%d (M >= 0, the others positive)", who, M, K, N, G);
    if (K > kMaxWidth || N > kMaxWidth || G > kMaxTypes)
        return fail(JGAMD_ERR_SIZE, "%s: K=%d N=%d (at most %d), G=%d (at most %d)", who, K, N, kMaxWidth, G, kMaxTypes);
    if (dtype != JGAMD_F32 && dtype != JGAMD_BF16) return fail(JGAMD_ERR_UNSUPPORTED, "%s: unknown dtype %d", who, dtype);
    return 0;
}

// every array starts at a multiple of its element's size
static bool off_element(int32_t dtype, const void *p) { return ((uintptr_t)p & (dtype == JGAMD_F32 ? 3 : 1)) != 0; }

template <typename T, typename S, Layout WL> static int32_t launch_rows(const GroupedArgs &a, hipStream_t s)
{
    const int64_t mtiles = (int64_t)a.M / S::BM + std::min<int64_t>(a.G, a.M) + 2;
    const int64_t blocks = grid_of_groups(mtiles, ceil_div(a.N, S::BN));
    if (blocks > 0x7fffffffLL) return fail(JGAMD_ERR_SIZE, "grouped_rows: M=%d N=%d G=%d is too large", a.M, a.N, a.G);
    hipLaunchKernelGGL((grouped_rows<T, S, WL>), grid_of_blocks(blocks), dim3(S::kThreads), 0, s, a);
    return launch_status("grouped_rows");
}

// Tiles of 64 columns where they cover n with at most three quarters of what tiles of 128 do (129: 192
// against 256).  169343 rows of 200 floats to 129: 175 us with two tiles of 128, 142 with three of 64.
static bool narrow_tiles(int n) { return ceil_div(n, 64) * 64 * 4 <= ceil_div(n, 128) * 128 * 3; }

// Workgroups of a streaming launch: those resident at once, more only if one had over kRunsKept tiles.  Beside the
// stages LDS holds the runs: tiles of 64 columns, two of whose 80 KB would fill a compute unit, have one workgroup
// on each (120000 rows, 256 -> 64: 18.0 us, 20.7 with a grid for two; 60000 rows, 1024 x 64, dW: 70 and 74)
template <typename S> static unsigned stream_grid(int64_t tiles)
{
    constexpr int kRunBytes = kRunsKept * (int)sizeof(Run) + S::kWaves * (int)sizeof(int);
    const int64_t resident = 256 * (160 * 1024 / (S::kLds + kRunBytes));
    return (unsigned)std::min<int64_t>(tiles, std::max<int64_t>(resident, ceil_div(ceil_div(tiles, kRunsKept), 8) * 8));
}
// 256 x 128 results (two workgroups a compute unit, steps of 32) against 256 x 256 (one, steps of 64): 65521 rows,
// 32 types, 1024 x 2048: 423 and 420 us against 380 and 358 (the two directions); 120011 rows, 256 x 256: 45, 38
// against 42, 35
template <int WIDTH> using TypedStream = typename StreamOfWidth<1, WIDTH, 64>::S;
using GradOfFewK = StreamShape<1, 256, 64, 4, 1, 64, 2>;      // dW of up to 64 rows

template <typename S, Layout WL> static int32_t launch_rows_stream(const GroupedArgs &a, hipStream_t s)
{
    const int64_t mtiles = (int64_t)a.M / S::BM + std::min<int64_t>(a.G, a.M) + 2;
    const int64_t tiles = mtiles * ceil_div(a.N, S::BN);
    if (tiles > 0x3fffffffLL) return fail(JGAMD_ERR_SIZE, "grouped_rows: M=%d N=%d G=%d is too large", a.M, a.N, a.G);
    raise_lds<&grouped_rows_stream<S, WL>>(S::kLds);
    hipLaunchKernelGGL((grouped_rows_stream<S, WL>), dim3(stream_grid<S>(tiles)), dim3(S::kThreads), S::kLds, s, a, (int)mtiles);
    return launch_status("grouped_rows");
}
template <Layout WL> static int32_t rows_stream(const GroupedArgs &a, hipStream_t s)
{
    const int width = stream_width(a.N);
    if (width == 64) return launch_rows_stream<TypedStream<64>, WL>(a, s);
    if (width == 128) return launch_rows_stream<TypedStream<128>, WL>(a, s);
    return launch_rows_stream<TypedStream<256>, WL>(a, s);
}

template <typename T> static int32_t launch_thin(const GroupedArgs &a, bool transposed, hipStream_t s)
{
    const unsigned runs = a.M / kThinRows + std::min(a.G, a.M) + 2;
    const unsigned wide = (unsigned)ceil_div(a.N, 128), narrow = (unsigned)ceil_div(a.N, 32);
    if (transposed) hipLaunchKernelGGL((grouped_thin_along<T>), dim3(runs * narrow), dim3(kThinThreads), 0, s, a);
    // 32 columns a workgroup where 128 would leave compute units without one
    else if (runs * wide < 256) hipLaunchKernelGGL((grouped_thin_across<T, 32>), dim3(runs * narrow), dim3(kThinThreads), 0, s, a);
    else hipLaunchKernelGGL((grouped_thin_across<T, 128>), dim3(runs * wide), dim3(kThinThreads), 0, s, a);
    return launch_status("grouped_rows");
}

template <typename T> static int32_t rows_of_type(const GroupedArgs &a, bool transposed, hipStream_t s)
{
    // on average at most kThinRows rows a type; all of them of one type read its weight up to 16 times
    if (a.M <= kThinMost && a.M <= (int64_t)kThinRows * a.G) return launch_thin<T>(a, transposed, s);
    // streaming tiles, unless too few of 256 x 256 to fill half of the chip: 3000 rows, 2000 -> 504 bfloat16,
    // 24 of them: 57 us, 25 in tiles of 64 x 64 from registers; 6000 rows, 1024 -> 1024, 108 of them: 35 and 34
    auto tiles_of = [&](int of) { return ((int64_t)a.M / of + std::min(a.G, a.M)) * ceil_div(a.N, of); };
    if (sizeof(T) == 2 && a.K % 8 == 0 && a.N % 8 == 0 && (((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.out) & 15) == 0 &&
        tiles_of(256) >= 128)
        return transposed ? rows_stream<kAlongK>(a, s) : rows_stream<kAcrossK>(a, s);
    using Wide = Shape<T, 128, 128, 2, 2>;
    using Narrow = Shape<T, 64, 128, 2, 2>;
    using Small = Shape<T, 64, 64, 2, 2>;
    // 150 rows, 2047 -> 100 floats, 2 tiles of 128 x 128: 144 us, 68 in those of 64 x 64; 20000 rows, 256 -> 256,
    // 320 tiles: 29 and 26; 6000 rows, 1024 -> 1024, 400 tiles: 82 and 95
    if (tiles_of(128) < 384)
        return transposed ? launch_rows<T, Small, kAlongK>(a, s) : launch_rows<T, Small, kAcrossK>(a, s);
    if (narrow_tiles(a.N)) return transposed ? launch_rows<T, Narrow, kAlongK>(a, s) : launch_rows<T, Narrow, kAcrossK>(a, s);
    return transposed ? launch_rows<T, Wide, kAlongK>(a, s) : launch_rows<T, Wide, kAcrossK>(a, s);
}

template <typename S> static int64_t launch_grad_stream(const GradArgs &a, int64_t pieces, hipStream_t s)
{
    const int64_t tiles = ceil_div(a.N, S::BN) * ceil_div(a.K, S::BM) * pieces;
    if (tiles > 0x3fffffffLL) return tiles;
    const dim3 grid(stream_grid<S>(tiles)), threads(S::kThreads);
    if (a.db) {
        raise_lds<&grouped_weight_grad_stream<S, kSumP>>(S::kLds);
        hipLaunchKernelGGL((grouped_weight_grad_stream<S, kSumP>), grid, threads, S::kLds, s, a, (int)pieces);
    } else {
        raise_lds<&grouped_weight_grad_stream<S, kNoSums>>(S::kLds);
        hipLaunchKernelGGL((grouped_weight_grad_stream<S, kNoSums>), grid, threads, S::kLds, s, a, (int)pieces);
    }
    return tiles;
}

template <typename T, int BN, int BM> static int64_t launch_grad(const GradArgs &a, int64_t pieces, hipStream_t s)
{
    using S = Shape<T, BN, BM, 2, 2>;
    const int64_t tiles = grid_of_groups(pieces, ceil_div(a.N, BN) * ceil_div(a.K, BM));
    if (tiles <= 0x3fffffffLL)
        hipLaunchKernelGGL((grouped_weight_grad<T, S>), grid_of_blocks(tiles), dim3(S::kThreads), 0, s, a);
    return tiles;
}

template <typename T> static int32_t weight_grad_of_type(const GradArgs &a, hipStream_t s)
{
    const int64_t pieces = (int64_t)a.M / a.piece + a.G;
    const bool stream = sizeof(T) == 2 && a.K % 8 == 0 && a.N % 8 == 0 && (((uintptr_t)a.x | (uintptr_t)a.dout) & 15) == 0;
    int64_t tiles;
    if (stream) {
        const int width = stream_width(a.N);
        if (a.K <= 64 && width > 64) tiles = launch_grad_stream<GradOfFewK>(a, pieces, s);
        else if (width == 64) tiles = launch_grad_stream<TypedStream<64>>(a, pieces, s);
        else if (width == 128) tiles = launch_grad_stream<TypedStream<128>>(a, pieces, s);
        else tiles = launch_grad_stream<TypedStream<256>>(a, pieces, s);
    } else if (narrow_tiles(a.N)) {
        tiles = narrow_tiles(a.K) ? launch_grad<T, 64, 64>(a, pieces, s) : launch_grad<T, 64, 128>(a, pieces, s);
    } else {
        tiles = narrow_tiles(a.K) ? launch_grad<T, 128, 64>(a, pieces, s) : launch_grad<T, 128, 128>(a, pieces, s);
    }
    if (tiles > 0x3fffffffLL)
        return fail(JGAMD_ERR_SIZE, "grouped_rows_weight_grad: K=%d N=%d G=%d is too large", a.K, a.N, a.G);
    if (int32_t rc = launch_status("grouped_rows_weight_grad")) return rc;
    if (a.M <= a.piece) return 0;
    const unsigned types = (unsigned)std::min(a.G, a.M / a.piece);
    const int64_t blocks = ceil_div((int64_t)a.K * a.N, 4 * kWave);
    const unsigned gx = (unsigned)std::min<int64_t>(blocks, std::max<int64_t>(64, kSumBlocks / types));
    hipLaunchKernelGGL((grouped_weight_grad_sum<T>), dim3(gx, types), dim3(256), 0, s, a);
    return launch_status("grouped_rows_weight_grad");
}

}  // namespace jg

using namespace jg;
#define JG_EXPORT extern "C" __attribute__((visibility("default")))

JG_EXPORT int32_t jgamd_grouped_rows(const void *x, const void *w, const void *bias, const int32_t *off, void *out,
                                     int32_t M, int32_t K, int32_t N, int32_t G, int32_t dtype, int32_t flags,
                                     void *stream)
{
    if (int32_t rc = grouped_check("grouped_rows", M, K, N, G, dtype)) return rc;
    if (flags & ~JGAMD_WEIGHT_TRANSPOSED) return fail(JGAMD_ERR_SIZE, "grouped_rows: unknown flags %d", flags);
    if (M == 0) return 0;
    if (!x || !w || !off || !out) return fail(JGAMD_ERR_NULL, "grouped_rows: NULL array");
    if (off_element(dtype, x) || off_element(dtype, w) || off_element(dtype, bias) || off_element(dtype, out) ||
        ((uintptr_t)off & 3) != 0)
        return fail(JGAMD_ERR_ALIGN, "grouped_rows: an array does not start at a multiple of its element's size");
    const bool f32 = dtype == JGAMD_F32;
    const int whole = N % 4 == 0 && ((uintptr_t)out & (f32 ? 15 : 7)) == 0;
    const GroupedArgs a{x, w, bias, off, out, M, K, N, G, whole};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool transposed = (flags & JGAMD_WEIGHT_TRANSPOSED) != 0;
    return f32 ? rows_of_type<float>(a, transposed, s) : rows_of_type<bf16>(a, transposed, s);
}

static size_t grad_part_floats(int32_t M, int32_t K, int32_t N, int32_t G, size_t *bias_floats)
{
    const int piece = grad_piece(M, K, N);
    const size_t slots = M > piece ? (size_t)grad_slots(M, G, piece) : 0;
    *bias_floats = slots * N;
    return slots * K * N;
}

JG_EXPORT int32_t jgamd_grouped_rows_weight_grad_workspace(int32_t M, int32_t K, int32_t N, int32_t G, size_t *bytes)
{
    if (!bytes) return fail(JGAMD_ERR_NULL, "grouped_rows_weight_grad_workspace: bytes is NULL");
    if (int32_t rc = grouped_check("grouped_rows_weight_grad_workspace", M, K, N, G, JGAMD_F32)) return rc;
    size_t nb;
    const size_t n = grad_part_floats(M, K, N, G, &nb);
    *bytes = carve_bytes(n, 4) + carve_bytes(nb, 4);
    return 0;
}

JG_EXPORT int32_t jgamd_grouped_rows_weight_grad(const void *x, const void *dout, const int32_t *off, void *dw, void *db,
                                                 int32_t M, int32_t K, int32_t N, int32_t G, int32_t dtype, void *ws,
                                                 size_t ws_bytes, void *stream)
{
    if (int32_t rc = grouped_check("grouped_rows_weight_grad", M, K, N, G, dtype)) return rc;
    if (!off || !dw || (M > 0 && (!x || !dout))) return fail(JGAMD_ERR_NULL, "grouped_rows_weight_grad: NULL array");
    if (off_element(dtype, x) || off_element(dtype, dout) || off_element(dtype, dw) || off_element(dtype, db) ||
        ((uintptr_t)off & 3) != 0)
        return fail(JGAMD_ERR_ALIGN, "grouped_rows_weight_grad: an array does not start at a multiple of its element's size");
    size_t nb;
    const size_t n = grad_part_floats(M, K, N, G, &nb);
    const size_t need = carve_bytes(n, 4) + carve_bytes(nb, 4);
    if (need > 0 && (!ws || ws_bytes < need))
        return fail(JGAMD_ERR_WORKSPACE, "grouped_rows_weight_grad: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
    if (need > 0 && ((uintptr_t)ws & 255) != 0)
        return fail(JGAMD_ERR_ALIGN, "grouped_rows_weight_grad: workspace not 256-byte aligned");
    Carver carve(ws);
    const bool f32 = dtype == JGAMD_F32;
    const int whole = N % 4 == 0 && (((uintptr_t)dw | (uintptr_t)db) & (f32 ? 15 : 7)) == 0;
    GradArgs a{x, dout, off, dw, db, nullptr, nullptr, M, K, N, G, grad_piece(M, K, N), whole};
    if (need > 0) {
        a.part = carve.take<float>(n);
        a.part_b = carve.take<float>(nb);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    return f32 ? weight_grad_of_type<float>(a, s) : weight_grad_of_type<bf16>(a, s);
}
