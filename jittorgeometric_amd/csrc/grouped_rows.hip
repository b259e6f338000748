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

#include "tile_product.h"

namespace jg {

constexpr int kMaxTypes = 65535;      // the summing kernel's grid.y
constexpr int kMaxWidth = 1 << 20;

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

// The `wanted`-th piece of at most `step` rows, counted over the types in order.  With `typed`
// false the rows before the first and behind the last type are runs of their own; with it true
// only types count, and a type without rows has one (empty) piece.  Returns false past the last.
template <int THREADS>
__device__ __forceinline__ bool find_run(const int32_t *__restrict__ off, int G, int M, int step, int wanted, bool typed,
                                         Run *run)
{
    __shared__ int wave_totals[THREADS / kWave];
    __shared__ Run found;
    __shared__ int hit;
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
            body(i - 1, begin, rows, np);
            begin = high;
        }
    };
    each([&](int, int, int, int np) {
        pieces += np;
        slots += np > 1 ? np : 0;
    });
    int all, ignored;
    int at = block_exclusive<THREADS, false>(pieces, wave_totals, &all);
    int slot = block_exclusive<THREADS, false>(slots, wave_totals, &ignored);
    if (threadIdx.x == 0) hit = 0;
    __syncthreads();
    if (wanted >= at && wanted < at + pieces) {
        each([&](int type, int begin, int rows, int np) {
            if (wanted >= at && wanted < at + np) {
                const int piece = wanted - at;
                found = Run{type, begin + piece * step, min(step, rows - piece * step), piece, np, slot};
                hit = 1;
            }
            at += np;
            slot += np > 1 ? np : 0;
        });
    }
    __syncthreads();
    *run = found;
    return hit != 0;
}

struct GroupedArgs {
    const void *x, *w, *bias;
    const int32_t *off;
    void *out;
    int M, K, N, G;
    int whole;      // four neighbouring results always lie on an address that one store can take
};

// grid: x = tiles of rows x tiles of columns, columns fastest
template <typename T, typename S, Layout WL> __global__ __launch_bounds__(S::kThreads) void grouped_rows(GroupedArgs a)
{
    using Product = TileProduct<T, S, WL, kAlongK>;
    __shared__ __align__(16) char lds[Product::kLds];
    const int ntiles = (a.N + S::BN - 1) / S::BN;
    Run run;
    if (!find_run<S::kThreads>(a.off, a.G, a.M, S::BM, blockIdx.x / ntiles, false, &run)) return;
    const int type = uniform(run.type), row0 = uniform(run.row), rows = uniform(run.rows);
    const int n0 = (blockIdx.x % ntiles) * S::BN;
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

struct GradArgs {
    const void *x, *dout;
    const int32_t *off;
    void *dw, *db;
    float *part, *part_b;      // [slots][K][N], [slots][N]: pieces of types that have several
    int M, K, N, G, piece;
    int whole;
};

// grid: x = pieces x tiles of dW, the tiles of one piece next to each other
template <typename T, typename S> __global__ __launch_bounds__(S::kThreads) void grouped_weight_grad(GradArgs a)
{
    using Product = TileProduct<T, S, kAcrossK, kAcrossK>;
    __shared__ __align__(16) char lds[Product::kLds];
    const int ntiles = (a.N + S::BN - 1) / S::BN, ktiles = (a.K + S::BM - 1) / S::BM;
    const int tile = blockIdx.x % (ntiles * ktiles);
    Run run;
    if (!find_run<S::kThreads>(a.off, a.G, a.M, a.piece, blockIdx.x / (ntiles * ktiles), true, &run)) return;
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

// Adds the pieces of the types that have several, in order.  grid: x = 1024 results each, y = types
template <typename T> __global__ __launch_bounds__(256) void grouped_weight_grad_sum(GradArgs a)
{
    __shared__ int s_pieces;
    __shared__ int wave_totals[4];
    const int type = blockIdx.y;
    // this type's pieces and the slots of the types before it, from offsets 0 .. type + 1
    int totals_ignored;
    const int n = type + 2;
    const int per = (n + 255) / 256;
    const int first = min((int)threadIdx.x * per, n), last = min(first + per, n);
    auto clean = [&](int i) { return min(max(a.off[i], 0), a.M); };
    int top = 0;
    for (int i = first; i < last; i++) top = max(top, clean(i));
    const int before = block_exclusive<256, true>(top, wave_totals, &totals_ignored);
    int slots = 0, mine = 0, begin = before, high = before;
    for (int i = first; i < last; i++) {
        high = max(high, clean(i));
        const int np = i >= 1 && high > begin ? (high - begin - 1) / a.piece + 1 : 0;
        if (i == type + 1) mine = np;
        else slots += np > 1 ? np : 0;
        begin = high;
    }
    int slots_before;
    block_exclusive<256, false>(slots, wave_totals, &slots_before);
    if (first <= type + 1 && type + 1 < last) s_pieces = mine;
    __syncthreads();
    const int pieces = uniform(s_pieces);
    if (pieces <= 1) return;
    const int64_t slot = slots_before, size = (int64_t)a.K * a.N;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int64_t e = (int64_t)blockIdx.x * 1024 + u * 256 + threadIdx.x;
        if (e < size) {
            float v = 0.f;
            for (int p = 0; p < pieces; p++) v += a.part[(slot + p) * size + e];
            static_cast<T *>(a.dw)[type * size + e] = from_float<T>(v);
        }
        if (a.db && e < a.N) {
            float v = 0.f;
            for (int p = 0; p < pieces; p++) v += a.part_b[(slot + p) * a.N + e];
            static_cast<T *>(a.db)[(int64_t)type * a.N + e] = from_float<T>(v);
        }
    }
}

// Rows a piece of the weight gradient sums: so many that about four workgroups per compute unit
// result, but whole steps of the product and at least 256
static int grad_piece(int32_t M, int32_t K, int32_t N)
{
    const int64_t tiles = ceil_div(K, 128) * ceil_div(N, 128);
    const int64_t pieces = std::max<int64_t>(1, 1024 / tiles);
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
    const int64_t blocks = mtiles * ceil_div(a.N, S::BN);
    if (blocks > 0x7fffffffLL) return fail(JGAMD_ERR_SIZE, "grouped_rows: M=%d N=%d G=%d is too large", a.M, a.N, a.G);
    hipLaunchKernelGGL((grouped_rows<T, S, WL>), dim3((unsigned)blocks), dim3(S::kThreads), 0, s, a);
    return launch_status("grouped_rows");
}

template <typename T> static int32_t rows_of_type(const GroupedArgs &a, bool transposed, hipStream_t s)
{
    using S = Shape<T, 128, 128, 2, 2>;
    return transposed ? launch_rows<T, S, kAlongK>(a, s) : launch_rows<T, S, kAcrossK>(a, s);
}

template <typename T> static int32_t weight_grad_of_type(const GradArgs &a, hipStream_t s)
{
    using S = Shape<T, 128, 128, 2, 2>;
    const int64_t tiles = ceil_div(a.N, S::BN) * ceil_div(a.K, S::BM);
    const int64_t blocks = tiles * ((int64_t)a.M / a.piece + a.G);
    if (blocks > 0x7fffffffLL)
        return fail(JGAMD_ERR_SIZE, "grouped_rows_weight_grad: K=%d N=%d G=%d is too large", a.K, a.N, a.G);
    hipLaunchKernelGGL((grouped_weight_grad<T, S>), dim3((unsigned)blocks), dim3(S::kThreads), 0, s, a);
    if (int32_t rc = launch_status("grouped_rows_weight_grad")) return rc;
    if (a.M <= a.piece) return 0;
    const unsigned gx = (unsigned)ceil_div((int64_t)a.K * a.N, 1024);
    hipLaunchKernelGGL((grouped_weight_grad_sum<T>), dim3(gx, (unsigned)a.G), dim3(256), 0, s, a);
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
