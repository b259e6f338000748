// Products of tiles on the matrix cores, shared by the typed product (grouped_rows.hip) and the
// class head (class_head.hip).
//
//     acc[n][m] += sum_k P[n][k] Q[m][k]
//
// P is the operand whose index runs along the registers of a lane (four consecutive n: the
// contiguous direction of what is stored), Q the one whose index runs along the lanes.  An operand
// lies in memory either with k contiguous (kAlongK: [row][k]) or with its row index contiguous
// (kAcrossK: [k][row]); the second kind is transposed on the way from LDS to the registers
// (ds_read_b64_tr_b16), so no operand is ever copied into another order.
//
// bfloat16 enters v_mfma_f32_16x16x32_bf16 as it is.  A float is split into three bfloat16 parts
// a = a1 + a2 + a3, each the remainder rounded to 8 bits, which together hold its 24 bits; six of
// the nine products of parts are summed in fp32 (a1b1, a1b2, a2b1, a1b3, a2b2, a3b1).  The parts are
// at most 2^-8 and 2^-17 of a, so the dropped products (a2b3, a3b2, a3b3) are under 2^-23.9 of a * b: about
// one rounding of a float, which each of the fp32 sums has too.  Six bfloat16 steps cost 6 / 16 of the fp32
// matrix instruction's time on this chip (2.5 PFLOP/s against 157 TFLOP/s).  Infinities and NaN have no such
// parts: results they enter are NaN.
#pragma once
#include "common.h"

namespace jg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
// the same 16 bytes at any element's address: rows of odd widths start anywhere
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));

struct bf16 {      // storage only
    uint16_t u;
};

enum Layout { kAlongK, kAcrossK };
enum Sums { kNoSums, kSumP, kSumQ };

// two floats, rounded to nearest even, as two bfloat16 in one register
__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __uint_as_float((uint32_t)v.u << 16); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float v)
{
    return bf16{(uint16_t)__builtin_bit_cast(uint16_t, (__bf16)v)};
}

// What the first part of a float is rounded from: past the largest bfloat16 (3.39e38) that one, and the second
// part takes the rest.  An infinity or a NaN gives something finite here and NaN as the last part.  60000 rows,
// 512 x 500 floats, forward: 201 us without it, 205 with it.
__device__ __forceinline__ float finite(float v) { return __builtin_amdgcn_fmed3f(v, -0x1.fep+127f, 0x1.fep+127f); }

// eight elements on their way from memory to LDS
template <typename T> struct Eight;
template <> struct Eight<bf16> {
    u32x4 v;
    static constexpr int kParts = 1;
    __device__ __forceinline__ void load(const bf16 *p) { v = *reinterpret_cast<const u32x4_at2 *>(p); }
    __device__ __forceinline__ void load_some(const bf16 *p, int n)      // the first n, zero behind them
    {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) w[i / 2] |= (uint32_t)p[i].u << (16 * (i & 1));
        v = u32x4{w[0], w[1], w[2], w[3]};
    }
    __device__ __forceinline__ void clear() { v = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void store(char *lds, int) const { *reinterpret_cast<u32x4 *>(lds) = v; }
    __device__ __forceinline__ void scale(float g)      // zero makes zero of anything
    {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = g == 0.f ? 0u : pack_bf16(g * bf16_lo(v[i]), g * bf16_hi(v[i]));
    }
};
template <> struct Eight<float> {
    f32x4 a, b;
    static constexpr int kParts = 3;
    __device__ __forceinline__ void load(const float *p)
    {
        a = *reinterpret_cast<const f32x4_at4 *>(p);
        b = *reinterpret_cast<const f32x4_at4 *>(p + 4);
    }
    __device__ __forceinline__ void load_some(const float *p, int n)
    {
        clear();
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) (i < 4 ? a : b)[i & 3] = p[i];
    }
    __device__ __forceinline__ void clear() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ void scale(float g)
    {
        if (g == 0.f) clear();
        else a *= g, b *= g;
    }
    // the three parts, `part_bytes` apart in LDS
    __device__ __forceinline__ void store(char *lds, int part_bytes) const
    {
        float r[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
        for (int s = 0; s < 3; s++) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[i] = s == 0 ? pack_bf16(finite(r[2 * i]), finite(r[2 * i + 1])) : pack_bf16(r[2 * i], r[2 * i + 1]);
                r[2 * i] -= bf16_lo(w[i]);
                r[2 * i + 1] -= bf16_hi(w[i]);
            }
            *reinterpret_cast<u32x4 *>(lds + s * part_bytes) = w;
        }
    }
};

// One operand of a tile: `base` points at row 0 of the tile and k = 0, `rows` of the tile's rows
// exist, `ld` elements lie between memory rows.
template <typename T> struct Operand {
    const T *base;
    int64_t ld;
    int rows;
};

// Where the 8 elements (row, k .. k + 7) (kAlongK) or (k, row .. row + 7) (kAcrossK) of a staged
// tile of BR rows and BK steps lie in LDS, in bytes.  kAlongK: 16-byte pieces of a row are permuted
// by the row, so that the 8 rows a read touches at a time fall on different banks.  kAcrossK: the
// 32-byte runs of 16 rows that a transposing read collects are permuted by k.
template <int BR, int BK, Layout LAY> struct Place {
    static constexpr int kBytes = BR * BK * 2;
    __device__ __forceinline__ static int at(int row, int k)
    {
        if (LAY == kAlongK) {
            constexpr int pieces = BK / 8;
            const int turn = pieces >= 8 ? row : row >> 1;
            return row * (BK * 2) + ((((k >> 3) ^ turn) & (pieces - 1)) << 4);
        }
        constexpr int runs = BR / 16;
        const int turn = (k & 3) | ((k >> 1) & 4);
        return k * (BR * 2) + ((((row >> 4) ^ turn) & (runs - 1)) << 5) + ((row & 15) << 1);
    }
};

// Moves one operand's tile from memory to registers (load) and on to LDS (store); the two are
// apart so that the loads of the next step are under way while this step's products run.
template <typename T, int BR, int BK, Layout LAY, int THREADS> struct Stage {
    static constexpr int kAcross = (LAY == kAlongK ? BK : BR) / 8;      // pieces of 8 per memory row
    static constexpr int kPieces = BR * BK / 8;
    static constexpr int kPasses = (kPieces + THREADS - 1) / THREADS;
    static constexpr int kPartBytes = Place<BR, BK, LAY>::kBytes;
    static constexpr int kBytes = kPartBytes * Eight<T>::kParts;
    Eight<T> r[kPasses];

    __device__ __forceinline__ static bool mine(int id) { return kPieces % THREADS == 0 || id < kPieces; }

    // steps k0 .. k0 + BK - 1, of which those from k_end on count as zero
    __device__ __forceinline__ void load(const Operand<T> &o, int k0, int k_end)
    {
#pragma unroll
        for (int p = 0; p < kPasses; p++) {
            const int id = threadIdx.x + p * THREADS;
            if (!mine(id)) continue;
            const int line = id / kAcross, c = (id % kAcross) * 8;
            if (LAY == kAlongK) {
                const int row = min(line, o.rows - 1);      // rows past the last repeat it: never stored
                const int left = k_end - (k0 + c);
                const T *src = o.base + (int64_t)row * o.ld + (k0 + c);
                if (left >= 8) r[p].load(src);
                else if (left > 0) r[p].load_some(src, left);
                else r[p].clear();
            } else {
                const int left = o.rows - c;
                const T *src = o.base + (int64_t)(k0 + line) * o.ld + c;
                if (k0 + line >= k_end || left <= 0) r[p].clear();
                else if (left >= 8) r[p].load(src);
                else r[p].load_some(src, left);
            }
        }
    }
    __device__ __forceinline__ void store(char *lds) const
    {
#pragma unroll
        for (int p = 0; p < kPasses; p++) {
            const int id = threadIdx.x + p * THREADS;
            if (!mine(id)) continue;
            const int line = id / kAcross, c = (id % kAcross) * 8;
            r[p].store(lds + (LAY == kAlongK ? Place<BR, BK, LAY>::at(line, c) : Place<BR, BK, LAY>::at(c, line)),
                       kPartBytes);
        }
    }
};

// the 8 steps k .. k + 7 of row `row` that lane l = 16 g + t holds: row = row0 + t, k = k0 + 8 g
template <int BR, int BK, Layout LAY> __device__ __forceinline__ bf16x8 fragment(const char *lds, int row0, int k0)
{
    const int t = lane_id() & 15, g = lane_id() >> 4;
    if (LAY == kAlongK) {
        return *reinterpret_cast<const bf16x8 *>(lds + Place<BR, BK, LAY>::at(row0 + t, k0 + 8 * g));
    }
    // a transposing read: the 16 lanes of a group name four lines of 16 rows (8 bytes a lane) and
    // lane t receives row t of all four
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int k = k0 + 8 * g + (t >> 2);
    const char *lo = lds + Place<BR, BK, LAY>::at(row0 + 4 * (t & 3), k);
    const char *hi = lds + Place<BR, BK, LAY>::at(row0 + 4 * (t & 3), k + 4);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)lo);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)hi);
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(bf16x8, v);
}

// The shape of a workgroup's tile: BN x BM results, WN x WM wavefronts.
template <typename T, int BN_, int BM_, int WN_, int WM_> struct Shape {
    static constexpr int BN = BN_, BM = BM_, WN = WN_, WM = WM_;
    static constexpr int kThreads = WN * WM * kWave;
    static constexpr int BK = sizeof(T) == 2 ? 64 : 32;
    static constexpr int FN = BN / WN / 16, FM = BM / WM / 16;      // 16 x 16 fragments of a wavefront
};

// acc of fragment (i, j): n = n_of(i) + r, m = m_of(j) for register r = 0..3
template <typename S> __device__ __forceinline__ int n_of(int i)
{
    return (wave_in_block() / S::WM) * (S::BN / S::WN) + i * 16 + 4 * (lane_id() >> 4);
}
template <typename S> __device__ __forceinline__ int m_of(int j)
{
    return (wave_in_block() % S::WM) * (S::BM / S::WM) + j * 16 + (lane_id() & 15);
}

template <typename T, typename S, Layout PL, Layout QL> struct TileProduct {
    using StageP = Stage<T, S::BN, S::BK, PL, S::kThreads>;
    using StageQ = Stage<T, S::BM, S::BK, QL, S::kThreads>;
    static constexpr int kLds = StageP::kBytes + StageQ::kBytes;
    static constexpr int kParts = Eight<T>::kParts;

    // acc += products over k_beg .. k_end - 1.  SUMS: also the sums of one operand over k, as products
    // with ones: kSumP: sums[i] += sum_k P[n][k] in every lane, at the registers of n; kSumQ:
    // sums[j] += sum_k Q[m][k] in every register, at the lanes of m.
    // Every wavefront of the workgroup calls it, with the same arguments.
    template <Sums SUMS = kNoSums>
    __device__ __forceinline__ static void run(f32x4 (&acc)[S::FN][S::FM], const Operand<T> &p, const Operand<T> &q,
                                               int k_beg, int k_end, char *lds, f32x4 *sums = nullptr)
    {
        if (k_beg >= k_end) return;
        StageP sp;
        StageQ sq;
        char *lp = lds, *lq = lds + StageP::kBytes;
        const int wn = (wave_in_block() / S::WM) * (S::BN / S::WN), wm = (wave_in_block() % S::WM) * (S::BM / S::WM);
        sp.load(p, k_beg, k_end);
        sq.load(q, k_beg, k_end);
        for (int k0 = k_beg; k0 < k_end; k0 += S::BK) {
            __syncthreads();      // everyone has read the step before
            sp.store(lp);
            sq.store(lq);
            __syncthreads();
            if (k0 + S::BK < k_end) {
                sp.load(p, k0 + S::BK, k_end);
                sq.load(q, k0 + S::BK, k_end);
            }
#pragma unroll
            for (int kk = 0; kk < S::BK; kk += 32) {
                bf16x8 fp[kParts][S::FN], fq[kParts][S::FM];
#pragma unroll
                for (int s = 0; s < kParts; s++) {
#pragma unroll
                    for (int i = 0; i < S::FN; i++)
                        fp[s][i] = fragment<S::BN, S::BK, PL>(lp + s * StageP::kPartBytes, wn + 16 * i, kk);
#pragma unroll
                    for (int j = 0; j < S::FM; j++)
                        fq[s][j] = fragment<S::BM, S::BK, QL>(lq + s * StageQ::kPartBytes, wm + 16 * j, kk);
                }
                // parts from the smallest products to the largest
#pragma unroll
                for (int sum = kParts - 1; sum >= 0; sum--)
#pragma unroll
                    for (int a = 0; a <= sum; a++)
#pragma unroll
                        for (int i = 0; i < S::FN; i++)
#pragma unroll
                            for (int j = 0; j < S::FM; j++)
                                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp[a][i], fq[sum - a][j], acc[i][j],
                                                                                    0, 0, 0);
                if (SUMS != kNoSums) {
                    const uint32_t one = 0x3f803f80u;      // two bfloat16 ones
                    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{one, one, one, one});
#pragma unroll
                    for (int s = kParts - 1; s >= 0; s--) {
                        if (SUMS == kSumP)
#pragma unroll
                            for (int i = 0; i < S::FN; i++)
                                sums[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp[s][i], ones, sums[i], 0, 0, 0);
                        else
#pragma unroll
                            for (int j = 0; j < S::FM; j++)
                                sums[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, fq[s][j], sums[j], 0, 0, 0);
                    }
                }
            }
        }
    }
};

// v[0..3] to out[0 .. n - 1] (n > 0): one store where four exist and lie on a whole address
template <typename T> __device__ __forceinline__ void store4(T *out, f32x4 v, int n, bool whole);
template <> __device__ __forceinline__ void store4<float>(float *out, f32x4 v, int n, bool whole)
{
    if (whole && n >= 4) {
        *reinterpret_cast<f32x4 *>(out) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) out[i] = v[i];
}
template <> __device__ __forceinline__ void store4<bf16>(bf16 *out, f32x4 v, int n, bool whole)
{
    if (whole && n >= 4) {
        *reinterpret_cast<u32x2 *>(out) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) out[i] = from_float<bf16>(v[i]);
}

}  // namespace jg
