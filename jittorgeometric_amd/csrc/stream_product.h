// The products of tile_product.h for operands that lie in memory as bfloat16 parts (one, or three for
// floats) on 16-byte addresses: tiles go from memory to LDS directly (buffer_load ... lds), several steps
// ahead, and a workgroup that owns several tiles keeps loading across their borders.
//
// A step is 32 or 64 values of k.  STAGES steps have room in LDS; while one is multiplied, the next
// STAGES - 1 are loaded or on their way.  Per step a wavefront waits until its own loads of that step
// have landed (all but the newest (STAGES - 2) steps' loads) and until its LDS reads of the step
// before are done, then one barrier makes every wavefront's loads visible and the oldest stage free
// for the loads of a later step.  Lanes whose data does not exist ask for an address past the
// descriptor's range, which the hardware answers with zeros: k past the end adds nothing.  Rows past
// the last of a tile repeat a row that exists and are not stored.
//
// The LDS image is in lines of 32 or 64 k, or of the tile's rows: a wavefront's load writes 1 KB in lane
// order, so the permutation is applied to the address each lane asks for.
//
// Which row of P stands at which row of a 16 x 16 fragment is free.  In pairs the fragments 2 i and
// 2 i + 1 of a wavefront share 32 rows such that a lane's two times four results are eight
// neighbouring n: the four lanes of an m then store 64 contiguous bytes of bfloat16 at a time
// instead of 32 (65521 rows of 32 types, 1024 x 2048: 402 -> 362 us).  Otherwise n is natural, four of a
// lane and sixteen of a fragment: 64 contiguous bytes of floats.
#pragma once
#include <type_traits>

#include "tile_product.h"

namespace jg {

constexpr uint32_t kStreamRange = 0x40000000u;      // bytes a lane's offset may span; past it reads zero

// One tile of the product: p[row][k] or p[k][row] as parts `part` elements apart.
// kAlongK: ld and K multiples of 8; kAcrossK: ld and rows multiples of 8.  p, q on 16-byte addresses.
struct StreamTile {
    const bf16 *p, *q;
    int64_t part_p, part_q;
    int ldp, ldq;
    int rows_p, rows_q;
    int K;
};

template <int PARTS, int BN_, int BM_, int WN_, int WM_, int STEP_, int STAGES_> struct StreamShape {
    static constexpr int BN = BN_, BM = BM_, WN = WN_, WM = WM_, kStep = STEP_, kStages = STAGES_, kParts = PARTS;
    static_assert(PARTS == 1 || PARTS == 3, "of a bfloat16 or of a float");
    static constexpr int kWaves = WN * WM, kThreads = kWaves * kWave;
    static constexpr int FN = BN / WN / 16, FM = BM / WM / 16;
    // of a wavefront, step and part
    static constexpr int kLoadsP = BN * kStep / 512 / kWaves, kLoadsQ = BM * kStep / 512 / kWaves;
    static constexpr int kLoads = (kLoadsP + kLoadsQ) * PARTS;
    static constexpr int kPartP = BN * kStep * 2, kPartQ = BM * kStep * 2;
    static constexpr int kStage = (kPartP + kPartQ) * PARTS;
    static constexpr int kLds = kStage * kStages;
    static_assert(kLoadsP >= 1 && kLoadsQ >= 1 && kLoads * (kStages - 2) < 64 && (kStep == 32 || kStep == 64), "");
};

// Four fragments of 16 rows whose LDS lines run along the rows, by transposing reads (tile_product.h's
// `fragment`); at[]: this lane's LDS address of the first line of each, the second line is `LINE`
// bytes on, both OFFSET further.  Written out with its wait: the compiler takes the builtin of this
// read to depend on every load into LDS under way and would wait for all of them in each step.
template <int OFFSET, int LINE> __device__ __forceinline__ void fragments_across(const uint32_t *at, bf16x8 *out)
{
    u32x2 v[8];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%c12\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:%c13\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%c12\n\t"
        "ds_read_b64_tr_b16 %3, %9 offset:%c13\n\t"
        "ds_read_b64_tr_b16 %4, %10 offset:%c12\n\t"
        "ds_read_b64_tr_b16 %5, %10 offset:%c13\n\t"
        "ds_read_b64_tr_b16 %6, %11 offset:%c12\n\t"
        "ds_read_b64_tr_b16 %7, %11 offset:%c13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "i"(OFFSET), "i"(OFFSET + LINE));
#pragma unroll
    for (int i = 0; i < 4; i++)
        out[i] = __builtin_bit_cast(bf16x8, u32x4{v[2 * i][0], v[2 * i][1], v[2 * i + 1][0], v[2 * i + 1][1]});
}

// Widths of tiles for an n that is a fraction of 256.  The fewer n a tile has, the more of its time goes into
// loading Q: a column of a tile of 128 is taken to cost 1.1 of one of 256, and tiles of 64 are for an n of up to 64
// (typed, 120000 rows, 256 -> 64 bfloat16: 18.0 us, 20.6 in tiles of 128; n = 192 in three tiles of 64 or one of 256:
// typed, 60000 rows of 1024: 46 and 37 us, class head, 8000 rows, 20000 classes, training: floats 1.96 and 1.71 ms,
// bfloat16 495 and 460 us; n = 320 in five of 64 or three of 128: 52 and 45 us, 2.99 and 2.56 ms, 727 and 686 us).
inline int stream_width(int64_t n)
{
    const double full = (double)((n + 255) / 256 * 256), half = 1.1 * (double)((n + 127) / 128 * 128);
    return n <= 64 ? 64 : half <= full ? 128 : 256;
}
template <int PARTS, int WIDTH, int STEP> struct StreamOfWidth;
template <int PARTS, int STEP> struct StreamOfWidth<PARTS, 256, STEP> {
    using S = StreamShape<PARTS, 256, 256, 2, 4, STEP, 2>;
};
template <int STEP> struct StreamOfWidth<3, 256, STEP> {      // 256 x 256 of three parts do not fit into LDS twice
    using S = StreamShape<3, 256, 128, 4, 2, STEP, 2>;
};
template <int PARTS, int STEP> struct StreamOfWidth<PARTS, 128, STEP> {
    using S = StreamShape<PARTS, 128, 256, 2, 4, STEP, PARTS == 1 ? 3 : 2>;
};
template <int PARTS, int STEP> struct StreamOfWidth<PARTS, 64, STEP> {
    using S = StreamShape<PARTS, 64, 256, 1, 4, STEP, 2>;
};

template <int N> __device__ __forceinline__ void wait_all_but()
{
    // vmcnt <= N and lgkmcnt == 0 (expcnt is not waited for)
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
}

__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <typename S, Layout PL, Layout QL, bool PAIRS = PL == kAlongK> struct StreamProduct {
    typedef __attribute__((address_space(3))) void lds_void;
    typedef __attribute__((address_space(3))) char lds_char;
    static constexpr bool kPairs = PAIRS;
    static_assert(!kPairs || S::FN % 2 == 0, "fragments of P come in pairs");

    // n of register 0 of fragment i (the other three follow), m of fragment j
    __device__ __forceinline__ static int n_of(int i)
    {
        const int n = (wave_in_block() / S::WM) * (S::BN / S::WN), g = lane_id() >> 4;
        return kPairs ? n + (i >> 1) * 32 + 8 * g + (i & 1) * 4 : n + i * 16 + 4 * g;
    }
    __device__ __forceinline__ static int m_of(int j)
    {
        return (wave_in_block() % S::WM) * (S::BM / S::WM) + j * 16 + (lane_id() & 15);
    }

    static constexpr int kRowPieces = S::kStep / 8;      // of 16 bytes, of a row along k

    // The turn of a row's pieces: the eight rows that are read at a time (0 .. 7 of Q; 0 .. 3 and 8 .. 11
    // of P in pairs) fall on different banks.  Rows of 64 bytes alternate between two halves by themselves.
    template <bool ROWS_IN_PAIRS> __device__ __forceinline__ static int turn(int row)
    {
        const int eight = ROWS_IN_PAIRS ? (row & 3) | ((row >> 1) & 4) : row & 7;
        return kRowPieces == 8 ? eight : eight >> 1;
    }
    // fragment of 16 rows along k at step kk of a stage, this lane's row given
    template <bool ROWS_IN_PAIRS> __device__ __forceinline__ static bf16x8 fragment_along(const char *lds, int row, int kk)
    {
        const int g = lane_id() >> 4;
        return *reinterpret_cast<const bf16x8 *>(lds + row * (2 * S::kStep) + (((kk / 8 + g) ^ turn<ROWS_IN_PAIRS>(row)) << 4));
    }

    // the addresses that this lane asks for, relative to the tile's (k = k0) corner
    template <int BR, int LOADS, Layout LAY, bool ROWS_IN_PAIRS> struct Lane {
        uint32_t off[LOADS];
        __device__ __forceinline__ static int k_of(int u)
        {
            const int id = (wave_in_block() * LOADS + u) * kWave + lane_id();
            if (LAY == kAlongK) return ((id % kRowPieces) ^ turn<ROWS_IN_PAIRS>(id / kRowPieces)) * 8;
            return id / (BR / 8);
        }
        __device__ __forceinline__ void place(int ld, int rows)
        {
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const int id = (wave_in_block() * LOADS + u) * kWave + lane_id();
                if (LAY == kAlongK) {
                    off[u] = (uint32_t)min(id / kRowPieces, rows - 1) * (uint32_t)(2 * ld) + 2 * k_of(u);
                } else {
                    const int k = id / (BR / 8), pos = id % (BR / 8);
                    const int by = (k & 3) | ((k >> 1) & 4);
                    const int col = ((((pos >> 1) ^ by) & (BR / 16 - 1)) << 4) + ((pos & 1) << 3);
                    off[u] = (uint32_t)k * (uint32_t)(2 * ld) + 2 * (col < rows ? col : 0);
                }
            }
        }
    };
    using LaneP = Lane<S::BN, S::kLoadsP, PL, kPairs>;
    using LaneQ = Lane<S::BM, S::kLoadsQ, QL, false>;

    template <int LOADS, typename L>
    __device__ __forceinline__ static void load(const bf16 *base, const L &lane, int left, char *lds)
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)kStreamRange, 0x00020000);
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            const uint32_t off = L::k_of(u) < left ? lane.off[u] : kStreamRange;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                r, (lds_void *)(lds + (wave_in_block() * LOADS + u) * 1024), 16, (int)off, 0, 0, 0);
        }
    }

    // 16 bytes to base + at where they exist
    __device__ __forceinline__ static void store(bf16 *base, uint32_t at, bool exists, u32x4 v)
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)kStreamRange, 0x00020000);
        __builtin_amdgcn_raw_buffer_store_b128(v, r, (int)(exists ? at : kStreamRange), 0, 0);
    }

    // the products of fragments i0 .. i1 - 1 of P, parts from the smallest products to the largest
    template <int PARTS>
    __device__ __forceinline__ static void multiply(f32x4 (&acc)[S::FN][S::FM], const bf16x8 (&fp)[S::kParts][S::FN],
                                                    const bf16x8 (&fq)[S::kParts][S::FM], int i0, int i1)
    {
#pragma unroll
        for (int sum = PARTS - 1; sum >= 0; sum--)
#pragma unroll
            for (int a = 0; a <= sum; a++)
#pragma unroll
                for (int i = i0; i < i1; i++)
#pragma unroll
                    for (int j = 0; j < S::FM; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp[a][i], fq[sum - a][j], acc[i][j], 0, 0, 0);
    }

    // Multiplies tiles 0 .. tiles - 1: tile(t) describes one (a StreamTile; cheap, called twice),
    // done(t, acc, sums) takes its results.  SUMS as in TileProduct.  The whole workgroup calls it.
    // On return LDS is free again.
    template <Sums SUMS, typename Tile, typename Done>
    __device__ __forceinline__ static void run(int tiles, char *lds, Tile &&tile, Done &&done)
    {
        constexpr int kSums = SUMS == kSumP ? S::FN : SUMS == kSumQ ? S::FM : 1;
        if (tiles <= 0) return;
        // the load side: next step to ask for
        int load_tile = 0, load_k = 0, load_stage = 0;
        StreamTile in = tile(0);
        LaneP lane_p;
        LaneQ lane_q;
        lane_p.place(in.ldp, in.rows_p);
        lane_q.place(in.ldq, in.rows_q);
        auto ask = [&]() {
            const int left = load_tile < tiles ? in.K - load_k : 0;      // past the last tile: zeros, never read
            char *stage = lds + load_stage * S::kStage;
#pragma unroll
            for (int s = 0; s < S::kParts; s++) {
                load<S::kLoadsP>(in.p + s * in.part_p + (PL == kAlongK ? (int64_t)load_k : (int64_t)load_k * in.ldp), lane_p,
                                 left, stage + s * S::kPartP);
                load<S::kLoadsQ>(in.q + s * in.part_q + (QL == kAlongK ? (int64_t)load_k : (int64_t)load_k * in.ldq), lane_q,
                                 left, stage + S::kParts * S::kPartP + s * S::kPartQ);
            }
            load_stage = load_stage + 1 == S::kStages ? 0 : load_stage + 1;
            load_k += S::kStep;
            if (load_k >= in.K && load_tile < tiles) {
                load_k = 0;
                if (++load_tile < tiles) {
                    in = tile(load_tile);
                    lane_p.place(in.ldp, in.rows_p);
                    lane_q.place(in.ldq, in.rows_q);
                }
            }
        };
#pragma unroll
        for (int s = 0; s < S::kStages - 1; s++) ask();
        const int wn = (wave_in_block() / S::WM) * (S::BN / S::WN), wm = (wave_in_block() % S::WM) * (S::BM / S::WM);
        // this lane's first line of each fragment across k, from the start of the operand's part
        uint32_t across_p[S::FN], across_q[S::FM];
        const int line_row = 4 * (lane_id() & 3), line_k = 8 * (lane_id() >> 4) + ((lane_id() >> 2) & 3);
        const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_char *)lds;
#pragma unroll
        for (int i = 0; i < S::FN; i++)
            across_p[i] = lds_at + Place<S::BN, S::kStep, kAcrossK>::at(
                                       kPairs ? wn + (i >> 1) * 32 + 2 * line_row + (i & 1) * 4 : wn + 16 * i + line_row, line_k);
#pragma unroll
        for (int j = 0; j < S::FM; j++)
            across_q[j] = lds_at + S::kParts * S::kPartP + Place<S::BM, S::kStep, kAcrossK>::at(wm + 16 * j + line_row, line_k);
        int stage_at = 0;
        for (int t = 0; t < tiles; t++) {
            f32x4 acc[S::FN][S::FM], sums[kSums];
#pragma unroll
            for (int i = 0; i < S::FN; i++)
#pragma unroll
                for (int j = 0; j < S::FM; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kSums; i++) sums[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            const int K = tile(t).K;
            int k = 0;
            do {      // a tile of no steps takes one, of zeros
                wait_all_but<S::kLoads *(S::kStages - 2)>();
                lds_barrier();
                ask();
                const uint32_t stage = stage_at * S::kStage;
                const char *lp = lds + stage, *lq = lp + S::kParts * S::kPartP;
                stage_at = stage_at + 1 == S::kStages ? 0 : stage_at + 1;
                bf16x8 fp[S::kParts][S::FN], fq[S::kParts][S::FM];
                auto read = [&](auto part, auto at_k) {
                    constexpr int s = decltype(part)::value, kk = decltype(at_k)::value;
                    if constexpr (QL == kAlongK) {
#pragma unroll
                        for (int j = 0; j < S::FM; j++)
                            fq[s][j] = fragment_along<false>(lq + s * S::kPartQ, wm + 16 * j + (lane_id() & 15), kk);
                    } else {
                        uint32_t at[S::FM];
#pragma unroll
                        for (int j = 0; j < S::FM; j++) at[j] = across_q[j] + stage;
#pragma unroll
                        for (int j = 0; j < S::FM; j += 4)
                            fragments_across<s * S::kPartQ + kk * 2 * S::BM, 8 * S::BM>(at + j, &fq[s][j]);
                    }
                    if constexpr (PL == kAlongK) {
                        const int t = lane_id() & 15;
#pragma unroll
                        for (int i = 0; i < S::FN; i++)
                            fp[s][i] = fragment_along<true>(
                                lp + s * S::kPartP, wn + (i >> 1) * 32 + (t >> 2) * 8 + (i & 1) * 4 + (t & 3), kk);
                    } else {
                        uint32_t at[S::FN];
#pragma unroll
                        for (int i = 0; i < S::FN; i++) at[i] = across_p[i] + stage;
#pragma unroll
                        for (int i = 0; i < S::FN; i += 4) {
                            fragments_across<s * S::kPartP + kk * 2 * S::BN, 8 * S::BN>(at + i, &fp[s][i]);
                            if constexpr (S::kParts == 1) multiply<1>(acc, fp, fq, i, i + 4);      // while the next are read
                        }
                    }
                };
                auto step = [&](auto at_k) {
                    read(std::integral_constant<int, 0>(), at_k);
                    if constexpr (S::kParts == 3) {
                        read(std::integral_constant<int, 1>(), at_k);
                        read(std::integral_constant<int, 2>(), at_k);
                    }
                    if constexpr (S::kParts > 1 || PL == kAlongK) multiply<S::kParts>(acc, fp, fq, 0, S::FN);
                    if (SUMS != kNoSums) {
                        const uint32_t one = 0x3f803f80u;      // two bfloat16 ones
                        const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{one, one, one, one});
#pragma unroll
                        for (int s = S::kParts - 1; s >= 0; s--)
#pragma unroll
                            for (int i = 0; i < kSums; i++)
                                sums[i] = SUMS == kSumP
                                              ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp[s][i], ones, sums[i], 0, 0, 0)
                                              : __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, fq[s][i], sums[i], 0, 0, 0);
                    }
                };
                step(std::integral_constant<int, 0>());
                if constexpr (S::kStep == 64) step(std::integral_constant<int, 32>());
                k += S::kStep;
            } while (k < K);
            done(t, acc, sums);
        }
        wait_all_but<0>();      // nothing may land in LDS after the workgroup has gone on
        lds_barrier();
    }
};

}  // namespace jg
