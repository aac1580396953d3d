// Weight gradient of a linear layer (or 1 x 1 convolution, channels last) from the 8-bit checkpoint of its input (elem8.inc):
//
//     gw[o][i] = alpha * sum over r of gy[r][o] * x8[r][i],     gb[o] = sum over r of gy[r][o]
//
// on the 16-bit matrix cores with fp32 accumulation, without a rounding in front of the sum:
//     x8 = q * 2^k has 8 significant bits at most: a bf16 (and, with k >= -24, an f16) value exactly
//     gy in bf16 / f16 is taken as it is
//     gy in f32 is cut into three bf16 pieces of 8 bits each and takes three products; high + middle + low = gy exactly from
//     |gy| = 2^-110 up.  Below, the pieces end at the last place of bf16's subnormals, 2^-133, and lose less than 2^-132 of a value
//     (gy of 1e-36 everywhere: 3e-5 of gw, where fp32 sums alone are good for 2e-7)
// v_mfma_f32_32x32x16 at 3 products has five times the rate of v_mfma_f32_32x32x2_f32: keeping x in 8 bits makes the f32 weight
// gradient faster than the exact f32 product of the full-width tensors, not only smaller.
//
// Tile: BM channels of gy x 128 channels of x, 32 rows (f32) or 64 at a time; 256 x 128 in eight waves of 64 x 128, each group of four
// with half of a step's rows, where there is work for it, 128 and 64 in four waves where not.  The sum runs over ROWS, the slow axis of
// both tensors, while a matrix-core operand wants 8 rows of one channel next to each other: a thread loads 16 bytes (4 or 8 channels) of
// 4 rows of gy and 4 codes of 4 rows, and writes for each of its channels the 4 rows packed to 8 bytes.  LDS holds 16-byte cells
// [k octet][position], where the j-th channel of the q-th thread sits at G j + q of its group of 128: lanes that stage neighbouring
// channels write neighbouring cells, and an operand is one 16-byte read with neighbouring lanes on neighbouring cells (no bank conflict,
// by the counters).  For the codes G = 32, and a lane ends up with 4 neighbouring output channels in its 4 accumulators: whole 16-byte
// stores, no shuffle.
//
// What bounds it: a wave issues in order, so everything a step needs beside its products -- cutting gy, decoding codes, LDS writes,
// the loads two and three steps ahead -- is dealt out between them (`multiply`), 6 to 7 vector instructions a product, and two waves a
// SIMD cover each other.  Measured (f32 16384 x 1024 x 2048, bf16 65536 x 512 x 512, with the reduction):
//     340, 140 us   one set of cells, a burst of loads, then of vector work, then of products
//     229, 100      two groups of four waves that stage and multiply in turn; their loads, one step ahead, are waited for
//     207, 65       four waves, dealt out; operands read ahead
//     201, 58       eight waves, two on a SIMD
//     192, 58       f32: no branch in a step, no code decoded twice (this form)
// f32: 990 - 1070 TFLOP/s on the matrix cores (192 - 208 us, by the card), where a library's bf16 product of 8192^3 reaches 1217 - 1362; the clock is what is left
// (with gy = 0 the same launch takes 15 % less).  bf16: 45 us here and 12 in the kernel that adds the slices; of the 45, some 10 are
// the first loads and the last stores.  65536 x 1024 x 2048 runs at 870 TFLOP/s.
//
// Few tiles: the rows are cut into slices, one work-group each, whose fp32 tiles a second kernel adds in order.
#include "elem8.inc"

namespace sae {
namespace {

constexpr int kBN = 128;       // channels of x of a tile

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == SAE_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// the low or high halves of two words, as a word (low half: a's)
template <bool HIGH>
__device__ __forceinline__ unsigned halves(unsigned a, unsigned b) {
#ifdef HIPEMU
    return HIGH ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | (b << 16);
#else
    return __builtin_amdgcn_perm(b, a, HIGH ? 0x07060302u : 0x05040100u);
#endif
}
// two values that are exact in 16 bits, as a word
template <int DT>
__device__ __forceinline__ unsigned pack_exact(float a, float b) {
    if constexpr (DT == SAE_F16) return (unsigned)narrow<DT>(a) | ((unsigned)narrow<DT>(b) << 16);
    else return halves<true>(f_bits(a), f_bits(b));
}

// sum + the two 16-bit values of a word, widened
template <int DT>
__device__ __forceinline__ float add_pair(float sum, unsigned w) {
#ifdef HIPEMU
    return sum + (widen<DT>((uint16_t)(w & 0xffffu)) + widen<DT>((uint16_t)(w >> 16)));
#else
    if constexpr (DT == SAE_BF16) {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, w), __builtin_bit_cast(v2, 0x3f803f80u), sum, false);
    } else {
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, w), __builtin_bit_cast(v2, 0x3c003c00u), sum, false);
    }
#endif
}

struct WgShape {
    int64_t rows;
    int out, c, blocks;
    int tiles_m, tiles_n, slices;
    int64_t slice_rows;
};

// A slice's rows of a tensor behind a range-checked descriptor: a row behind the last reads as zero, without a mask
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

// A thread's 4 rows x CH channels of gy, as loaded: 16 bytes of each row (4 or 8 channels), at dword addresses.  Where a row ends inside
// them, the channels behind its end are whatever follows; they only meet outputs that are not there.  ODD: 16-bit rows of odd length,
// every other one of which starts in the middle of a dword -- rows 1 and 3: five dwords from half a dword in front.
template <int DT, bool ODD>
struct GyBox {
    using T = typename Elem<DT>::T;
    static constexpr int CH = 16 / (int)sizeof(T);
    u32x4 q[4];
    unsigned fifth[2]; // of rows 1 and 3
    // row i: r0 + mine + i of a slice of `rows` (r0, the same in a wave, is in the scalar offset, which stays within the descriptor;
    // mine, a multiple of four, and the channel are in the lane's offset `at`)
    __device__ __forceinline__ void load(int i, __amdgpu_buffer_rsrc_t all, unsigned at, int r0, int rows, int out) {
        const bool on = r0 + i < rows;
        const unsigned from = (unsigned)(on ? r0 + i : rows) * (unsigned)out * (unsigned)sizeof(T);
        if (ODD && (i & 1)) {
            const unsigned whole = on ? from - 2u : (from + 3u) & ~3u;
            q[i] = __builtin_amdgcn_raw_buffer_load_b128(all, at, whole, 0);
            fifth[i >> 1] = __builtin_amdgcn_raw_buffer_load_b32(all, at + 16u, whole, 0);
        } else {
            q[i] = __builtin_amdgcn_raw_buffer_load_b128(all, at, ODD ? (from + 3u) & ~3u : from, 0);
        }
    }
    __device__ __forceinline__ float value(int i, int j) const { return bits_f(q[i][j]); }      // (f32)
    // channels 2 k and 2 k + 1 of row i (16-bit types); have: rows that are there (ODD: half a dword behind the last one is not)
    __device__ __forceinline__ unsigned word(int i, int k, int have) const {
        unsigned w = q[i][k];
        if constexpr (ODD) {
            if (i & 1) w = (w >> 16) | ((k < 3 ? q[i][(k + 1) & 3] : fifth[i >> 1]) << 16);
            if (i >= have) w = 0u;
        }
        return w;
    }
    // channel j of rows i and i + 1, as a word
    __device__ __forceinline__ unsigned pair(int i, int j, int have) const {
        const unsigned a = word(i, j >> 1, have), b = word(i + 1, j >> 1, have);
        return j & 1 ? halves<true>(a, b) : halves<false>(a, b);
    }
};

// the rest of v behind its high 8 bits (cut, not rounded: the rest is exact); ODD: an infinity or NaN has none
template <bool ODD>
__device__ __forceinline__ float rest8(float v) {
    const float rest = v - bits_f(f_bits(v) & 0xffff0000u);
    if constexpr (ODD) return (f_bits(v) & 0x7f800000u) == 0x7f800000u ? 0.0f : rest;
    else return rest;
}

template <int DT, int BM>
struct WgTile {
    static constexpr int PL = DT == SAE_F32 ? 3 : 1;              // pieces of gy
    static constexpr int KR = DT == SAE_F32 ? 32 : 64;            // rows of a step: 2 x 56 (f32) or 2 x 48 KB of LDS at BM = 256
    static constexpr int OCT = KR / 8;
    static constexpr int GROUPS = BM == 256 ? 2 : 1;              // of four waves, each with a share of a step's rows: two waves a SIMD
    static constexpr int T = 256 * GROUPS;                        // threads
    static constexpr int CH = DT == SAE_F32 ? 4 : 8;              // channels of gy of a thread's box (4 rows of them: GyBox)
    static constexpr int AQ = BM / CH * (KR / 4);                 // boxes of a step
    static constexpr int NA = AQ / T > 0 ? AQ / T : 1;            // of a thread
    static constexpr int AR = T / (BM / CH);                      // row quads that the threads cover at once
    static constexpr int BQ = kBN / 4 * (KR / 4);                 // codes quads of a step
    static constexpr int NB = BQ / T > 0 ? BQ / T : 1;            // of a thread
    static constexpr int BR = (T < BQ ? T : BQ) / 32;             // row quads of codes at once
    static constexpr int BJ = T > BQ ? 2 : 4;                     // codes of a quad that a thread takes of each row
    static constexpr int WM = BM == 256 ? 2 : 1;                  // 32-channel tiles of a wave: 64 x 128 (BM 256),
    static constexpr int WN = BM == 64 ? 2 : 4;                   // 32 x 128 (128), 32 x 64 (64)
    static constexpr int CELLS = OCT * (PL * BM + kBN);           // 16-byte cells of a step
    // position of channel CH q + j of gy: groups of 128 channels, G j + q inside; and the channel of a position
    static constexpr int G = (BM < 128 ? BM : 128) / CH;
    static __device__ __forceinline__ int place(int q, int j) { return q / G * 128 + G * j + q % G; }
    static __device__ __forceinline__ int channel(int at) { return (at >> 7) * 128 + CH * (at % G) + (at & 127) / G; }
};

template <int DT, int BM, bool ODD, bool WHOLE>
__global__ __launch_bounds__((WgTile<DT, BM>::T), 2)
void linear_wgrad8_kernel(const typename Elem<DT>::T* __restrict__ gy, const int8_t* __restrict__ codes,
                          const uint8_t* __restrict__ scales, float* __restrict__ part, float* __restrict__ part_b,
                          typename Elem<DT>::T* __restrict__ gw, typename Elem<DT>::T* __restrict__ gb, float alpha, const WgShape p) {
    using W = WgTile<DT, BM>;
    using T = typename Elem<DT>::T;
    constexpr int PL = W::PL, KR = W::KR, OCT = W::OCT, NA = W::NA, NB = W::NB, WM = W::WM, WN = W::WN, AR = W::AR,
                  CH = W::CH, BR = W::BR, BJ = W::BJ, GROUPS = W::GROUPS;
    __shared__ u32x4 cells[2][W::CELLS];                          // of a step: gy [PL][OCT][BM], codes [OCT][kBN]
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wid = wave & 3, group = wave >> 2;
    // Work-groups go round the eight XCDs.  Each XCD takes a run of neighbouring (slice, tile row, tile column): whole slices where
    // there are eight or more, else tile rows of one, so that its L2 reads a tile of gy once for all the columns beside it.
    const int tiles = p.tiles_m * p.tiles_n, all = (int)gridDim.x, xcd = blockIdx.x & 7;
    const int run = xcd * (all >> 3) + (xcd < (all & 7) ? xcd : (all & 7)) + (int)(blockIdx.x >> 3);
    const int slice = run / tiles, tile = run - slice * tiles;
    const int tn = tile % p.tiles_n, tm = tile / p.tiles_n;
    const int o0 = tm * BM, i0 = tn * kBN;
    const int64_t r_begin = slice * p.slice_rows;
    const int64_t r_end = r_begin + p.slice_rows < p.rows ? r_begin + p.slice_rows : p.rows;
    const int rows = (int)(r_end - r_begin), steps = (rows + KR - 1) / KR;
    const int64_t behind = p.rows - r_begin;                      // (a slice has fewer than 2^26 rows)
    const int last = (int)(behind < (1 << 30) ? behind : 1 << 30) - 4;
    const int64_t ld = (int64_t)p.blocks * kBlk8;

    f32x16 acc[WM][WN];
    float sum[2 * CH];                                            // gb (the thread's channels are the same in every step), in two shares
    float pace[NB][4];                                            // steps 2^k of the codes' rows

    // what a step's loads bring a thread; two steps are under way
    struct Load {
        GyBox<DT, ODD> g[NA];
        unsigned cw[NB][4], ce[NB];
    };
    Load load[2];
    // neighbouring lanes take the two row quads of a cell: their 8-byte writes fill whole cells, without a bank conflict
    const int oq = (tid >> 1) % (BM / CH), ar = (tid & 1) + 2 * (tid / (2 * BM / CH));   // gy: channels, row quad (of every AR)
    const int bt = tid % (32 * BR), bj = BJ * (tid / (32 * BR));  // (twice as many threads as quads: two codes of each)
    const int bq = (bt >> 1) & 31, br = (bt & 1) + 2 * (bt >> 6);                        // codes: channel quad, row quad (of every BR)
    const bool a_in = W::AQ >= W::T || ar < KR / 4, b_in = i0 + 4 * bq < ld;
    const __amdgpu_buffer_rsrc_t grows = rows_of(gy + r_begin * p.out, ((int64_t)rows * p.out * (int64_t)sizeof(T) + 3) & ~(int64_t)3);
    const __amdgpu_buffer_rsrc_t crows = rows_of(codes + r_begin * ld, rows * ld);
    const uint8_t* const ssrc = scales + (int64_t)(b_in ? (i0 + 4 * bq) / kBlk8 : 0) * p.rows + r_begin;
    const unsigned nowhere = 0xfffffff0u;                         // behind every descriptor
    const unsigned gat = a_in && o0 + CH * oq < p.out
                             ? ((unsigned)(4 * ar) * (unsigned)p.out + (unsigned)(o0 + CH * oq)) * (unsigned)sizeof(T) : nowhere;
    const unsigned cat = b_in ? (unsigned)(4 * br) * (unsigned)ld + (unsigned)(i0 + 4 * bq + bj) : nowhere;

    auto fetch_gy = [&](Load& to, int step, int n) {              // n < 4 NA: one row of a box
        to.g[n >> 2].load(n & 3, grows, gat, step * KR + 4 * AR * (n >> 2), rows, p.out);
    };
    auto fetch_codes = [&](Load& to, int step, int n) {           // n < 5 NB: four rows of a quad, and their exponents
        const int q = n / 5, i = n % 5;
        if (i < 4) {
            const int from = step * KR + 4 * BR * q + i;
            const unsigned at = (unsigned)(from < rows ? from : rows) * (unsigned)ld;
            if constexpr (BJ == 4) to.cw[q][i] = __builtin_amdgcn_raw_buffer_load_b32(crows, cat, at, 0);
            else to.cw[q][i] = __builtin_amdgcn_raw_buffer_load_b16(crows, cat, at, 0);
            return;
        }
        const int r = step * KR + 4 * (br + BR * q);
        // (f32: no branch in a step's schedule, 202 -> 198 us; in the 16-bit types the same branch, never taken, is worth 59.4 -> 57.8)
        if ((DT == SAE_F32 && !(BM == 64 && WHOLE)) || p.rows >= 4) {          // a word that ends at the block's last row at most
            __builtin_memcpy(&to.ce[q], ssrc + (r < last ? r : last), 4);
        } else {                                                  // (wg_plan: 64-tall tiles, one slice)
            to.ce[q] = 0;
            for (int i = 0; i < rows; ++i) to.ce[q] |= (unsigned)ssrc[i] << (8 * i);
            to.ce[q] <<= 8 * -last;
        }
    };
    auto fetch = [&](Load& to, int step, bool all_of_it) {
#pragma unroll
        for (int n = 0; n < 4 * NA; ++n) fetch_gy(to, step, n);
        if (all_of_it)
#pragma unroll
            for (int n = 0; n < 5 * NB; ++n) fetch_codes(to, step, n);
    };
    auto put = [&](u32x4* cell, int rq, unsigned lo, unsigned hi) { *(reinterpret_cast<u32x2*>(cell) + (rq & 1)) = u32x2{lo, hi}; };
    // One channel of a box: of gy (n < CH NA) or of the codes.  odd: with infinities and NaN among the values (f32)
    constexpr int PIECES = CH * NA + BJ * NB;
    auto stage = [&](const Load& from, int step, u32x4* to, int n, auto odd) {
        if (n < CH * NA) {
            const int q = n / CH, j = n % CH, rq = ar + AR * q;
            u32x4* const row = to + (rq >> 1) * BM + W::place(oq, j);
            if constexpr (DT == SAE_F32) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = from.g[q].value(i, j);
                    sum[(i & 1) * CH + j] += v[i];
                    if (odd.value && v[i] != v[i]) v[i] = bits_f(0x7fc00000u);       // (a NaN of low bits alone is cut to infinity)
                }
#pragma unroll
                for (int s = 0; s < 3; ++s) {
                    if (W::AQ >= W::T || rq < KR / 4)
                        put(row + s * OCT * BM, rq, pack_exact<DT>(v[0], v[1]), pack_exact<DT>(v[2], v[3]));
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = rest8<odd.value>(v[i]);
                }
            } else {
                const int have = rows - (step * KR + 4 * rq);
                const unsigned lo = from.g[q].pair(0, j, have), hi = from.g[q].pair(2, j, have);
                sum[j] = add_pair<DT>(sum[j], lo);
                sum[CH + j] = add_pair<DT>(sum[CH + j], hi);
                if (W::AQ >= W::T || rq < KR / 4) put(row, rq, lo, hi);
            }
        } else {
            const int m = n - CH * NA, q = m / BJ, j = m % BJ, rq = br + BR * q;
            if (j == 0) {                                         // the word of exponents shifted, and cut to the slice's rows
                const int r = step * KR + 4 * rq, by = r > last ? r - last : 0;
                const int have = rows - r < 0 ? 0 : rows - r < 4 ? rows - r : 4;
                const unsigned e = (from.ce[q] >> (8 * (by & 3))) & (unsigned)(((uint64_t)1 << (8 * have)) - 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) pace[q][i] = block8_step((e >> (8 * i)) & 0xffu);
            }
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(from.cw[q][i] >> (8 * j)) * pace[q][i];
            put(to + PL * OCT * BM + (rq >> 1) * kBN + 32 * (bj + j) + bq, rq, pack_exact<DT>(v[0], v[1]), pack_exact<DT>(v[2], v[3]));
        }
    };
    // The products of a step out of `from`, and between them, a share behind each PL-th part, whatever `beside` does: matrix cores
    // and vector units work at the same time.  Operands are read one part ahead.
    constexpr int PARTS = KR / 16 / GROUPS * PL;
    auto multiply = [&](const u32x4* from, auto beside) {
        u32x4 bf[2][WN], af[2][WM];
        auto read = [&](int part) {
            const int sixteen = part / PL, k = part % PL, s = GROUPS * sixteen + group;
            if (k == 0)
#pragma unroll
                for (int n = 0; n < WN; ++n)
                    bf[sixteen & 1][n] = from[PL * OCT * BM + (2 * s + half) * kBN + 32 * (BM == 64 ? 2 * (wid & 1) + n : n) + l31];
#pragma unroll
            for (int m = 0; m < WM; ++m)
                af[part & 1][m] = from[(k * OCT + 2 * s + half) * BM + 32 * (BM == 64 ? wid >> 1 : wid * WM + m) + l31];
        };
        read(0);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            if (part + 1 < PARTS) read(part + 1);
#pragma unroll
            for (int m = 0; m < WM; ++m)
#pragma unroll
                for (int n = 0; n < WN; ++n) acc[m][n] = mma<DT>(af[part & 1][m], bf[(part / PL) & 1][n], acc[m][n]);
            beside(part);
            // operand reads, then a product, a share of the vector work and of the memory instructions in turn: a wave issues in
            // order, and loads that come in a burst wait for the CU's one address unit with every product behind them
            __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
            for (int i = 0; i < WM * WN; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, DT == SAE_F32 ? 6 : 9, 0);    // (the other way round: 1 % more each)
                __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto clear = [&]() {
#pragma unroll
        for (int m = 0; m < WM; ++m)
#pragma unroll
            for (int n = 0; n < WN; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[m][n][r] = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * CH; ++j) sum[j] = 0.0f;
    };

    clear();
    fetch(load[0], 0, true);
    fetch(load[1], 1, true);
#pragma unroll
    for (int n = 0; n < PIECES; ++n) stage(load[0], 0, cells[0], n, BoolTag<false>());
    fetch(load[0], 2, false);
    __syncthreads();
    // Step t: products of cells[t & 1]; what was loaded of step t + 1 goes to the other cells, and step t + 3 of gy is asked for into
    // the registers that this frees, step t + 2 of the codes into those freed in the step before.  (Steps behind the last are zeros.)
    constexpr int LOADS = 5 * NB + 4 * NA;
    auto turn = [&](int step, Load& next, Load& before, const u32x4* from, u32x4* to) {
        multiply(from, [&](int part) {
#pragma unroll
            for (int n = PIECES * part / PARTS; n < PIECES * (part + 1) / PARTS; ++n) stage(next, step + 1, to, n, BoolTag<false>());
#pragma unroll
            for (int n = 0; n < LOADS; ++n) {
                if (n * PARTS / LOADS != part) continue;
                if (n < 5 * NB) {
                    fetch_codes(before, step + 2, n);
                } else {
                    const int m = n - 5 * NB;                     // (its box is staged by then)
                    static_assert(5 * NB * PARTS / LOADS >= (CH - 1) * PARTS / PIECES && (LOADS - 4) * PARTS / LOADS >= (CH * NA - 1) * PARTS / PIECES, "order");
                    fetch_gy(next, step + 3, m);
                }
            }
        });
        __syncthreads();
    };
    for (int step = 0; step < steps; step += 2) {
        turn(step, load[1], load[0], cells[0], cells[1]);
        if (step + 1 < steps) turn(step + 1, load[0], load[1], cells[1], cells[0]);
    }
    if constexpr (DT == SAE_F32) {
        // An infinity or NaN in gy makes the rest behind its high piece a NaN, and with it the whole row of the tile: such a tile is
        // computed again with the pieces of these values set right.
        float zero = 0.0f;
#pragma unroll
        for (int m = 0; m < WM; ++m)
#pragma unroll
            for (int n = 0; n < WN; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) zero = fmaf(acc[m][n][r], 0.0f, zero);
        int* const flag = reinterpret_cast<int*>(&cells[0][0]);
        if (tid == 0) *flag = 0;
        __syncthreads();
        if (zero != 0.0f || zero != zero) *flag = 1;
        __syncthreads();
        const bool again = *flag != 0;
        __syncthreads();
        if (again) {
            clear();
            for (int step = 0; step < steps; ++step) {
                fetch(load[0], step, true);
#pragma unroll
                for (int n = 0; n < PIECES; ++n) stage(load[0], step, cells[0], n, BoolTag<true>());
                __syncthreads();
                multiply(cells[0], [](int) {});
                __syncthreads();
            }
        }
    }

    // Two groups: each keeps half of the accumulator registers, 8 g ... 8 g + 7, and takes the other's share of them through LDS.
    // Register r of the lane: tile row (r & 3) + 8 (r >> 2) + 4 half, tile column l31.
    float* const swap = reinterpret_cast<float*>(&cells[0][0]);
    static_assert(GROUPS == 1 || 2 * W::CELLS * 16 >= 8 * WN * 8 * 64 * 4, "the exchange fits into the cells");
#pragma unroll
    for (int m = 0; m < WM; ++m) {
        if constexpr (GROUPS == 2) {
            if (m > 0) __syncthreads();
#pragma unroll
            for (int n = 0; n < WN; ++n)
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const float low = acc[m][n][r], high = acc[m][n][r + 8];
                    swap[((wave * WN + n) * 8 + r) * 64 + lane] = group == 0 ? high : low;
                }
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < 16 / GROUPS; ++r) {
            const int rr = r + 8 * group;
            const int at = 32 * (BM == 64 ? wid >> 1 : wid * WM + m) + (rr & 3) + 8 * (rr >> 2) + 4 * half;
            const int o = o0 + W::channel(at), i = i0 + 4 * l31 + (BM == 64 ? 2 * (wid & 1) : 0);
            float v[WN];
#pragma unroll
            for (int n = 0; n < WN; ++n) {
                if constexpr (GROUPS == 2) {
                    const float low = acc[m][n][r], high = acc[m][n][(r + 8) & 15];
                    v[n] = (group == 0 ? low : high) + swap[(((wave ^ 4) * WN + n) * 8 + r) * 64 + lane];
                } else {
                    v[n] = acc[m][n][r];
                }
            }
            if (o >= p.out) continue;
            if constexpr (WHOLE) {
                T* const dst = gw + (int64_t)o * p.c + i;
#pragma unroll
                for (int n = 0; n < WN; ++n)
                    if (i + n < p.c) store_one<DT>(dst + n, alpha * v[n]);
            } else if (i < ld) {
                float* const dst = part + ((int64_t)slice * p.out + o) * ld + i;
                // (past the caches: written once, read once; 67 -> 64 us on bf16 65536 x 512 x 512)
                if constexpr (WN == 4) __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(dst));
                else __builtin_nontemporal_store(f32x2{v[0], v[1]}, reinterpret_cast<f32x2*>(dst));
            }
        }
    }
    if (tn == 0 && (WHOLE ? gb != nullptr : part_b != nullptr)) {      // the row quads' sums of each channel, added in order
        constexpr int AG = AR < KR / 4 ? AR : KR / 4;                  // row quads that have one
        float* const fold = swap;
        __syncthreads();
        if (ar < AG)
#pragma unroll
            for (int j = 0; j < CH; ++j) fold[ar * BM + CH * oq + j] = sum[j] + sum[CH + j];
        __syncthreads();
        for (int o = tid; o < BM; o += W::T) {
            float t = fold[o];
            for (int rq = 1; rq < AG; ++rq) t += fold[rq * BM + o];
            if (o0 + o >= p.out) continue;
            if constexpr (WHOLE) store_one<DT>(gb + o0 + o, t);
            else part_b[(int64_t)slice * p.out + o0 + o] = t;
        }
    }
}

// gw[o][i] = alpha * the sum of the slices' tiles; gb likewise.  64 quads of channels a work-group, four threads each: a quarter of
// the slices in order, the quarters in order behind it.
template <int DT>
__global__ __launch_bounds__(kBlock) void linear_wgrad8_reduce_kernel(const float* __restrict__ part, const float* __restrict__ part_b,
                                                                      typename Elem<DT>::T* __restrict__ gw,
                                                                      typename Elem<DT>::T* __restrict__ gb, float alpha, const WgShape p) {
    __shared__ f32x4 quarter[3][64];
    const int64_t ld = (int64_t)p.blocks * kBlk8, size = (int64_t)p.out * ld;
    const int lane = threadIdx.x & 63, part4 = threadIdx.x >> 6;
    const int64_t e = ((int64_t)blockIdx.x * 64 + lane) * 4;
    const int per = (p.slices + 3) / 4, first = part4 * per, end = first + per < p.slices ? first + per : p.slices;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (e < size)
#pragma unroll 8
        for (int s = first; s < end; ++s) {
            const f32x4 t = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(part + s * size + e));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += t[j];
        }
    if (part4 > 0) quarter[part4 - 1][lane] = v;
    __syncthreads();
    if (part4 == 0 && e < size) {
        const int64_t o = e / ld, i = e - o * ld;
        float one[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) one[j] = alpha * (((v[j] + quarter[0][lane][j]) + quarter[1][lane][j]) + quarter[2][lane][j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j < p.c) store_one<DT>(gw + o * p.c + i + j, one[j]);
        }
    }
    const int64_t u = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (gb && u < p.out) {
        float w = part_b[u];
        for (int s = 1; s < p.slices; ++s) w += part_b[(int64_t)s * p.out + u];
        store_one<DT>(gb + u, w);
    }
}

template <int DT>
__global__ __launch_bounds__(kBlock) void fill_zero_kernel(typename Elem<DT>::T* __restrict__ gw, typename Elem<DT>::T* __restrict__ gb,
                                                           int64_t size, int64_t out) {
    const int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (e < size) gw[e] = 0;
    if (gb && e < out) gb[e] = 0;
}

int wg_rows(int32_t dtype) { return dtype == SAE_F32 ? 32 : 64; }      // WgTile::KR

struct WgPlan {
    int bm;
    WgShape p;
};

// The tallest tile that leaves no CU without a work-group of four steps (256: one of eight waves a CU; 128, 64: two of four; bf16
// 65536 x 512 x 512 takes 58 us in tiles of 256, 65 of 128 and 90 of 64).  Slices so that the work-groups fill the chip once.
WgPlan wg_plan(int64_t rows, int64_t out, int64_t c, int32_t dtype) {
    const int kr = wg_rows(dtype);
    const int64_t steps = ceil_div64(rows, kr), pairs = ceil_div64(steps, 4), tiles_n = ceil_div64(c, kBN);
    int bm = 64;                                                            // (fewer than four rows: the form that reads so few)
    for (int t = 256; t > 64 && rows >= 4; t /= 2)
        if (out > t / 2 && ceil_div64(out, t) * tiles_n * pairs >= 256) { bm = t; break; }
    const int forced = tuning_knob("SAE_WG_TILE", 0);                       // (tests: every height at small sizes)
    if (forced && rows >= 4) bm = forced;
    const int64_t full = bm == 256 ? 256 : 512;
    WgPlan w;
    w.bm = bm;
    w.p.rows = rows;
    w.p.out = (int)out;
    w.p.c = (int)c;
    w.p.blocks = (int)ceil_div64(c, kBlk8);
    w.p.tiles_m = (int)ceil_div64(out, bm);
    w.p.tiles_n = (int)tiles_n;
    const int64_t tiles = ceil_div64(out, bm) * tiles_n;
    int64_t best = 1;
    if (tiles < full) {
        best = full / tiles;
        if (best > 8) best = best / 8 * 8;                                  // (whole slices on each of the eight XCDs)
    }
    if (best > pairs) best = pairs;
    // a slice's rows lie behind one descriptor with 32-bit offsets
    const int64_t widest = ceil_div64(c, kBlk8) * kBlk8 > 4 * out ? ceil_div64(c, kBlk8) * kBlk8 : 4 * out;
    const int64_t least = ceil_div64(rows, ((int64_t)1 << 30) / widest / kr * kr);
    if (best < least) best = least;
    w.p.slice_rows = ceil_div64(steps, best) * kr;
    w.p.slices = (int)ceil_div64(rows, w.p.slice_rows);
    return w;
}

int64_t wg_workspace(const WgPlan& w) {
    return w.p.slices == 1 ? 0 : (int64_t)w.p.slices * w.p.out * ((int64_t)w.p.blocks * kBlk8 + 1);
}

bool wg_shape_ok(int64_t rows, int64_t out, int64_t c) {
    return rows >= 0 && out >= 1 && c >= 1 && out <= (1 << 20) && c <= (1 << 20) && out * c <= ((int64_t)1 << 31) &&
           rows <= ((int64_t)1 << 40) / (out + c);
}

template <int DT, int BM, bool ODD>
void wg_launch(const void* gy, const int8_t* codes, const uint8_t* scales, float* part, float* part_b, void* gw, void* gb, float alpha,
               const WgShape& p, hipStream_t s) {
    using T = typename Elem<DT>::T;
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n * p.slices)), block((unsigned)WgTile<DT, BM>::T);
    if (p.slices == 1)
        hipLaunchKernelGGL((linear_wgrad8_kernel<DT, BM, ODD, true>), grid, block, 0, s, (const T*)gy, codes, scales, part, part_b,
                           (T*)gw, (T*)gb, alpha, p);
    else
        hipLaunchKernelGGL((linear_wgrad8_kernel<DT, BM, ODD, false>), grid, block, 0, s, (const T*)gy, codes, scales, part, part_b,
                           (T*)gw, (T*)gb, alpha, p);
}

template <int DT>
int wg_run(const void* gy, const int8_t* codes, const uint8_t* scales, void* gw, void* gb, int64_t rows, int64_t out, int64_t c,
           float alpha, float* ws, hipStream_t s) {
    using T = typename Elem<DT>::T;
    if (rows == 0) {
        hipLaunchKernelGGL((fill_zero_kernel<DT>), dim3((unsigned)ceil_div64(out * c, kBlock)), dim3(kBlock), 0, s, (T*)gw, (T*)gb,
                           out * c, out);
        return check_launch("sae_linear_wgrad8");
    }
    const WgPlan w = wg_plan(rows, out, c, DT);
    const WgShape& p = w.p;
    float* part_b = gb ? ws + (int64_t)p.slices * out * p.blocks * kBlk8 : nullptr;
#define SAE_WG(BM)                                                                                                              \
    if (DT != SAE_F32 && out % 2 != 0)                                                                                          \
        wg_launch<DT, BM, DT != SAE_F32>(gy, codes, scales, ws, part_b, gw, gb, alpha, p, s);                                   \
    else wg_launch<DT, BM, false>(gy, codes, scales, ws, part_b, gw, gb, alpha, p, s)
    if (w.bm == 64) { SAE_WG(64); }
    else if (w.bm == 128) { SAE_WG(128); }
    else { SAE_WG(256); }
#undef SAE_WG
    if (p.slices > 1)
        hipLaunchKernelGGL((linear_wgrad8_reduce_kernel<DT>), dim3((unsigned)ceil_div64(out * p.blocks * kBlk8, 256)),
                           dim3(kBlock), 0, s, (const float*)ws, (const float*)part_b, (T*)gw, (T*)gb, alpha, p);
    return check_launch("sae_linear_wgrad8");
}

}  // namespace
}  // namespace sae

using namespace sae;

extern "C" int64_t sae_linear_wgrad8_workspace(int64_t rows, int64_t out, int64_t c, int32_t dtype) {
    if (!wg_shape_ok(rows, out, c) || !elem_known(dtype) || rows == 0) return 0;
    return wg_workspace(wg_plan(rows, out, c, dtype));
}

extern "C" int sae_linear_wgrad8(const void* gy, const int8_t* codes, const uint8_t* scales, void* gw, void* gb, int64_t rows,
                                 int64_t out, int64_t c, float alpha, int32_t dtype, float* workspace, int64_t workspace_floats,
                                 sae_stream_t stream) {
    sae::clear_stale_error();
    if (!elem_known(dtype)) return fail(SAE_EINVAL, "sae_linear_wgrad8: unknown element type %d", (int)dtype);
    if (!wg_shape_ok(rows, out, c)) return fail(SAE_EINVAL, "sae_linear_wgrad8: bad shape");
    if (!gw || (rows > 0 && (!gy || !codes || !scales))) return fail(SAE_EINVAL, "sae_linear_wgrad8: null tensor");
    if (rows > 0 && (!aligned16(codes) || !aligned16(workspace) || !aligned16(gy)))
        return fail(SAE_EINVAL, "sae_linear_wgrad8: misaligned tensor");
    const int64_t need = sae_linear_wgrad8_workspace(rows, out, c, dtype);
    if (need > 0 && (!workspace || workspace_floats < need))
        return fail(SAE_EWORKSPACE, "sae_linear_wgrad8: workspace %lld < %lld floats (sae_linear_wgrad8_workspace)",
                    (long long)workspace_floats, (long long)need);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == SAE_F32) return wg_run<SAE_F32>(gy, codes, scales, gw, gb, rows, out, c, alpha, workspace, s);
    if (dtype == SAE_BF16) return wg_run<SAE_BF16>(gy, codes, scales, gw, gb, rows, out, c, alpha, workspace, s);
    return wg_run<SAE_F16>(gy, codes, scales, gw, gb, rows, out, c, alpha, workspace, s);
}
