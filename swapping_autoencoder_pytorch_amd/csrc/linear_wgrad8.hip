// Weight gradient of a linear layer (or 1 x 1 convolution, channels last) from the 8-bit checkpoint of its input (elem8.inc):
//
//     gw[o][i] = alpha * sum over r of gy[r][o] * x8[r][i],     gb[o] = sum over r of gy[r][o]
//
// on the 16-bit matrix cores with fp32 accumulation, without a rounding in front of the sum:
//     x8 = q * 2^k has 8 significant bits at most: a bf16 (and, with k >= -24, an f16) value exactly
//     gy in bf16 / f16 is taken as it is
//     gy in f32 is cut into three bf16 pieces of 8 bits each, high + middle + low = gy exactly, and takes three products
// v_mfma_f32_32x32x16 at 3 products is ~5 times v_mfma_f32_32x32x2_f32's rate: keeping x in 8 bits makes the f32 weight gradient
// faster than the exact f32 product of the full-width tensors, not only smaller.
//
// Tile: BM channels of gy x 128 channels of x, 32 rows at a time.  The sum runs over ROWS, the slow axis of both tensors, while a
// matrix-core operand wants 8 rows of one channel next to each other: a thread loads 4 channels of 4 rows (16 bytes a row of f32
// gy, 4 bytes a row of codes), and writes for each of its 4 channels the 4 rows packed to 8 bytes.  LDS holds 16-byte cells
// [k octet][position], where channel 4 j + m of a group of 128 sits at position 32 m + j: lanes that stage neighbouring quads
// write neighbouring cells, an operand is one 16-byte read with neighbouring lanes on neighbouring cells, and a lane ends up with
// the 4 neighbouring output channels 4 j ... 4 j + 3 in its 4 accumulators -- whole 16-byte stores, no shuffle.
//
// Few tiles: the rows are cut into slices, one work-group each, whose fp32 tiles a second kernel adds in order.
#include "elem8.inc"

namespace sae {
namespace {

constexpr int kBN = 128;       // channels of x of a tile
constexpr int kRows = 32;      // rows of a step
constexpr int kOct = kRows / 8;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == SAE_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two values that are exact in 16 bits, as a word (low half: the first)
template <int DT>
__device__ __forceinline__ unsigned pack_exact(float a, float b) {
    if constexpr (DT == SAE_F16) return (unsigned)narrow<DT>(a) | ((unsigned)narrow<DT>(b) << 16);
    else return (f_bits(a) >> 16) | (f_bits(b) & 0xffff0000u);
}

struct WgShape {
    int64_t rows;
    int out, c, blocks;
    int tiles_m, tiles_n, slices;
    int64_t slice_rows;
};

// A thread's 4 rows x 4 channels of gy, as loaded
template <int DT, bool VEC>
struct GyQuad {
    float f[4][4];     // f32
    u32x2 h[4];        // 16-bit types: 4 channels of a row
    __device__ __forceinline__ void load(const typename Elem<DT>::T* __restrict__ gy, int64_t r0, int64_t r_end, int o, int out) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool on = r0 + i < r_end;
            const typename Elem<DT>::T* p = gy + (r0 + i) * (int64_t)out + o;
            if constexpr (VEC) {                                   // out % 4 == 0: the quad is there or not
                const bool in = on && o < out;
                if constexpr (DT == SAE_F32) {
                    f32x4 q = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (in) q = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[i][j] = q[j];
                } else {
                    h[i] = u32x2{0u, 0u};
                    if (in) h[i] = *reinterpret_cast<const u32x2*>(p);
                }
            } else if constexpr (DT == SAE_F32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) f[i][j] = on && o + j < out ? p[j] : 0.0f;
            } else {
                unsigned v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = on && o + j < out ? p[j] : 0u;
                h[i] = u32x2{v[0] | (v[1] << 16), v[2] | (v[3] << 16)};
            }
        }
    }
    __device__ __forceinline__ unsigned half(int i, int j) const { return (h[i][j >> 1] >> (16 * (j & 1))) & 0xffffu; }
    __device__ __forceinline__ float value(int i, int j) const {
        if constexpr (DT == SAE_F32) return f[i][j];
        else return widen<DT>((uint16_t)half(i, j));
    }
};

// high part of v in 8 bits (cut, not rounded: the rest is exact); an infinity or NaN has no rest
__device__ __forceinline__ float cut8(float v) { return bits_f(f_bits(v) & 0xffff0000u); }

template <int DT, int BM, bool VEC>
__global__ __launch_bounds__(kBlock) void linear_wgrad8_kernel(const typename Elem<DT>::T* __restrict__ gy,
                                                               const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                               float* __restrict__ part, float* __restrict__ part_b, const WgShape p) {
    constexpr int PL = DT == SAE_F32 ? 3 : 1;                     // pieces of gy
    constexpr int NQ = BM / 4 * (kRows / 4) / kBlock > 0 ? BM / 4 * (kRows / 4) / kBlock : 1;   // gy quads of a thread
    constexpr int MT = BM / 64;                                   // 32-channel tiles of gy in a wave: 64 x 128 (BM 256) ...
    constexpr int WN = BM >= 128 ? 4 : 2;                         // ... 32 x 128 (128), 32 x 64 (64)
    static_assert(BM == 64 || BM == 128 || BM == 256, "tile");
    constexpr int WM = BM == 256 ? 2 : 1;
    (void)MT;
    __shared__ u32x4 As[PL][kOct][BM];
    __shared__ u32x4 Bs[kOct][kBN];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, l31 = lane & 31, half = lane >> 5;
    // slices of the same rows on one XCD (work-groups go round the eight of them): its L2 serves the tiles' shared reads
    const int tiles = p.tiles_m * p.tiles_n;
    const int slice = blockIdx.x / tiles, tile = blockIdx.x - slice * tiles;
    const int tn = tile % p.tiles_n, tm = tile / p.tiles_n;
    const int o0 = tm * BM, i0 = tn * kBN;
    const int64_t r_begin = slice * p.slice_rows;
    const int64_t r_end = r_begin + p.slice_rows < p.rows ? r_begin + p.slice_rows : p.rows;

    f32x16 acc[WM][WN];
#pragma unroll
    for (int m = 0; m < WM; ++m)
#pragma unroll
        for (int n = 0; n < WN; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[m][n][r] = 0.0f;
    float sum[NQ][4];
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[q][j] = 0.0f;

    const int bq = tid & 31, br = tid >> 5;                       // codes: channel quad, row quad
    const int bc = i0 + 4 * bq;
    const bool b_in = bc < p.blocks * kBlk8;
    const int8_t* const bsrc = codes + (b_in ? bc : 0);
    const uint8_t* const ssrc = scales + (int64_t)(b_in ? bc / kBlk8 : 0) * p.rows;
    const int64_t ld = (int64_t)p.blocks * kBlk8;

    for (int64_t r0 = r_begin; r0 < r_end; r0 += kRows) {
        GyQuad<DT, VEC> g[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int e = tid + q * kBlock, oq = e % (BM / 4), rq = e / (BM / 4);
            g[q].load(gy, r0 + 4 * rq, rq < kRows / 4 ? r_end : r_begin, o0 + 4 * oq, p.out);
        }
        unsigned cw[4], ce[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = r0 + 4 * br + i;
            const bool on = b_in && r < r_end;
            cw[i] = on ? *reinterpret_cast<const unsigned*>(bsrc + r * ld) : 0u;
            ce[i] = on ? ssrc[r] : 0u;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int e = tid + q * kBlock, oq = e % (BM / 4), rq = e / (BM / 4);
            if (rq < kRows / 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // channel 4 oq + j: group of 128, position 32 j + (oq & 31) in it (BM = 64: 16 j + oq)
                    const int pos = BM == 64 ? 16 * j + oq : (oq >> 5) * 128 + 32 * j + (oq & 31);
                    if constexpr (DT == SAE_F32) {
                        float v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = g[q].f[i][j];
#pragma unroll
                        for (int s = 0; s < 3; ++s) {
                            u32x2* cell = reinterpret_cast<u32x2*>(&As[s][rq >> 1][pos]) + (rq & 1);
                            *cell = u32x2{pack_exact<DT>(v[0], v[1]), pack_exact<DT>(v[2], v[3])};
                            if (s < 2)
#pragma unroll
                                for (int i = 0; i < 4; ++i) v[i] = (f_bits(v[i]) & 0x7f800000u) == 0x7f800000u ? 0.0f : v[i] - cut8(v[i]);
                        }
                    } else {
                        u32x2* cell = reinterpret_cast<u32x2*>(&As[0][rq >> 1][pos]) + (rq & 1);
                        *cell = u32x2{g[q].half(0, j) | (g[q].half(1, j) << 16), g[q].half(2, j) | (g[q].half(3, j) << 16)};
                    }
                    if (tn == 0)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sum[q][j] += g[q].value(i, j);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(cw[i] >> (8 * j)) * block8_step(ce[i]);
            u32x2* cell = reinterpret_cast<u32x2*>(&Bs[br >> 1][32 * j + bq]) + (br & 1);
            *cell = u32x2{pack_exact<DT>(v[0], v[1]), pack_exact<DT>(v[2], v[3])};
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < kRows / 16; ++s) {
            u32x4 bf[WN], af[WM][PL];
#pragma unroll
            for (int n = 0; n < WN; ++n) bf[n] = Bs[2 * s + half][32 * (BM == 64 ? 2 * (wid & 1) + n : n) + l31];
#pragma unroll
            for (int m = 0; m < WM; ++m)
#pragma unroll
                for (int k = 0; k < PL; ++k) af[m][k] = As[k][2 * s + half][32 * (BM == 64 ? wid >> 1 : wid * WM + m) + l31];
#pragma unroll
            for (int k = 0; k < PL; ++k)
#pragma unroll
                for (int m = 0; m < WM; ++m)
#pragma unroll
                    for (int n = 0; n < WN; ++n) acc[m][n] = mma<DT>(af[m][k], bf[n], acc[m][n]);
        }
    }
    // accumulator register r of the lane: tile row (r & 3) + 8 (r >> 2) + 4 half, tile column l31
    float* const dst = part + (int64_t)slice * p.out * ld;
#pragma unroll
    for (int m = 0; m < WM; ++m) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int at = 32 * (BM == 64 ? wid >> 1 : wid * WM + m) + (r & 3) + 8 * (r >> 2) + 4 * half;    // position of the row
            const int o = o0 + (BM == 64 ? 4 * (at & 15) + (at >> 4) : (at >> 7) * 128 + 4 * (at & 31) + ((at >> 5) & 3));
            const int i = i0 + 4 * l31;
            if (o < p.out && i < p.blocks * kBlk8) {
                if constexpr (WN == 4)
                    *reinterpret_cast<f32x4*>(dst + (int64_t)o * ld + i) = f32x4{acc[m][0][r], acc[m][1][r], acc[m][2][r], acc[m][3][r]};
                else
#pragma unroll
                    for (int n = 0; n < WN; ++n) dst[(int64_t)o * ld + i + 2 * (wid & 1) + n] = acc[m][n][r];
            }
        }
    }
    if (tn == 0 && part_b) {       // the row quads' sums of each channel, added in order
        __syncthreads();
        float* const fold = reinterpret_cast<float*>(&As[0][0][0]);          // [kRows / 4][BM]
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int e = tid + q * kBlock, oq = e % (BM / 4), rq = e / (BM / 4);
            if (rq < kRows / 4)
#pragma unroll
                for (int j = 0; j < 4; ++j) fold[rq * BM + 4 * oq + j] = sum[q][j];
        }
        __syncthreads();
        for (int o = tid; o < BM; o += kBlock) {
            float t = fold[o];
            for (int rq = 1; rq < kRows / 4; ++rq) t += fold[rq * BM + o];
            if (o0 + o < p.out) part_b[(int64_t)slice * p.out + o0 + o] = t;
        }
    }
}

// gw[o][i] = alpha * the slices' tiles in order; gb likewise
template <int DT>
__global__ __launch_bounds__(kBlock) void linear_wgrad8_reduce_kernel(const float* __restrict__ part, const float* __restrict__ part_b,
                                                                      typename Elem<DT>::T* __restrict__ gw,
                                                                      typename Elem<DT>::T* __restrict__ gb, float alpha, const WgShape p) {
    const int64_t ld = (int64_t)p.blocks * kBlk8, size = (int64_t)p.out * ld;
    const int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (e < (int64_t)p.out * p.c) {
        const int64_t o = e / p.c, i = e - o * p.c;
        float v[1] = {part[o * ld + i]};
        for (int s = 1; s < p.slices; ++s) v[0] += part[s * size + o * ld + i];
        v[0] *= alpha;
        store_vec<DT, 1>(gw + e, v);
    }
    if (gb && e < p.out) {
        float v[1] = {part_b[e]};
        for (int s = 1; s < p.slices; ++s) v[0] += part_b[(int64_t)s * p.out + e];
        store_vec<DT, 1>(gb + e, v);
    }
}

template <int DT>
__global__ __launch_bounds__(kBlock) void fill_zero_kernel(typename Elem<DT>::T* __restrict__ gw, typename Elem<DT>::T* __restrict__ gb,
                                                           int64_t size, int64_t out) {
    const int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (e < size) gw[e] = 0;
    if (gb && e < out) gb[e] = 0;
}

int wg_tile(int64_t out) { return out <= 64 ? 64 : out <= 128 ? 128 : 256; }

WgShape wg_plan(int64_t rows, int64_t out, int64_t c) {
    WgShape p;
    p.rows = rows;
    p.out = (int)out;
    p.c = (int)c;
    p.blocks = (int)ceil_div64(c, kBlk8);
    p.tiles_m = (int)ceil_div64(out, wg_tile(out));
    p.tiles_n = (int)ceil_div64(c, kBN);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, steps = ceil_div64(rows, kRows);
    int64_t s = ceil_div64(512, tiles);                  // two work-groups per CU
    if (s > steps) s = steps;
    if (s < 1) s = 1;
    p.slice_rows = ceil_div64(steps, s) * kRows;
    p.slices = (int)ceil_div64(rows, p.slice_rows);
    return p;
}

bool wg_shape_ok(int64_t rows, int64_t out, int64_t c) {
    return rows >= 0 && out >= 1 && c >= 1 && out <= (1 << 20) && c <= (1 << 20) && out * c <= ((int64_t)1 << 31) &&
           rows <= ((int64_t)1 << 40) / (out + c);
}

template <int DT, int BM>
void wg_launch(const void* gy, const int8_t* codes, const uint8_t* scales, float* part, float* part_b, const WgShape& p, bool vec,
               hipStream_t s) {
    using T = typename Elem<DT>::T;
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n * p.slices)), block(kBlock);
    if (vec) hipLaunchKernelGGL((linear_wgrad8_kernel<DT, BM, true>), grid, block, 0, s, (const T*)gy, codes, scales, part, part_b, p);
    else hipLaunchKernelGGL((linear_wgrad8_kernel<DT, BM, false>), grid, block, 0, s, (const T*)gy, codes, scales, part, part_b, p);
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
    const WgShape p = wg_plan(rows, out, c);
    const bool vec = out % 4 == 0 && reinterpret_cast<uintptr_t>(gy) % (4 * sizeof(T)) == 0;
    float* part_b = gb ? ws + (int64_t)p.slices * out * p.blocks * kBlk8 : nullptr;
    switch (wg_tile(out)) {
        case 64: wg_launch<DT, 64>(gy, codes, scales, ws, part_b, p, vec, s); break;
        case 128: wg_launch<DT, 128>(gy, codes, scales, ws, part_b, p, vec, s); break;
        default: wg_launch<DT, 256>(gy, codes, scales, ws, part_b, p, vec, s); break;
    }
    hipLaunchKernelGGL((linear_wgrad8_reduce_kernel<DT>), dim3((unsigned)ceil_div64(out * c, kBlock)), dim3(kBlock), 0, s,
                       (const float*)ws, (const float*)part_b, (T*)gw, (T*)gb, alpha, p);
    return check_launch("sae_linear_wgrad8");
}

}  // namespace
}  // namespace sae

using namespace sae;

extern "C" int64_t sae_linear_wgrad8_workspace(int64_t rows, int64_t out, int64_t c) {
    if (!wg_shape_ok(rows, out, c) || rows == 0) return 0;
    const WgShape p = wg_plan(rows, out, c);
    return (int64_t)p.slices * out * ((int64_t)p.blocks * kBlk8 + 1);
}

extern "C" int sae_linear_wgrad8(const void* gy, const int8_t* codes, const uint8_t* scales, void* gw, void* gb, int64_t rows,
                                 int64_t out, int64_t c, float alpha, int32_t dtype, float* workspace, int64_t workspace_floats,
                                 sae_stream_t stream) {
    sae::clear_stale_error();
    if (!elem_known(dtype)) return fail(SAE_EINVAL, "sae_linear_wgrad8: unknown element type %d", (int)dtype);
    if (!wg_shape_ok(rows, out, c)) return fail(SAE_EINVAL, "sae_linear_wgrad8: bad shape");
    if (!gw || (rows > 0 && (!gy || !codes || !scales))) return fail(SAE_EINVAL, "sae_linear_wgrad8: null tensor");
    if (rows > 0 && (!aligned16(codes) || !aligned16(workspace) || reinterpret_cast<uintptr_t>(gy) % (uintptr_t)elem_bytes(dtype)))
        return fail(SAE_EINVAL, "sae_linear_wgrad8: misaligned tensor");
    if (rows > 0 && (!workspace || workspace_floats < sae_linear_wgrad8_workspace(rows, out, c)))
        return fail(SAE_EWORKSPACE, "sae_linear_wgrad8: workspace %lld < %lld floats (sae_linear_wgrad8_workspace)",
                    (long long)workspace_floats, (long long)sae_linear_wgrad8_workspace(rows, out, c));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == SAE_F32) return wg_run<SAE_F32>(gy, codes, scales, gw, gb, rows, out, c, alpha, workspace, s);
    if (dtype == SAE_BF16) return wg_run<SAE_BF16>(gy, codes, scales, gw, gb, rows, out, c, alpha, workspace, s);
    return wg_run<SAE_F16>(gy, codes, scales, gw, gb, rows, out, c, alpha, workspace, s);
}
