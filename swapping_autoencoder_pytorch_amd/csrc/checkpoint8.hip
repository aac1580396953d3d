// 8-bit activation checkpoints (format: elem8.inc): an activation written as codes + block exponents, and given back.
//
//   pack     reads x [rows][c] (f32 / bf16 / f16), writes codes [rows][32 * blocks] and exponents [blocks][rows]
//   unpack   the values the codes stand for, in the element type
//
// blocks = ceil(c / 32).  The code rows are padded with zeros to whole blocks and the exponents are stored block-major so that the
// product that reads them (linear_wgrad8.hip) loads four channels and four rows' exponents as one word each, with no remainder.
// HBM-bound: S + S / 4 bytes in f32.
#include "elem8.inc"

namespace sae {
namespace {

// One thread per V neighbours of a row padded to whole blocks; a block's LB = 32 / V lanes lie in one wave and meet in shuffles.
template <int DT, int V>
__global__ __launch_bounds__(kBlock) void checkpoint8_pack_kernel(const typename Elem<DT>::T* __restrict__ x,
                                                                  int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                  int64_t rows, int64_t c, int64_t blocks) {
    constexpr int LB = kBlk8 / V;
    const int64_t stride = (int64_t)gridDim.x * (kBlock / LB);
    for (int64_t base = (int64_t)blockIdx.x * (kBlock / LB); base < rows * blocks; base += stride) {
        const int64_t block = base + threadIdx.x / LB;
        const bool live = block < rows * blocks;      // (whole groups of LB lanes are live or not)
        const int64_t row = live ? block / blocks : 0, cb = live ? block - row * blocks : 0;
        const int64_t col = cb * kBlk8 + (int64_t)(threadIdx.x % LB) * V;
        Raw<DT, V> raw;
        raw.zero();
        if (live && col < c) raw.load(x + row * c + col);
        const unsigned e = block8_exponent<DT>(block8_amax<LB>(raw.amax()));
        if (!live) continue;
        float v[V];
        raw.get(v);
        store_codes<V>(codes + row * blocks * kBlk8 + col, v, block8_inverse(e));
        if (threadIdx.x % LB == 0) scales[cb * rows + row] = (uint8_t)e;
    }
}

template <int DT, int V>
__global__ __launch_bounds__(kBlock) void checkpoint8_unpack_kernel(const int8_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ scales,
                                                                    typename Elem<DT>::T* __restrict__ x, int64_t rows,
                                                                    int64_t c, int64_t blocks) {
    constexpr int LB = kBlk8 / V;
    const int64_t stride = (int64_t)gridDim.x * (kBlock / LB);
    for (int64_t block = (int64_t)blockIdx.x * (kBlock / LB) + threadIdx.x / LB; block < rows * blocks; block += stride) {
        const int64_t row = block / blocks, cb = block - row * blocks;
        const int64_t col = cb * kBlk8 + (int64_t)(threadIdx.x % LB) * V;
        if (col >= c) continue;
        RawCodes<V> raw;
        raw.load(codes + row * blocks * kBlk8 + col);
        float v[V];
        raw.get(block8_step(scales[cb * rows + row]), v);
        store_vec<DT, V>(x + row * c + col, v);
    }
}

// work-groups of the two kernels, which walk what is behind them in strides of the grid (a launch holds 2^32 threads at most)
unsigned checkpoint8_grid(int64_t rows, int64_t blocks, int lanes) {
    const int64_t g = ceil_div64(rows * blocks, kBlock / lanes);
    return (unsigned)(g > (1 << 20) ? 1 << 20 : g);
}

template <int DT>
int pack(const void* x, int8_t* codes, uint8_t* scales, int64_t rows, int64_t c, hipStream_t s) {
    using T = typename Elem<DT>::T;
    const int64_t blocks = ceil_div64(c, kBlk8);
    const bool vec = c % Elem<DT>::kVec == 0 && aligned16(x);
    const unsigned g = checkpoint8_grid(rows, blocks, vec ? kBlk8 / Elem<DT>::kVec : kBlk8);
    if (vec)
        hipLaunchKernelGGL((checkpoint8_pack_kernel<DT, Elem<DT>::kVec>), dim3(g), dim3(kBlock), 0, s, (const T*)x, codes,
                           scales, rows, c, blocks);
    else
        hipLaunchKernelGGL((checkpoint8_pack_kernel<DT, 1>), dim3(g), dim3(kBlock), 0, s, (const T*)x, codes, scales, rows,
                           c, blocks);
    return check_launch("sae_checkpoint8_pack");
}

template <int DT>
int unpack(const int8_t* codes, const uint8_t* scales, void* x, int64_t rows, int64_t c, hipStream_t s) {
    using T = typename Elem<DT>::T;
    const int64_t blocks = ceil_div64(c, kBlk8);
    const bool vec = c % Elem<DT>::kVec == 0 && aligned16(x);
    const unsigned g = checkpoint8_grid(rows, blocks, vec ? kBlk8 / Elem<DT>::kVec : kBlk8);
    if (vec)
        hipLaunchKernelGGL((checkpoint8_unpack_kernel<DT, Elem<DT>::kVec>), dim3(g), dim3(kBlock), 0, s, codes, scales,
                           (T*)x, rows, c, blocks);
    else
        hipLaunchKernelGGL((checkpoint8_unpack_kernel<DT, 1>), dim3(g), dim3(kBlock), 0, s, codes, scales, (T*)x, rows, c,
                           blocks);
    return check_launch("sae_checkpoint8_unpack");
}

int check_checkpoint8(const char* what, const void* x, const void* codes, const void* scales, int64_t rows, int64_t c,
                      int32_t dtype) {
    if (!elem_known(dtype)) return fail(SAE_EINVAL, "%s: unknown element type %d", what, (int)dtype);
    if (rows < 0 || c < 1 || c > ((int64_t)1 << 46) || rows > ((int64_t)1 << 46) / c) return fail(SAE_EINVAL, "%s: bad shape", what);
    if (rows == 0) return SAE_OK;
    if (!x || !codes || !scales) return fail(SAE_EINVAL, "%s: null tensor", what);
    if (!aligned16(codes)) return fail(SAE_EINVAL, "%s: the codes must be 16-byte aligned", what);
    if (reinterpret_cast<uintptr_t>(x) % (uintptr_t)elem_bytes(dtype)) return fail(SAE_EINVAL, "%s: misaligned tensor", what);
    return SAE_OK;
}

}  // namespace
}  // namespace sae

using namespace sae;

extern "C" int sae_checkpoint8_pack(const void* x, int8_t* codes, uint8_t* scales, int64_t rows, int64_t c, int32_t dtype,
                                    sae_stream_t stream) {
    sae::clear_stale_error();
    const int rc = check_checkpoint8("sae_checkpoint8_pack", x, codes, scales, rows, c, dtype);
    if (rc != SAE_OK || rows == 0) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == SAE_F32) return pack<SAE_F32>(x, codes, scales, rows, c, s);
    if (dtype == SAE_BF16) return pack<SAE_BF16>(x, codes, scales, rows, c, s);
    return pack<SAE_F16>(x, codes, scales, rows, c, s);
}

extern "C" int sae_checkpoint8_unpack(const int8_t* codes, const uint8_t* scales, void* x, int64_t rows, int64_t c, int32_t dtype,
                                      sae_stream_t stream) {
    sae::clear_stale_error();
    const int rc = check_checkpoint8("sae_checkpoint8_unpack", x, codes, scales, rows, c, dtype);
    if (rc != SAE_OK || rows == 0) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == SAE_F32) return unpack<SAE_F32>(codes, scales, x, rows, c, s);
    if (dtype == SAE_BF16) return unpack<SAE_BF16>(codes, scales, x, rows, c, s);
    return unpack<SAE_F16>(codes, scales, x, rows, c, s);
}
