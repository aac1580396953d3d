// 8-bit activation checkpoints (format: elem8.inc): an activation written as codes + block exponents, and given back.
//
//   pack     reads x [rows][c] (f32 / bf16 / f16), writes codes [rows][32 * blocks] and exponents [blocks][rows]
//   unpack   the values the codes stand for, in the element type
//
// blocks = ceil(c / 32).  The code rows are padded with zeros to whole blocks and the exponents are stored block-major so that the
// product that reads them (linear_wgrad8.hip) loads four channels and four rows' exponents as one word each, with no remainder.
// HBM-bound: S + S / 4 bytes in f32.  f32 524288 x 256 (537 MB): pack 119 us, 5.7 TB/s; unpack 113 us, 5.9 TB/s.  bf16 6561 x 515 (7 MB,
// rows that start anywhere): 6.3 and 5.3 us, of which 2 - 3 are the launch; with four rows a thread and whole vectors up to the row's end
// 22 -> 12 us for both (element-wise ends wait for one load after the other).
#include "elem8.inc"

namespace sae {
namespace {

constexpr int kQ = 4;              // rows a thread takes: four loads under way, and the exponents of a block's four rows are a word

struct PackShape {
    int64_t rows, c, blocks;
    int64_t lanes;             // channel vectors of a row padded to whole blocks
    int tile, rp;              // of a work-group: lanes at a time, threads / tile (rows at a time: kQ of each)
    int64_t tiles, chunks;     // of a row, of the rows
};

// A work-group takes one (chunk of rows, tile of lanes) after the other in strides of the grid.  ANY: rows that start anywhere and end
// inside a vector.
template <int DT, bool ANY>
__global__ __launch_bounds__(kBlock) void checkpoint8_pack_kernel(const typename Elem<DT>::T* __restrict__ x,
                                                                  int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                  const PackShape p) {
    constexpr int V = Elem<DT>::kVec, LB = kBlk8 / V;
    const int tx = (int)threadIdx.x % p.tile, ty = (int)threadIdx.x / p.tile;
    for (int64_t id = blockIdx.x; id < p.tiles * p.chunks; id += gridDim.x) {
        const int64_t chunk = id / p.tiles, lane = (id - chunk * p.tiles) * p.tile + tx, c0 = lane * V;
        const int64_t r = (chunk * p.rp + ty) * kQ;
        const int have = ty >= p.rp || lane >= p.lanes || r >= p.rows ? 0 : p.rows - r < kQ ? (int)(p.rows - r) : kQ;
        const int n = p.c - c0 < V ? (int)(p.c - c0) : V;           // (not positive in a row's padding)
        Raw<DT> raw[kQ];
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
            raw[i].zero();
            if (i < have && n > 0) {
                if constexpr (ANY) raw[i].load_some(x + (r + i) * p.c + c0, n, p.c >= V);
                else raw[i].load(x + (r + i) * p.c + c0);
            }
        }
        unsigned word = 0;
#pragma unroll
        for (int i = 0; i < kQ; ++i) {                              // (whole blocks of lanes have the same rows)
            const unsigned e = block8_exponent<DT>(block8_amax<LB>(raw[i].amax()));
            word |= e << (8 * i);
            if (i < have) {
                float v[V];
                raw[i].get(v);
                store_codes<V>(codes + (r + i) * p.blocks * kBlk8 + c0, v, block8_inverse(e));
            }
        }
        if (have > 0 && lane % LB == 0) store_exponents(scales + c0 / kBlk8 * p.rows + r, word, have);
    }
}

template <int DT, bool ANY, bool STREAM>
__global__ __launch_bounds__(kBlock) void checkpoint8_unpack_kernel(const int8_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ scales,
                                                                    typename Elem<DT>::T* __restrict__ x, const PackShape p) {
    constexpr int V = Elem<DT>::kVec;
    const int tx = (int)threadIdx.x % p.tile, ty = (int)threadIdx.x / p.tile;
    if (ty >= p.rp) return;
    for (int64_t id = blockIdx.x; id < p.tiles * p.chunks; id += gridDim.x) {
        const int64_t chunk = id / p.tiles, lane = (id - chunk * p.tiles) * p.tile + tx, c0 = lane * V;
        const int64_t r = (chunk * p.rp + ty) * kQ;
        if (c0 >= p.c || r >= p.rows) continue;
        const int have = p.rows - r < kQ ? (int)(p.rows - r) : kQ, n = p.c - c0 < V ? (int)(p.c - c0) : V;
        RawCodes<V> code[kQ];
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < have) code[i].load(codes + (r + i) * p.blocks * kBlk8 + c0);
        const unsigned word = load_exponents(scales + c0 / kBlk8 * p.rows + r, have);
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < have) {
                float v[V];
                code[i].get(block8_step((word >> (8 * i)) & 0xffu), v);
                Raw<DT> raw;
                raw.set(v);
                if constexpr (ANY) raw.store_some(x + (r + i) * p.c + c0, n);
                else raw.template store<STREAM>(x + (r + i) * p.c + c0);
            }
    }
}

PackShape pack_plan(int64_t rows, int64_t c, int v) {
    PackShape p;
    const int lb = kBlk8 / v;
    p.rows = rows;
    p.c = c;
    p.blocks = ceil_div64(c, kBlk8);
    p.lanes = p.blocks * lb;
    const int64_t tiles = ceil_div64(p.lanes, kBlock);
    p.tile = (int)(ceil_div64(ceil_div64(p.lanes, tiles), lb) * lb);       // tiles of even width, of whole blocks
    p.tiles = ceil_div64(p.lanes, p.tile);
    p.rp = kBlock / p.tile;
    p.chunks = ceil_div64(rows, (int64_t)p.rp * kQ);
    return p;
}
dim3 pack_grid(const PackShape& p) {
    const int64_t g = p.tiles * p.chunks;                                   // (a launch holds 2^32 threads at most)
    return dim3((unsigned)(g > (1 << 20) ? 1 << 20 : g));
}

template <int DT>
int pack(const void* x, int8_t* codes, uint8_t* scales, int64_t rows, int64_t c, hipStream_t s) {
    using T = typename Elem<DT>::T;
    const PackShape p = pack_plan(rows, c, Elem<DT>::kVec);
    if (c % Elem<DT>::kVec == 0 && aligned16(x))
        hipLaunchKernelGGL((checkpoint8_pack_kernel<DT, false>), pack_grid(p), dim3(kBlock), 0, s, (const T*)x, codes, scales, p);
    else
        hipLaunchKernelGGL((checkpoint8_pack_kernel<DT, true>), pack_grid(p), dim3(kBlock), 0, s, (const T*)x, codes, scales, p);
    return check_launch("sae_checkpoint8_pack");
}

template <int DT>
int unpack(const int8_t* codes, const uint8_t* scales, void* x, int64_t rows, int64_t c, hipStream_t s) {
    using T = typename Elem<DT>::T;
    const PackShape p = pack_plan(rows, c, Elem<DT>::kVec);
    const bool whole = c % Elem<DT>::kVec == 0 && aligned16(x), stream = rows * c * (int64_t)sizeof(T) > ((int64_t)32 << 20);   // > the L2s
    if (whole && stream)
        hipLaunchKernelGGL((checkpoint8_unpack_kernel<DT, false, true>), pack_grid(p), dim3(kBlock), 0, s, codes, scales, (T*)x, p);
    else if (whole)
        hipLaunchKernelGGL((checkpoint8_unpack_kernel<DT, false, false>), pack_grid(p), dim3(kBlock), 0, s, codes, scales, (T*)x, p);
    else
        hipLaunchKernelGGL((checkpoint8_unpack_kernel<DT, true, false>), pack_grid(p), dim3(kBlock), 0, s, codes, scales, (T*)x, p);
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
