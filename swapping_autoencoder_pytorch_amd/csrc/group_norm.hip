// Group normalisation with its activation on channels-last tensors x [n][l][c] (l: positions of a sample), f32 / bf16 / f16:
//
//     z = (x - mean) * rstd * w[c] + b[c],   y = scale * act(z)          mean, rstd over the l * (c / groups) values of a group
//
// and its backward, from x itself or from its 8-bit checkpoint (elem8.inc), which the forward writes next to y:
//
//     dz = gy * scale * act'(z),   gb = sum dz,   gw = sum dz xhat,
//     gx = rstd * (w dz - m1 - xhat m2),    m1 = mean over the group of w dz,   m2 = of w dz xhat,    xhat = (x - mean) * rstd
//
// Every statistic needs the whole group before the first result can be written, so each direction walks its tensors twice:
//     sums      per (sample, chunk of rows, channel), in registers, one record per chunk
//     totals    the chunks' records added in order: mean / rstd, or m1 / m2 and the channel sums (few records: by the apply kernel)
//     apply     the elementwise pass, last chunk first: what the sums read last is what the caches still hold
// or, where a sample's groups are small, all of it in one work-group per (sample, slab of whole groups): one launch.
//
// Layout of a walk: a lane owns V neighbouring channels (16 bytes) and takes four rows at a time, so that four loads are under way
// and the exponents of four rows are one word.  ANY: rows (or slabs of them) that start anywhere and end inside a vector.
//
// What bounds it: HBM, each tensor's bytes twice less what the caches keep.  f32 [16, 128, 256, 256] kept in 8 bits (537 MB): sums 131 us
// (678 MB, 5.2 TB/s), apply 201 (1074 MB, 5.3), backward sums 120 (678 MB, 5.6), apply 212 (1213 MB, 5.7).  f32 [16, 512, 64, 64]
// (134 MB): 26 + 5 + 42 us, 43 + 6 + 61 back, 212 in all a row at a time, stores through the caches, first chunk first.  bf16
// [16, 256, 64, 64] forward: 9.3 + 14.5 us (36 so).  In groups of samples that the 256 MB cache would hold the
// largest takes 2 - 50 % longer (more kernels' ends).
//
// Numerics: a thread adds x - x0 and (x - x0)^2 over its rows, x0 the first value it meets in the channel: at most the number of
// its rows times the rounding of a plain sum, whatever the channel's mean.  The records are moments about zero in 64 bits, which
// only have to be added.  mean and rstd are fp32; nothing is held in less.
#include "elem8.inc"

namespace sae {
namespace {

constexpr int kQ = 4;              // rows a thread takes at a time
constexpr int kFused = 512;        // most threads of a one-launch work-group

struct GnShape {
    int64_t l;                 // positions of a sample
    int64_t rows;              // n * l: rows of codes, stride of a block's exponents
    int c, groups, cg;
    int lanes;                 // channel vectors of a row (of a slab); padded to whole 8-bit blocks where codes are written
    int tile;                  // lanes a work-group covers at a time
    int rp;                    // rows it covers at a time: threads / tile, kQ of each
    int chunk_rows;            // rows of a work-group
    int chunks;                // chunks of a sample
    int units;                 // records of a chunk: channel vectors if a vector lies in one group, channels if not
    int blocks;                // 8-bit blocks of a row
    bool any;                  // vectors that start anywhere or end inside
    int slab, slabs;           // groups of a one-launch work-group (0: not that form), slabs of a sample
};

#ifdef HIPEMU
__device__ __forceinline__ float exp2_fast(float v) { return exp2f(v); }
__device__ __forceinline__ float rcp_fast(float v) { return 1.0f / v; }
#else
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }    // 1 ulp
__device__ __forceinline__ float rcp_fast(float v) { return __builtin_amdgcn_rcpf(v); }      // 1 ulp
#endif

// Activations of t = kArg * z (SiLU's exponent has base 2, so its factor goes into the affine map in front):
//   value   act(z) * scale;      slope   act'(z)
template <int ACT>
struct Act {
    static constexpr float kArg = ACT == SAE_ACT_SILU ? 1.44269504088896341f : 1.0f;
    static constexpr float kLn2 = 0.693147180559945309f;
    // z -> -infinity: exp2 gives infinity and the quotient 0
    static __device__ __forceinline__ float sigmoid(float t) { return rcp_fast(1.0f + exp2_fast(-t)); }
    static __device__ __forceinline__ float value(float t, float slope, float scale) {
        if constexpr (ACT == SAE_ACT_LRELU) return t * (t > 0.0f ? scale : scale * slope);
        else if constexpr (ACT == SAE_ACT_SILU) return t * (kLn2 * scale) * sigmoid(t);
        else return t * scale;
    }
    static __device__ __forceinline__ float derivative(float t, float slope) {
        if constexpr (ACT == SAE_ACT_LRELU) return t > 0.0f ? 1.0f : slope;
        else if constexpr (ACT == SAE_ACT_SILU) {
            const float s = sigmoid(t);
            return s * fmaf(t, fmaf(-kLn2, s, kLn2), 1.0f);
        } else return 1.0f;
    }
};

// The groups of a lane's V channels, one division for all of them
template <int V>
__device__ __forceinline__ void groups_of(int c0, int cg, int most, int (&g)[V]) {
    int at = c0 / cg, left = cg - (c0 - at * cg);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        g[j] = at < most ? at : most - 1;                          // (behind the row's end: any that is there)
        if (--left == 0) { ++at; left = cg; }
    }
}

// V neighbours of a parameter (absent: all `none`)
template <int V>
__device__ __forceinline__ void load_param(const float* __restrict__ w, int c0, int n, float none, float (&v)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = none;
    if (!w) return;
    if (n >= V) {
        __builtin_memcpy(v, w + c0, sizeof(v));
        return;
    }
#pragma unroll
    for (int j = 0; j < V - 1; ++j)
        if (j < n) v[j] = w[c0 + j];
}

// Where a thread stands in a walk over rows [r_begin, r_end) of sample n
struct Walk {
    int tx, ty, c0, rp;
    int64_t first, r_end, row0;        // row0: the sample's first row
    int n;                             // channels of the lane: V, fewer at the row's (the slab's) end, 0 if it has none
};

template <bool ANY, typename R, typename T>
__device__ __forceinline__ void load_lane(R& raw, const T* p, int n, int c) {
    if constexpr (ANY) raw.load_some(p, n, c >= 16 / (int)sizeof(T));
    else raw.load(p);
}
template <bool ANY, bool STREAM, int DT, int V>
__device__ __forceinline__ void store_lane(typename Elem<DT>::T* p, const float (&v)[V], int n) {
    Raw<DT> raw;
    raw.set(v);
    if constexpr (ANY) raw.store_some(p, n);
    else raw.template store<STREAM>(p);
}
// n of a lane whose channels start `left` in front of the end
template <int V>
__device__ __forceinline__ int lane_channels(bool on, int left) { return !on || left <= 0 ? 0 : left < V ? left : V; }

// sum over ty of the threads' values (red[ty * width + tx], every thread's written): at red[tx] behind it, in a fixed order
template <typename P>
__device__ __forceinline__ void fold_rows(P* red, int tx, int ty, int width, int rp, bool on) {
    int half = 1;
    while (half < rp) half <<= 1;
    for (half >>= 1; half >= 1; half >>= 1) {
        __syncthreads();
        if (on && ty < half && ty + half < rp) {
            P& a = red[ty * width + tx];
            const P b = red[(ty + half) * width + tx];
            a.x += b.x;
            a.y += b.y;
        }
    }
    __syncthreads();
}

// ---- forward ----------------------------------------------------------------------------------------------------------------

// a thread's moments over its rows, and (KEEP) the checkpoint of them; every thread of the work-group makes the same trips
template <int DT, bool ANY, bool KEEP, int V>
__device__ __forceinline__ void walk_sums(const typename Elem<DT>::T* __restrict__ x, int8_t* __restrict__ codes,
                                          uint8_t* __restrict__ scales, const Walk& w, const GnShape& p, double (&sx)[V], double (&sxx)[V]) {
    constexpr int LB = kBlk8 / V;
    float k[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) k[j] = s1[j] = s2[j] = 0.0f;
    const int64_t begin = w.first + kQ * w.ty;
    if (w.n > 0 && begin < w.r_end) {
        Raw<DT> raw;
        load_lane<ANY>(raw, x + (w.row0 + begin) * p.c + w.c0, w.n, p.c);
        raw.get(k);
    }
    int64_t count = 0;
    const int cb = w.c0 / kBlk8;
    const bool kept = KEEP && w.ty < w.rp && cb < p.blocks;
    for (int64_t r0 = w.first; r0 < w.r_end; r0 += kQ * w.rp) {
        const int64_t r = r0 + kQ * w.ty;
        Raw<DT> raw[kQ];
        const int have = w.n <= 0 || r >= w.r_end ? 0 : w.r_end - r < kQ ? (int)(w.r_end - r) : kQ;
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
            raw[i].zero();
            if (i < have) load_lane<ANY>(raw[i], x + (w.row0 + r + i) * p.c + w.c0, w.n, p.c);
        }
        unsigned e[kQ];
        if constexpr (KEEP)
#pragma unroll
            for (int i = 0; i < kQ; ++i) e[i] = block8_exponent<DT>(block8_amax<LB>(raw[i].amax()));
        count += have;
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
            float v[V];
            raw[i].get(v);
            if (i < have)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[j] - k[j];
                    s1[j] += d;
                    s2[j] = fmaf(d, d, s2[j]);
                }
            if constexpr (KEEP)
                if (kept && r + i < w.r_end) store_codes<V>(codes + (w.row0 + r + i) * p.blocks * kBlk8 + w.c0, v, block8_inverse(e[i]));
        }
        if constexpr (KEEP)
            if (kept && w.c0 % kBlk8 == 0 && r < w.r_end)
                store_exponents(scales + (int64_t)cb * p.rows + w.row0 + r, e[0] | (e[1] << 8) | (e[2] << 16) | (e[3] << 24),
                                w.r_end - r < kQ ? (int)(w.r_end - r) : kQ);
    }
    const double m = (double)count;
#pragma unroll
    for (int j = 0; j < V; ++j) {                                  // about zero
        const double kd = k[j], d1 = s1[j];
        sx[j] = m * kd + d1;
        sxx[j] = (double)s2[j] + 2.0 * kd * d1 + m * kd * kd;
    }
}

// mean and rstd of m values from their moments about zero
__device__ __forceinline__ float2 moments(double a, double b, double m, float eps) {
    const double mu = a / m;
    double var = b / m - mu * mu;
    if (var < 0.0) var = 0.0;                                      // (a NaN stays one)
    return float2{(float)mu, (float)(1.0 / sqrt(var + (double)eps))};
}

template <int DT, bool ANY, int ACT, bool STREAM, int V>
__device__ __forceinline__ void walk_apply(const typename Elem<DT>::T* __restrict__ x, typename Elem<DT>::T* __restrict__ y, const Walk& w,
                                           const GnShape& p, const float (&mu)[V], const float (&a)[V], const float (&b)[V], float slope,
                                           float scale) {
    for (int64_t r = w.first + kQ * w.ty; r < w.r_end; r += kQ * w.rp) {
        const int64_t at = (w.row0 + r) * p.c + w.c0;
        const int have = w.r_end - r < kQ ? (int)(w.r_end - r) : kQ;
        Raw<DT> raw[kQ];
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < have) load_lane<ANY>(raw[i], x + at + (int64_t)i * p.c, w.n, p.c);
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < have) {
                float v[V];
                raw[i].get(v);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = Act<ACT>::value(fmaf(v[j] - mu[j], a[j], b[j]), slope, scale);
                store_lane<ANY, STREAM, DT>(y + at + (int64_t)i * p.c, v, w.n);
            }
    }
}

// record [n][chunk][unit]: sum x and sum x^2 of the unit over the chunk's rows
template <int DT, bool ANY, bool KEEP>
__global__ __launch_bounds__(kBlock) void gn_sums_kernel(const typename Elem<DT>::T* __restrict__ x, double2* __restrict__ rec,
                                                         int8_t* __restrict__ codes, uint8_t* __restrict__ scales, const GnShape p) {
    constexpr int V = Elem<DT>::kVec;
    __shared__ double2 red[kBlock];
    const int n = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
    Walk w;
    w.tx = tid % p.tile;
    w.ty = tid / p.tile;
    w.rp = p.rp;
    w.row0 = (int64_t)n * p.l;
    w.first = (int64_t)chunk * p.chunk_rows;
    w.r_end = w.first + p.chunk_rows < p.l ? w.first + p.chunk_rows : p.l;
    const bool whole = p.cg % V == 0;
    for (int lane0 = 0; lane0 < p.lanes; lane0 += p.tile) {
        w.c0 = (lane0 + w.tx) * V;
        w.n = lane_channels<V>(w.ty < w.rp, p.c - w.c0);
        double sx[V], sxx[V];
        walk_sums<DT, ANY, KEEP>(x, codes, scales, w, p, sx, sxx);
        const int rounds = whole ? 1 : V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j >= rounds) break;
            double2 t{sx[j], sxx[j]};
            if (whole)
#pragma unroll
                for (int i = 1; i < V; ++i) { t.x += sx[i]; t.y += sxx[i]; }
            __syncthreads();
            red[tid] = t;
            fold_rows(red, w.tx, w.ty, p.tile, p.rp, w.ty < p.rp);
            const int unit = whole ? lane0 + w.tx : w.c0 + j;
            if (w.ty == 0 && j < w.n) rec[((int64_t)n * p.chunks + chunk) * p.units + unit] = red[w.tx];
        }
    }
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// one wave per (sample, group)
__global__ __launch_bounds__(kWave) void gn_totals_kernel(const double2* __restrict__ rec, float* __restrict__ mean,
                                                          float* __restrict__ rstd, float eps, const GnShape p) {
    const int g = blockIdx.x, n = blockIdx.y;
    const int per = p.units / p.groups;
    double a = 0.0, b = 0.0;
    const unsigned records = (unsigned)p.chunks * (unsigned)per;   // (below 2^31)
    for (unsigned i = threadIdx.x; i < records; i += kWave) {
        const unsigned chunk = i / (unsigned)per, u = i - chunk * (unsigned)per;
        const double2 t = rec[((int64_t)n * p.chunks + chunk) * p.units + g * per + u];
        a += t.x;
        b += t.y;
    }
    a = wave_sum_d(a);
    b = wave_sum_d(b);
    if (threadIdx.x == 0) {
        const float2 s = moments(a, b, (double)p.l * p.cg, eps);
        mean[(int64_t)n * p.groups + g] = s.x;
        rstd[(int64_t)n * p.groups + g] = s.y;
    }
}

// Totals by the apply kernels: each work-group adds its sample's records for itself, where they are few (fold_totals); a launch fewer.
// `per` lanes of a wave, a power of two, for each group; every work-group adds in the same order.
constexpr int kFoldGroups = kBlock, kFoldChannels = 512;
__device__ __forceinline__ int fold_lanes(int groups) {
    int per = kWave;
    while (per * groups > kBlock) per >>= 1;
    return per;
}
__device__ __forceinline__ double lanes_sum_d(double v, int per) {
    for (int off = per >> 1; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// TOTALS: the statistics too
template <int DT, bool ANY, int ACT, bool TOTALS>
__global__ __launch_bounds__(kBlock) void gn_apply_kernel(const typename Elem<DT>::T* __restrict__ x, const double2* __restrict__ rec,
                                                          float* __restrict__ mean, float* __restrict__ rstd,
                                                          const float* __restrict__ weight, const float* __restrict__ bias,
                                                          typename Elem<DT>::T* __restrict__ y, float eps, float slope, float scale,
                                                          const GnShape p) {
    constexpr int V = Elem<DT>::kVec;
    const int n = (int)gridDim.y - 1 - (int)blockIdx.y, chunk = (int)gridDim.x - 1 - (int)blockIdx.x, tid = threadIdx.x;
    Walk w;
    w.tx = tid % p.tile;
    w.ty = tid / p.tile;
    w.rp = p.rp;
    w.row0 = (int64_t)n * p.l;
    w.first = (int64_t)chunk * p.chunk_rows;
    w.r_end = w.first + p.chunk_rows < p.l ? w.first + p.chunk_rows : p.l;
    __shared__ float2 stat[TOTALS ? kFoldGroups : 1];
    if constexpr (TOTALS) {
        const int units = p.units / p.groups, items = p.chunks * units, per = fold_lanes(p.groups), g = tid / per;
        double a = 0.0, b = 0.0;
        if (g < p.groups)
#pragma unroll 4
            for (int i = tid - g * per; i < items; i += per) {
                const int at = i / units, u = i - at * units;
                const double2 o = rec[((int64_t)n * p.chunks + at) * p.units + g * units + u];
                a += o.x;
                b += o.y;
            }
        a = lanes_sum_d(a, per);
        b = lanes_sum_d(b, per);
        if (g < p.groups && tid == g * per) {
            const float2 s = moments(a, b, (double)p.l * p.cg, eps);
            stat[g] = s;
            if (chunk == 0) {
                mean[(int64_t)n * p.groups + g] = s.x;
                rstd[(int64_t)n * p.groups + g] = s.y;
            }
        }
        __syncthreads();
    }
    if (w.ty >= w.rp) return;
    for (int lane0 = 0; lane0 < p.lanes; lane0 += p.tile) {
        w.c0 = (lane0 + w.tx) * V;
        w.n = lane_channels<V>(true, p.c - w.c0);
        if (w.n == 0) return;
        float mu[V], a[V], b[V];
        int g[V];
        groups_of<V>(w.c0, p.cg, p.groups, g);
        load_param<V>(weight, w.c0, w.n, 1.0f, a);
        load_param<V>(bias, w.c0, w.n, 0.0f, b);
        float2 s;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j == 0 || g[j] != g[j - 1]) {
                if constexpr (TOTALS) s = stat[g[j]];
                else s = float2{mean[(int64_t)n * p.groups + g[j]], rstd[(int64_t)n * p.groups + g[j]]};
            }
            mu[j] = s.x;
            a[j] *= s.y * Act<ACT>::kArg;
            b[j] *= Act<ACT>::kArg;
        }
        walk_apply<DT, ANY, ACT, true>(x, y, w, p, mu, a, b, slope, scale);
    }
}

// The place of a one-launch work-group: slab blockIdx.x (p.slab groups) of sample blockIdx.y; the walk covers all of its rows
template <int V>
__device__ __forceinline__ Walk slab_walk(const GnShape& p, int& g0, int& gs, int& width) {
    g0 = (int)blockIdx.x * p.slab;
    gs = p.groups - g0 < p.slab ? p.groups - g0 : p.slab;
    width = gs * p.cg;
    Walk w;
    w.tx = (int)threadIdx.x % p.tile;
    w.ty = (int)threadIdx.x / p.tile;
    w.rp = p.rp;
    w.row0 = (int64_t)blockIdx.y * p.l;
    w.first = 0;
    w.r_end = p.l;
    w.c0 = g0 * p.cg + w.tx * V;
    w.n = lane_channels<V>(w.ty < w.rp, width - w.tx * V);
    return w;
}

template <int DT, bool ANY, int ACT, bool KEEP>
__global__ __launch_bounds__(kFused) void gn_fused_kernel(const typename Elem<DT>::T* __restrict__ x, const float* __restrict__ weight,
                                                          const float* __restrict__ bias, typename Elem<DT>::T* __restrict__ y,
                                                          float* __restrict__ mean, float* __restrict__ rstd, int8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, float eps, float slope, float scale,
                                                          const GnShape p) {
    constexpr int V = Elem<DT>::kVec;
    __shared__ double2 red[kFused];
    __shared__ double2 unit[kFused];
    __shared__ float2 stat[kFused];
    int g0, gs, width;
    const Walk w = slab_walk<V>(p, g0, gs, width);
    const int tid = threadIdx.x;
    const bool whole = p.cg % V == 0;
    double sx[V], sxx[V];
    walk_sums<DT, ANY, KEEP>(x, codes, scales, w, p, sx, sxx);
    // unit sums of the slab: of its channel vectors, or of its channels (at most kFused of them: gn_slab)
    const int rounds = whole ? 1 : V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (j >= rounds) break;
        double2 t{sx[j], sxx[j]};
        if (whole)
#pragma unroll
            for (int i = 1; i < V; ++i) { t.x += sx[i]; t.y += sxx[i]; }
        __syncthreads();
        red[tid] = t;
        fold_rows(red, w.tx, w.ty, p.tile, p.rp, w.ty < p.rp);
        if (w.ty == 0 && j < w.n) unit[whole ? w.tx : w.tx * V + j] = red[w.tx];
    }
    __syncthreads();
    const int per = whole ? p.cg / V : p.cg;
    for (int g = tid; g < gs; g += (int)blockDim.x) {
        double2 t = unit[g * per];
        for (int u = 1; u < per; ++u) {
            t.x += unit[g * per + u].x;
            t.y += unit[g * per + u].y;
        }
        const float2 s = moments(t.x, t.y, (double)p.l * p.cg, eps);
        stat[g] = s;
        mean[(int64_t)blockIdx.y * p.groups + g0 + g] = s.x;
        rstd[(int64_t)blockIdx.y * p.groups + g0 + g] = s.y;
    }
    __syncthreads();
    if (w.n == 0) return;
    float mu[V], a[V], b[V];
    int g[V];
    groups_of<V>(w.tx * V, p.cg, gs, g);
    load_param<V>(weight, w.c0, w.n, 1.0f, a);
    load_param<V>(bias, w.c0, w.n, 0.0f, b);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 s = stat[g[j]];
        mu[j] = s.x;
        a[j] *= s.y * Act<ACT>::kArg;
        b[j] *= Act<ACT>::kArg;
    }
    walk_apply<DT, ANY, ACT, false>(x, y, w, p, mu, a, b, slope, scale);
}

// ---- backward ---------------------------------------------------------------------------------------------------------------

// kQ rows of the input: from the tensor, or (KEPT) from their codes
template <int DT, bool ANY, bool KEPT>
struct Input {
    static constexpr int V = Elem<DT>::kVec;
    Raw<DT> raw[kQ];
    RawCodes<V> code[kQ];
    unsigned e;
    __device__ __forceinline__ void load(const typename Elem<DT>::T* x, const int8_t* codes, const uint8_t* scales, int64_t row, int c0,
                                         int n, int have, const GnShape& p) {
        if constexpr (KEPT) {
#pragma unroll
            for (int i = 0; i < kQ; ++i)
                if (i < have) code[i].load(codes + (row + i) * p.blocks * kBlk8 + c0);
            e = load_exponents(scales + (int64_t)(c0 / kBlk8) * p.rows + row, have);
        } else {
#pragma unroll
            for (int i = 0; i < kQ; ++i)
                if (i < have) load_lane<ANY>(raw[i], x + (row + i) * p.c + c0, n, p.c);
        }
    }
    __device__ __forceinline__ void get(int i, float (&v)[V]) const {
        if constexpr (KEPT) code[i].get(block8_step((e >> (8 * i)) & 0xffu), v);
        else raw[i].get(v);
    }
};

// what a lane needs of its channels: the mean, and t = (x - mean) * a + b (b: from zero)
template <int V>
struct Affine {
    float mu[V], a[V], b[V];
};

// a thread's sums over its rows of g = gy act'(z) and of g (x - mean)
template <int DT, bool ANY, int ACT, bool KEPT, int V>
__device__ __forceinline__ void walk_bwd_sums(const typename Elem<DT>::T* __restrict__ gy, const typename Elem<DT>::T* __restrict__ x,
                                              const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const Walk& w,
                                              const GnShape& p, const Affine<V>& f, float slope, float (&s1)[V], float (&s2)[V]) {
    for (int64_t r = w.first + kQ * w.ty; r < w.r_end; r += kQ * w.rp) {
        const int64_t row = w.row0 + r;
        const int have = w.r_end - r < kQ ? (int)(w.r_end - r) : kQ;
        Input<DT, ANY, KEPT> in;
        Raw<DT> raw[kQ];
        in.load(x, codes, scales, row, w.c0, w.n, have, p);
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < have) load_lane<ANY>(raw[i], gy + (row + i) * p.c + w.c0, w.n, p.c);
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < have) {
                float v[V], g[V];
                in.get(i, v);
                raw[i].get(g);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[j] - f.mu[j];
                    const float dz = g[j] * Act<ACT>::derivative(fmaf(d, f.a[j], f.b[j]), slope);
                    s1[j] += dz;
                    s2[j] = fmaf(dz, d, s2[j]);
                }
            }
    }
}

// gx = ga * g + (x - mean) * gd + ge, g as above
template <int DT, bool ANY, int ACT, bool KEPT, bool STREAM, int V>
__device__ __forceinline__ void walk_bwd_apply(const typename Elem<DT>::T* __restrict__ gy, const typename Elem<DT>::T* __restrict__ x,
                                               const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                               typename Elem<DT>::T* __restrict__ gx, const Walk& w, const GnShape& p, const Affine<V>& f,
                                               const float (&ga)[V], const float (&gd)[V], const float (&ge)[V], float slope) {
    for (int64_t r = w.first + kQ * w.ty; r < w.r_end; r += kQ * w.rp) {
        const int64_t row = w.row0 + r;
        const int have = w.r_end - r < kQ ? (int)(w.r_end - r) : kQ;
        Input<DT, ANY, KEPT> in;
        Raw<DT> raw[kQ];
        in.load(x, codes, scales, row, w.c0, w.n, have, p);
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < have) load_lane<ANY>(raw[i], gy + (row + i) * p.c + w.c0, w.n, p.c);
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < have) {
                float v[V], g[V];
                in.get(i, v);
                raw[i].get(g);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[j] - f.mu[j];
                    const float dz = g[j] * Act<ACT>::derivative(fmaf(d, f.a[j], f.b[j]), slope);
                    v[j] = fmaf(ga[j], dz, fmaf(d, gd[j], ge[j]));
                }
                store_lane<ANY, STREAM, DT>(gx + (row + i) * p.c + w.c0, v, w.n);
            }
    }
}

// the four tensors every backward kernel reads besides gy
struct BwdIn {
    const float *mean, *rstd, *weight, *bias;
};

template <int V, int ACT>
__device__ __forceinline__ void load_affine(const BwdIn& in, int64_t n, int c0, int channels, const GnShape& p, Affine<V>& f) {
    int g[V];
    groups_of<V>(c0, p.cg, p.groups, g);
    load_param<V>(in.weight, c0, channels, 1.0f, f.a);
    load_param<V>(in.bias, c0, channels, 0.0f, f.b);
    float mu = 0.0f, rs = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (j == 0 || g[j] != g[j - 1]) {
            mu = in.mean[n * p.groups + g[j]];
            rs = in.rstd[n * p.groups + g[j]];
        }
        f.mu[j] = mu;
        f.a[j] *= rs * Act<ACT>::kArg;
        f.b[j] *= Act<ACT>::kArg;
    }
}

// record [n][chunk][channel]: the two sums over the chunk's rows
template <int DT, bool ANY, int ACT, bool KEPT>
__global__ __launch_bounds__(kBlock) void gn_bwd_sums_kernel(const typename Elem<DT>::T* __restrict__ gy,
                                                             const typename Elem<DT>::T* __restrict__ x,
                                                             const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             const BwdIn in, float2* __restrict__ rec, float slope, const GnShape p) {
    constexpr int V = Elem<DT>::kVec;
    __shared__ float2 red[V][kBlock];
    const int n = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
    Walk w;
    w.tx = tid % p.tile;
    w.ty = tid / p.tile;
    w.rp = p.rp;
    w.row0 = (int64_t)n * p.l;
    w.first = (int64_t)chunk * p.chunk_rows;
    w.r_end = w.first + p.chunk_rows < p.l ? w.first + p.chunk_rows : p.l;
    for (int lane0 = 0; lane0 < p.lanes; lane0 += p.tile) {
        w.c0 = (lane0 + w.tx) * V;
        w.n = lane_channels<V>(w.ty < w.rp, p.c - w.c0);
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
        if (w.n > 0) {
            Affine<V> f;
            load_affine<V, ACT>(in, n, w.c0, w.n, p, f);
            walk_bwd_sums<DT, ANY, ACT, KEPT>(gy, x, codes, scales, w, p, f, slope, s1, s2);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) red[j][tid] = float2{s1[j], s2[j]};
        int half = 1;
        while (half < p.rp) half <<= 1;
        for (half >>= 1; half >= 1; half >>= 1) {
            __syncthreads();
            if (w.ty < half && w.ty + half < p.rp)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 o = red[j][(w.ty + half) * p.tile + w.tx];
                    red[j][tid].x += o.x;
                    red[j][tid].y += o.y;
                }
        }
        if (w.ty == 0)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < w.n) rec[((int64_t)n * p.chunks + chunk) * p.c + w.c0 + j] = red[j][tid];
    }
}

// one work-group per (sample, group): the channels' totals {sum dz, sum dz xhat} and the group's two means
__global__ __launch_bounds__(kBlock) void gn_bwd_totals_kernel(const float2* __restrict__ rec, const float* __restrict__ weight,
                                                               const float* __restrict__ rstd, float2* __restrict__ totals,
                                                               float2* __restrict__ means, float scale, const GnShape p) {
    __shared__ double2 red[kBlock];
    const int g = blockIdx.x, n = blockIdx.y, tid = threadIdx.x;
    const int width = p.cg < kBlock ? p.cg : kBlock, depth = kBlock / width;
    const int tx = tid % width, ty = tid / width;
    const double s1 = scale, s2 = (double)scale * rstd[(int64_t)n * p.groups + g];
    double m1 = 0.0, m2 = 0.0;
    for (int u0 = 0; u0 < p.cg; u0 += width) {
        const int ch = g * p.cg + u0 + tx;
        const bool on = u0 + tx < p.cg && ty < depth;
        double a = 0.0, b = 0.0;
        if (on)
            for (int chunk = ty; chunk < p.chunks; chunk += depth) {
                const float2 t = rec[((int64_t)n * p.chunks + chunk) * p.c + ch];
                a += t.x;
                b += t.y;
            }
        __syncthreads();
        red[tid] = double2{a * s1, b * s2};
        fold_rows(red, tx, ty, width, depth, ty < depth);
        if (on && ty == 0) {
            const double2 t = red[tx];
            totals[(int64_t)n * p.c + ch] = float2{(float)t.x, (float)t.y};
            const double w = weight ? weight[ch] : 1.0;
            m1 += w * t.x;
            m2 += w * t.y;
        }
    }
    __syncthreads();
    red[tid] = double2{m1, m2};
    fold_rows(red, 0, tid, 1, kBlock, true);
    if (tid == 0) {
        const double m = (double)p.l * p.cg;
        means[(int64_t)n * p.groups + g] = float2{(float)(red[0].x / m), (float)(red[0].y / m)};
    }
}

// gw, gb: the samples' channel totals added in order
__device__ __forceinline__ void weight_grads(const float2* __restrict__ totals, float* __restrict__ gw, float* __restrict__ gb, int n,
                                             int c, int ch) {
    double a = 0.0, b = 0.0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
        const float2 t = totals[(int64_t)i * c + ch];
        a += t.x;
        b += t.y;
    }
    if (gb) gb[ch] = (float)a;
    if (gw) gw[ch] = (float)b;
}
__global__ __launch_bounds__(kBlock) void gn_bwd_weight_kernel(const float2* __restrict__ totals, float* __restrict__ gw,
                                                               float* __restrict__ gb, int n, int c) {
    const int ch = blockIdx.x * kBlock + threadIdx.x;
    if (ch < c) weight_grads(totals, gw, gb, n, c, ch);
}

template <int V>
__device__ __forceinline__ void bwd_factors(float rs, float2 m, float w, float scale, float& ga, float& gd, float& ge) {
    ga = rs * w * scale;
    gd = -rs * rs * m.y;
    ge = -rs * m.x;
}

// TOTALS: the two means and the weights' gradients too, from the records of the sums
template <int DT, bool ANY, int ACT, bool KEPT, bool TOTALS>
__global__ __launch_bounds__(kBlock) void gn_bwd_apply_kernel(const typename Elem<DT>::T* __restrict__ gy,
                                                              const typename Elem<DT>::T* __restrict__ x,
                                                              const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                              const BwdIn in, const float2* __restrict__ rec,
                                                              const float2* __restrict__ means,
                                                              const float2* __restrict__ totals, float* __restrict__ gw,
                                                              float* __restrict__ gb, typename Elem<DT>::T* __restrict__ gx, float slope,
                                                              float scale, const GnShape p) {
    constexpr int V = Elem<DT>::kVec;
    const int n = (int)gridDim.y - 1 - (int)blockIdx.y, chunk = (int)gridDim.x - 1 - (int)blockIdx.x, tid = threadIdx.x;
    __shared__ double2 red[TOTALS ? kBlock : 1];
    __shared__ double2 sums[TOTALS ? kFoldChannels : 1];
    __shared__ float2 stat[TOTALS ? kFoldGroups : 1];
    if constexpr (TOTALS) {
        const int lane = tid & (kWave - 1), waves = (int)(gridDim.x * gridDim.y) * (kBlock / kWave);
        if (gw || gb)                                              // a wave a channel, over all samples
            for (int ch = (int)(blockIdx.y * gridDim.x + blockIdx.x) * (kBlock / kWave) + (tid >> 6); ch < p.c; ch += waves) {
                double a = 0.0, b = 0.0;
                for (int i = lane; i < p.chunks * (int)gridDim.y; i += kWave) {
                    const float2 t = rec[(int64_t)i * p.c + ch];
                    a += t.x;
                    b += (double)t.y * in.rstd[(int64_t)(i / p.chunks) * p.groups + ch / p.cg];
                }
                a = wave_sum_d(a) * scale;
                b = wave_sum_d(b) * scale;
                if (lane == 0 && gb) gb[ch] = (float)a;
                if (lane == 0 && gw) gw[ch] = (float)b;
            }
        if (!gx) return;
        const int width = p.c < kBlock ? p.c : kBlock, depth = kBlock / width, tx = tid % width, ty = tid / width;
        for (int u0 = 0; u0 < p.c; u0 += width) {                  // the sample's channels
            const int ch = u0 + tx;
            double2 t{0.0, 0.0};
            if (ch < p.c && ty < depth)
#pragma unroll 4
                for (int i = ty; i < p.chunks; i += depth) {
                    const float2 o = rec[((int64_t)n * p.chunks + i) * p.c + ch];
                    t.x += o.x;
                    t.y += o.y;
                }
            __syncthreads();
            red[tid] = t;
            fold_rows(red, tx, ty, width, depth, ty < depth);
            if (ty == 0 && ch < p.c) sums[ch] = red[tx];
        }
        __syncthreads();
        const int per = fold_lanes(p.groups), g = tid / per;
        double m1 = 0.0, m2 = 0.0;
        if (g < p.groups)
            for (int u = tid - g * per; u < p.cg; u += per) {
                const int ch = g * p.cg + u;
                const double weight = in.weight ? in.weight[ch] : 1.0;
                m1 += weight * sums[ch].x;
                m2 += weight * sums[ch].y;
            }
        m1 = lanes_sum_d(m1, per);
        m2 = lanes_sum_d(m2, per);
        if (g < p.groups && tid == g * per) {
            const double m = (double)scale / ((double)p.l * p.cg);
            stat[g] = float2{(float)(m1 * m), (float)(m2 * m * in.rstd[(int64_t)n * p.groups + g])};
        }
        __syncthreads();
    } else if (totals) {                                           // gw and gb on the way, 256 channels a work-group
        const int blocks = (int)(gridDim.x * gridDim.y);
        for (int ch = (int)(blockIdx.y * gridDim.x + blockIdx.x) * kBlock + tid; ch < p.c; ch += blocks * kBlock)
            weight_grads(totals, gw, gb, (int)gridDim.y, p.c, ch);
    }
    Walk w;
    w.tx = tid % p.tile;
    w.ty = tid / p.tile;
    w.rp = p.rp;
    w.row0 = (int64_t)n * p.l;
    w.first = (int64_t)chunk * p.chunk_rows;
    w.r_end = w.first + p.chunk_rows < p.l ? w.first + p.chunk_rows : p.l;
    if (w.ty >= w.rp) return;
    for (int lane0 = 0; lane0 < p.lanes; lane0 += p.tile) {
        w.c0 = (lane0 + w.tx) * V;
        w.n = lane_channels<V>(true, p.c - w.c0);
        if (w.n == 0) return;
        Affine<V> f;
        load_affine<V, ACT>(in, n, w.c0, w.n, p, f);
        float ga[V], gd[V], ge[V];
        int g[V];
        groups_of<V>(w.c0, p.cg, p.groups, g);
        load_param<V>(in.weight, w.c0, w.n, 1.0f, ga);
        float rs = 0.0f;
        float2 m{0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j == 0 || g[j] != g[j - 1]) {
                rs = in.rstd[(int64_t)n * p.groups + g[j]];
                if constexpr (TOTALS) m = stat[g[j]];
                else m = means[(int64_t)n * p.groups + g[j]];
            }
            bwd_factors<V>(rs, m, ga[j], scale, ga[j], gd[j], ge[j]);
        }
        walk_bwd_apply<DT, ANY, ACT, KEPT, true>(gy, x, codes, scales, gx, w, p, f, ga, gd, ge, slope);
    }
}

// one launch: a sample's slab of groups; totals [n][c] for the weights' kernel, or (one sample) gw and gb themselves
template <int DT, bool ANY, int ACT, bool KEPT>
__global__ __launch_bounds__(kFused) void gn_bwd_fused_kernel(const typename Elem<DT>::T* __restrict__ gy,
                                                              const typename Elem<DT>::T* __restrict__ x,
                                                              const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                              const BwdIn in, float2* __restrict__ totals, float* __restrict__ gw,
                                                              float* __restrict__ gb, typename Elem<DT>::T* __restrict__ gx, float slope,
                                                              float scale, const GnShape p) {
    constexpr int V = Elem<DT>::kVec;
    __shared__ float2 red[V][kFused];
    __shared__ float2 mean[kFused];
    int g0, gs, width;
    const Walk w = slab_walk<V>(p, g0, gs, width);
    const int tid = threadIdx.x;
    Affine<V> f;
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
    if (w.n > 0) {
        load_affine<V, ACT>(in, blockIdx.y, w.c0, w.n, p, f);
        walk_bwd_sums<DT, ANY, ACT, KEPT>(gy, x, codes, scales, w, p, f, slope, s1, s2);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) red[j][tid] = float2{s1[j], s2[j]};
    int half = 1;
    while (half < p.rp) half <<= 1;
    for (half >>= 1; half >= 1; half >>= 1) {
        __syncthreads();
        if (w.ty < half && w.ty + half < p.rp)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 o = red[j][(w.ty + half) * p.tile + w.tx];
                red[j][tid].x += o.x;
                red[j][tid].y += o.y;
            }
    }
    __syncthreads();
    for (int i = tid; i < gs; i += (int)blockDim.x) {              // the group's channels in order
        const int64_t g = (int64_t)blockIdx.y * p.groups + g0 + i;
        const double k1 = scale, k2 = (double)scale * in.rstd[g];
        double m1 = 0.0, m2 = 0.0;
        for (int u = i * p.cg; u < (i + 1) * p.cg; ++u) {
            const float2 t = red[u % V][u / V];
            const int ch = g0 * p.cg + u;
            const double w1 = in.weight ? in.weight[ch] : 1.0, a = t.x * k1, b = t.y * k2;
            m1 += w1 * a;
            m2 += w1 * b;
            if (totals) totals[(int64_t)blockIdx.y * p.c + ch] = float2{(float)a, (float)b};
            if (gb) gb[ch] = (float)a;
            if (gw) gw[ch] = (float)b;
        }
        const double m = (double)p.l * p.cg;
        mean[i] = float2{(float)(m1 / m), (float)(m2 / m)};
    }
    __syncthreads();
    if (w.n == 0 || !gx) return;
    float ga[V], gd[V], ge[V];
    int g[V];
    groups_of<V>(w.tx * V, p.cg, gs, g);
    load_param<V>(in.weight, w.c0, w.n, 1.0f, ga);
#pragma unroll
    for (int j = 0; j < V; ++j)
        bwd_factors<V>(in.rstd[(int64_t)blockIdx.y * p.groups + g0 + g[j]], mean[g[j]], ga[j], scale, ga[j], gd[j], ge[j]);
    walk_bwd_apply<DT, ANY, ACT, KEPT, false>(gy, x, codes, scales, gx, w, p, f, ga, gd, ge, slope);
}

// ---- host -------------------------------------------------------------------------------------------------------------------

constexpr int64_t kMostChannels = 1 << 20, kMostSamples = 65535;

constexpr int64_t kMostValues = (int64_t)1 << 40;

// what a shape breaks (nullptr: nothing).  Samples are the grid's second dimension; a chunk's rows and its records are counted in 32 bits
const char* gn_shape_fault(int64_t n, int64_t l, int64_t c, int64_t groups) {
    if (n < 0 || l < 0 || c < 1 || groups < 1 || c % groups != 0) return "bad shape (n, l >= 0; c a multiple of groups >= 1)";
    if (n > kMostSamples) return "more than 65535 samples";
    if (c > kMostChannels) return "more than 1048576 channels";
    if (groups > 65535) return "more than 65535 groups";
    if (l > kMostValues / c || n * l > kMostValues / c) return "more than 2^40 values";
    return nullptr;
}

// Groups of a one-launch work-group: at least 64 bytes of a row (one group's share is often less, and every 64-byte piece is read
// whole); with codes whole 8-bit blocks where it writes them and whole vectors where it reads them; 0 if there is no such slab.
enum GnCodes { kNoCodes, kWriteCodes, kReadCodes };
int gn_slab(int64_t c, int64_t groups, int v, int esize, GnCodes codes) {
    const int64_t cg = c / groups, whole = codes == kWriteCodes ? kBlk8 : codes == kReadCodes ? v : 1;
    for (int64_t s = 1; s <= groups; ++s) {
        const int64_t w = s * cg;
        if (w > kFused || s > kFused) return 0;                    // a lane, a unit and a group at most for each thread
        if (s == groups || (w % whole == 0 && w * esize >= 64)) return (int)s;
    }
    return 0;
}

GnShape gn_plan(int64_t n, int64_t l, int64_t c, int64_t groups, int esize, GnCodes codes, bool backward) {
    const int v = 16 / esize;
    GnShape p;
    p.l = l;
    p.rows = n * l;
    p.c = (int)c;
    p.groups = (int)groups;
    p.cg = (int)(c / groups);
    p.blocks = (int)ceil_div64(c, kBlk8);
    p.units = p.cg % v == 0 ? (int)c / v : (int)c;
    p.slab = gn_slab(c, groups, v, esize, codes);
    p.slabs = p.slab ? (int)ceil_div64(groups, p.slab) : 0;
    // One launch where a thread of kFused has at most 64 values of its slab (backward: 32) and the tensor is small; backward of groups of
    // up to 16 channels only, which one thread adds up at the end.  Time against that of two or three launches, captured, f32 and bf16,
    // n of 1 ... 32, c of 128 ... 512 in groups of 4 ... 512, 546 shapes:
    //   forward, <= 10 MB    values a thread   < 16: 0.54 ... 0.94     16, 32: 0.60 ... 0.94     64: 0.66 ... 1.22, median 1.0 (a launch fewer)
    //                        (any group: one of 512 channels 0.73 ... 1.11);  beyond: 128 values 1.22 ... 1.43, 12 to 18 MB 0.89 ... 1.21
    //   backward, <= 4 MB, up to 32 values   groups of 4 channels 0.51 ... 0.99, 8 0.57 ... 1.02, 16 0.69 ... 1.13; of 32 11 ... 20 us, 64
    //                        16 ... 25, 128 27 ... 34, 256 48 ... 57, against 10 ... 17 in more launches
    // (knob 0, for tests: never)
    if (p.slab) {
        const int64_t values = l * p.slab * p.cg, bytes = n * l * c * esize;
        const bool small = backward ? p.cg <= 16 && values <= kFused * 32 && bytes <= ((int64_t)4 << 20)
                                    : values <= kFused * 64 && bytes <= ((int64_t)10 << 20);
        if (!small || tuning_knob("SAE_GN_ONE_LAUNCH", 1) == 0) p.slab = 0;
    }
    // lanes of so many channels; a walk that writes codes has all lanes of a block
    auto lanes_of = [&](int64_t w) { return (int)(codes == kWriteCodes ? ceil_div64(w, kBlk8) * (kBlk8 / v) : ceil_div64(w, v)); };
    p.any = c % v != 0 || (p.slab && (int64_t)p.slab * p.cg % v != 0);
    if (p.slab) {
        p.lanes = lanes_of((int64_t)p.slab * p.cg);
        p.tile = p.lanes;
        p.rp = kFused / p.tile;
        while (p.rp > 1 && (int64_t)(p.rp / 2) * kQ >= l) p.rp /= 2;          // (no more threads than rows)
        p.chunk_rows = 0;
        p.chunks = 1;
        return p;
    }
    p.lanes = lanes_of(c);
    p.tile = p.lanes < kBlock ? p.lanes : kBlock;
    p.rp = kBlock / p.tile;
    // Up to 8 work-groups per CU over the whole batch, while each thread has four trips of kQ rows (one trip alone is all prologue:
    // [16, 256, 64, 64] bf16 took 36 us so); down to 2 per CU with fewer trips than that.
    const int64_t step = (int64_t)kQ * p.rp, each = n > 0 ? n : 1;
    int64_t chunks = ceil_div64(l, 4 * step);
    if (chunks > ceil_div64(2048, each)) chunks = ceil_div64(2048, each);
    if (chunks < ceil_div64(512, each)) chunks = ceil_div64(512, each);
    if (chunks > ceil_div64(l, step)) chunks = ceil_div64(l, step);
    p.chunk_rows = (int)(ceil_div64(ceil_div64(l, chunks > 0 ? chunks : 1), step) * step);
    p.chunks = (int)ceil_div64(l, p.chunk_rows > 0 ? p.chunk_rows : 1);
    return p;
}

int64_t gn_workspace(const GnShape& p, int64_t n, bool backward) {
    if (p.slab) return backward && n > 1 ? n * p.c * (int64_t)sizeof(float2) : 0;
    if (!backward) return n * p.chunks * p.units * (int64_t)sizeof(double2);
    return (n * p.chunks * (int64_t)p.c + n * p.c + n * p.groups) * (int64_t)sizeof(float2);
}

struct GnArgs {
    const void *gy, *x;
    int8_t* codes;
    uint8_t* scales;
    float *mean, *rstd;
    const float *weight, *bias;
    void* out;
    float *gw, *gb;
    int64_t n;
    float eps, slope, scale;
    int act;
    void* ws;
    hipStream_t stream;
};

// The apply kernel adds a sample's records (`bytes` of them) itself: up to 64 KB for each work-group and 32 MB for all.  Captured, forward
// / backward, against a launch for the totals: few groups gain (bf16 [2, 64, 128, 128] in one group 10.8 / 17.2 against 14.5 / 22.6 us,
// f16 [3, 100, 33, 65] in one 21.2 / 19.0 against 29.4 / 21.1, in 25 17.8 / 18.9 against 17.2 / 18.8), the most that is lost is 6 %
// (bf16 [2, 64, 128, 128] in 16: 17.6 / 17.2 against 17.6 / 16.2); an eager training step of two launches fewer takes 4 % less.  At 128 KB
// it takes longer (f16 [8, 320, 1000] backward 26.2 against 18.5).
// (knob 0, for tests: never)
bool fold_totals(const GnShape& p, int64_t n, int64_t bytes) {
    return p.groups <= kFoldGroups && bytes <= ((int64_t)64 << 10) && bytes * p.chunks * n <= ((int64_t)32 << 20) &&
           tuning_knob("SAE_GN_FOLD", 1) != 0;
}

template <int DT, bool ANY, int ACT>
void gn_forward_as(const GnArgs& a, const GnShape& p) {
    using T = typename Elem<DT>::T;
    if (p.slab) {
        const dim3 grid((unsigned)p.slabs, (unsigned)a.n), block((unsigned)(p.tile * p.rp));
        if (a.codes)
            hipLaunchKernelGGL((gn_fused_kernel<DT, ANY, ACT, true>), grid, block, 0, a.stream, (const T*)a.x, a.weight, a.bias, (T*)a.out,
                               a.mean, a.rstd, a.codes, a.scales, a.eps, a.slope, a.scale, p);
        else
            hipLaunchKernelGGL((gn_fused_kernel<DT, ANY, ACT, false>), grid, block, 0, a.stream, (const T*)a.x, a.weight, a.bias,
                               (T*)a.out, a.mean, a.rstd, a.codes, a.scales, a.eps, a.slope, a.scale, p);
        return;
    }
    const dim3 grid((unsigned)p.chunks, (unsigned)a.n), block(kBlock);
    double2* rec = (double2*)a.ws;
    if (a.codes)
        hipLaunchKernelGGL((gn_sums_kernel<DT, ANY, true>), grid, block, 0, a.stream, (const T*)a.x, rec, a.codes, a.scales, p);
    else
        hipLaunchKernelGGL((gn_sums_kernel<DT, ANY, false>), grid, block, 0, a.stream, (const T*)a.x, rec, a.codes, a.scales, p);
    if (fold_totals(p, a.n, (int64_t)p.chunks * p.units * (int64_t)sizeof(double2))) {
        hipLaunchKernelGGL((gn_apply_kernel<DT, ANY, ACT, true>), grid, block, 0, a.stream, (const T*)a.x, (const double2*)rec, a.mean,
                           a.rstd, a.weight, a.bias, (T*)a.out, a.eps, a.slope, a.scale, p);
        return;
    }
    hipLaunchKernelGGL(gn_totals_kernel, dim3((unsigned)p.groups, (unsigned)a.n), dim3(kWave), 0, a.stream, (const double2*)rec,
                       a.mean, a.rstd, a.eps, p);
    hipLaunchKernelGGL((gn_apply_kernel<DT, ANY, ACT, false>), grid, block, 0, a.stream, (const T*)a.x, (const double2*)rec, a.mean,
                       a.rstd, a.weight, a.bias, (T*)a.out, a.eps, a.slope, a.scale, p);
}

template <int DT, bool ANY, int ACT, bool KEPT>
void gn_backward_as(const GnArgs& a, const GnShape& p) {
    using T = typename Elem<DT>::T;
    const BwdIn in{a.mean, a.rstd, a.weight, a.bias};
    const bool weights = a.gw || a.gb;
    if (p.slab) {
        const dim3 grid((unsigned)p.slabs, (unsigned)a.n), block((unsigned)(p.tile * p.rp));
        float2* totals = a.n > 1 && weights ? (float2*)a.ws : nullptr;
        hipLaunchKernelGGL((gn_bwd_fused_kernel<DT, ANY, ACT, KEPT>), grid, block, 0, a.stream, (const T*)a.gy, (const T*)a.x,
                           (const int8_t*)a.codes, (const uint8_t*)a.scales, in, totals, totals ? nullptr : a.gw,
                           totals ? nullptr : a.gb, (T*)a.out, a.slope, a.scale, p);
        if (totals)
            hipLaunchKernelGGL(gn_bwd_weight_kernel, dim3((unsigned)ceil_div(p.c, kBlock)), dim3(kBlock), 0, a.stream,
                               (const float2*)totals, a.gw, a.gb, (int)a.n, p.c);
        return;
    }
    const dim3 grid((unsigned)p.chunks, (unsigned)a.n), block(kBlock);
    float2* rec = (float2*)a.ws;
    float2* totals = rec + a.n * p.chunks * (int64_t)p.c;
    float2* means = totals + a.n * p.c;
    hipLaunchKernelGGL((gn_bwd_sums_kernel<DT, ANY, ACT, KEPT>), grid, block, 0, a.stream, (const T*)a.gy, (const T*)a.x,
                       (const int8_t*)a.codes, (const uint8_t*)a.scales, in, rec, a.slope, p);
    // (a wave adds two channels' weight gradients at most: where few work-groups share many channels, that is what everything waits
    // for -- f32 [1, 512, 4, 4] 49 us against 12 with a launch for the totals, [1, 128, 8, 8] 20 against 12, [4, 256, 8, 8], four
    // channels a wave, 13 against 12; two: [8, 256, 8, 8] 11 against 13, bf16 [4, 128, 32, 32] 14 against 16)
    const bool waves = p.c <= 2 * (kBlock / kWave) * (int64_t)p.chunks * a.n;
    if (waves && p.c <= kFoldChannels && fold_totals(p, a.n, (int64_t)p.chunks * p.c * (int64_t)sizeof(float2))) {
        hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, ANY, ACT, KEPT, true>), grid, block, 0, a.stream, (const T*)a.gy, (const T*)a.x,
                           (const int8_t*)a.codes, (const uint8_t*)a.scales, in, (const float2*)rec, (const float2*)nullptr,
                           (const float2*)nullptr, a.gw, a.gb, (T*)a.out, a.slope, a.scale, p);
        return;
    }
    hipLaunchKernelGGL(gn_bwd_totals_kernel, dim3((unsigned)p.groups, (unsigned)a.n), block, 0, a.stream, (const float2*)rec,
                       a.weight, (const float*)a.rstd, totals, means, a.scale, p);
    if (a.out)
        hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, ANY, ACT, KEPT, false>), grid, block, 0, a.stream, (const T*)a.gy, (const T*)a.x,
                           (const int8_t*)a.codes, (const uint8_t*)a.scales, in, (const float2*)nullptr, (const float2*)means,
                           weights ? (const float2*)totals : (const float2*)nullptr, a.gw, a.gb, (T*)a.out, a.slope, a.scale, p);
    else
        hipLaunchKernelGGL(gn_bwd_weight_kernel, dim3((unsigned)ceil_div(p.c, kBlock)), block, 0, a.stream, (const float2*)totals,
                           a.gw, a.gb, (int)a.n, p.c);
}

template <int DT, bool ANY, int ACT>
void gn_run(const GnArgs& a, const GnShape& p, bool backward) {
    if (!backward) gn_forward_as<DT, ANY, ACT>(a, p);
    else if (a.codes) gn_backward_as<DT, ANY, ACT, true>(a, p);
    else gn_backward_as<DT, ANY, ACT, false>(a, p);
}

template <int DT, bool ANY>
void gn_run(const GnArgs& a, const GnShape& p, bool backward) {
    if (a.act == SAE_ACT_LRELU) gn_run<DT, ANY, SAE_ACT_LRELU>(a, p, backward);
    else if (a.act == SAE_ACT_SILU) gn_run<DT, ANY, SAE_ACT_SILU>(a, p, backward);
    else gn_run<DT, ANY, SAE_ACT_NONE>(a, p, backward);
}

template <int DT>
void gn_run(const GnArgs& a, const GnShape& p, bool backward) {
    if (p.any) gn_run<DT, true>(a, p, backward);
    else gn_run<DT, false>(a, p, backward);
}

int gn_dispatch(const char* what, GnArgs& a, int64_t l, int64_t c, int64_t groups, int32_t dtype, int64_t ws_bytes, bool backward) {
    const GnCodes codes = !a.codes ? kNoCodes : backward ? kReadCodes : kWriteCodes;
    const GnShape p = gn_plan(a.n, l, c, groups, elem_bytes(dtype), codes, backward);
    const int64_t need = gn_workspace(p, a.n, backward);
    if (need > 0 && (!a.ws || ws_bytes < need))
        return fail(SAE_EWORKSPACE, "%s: workspace %lld < %lld bytes (sae_group_norm_act_workspace)", what, (long long)ws_bytes,
                    (long long)need);
    for (const void* t : {a.gy, a.x, (const void*)a.out, (const void*)a.ws, (const void*)a.codes})
        if (!aligned16(t)) return fail(SAE_EINVAL, "%s: tensors must be 16-byte aligned", what);
    if (dtype == SAE_F32) gn_run<SAE_F32>(a, p, backward);
    else if (dtype == SAE_BF16) gn_run<SAE_BF16>(a, p, backward);
    else gn_run<SAE_F16>(a, p, backward);
    return check_launch(what);
}

}  // namespace
}  // namespace sae

using namespace sae;

extern "C" int64_t sae_group_norm_act_workspace(int64_t n, int64_t l, int64_t c, int64_t groups, int32_t dtype, int32_t backward) {
    if (gn_shape_fault(n, l, c, groups) || !elem_known(dtype) || n == 0 || l == 0) return 0;
    const int64_t without = gn_workspace(gn_plan(n, l, c, groups, elem_bytes(dtype), kNoCodes, backward != 0), n, backward != 0);
    const int64_t with = gn_workspace(gn_plan(n, l, c, groups, elem_bytes(dtype), backward ? kReadCodes : kWriteCodes, backward != 0), n,
                                       backward != 0);
    return with > without ? with : without;
}

extern "C" int sae_group_norm_act(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                                  int8_t* codes, uint8_t* scales, int64_t n, int64_t l, int64_t c, int64_t groups, float eps,
                                  int32_t act, float slope, float scale, int32_t dtype, void* workspace, int64_t workspace_bytes,
                                  sae_stream_t stream) {
    sae::clear_stale_error();
    if (!elem_known(dtype) || act < SAE_ACT_NONE || act > SAE_ACT_SILU)
        return fail(SAE_EINVAL, "sae_group_norm_act: unknown element type or activation");
    if (const char* fault = gn_shape_fault(n, l, c, groups)) return fail(SAE_EINVAL, "sae_group_norm_act: %s", fault);
    if (!(eps >= 0.0f)) return fail(SAE_EINVAL, "sae_group_norm_act: negative eps");
    if ((codes == nullptr) != (scales == nullptr)) return fail(SAE_EINVAL, "sae_group_norm_act: codes and scales go together");
    if (n == 0 || l == 0) return SAE_OK;
    if (!x || !y || !mean || !rstd) return fail(SAE_EINVAL, "sae_group_norm_act: null tensor");
    GnArgs a{nullptr, x, codes, scales, mean, rstd, weight, bias, y, nullptr, nullptr, n, eps, slope, scale, act, workspace,
             (hipStream_t)stream};
    return gn_dispatch("sae_group_norm_act", a, l, c, groups, dtype, workspace_bytes, false);
}

extern "C" int sae_group_norm_act_bwd(const void* gy, const void* x, const int8_t* codes, const uint8_t* scales, const float* mean,
                                      const float* rstd, const float* weight, const float* bias, void* gx, float* gw, float* gb,
                                      int64_t n, int64_t l, int64_t c, int64_t groups, int32_t act, float slope, float scale,
                                      int32_t dtype, void* workspace, int64_t workspace_bytes, sae_stream_t stream) {
    sae::clear_stale_error();
    if (!elem_known(dtype) || act < SAE_ACT_NONE || act > SAE_ACT_SILU)
        return fail(SAE_EINVAL, "sae_group_norm_act_bwd: unknown element type or activation");
    if (const char* fault = gn_shape_fault(n, l, c, groups)) return fail(SAE_EINVAL, "sae_group_norm_act_bwd: %s", fault);
    if ((codes == nullptr) != (scales == nullptr) || (codes == nullptr) == (x == nullptr && n > 0 && l > 0))
        return fail(SAE_EINVAL, "sae_group_norm_act_bwd: either x or codes and scales");
    if (n == 0 || l == 0) {
        if (gw || gb) {
            hipLaunchKernelGGL(gn_bwd_weight_kernel, dim3((unsigned)ceil_div64(c, kBlock)), dim3(kBlock), 0, (hipStream_t)stream,
                               (const float2*)nullptr, gw, gb, 0, (int)c);
            return check_launch("sae_group_norm_act_bwd");
        }
        return SAE_OK;
    }
    if (!gy || !mean || !rstd || (!gx && !gw && !gb)) return fail(SAE_EINVAL, "sae_group_norm_act_bwd: null tensor");
    GnArgs a{gy, x, const_cast<int8_t*>(codes), const_cast<uint8_t*>(scales), const_cast<float*>(mean), const_cast<float*>(rstd),
             weight, bias, gx, gw, gb, n, 0.0f, slope, scale, act, workspace, (hipStream_t)stream};
    return gn_dispatch("sae_group_norm_act_bwd", a, l, c, groups, dtype, workspace_bytes, true);
}
