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
//     totals    the chunks' records added in order: mean / rstd, or m1 / m2 and the channel sums
//     apply     the elementwise pass
// All of them are HBM-bound: forward 2 reads + 1 write (the floor is 1 + 1), backward 4 + 1 (2 + 1).
//
// Numerics: a thread adds x - x0 and (x - x0)^2 over its rows, x0 the first value it meets in the channel: at most the number of
// its rows times the rounding of a plain sum, whatever the channel's mean.  The records are moments about zero in 64 bits, which
// only have to be added.  mean and rstd are fp32; nothing is held in less.
#include "elem8.inc"

namespace sae {
namespace {

struct GnShape {
    int64_t l;                 // positions of a sample
    int64_t rows;              // n * l: rows of codes, stride of a block's exponents
    int c, groups, cg;
    int lanes;                 // channel vectors of a row, padded to whole 8-bit blocks
    int tile;                  // lanes a work-group covers at a time: min(lanes, kBlock)
    int rp;                    // rows it covers at a time: kBlock / tile
    int chunk_rows;            // rows of a work-group
    int chunks;                // chunks of a sample
    int units;                 // records of a chunk: channel vectors if a vector lies in one group, channels if not
    int blocks;                // 8-bit blocks of a row
};

#ifdef HIPEMU
__device__ __forceinline__ float exp2_fast(float v) { return exp2f(v); }
__device__ __forceinline__ float rcp_fast(float v) { return 1.0f / v; }
#else
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }    // 1 ulp
__device__ __forceinline__ float rcp_fast(float v) { return __builtin_amdgcn_rcpf(v); }      // 1 ulp
#endif

// 1 / (1 + exp(-z)); z -> -infinity: exp2 gives infinity and the quotient 0
__device__ __forceinline__ float sigmoid_f(float z) { return rcp_fast(1.0f + exp2_fast(z * -1.44269504088896341f)); }

template <int ACT>
__device__ __forceinline__ float act_f(float z, float slope) {
    if constexpr (ACT == SAE_ACT_LRELU) return z > 0.0f ? z : z * slope;
    else if constexpr (ACT == SAE_ACT_SILU) return z * sigmoid_f(z);
    else return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope_f(float z, float slope) {
    if constexpr (ACT == SAE_ACT_LRELU) return z > 0.0f ? 1.0f : slope;
    else if constexpr (ACT == SAE_ACT_SILU) {
        const float s = sigmoid_f(z);
        return s * fmaf(z, 1.0f - s, 1.0f);
    } else return 1.0f;
}

// ---- forward ----------------------------------------------------------------------------------------------------------------

// record [n][chunk][unit]: sum x and sum x^2 of the unit over the chunk's rows
template <int DT, int V, bool KEEP>
__global__ __launch_bounds__(kBlock) void gn_sums_kernel(const typename Elem<DT>::T* __restrict__ x, double2* __restrict__ rec,
                                                         int8_t* __restrict__ codes, uint8_t* __restrict__ scales, const GnShape p) {
    constexpr int LB = kBlk8 / V;
    __shared__ double2 red[kBlock * V];
    const int n = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
    const int tx = tid % p.tile, ty = tid / p.tile;
    const int64_t r_begin = (int64_t)chunk * p.chunk_rows;
    const int64_t r_end = r_begin + p.chunk_rows < p.l ? r_begin + p.chunk_rows : p.l;
    const bool whole = p.cg % V == 0;
    for (int lane0 = 0; lane0 < p.lanes; lane0 += p.tile) {
        const int c0 = (lane0 + tx) * V;
        const bool live = ty < p.rp && c0 < p.c;
        float k[V], s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) k[j] = s1[j] = s2[j] = 0.0f;
        int64_t count = 0;
        if (live && r_begin + ty < r_end) load_vec<DT, V>(x + ((int64_t)n * p.l + r_begin + ty) * p.c + c0, k);
        // (every lane of a work-group makes the same trips: the blocks' lanes meet in shuffles)
        for (int64_t r0 = r_begin; r0 < r_end; r0 += p.rp) {
            const int64_t r = r0 + ty;
            const bool on = live && r < r_end;
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = 0.0f;
            if (on) {
                load_vec<DT, V>(x + ((int64_t)n * p.l + r) * p.c + c0, v);
                ++count;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[j] - k[j];
                    s1[j] += d;
                    s2[j] = fmaf(d, d, s2[j]);
                }
            }
            if constexpr (KEEP) {
                const unsigned e = block8_exponent<DT>(block8_amax<LB>(vec_amax<V>(v)));
                const int cb = (lane0 + tx) / LB;
                const int64_t row = (int64_t)n * p.l + r;
                if (ty < p.rp && cb < p.blocks && r < r_end) {
                    store_codes<V>(codes + row * p.blocks * kBlk8 + c0, v, block8_inverse(e));
                    if ((lane0 + tx) % LB == 0) scales[(int64_t)cb * p.rows + row] = (uint8_t)e;
                }
            }
        }
        // moments about zero, then the sum over the rows' threads
        __syncthreads();
        const double m = (double)count;
        double a = 0.0, b = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const double kd = k[j], d1 = s1[j];
            const double sx = m * kd + d1, sxx = (double)s2[j] + 2.0 * kd * d1 + m * kd * kd;
            if (whole) { a += sx; b += sxx; }
            else red[tid * V + j] = double2{sx, sxx};
        }
        if (whole) red[tid] = double2{a, b};
        __syncthreads();
        const int per = whole ? 1 : V;
        for (int u = tid; u < p.tile * per; u += kBlock) {
            const int unit = lane0 * per + u;
            if (unit >= p.units) continue;
            double2 t = red[u];
            for (int y = 1; y < p.rp; ++y) {
                const double2 o = red[y * p.tile * per + u];
                t.x += o.x;
                t.y += o.y;
            }
            rec[((int64_t)n * p.chunks + chunk) * p.units + unit] = t;
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
    for (int i = threadIdx.x; i < p.chunks * per; i += kWave) {
        const int chunk = i / per, u = i - chunk * per;
        const double2 t = rec[((int64_t)n * p.chunks + chunk) * p.units + g * per + u];
        a += t.x;
        b += t.y;
    }
    a = wave_sum_d(a);
    b = wave_sum_d(b);
    if (threadIdx.x == 0) {
        const double m = (double)p.l * p.cg, mu = a / m;
        double var = b / m - mu * mu;
        if (var < 0.0) var = 0.0;            // (a NaN stays one)
        mean[(int64_t)n * p.groups + g] = (float)mu;
        rstd[(int64_t)n * p.groups + g] = (float)(1.0 / sqrt(var + (double)eps));
    }
}

template <int DT, int V, int ACT>
__global__ __launch_bounds__(kBlock) void gn_apply_kernel(const typename Elem<DT>::T* __restrict__ x, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, const float* __restrict__ weight,
                                                          const float* __restrict__ bias, typename Elem<DT>::T* __restrict__ y,
                                                          float slope, float scale, const GnShape p) {
    const int n = blockIdx.y, tid = threadIdx.x;
    const int tx = tid % p.tile, ty = tid / p.tile;
    const int64_t r_begin = (int64_t)blockIdx.x * p.chunk_rows;
    const int64_t r_end = r_begin + p.chunk_rows < p.l ? r_begin + p.chunk_rows : p.l;
    if (ty >= p.rp) return;
    for (int lane0 = 0; lane0 < p.lanes; lane0 += p.tile) {
        const int c0 = (lane0 + tx) * V;
        if (c0 >= p.c) return;
        float mu[V], a[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int64_t g = (int64_t)n * p.groups + (c0 + j) / p.cg;
            mu[j] = mean[g];
            a[j] = rstd[g] * (weight ? weight[c0 + j] : 1.0f);
            b[j] = bias ? bias[c0 + j] : 0.0f;
        }
        for (int64_t r = r_begin + ty; r < r_end; r += p.rp) {
            const int64_t at = ((int64_t)n * p.l + r) * p.c + c0;
            float v[V];
            load_vec<DT, V>(x + at, v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = act_f<ACT>(fmaf(v[j] - mu[j], a[j], b[j]), slope) * scale;
            store_vec<DT, V>(y + at, v);
        }
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------

// V neighbours of the input: from the tensor, or (KEPT) what their codes stand for
template <int DT, int V, bool KEPT>
__device__ __forceinline__ void load_input(const typename Elem<DT>::T* x, const int8_t* codes, const uint8_t* scales, int64_t row,
                                           int c0, const GnShape& p, float (&v)[V]) {
    if constexpr (KEPT) load_codes<V>(codes + row * p.blocks * kBlk8 + c0, block8_step(scales[(int64_t)(c0 / kBlk8) * p.rows + row]), v);
    else load_vec<DT, V>(x + row * p.c + c0, v);
}

// record [n][chunk][channel]: sum dz and sum dz xhat over the chunk's rows
template <int DT, int V, int ACT, bool KEPT>
__global__ __launch_bounds__(kBlock) void gn_bwd_sums_kernel(const typename Elem<DT>::T* __restrict__ gy,
                                                             const typename Elem<DT>::T* __restrict__ x,
                                                             const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             const float* __restrict__ weight, const float* __restrict__ bias,
                                                             float2* __restrict__ rec, float slope, float scale, const GnShape p) {
    __shared__ float2 red[kBlock * V];
    const int n = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
    const int tx = tid % p.tile, ty = tid / p.tile;
    const int64_t r_begin = (int64_t)chunk * p.chunk_rows;
    const int64_t r_end = r_begin + p.chunk_rows < p.l ? r_begin + p.chunk_rows : p.l;
    for (int lane0 = 0; lane0 < p.lanes; lane0 += p.tile) {
        const int c0 = (lane0 + tx) * V;
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
        if (ty < p.rp && c0 < p.c) {
            float mu[V], rs[V], w[V], b[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int64_t g = (int64_t)n * p.groups + (c0 + j) / p.cg;
                mu[j] = mean[g];
                rs[j] = rstd[g];
                w[j] = weight ? weight[c0 + j] : 1.0f;
                b[j] = bias ? bias[c0 + j] : 0.0f;
            }
            for (int64_t r = r_begin + ty; r < r_end; r += p.rp) {
                const int64_t row = (int64_t)n * p.l + r;
                float v[V], g[V];
                load_input<DT, V, KEPT>(x, codes, scales, row, c0, p, v);
                load_vec<DT, V>(gy + row * p.c + c0, g);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xh = (v[j] - mu[j]) * rs[j];
                    const float dz = g[j] * (act_slope_f<ACT>(fmaf(xh, w[j], b[j]), slope) * scale);
                    s1[j] += dz;
                    s2[j] = fmaf(dz, xh, s2[j]);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) red[tid * V + j] = float2{s1[j], s2[j]};
        __syncthreads();
        for (int u = tid; u < p.tile * V; u += kBlock) {
            const int ch = lane0 * V + u;
            if (ch >= p.c) continue;
            float2 t = red[u];
            for (int y = 1; y < p.rp; ++y) {
                const float2 o = red[y * p.tile * V + u];
                t.x += o.x;
                t.y += o.y;
            }
            rec[((int64_t)n * p.chunks + chunk) * p.c + ch] = t;
        }
    }
}

// one work-group per (sample, group): the channels' totals and the group's two means
__global__ __launch_bounds__(kBlock) void gn_bwd_totals_kernel(const float2* __restrict__ rec, const float* __restrict__ weight,
                                                               float2* __restrict__ totals, float2* __restrict__ means,
                                                               const GnShape p) {
    __shared__ double2 red[kBlock];
    const int g = blockIdx.x, n = blockIdx.y, tid = threadIdx.x;
    const int width = p.cg < kBlock ? p.cg : kBlock, depth = kBlock / width;
    const int tx = tid % width, ty = tid / width;
    double m1 = 0.0, m2 = 0.0;
    for (int u0 = 0; u0 < p.cg; u0 += width) {
        const int ch = g * p.cg + u0 + tx;
        const bool on = u0 + tx < p.cg;
        double a = 0.0, b = 0.0;
        if (on && ty < depth)
            for (int chunk = ty; chunk < p.chunks; chunk += depth) {
                const float2 t = rec[((int64_t)n * p.chunks + chunk) * p.c + ch];
                a += t.x;
                b += t.y;
            }
        __syncthreads();
        red[tid] = double2{a, b};
        __syncthreads();
        if (on && ty == 0) {
            for (int y = 1; y < depth; ++y) {
                a += red[y * width + tx].x;
                b += red[y * width + tx].y;
            }
            totals[(int64_t)n * p.c + ch] = float2{(float)a, (float)b};
            const double w = weight ? weight[ch] : 1.0;
            m1 += w * a;
            m2 += w * b;
        }
    }
    __syncthreads();
    red[tid] = double2{m1, m2};
    __syncthreads();
    for (int half = kBlock / 2; half >= 1; half >>= 1) {
        if (tid < half) {
            red[tid].x += red[tid + half].x;
            red[tid].y += red[tid + half].y;
        }
        __syncthreads();
    }
    if (tid == 0) {
        const double m = (double)p.l * p.cg;
        means[(int64_t)n * p.groups + g] = float2{(float)(red[0].x / m), (float)(red[0].y / m)};
    }
}

// gw, gb: the samples' channel totals added in order
__global__ __launch_bounds__(kBlock) void gn_bwd_weight_kernel(const float2* __restrict__ totals, float* __restrict__ gw,
                                                               float* __restrict__ gb, int n, int c) {
    const int ch = blockIdx.x * kBlock + threadIdx.x;
    if (ch >= c) return;
    double a = 0.0, b = 0.0;
    for (int i = 0; i < n; ++i) {
        const float2 t = totals[(int64_t)i * c + ch];
        a += t.x;
        b += t.y;
    }
    if (gb) gb[ch] = (float)a;
    if (gw) gw[ch] = (float)b;
}

template <int DT, int V, int ACT, bool KEPT>
__global__ __launch_bounds__(kBlock) void gn_bwd_apply_kernel(const typename Elem<DT>::T* __restrict__ gy,
                                                              const typename Elem<DT>::T* __restrict__ x,
                                                              const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              const float* __restrict__ weight, const float* __restrict__ bias,
                                                              const float2* __restrict__ means, typename Elem<DT>::T* __restrict__ gx,
                                                              float slope, float scale, const GnShape p) {
    const int n = blockIdx.y, tid = threadIdx.x;
    const int tx = tid % p.tile, ty = tid / p.tile;
    const int64_t r_begin = (int64_t)blockIdx.x * p.chunk_rows;
    const int64_t r_end = r_begin + p.chunk_rows < p.l ? r_begin + p.chunk_rows : p.l;
    if (ty >= p.rp) return;
    for (int lane0 = 0; lane0 < p.lanes; lane0 += p.tile) {
        const int c0 = (lane0 + tx) * V;
        if (c0 >= p.c) return;
        float mu[V], rs[V], w[V], b[V], m1[V], m2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int64_t g = (int64_t)n * p.groups + (c0 + j) / p.cg;
            mu[j] = mean[g];
            rs[j] = rstd[g];
            w[j] = weight ? weight[c0 + j] : 1.0f;
            b[j] = bias ? bias[c0 + j] : 0.0f;
            m1[j] = means[g].x;
            m2[j] = means[g].y;
        }
        for (int64_t r = r_begin + ty; r < r_end; r += p.rp) {
            const int64_t row = (int64_t)n * p.l + r;
            float v[V], g[V];
            load_input<DT, V, KEPT>(x, codes, scales, row, c0, p, v);
            load_vec<DT, V>(gy + row * p.c + c0, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (v[j] - mu[j]) * rs[j];
                const float dz = g[j] * (act_slope_f<ACT>(fmaf(xh, w[j], b[j]), slope) * scale);
                v[j] = rs[j] * (fmaf(w[j], dz, -m1[j]) - xh * m2[j]);
            }
            store_vec<DT, V>(gx + row * p.c + c0, v);
        }
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------

constexpr int64_t kMostChannels = 1 << 20, kMostSamples = 65535;

bool gn_shape_ok(int64_t n, int64_t l, int64_t c, int64_t groups) {
    return n >= 0 && n <= kMostSamples && l >= 0 && c >= 1 && c <= kMostChannels && groups >= 1 && groups <= 65535 &&
           c % groups == 0 && l <= ((int64_t)1 << 40) / c;
}

GnShape gn_plan(int64_t n, int64_t l, int64_t c, int64_t groups, int v) {
    GnShape p;
    p.l = l;
    p.rows = n * l;
    p.c = (int)c;
    p.groups = (int)groups;
    p.cg = (int)(c / groups);
    p.blocks = (int)ceil_div64(c, kBlk8);
    p.lanes = p.blocks * (kBlk8 / v);
    p.tile = p.lanes < kBlock ? p.lanes : kBlock;
    p.rp = kBlock / p.tile;
    // ~8 work-groups per CU over the whole batch, at least four rows for each thread
    const int64_t most = ceil_div64(l, 4 * (int64_t)p.rp), want = ceil_div64(2048, n > 0 ? n : 1);
    const int64_t chunks = most < want ? most : want;
    p.chunk_rows = (int)(ceil_div64(ceil_div64(l, chunks > 0 ? chunks : 1), p.rp) * p.rp);
    p.chunks = (int)ceil_div64(l, p.chunk_rows > 0 ? p.chunk_rows : 1);
    p.units = p.cg % v == 0 ? (int)c / v : (int)c;
    return p;
}

int64_t gn_workspace(const GnShape& p, int64_t n, bool backward) {
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

template <int DT, int V>
int gn_forward(const GnArgs& a, const GnShape& p) {
    using T = typename Elem<DT>::T;
    const dim3 grid((unsigned)p.chunks, (unsigned)a.n), block(kBlock);
    double2* rec = (double2*)a.ws;
    if (a.codes)
        hipLaunchKernelGGL((gn_sums_kernel<DT, V, true>), grid, block, 0, a.stream, (const T*)a.x, rec, a.codes, a.scales, p);
    else
        hipLaunchKernelGGL((gn_sums_kernel<DT, V, false>), grid, block, 0, a.stream, (const T*)a.x, rec, a.codes, a.scales, p);
    hipLaunchKernelGGL(gn_totals_kernel, dim3((unsigned)p.groups, (unsigned)a.n), dim3(kWave), 0, a.stream, (const double2*)rec,
                       a.mean, a.rstd, a.eps, p);
#define SAE_GN_APPLY(ACT)                                                                                                      \
    hipLaunchKernelGGL((gn_apply_kernel<DT, V, ACT>), grid, block, 0, a.stream, (const T*)a.x, (const float*)a.mean,           \
                       (const float*)a.rstd, a.weight, a.bias, (T*)a.out, a.slope, a.scale, p)
    if (a.act == SAE_ACT_LRELU) SAE_GN_APPLY(SAE_ACT_LRELU);
    else if (a.act == SAE_ACT_SILU) SAE_GN_APPLY(SAE_ACT_SILU);
    else SAE_GN_APPLY(SAE_ACT_NONE);
#undef SAE_GN_APPLY
    return check_launch("sae_group_norm_act");
}

template <int DT, int V, int ACT, bool KEPT>
int gn_backward_as(const GnArgs& a, const GnShape& p) {
    using T = typename Elem<DT>::T;
    const dim3 grid((unsigned)p.chunks, (unsigned)a.n), block(kBlock);
    float2* rec = (float2*)a.ws;
    float2* totals = rec + a.n * p.chunks * (int64_t)p.c;
    float2* means = totals + a.n * p.c;
    hipLaunchKernelGGL((gn_bwd_sums_kernel<DT, V, ACT, KEPT>), grid, block, 0, a.stream, (const T*)a.gy, (const T*)a.x,
                       (const int8_t*)a.codes, (const uint8_t*)a.scales, (const float*)a.mean, (const float*)a.rstd, a.weight,
                       a.bias, rec, a.slope, a.scale, p);
    hipLaunchKernelGGL(gn_bwd_totals_kernel, dim3((unsigned)p.groups, (unsigned)a.n), block, 0, a.stream, (const float2*)rec,
                       a.weight, totals, means, p);
    if (a.gw || a.gb)
        hipLaunchKernelGGL(gn_bwd_weight_kernel, dim3((unsigned)ceil_div(p.c, kBlock)), block, 0, a.stream, (const float2*)totals,
                           a.gw, a.gb, (int)a.n, p.c);
    if (a.out)
        hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, V, ACT, KEPT>), grid, block, 0, a.stream, (const T*)a.gy, (const T*)a.x,
                           (const int8_t*)a.codes, (const uint8_t*)a.scales, (const float*)a.mean, (const float*)a.rstd, a.weight,
                           a.bias, (const float2*)means, (T*)a.out, a.slope, a.scale, p);
    return check_launch("sae_group_norm_act_bwd");
}

template <int DT, int V, bool KEPT>
int gn_backward(const GnArgs& a, const GnShape& p) {
    if (a.act == SAE_ACT_LRELU) return gn_backward_as<DT, V, SAE_ACT_LRELU, KEPT>(a, p);
    if (a.act == SAE_ACT_SILU) return gn_backward_as<DT, V, SAE_ACT_SILU, KEPT>(a, p);
    return gn_backward_as<DT, V, SAE_ACT_NONE, KEPT>(a, p);
}

// V channels per lane in 16-byte accesses where the rows allow it, one channel where not
bool gn_vector(int64_t c, int32_t dtype) { return c % (16 / elem_bytes(dtype)) == 0; }

template <int DT>
int gn_run(const GnArgs& a, const GnShape& p, bool vec, bool backward) {
    if (!backward) return vec ? gn_forward<DT, Elem<DT>::kVec>(a, p) : gn_forward<DT, 1>(a, p);
    if (a.codes) return vec ? gn_backward<DT, Elem<DT>::kVec, true>(a, p) : gn_backward<DT, 1, true>(a, p);
    return vec ? gn_backward<DT, Elem<DT>::kVec, false>(a, p) : gn_backward<DT, 1, false>(a, p);
}

int gn_dispatch(const char* what, GnArgs& a, int64_t l, int64_t c, int64_t groups, int32_t dtype, int64_t ws_bytes, bool backward) {
    const bool vec = gn_vector(c, dtype);
    const GnShape p = gn_plan(a.n, l, c, groups, vec ? 16 / elem_bytes(dtype) : 1);
    const int64_t need = gn_workspace(p, a.n, backward);
    if (!a.ws || ws_bytes < need)
        return fail(SAE_EWORKSPACE, "%s: workspace %lld < %lld bytes (sae_group_norm_act_workspace)", what, (long long)ws_bytes,
                    (long long)need);
    for (const void* t : {a.gy, a.x, (const void*)a.out, (const void*)a.ws, (const void*)a.codes})
        if (!aligned16(t)) return fail(SAE_EINVAL, "%s: tensors must be 16-byte aligned", what);
    if (dtype == SAE_F32) return gn_run<SAE_F32>(a, p, vec, backward);
    if (dtype == SAE_BF16) return gn_run<SAE_BF16>(a, p, vec, backward);
    return gn_run<SAE_F16>(a, p, vec, backward);
}

}  // namespace
}  // namespace sae

using namespace sae;

extern "C" int64_t sae_group_norm_act_workspace(int64_t n, int64_t l, int64_t c, int64_t groups, int32_t dtype, int32_t backward) {
    if (!gn_shape_ok(n, l, c, groups) || !elem_known(dtype) || n == 0 || l == 0) return 0;
    return gn_workspace(gn_plan(n, l, c, groups, gn_vector(c, dtype) ? 16 / elem_bytes(dtype) : 1), n, backward != 0);
}

extern "C" int sae_group_norm_act(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                                  int8_t* codes, uint8_t* scales, int64_t n, int64_t l, int64_t c, int64_t groups, float eps,
                                  int32_t act, float slope, float scale, int32_t dtype, void* workspace, int64_t workspace_bytes,
                                  sae_stream_t stream) {
    sae::clear_stale_error();
    if (!elem_known(dtype) || act < SAE_ACT_NONE || act > SAE_ACT_SILU)
        return fail(SAE_EINVAL, "sae_group_norm_act: unknown element type or activation");
    if (!gn_shape_ok(n, l, c, groups) || !(eps >= 0.0f)) return fail(SAE_EINVAL, "sae_group_norm_act: bad shape or eps");
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
    if (!gn_shape_ok(n, l, c, groups)) return fail(SAE_EINVAL, "sae_group_norm_act_bwd: bad shape");
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
