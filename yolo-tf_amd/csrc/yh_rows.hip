// Row operators bound by memory: row codes (write and read) and batch normalisation with leaky ReLU on an 8-bit
// checkpoint, forward and backward.
#include <algorithm>
#include "yh_rows.h"

namespace yh {
namespace {

constexpr int kThreads = 256;

// How a wavefront holds rows in registers: `lanes` neighbouring lanes a row, each with `vecs` vectors of V elements,
// `lanes` vectors apart.  `most` vectors a lane (four: 4 KiB of loads in flight a wavefront); rows shorter than that share
// the wavefront, with at least eight lanes (128 contiguous bytes) each.  Below 2^20 lanes in all (64 wavefronts a compute
// unit) more lanes a row fill the card better: normalisation of 10816 x 512 in float32 29.3 us with four vectors a lane, 26.8
// with two; of 173056 x 128, with lanes enough, 57.8 and 60.2.
struct RowPlan { int lanes, vecs; };
RowPlan plan_row(int64_t rows, int cols, int V, int most)
{
    const int nv = (cols + V - 1) / V, all = std::min(64, pow2_at_least(nv));
    RowPlan p;
    p.lanes = std::min(64, std::max(std::min(8, pow2_at_least(nv)), pow2_at_least((nv + most - 1) / most)));
    while (p.lanes < all && rows * p.lanes < 1 << 20) p.lanes *= 2;
    p.vecs = (nv + p.lanes - 1) / p.lanes;
    return p;
}

// Row codes, written: one read of x, one write of the codes; the row waits in registers for its maximum (lanes of a row
// exchange it by data-parallel moves).  Bound by memory: 173056 x 128 in float32 20 us (112 MB, 5.6 TB/s), 43264 x 1536 in
// bfloat16 37.6 us (5.3 TB/s; 43 where the launch before still writes).
template <class T, int IT>
__global__ __launch_bounds__(kThreads) void k_quantize(const T *x, int64_t rows, int cols, int64_t ldx, int8_t *codes, int64_t ldc,
                                                       float *scale, int lanes, int64_t spare)
{
    constexpr int V = RowVec<T>::V;
    const int lane = threadIdx.x & 63, sub = lane & (lanes - 1);
    const int64_t wave = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    const int64_t row = wave * (64 / lanes) + lane / lanes;
    const int read = left_of(row, rows, spare, cols, 0, V);
    float v[IT][V];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * lanes + sub) * V;
        load_vec<T, V>(v[i], x + row * ldx + c, read - c);
    }
    if (cols % V)
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if ((i * lanes + sub) * V + j >= cols) v[i][j] = 0.0f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) m = max(m, __float_as_uint(v[i][j]) & 0x7fffffffu);
    const RowScale k = row_scale(row_max(m, lanes), (float)kCodeMax);
    if (row >= rows) return;
    if (sub == 0) scale[row] = k.s;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * lanes + sub) * V;
        uint32_t w[V / 4];
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const uint32_t q = pack4(code_bits(v[i][j], k.r), code_bits(v[i][j + 1], k.r), code_bits(v[i][j + 2], k.r), code_bits(v[i][j + 3], k.r));
            w[j / 4] = k.live ? q : 0u;
        }
        store_bytes<V>(codes + row * ldc + c, w, cols - c);
    }
}

// The largest of a workgroup's values; `top`: one word a wavefront, free again when the call returns everywhere.
__device__ __forceinline__ uint32_t workgroup_max(uint32_t m, uint32_t *top)
{
    m = row_max(m, 64);
    __syncthreads();                                 // the last call's words have been read
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) m = max(m, top[i]);
    return m;
}

// Rows longer than the registers of a wavefront (eight vectors a lane: 20000 x 2048 in float32 35 us so, 41 us here): a
// workgroup a row, read twice (the second time from the caches).
template <class T>
__global__ __launch_bounds__(kThreads) void k_quantize_long(const T *x, int64_t rows, int cols, int64_t ldx, int8_t *codes, int64_t ldc, float *scale)
{
    constexpr int V = RowVec<T>::V;
    __shared__ uint32_t top[kThreads / 64];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *p = x + row * ldx;
        uint32_t m = 0;
        for (int c = threadIdx.x * V; c < cols; c += kThreads * V) {
            float v[V];
            load_vec<T, V>(v, p + c, cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
        }
        m = workgroup_max(m, top);
        const RowScale k = row_scale(m, (float)kCodeMax);
        if (threadIdx.x == 0) scale[row] = k.s;
        for (int c = threadIdx.x * V; c < cols; c += kThreads * V) {
            float v[V];
            load_vec<T, V>(v, p + c, cols - c);
            uint32_t w[V / 4];
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const uint32_t q = pack4(code_bits(v[j], k.r), code_bits(v[j + 1], k.r), code_bits(v[j + 2], k.r), code_bits(v[j + 3], k.r));
                w[j / 4] = k.live ? q : 0u;
            }
            store_bytes<V>(codes + row * ldc + c, w, cols - c);
        }
    }
}

// Row codes, read: 173056 x 128 to float32 18.6 us (111 MB, 6.0 TB/s), 43264 x 1536 to bfloat16 30.2 us (200 MB, 6.6 TB/s).
template <class T, int IT>
__global__ __launch_bounds__(kThreads) void k_dequantize(const int8_t *codes, int64_t ldc, const float *scale, int64_t rows, int cols,
                                                         T *out, int64_t ldo, int lanes, int64_t spare)
{
    constexpr int V = RowVec<T>::V;
    const int lane = threadIdx.x & 63, sub = lane & (lanes - 1);
    const int64_t wave = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    const int64_t row = wave * (64 / lanes) + lane / lanes;
    if (row >= rows) return;
    const float s = scale[row];
    const int read = left_of(row, rows, spare, cols, 0, V);
    for (int base = 0; base < cols; base += IT * lanes * V) {
        uint32_t w[IT][V / 4];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = base + (i * lanes + sub) * V;
            load_bytes<V>(w[i], codes + row * ldc + c, read - c);
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = base + (i * lanes + sub) * V;
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = code_value(w[i][j / 4], j % 4) * s;
            store_vec<T, V>(out + row * ldo + c, v, cols - c);
        }
    }
}

// ---- batch normalisation + leaky ReLU (+ shortcut) on an 8-bit checkpoint ----
// Forward, per channel c over all rows:  mean = sum z / M, var = sum (z - mean)^2 / M, both in 64 bits (the differences to
// the channel's first value are exact there, so neither a large mean nor many rows cost anything), then rounded once:
// mean, invstd = 1 / sqrt(var + eps) in float32.  Per element in float32, each operation rounded by itself:
//   xhat = (z - mean) * invstd,  u = xhat * gamma + beta,  a = (u > 0 ? u : slope * u) [+ residual].
// The checkpoint is one byte an element: the sign of u in the lowest bit, exactly as the forward pass decided it, and
// xhat in seven bits above it, relative to the row's largest |xhat| / 63.  The backward pass needs the sign for every
// element's gradient and xhat only for a sum over the rows (dgamma) and for that sum's small share of each element, where
// the rounding of the code averages out; eight bits for xhat and the sign taken from them would be off on the elements
// next to zero.
// Backward:  du = sign ? da : slope * da,  dbeta = sum du,  dgamma = sum du * xq,
//            dz = gamma * invstd * (du - dbeta / M - xq * dgamma / M).
// Both directions read their input twice, with the per-channel sums in between: a reduction into one partial pair a
// workgroup and channel, a small launch that adds the partials in a fixed order, and an elementwise pass.

// A workgroup's threads over (channel vectors, rows) in the reductions.
struct ReducePlan { int tx, ty, slabs, blocks; };
ReducePlan plan_reduce(int64_t rows, int cols, int V)
{
    const int cv = (cols + V - 1) / V;
    ReducePlan p;
    // Up to 1024 rows one workgroup takes all rows of a slab of four vectors (64 bytes a row) and finishes by itself: the
    // launch that adds the partials costs more than what the spread over workgroups wins (forward pass,
    // 169 x 1024 in bfloat16: 9.7 us so, 12.0 with it; 1024 x 1024: 10.7 and 12.8; 4096 x 1024: 25.1 and 22.6).
    const bool alone = rows <= 1024;
    p.tx = std::min(alone ? 4 : 64, pow2_at_least(cv));
    p.ty = kThreads / p.tx;
    p.slabs = (cv + p.tx - 1) / p.tx;
    if (alone) {
        p.blocks = 1;
        return p;
    }
    // about 1024 workgroups in all (four a compute unit), each thread with at least eight rows
    const int64_t by_rows = (rows + p.ty * 8 - 1) / ((int64_t)p.ty * 8);
    const int64_t want = std::max(1, 1024 / p.slabs);
    p.blocks = (int)std::max<int64_t>(1, std::min(want, by_rows));
    return p;
}

// Adds the threads' pairs over ty: first over the lanes of a wavefront that hold the same channels, then over the four
// wavefronts through LDS, a thread a channel.  Where there is more than one workgroup its pair goes to
// part[2][cols][blocks], otherwise to out.finish(channel, sum, sum).
template <int V, class Out>
__device__ __forceinline__ void reduce_pairs(double (&s1)[V], double (&s2)[V], int TX, int cols, double *part, const Out &out)
{
    constexpr int W = kThreads / 64;
    __shared__ double buf[2 * V][W][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int o = TX; o < 64; o <<= 1)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s1[j] += __shfl_xor(s1[j], o);
            s2[j] += __shfl_xor(s2[j], o);
        }
    if (lane < TX)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            buf[2 * j][wave][lane] = s1[j];
            buf[2 * j + 1][wave][lane] = s2[j];
        }
    __syncthreads();
    for (int t = threadIdx.x; t < TX * V; t += kThreads) {
        const int c = blockIdx.y * TX * V + t, x = t / V, j = t % V;
        if (c >= cols) continue;
        const double a = (buf[2 * j][0][x] + buf[2 * j][1][x]) + (buf[2 * j][2][x] + buf[2 * j][3][x]);
        const double b = (buf[2 * j + 1][0][x] + buf[2 * j + 1][1][x]) + (buf[2 * j + 1][2][x] + buf[2 * j + 1][3][x]);
        if (gridDim.x > 1) {
            part[(int64_t)c * gridDim.x + blockIdx.x] = a;
            part[((int64_t)cols + c) * gridDim.x + blockIdx.x] = b;
        } else {
            out.finish(c, a, b);
        }
    }
}

// What follows from a channel's sums of (z - first) and of its square.
template <class T>
struct NormStats {
    const T *first;                                      // z's first row
    int64_t rows;
    double eps, momentum;
    float *mean, *invstd, *running_mean, *running_var;
    __device__ __forceinline__ void finish(int c, double s1, double s2) const
    {
        const double m = (double)rows, d = s1 / m, mu = (double)(float)first[c] + d;
        double var = s2 / m - d * d;
        if (var < 0.0) var = 0.0;                        // a NaN stays one
        mean[c] = (float)mu;
        invstd[c] = (float)(1.0 / sqrt(var + eps));
        if (running_mean) {
            running_mean[c] = (float)((1.0 - momentum) * (double)running_mean[c] + momentum * mu);
            running_var[c] = (float)((1.0 - momentum) * (double)running_var[c] + momentum * (rows > 1 ? var * (m / (m - 1.0)) : var));
        }
    }
};

struct NormGrads {
    float *dgamma, *dbeta;
    __device__ __forceinline__ void finish(int c, double b, double g) const
    {
        dbeta[c] = (float)b;
        dgamma[c] = (float)g;
    }
};

// NormGrads, and a workgroup's own channels, from `first` on, in LDS.
struct NormGradsHere {
    NormGrads out;
    float *b_here, *g_here;
    int first;
    __device__ __forceinline__ void finish(int c, double b, double g) const
    {
        out.finish(c, b, g);
        b_here[c - first] = (float)b;
        g_here[c - first] = (float)g;
    }
};

// Statistics: one read of z.  346112 x 128 in float32 (177 MB): 46 us (3.9 TB/s), the adding of the partials 5 us; sums
// in float32, loads one round ahead, half or twice the workgroups: 44 to 49 us.
template <class T>
__global__ __launch_bounds__(kThreads) void k_norm_stats(const T *z, int64_t rows, int cols, int64_t ldz, int64_t spare, int TX, double *part,
                                                         NormStats<T> out)
{
    constexpr int V = RowVec<T>::V, U = 4;
    const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x / TX, TY = kThreads / TX;
    const int cvec = blockIdx.y * TX + tx, c = cvec * V, left = cols - c;
    double s1[V], s2[V];
    float first[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0;
    load_vec<T, V>(first, z + c, left);
    const int64_t step = (int64_t)gridDim.x * U * TY, rows_whole = left >= V ? rows : spare;
    const T *p = z + c;
    const auto add = [&](const float (&v)[V]) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const double d = (double)v[j] - (double)first[j];
            s1[j] += d;
            s2[j] = __builtin_fma(d, d, s2[j]);
        }
    };
    int64_t r = (int64_t)blockIdx.x * U * TY + ty;
    if (left > 0)                                    // whole vectors, whole groups of rows: nothing to ask in the loop
        for (; r + (U - 1) * TY < rows_whole; r += step) {
            float v[U][V];
#pragma unroll
            for (int i = 0; i < U; ++i) load_vec<T, V>(v[i], p + (r + i * TY) * ldz, V);
#pragma unroll
            for (int i = 0; i < U; ++i) add(v[i]);
        }
    for (; left > 0 && r < rows; r += step) {        // rows past the end are read as the last one and left out
        float v[U][V];
#pragma unroll
        for (int i = 0; i < U; ++i) load_vec<T, V>(v[i], p + min(r + i * TY, rows - 1) * ldz, left);
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (r + i * TY < rows) add(v[i]);
    }
    reduce_pairs<V>(s1, s2, TX, cols, part, out);
}

// A channel's pair of sums over its partials, by `lanes` threads (64: a wavefront, or 256: the workgroup; few partials
// take the wavefront) in a fixed order, whatever ran first.  Whole in the thread with at == 0.
__device__ __forceinline__ void sum_partials(const double *p, const double *q, int blocks, int at, int lanes, double &s1, double &s2)
{
    __shared__ double buf[2][kThreads / 64];
    s1 = s2 = 0.0;
#pragma unroll 4
    for (int i = at; i < blocks; i += lanes) {
        s1 += p[i];
        s2 += q[i];
    }
    for (int o = 1; o < 64; o <<= 1) {
        s1 += __shfl_xor(s1, o);
        s2 += __shfl_xor(s2, o);
    }
    if (lanes == 64) return;
    if ((at & 63) == 0) {
        buf[0][at >> 6] = s1;
        buf[1][at >> 6] = s2;
    }
    __syncthreads();
    if (at == 0)
        for (int i = 1; i < kThreads / 64; ++i) {
            s1 += buf[0][i];
            s2 += buf[1][i];
        }
}

template <class T>
__global__ __launch_bounds__(kThreads) void k_norm_stats_finish(const double *part, int blocks, int cols, int lanes, NormStats<T> out)
{
    const int per = kThreads / lanes, c = min((int)blockIdx.x * per + (int)threadIdx.x / lanes, cols - 1), at = threadIdx.x & (lanes - 1);
    double s1, s2;
    sum_partials(part + (int64_t)c * blocks, part + ((int64_t)cols + c) * blocks, blocks, at, lanes, s1, s2);
    if (at == 0 && (int)blockIdx.x * per + (int)threadIdx.x / lanes < cols) out.finish(c, s1, s2);
}

// The elementwise pass: z (and the shortcut) in, the activation and the checkpoint out, a row's maximum between its lanes.
// Bound by memory: 346112 x 128 in float32 with a shortcut 98 us (577 MB, 5.9 TB/s).
template <class T, int IT>
__global__ __launch_bounds__(kThreads) void k_norm_apply(const T *z, int64_t ldz, const T *res, int64_t ldr, int64_t rows, int cols,
                                                         const float *mean, const float *invstd, const float *gamma, const float *beta, float slope,
                                                         T *a, int64_t lda, int8_t *kept, int64_t ldk, float *scale, int64_t spare, int lanes, int64_t waves)
{
    constexpr int V = RowVec<T>::V;
    const int lane = threadIdx.x & 63, sub = lane & (lanes - 1), rpw = 64 / lanes;
    float mu[IT][V], is[IT][V], ga[IT][V], be[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * lanes + sub) * V;
        load_vec<float, V>(mu[i], mean + c, cols - c);
        load_vec<float, V>(is[i], invstd + c, cols - c);
        load_vec<float, V>(ga[i], gamma + c, cols - c);
        load_vec<float, V>(be[i], beta + c, cols - c);
    }
    // every lane of a wavefront takes part in the row maximum: the loop's bound is the wavefront's first row
    for (int64_t g = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); g * rpw < rows; g += waves) {
        const int64_t row = g * rpw + lane / lanes;
        const bool in = row < rows;
        const int read = left_of(row, rows, spare, cols, 0, V);
        float v[IT][V], rs[IT][V];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * lanes + sub) * V;
            load_vec<T, V>(v[i], z + row * ldz + c, read - c);
            if (res) load_vec<T, V>(rs[i], res + row * ldr + c, read - c);
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = (i * lanes + sub) * V + j;
                v[i][j] = (v[i][j] - mu[i][j]) * is[i][j];
                if (c < cols) m = max(m, __float_as_uint(v[i][j]) & 0x7fffffffu);
            }
        const RowScale k = row_scale(row_max(m, lanes), (float)kKeptMax);
        if (!in) continue;
        if (kept && sub == 0) scale[row] = k.s;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * lanes + sub) * V;
            uint32_t w[V / 4], b[V];
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float u = v[i][j] * ga[i][j] + be[i][j];
                const bool up = u > 0.0f;
                o[j] = up ? u : slope * u;
                if (res) o[j] += rs[i][j];
                const uint32_t q = k.live ? code_bits(v[i][j], k.r) : 0u;
                b[j] = (q << 1) | (up ? 1u : 0u);
            }
            store_vec<T, V>(a + row * lda + c, o, cols - c);
            if (kept) {
#pragma unroll
                for (int j = 0; j < V; j += 4) w[j / 4] = pack4(b[j], b[j + 1], b[j + 2], b[j + 3]);
                store_bytes<V>(kept + row * ldk + c, w, cols - c);
            }
        }
    }
}

// Rows over the whole workgroup, R at a time; the wavefronts exchange their maxima through LDS, in two sets of words in
// turn, so that one barrier a turn is enough.
template <class T, int IT, int R>
__global__ __launch_bounds__(kThreads) void k_norm_apply_wide(const T *z, int64_t ldz, const T *res, int64_t ldr, int64_t rows, int cols,
                                                              const float *mean, const float *invstd, const float *gamma, const float *beta, float slope,
                                                              T *a, int64_t lda, int8_t *kept, int64_t ldk, float *scale, int64_t spare)
{
    constexpr int V = RowVec<T>::V;
    __shared__ uint32_t top[2][R][kThreads / 64];
    float mu[IT][V], is[IT][V], ga[IT][V], be[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * kThreads + threadIdx.x) * V;
        load_vec<float, V>(mu[i], mean + c, cols - c);
        load_vec<float, V>(is[i], invstd + c, cols - c);
        load_vec<float, V>(ga[i], gamma + c, cols - c);
        load_vec<float, V>(be[i], beta + c, cols - c);
    }
    int at = 0;
    for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < rows; row0 += (int64_t)gridDim.x * R, at ^= 1) {
        float v[R][IT][V], rs[R][IT][V];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int c = (i * kThreads + threadIdx.x) * V, left = left_of(row0 + r, rows, spare, cols, c, V);
                load_vec<T, V>(v[r][i], z + (row0 + r) * ldz + c, left);
                if (res) load_vec<T, V>(rs[r][i], res + (row0 + r) * ldr + c, left);
            }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[r][i][j] = (v[r][i][j] - mu[i][j]) * is[i][j];
                    if ((i * kThreads + (int)threadIdx.x) * V + j < cols) m = max(m, __float_as_uint(v[r][i][j]) & 0x7fffffffu);
                }
            m = row_max(m, 64);
            if ((threadIdx.x & 63) == 0) top[at][r][threadIdx.x >> 6] = m;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + r;
            if (row >= rows) break;
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 64; ++i) m = max(m, top[at][r][i]);
            const RowScale k = row_scale(m, (float)kKeptMax);
            if (kept && threadIdx.x == 0) scale[row] = k.s;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int c = (i * kThreads + threadIdx.x) * V;
                uint32_t w[V / 4], b[V];
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = v[r][i][j] * ga[i][j] + be[i][j];
                    const bool up = u > 0.0f;
                    o[j] = up ? u : slope * u;
                    if (res) o[j] += rs[r][i][j];
                    b[j] = ((k.live ? code_bits(v[r][i][j], k.r) : 0u) << 1) | (up ? 1u : 0u);
                }
                store_vec<T, V>(a + row * lda + c, o, cols - c);
                if (kept) {
#pragma unroll
                    for (int j = 0; j < V; j += 4) w[j / 4] = pack4(b[j], b[j + 1], b[j + 2], b[j + 3]);
                    store_bytes<V>(kept + row * ldk + c, w, cols - c);
                }
            }
        }
    }
}

// Rows of any length: a workgroup a row, read twice.
template <class T>
__global__ __launch_bounds__(kThreads) void k_norm_apply_long(const T *z, int64_t ldz, const T *res, int64_t ldr, int64_t rows, int cols,
                                                              const float *mean, const float *invstd, const float *gamma, const float *beta, float slope,
                                                              T *a, int64_t lda, int8_t *kept, int64_t ldk, float *scale)
{
    constexpr int V = RowVec<T>::V;
    __shared__ uint32_t top[kThreads / 64];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        uint32_t m = 0;
        for (int c = threadIdx.x * V; c < cols; c += kThreads * V) {
            float v[V], mu[V], is[V];
            load_vec<T, V>(v, z + row * ldz + c, cols - c);
            load_vec<float, V>(mu, mean + c, cols - c);
            load_vec<float, V>(is, invstd + c, cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < cols) m = max(m, __float_as_uint((v[j] - mu[j]) * is[j]) & 0x7fffffffu);
        }
        m = workgroup_max(m, top);
        const RowScale k = row_scale(m, (float)kKeptMax);
        if (kept && threadIdx.x == 0) scale[row] = k.s;
        for (int c = threadIdx.x * V; c < cols; c += kThreads * V) {
            float v[V], rs[V], mu[V], is[V], ga[V], be[V], o[V];
            uint32_t w[V / 4], b[V];
            load_vec<T, V>(v, z + row * ldz + c, cols - c);
            if (res) load_vec<T, V>(rs, res + row * ldr + c, cols - c);
            load_vec<float, V>(mu, mean + c, cols - c);
            load_vec<float, V>(is, invstd + c, cols - c);
            load_vec<float, V>(ga, gamma + c, cols - c);
            load_vec<float, V>(be, beta + c, cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (v[j] - mu[j]) * is[j], u = xh * ga[j] + be[j];
                const bool up = u > 0.0f;
                o[j] = up ? u : slope * u;
                if (res) o[j] += rs[j];
                b[j] = ((k.live ? code_bits(xh, k.r) : 0u) << 1) | (up ? 1u : 0u);
            }
            store_vec<T, V>(a + row * lda + c, o, cols - c);
            if (kept) {
#pragma unroll
                for (int j = 0; j < V; j += 4) w[j / 4] = pack4(b[j], b[j + 1], b[j + 2], b[j + 3]);
                store_bytes<V>(kept + row * ldk + c, w, cols - c);
            }
        }
    }
}

// The checkpoint's byte: xhat's code and the activation's side.
__device__ __forceinline__ float kept_code(uint32_t w, int i) { return (float)((int8_t)(w >> (8 * i)) >> 1); }
__device__ __forceinline__ bool kept_side(uint32_t w, int i) { return (w >> (8 * i)) & 1u; }

// da -> dz, from a row's bytes and scale and the channels' factors.
template <int V>
__device__ __forceinline__ void input_grads(float (&v)[V], const uint32_t (&w)[V / 4], float s, float slope, const float (&g)[V],
                                            const float (&cb)[V], const float (&cg)[V])
{
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float du = kept_side(w[j / 4], j % 4) ? v[j] : slope * v[j];
        const float xq = kept_code(w[j / 4], j % 4) * s;
        v[j] = g[j] * (du - cb[j] - xq * cg[j]);
    }
}

// Sums of the backward pass: da and the checkpoint in.  346112 x 128 in float32 (223 MB): 57 us (3.9 TB/s).
template <class T>
__global__ __launch_bounds__(kThreads) void k_norm_grad_sums(const T *da, int64_t ldd, const int8_t *kept, int64_t ldk, const float *scale,
                                                             int64_t rows, int cols, float slope, int64_t spare, int TX, double *part,
                                                             NormGrads out)
{
    constexpr int V = RowVec<T>::V, U = 4;
    const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x / TX, TY = kThreads / TX;
    const int cvec = blockIdx.y * TX + tx, c = cvec * V, left = cols - c;
    double s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0;
    const int64_t step = (int64_t)gridDim.x * U * TY, rows_whole = left >= V ? rows : spare;
    const auto add = [&](const float (&v)[V], const uint32_t (&w)[V / 4], float s) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float du = kept_side(w[j / 4], j % 4) ? v[j] : slope * v[j];
            const float xq = kept_code(w[j / 4], j % 4) * s;
            s1[j] += (double)du;
            s2[j] = __builtin_fma((double)du, (double)xq, s2[j]);
        }
    };
    int64_t r = (int64_t)blockIdx.x * U * TY + ty;
    if (left > 0)
        for (; r + (U - 1) * TY < rows_whole; r += step) {
            float v[U][V], s[U];
            uint32_t w[U][V / 4];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int64_t rr = r + i * TY;
                load_vec<T, V>(v[i], da + rr * ldd + c, V);
                load_bytes<V>(w[i], kept + rr * ldk + c, V);
                s[i] = scale[rr];
            }
#pragma unroll
            for (int i = 0; i < U; ++i) add(v[i], w[i], s[i]);
        }
    for (; left > 0 && r < rows; r += step) {
        float v[U][V], s[U];
        uint32_t w[U][V / 4];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t rr = min(r + i * TY, rows - 1);
            load_vec<T, V>(v[i], da + rr * ldd + c, left);
            load_bytes<V>(w[i], kept + rr * ldk + c, left);
            s[i] = scale[rr];
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (r + i * TY < rows) add(v[i], w[i], s[i]);
    }
    reduce_pairs<V>(s1, s2, TX, cols, part, out);
}

// The whole backward pass for few rows: a workgroup holds its channels' rows, U a thread, and gives both the sums and the
// input gradients.  169 x 1024 in bfloat16: 6.6 us, 9.3 in two launches; 512 x 1024: 8.6 and
// 10.1.
template <class T, int U>
__global__ __launch_bounds__(kThreads) void k_norm_grad_few(const T *da, int64_t ldd, const int8_t *kept, int64_t ldk, const float *scale,
                                                            int64_t rows, int cols, float slope, int64_t spare, int TX, const float *gamma,
                                                            const float *invstd, float *dgamma, float *dbeta, T *dz, int64_t ldz)
{
    constexpr int V = RowVec<T>::V;
    __shared__ float sums[2][4 * V];
    const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x / TX, TY = kThreads / TX;
    const int c = (blockIdx.y * TX + tx) * V;
    float v[U][V], s[U], g[V], is[V], cb[V], cg[V];
    uint32_t w[U][V / 4];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t row = ty + i * TY;
        const int read = left_of(row, rows, spare, cols, c, V);
        load_vec<T, V>(v[i], da + row * ldd + c, read);
        load_bytes<V>(w[i], kept + row * ldk + c, read);
        s[i] = row < rows ? scale[row] : 0.0f;
    }
    load_vec<float, V>(g, gamma + c, cols - c);
    load_vec<float, V>(is, invstd + c, cols - c);
    double s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        s1[j] = s2[j] = 0.0;
#pragma unroll
        for (int i = 0; i < U; ++i) {                // rows past the end are zeros
            const float du = kept_side(w[i][j / 4], j % 4) ? v[i][j] : slope * v[i][j];
            const float xq = kept_code(w[i][j / 4], j % 4) * s[i];
            s1[j] += (double)du;
            s2[j] = __builtin_fma((double)du, (double)xq, s2[j]);
        }
    }
    reduce_pairs<V>(s1, s2, TX, cols, nullptr, NormGradsHere{{dgamma, dbeta}, sums[0], sums[1], (int)blockIdx.y * TX * V});
    __syncthreads();
    const float per_row = 1.0f / (float)rows;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        g[j] *= is[j];
        cb[j] = sums[0][tx * V + j] * per_row;
        cg[j] = sums[1][tx * V + j] * per_row;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t row = ty + i * TY;
        input_grads<V>(v[i], w[i], s[i], slope, g, cb, cg);
        if (row < rows) store_vec<T, V>(dz + row * ldz + c, v[i], cols - c);
    }
}

__global__ __launch_bounds__(kThreads) void k_norm_grad_finish(const double *part, int blocks, int cols, int lanes, NormGrads out)
{
    const int per = kThreads / lanes, c = min((int)blockIdx.x * per + (int)threadIdx.x / lanes, cols - 1), at = threadIdx.x & (lanes - 1);
    double b, g;
    sum_partials(part + (int64_t)c * blocks, part + ((int64_t)cols + c) * blocks, blocks, at, lanes, b, g);
    if (at == 0 && (int)blockIdx.x * per + (int)threadIdx.x / lanes < cols) out.finish(c, b, g);
}

// Input gradient: da and the checkpoint again, dz out.  346112 x 128 in float32 (400 MB): 68 us (5.9 TB/s).
template <class T, int IT>
__global__ __launch_bounds__(kThreads) void k_norm_grad_apply(const T *da, int64_t ldd, const int8_t *kept, int64_t ldk, const float *scale,
                                                              int64_t rows, int cols, float slope, const float *gamma, const float *invstd,
                                                              const float *dgamma, const float *dbeta, T *dz, int64_t ldz, int64_t spare, int lanes, int64_t waves)
{
    constexpr int V = RowVec<T>::V;
    const int lane = threadIdx.x & 63, sub = lane & (lanes - 1), rpw = 64 / lanes;
    const int c0 = blockIdx.y * IT * lanes * V;
    const float per_row = 1.0f / (float)rows;
    float g[IT][V], cb[IT][V], cg[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = c0 + (i * lanes + sub) * V;
        float is[V];
        load_vec<float, V>(g[i], gamma + c, cols - c);
        load_vec<float, V>(is, invstd + c, cols - c);
        load_vec<float, V>(cb[i], dbeta + c, cols - c);
        load_vec<float, V>(cg[i], dgamma + c, cols - c);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            g[i][j] *= is[j];
            cb[i][j] *= per_row;
            cg[i][j] *= per_row;
        }
    }
    for (int64_t w0 = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); w0 * rpw < rows; w0 += waves) {
        const int64_t row = w0 * rpw + lane / lanes;
        if (row >= rows) continue;
        const int read = left_of(row, rows, spare, cols, 0, V);
        float v[IT][V];
        uint32_t w[IT][V / 4];
        const float s = scale[row];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = c0 + (i * lanes + sub) * V;
            load_vec<T, V>(v[i], da + row * ldd + c, read - c);
            load_bytes<V>(w[i], kept + row * ldk + c, read - c);
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = c0 + (i * lanes + sub) * V;
            input_grads<V>(v[i], w[i], s, slope, g[i], cb[i], cg[i]);
            store_vec<T, V>(dz + row * ldz + c, v[i], cols - c);
        }
    }
}

// The kernels' vector counts.
#define YH_WITH_VECS(vecs, CALL)            \
    do {                                    \
        if ((vecs) <= 1) { CALL(1); }       \
        else if ((vecs) <= 2) { CALL(2); }  \
        else if ((vecs) <= 4) { CALL(4); }  \
        else { CALL(8); }                   \
    } while (0)

unsigned row_blocks(int64_t rows) { return (unsigned)std::min<int64_t>(rows, 1 << 20); }
unsigned waves_to_blocks(int64_t waves) { return (unsigned)((waves + kThreads / 64 - 1) / (kThreads / 64)); }

}  // namespace

hipError_t launch_quantize(const Rows &x, int64_t rows, int32_t cols, int8_t *codes, int64_t ldc, float *scale, hipStream_t st)
{
    with_type(x.type, [&](auto t) {
        using T = decltype(t);
        const T *p = static_cast<const T *>(x.p);
        const RowPlan r = plan_row(rows, cols, RowVec<T>::V, 4);
        if (r.vecs > 8) {
            k_quantize_long<T><<<dim3(row_blocks(rows)), kThreads, 0, st>>>(p, rows, cols, x.ld, codes, ldc, scale);
            return;
        }
        const unsigned blocks = waves_to_blocks((rows * r.lanes + 63) / 64);
#define CALL(IT) k_quantize<T, IT><<<dim3(blocks), kThreads, 0, st>>>(p, rows, cols, x.ld, codes, ldc, scale, r.lanes, spare_rows(rows, x.ld, RowVec<T>::V))
        YH_WITH_VECS(r.vecs, CALL);
#undef CALL
    });
    return hipGetLastError();
}

hipError_t launch_dequantize(const int8_t *codes, int64_t ldc, const float *scale, int64_t rows, int32_t cols,
                             void *out, int64_t ldo, int32_t type, hipStream_t st)
{
    with_type(type, [&](auto t) {
        using T = decltype(t);
        const RowPlan r = plan_row(rows, cols, RowVec<T>::V, 4);
        const unsigned blocks = waves_to_blocks((rows * r.lanes + 63) / 64);
#define CALL(IT) k_dequantize<T, IT><<<dim3(blocks), kThreads, 0, st>>>(codes, ldc, scale, rows, cols, static_cast<T *>(out), ldo, r.lanes, spare_rows(rows, ldc, RowVec<T>::V))
        YH_WITH_VECS(r.vecs, CALL);
#undef CALL
    });
    return hipGetLastError();
}

int norm_blocks(int64_t rows, int32_t cols, int32_t type)
{
    return plan_reduce(rows, cols, type == YH_FLOAT32 ? RowVec<float>::V : RowVec<__bf16>::V).blocks;
}

hipError_t launch_norm_forward(const Rows &z, const Rows &res, int64_t rows, int32_t cols, const float *gamma, const float *beta,
                               double eps, float slope, void *a, int64_t lda, int8_t *kept, int64_t ldk, float *scale,
                               float *mean, float *invstd, float *running_mean, float *running_var, double momentum,
                               void *workspace, hipStream_t st)
{
    double *part = static_cast<double *>(workspace);
    with_type(z.type, [&](auto t) {
        using T = decltype(t);
        const T *p = static_cast<const T *>(z.p), *q = static_cast<const T *>(res.p);
        const ReducePlan d = plan_reduce(rows, cols, RowVec<T>::V);
        const NormStats<T> out{p, rows, eps, momentum, mean, invstd, running_mean, running_var};
        k_norm_stats<T><<<dim3(d.blocks, d.slabs), kThreads, 0, st>>>(p, rows, cols, z.ld, spare_rows(rows, z.ld, RowVec<T>::V), d.tx, part, out);
        const int lanes = d.blocks > 64 ? kThreads : 64;
        if (d.blocks > 1)
            k_norm_stats_finish<T><<<dim3((cols * lanes + kThreads - 1) / kThreads), kThreads, 0, st>>>(part, d.blocks, cols, lanes, out);
        // Per channel four numbers stay in registers, so a lane holds at most 16 channels and beyond a wavefront's 1024 the
        // workgroup takes the row (20000 x 2048 in float32: 138 us in all, 171 by the kernel for any length; 20000 x 1536 in
        // bfloat16 77 us, 101 with 24 channels a lane).  With 16-bit vectors one a lane is best where lanes are enough
        // (173056 x 256 with a shortcut: 94 us, two: 104, four: 121), with float32 four.
        constexpr int V = RowVec<T>::V, kMost = 16 / V, kLane = V == 4 ? 4 : 1, R = 2;
        const int64_t spare = std::min(spare_rows(rows, z.ld, V), q ? spare_rows(rows, res.ld, V) : rows);
        const RowPlan r = plan_row(rows, cols, V, kLane);
        if (cols > kThreads * 16) {
            k_norm_apply_long<T><<<dim3(row_blocks(rows)), kThreads, 0, st>>>(p, z.ld, q, res.ld, rows, cols, mean, invstd, gamma, beta, slope,
                                                                            static_cast<T *>(a), lda, kept, ldk, scale);
            return;
        }
        if (r.vecs > kMost) {
            const int per = (cols + kThreads * V - 1) / (kThreads * V);
            const unsigned blocks = (unsigned)std::min<int64_t>(2048, (rows + R - 1) / R);
#define CALL(IT) k_norm_apply_wide<T, IT, R><<<dim3(blocks), kThreads, 0, st>>>(p, z.ld, q, res.ld, rows, cols, mean, invstd, gamma, beta, slope, \
                                                                               static_cast<T *>(a), lda, kept, ldk, scale, spare)
            if (per <= 1) CALL(1);
            else if (per <= 2) CALL(2);
            else if constexpr (kMost == 4) CALL(4);
#undef CALL
            return;
        }
        const unsigned blocks = std::min(2048u, waves_to_blocks((rows * r.lanes + 63) / 64));
#define CALL(IT) k_norm_apply<T, IT><<<dim3(blocks), kThreads, 0, st>>>(p, z.ld, q, res.ld, rows, cols, mean, invstd, gamma, beta, slope, \
                                                                        static_cast<T *>(a), lda, kept, ldk, scale, spare, r.lanes, (int64_t)blocks * (kThreads / 64))
        if (r.vecs <= 1) CALL(1);
        else if (r.vecs <= 2) CALL(2);
        else if constexpr (kMost == 4) CALL(4);
#undef CALL
    });
    return hipGetLastError();
}

hipError_t launch_norm_backward(const Rows &da, int64_t rows, int32_t cols, const int8_t *kept, int64_t ldk, const float *scale,
                                const float *gamma, const float *invstd, float slope, void *dz, int64_t lddz,
                                float *dgamma, float *dbeta, void *workspace, hipStream_t st)
{
    double *part = static_cast<double *>(workspace);
    with_type(da.type, [&](auto t) {
        using T = decltype(t);
        const T *p = static_cast<const T *>(da.p);
        const ReducePlan d = plan_reduce(rows, cols, RowVec<T>::V);
        const int64_t spare = std::min(spare_rows(rows, da.ld, RowVec<T>::V), spare_rows(rows, ldk, RowVec<T>::V));
        // up to eight rows a thread in registers, where four vectors a row and no more are one workgroup's
        if (d.tx <= 4 && rows <= 8 * d.ty) {
#define CALL(U) k_norm_grad_few<T, U><<<dim3(1, d.slabs), kThreads, 0, st>>>(p, da.ld, kept, ldk, scale, rows, cols, slope, spare, d.tx, gamma, \
                                                                            invstd, dgamma, dbeta, static_cast<T *>(dz), lddz)
            if (rows <= 4 * d.ty) CALL(4);
            else CALL(8);
#undef CALL
            return;
        }
        const NormGrads out{dgamma, dbeta};
        k_norm_grad_sums<T><<<dim3(d.blocks, d.slabs), kThreads, 0, st>>>(p, da.ld, kept, ldk, scale, rows, cols, slope, spare, d.tx, part, out);
        const int lanes = d.blocks > 64 ? kThreads : 64;
        if (d.blocks > 1)
            k_norm_grad_finish<<<dim3((cols * lanes + kThreads - 1) / kThreads), kThreads, 0, st>>>(part, d.blocks, cols, lanes, out);
        // the forward pass's lanes; 16 channels at most, further ones in workgroups of their own
        constexpr int V = RowVec<T>::V, kMost = 16 / V, kLane = V == 4 ? 4 : 1;
        const RowPlan r = plan_row(rows, cols, V, kLane);
        const int vecs = std::min(kMost, r.vecs), step = (vecs <= 1 ? 1 : vecs <= 2 ? 2 : 4) * r.lanes * V;
        const unsigned blocks = std::min(2048u, waves_to_blocks((rows * r.lanes + 63) / 64));
#define CALL(IT) k_norm_grad_apply<T, IT><<<dim3(blocks, (cols + step - 1) / step), kThreads, 0, st>>>( \
            p, da.ld, kept, ldk, scale, rows, cols, slope, gamma, invstd, dgamma, dbeta, static_cast<T *>(dz), lddz, spare, r.lanes, (int64_t)blocks * (kThreads / 64))
        if (vecs <= 1) CALL(1);
        else if (vecs <= 2) CALL(2);
        else if constexpr (kMost == 4) CALL(4);
#undef CALL
    });
    return hipGetLastError();
}

}  // namespace yh
