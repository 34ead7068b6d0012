// Products of row codes on the matrix cores: the integer product of a pointwise convolution, and its gradients, which
// multiply a float matrix by an integer one.
#include <algorithm>
#include "yh_rows.h"

namespace yh {
namespace {

constexpr int kThreads = 256;
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

// Workgroups with neighbouring tile numbers read the same rows; the hardware deals consecutive workgroups out to the 8
// XCDs in turn, each with an L2 of its own.  This gives each XCD a contiguous run of tile numbers.
__device__ __forceinline__ int64_t xcd_run(int64_t id, int64_t total)
{
    const int64_t per = total / 8, rest = total - per * 8, x = id & 7, i = id >> 3;
    return x * per + min(x, rest) + i;
}

// A 64-byte LDS row holds four 16-byte chunks; chunk c of row r sits at c ^ ((r >> 1) & 3), so that eight lanes that read
// (or write) one chunk each of eight neighbouring rows touch all 32 banks once.
__device__ __forceinline__ int chunk_at(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }

// ---- y = (codes . w codes^T) * scale * w_scale + bias ---------------------
// The sums are whole numbers in 32 bits (exact up to 65536 terms of 127^2); one product by each scale in float32 and one
// rounding to the output's type follow.  The weights are the matrix instruction's first operand: a lane then holds four
// neighbouring output channels of one row and stores them together.

__device__ __forceinline__ v4i load_chunk(const int8_t *p, int left)
{
    v4i v = {0, 0, 0, 0};
    if (left >= 16) {
        const LooseBytes<16>::type t = *reinterpret_cast<const LooseBytes<16>::type *>(p);
        __builtin_memcpy(&v, &t, 16);
    } else if (left > 0) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 15; ++i)
            if (i < left) w[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
        __builtin_memcpy(&v, w, 16);
    }
    return v;
}

template <int R>
struct CodeTile {
    static constexpr int N = (R * 4 + kThreads - 1) / kThreads;
    v4i v[N];
    __device__ __forceinline__ void load(const int8_t *p, int64_t ld, int64_t row0, int64_t rows, int k0, int k)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = threadIdx.x + i * kThreads, r = u >> 2, c = k0 + (u & 3) * 16;
            v[i] = load_chunk(p + (row0 + r) * ld + c, (R * 4 >= kThreads || u < R * 4) && row0 + r < rows ? k - c : 0);
        }
    }
    __device__ __forceinline__ void store(int8_t *lds) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = threadIdx.x + i * kThreads;
            if (R * 4 >= kThreads || u < R * 4) *reinterpret_cast<v4i *>(lds + chunk_at(u >> 2, u & 3)) = v[i];
        }
    }
};

template <class T, int BM, int BN>
__global__ __launch_bounds__(kThreads) void k_int8_tile(const int8_t *x, int64_t ldx, const float *xs, int64_t rows, int k,
                                                        const int8_t *w, int64_t ldw, const float *ws, int n, const float *bias,
                                                        T *y, int64_t ldy, int tiles_n)
{
    constexpr int TM = BM / 32, TN = BN / 32;            // 16 x 16 blocks of a wavefront (2 x 2 wavefronts)
    __shared__ __attribute__((aligned(16))) int8_t sx[2][BM * 64], sw[2][BN * 64];
    const int64_t tile = xcd_run(blockIdx.x, gridDim.x);
    const int64_t m0 = tile / tiles_n * BM;
    const int n0 = (int)(tile % tiles_n) * BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
    const int r16 = lane & 15, quad = lane >> 4;
    v4i acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = v4i{0, 0, 0, 0};
    CodeTile<BM> tx;
    CodeTile<BN> tw;
    const int steps = (k + 63) / 64;
    tx.load(x, ldx, m0, rows, 0, k);
    tw.load(w, ldw, n0, n, 0, k);
    tx.store(sx[0]);
    tw.store(sw[0]);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const int at = s & 1;
        if (s + 1 < steps) {
            tx.load(x, ldx, m0, rows, (s + 1) * 64, k);
            tw.load(w, ldw, n0, n, (s + 1) * 64, k);
        }
        v4i a[TN], b[TM];
#pragma unroll
        for (int i = 0; i < TN; ++i) a[i] = *reinterpret_cast<const v4i *>(sw[at] + chunk_at(wn + i * 16 + r16, quad));
#pragma unroll
        for (int j = 0; j < TM; ++j) b[j] = *reinterpret_cast<const v4i *>(sx[at] + chunk_at(wm + j * 16 + r16, quad));
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], b[j], acc[i][j], 0, 0, 0);
        if (s + 1 < steps) {
            tx.store(sx[at ^ 1]);
            tw.store(sw[at ^ 1]);
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        const int c = n0 + wn + i * 16 + quad * 4;
        float sc[4], bi[4];
        load_vec<float, 4>(sc, ws + c, n - c);
        if (bias) load_vec<float, 4>(bi, bias + c, n - c);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int64_t r = m0 + wm + j * 16 + r16;
            if (r >= rows) continue;
            const float s = xs[r];
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[e] = (float)acc[i][j][e] * s * sc[e];
                if (bias) o[e] += bi[e];
            }
            store_vec<T, 4>(y + r * ldy + c, o, n - c);
        }
    }
}

// ---- float x integer products ---------------------------------------------
// A float32 number is the exact sum of three bfloat16 numbers, its significand cut in three pieces of eight bits (an
// infinity has no such sum and comes out as NaN; below 2^-110 the last pieces run out of exponents).  A code of at most
// seven bits and a sign is one bfloat16 number.  Three bfloat16 matrix instructions therefore give the product of a
// float32 matrix and a code matrix with exact terms, added in float32, at a third of the bfloat16 rate: some five times
// the rate of the float32 matrix instructions.
//
//   weight gradient   dw[n, k] = sum over rows m of (dy[m, n] * scale[m]) * codes[m, k]
//   input gradient    dx[m, k] = sum over channels n of (dy[m, n] * w_scale[n]) * w[n, k]
//
// In both the integer matrix runs along the sum ("red") with its rows, so its tile is transposed on the way into LDS.
// The scale belongs to an index of the sum and is taken into the float operand, one rounding in float32.

__device__ __forceinline__ uint32_t high_halves(float a, float b)      // the upper 16 bits of a and of b: a in the low half
{
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float cut8(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// Eight numbers to three 16-byte chunks of bfloat16.
__device__ __forceinline__ void split8(const float (&x)[8], v4i (&out)[3])
{
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float r0 = x[i] - cut8(x[i]), r1 = x[i + 1] - cut8(x[i + 1]);
        const float l0 = r0 - cut8(r0), l1 = r1 - cut8(r1);
        out[0][i / 2] = (int)high_halves(x[i], x[i + 1]);
        out[1][i / 2] = (int)high_halves(r0, r1);
        out[2][i / 2] = (int)high_halves(l0, l1);
    }
}

// The float operand's tile: BA rows (output index) x 32 of the sum.
// kDown: the sum runs down the rows of dy (weight gradient): a thread takes eight rows of a column, the 64 lanes of a
//        wavefront neighbouring columns.  Otherwise it runs along a row (input gradient): eight neighbouring numbers.
template <class T, bool kDown, int BA>
struct FloatTile {
    static constexpr int N = BA / 64;
    float v[N][8], s[8];
    __device__ __forceinline__ void load(const T *p, int64_t ld, const float *scale, int64_t a0, int64_t na, int64_t r0, int64_t nr)
    {
        if (kDown) {
            const int64_t r = r0 + (threadIdx.x >> 6) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = r + e < nr ? scale[r + e] : 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t a = a0 + i * 64 + (threadIdx.x & 63);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = a < na && r + e < nr ? (float)p[(r + e) * ld + a] : 0.0f;
            }
        } else {
            const int64_t r = r0 + (threadIdx.x & 3) * 8;
            const int left = (int)min((int64_t)8, nr - r);
            load_vec<float, 8>(s, scale + r, left);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t a = a0 + i * 64 + (threadIdx.x >> 2);
                load_vec<T, 8>(v[i], p + a * ld + r, a < na ? left : 0);
            }
        }
    }
    // the sum of this tile's values in each of the thread's columns (kDown)
    __device__ __forceinline__ void column_sums(float (&sum)[N]) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
            sum[i] += ((v[i][0] + v[i][1]) + (v[i][2] + v[i][3])) + ((v[i][4] + v[i][5]) + (v[i][6] + v[i][7]));
    }
    __device__ __forceinline__ void store(int8_t *lds) const      // [3][BA] rows of 64 bytes
    {
        const int chunk = kDown ? threadIdx.x >> 6 : threadIdx.x & 3;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = i * 64 + (kDown ? threadIdx.x & 63 : threadIdx.x >> 2);
            float x[8];
            v4i w[3];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = v[i][e] * s[e];
            split8(x, w);
#pragma unroll
            for (int q = 0; q < 3; ++q) *reinterpret_cast<v4i *>(lds + q * BA * 64 + chunk_at(row, chunk)) = w[q];
        }
    }
};

// The integer operand's tile: BB columns x 32 of the sum, transposed.  A unit is four columns x four rows of the sum.
template <int BB>
struct TurnedTile {
    uint32_t v[4];
    __device__ __forceinline__ void load(const int8_t *q, int64_t ld, int b0, int nb, int64_t r0, int64_t nr)
    {
        const int u = threadIdx.x, b = b0 + (u >> 3) * 4;
        const int64_t r = r0 + (u & 7) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[1];
            load_bytes<4>(w, q + (r + i) * ld + b, (BB * 2 >= kThreads || u < BB * 2) && r + i < nr ? nb - b : 0);
            v[i] = w[0];
        }
    }
    __device__ __forceinline__ void store(int8_t *lds) const
    {
        const int u = threadIdx.x;
        if (BB * 2 < kThreads && u >= BB * 2) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = (u >> 3) * 4 + j;
            uint32_t w[2] = {high_halves(code_value(v[0], j), code_value(v[1], j)), high_halves(code_value(v[2], j), code_value(v[3], j))};
            __builtin_memcpy(__builtin_assume_aligned(lds + chunk_at(row, (u & 7) >> 1) + (u & 1) * 8, 8), w, 8);
        }
    }
};

// out[a, b] over a tile of BA x BB, sum over [r0, r1).
template <class T, bool kDown, int BA, int BB>
struct SplitProduct {
    static constexpr int TA = BA / 32, TB = BB / 32;
    v4f acc[TB][TA];
    __device__ __forceinline__ void step(const int8_t *sa, const int8_t *sb)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wa = (wave >> 1) * (BA / 2), wb = (wave & 1) * (BB / 2);
        v8b b[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) b[i] = *reinterpret_cast<const v8b *>(sb + chunk_at(wb + i * 16 + (lane & 15), lane >> 4));
#pragma unroll
        for (int q = 2; q >= 0; --q) {                    // small pieces first
            v8b a[TA];
#pragma unroll
            for (int j = 0; j < TA; ++j) a[j] = *reinterpret_cast<const v8b *>(sa + q * BA * 64 + chunk_at(wa + j * 16 + (lane & 15), lane >> 4));
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int j = 0; j < TA; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[i], a[j], acc[i][j], 0, 0, 0);
        }
    }
};

template <class T, bool kDown, int BA, int BB, class TO, bool kSums>
__device__ __forceinline__ void split_tile(const T *dy, int64_t ldd, const float *scale, const int8_t *q, int64_t ldq,
                                           int64_t a0, int64_t na, int b0, int nb, int64_t r0, int64_t r1,
                                           TO *out, int64_t ldo, float *sums)
{
    __shared__ __attribute__((aligned(16))) int8_t sa[2][3 * BA * 64], sb[2][BB * 64];
    SplitProduct<T, kDown, BA, BB> p;
    constexpr int TA = p.TA, TB = p.TB;
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
        for (int j = 0; j < TA; ++j) p.acc[i][j] = v4f{0, 0, 0, 0};
    FloatTile<T, kDown, BA> ta;
    TurnedTile<BB> tb;
    float col[FloatTile<T, kDown, BA>::N];
#pragma unroll
    for (int i = 0; i < ta.N; ++i) col[i] = 0.0f;
    ta.load(dy, ldd, scale, a0, na, r0, r1);
    tb.load(q, ldq, b0, nb, r0, r1);
    ta.store(sa[0]);
    tb.store(sb[0]);
    if (kSums) ta.column_sums(col);
    __syncthreads();
    int at = 0;
    for (int64_t r = r0; r < r1; r += 32, at ^= 1) {
        const bool more = r + 32 < r1;
        if (more) {
            ta.load(dy, ldd, scale, a0, na, r + 32, r1);
            tb.load(q, ldq, b0, nb, r + 32, r1);
        }
        p.step(sa[at], sb[at]);
        if (more) {
            ta.store(sa[at ^ 1]);
            tb.store(sb[at ^ 1]);
            if (kSums) ta.column_sums(col);
            __syncthreads();
        }
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wa = (wave >> 1) * (BA / 2), wb = (wave & 1) * (BB / 2);
#pragma unroll
    for (int j = 0; j < TA; ++j) {
        const int64_t a = a0 + wa + j * 16 + (lane & 15);
        if (a >= na) continue;
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            const int b = b0 + wb + i * 16 + (lane >> 4) * 4;
            float o[4] = {p.acc[i][j][0], p.acc[i][j][1], p.acc[i][j][2], p.acc[i][j][3]};
            store_vec<TO, 4>(out + a * ldo + b, o, nb - b);
        }
    }
    if (kSums && sums) {                                   // the four wavefronts hold the four eights of every 32 rows
        __syncthreads();
        float *f = reinterpret_cast<float *>(sa[0]);
#pragma unroll
        for (int i = 0; i < ta.N; ++i) f[wave * BA + i * 64 + lane] = col[i];
        __syncthreads();
        for (int c = threadIdx.x; c < BA; c += kThreads)
            if (a0 + c < na) sums[a0 + c] = (f[c] + f[BA + c]) + (f[2 * BA + c] + f[3 * BA + c]);
    }
}

// Weight gradient: workgroup (tile of dw, piece of the rows).  The pieces' results are added by k_add_pieces in a fixed
// order (no atomics: the same bits on every run).
template <class T, int BA, int BB>
__global__ __launch_bounds__(kThreads, 2) void k_weight_grad(const T *dy, int64_t ldd, const int8_t *codes, int64_t ldc, const float *scale,
                                                             int64_t rows, int n, int k, int64_t rows_per_piece, int tiles_k, int tiles,
                                                             float *dw, float *db, int64_t pitch)
{
    const int64_t id = xcd_run(blockIdx.x, gridDim.x);
    const int64_t piece = id / tiles;
    const int tile = (int)(id % tiles), a0 = tile / tiles_k * BA, b0 = tile % tiles_k * BB;
    const int64_t r0 = piece * rows_per_piece, r1 = min(rows, r0 + rows_per_piece);
    split_tile<T, true, BA, BB, float, true>(dy, ldd, scale, codes, ldc, a0, n, b0, k, r0, r1,
                                             dw + piece * pitch, k, db && b0 == 0 ? db + piece * pitch : nullptr);
}

// out[i] = sum of part[p][i] over the pieces, in 64 bits; the first `cut` values are dw, the others db.  A workgroup takes
// `wide` values; its 256 / wide groups of threads add pieces in turn, and their sums are added in order.
__global__ __launch_bounds__(kThreads) void k_add_pieces(const float *part, int pieces, int64_t count, int64_t cut, int wide, float *dw, float *db)
{
    __shared__ double buf[kThreads];
    const int col = threadIdx.x & (wide - 1), group = threadIdx.x / wide, groups = kThreads / wide;
    const int64_t i = (int64_t)blockIdx.x * wide + col;
    double s = 0.0;
    if (i < count) {
#pragma unroll 8
        for (int p = group; p < pieces; p += groups) s += (double)part[p * count + i];
    }
    buf[threadIdx.x] = s;
    __syncthreads();
    if (group == 0 && i < count) {
        for (int g = 1; g < groups; ++g) s += buf[g * wide + col];
        if (i < cut) dw[i] = (float)s;
        else db[i - cut] = (float)s;
    }
}

__global__ __launch_bounds__(kThreads) void k_fill_zero(float *p, int64_t count)
{
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i < count) p[i] = 0.0f;
}

template <class T, int BA, int BB>
__global__ __launch_bounds__(kThreads, 2) void k_input_grad(const T *dy, int64_t ldd, const int8_t *w, int64_t ldw, const float *ws,
                                                            int64_t rows, int n, int k, int tiles_k, T *dx, int64_t lddx)
{
    const int64_t tile = xcd_run(blockIdx.x, gridDim.x);
    split_tile<T, false, BA, BB, T, false>(dy, ldd, ws, w, ldw, tile / tiles_k * BA, rows, (int)(tile % tiles_k) * BB, k, 0, n,
                                           dx, lddx, nullptr);
}

template <class F>
void with_type(int32_t type, F f)
{
    if (type == YH_FLOAT32) f(float());
    else if (type == YH_BFLOAT16) f((__bf16)0.0f);
    else f((_Float16)0.0f);
}

struct GradPlan { int ba, bb, tiles_k, tiles, pieces; int64_t rows_per_piece; };
GradPlan plan_weight_grad(int64_t rows, int n, int k)
{
    GradPlan p;
    p.ba = n <= 64 ? 64 : 128;
    p.bb = k <= 64 ? 64 : 128;
    p.tiles_k = (k + p.bb - 1) / p.bb;
    p.tiles = (n + p.ba - 1) / p.ba * p.tiles_k;
    // two workgroups a compute unit (their LDS allows no more), each with at least four steps of 32 rows
    const int64_t want = std::max(1, 2 * 256 / p.tiles), steps = (rows + 31) / 32;
    const int64_t pieces = std::max<int64_t>(1, std::min(want, (steps + 3) / 4));
    p.rows_per_piece = (steps + pieces - 1) / pieces * 32;
    p.pieces = (int)((rows + p.rows_per_piece - 1) / p.rows_per_piece);
    return p;
}

unsigned blocks_for(int64_t count) { return (unsigned)((count + kThreads - 1) / kThreads); }

}  // namespace

hipError_t launch_int8_product(const int8_t *x, int64_t ldx, const float *x_scale, int64_t rows, int32_t k,
                               const int8_t *w, int64_t ldw, const float *w_scale, int32_t n, const float *bias,
                               void *y, int64_t ldy, int32_t type, hipStream_t st)
{
    with_type(type, [&](auto t) {
        using T = decltype(t);
#define CALL(BM, BN)                                                                                                        \
        do {                                                                                                                \
            const int tn = (n + BN - 1) / BN;                                                                               \
            k_int8_tile<T, BM, BN><<<dim3((unsigned)((rows + BM - 1) / BM * tn)), kThreads, 0, st>>>(                       \
                x, ldx, x_scale, rows, k, w, ldw, w_scale, n, bias, static_cast<T *>(y), ldy, tn);                          \
        } while (0)
        // large tiles where they fill the card, small ones where there are few rows
        if ((rows + 127) / 128 * ((n + 127) / 128) >= 256) CALL(128, 128);
        else CALL(32, 64);
#undef CALL
    });
    return hipGetLastError();
}

int weight_grad_chunks(int64_t rows, int32_t n, int32_t k) { return plan_weight_grad(rows, n, k).pieces; }

hipError_t launch_weight_grad(const Rows &dy, const int8_t *codes, int64_t ldc, const float *scale, int64_t rows,
                              int32_t n, int32_t k, float *dw, float *db, void *workspace, hipStream_t st)
{
    const int64_t count = (int64_t)n * k;
    if (rows == 0) {
        k_fill_zero<<<dim3(blocks_for(count)), kThreads, 0, st>>>(dw, count);
        if (db) k_fill_zero<<<dim3(blocks_for(n)), kThreads, 0, st>>>(db, n);
        return hipGetLastError();
    }
    const GradPlan p = plan_weight_grad(rows, n, k);
    float *pw = p.pieces > 1 ? static_cast<float *>(workspace) : dw;
    float *pb = !db ? nullptr : p.pieces > 1 ? pw + count : db;
    const int64_t pitch = db ? count + n : count;              // a piece: dw, then db
    with_type(dy.type, [&](auto t) {
        using T = decltype(t);
#define CALL(BA, BB) k_weight_grad<T, BA, BB><<<dim3((unsigned)(p.tiles * p.pieces)), kThreads, 0, st>>>(                   \
            static_cast<const T *>(dy.p), dy.ld, codes, ldc, scale, rows, n, k, p.rows_per_piece, p.tiles_k, p.tiles, pw, pb, pitch)
        if (p.ba == 64 && p.bb == 64) CALL(64, 64);
        else if (p.ba == 64) CALL(64, 128);
        else if (p.bb == 64) CALL(128, 64);
        else CALL(128, 128);
#undef CALL
    });
    if (p.pieces > 1) {
        // few pieces: a thread a value; many: eight pieces a thread, down to 16 neighbouring values (64 bytes) a workgroup
        int wide = kThreads;
        while (wide > 16 && p.pieces * wide > 8 * kThreads) wide /= 2;
        k_add_pieces<<<dim3((unsigned)((pitch + wide - 1) / wide)), kThreads, 0, st>>>(pw, p.pieces, pitch, count, wide, dw, db);
    }
    return hipGetLastError();
}

hipError_t launch_input_grad(const Rows &dy, const int8_t *w, int64_t ldw, const float *w_scale, int64_t rows,
                             int32_t n, int32_t k, void *dx, int64_t lddx, int32_t type, hipStream_t st)
{
    (void)type;
    with_type(dy.type, [&](auto t) {
        using T = decltype(t);
#define CALL(BA, BB)                                                                                                        \
        do {                                                                                                                \
            const int tk = (k + BB - 1) / BB;                                                                               \
            k_input_grad<T, BA, BB><<<dim3((unsigned)((rows + BA - 1) / BA * tk)), kThreads, 0, st>>>(                      \
                static_cast<const T *>(dy.p), dy.ld, w, ldw, w_scale, rows, n, k, tk, static_cast<T *>(dx), lddx);          \
        } while (0)
        if (k <= 64) CALL(64, 64);
        else if ((rows + 127) / 128 * ((k + 127) / 128) >= 256) CALL(128, 128);
        else CALL(64, 64);
#undef CALL
    });
    return hipGetLastError();
}

}  // namespace yh
