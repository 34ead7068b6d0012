// Products of row codes on the matrix cores: the integer product of a pointwise convolution, and its gradients, which
// multiply a float matrix by an integer one.
#include <algorithm>
#include <type_traits>
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

// Loads through a buffer descriptor: a uniform 64-bit base, a uniform 32-bit offset that changes from load to load and a
// lane offset of 32 bits that does not change at all.  (With plain pointers the compiler keeps and advances one 64-bit
// address a lane and load, some forty register pairs here.)  The descriptor's bound is the address space's end: every
// offset is inside of the matrix by construction.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_at(const void *p)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, -1, 0x00027000);
}
__device__ __forceinline__ void load_at(Buffer b, uint32_t lane, uint32_t uniform, uint32_t &v) { v = __builtin_amdgcn_raw_buffer_load_b32(b, lane, uniform, 0); }
__device__ __forceinline__ void load_at(Buffer b, uint32_t lane, uint32_t uniform, float &v)
{
    v = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, lane, uniform, 0));
}
template <class T>
__device__ __forceinline__ void load_at(Buffer b, uint32_t lane, uint32_t uniform, T &v)      // 16-bit numbers
{
    const uint16_t w = __builtin_amdgcn_raw_buffer_load_b16(b, lane, uniform, 0);
    __builtin_memcpy(&v, &w, 2);
}
__device__ __forceinline__ v4i load_at16(Buffer b, uint32_t lane, uint32_t uniform) { return __builtin_amdgcn_raw_buffer_load_b128(b, lane, uniform, 0); }

// ---- y = (codes . w codes^T) * scale * w_scale + bias ---------------------
// The sums are whole numbers in 32 bits (exact up to 65536 terms of 127^2); one product by each scale in float32 and one
// rounding to the output's type follow.  The weights are the matrix instruction's first operand: a lane then holds four
// neighbouring output channels of one row and stores them together.

__device__ __forceinline__ v4i load_chunk(const int8_t *p, int left)
{
    uint32_t w[4];
    load_bytes<16>(w, p, left);
    v4i v;
    __builtin_memcpy(&v, w, 16);
    return v;
}

// R rows x 64 of the sum.  Rows past the matrix's end read its last row again (their results are not stored), so that a
// whole step asks nothing; load_part() reads what is left of the sum and zeros behind it.
template <int R>
struct CodeTile {
    static constexpr int N = R * 4 / kThreads;
    v4i v[N];
    uint32_t off[N];
    const int8_t *base;
    int64_t ld, last;
    __device__ __forceinline__ void place(const int8_t *p, int64_t pitch, int64_t row0, int64_t rows)
    {
        base = p + row0 * pitch;
        ld = pitch, last = rows - 1 - row0;
#pragma unroll
        for (int i = 0; i < N; ++i) off[i] = (uint32_t)(min((int64_t)(threadIdx.x + i * kThreads) >> 2, last) * ld + (threadIdx.x & 3) * 16);
    }
    __device__ __forceinline__ void load_whole(int k0)
    {
        const Buffer b = buffer_at(base + k0);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = load_at16(b, off[i], 0);
    }
    __device__ __forceinline__ void load_part(int k0, int k)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = k0 + (threadIdx.x & 3) * 16;
            v[i] = load_chunk(base + min((int64_t)(threadIdx.x + i * kThreads) >> 2, last) * ld + c, k - c);
        }
    }
    __device__ __forceinline__ void store(int8_t *lds) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = threadIdx.x + i * kThreads;
            *reinterpret_cast<v4i *>(lds + chunk_at(u >> 2, u & 3)) = v[i];
        }
    }
};

// Orders a wavefront's LDS writes before its other lanes' reads.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr int kOutPitch = 64 * 4 + 16;                     // 16 rows of 64 results on their way out of a wavefront

// 16 x 64 results of a wavefront: scaled, in LDS with neighbouring columns together, out.  acc[i] holds channels
// n0 + 16 i + 4 (lane >> 4) + 0..3 of row lane & 15.
template <class T>
__device__ __forceinline__ void out_16x64(const v4i (&acc)[4], float s, const float *ws, const float *bias, int8_t *turn,
                                          T *y, int64_t ldy, int64_t first, int64_t rows, int n0, int n)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = i * 16 + (lane >> 4) * 4;
        v4f o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (float)acc[i][e] * s * ws[c + e] + bias[c + e];
        *reinterpret_cast<v4f *>(turn + (lane & 15) * kOutPitch + c * 4) = o;
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 4 + (lane >> 4), c = (lane & 15) * 4;
        float o[4];
        __builtin_memcpy(o, __builtin_assume_aligned(turn + row * kOutPitch + c * 4, 16), 16);
        if (first + row < rows) store_vec<T, 4>(y + (first + row) * ldy + n0 + c, o, n - n0 - c);
    }
    wave_sync();
}

// The tile form, from codes in memory: 43264 rows, 1536 -> 425 56 us (1.0 POP/s, half of what a large library product
// reaches), 21632 rows, 1024 -> 512 22.6 us.  A wavefront's 64 x 64 results ask LDS for as many cycles as the matrix
// instructions take (counted over a launch: matrix instructions busy 24 % of the time, LDS 31 %).  Operands read a step
// ahead win 3 to 9 % where few wavefronts share a compute unit (2704 rows, 1024 -> 512 7.6 us, 8.3 without); larger tiles,
// longer steps, loads further ahead and wave priorities won nothing.  Three workgroups a compute unit: 168 registers.
template <class T, int BM, int BN>
__global__ __launch_bounds__(kThreads, 3) void k_int8_tile(const int8_t *x, int64_t ldx, const float *xs, int64_t rows, int k,
                                                        const int8_t *w, int64_t ldw, const float *ws, int n, const float *bias,
                                                        T *y, int64_t ldy, int tiles_n)
{
    constexpr int WN = BN / 64, WM = 4 / WN, TM = BM / WM / 16, TN = 4;       // wavefronts of 64 channels, 16 x 16 blocks of one
    constexpr int kStage = (BM + BN) * 64, kTurn = 4 * 16 * kOutPitch;
    __shared__ __attribute__((aligned(16))) int8_t lds[2 * kStage > kTurn ? 2 * kStage : kTurn];
    __shared__ float lsc[BN], lb[BN];
    const uint32_t tile = (uint32_t)xcd_run(blockIdx.x, gridDim.x);
    const int64_t m0 = (int64_t)(tile / (uint32_t)tiles_n) * BM;
    const int n0 = (int)(tile % (uint32_t)tiles_n) * BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN * (BM / WM), wn = wave % WN * 64;
    const int r16 = lane & 15, quad = lane >> 4;
    for (int u = threadIdx.x; u < BN; u += kThreads) {
        lsc[u] = n0 + u < n ? ws[n0 + u] : 0.0f;
        lb[u] = bias && n0 + u < n ? bias[n0 + u] : 0.0f;
    }
    v4i acc[TM][TN];
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int i = 0; i < TN; ++i) acc[j][i] = v4i{0, 0, 0, 0};
    CodeTile<BM> tx;
    CodeTile<BN> tw;
    tx.place(x, ldx, m0, rows);
    tw.place(w, ldw, n0, n);
    const auto store = [&](int8_t *stage) {
        tx.store(stage);
        tw.store(stage + BM * 64);
    };
    struct Parts { v4i a[TN], b[TM]; };
    const auto read = [&](Parts &f, const int8_t *sx) {
        const int8_t *sw = sx + BM * 64;
#pragma unroll
        for (int i = 0; i < TN; ++i) f.a[i] = *reinterpret_cast<const v4i *>(sw + chunk_at(wn + i * 16 + r16, quad));
#pragma unroll
        for (int j = 0; j < TM; ++j) f.b[j] = *reinterpret_cast<const v4i *>(sx + chunk_at(wm + j * 16 + r16, quad));
    };
    const auto multiply = [&](const Parts &f) {
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int i = 0; i < TN; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.a[i], f.b[j], acc[j][i], 0, 0, 0);
    };
    const int whole = ldx < (1 << 22) && ldw < (1 << 22) ? k & ~63 : 0;
    if (whole) {
        // a step's operands are read from LDS while the step before is multiplied, stored while the one before that is, and
        // loaded one step earlier still
        Parts f[2];
        const auto fetch = [&](int q) {
            if (q < whole) {
                tx.load_whole(q);
                tw.load_whole(q);
            }
        };
        fetch(0);
        store(lds);
        fetch(64);
        __syncthreads();
        read(f[0], lds);
        if (64 < whole) store(lds + kStage);
        fetch(128);
        __syncthreads();
        const auto step = [&](int q, const Parts &now, Parts &next, int8_t *here, int8_t *there) {
            if (q + 64 < whole) read(next, there);
            multiply(now);
            // this stage was read in the step before, and every wavefront has passed the barrier since
            if (q + 128 < whole) store(here);
            fetch(q + 192);
            __syncthreads();
        };
        for (int q = 0; q < whole; q += 128) {
            step(q, f[0], f[1], lds, lds + kStage);
            if (q + 64 < whole) step(q + 64, f[1], f[0], lds + kStage, lds);
        }
    }
    for (int q = whole; q < k; q += 64) {
        tx.load_part(q, k);
        tw.load_part(q, k);
        store(lds);
        __syncthreads();
        Parts f;
        read(f, lds);
        multiply(f);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int64_t r = m0 + wm + j * 16;
        out_16x64<T>(acc[j], r + r16 < rows ? xs[r + r16] : 0.0f, lsc + wn, lb + wn, lds + wave * 16 * kOutPitch, y, ldy, r, rows, n0 + wn, n);
    }
}

// 16 bytes of a row's elements from p on, `left` of them to be read; zeros behind.
template <class TX, bool kWhole = false>                   // kWhole: 16 bytes or nothing
__device__ __forceinline__ v4i load_elements(const TX *p, int left)
{
    constexpr int V = 16 / (int)sizeof(TX);
    v4i v = {0, 0, 0, 0};
    if (left >= V) {
        const LooseBytes<16>::type t = *reinterpret_cast<const LooseBytes<16>::type *>(p);
        __builtin_memcpy(&v, &t, 16);
    } else if (!kWhole && left > 0) {
        uint32_t w[4];
        load_end<sizeof(TX), 4>(w, p, left * (int)sizeof(TX));
        __builtin_memcpy(&v, w, 16);
    }
    return v;
}

// Zeros in the place of the elements from `left` on.
template <class TX, int V>
__device__ __forceinline__ void clear_end(TX (&t)[V], int left)
{
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j >= left) t[j] = (TX)0;
}

// ---- the same from float rows: codes taken on the way --------------------------
// Reading x once and writing y once is all the product has to move, so where it can the product takes the codes itself
// and they stay in LDS.  A wavefront turns 16 rows into codes at a time: `lanes` (4 to 16) neighbouring lanes a row, four
// vectors of 16 bytes each, so rows of up to 1024 bytes, and leaves them in LDS rows of k64 + 16 bytes (k64: K rounded up to 64, zeros
// behind K; the 16 bytes shift each row by a bank group, so that 16 rows are read without a conflict).
template <class TX, int G, bool kWhole>                  // kWhole: K is a multiple of 16
struct CodeRows {
    static constexpr int V = 16 / (int)sizeof(TX);
    v4i raw[G][4];                                       // G = lanes / 4 passes of 64 / lanes rows, as they are in memory
    const TX *x;
    int64_t ldx, rows;
    int k, k64, lanes;
    __device__ __forceinline__ void load(int64_t first)
    {
        const int lane = threadIdx.x & 63, sub = lane & (lanes - 1), per = 64 / lanes;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int64_t row = first + g * per + lane / lanes;
            const TX *p = x + row * ldx;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = (i * lanes + sub) * V;
                raw[g][i] = load_elements<TX, kWhole>(p + c, row < rows ? k - c : 0);
            }
        }
    }
    // what is loaded, the 16 rows from `first` on, as codes to `lds` and scales to `ls`, and to codes / scale if they are
    // not null
    __device__ __forceinline__ void put(int64_t first, int8_t *lds, float *ls, int8_t *codes, int64_t ldc, float *scale) const
    {
        const int lane = threadIdx.x & 63, sub = lane & (lanes - 1), per = 64 / lanes;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int r = g * per + lane / lanes;
            float v[4][V];
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                TX t[V];
                __builtin_memcpy(t, &raw[g][i], 16);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[i][j] = (float)t[j];
                    m = max(m, __float_as_uint(v[i][j]) & 0x7fffffffu);
                }
            }
            const RowScale s = row_scale(row_max(m, lanes), (float)kCodeMax);
            const bool in = first + r < rows;
            if (sub == 0) {
                ls[r] = s.s;
                if (scale && in) scale[first + r] = s.s;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = (i * lanes + sub) * V;
                uint32_t w[V / 4];
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const uint32_t q = pack4(code_bits(v[i][j], s.r), code_bits(v[i][j + 1], s.r), code_bits(v[i][j + 2], s.r), code_bits(v[i][j + 3], s.r));
                    w[j / 4] = s.live ? q : 0u;
                }
                if (c < k64) __builtin_memcpy(__builtin_assume_aligned(lds + r * (k64 + 16) + c, V), w, V);
                if (codes && in) store_bytes<V>(codes + (first + r) * ldc + c, w, k - c);
            }
        }
    }
};
template <int G, bool kWhole>
struct CodeRows<int8_t, G, kWhole> {                     // codes already
    static constexpr int V = 16;
    v4i raw[G][4];
    const int8_t *x;
    int64_t ldx, rows;
    int k, k64, lanes;
    __device__ __forceinline__ void load(int64_t first)
    {
        const int lane = threadIdx.x & 63, sub = lane & (lanes - 1), per = 64 / lanes;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t row = first + g * per + lane / lanes;
                const int c = (i * lanes + sub) * V;
                raw[g][i] = load_elements<int8_t, kWhole>(x + row * ldx + c, row < rows ? k - c : 0);
            }
    }
    __device__ __forceinline__ void put(int64_t, int8_t *lds, float *, int8_t *, int64_t, float *) const
    {
        const int lane = threadIdx.x & 63, sub = lane & (lanes - 1), per = 64 / lanes;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = (i * lanes + sub) * V;
                if (c < k64) *reinterpret_cast<v4i *>(lds + (g * per + lane / lanes) * (k64 + 16) + c) = raw[g][i];
            }
    }
};

// Many rows, weights that fit: a workgroup keeps all weights in LDS for good and its eight wavefronts, which have nothing
// more to say to each other, take blocks of 16 rows in turn, the next block's loads under this block's arithmetic.  Bound
// by memory: 173056 rows, 256 -> 128 in float32 move 266 MB in 56 us (4.8 TB/s), 692224 rows, 128 -> 64 532 MB in 108 us
// (4.9 TB/s); through codes in memory they take 77 and 179 us.
constexpr int kRowWaves = 8;

template <class TX, class T, int G, bool kWhole>
__global__ __launch_bounds__(64 * kRowWaves) void k_int8_rows(const TX *x, int64_t ldx, const float *xs, int64_t rows, int k, int lanes,
                                                   const int8_t *w, int64_t ldw, const float *ws, int n, const float *bias,
                                                   T *y, int64_t ldy, int8_t *codes, int64_t ldc, float *scale)
{
    extern __shared__ __attribute__((aligned(16))) int8_t lds[];
    const int k64 = (k + 63) / 64 * 64, pitch = k64 + 16, nw = (n + 63) / 64 * 64;
    int8_t *lw = lds;
    float *lsc = reinterpret_cast<float *>(lds + nw * pitch), *lb = lsc + nw;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int8_t *mine = reinterpret_cast<int8_t *>(lb + nw) + wave * (16 * pitch + 16 * kOutPitch + 64);
    int8_t *lx = mine, *turn = mine + 16 * pitch;
    float *ls = reinterpret_cast<float *>(turn + 16 * kOutPitch);
    const int per = k64 / 16;
    for (int u = threadIdx.x; u < nw * per; u += blockDim.x) {
        const int r = u / per, c = (u - r * per) * 16;
        *reinterpret_cast<v4i *>(lw + r * pitch + c) = load_chunk(w + (int64_t)r * ldw + c, r < n ? k - c : 0);
    }
    for (int u = threadIdx.x; u < nw; u += blockDim.x) {
        lsc[u] = u < n ? ws[u] : 0.0f;
        lb[u] = bias && u < n ? bias[u] : 0.0f;
    }
    __syncthreads();
    CodeRows<TX, G, kWhole> in;
    in.x = x, in.ldx = ldx, in.rows = rows, in.k = k, in.k64 = k64, in.lanes = lanes;
    const int64_t stride = (int64_t)gridDim.x * kRowWaves;
    int64_t b = (int64_t)blockIdx.x * kRowWaves + wave;
    if (b * 16 < rows) in.load(b * 16);
    for (; b * 16 < rows; b += stride) {
        in.put(b * 16, lx, ls, codes, ldc, scale);
        in.load((b + stride) * 16);                        // under this block's products
        wave_sync();
        const float s = sizeof(TX) == 1 ? (b * 16 + (lane & 15) < rows ? xs[b * 16 + (lane & 15)] : 0.0f) : ls[lane & 15];
        const int at = (lane & 15) * pitch + (lane >> 4) * 16;
        for (int c0 = 0; c0 < nw; c0 += 64) {
            v4i acc[4] = {};
            for (int q = 0; q < k64; q += 64) {
                const v4i xv = *reinterpret_cast<const v4i *>(lx + at + q);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const v4i *>(lw + (c0 + i * 16) * pitch + at + q), xv, acc[i], 0, 0, 0);
            }
            out_16x64<T>(acc, s, lsc + c0, lb + c0, turn, y, ldy, b * 16, rows, c0, n);
        }
    }
}

// The 16 rows of codes from LDS (pitch `pitch`) to memory, by the workgroup.
__device__ __forceinline__ void codes_out(const int8_t *lx, int pitch, int64_t first, int64_t rows, int k, int8_t *codes, int64_t ldc)
{
    const int per = (k + 15) / 16;
    for (int u = threadIdx.x; u < 16 * per; u += kThreads) {
        const int r = u / per, c = (u - r * per) * 16;
        uint32_t w[4];
        __builtin_memcpy(w, __builtin_assume_aligned(lx + r * pitch + c, 16), 16);
        if (first + r < rows) store_bytes<16>(codes + (first + r) * ldc + c, w, k - c);
    }
}

// What a lane reads of a row in whole vectors; the one that ends the row, where it may not be read whole (the matrix's
// last rows), comes by a load of its own: a short call is a straight run through its code, and lasts as long as that.
template <class TX, int N, bool kWhole>
__device__ __forceinline__ void load_row(v4i (&v)[N], const TX *p, int at, int step, int read, int k)
{
    constexpr int V = 16 / (int)sizeof(TX);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = v4i{0, 0, 0, 0};
        if (at + i * step + V <= read) {
            const LooseBytes<16>::type t = *reinterpret_cast<const LooseBytes<16>::type *>(p + at + i * step);
            __builtin_memcpy(&v[i], &t, 16);
        }
    }
    if (!kWhole && k % V && read == k) {
        const int end = k / V * V;
        const v4i e = load_elements<TX>(p + end, k - end);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i * step == end) v[i] = e;
    }
}

// Four rows of a workgroup's 16 a wavefront, each by all its lanes: codes at lx, scales at ls (k_int8_few).
template <class TX, int IT, bool kWhole>
__device__ __forceinline__ void code_four_rows(const TX *x, int64_t ldx, int64_t spare, int64_t first, int64_t rows, int k, int k64,
                                               int8_t *lx, float *ls, float *scale)
{
    constexpr int V = RowVec<TX>::V;
    const int lane = threadIdx.x & 63, r0 = (threadIdx.x >> 6) * 4, pitch = k64 + 16;
    const bool once = IT == 1 || k <= IT * 64 * V;        // the row fits the wavefront's registers
    v4i raw[4][IT];
    uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < 4; ++r)
        load_row<TX, IT, kWhole>(raw[r], x + (first + r0 + r) * ldx, lane * V, 64 * V, left_of(first + r0 + r, rows, spare, k, 0, V), k);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float v[IT][V];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            TX t[V];
            __builtin_memcpy(t, &raw[r][i], 16);
            if (!kWhole && k % V) clear_end(t, k - (i * 64 + lane) * V);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] = (float)t[j];
                m[r] = max(m[r], __float_as_uint(v[i][j]) & 0x7fffffffu);
            }
        }
        if (!once && first + r0 + r < rows)
            for (int c = (IT * 64 + lane) * V; c < k; c += 64 * V) {
                float t[V];
                load_vec<TX, V>(t, x + (first + r0 + r) * ldx + c, k - c);
#pragma unroll
                for (int j = 0; j < V; ++j) m[r] = max(m[r], __float_as_uint(t[j]) & 0x7fffffffu);
            }
        const RowScale s = row_scale(row_max(m[r], 64), (float)kCodeMax);
        const bool in = first + r0 + r < rows;
        if (lane == 0) {
            ls[r0 + r] = s.s;
            if (scale && in) scale[first + r0 + r] = s.s;
        }
        const auto put = [&](const float (&t)[V], int c) {
            uint32_t w[V / 4];
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const uint32_t q = pack4(code_bits(t[j], s.r), code_bits(t[j + 1], s.r), code_bits(t[j + 2], s.r), code_bits(t[j + 3], s.r));
                w[j / 4] = s.live ? q : 0u;
            }
            if (c < k64) __builtin_memcpy(__builtin_assume_aligned(lx + (r0 + r) * pitch + c, V), w, V);
        };
#pragma unroll
        for (int i = 0; i < IT; ++i) put(v[i], (i * 64 + lane) * V);
        if (!once)
            for (int c = (IT * 64 + lane) * V; c < k64; c += 64 * V) {
                float t[V];
                load_vec<TX, V>(t, x + (first + r0 + r) * ldx + c, in ? k - c : 0);
                put(t, c);
            }
    }
}
__device__ __forceinline__ void code_rows_given(const int8_t *x, int64_t ldx, const float *xs, int64_t first, int64_t rows, int k, int k64, int8_t *lx, float *ls)
{
    const int per = k64 / 16;
    if (threadIdx.x < 16) ls[threadIdx.x] = first + threadIdx.x < rows ? xs[first + threadIdx.x] : 0.0f;
    for (int u = threadIdx.x; u < 16 * per; u += kThreads) {
        const int r = u / per, c = (u - r * per) * 16;
        *reinterpret_cast<v4i *>(lx + r * (k64 + 16) + c) = load_elements<int8_t>(x + (first + r) * ldx + c, first + r < rows ? k - c : 0);
    }
}

// Few rows: a workgroup takes 16 rows and 64 channels, 16 a wavefront.  The weights' loads are under way before the rows
// are turned into codes (four rows a wavefront); nothing is read in turns, so a call lasts about three memory latencies
// and one pass through its code, which is why rows of up to 256 channels have a form of their own (S = 1; 300 rows,
// 256 -> 128: 5.0 us, 6.0 with S = 4).  169 rows, 1024 -> 512: 7.0 us.
template <class TX, class T, int S, bool kWhole>             // kWhole: K is a multiple of 16
__global__ __launch_bounds__(kThreads) void k_int8_few(const TX *x, int64_t ldx, int64_t spare, const float *xs, int64_t rows, int k,
                                                       const int8_t *w, int64_t ldw, int64_t spare_w, const float *ws, int n, const float *bias,
                                                       T *y, int64_t ldy, int8_t *codes, int64_t ldc, float *scale)
{
    constexpr int kAhead = 4 * S;                          // steps of 64 whose weights are fetched first
    extern __shared__ __attribute__((aligned(16))) int8_t lds[];
    const int k64 = (k + 63) / 64 * 64, pitch = k64 + 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, quad = lane >> 4;
    const int64_t first = (int64_t)blockIdx.x * 16;
    const int n0 = blockIdx.y * 64 + wave * 16;
    int8_t *turn = lds + wave * 4096, *lx = lds + 4 * 4096;      // a wavefront's weights on their way to its operands: 4 steps
    float *ls = reinterpret_cast<float *>(lx + 16 * pitch);
    // four lanes take a row's 64 bytes of a step
    const int wrow = min(n0 + (lane >> 2), n - 1), part = (lane & 3) * 16;
    const int8_t *wr = w + (int64_t)wrow * ldw;
    const int read = left_of(wrow, n, spare_w, k, 0, 16);      // weights beyond K meet codes that are zero
    v4i a[kAhead];
    load_row<int8_t, kAhead, kWhole>(a, wr, part, 64, read, k);
    const int64_t row = first + r16;
    const int c = n0 + quad * 4;
    float sc[4], bi[4] = {0.0f, 0.0f, 0.0f, 0.0f}, o[4];
    load_vec<float, 4>(sc, ws + c, n - c);
    if (bias) load_vec<float, 4>(bi, bias + c, n - c);
    if (blockIdx.y) codes = nullptr, scale = nullptr;
    if constexpr (sizeof(TX) == 1) code_rows_given(x, ldx, xs, first, rows, k, k64, lx, ls);
    else code_four_rows<TX, S, kWhole>(x, ldx, spare, first, rows, k, k64, lx, ls, scale);
    __syncthreads();
    if (codes) codes_out(lx, pitch, first, rows, k, codes, ldc);
    v4i acc = {0, 0, 0, 0}, odd = {0, 0, 0, 0};            // two chains of sums: one would wait for itself
    const int8_t *at = lx + r16 * pitch + quad * 16;
    const auto four_steps = [&](const v4i *wv, int q) {
        wave_sync();
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<v4i *>(turn + i * 1024 + chunk_at(lane >> 2, lane & 3)) = wv[i];
        wave_sync();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (q + i * 64 >= k64) break;
            v4i &sum = i & 1 ? odd : acc;
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const v4i *>(turn + i * 1024 + chunk_at(r16, quad)),
                                                        *reinterpret_cast<const v4i *>(at + q + i * 64), sum, 0, 0, 0);
        }
    };
#pragma unroll
    for (int i = 0; i < kAhead; i += 4)
        if (i * 64 < k64) four_steps(a + i, i * 64);
    for (int q = kAhead * 64; S > 1 && q < k64; q += 256) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = load_elements<int8_t>(wr + q + i * 64 + part, read - q - i * 64 - part);
        four_steps(a, q);
    }
    acc += odd;
    if (row >= rows) return;
    const float s = ls[r16];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (float)acc[e] * s * sc[e] + bi[e];
    store_vec<T, 4>(y + row * ldy + c, o, n - c);
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

// Eight numbers to three operands of bfloat16 numbers.  Two would be enough for the rounding of a 16-bit result, but not
// for a sum that cancels: what the third holds is up to 2^-16 of every term.
__device__ __forceinline__ void split8(const float (&x)[8], v8b (&out)[3])
{
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float r0 = x[i] - cut8(x[i]), r1 = x[i + 1] - cut8(x[i + 1]);
        const float l0 = r0 - cut8(r0), l1 = r1 - cut8(r1);
        w[0][i / 2] = high_halves(x[i], x[i + 1]);
        w[1][i / 2] = high_halves(r0, r1);
        w[2][i / 2] = high_halves(l0, l1);
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) __builtin_memcpy(&out[q], w[q], 16);
}

// A workgroup's four wavefronts have different rows of the float operand (16 each) and share the integer tile
// (TB blocks of 16 columns).  A lane's operand is eight numbers along the sum, from (lane >> 4) * 8 on, of output index
// lane & 15.  The memory pipeline takes neighbouring lanes' addresses together, so every load and store here gives
// neighbouring lanes neighbouring addresses; what the matrix layout wants otherwise is turned in LDS.
// Output indexes past the matrix's end read its last row or column again (what they give is not stored), so that a step
// of 32 whole indexes of the sum asks nothing; offsets are 32 bits from a uniform base (pitches below 2^22: 128 rows of 4-byte elements).

// Four wavefronts work on a tile together: a team.  Where a workgroup has several, each takes some of the sum's steps.
__device__ __forceinline__ int team_thread() { return threadIdx.x & (kThreads - 1); }

// Weight gradient: the sum runs down the rows of dy; a lane takes eight rows of a column straight into its operand, 16
// lanes 16 neighbouring columns.
template <class T>
struct DownOperand {
    static constexpr int kLds = 0;
    float v[8];
    uint32_t off;
    const T *base;
    int64_t ld;
    __device__ __forceinline__ void place(const T *p, int64_t pitch, int64_t a0, int64_t na)
    {
        const int lane = team_thread() & 63;
        const int64_t aw = min(a0 + __builtin_amdgcn_readfirstlane(team_thread() >> 6) * 16, na - 1);
        base = p + aw;
        ld = pitch;
        off = (uint32_t)(((lane >> 4) * 8 * ld + min(aw + (lane & 15), na - 1) - aw) * sizeof(T));
    }
    __device__ __forceinline__ void load_whole(int64_t r)
    {
        const Buffer p = buffer_at(base + r * ld);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            T t;
            load_at(p, off, (uint32_t)(e * ld * sizeof(T)), t);
            v[e] = (float)t;
        }
    }
    __device__ __forceinline__ void load_part(int64_t r, int left)
    {
        const int k = ((team_thread() & 63) >> 4) * 8;
        const uint32_t a = off - (uint32_t)(k * ld * sizeof(T));                  // the column alone, whatever the pitch
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < left ? (float)*(base + (r + k + e) * ld + a / sizeof(T)) : 0.0f;
    }
    __device__ __forceinline__ void store(int8_t *) const {}
    __device__ __forceinline__ void fetch(const int8_t *, float (&x)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = v[e];
    }
};

// Input gradient: the sum runs along the rows of dy.  A tile of 64 rows x 32 goes through LDS as it is, in chunks of 16
// bytes that sit where eight lanes reading a chunk each of eight rows touch all banks once.
template <class T>
struct AlongOperand {
    static constexpr int E = 16 / (int)sizeof(T), C = 32 / E, N = 64 * C / kThreads, kLds = 64 * C * 16;
    v4i v[N];
    uint32_t off[N];
    const T *base;
    int64_t ld, a0, na;
    __device__ __forceinline__ static int place_of(int row, int chunk)
    {
        return row * (C * 16) + ((chunk ^ (C == 8 ? row & 7 : (row >> 1) & 3)) << 4);
    }
    __device__ __forceinline__ void place(const T *p, int64_t pitch, int64_t first, int64_t rows)
    {
        base = p + first * pitch;
        ld = pitch, a0 = first, na = rows;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int u = team_thread() + n * kThreads;
            off[n] = (uint32_t)((min((int64_t)(u / C), na - 1 - a0) * ld + u % C * E) * sizeof(T));
        }
    }
    __device__ __forceinline__ void load_whole(int64_t r)
    {
        const Buffer p = buffer_at(base + r);
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = load_at16(p, off[n], 0);
    }
    __device__ __forceinline__ void load_part(int64_t r, int left)
    {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int u = team_thread() + n * kThreads, c = u % C * E;
            const T *p = base + min((int64_t)(u / C), na - 1 - a0) * ld + r + c;
            v[n] = load_elements<T>(p, left - c);
        }
    }
    __device__ __forceinline__ void store(int8_t *lds) const
    {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int u = team_thread() + n * kThreads;
            __builtin_memcpy(__builtin_assume_aligned(lds + place_of(u / C, u % C), 16), &v[n], 16);
        }
    }
    __device__ __forceinline__ void fetch(const int8_t *lds, float (&x)[8]) const
    {
        const int lane = team_thread() & 63, row = (team_thread() >> 6) * 16 + (lane & 15);
#pragma unroll
        for (int h = 0; h < 8 / E; ++h) {
            T t[E];
            __builtin_memcpy(t, __builtin_assume_aligned(lds + place_of(row, (lane >> 4) * (8 / E) + h), 16), 16);
#pragma unroll
            for (int e = 0; e < E; ++e) x[h * E + e] = (float)t[e];
        }
    }
};

// The integer operand's tile: BB columns x 32 of the sum, transposed on its way into LDS and made bfloat16 there, once
// for the four wavefronts.  A unit is four columns x four rows of the sum; the lanes of a row of units read neighbouring
// words.  Column 4 q + j of the tile becomes LDS row j * BB / 4 + q: the lanes that write column j of their units then
// write neighbouring rows.  The last columns' unit starts where four are left and shifts them down; units past the end
// read the last ones.  Of a matrix of fewer than four columns a word runs over into the next row, which its last rows
// (those from `spare` on) do not have.
template <int BB>
struct TurnedTile {
    static constexpr int Q = BB / 4, N = (BB * 2 + kThreads - 1) / kThreads;
    uint32_t v[N][4], off[N];
    int shift;
    __device__ __forceinline__ bool idle() const { return BB * 2 < kThreads && team_thread() >= BB * 2; }
    // The tile's first column in a matrix of nb, and where the whole words' base column is: `before` columns ahead of it.
    __device__ __forceinline__ void place(int64_t ld, int b0, int nb, int &before)
    {
        const int last = max(nb - 4, 0), base = min(b0, last), b = b0 + team_thread() % Q * 4, c = min(b, last) - base;
        before = b0 - base;
        shift = min(b - base - c, 3) * 8;
#pragma unroll
        for (int n = 0; n < N; ++n) off[n] = (uint32_t)((team_thread() + n * kThreads) / Q * 4 * ld + c);
    }
    __device__ __forceinline__ void load_whole(const int8_t *base, int64_t ld)
    {
        if (idle()) return;
        const Buffer p = buffer_at(base);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < N; ++n) load_at(p, off[n], (uint32_t)(i * ld), v[n][i]);
    }
    __device__ __forceinline__ void load_part(const int8_t *base, int64_t ld, int cols, int left)
    {
        if (idle()) return;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int b = team_thread() % Q * 4, r = (team_thread() + n * kThreads) / Q * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[1];
                load_bytes<4>(w, base + (int64_t)(r + i) * ld + b, r + i < left ? cols - b : 0);
                v[n][i] = w[0] << shift;                             // store() takes it back
            }
        }
    }
    __device__ __forceinline__ void store(int8_t *lds) const
    {
        if (idle()) return;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int q = team_thread() % Q, r = (team_thread() + n * kThreads) / Q;
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = v[n][i] >> shift;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t w[2] = {high_halves(code_value(x[0], j), code_value(x[1], j)), high_halves(code_value(x[2], j), code_value(x[3], j))};
                __builtin_memcpy(__builtin_assume_aligned(lds + chunk_at(j * Q + q, r >> 1) + (r & 1) * 8, 8), w, 8);
            }
        }
    }
};

// out[a, b] over 64 x 16 TB values from (a0, b0) on, the sum over [r0, r1) in steps of 32, which the teams take in turn.
// kSums: the float operand's own sums over [r0, r1), in 64 bits, go to `piece` as they are or to `sums` rounded once
// (nowhere if both are null).  Every tile adds them, beside its matrix instructions and without a branch: 1 % of a call
// more than float32 sums took (left to the one tile that stores them 2 to 6 %, the branch keeps loads and sums apart).
template <class T, bool kDown, int TB, int kTeams, class TO, bool kSums>
__device__ __forceinline__ void split_tile(const T *dy, int64_t ldd, const float *scale, const int8_t *q, int64_t ldq,
                                           int64_t spare, int64_t a0, int64_t na, int b0, int nb, int64_t r0, int64_t r1,
                                           TO *out, int64_t ldo, double *piece, float *sums)
{
    typedef typename std::conditional<kDown, DownOperand<T>, AlongOperand<T>>::type Operand;
    constexpr int BB = 16 * TB, kB = BB * 64, kS = 128, kStage = Operand::kLds + kB + kS;
    constexpr int kPitch = BB * 4 + 16, kTurn = 4 * 16 * kPitch;      // the results' way out
    constexpr int kTeam = kTurn > 2 * kStage ? kTurn : 2 * kStage;
    __shared__ __attribute__((aligned(16))) int8_t all[kTeams * kTeam];
    const int thread = team_thread(), team = kTeams > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads) : 0;
    const int lane = thread & 63, wave = thread >> 6;
    int8_t *lds = all + team * kTeam;
    v4f acc[TB];
#pragma unroll
    for (int i = 0; i < TB; ++i) acc[i] = v4f{0, 0, 0, 0};
    Operand fa;
    TurnedTile<BB> tb;
    float scale_v = 0.0f;
    double col = 0.0;
    fa.place(dy, ldd, a0, na);
    int before;
    tb.place(ldq, b0, nb, before);
    const int8_t *pb = q + b0;
    const bool near = ldd < (1 << 22) && ldq < (1 << 22);
    const auto store = [&](int8_t *stage) {
        fa.store(stage);
        tb.store(stage + Operand::kLds);
        if (thread < 32) reinterpret_cast<float *>(stage + Operand::kLds + kB)[thread] = scale_v;
    };
    // the stage's float operand, scaled and split
    const auto split = [&](const int8_t *stage, v8b (&a)[3], float (&x)[8]) {
        float s[8];
        fa.fetch(stage, x);
        __builtin_memcpy(s, __builtin_assume_aligned(stage + Operand::kLds + kB + (lane >> 4) * 32, 16), 32);
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = x[e] * s[e];
        split8(t, a);
    };
    const auto multiply = [&](const int8_t *stage, const v8b (&a)[3], const float (&x)[8]) {
        if constexpr (kSums) {
            double d[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = (double)x[e];
            col += ((d[0] + d[1]) + (d[2] + d[3])) + ((d[4] + d[5]) + (d[6] + d[7]));
        }
        // four blocks of columns at a time: an accumulator comes round again after four instructions, not at once
#pragma unroll
        for (int i = 0; i < TB; i += 4) {
            v8b b[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) b[c] = *reinterpret_cast<const v8b *>(stage + Operand::kLds + chunk_at((i + c) * 16 + (lane & 15), lane >> 4));
#pragma unroll
            for (int p = 2; p >= 0; --p)                              // small pieces first
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[c], a[p], acc[i + c], 0, 0, 0);
        }
    };
    // up to here: steps that ask nothing, loaded one ahead
    const int64_t whole = near ? r0 + max((int64_t)0, (nb < 4 ? min(r1, spare) : r1) - r0) / 32 * 32 : r0;
    constexpr int kRound = 32 * kTeams;
    if (r0 < whole) {
        const auto load = [&](int64_t x) {
            fa.load_whole(x);
            tb.load_whole(pb - before + x * ldq, ldq);
            if (thread < 32) scale_v = scale[x + thread];
        };
        int64_t r = r0 + team * 32;
        int at = 0;
        if (kTeams == 1 || r < whole) {
            load(r);
            store(lds);
        }
        __syncthreads();
        for (int64_t round = r0; round < whole; round += kRound, r += kRound, at ^= 1) {
            const int8_t *stage = lds + at * kStage;
            v8b a[3];
            float x[8];
            const bool on = kTeams == 1 || r < whole, more = r + kRound < whole;
            if (on) split(stage, a, x);
            if (more) load(r + kRound);
            if (on) multiply(stage, a, x);
            // the other stage was read in the round before, and every wavefront has passed the barrier since
            if (more) store(lds + (at ^ 1) * kStage);
            __syncthreads();
        }
    }
    for (int64_t round = whole; round < r1; round += kRound) {
        const int64_t r = round + team * 32;
        const int left = (int)max((int64_t)0, min((int64_t)32, r1 - r));
        fa.load_part(r, left);
        tb.load_part(pb + r * ldq, ldq, nb - b0, left);
        if (thread < 32) scale_v = thread < left ? scale[r + thread] : 0.0f;
        store(lds);
        __syncthreads();
        if (left > 0) {
            v8b a[3];
            float x[8];
            split(lds, a, x);
            multiply(lds, a, x);
        }
        __syncthreads();
    }
    if constexpr (kTeams > 1) {                                       // the teams' sums, added in order
        static_assert(!kSums, "the rows' own sums stay with one team");
        v4f *sums_of = reinterpret_cast<v4f *>(lds);
#pragma unroll
        for (int i = 0; i < TB; ++i)
            if (team > 0) sums_of[i * kThreads + thread] = acc[i];
        __syncthreads();
        if (team > 0) return;
#pragma unroll
        for (int o = 1; o < kTeams; ++o)
#pragma unroll
            for (int i = 0; i < TB; ++i) acc[i] += reinterpret_cast<const v4f *>(all + o * kTeam)[i * kThreads + thread];
    }
    // A lane's four rows of LDS order j * BB / 4 + q are four neighbouring columns of the result; through LDS neighbouring
    // lanes get neighbouring columns of a row.
    constexpr int H = TB / 4;
    int8_t *turn = lds + wave * 16 * kPitch;
    const int64_t first = a0 + wave * 16;
    if (kSums && (piece || sums)) {
        col += __shfl_xor(col, 16);
        col += __shfl_xor(col, 32);
        if (lane < 16 && first + lane < na) {
            if (piece) piece[first + lane] = col;
            else sums[first + lane] = (float)col;
        }
    }
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v4f o = {acc[h][e], acc[H + h][e], acc[2 * H + h][e], acc[3 * H + h][e]};
            *reinterpret_cast<v4f *>(turn + (lane & 15) * kPitch + (h * 16 + (lane >> 4) * 4 + e) * 16) = o;
        }
    wave_sync();
#pragma unroll
    for (int i = 0; i < TB; ++i) {
        const int u = i * 64 + lane, row = u / (BB / 4), b = u % (BB / 4) * 4;
        float o[4];
        __builtin_memcpy(o, __builtin_assume_aligned(turn + row * kPitch + b * 4, 16), 16);
        if (first + row < na && b0 + b < nb) store_vec<TO, 4>(out + (first + row) * ldo + b0 + b, o, nb - b0 - b);
    }
}

// Weight gradient: workgroup (tile of dw, piece of the rows).  The pieces' results are added by k_add_pieces in a fixed
// order (no atomics: the same bits on every run).  1024 x 512 weights from 10816 rows: 41 us (34 GFLOP as three bfloat16
// products, 0.82 PFLOP/s) and 7.3 us for the pieces; 128 x 64 from 692224 rows: 57 us (269 MB, 4.7 TB/s) and 7.4 us, from
// bfloat16 rows 63 us (180 MB: not bound by memory).
template <class T, int TB>
__global__ __launch_bounds__(kThreads, 2) void k_weight_grad(const T *dy, int64_t ldd, const int8_t *codes, int64_t ldc, const float *scale,
                                                             int64_t spare, int64_t rows, int n, int k, int64_t rows_per_piece, int tiles_k, int tiles,
                                                             float *dw, float *db, double *db_pieces)
{
    const uint32_t id = (uint32_t)xcd_run(blockIdx.x, gridDim.x);
    const int64_t piece = id / (uint32_t)tiles;
    const int tile = (int)(id % (uint32_t)tiles), a0 = tile / tiles_k * 64, b0 = tile % tiles_k * 16 * TB;
    const int64_t r0 = piece * rows_per_piece, r1 = min(rows, r0 + rows_per_piece);
    split_tile<T, true, TB, 1, float, true>(dy, ldd, scale, codes, ldc, spare, a0, n, b0, k, r0, r1, dw + piece * ((int64_t)n * k), k,
                                            db_pieces && b0 == 0 ? db_pieces + piece * n : nullptr, db && b0 == 0 ? db : nullptr);
}

// Sums over the pieces in 64 bits: the first `cut` of `count` values are dw, from float32 pieces, the others db, from pieces
// of 64 bits.  A workgroup takes `wide` values; its 256 / wide groups of threads add pieces in turn, and their sums are
// added in order.
__global__ __launch_bounds__(kThreads) void k_add_pieces(const float *dw_pieces, const double *db_pieces, int pieces, int64_t count, int64_t cut,
                                                         int wide, float *dw, float *db)
{
    __shared__ double buf[kThreads];
    const int col = threadIdx.x & (wide - 1), group = threadIdx.x / wide, groups = kThreads / wide;
    const int64_t i = (int64_t)(gridDim.x - 1 - blockIdx.x) * wide + col;      // db's few first, under dw's
    double s = 0.0;
    if (i < cut) {
#pragma unroll 8
        for (int p = group; p < pieces; p += groups) s += (double)dw_pieces[p * cut + i];
    } else if (i < count) {
#pragma unroll 8
        for (int p = group; p < pieces; p += groups) s += db_pieces[p * (count - cut) + i - cut];
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

// Input gradient: workgroup (64 rows, 16 TB columns), the whole sum over the output channels.  Bound by the matrix
// instructions and the vector instructions beside them: 43264 rows, 256 -> 512 in float32 43 us (34 GFLOP as three bfloat16
// products: 0.79 PFLOP/s; the memory's share is 26 us; 48 us a call back to back), 21632 rows, 255 -> 128 13.3 us
// (2.5 TB/s); in bfloat16 39.5 and 11.9 us.
template <class T, int TB, int kTeams>
__global__ __launch_bounds__(kThreads * kTeams, kTeams > 1 ? 1 : 3) void k_input_grad(const T *dy, int64_t ldd, const int8_t *w, int64_t ldw, const float *ws,
                                                            int64_t spare, int64_t rows, int n, int k, int tiles_k, T *dx, int64_t lddx)
{
    const uint32_t tile = (uint32_t)xcd_run(blockIdx.x, gridDim.x);
    split_tile<T, false, TB, kTeams, T, false>(dy, ldd, ws, w, ldw, spare, (int64_t)(tile / (uint32_t)tiles_k) * 64, rows, (int)(tile % (uint32_t)tiles_k) * 16 * TB, k,
                                                                   0, n, dx, lddx, nullptr, nullptr);
}

// Tiles of 64 x 16 tb values.  The widest reads and splits the float operand least often, which pays where each of 512
// workgroups has 16 steps of 32 rows and more and the tiles are filled (1024 x 512 weights from 10816 rows: 48 us in all
// with tb = 16, 53 with 8; from 2704 rows 512 x 256: 17.7 and 16.3; 384 x 255 from 43264 rows: 43.9 and 41.6).
struct GradPlan { int tb, tiles_k, tiles, pieces; int64_t rows_per_piece; };
GradPlan plan_weight_grad(int64_t rows, int n, int k)
{
    GradPlan p;
    const int64_t steps = (rows + 31) / 32, wide = (k + 255) / 256;
    p.tb = k <= 64 ? 4 : wide * 256 <= k + k / 4 && steps * ((n + 63) / 64) * wide >= 16 * 512 ? 16 : 8;
    p.tiles_k = (k + 16 * p.tb - 1) / (16 * p.tb);
    p.tiles = (n + 63) / 64 * p.tiles_k;
    // two workgroups a compute unit, each with at least four steps of 32 rows: more pieces cost more in k_add_pieces than
    // they win (692224 rows, 64 x 128: 64 us in all with 512 workgroups, 65 with 768, 69 with 1024)
    const int64_t want = std::max(1, 512 / p.tiles);
    const int64_t pieces = std::max<int64_t>(1, std::min(want, (steps + 3) / 4));
    p.rows_per_piece = (steps + pieces - 1) / pieces * 32;
    p.pieces = (int)((rows + p.rows_per_piece - 1) / p.rows_per_piece);
    return p;
}

unsigned blocks_for(int64_t count) { return (unsigned)((count + kThreads - 1) / kThreads); }

// How a product is computed.  All three give the same bits: the sums are whole numbers.
struct ProductPlan {
    enum { kTile, kRows, kFew } how;
    int lanes;                                           // kRows: of a row
    size_t lds;
};
ProductPlan plan_product(int64_t rows, int k, int n, int x_type)
{
    ProductPlan p{};
    const int k64 = (k + 63) / 64 * 64, n64 = (n + 63) / 64 * 64, V = x_type == YH_INT8 ? 16 : x_type == YH_FLOAT32 ? 4 : 8;
    const size_t pitch = k64 + 16, wave = 16 * pitch + 16 * kOutPitch + 64;
    // Up to two workgroups of 16 rows x 64 channels a compute unit: 828 rows, 1024 -> 512 take 8 us so, 12 us by tiles;
    // 3000 rows, with six rounds of workgroups, 25 and 15.
    if ((rows + 15) / 16 * (n64 / 64) <= 512 && 16 * pitch + 64 <= 64 * 1024) {
        p.how = ProductPlan::kFew;
        p.lds = 4 * 4096 + 16 * pitch + 64;
        return p;
    }
    // Rows of up to 1024 bytes and weights that leave LDS room for eight wavefronts' rows; with longer rows (512 -> 128:
    // 37 us by 16 rows, 31 by tiles) or with the weights in two halves the codes are better taken once, into memory.  Every
    // workgroup loads the weights first, which pays from four blocks of 16 rows a compute unit on (256 -> 128: 6000 rows 11.5
    // us so, 8.4 by tiles; 24000 rows 15.9 both; 100000 rows 37.6 and 41.2), with 8 KiB of weights always (32 -> 64, 6000
    // rows: 5.4 and 6.2 us).
    p.lds = n64 * (pitch + 8) + kRowWaves * wave;
    if (k64 <= 64 * V && p.lds <= 160 * 1024 && (rows >= 16384 || n64 * k64 <= 8192)) {
        p.how = ProductPlan::kRows;
        p.lanes = std::max(4, pow2_at_least((k64 / V + 3) / 4));
        return p;
    }
    p.how = ProductPlan::kTile;
    return p;
}

template <class TX, class T, bool kWhole>
void run_few(const ProductPlan &p, const TX *x, int64_t ldx, const float *xs, int64_t rows, int k, const int8_t *w, int64_t ldw, const float *ws,
             int n, const float *bias, T *y, int64_t ldy, int8_t *codes, int64_t ldc, float *scale, hipStream_t st)
{
    const int64_t spare = spare_rows(rows, ldx, 16 / (int)sizeof(TX));
#define CALL(S)                                                                                                             \
    k_int8_few<TX, T, S, kWhole><<<dim3((unsigned)((rows + 15) / 16), (n + 63) / 64), kThreads, p.lds, st>>>(               \
        x, ldx, spare, xs, rows, k, w, ldw, spare_rows(n, ldw, 16), ws, n, bias, y, ldy, codes, ldc, scale)
    if (k <= 256) CALL(1);
    else CALL(4);
#undef CALL
}

template <class TX, class T, bool kWhole>
void run_rows(const ProductPlan &p, const TX *x, int64_t ldx, const float *xs, int64_t rows, int k, const int8_t *w, int64_t ldw, const float *ws,
              int n, const float *bias, T *y, int64_t ldy, int8_t *codes, int64_t ldc, float *scale, hipStream_t st)
{
    // as many workgroups as the compute units hold at once, or as there are rows for
    const int64_t held = 256 * (int64_t)(160 * 1024 / p.lds), asked = (rows + 16 * kRowWaves - 1) / (16 * kRowWaves);
    const unsigned blocks = (unsigned)std::min(held, asked);
#define CALL(G) k_int8_rows<TX, T, G, kWhole><<<dim3(blocks), 64 * kRowWaves, p.lds, st>>>(x, ldx, xs, rows, k, p.lanes, w, ldw, ws, n, bias, y, ldy, codes, ldc, scale)
    if (p.lanes <= 4) CALL(1);
    else if (p.lanes <= 8) CALL(2);
    else CALL(4);
#undef CALL
}

}  // namespace

bool product_needs_codes(int64_t rows, int32_t k, int32_t n, int32_t x_type)
{
    return x_type != YH_INT8 && plan_product(rows, k, n, x_type).how == ProductPlan::kTile;
}

hipError_t launch_int8_product(const Rows &x, const float *x_scale, int64_t rows, int32_t k,
                               const int8_t *w, int64_t ldw, const float *w_scale, int32_t n, const float *bias,
                               void *y, int64_t ldy, int32_t type, int8_t *codes, int64_t ldc, float *scale, hipStream_t st)
{
    const ProductPlan p = plan_product(rows, k, n, x.type);
    if (p.how != ProductPlan::kTile) {
        with_type(type, [&](auto t) {
            using T = decltype(t);
            const auto go = [&](auto tx) {
                using TX = decltype(tx);
                const auto call = p.how == ProductPlan::kRows ? (k % 16 ? run_rows<TX, T, false> : run_rows<TX, T, true>)
                                                              : (k % 16 ? run_few<TX, T, false> : run_few<TX, T, true>);
                call(p, static_cast<const TX *>(x.p), x.ld, x_scale, rows, k, w, ldw, w_scale, n, bias, static_cast<T *>(y), ldy, codes, ldc, scale, st);
            };
            if (x.type == YH_INT8) go((int8_t)0);
            else with_type(x.type, go);
        });
        return hipGetLastError();
    }
    const int8_t *q = static_cast<const int8_t *>(x.p);
    int64_t ldq = x.ld;
    if (x.type != YH_INT8) {
        const hipError_t e = launch_quantize(x, rows, k, codes, ldc, scale, st);
        if (e != hipSuccess) return e;
        q = codes, ldq = ldc, x_scale = scale;
    }
    with_type(type, [&](auto t) {
        using T = decltype(t);
#define CALL(BM, BN)                                                                                                        \
        do {                                                                                                                \
            const int tn = (n + BN - 1) / BN;                                                                               \
            k_int8_tile<T, BM, BN><<<dim3((unsigned)((rows + BM - 1) / BM * tn)), kThreads, 0, st>>>(                       \
                q, ldq, x_scale, rows, k, w, ldw, w_scale, n, bias, static_cast<T *>(y), ldy, tn);                          \
        } while (0)
        // large tiles where they fill the card, small ones where there are few rows (1024 -> 512 in codes: 21632 rows 22.4 us
        // large, 29.5 small; 5408 rows 13.3 and 11.5)
        if ((rows + 127) / 128 * ((n + 127) / 128) >= 256) CALL(128, 128);
        else CALL(64, 64);
#undef CALL
    });
    return hipGetLastError();
}

size_t weight_grad_workspace(int64_t rows, int32_t n, int32_t k)
{
    if (rows == 0) return 0;
    const GradPlan p = plan_weight_grad(rows, n, k);
    return p.pieces > 1 ? (size_t)p.pieces * ((size_t)n * k * sizeof(float) + n * sizeof(double)) : 0;
}

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
    // in the workspace: db's pieces (64 bits), then dw's
    double *pb = p.pieces > 1 && db ? static_cast<double *>(workspace) : nullptr;
    float *pw = p.pieces > 1 ? reinterpret_cast<float *>(static_cast<double *>(workspace) + (int64_t)p.pieces * n) : dw;
    with_type(dy.type, [&](auto t) {
        using T = decltype(t);
#define CALL(TB) k_weight_grad<T, TB><<<dim3((unsigned)(p.tiles * p.pieces)), kThreads, 0, st>>>(                           \
            static_cast<const T *>(dy.p), dy.ld, codes, ldc, scale, spare_rows(rows, ldc, 4), rows, n, k, p.rows_per_piece, p.tiles_k, p.tiles, pw, db, pb)
        if (p.tb == 4) CALL(4);
        else if (p.tb == 8) CALL(8);
        else CALL(16);
#undef CALL
    });
    if (p.pieces > 1) {
        // A thread a value where that gives 512 workgroups (512 x 256 weights from 43264 rows, 64 pieces: 45.9 us in all, 47.9
        // with eight threads a value); otherwise several threads a value, down to 16 neighbouring values (64 bytes) a
        // workgroup (128 x 64 weights from 692224 rows, 512 pieces: 63 us, 81 with a thread a value).
        const int64_t values = db ? count + n : count;
        int wide = kThreads;
        while (wide > 16 && values / wide < 512 && kThreads / wide < p.pieces) wide /= 2;
        k_add_pieces<<<dim3((unsigned)((values + wide - 1) / wide)), kThreads, 0, st>>>(pw, pb, p.pieces, values, count, wide, dw, db);
    }
    return hipGetLastError();
}

hipError_t launch_input_grad(const Rows &dy, const int8_t *w, int64_t ldw, const float *w_scale, int64_t rows,
                             int32_t n, int32_t k, void *dx, int64_t lddx, hipStream_t st)
{
    with_type(dy.type, [&](auto t) {
        using T = decltype(t);
#define CALL(TB, TEAMS)                                                                                                     \
        do {                                                                                                                \
            const int tk = (k + 16 * TB - 1) / (16 * TB);                                                                   \
            k_input_grad<T, TB, TEAMS><<<dim3((unsigned)((rows + 63) / 64 * tk)), kThreads * TEAMS, 0, st>>>(               \
                static_cast<const T *>(dy.p), dy.ld, w, ldw, w_scale, spare_rows(n, ldw, 4), rows, n, k, tk, static_cast<T *>(dx), lddx);          \
        } while (0)
        // Tiles of 64 x 128 (43264 rows, 256 -> 512: 64 x 256 takes 1.12 times as long, 64 x 64 1.27 times); half as wide where that gives
        // too few workgroups, and with the sum over four teams where even so they are few and the sum is long (169 rows,
        // 512 -> 1024, 48 workgroups: 8.2 us, 11.4 with one team; 32000 rows, 255 -> 60, 500 workgroups: 17.0 and 12.4; 2704
        // rows, 128 -> 256, four steps: 5.6 and 5.3).
        if (k > 64 && (rows + 63) / 64 * ((k + 127) / 128) >= 256) CALL(8, 1);
        else if ((rows + 63) / 64 * ((k + 63) / 64) <= 256 && n > 160) CALL(4, 4);
        else CALL(4, 1);
#undef CALL
    });
    return hipGetLastError();
}

}  // namespace yh
