// Row operators in 8 bits: declarations shared by their kernels and their C-ABI layer, and the device
// helpers for rows of float32 / bfloat16 / float16 whose length and pitch are arbitrary.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "yolohead.h"

namespace yh {

// yh_abi.hip: stores the thread's error message and returns `code`; looks for a HIP device.
int report(int code, const char *fmt, ...);
int report_hip(hipError_t e, const char *what);
int require_device();

// ---- what the launchers take --------------------------------------------
struct Rows {            // a matrix of rows: `ld` elements from one row to the next
    const void *p;
    int64_t ld;
    int32_t type;        // yh_dtype
};

hipError_t launch_quantize(const Rows &x, int64_t rows, int32_t cols, int8_t *codes, int64_t ldc, float *scale, hipStream_t st);
hipError_t launch_dequantize(const int8_t *codes, int64_t ldc, const float *scale, int64_t rows, int32_t cols,
                             void *out, int64_t ldo, int32_t type, hipStream_t st);

int norm_blocks(int64_t rows, int32_t cols, int32_t type);      // blocks per channel slab of the reductions
hipError_t launch_norm_forward(const Rows &z, const Rows &res, int64_t rows, int32_t cols, const float *gamma, const float *beta,
                               double eps, float slope, void *a, int64_t lda, int8_t *kept, int64_t ldk, float *scale,
                               float *mean, float *invstd, float *running_mean, float *running_var, double momentum,
                               void *workspace, hipStream_t st);
hipError_t launch_norm_backward(const Rows &da, int64_t rows, int32_t cols, const int8_t *kept, int64_t ldk, const float *scale,
                                const float *gamma, const float *invstd, float slope, void *dz, int64_t lddz,
                                float *dgamma, float *dbeta, void *workspace, hipStream_t st);

// codes, scale: where the codes of a float x are left; null if nobody wants them and product_needs_codes() says no.
bool product_needs_codes(int64_t rows, int32_t k, int32_t n, int32_t x_type);
hipError_t launch_int8_product(const Rows &x, const float *x_scale, int64_t rows, int32_t k,
                               const int8_t *w, int64_t ldw, const float *w_scale, int32_t n, const float *bias,
                               void *y, int64_t ldy, int32_t type, int8_t *codes, int64_t ldc, float *scale, hipStream_t st);

size_t weight_grad_workspace(int64_t rows, int32_t n, int32_t k);     // bytes
hipError_t launch_weight_grad(const Rows &dy, const int8_t *codes, int64_t ldc, const float *scale, int64_t rows,
                              int32_t n, int32_t k, float *dw, float *db, void *workspace, hipStream_t st);
hipError_t launch_input_grad(const Rows &dy, const int8_t *w, int64_t ldw, const float *w_scale, int64_t rows,
                             int32_t n, int32_t k, void *dx, int64_t lddx, hipStream_t st);

// ---- for the launchers ---------------------------------------------------
inline int pow2_at_least(int v)
{
    int p = 1;
    while (p < v) p <<= 1;
    return p;
}

// Calls f(T()) with the C++ type of a yh_dtype.
template <class F>
void with_type(int32_t type, F f)
{
    if (type == YH_FLOAT32) f(float());
    else if (type == YH_BFLOAT16) f((__bf16)0.0f);
    else f((_Float16)0.0f);
}

// ---- device helpers ------------------------------------------------------
constexpr float kRowMin = 0x1p-110f;      // a row whose largest value is below this is zero: its scale stays a normal number
constexpr int kCodeMax = 127;             // row codes: -127 .. 127
constexpr int kKeptMax = 63;              // norm checkpoint: seven bits beside the sign of the activation's input

template <class T> struct RowVec { static constexpr int V = 16 / (int)sizeof(T); };   // elements of a 16-byte access

// Vectors that may stand at any element (global memory on gfx950 takes unaligned accesses).  As vector types they stay
// one access each: an element-wise copy is taken apart and partly shared with the code for a row's end.
template <class T, int V> struct Loose { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)), may_alias)); };
template <int B> struct LooseBytes { typedef uint32_t type __attribute__((ext_vector_type(B / 4), aligned(1), may_alias)); };
template <> struct LooseBytes<4> { typedef uint32_t type __attribute__((aligned(1), may_alias)); };
template <> struct LooseBytes<2> { typedef uint16_t type __attribute__((aligned(1), may_alias)); };

template <int B>
__device__ __forceinline__ typename LooseBytes<B>::type loose_load(const uint8_t *p) { return *reinterpret_cast<const typename LooseBytes<B>::type *>(p); }
template <int B>
__device__ __forceinline__ void loose_store(uint8_t *p, typename LooseBytes<B>::type v) { *reinterpret_cast<typename LooseBytes<B>::type *>(p) = v; }

// A row's end: `bytes` of it (0 < bytes < 4 W, whole elements of E bytes) as words, zeros behind.  One access a bit of
// `bytes`, all under way together (element by element, each under a condition of its own, a lane's end took as long as
// all the rest of a short call).
template <int E, int W>
__device__ __forceinline__ void load_end(uint32_t (&w)[W], const void *from, int bytes)
{
    const uint8_t *p = static_cast<const uint8_t *>(from);
    uint32_t a[2] = {0, 0}, b = 0, c = 0, d = 0;
    if (W > 2 && (bytes & 8)) {
        const LooseBytes<8>::type t = loose_load<8>(p);
        a[0] = t[0], a[1] = t[1];
    }
    if (W > 1 && (bytes & 4)) b = loose_load<4>(p + (bytes & 8));
    if (E <= 2 && (bytes & 2)) c = loose_load<2>(p + (bytes & 12));
    if (E <= 1 && (bytes & 1)) d = p[bytes & 14];
    c |= d << ((bytes & 2) * 8);
    const uint32_t lo = bytes & 4 ? b : c, hi = bytes & 4 ? c : 0;
    const bool far = bytes & 8;
    w[0] = far ? a[0] : lo;
    if constexpr (W > 1) w[1] = far ? a[1] : hi;
    if constexpr (W > 2) w[2] = far ? lo : 0, w[3] = far ? hi : 0;
}
template <int E, int W>
__device__ __forceinline__ void store_end(void *to, const uint32_t (&w)[W], int bytes)
{
    uint8_t *p = static_cast<uint8_t *>(to);
    uint32_t lo = w[0], hi = W > 1 ? w[W > 1 ? 1 : 0] : 0;
    if constexpr (W > 2) {
        if (bytes & 8) {
            loose_store<8>(p, LooseBytes<8>::type{w[0], w[1]});
            lo = w[2], hi = w[3];
        }
    }
    if (W > 1 && (bytes & 4)) loose_store<4>(p + (bytes & 8), lo);
    const uint32_t c = bytes & 4 ? hi : lo;
    if (E <= 2 && (bytes & 2)) loose_store<2>(p + (bytes & 12), (uint16_t)c);
    if (E <= 1 && (bytes & 1)) p[bytes & 14] = (uint8_t)(c >> ((bytes & 2) * 8));
}

// `left` elements of a row from p on, as float32; what lies behind the row's end is not read and comes back zero.
// The address is aligned to an element only: rows of odd length start anywhere.
template <class T, int V>
__device__ __forceinline__ void load_vec(float (&out)[V], const T *p, int left)
{
    constexpr int W = V * (int)sizeof(T) / 4;
    if constexpr (W > 4) {
        float lo[V / 2], hi[V / 2];
        load_vec<T, V / 2>(lo, p, left);
        load_vec<T, V / 2>(hi, p + V / 2, left - V / 2);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) out[i] = lo[i], out[V / 2 + i] = hi[i];
    } else if (left >= V) {
        const typename Loose<T, V>::type t = *reinterpret_cast<const typename Loose<T, V>::type *>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = (float)t[i];
    } else {
        uint32_t w[W] = {};
        if (left > 0) load_end<sizeof(T), W>(w, p, left * (int)sizeof(T));
        T t[V];
        __builtin_memcpy(t, w, 4 * W);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = (float)t[i];
    }
}

// One rounding, to nearest even, of a float32 result to the row's type.
template <class T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[V], int left)
{
    constexpr int W = V * (int)sizeof(T) / 4;
    typename Loose<T, V>::type t;
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = (T)v[i];
    if (left >= V) {
        *reinterpret_cast<typename Loose<T, V>::type *>(p) = t;
    } else if (left > 0) {
        uint32_t w[W];
        __builtin_memcpy(w, &t, 4 * W);
        store_end<sizeof(T), W>(p, w, left * (int)sizeof(T));
    }
}

template <int V>
__device__ __forceinline__ void store_bytes(int8_t *p, const uint32_t (&w)[V / 4], int left)
{
    if (left >= V) {
        typename LooseBytes<V>::type t;
        __builtin_memcpy(&t, w, V);
        *reinterpret_cast<typename LooseBytes<V>::type *>(p) = t;
    } else if (left > 0) {
        store_end<1, V / 4>(p, w, left);
    }
}

template <int V>
__device__ __forceinline__ void load_bytes(uint32_t (&w)[V / 4], const int8_t *p, int left)
{
    if (left >= V) {
        const typename LooseBytes<V>::type t = *reinterpret_cast<const typename LooseBytes<V>::type *>(p);
        __builtin_memcpy(w, &t, V);
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) w[i] = 0;
        if (left > 0) load_end<1, V / 4>(w, p, left);
    }
}

// Rows of a matrix, from the first on, in which a vector of V elements that begins inside of the row may be read whole: it
// runs over into the pitch or the next rows, and the matrix goes on for as long.
inline int64_t spare_rows(int64_t rows, int64_t ld, int V) { return ld > 0 ? rows - (V - 2 + ld) / ld : 0; }
// Elements that may be read from column c on, of a row of `cols`; those beyond `cols` are somebody else's.
__device__ __forceinline__ int left_of(int64_t row, int64_t rows, int64_t spare, int cols, int c, int V)
{
    return row >= rows ? 0 : (row < spare ? (cols + V - 1) & -V : cols) - c;
}

__device__ __forceinline__ float code_value(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

// Round-half-even of the exact product x * r, |x * r| <= 127.0001: the fused multiply-add rounds once, to the unit of
// 1.5 * 2^23, so the whole number sits in the sum's low byte as two's complement.
__device__ __forceinline__ uint32_t code_bits(float x, float r) { return __float_as_uint(__builtin_fmaf(x, r, 12582912.0f)); }

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    // v_perm_b32: bytes 0..3 are the second operand's, 4..7 the first's
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return lo | hi;
}

// f over the `lanes` (a power of two) neighbouring lanes of a group, the result in all of them; the whole wavefront takes
// part.  Up to 16 lanes by data-parallel moves inside the vector unit, beyond by LDS permutes.
template <class F>
__device__ __forceinline__ uint32_t over_lanes(uint32_t m, int lanes, F f)
{
    if (lanes > 1) m = f(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));    // lane ^ 1
    if (lanes > 2) m = f(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));    // lane ^ 2
    if (lanes > 4) m = f(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, true));   // mirrored in eight
    if (lanes > 8) m = f(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xf, 0xf, true));   // mirrored in sixteen
    if (lanes > 16) m = f(m, (uint32_t)__shfl_xor((int)m, 16));
    if (lanes > 32) m = f(m, (uint32_t)__shfl_xor((int)m, 32));
    return m;
}

// Largest |value| bits of a row.  Magnitudes are compared as integers: every NaN is above infinity, infinity above every
// number.
__device__ __forceinline__ uint32_t row_max(uint32_t m, int lanes)
{
    return over_lanes(m, lanes, [](uint32_t a, uint32_t b) { return max(a, b); });
}

struct RowScale { float r, s; bool live; };
// r = levels / max, s = max / levels.  A row with an infinity or a NaN gets the scale NaN, so that everything computed
// from it is NaN; a row that is zero (or below kRowMin) the scale 0; both have codes 0.
__device__ __forceinline__ RowScale row_scale(uint32_t m, float levels)
{
    const float top = __uint_as_float(m);
    RowScale k;
    k.live = m < 0x7f800000u && top >= kRowMin;
    k.r = k.live ? levels / top : 0.0f;
    k.s = k.live ? top / levels : (m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : 0.0f);
    return k;
}

}  // namespace yh
