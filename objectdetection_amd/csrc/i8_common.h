// i8_common.h -- pieces shared by the 8-bit integer kernels (quantize.hip, linear_i8.hip).
#pragma once
#include "common.h"
#include <hip/hip_fp16.h>

// Element types of the entry points (frcnn_hip.h: FRCNN_F32 / FRCNN_BF16 / FRCNN_F16) as C++ types.
template <int T> struct I8Type;
template <> struct I8Type<FRCNN_F32> { typedef float type; };
template <> struct I8Type<FRCNN_BF16> { typedef __bf16 type; };
template <> struct I8Type<FRCNN_F16> { typedef _Float16 type; };

static inline int i8_type_bytes(int t) { return t == FRCNN_F32 ? 4 : 2; }
static inline bool i8_type_ok(int t) { return t == FRCNN_F32 || t == FRCNN_BF16 || t == FRCNN_F16; }

// V elements from an address that is aligned to one element only (rows of an odd length, views): the target reads
// such addresses with the same wide loads.
template <typename T, int V> struct I8Vec { T v[V]; };
template <typename T, int V> __device__ __forceinline__ I8Vec<T, V> i8_load(const T *p)
{
    I8Vec<T, V> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}

// Rows that a call works on: the device-side count where the caller has one (no host read), else all of them.
__device__ __forceinline__ int i8_rows(const int32_t *n_rows, int M)
{
    if (!n_rows) return M;
    const int n = *n_rows;
    return n < 0 ? 0 : (n < M ? n : M);
}

// ---- the row quantiser's arithmetic ----------------------------------------------------------------------------------
// top = max_k |x_k|; scale = top / 127 (fp32); code_k = the whole number nearest to the EXACT quotient 127 x_k / top, ties to
// even: codes do not depend on how a kernel happens to round.  A 32-bit product settles almost every one: t = x * (127 / top)
// with the hardware's reciprocal (one step off at most) is off by less than 5e-5, so its nearest whole number is right
// unless t is that close to a half.  There the comparison of 254 |x| with (2 n + 1) top decides, n + 1/2 being the half in
// question; both products are exact in 64 bits (32 bits each).
struct QrRow {
    float top, inv, scale;
    bool none; // codes are 0
    bool far;  // the row's numbers have to go through qr_lift first: 1 / top would leave fp32's normal numbers
    float lift;
};

__device__ __forceinline__ int qr_code(float x, const QrRow &q)
{
    const float t = x * q.inv;
    const float r = __builtin_rintf(t);
    if (__builtin_expect(fabsf(t - r) < 0.5f - 1.0e-4f, 1)) return (int)r;
    const float n = __builtin_floorf(fabsf(t));
    const double over = 254.0 * fabs((double)x) - (double)(2.0f * n + 1.0f) * (double)q.top;
    const int c = (int)n + (over > 0.0 || (over == 0.0 && ((int)n & 1)) ? 1 : 0);
    return x < 0.0f ? -c : c;
}

__device__ __forceinline__ uint32_t qr_pack(int a, int b, int c, int d)
{
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// What a row is quantised by, from the largest magnitude's bits (as integers, magnitudes keep their order: Inf above every
// number, NaN above Inf).  A row with an Inf or a NaN has scale NaN and codes 0: products of it are NaN, never a plausible
// number.
__device__ __forceinline__ QrRow qr_row(uint32_t top_bits)
{
    QrRow r;
    const bool finite = top_bits < 0x7f800000u;
    r.top = __uint_as_float(top_bits);
    r.none = !finite || top_bits == 0;
    r.far = r.top < 1e-30f || r.top > 1e30f;
    r.lift = r.top < 1e-30f ? 1.2676506002282294e30f : 7.888609052210118e-31f; // 2^100, 2^-100
    // correctly rounded: a quotient of a 24-bit number by 127 keeps 2^-32 away from the middle of two fp32 numbers
    r.scale = finite ? (float)((double)r.top * (1.0 / 127.0)) : __builtin_nanf("");
    if (r.far) r.top *= r.lift;
    r.inv = r.none ? 0.0f : 127.0f * __builtin_amdgcn_rcpf(r.top);
    return r;
}

// x by a power of two.  Exact where it counts: what 2^-100 pushes below the normal numbers is below top 2^-120.
template <typename T> __device__ __forceinline__ T qr_lift(T x, const QrRow &q) { return (T)((float)x * q.lift); }

__device__ __forceinline__ uint32_t qr_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t qr_max(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Largest value of a workgroup of THREADS; red: THREADS / 64 words of LDS.
template <int THREADS> __device__ __forceinline__ uint32_t qr_block_max(uint32_t v, uint32_t *red)
{
    for (int o = 32; o > 0; o >>= 1) v = qr_max(v, __shfl_xor(v, o));
    if (THREADS > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) v = qr_max(v, red[w]);
    }
    return v;
}

// A gradient's factor f of a row whose largest magnitude is `top`, as two fp16 numbers: v = f 2^i8_shift(top), |v| < 2^15;
// hi = v in fp16, lo = (v - hi) 2^12 in fp16, so that v ~ hi + lo 2^-12.  hi is off by at most 2^-11 of v's power of two and
// lo by 2^-12 of what is left, so f is off by at most 2^-23 of ITSELF down to 2^-27 of top (from there hi is a subnormal
// number), and by 2^-50 of top below.  A product with an 8-bit code (also fp16) is exact in fp32.
// Rounding to 23 bits is a choice: all 24 take a third piece, half as much again of the matrix instructions, for an error
// that the sums' own roundings in fp32 hide; fixed point relative to top, in three signed 8-bit digits on the integer
// instructions, takes three quarters of the time and loses the factors far below top: against a confident classifier's
// cross-entropy gradients one entry of dL/dw in a hundred was off by a fifth of itself.
// (top comes to [2^13, 2^14): the exact product may lie half above a top that is a subnormal fp32 number, and lo must not
// overflow.)
#define I8_LO 4096.0
__device__ __forceinline__ int i8_shift(float top) { return 14 - __builtin_amdgcn_frexp_expf(top); }
__device__ __forceinline__ double i8_pow2(int e) { return __builtin_amdgcn_ldexp(1.0, e); }
__device__ __forceinline__ void i8_pieces(double v, _Float16 &hi, _Float16 &lo)
{
    hi = (_Float16)(float)v;
    lo = (_Float16)(float)((v - (double)(float)hi) * I8_LO);
}

// Longest contraction: 2^17 - 1 products of at most 2^14 cannot leave 32 bits.
#define I8_MAX_K 131071
// Longest row of the quantiser alone: its column indices are 32-bit, and a step of the long-row form past the end stays one
#define I8_MAX_ROW (1 << 30)
// Most rows: a launch has fewer than 2^32 threads, up to 1,024 of them a row
#define I8_MAX_ROWS 4194303

// ---- quantize.hip, used by linear_i8.hip ---------------------------------------------------------------------------
struct I8Rows { // rows to quantise, and where to
    const void *x;
    int type;
    int64_t x_stride;
    int M;
    const int32_t *n_rows;
    int8_t *codes;
    int64_t c_stride;
    float *scale;
};
// A and, in the same launch where it is of the same type, B (B.M = 0: none)
int frcnn_i8_quantize(const I8Rows &A, const I8Rows &B, int K, hipStream_t stream);
int frcnn_i8_pad_rows(const int8_t *src, int64_t src_stride, int rows, int K, int8_t *dst, int64_t dst_stride,
                      hipStream_t stream);

struct I8Grad { // a training step's backward inputs, and what its products read
    const void *grad, *y; // y NULL: no ReLU
    int type;
    int64_t grad_stride, y_stride;
    const int8_t *a, *b;
    int64_t a_stride, b_stride;
    const float *a_scale, *b_scale;
    int M, N, K;
    // dL/dx: pieces (2, M, row_stride) of g b_scale, their magnitudes (M), b transposed (K, row_stride); NULL: not wanted
    _Float16 *row_pieces, *b_t;
    float *row_top;
    int64_t row_stride;
    // dL/dw: pieces (2, N, col_stride) of g a_scale, their magnitudes (N), a transposed (K, col_stride; NULL: only
    // dL/dbias wanted), partial magnitudes and sums of the columns (frcnn_i8_grad_parts(M), N)
    _Float16 *col_pieces, *a_t;
    float *col_top;
    int64_t col_stride;
    uint32_t *part_top;
    float *part_sum;
    float *grad_bias;
};
int frcnn_i8_grad_parts(int M);
int frcnn_i8_grad_prepare(const I8Grad &A, hipStream_t stream);
