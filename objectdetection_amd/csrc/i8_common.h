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

// A signed 24-bit fixed-point number T (|T| <= I8_FIX) as three signed 8-bit digits, T = d0 2^16 + d1 2^8 + d2 with
// d0 in [-127, 127] and d1, d2 in [-128, 127].
#define I8_FIX 8323072 /* 127 * 2^16 */
__device__ __forceinline__ void i8_digits(int T, int &d0, int &d1, int &d2)
{
    d0 = (T + 32896) >> 16;
    const int r = T - (d0 << 16); // in [-32896, 32639]
    d1 = (r + 128) >> 8;
    d2 = r - (d1 << 8);
}

// Longest contraction: 2^17 - 1 products of at most 2^14 cannot leave 32 bits.
#define I8_MAX_K 131071

// quantize.hip, used by linear_i8.hip
int frcnn_i8_pad_rows(const int8_t *src, int64_t src_stride, int rows, int K, int8_t *dst, int64_t dst_stride,
                      hipStream_t stream);
int frcnn_i8_transpose(const int8_t *src, int64_t src_stride, int rows, int cols, int8_t *dst, int64_t dst_stride,
                       hipStream_t stream);
int frcnn_i8_grad_row_digits(const void *grad, int type, int64_t grad_stride, const void *y, int64_t y_stride,
                             const float *col_scale, int M, int N, int8_t *digits, int64_t stride, int64_t plane,
                             float *row_top, hipStream_t stream);
size_t frcnn_i8_grad_col_partials(int M, int N);
int frcnn_i8_grad_col_digits(const void *grad, int type, int64_t grad_stride, const void *y, int64_t y_stride,
                             const float *row_scale, int M, int N, int8_t *digits, int64_t stride, int64_t plane,
                             float *col_top, float *col_sum, void *partials, hipStream_t stream);
