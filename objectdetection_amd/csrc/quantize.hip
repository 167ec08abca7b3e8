// quantize.hip -- what turns rows of numbers into 8-bit integers for linear_i8.hip: the row quantiser, and for the
// training step the byte transpose and the digits of the gradients.
//
// Row quantiser.  top = max_k |x_k|; scale = top / 127 (fp32); code_k = the whole number nearest to the EXACT quotient
// 127 x_k / top, ties to even.  Codes do not depend on how a kernel happens to round: 127 x (31 bits) and top (24 bits)
// are exact in 64-bit floating point, and a quotient of such numbers that is not a half is at least 2^-25 / 2^7 away
// from it relatively, far more than 2^-53, so one correctly rounded 64-bit division decides.  Almost every code is
// settled by a 32-bit product instead: t = x * (127 / top) is off by less than 3e-5, so it settles every t that is
// further than that from a half.
#include "i8_common.h"

#define QR_NEAR (0.5f - 3.0e-5f)

// The code of x in a row whose largest magnitude is `top`; inv = 127 / top in fp32, or NaN to ask for the division
// (a top so small that 127 / top leaves fp32).
__device__ __forceinline__ int qr_code(float x, float top, float inv)
{
    const float t = x * inv;
    const float r = __builtin_rintf(t);
    if (__builtin_expect(!(fabsf(t - r) < QR_NEAR), 0)) return (int)__builtin_rint((double)x * 127.0 / (double)top);
    return (int)r;
}

__device__ __forceinline__ uint32_t qr_pack(int a, int b, int c, int d)
{
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// One workgroup a row, the row held in registers between the maximum and the codes (V elements of 16 bytes a load,
// NV loads a thread), so that x is read once.  A row with an Inf or a NaN has scale NaN and codes 0: products of it
// are NaN, never a plausible number.
template <typename T, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS)
quantize_rows_kernel(const T *__restrict__ x, int64_t x_stride, int M, int K, const int32_t *__restrict__ n_rows,
                     int8_t *__restrict__ codes, int64_t c_stride, float *__restrict__ scale)
{
    constexpr int V = 16 / sizeof(T);
    __shared__ uint32_t red[THREADS / 64];
    const int row = blockIdx.x;
    if (row >= i8_rows(n_rows, M)) return;
    const T *xr = x + (int64_t)row * x_stride;
    int8_t *cr = codes + (int64_t)row * c_stride;
    I8Vec<T, V> v[NV];
    uint32_t top_bits = 0; // magnitudes as integers: order kept, Inf above every number and NaN above Inf
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * THREADS + (int)threadIdx.x) * V;
        if (k + V <= K) {
            v[i] = i8_load<T, V>(xr + k);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[i].v[j] = k + j < K ? xr[k + j] : (T)0.0f;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t m = __float_as_uint((float)v[i].v[j]) & 0x7fffffffu;
            top_bits = m > top_bits ? m : top_bits;
        }
    }
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t m = __shfl_xor(top_bits, o);
        top_bits = m > top_bits ? m : top_bits;
    }
    if (THREADS > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top_bits;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) top_bits = red[w] > top_bits ? red[w] : top_bits;
    }
    const bool finite = top_bits < 0x7f800000u;
    const float top = __uint_as_float(top_bits);
    const bool none = !finite || top_bits == 0;
    const float inv = none ? 0.0f : (top < 1e-30f ? __builtin_nanf("") : 127.0f / top);
    if (threadIdx.x == 0) scale[row] = finite ? top / 127.0f : __builtin_nanf("");
    // the stride is a multiple of 16 whenever K is not: bytes up to the next multiple belong to the row
    const int kp = (K + 15) & ~15;
    const bool wide = (c_stride & 15) == 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * THREADS + (int)threadIdx.x) * V;
        if (k >= (wide ? kp : K)) break;
        int c[V];
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = none ? 0 : qr_code((float)v[i].v[j], top, inv);
        if (wide) {
            uint32_t p[V / 4];
#pragma unroll
            for (int j = 0; j < V / 4; ++j) p[j] = qr_pack(c[4 * j], c[4 * j + 1], c[4 * j + 2], c[4 * j + 3]);
            __builtin_memcpy(__builtin_assume_aligned(cr + k, V), p, V);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (k + j < K) cr[k + j] = (int8_t)c[j];
        }
    }
}

// Rows too long for the registers of a workgroup: the same in two passes over the row.
template <typename T>
__global__ void __launch_bounds__(1024)
quantize_rows_long_kernel(const T *__restrict__ x, int64_t x_stride, int M, int K, const int32_t *__restrict__ n_rows,
                          int8_t *__restrict__ codes, int64_t c_stride, float *__restrict__ scale)
{
    __shared__ uint32_t red[16];
    const int row = blockIdx.x;
    if (row >= i8_rows(n_rows, M)) return;
    const T *xr = x + (int64_t)row * x_stride;
    int8_t *cr = codes + (int64_t)row * c_stride;
    uint32_t top_bits = 0;
    for (int k = threadIdx.x; k < K; k += 1024) {
        const uint32_t m = __float_as_uint((float)xr[k]) & 0x7fffffffu;
        top_bits = m > top_bits ? m : top_bits;
    }
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t m = __shfl_xor(top_bits, o);
        top_bits = m > top_bits ? m : top_bits;
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top_bits;
    __syncthreads();
    for (int w = 0; w < 16; ++w) top_bits = red[w] > top_bits ? red[w] : top_bits;
    const bool finite = top_bits < 0x7f800000u;
    const float top = __uint_as_float(top_bits);
    const bool none = !finite || top_bits == 0;
    const float inv = none ? 0.0f : (top < 1e-30f ? __builtin_nanf("") : 127.0f / top);
    if (threadIdx.x == 0) scale[row] = finite ? top / 127.0f : __builtin_nanf("");
    const int kp = (c_stride & 15) == 0 ? (K + 15) & ~15 : K;
    for (int k = threadIdx.x; k < kp; k += 1024) cr[k] = (int8_t)(none || k >= K ? 0 : qr_code((float)xr[k], top, inv));
}

template <typename T>
static int quantize_rows_t(const T *x, int64_t x_stride, int M, int K, const int32_t *n_rows, int8_t *codes,
                           int64_t c_stride, float *scale, hipStream_t st)
{
    constexpr int V = 16 / sizeof(T);
#define QR_LAUNCH(THREADS, NV)                                                                                      \
    if (K <= THREADS * NV * V) {                                                                                    \
        hipLaunchKernelGGL((quantize_rows_kernel<T, THREADS, NV>), dim3(M), dim3(THREADS), 0, st, x, x_stride, M, K, \
                           n_rows, codes, c_stride, scale);                                                         \
        FRCNN_CHECK_LAUNCH("quantize_rows");                                                                        \
        return FRCNN_OK;                                                                                            \
    }
    QR_LAUNCH(64, 4)
    QR_LAUNCH(256, 4)
    QR_LAUNCH(256, 16)
    QR_LAUNCH(512, 16)
#undef QR_LAUNCH
    hipLaunchKernelGGL((quantize_rows_long_kernel<T>), dim3(M), dim3(1024), 0, st, x, x_stride, M, K, n_rows, codes,
                       c_stride, scale);
    FRCNN_CHECK_LAUNCH("quantize_rows");
    return FRCNN_OK;
}

extern "C" int frcnn_quantize_rows_i8(const void *x, int x_type, int64_t x_stride, int M, int K, const int32_t *n_rows,
                                      int8_t *codes, int64_t codes_stride, float *scale, void *stream)
{
    FRCNN_REQUIRE(i8_type_ok(x_type), "quantize_rows: unknown element type %d", x_type);
    FRCNN_REQUIRE(M >= 0 && K > 0, "quantize_rows: bad shape (%d, %d)", M, K);
    FRCNN_REQUIRE(codes_stride >= K && x_stride >= 0, "quantize_rows: bad strides");
    if (M == 0) return FRCNN_OK;
    FRCNN_REQUIRE(x && codes && scale, "quantize_rows: null pointer");
    FRCNN_REQUIRE((codes_stride & 15) != 0 || ((uintptr_t)codes & 15) == 0,
                  "quantize_rows: codes of a padded row stride have to be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    if (x_type == FRCNN_F32)
        return quantize_rows_t((const float *)x, x_stride, M, K, n_rows, codes, codes_stride, scale, st);
    if (x_type == FRCNN_BF16)
        return quantize_rows_t((const __bf16 *)x, x_stride, M, K, n_rows, codes, codes_stride, scale, st);
    return quantize_rows_t((const _Float16 *)x, x_stride, M, K, n_rows, codes, codes_stride, scale, st);
}

// ---- rows copied to an aligned row stride -----------------------------------------------------------------------
__global__ void __launch_bounds__(256)
i8_pad_rows_kernel(const int8_t *__restrict__ src, int64_t s_stride, int K, int8_t *__restrict__ dst, int64_t d_stride)
{
    const int64_t row = blockIdx.x;
    const int8_t *s = src + row * s_stride;
    int8_t *d = dst + row * d_stride;
    for (int k = threadIdx.x * 16; k < (int)d_stride; k += 256 * 16) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (k + 16 <= K) {
            __builtin_memcpy(w, s + k, 16);
        } else {
            for (int j = 0; j < 16; ++j)
                if (k + j < K) w[j >> 2] |= (uint32_t)(uint8_t)s[k + j] << ((j & 3) * 8);
        }
        *(uint4 *)(d + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

int frcnn_i8_pad_rows(const int8_t *src, int64_t src_stride, int rows, int K, int8_t *dst, int64_t dst_stride,
                      hipStream_t stream)
{
    hipLaunchKernelGGL(i8_pad_rows_kernel, dim3(rows), dim3(256), 0, stream, src, src_stride, K, dst, dst_stride);
    FRCNN_CHECK_LAUNCH("i8_pad_rows");
    return FRCNN_OK;
}

// ---- byte transpose (rows, cols) -> (cols, rows): the operand of a gradient's product --------------------------------
// 64 x 64 tiles through LDS; a thread reads 16 bytes of a row and writes 16 bytes of a column.
__global__ void __launch_bounds__(256)
i8_transpose_kernel(const int8_t *__restrict__ src, int64_t s_stride, int rows, int cols, int8_t *__restrict__ dst,
                    int64_t d_stride)
{
    __shared__ int8_t tile[64][68];
    const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 64;
    const int tr = threadIdx.x >> 2, tc = (threadIdx.x & 3) * 16;
    uint32_t w[4] = {0, 0, 0, 0};
    if (r0 + tr < rows) {
        const int8_t *s = src + (r0 + tr) * s_stride + c0 + tc;
        if (c0 + tc + 16 <= cols) {
            __builtin_memcpy(w, s, 16);
        } else {
            for (int j = 0; j < 16; ++j)
                if (c0 + tc + j < cols) w[j >> 2] |= (uint32_t)(uint8_t)s[j] << ((j & 3) * 8);
        }
    }
    for (int j = 0; j < 4; ++j) *(uint32_t *)&tile[tr][tc + 4 * j] = w[j];
    __syncthreads();
    // thread: column tr of the tile, rows tc .. tc + 15
    if (c0 + tr >= cols || r0 + tc >= d_stride) return;
    for (int j = 0; j < 4; ++j)
        w[j] = qr_pack(tile[tc + 4 * j][tr], tile[tc + 4 * j + 1][tr], tile[tc + 4 * j + 2][tr], tile[tc + 4 * j + 3][tr]);
    *(uint4 *)(dst + (c0 + tr) * d_stride + r0 + tc) = make_uint4(w[0], w[1], w[2], w[3]);
}

int frcnn_i8_transpose(const int8_t *src, int64_t src_stride, int rows, int cols, int8_t *dst, int64_t dst_stride,
                       hipStream_t stream)
{
    hipLaunchKernelGGL(i8_transpose_kernel, dim3((cols + 63) / 64, (rows + 63) / 64), dim3(256), 0, stream, src,
                       src_stride, rows, cols, dst, dst_stride);
    FRCNN_CHECK_LAUNCH("i8_transpose");
    return FRCNN_OK;
}

// ---- digits of the gradients -----------------------------------------------------------------------------------------
// g_mn = grad_mn, or 0 where a ReLU's output y_mn is not above 0 (y = NULL: no ReLU; a NaN lets the gradient through, as
// torch's threshold backward does).
template <typename T> __device__ __forceinline__ float gd_grad(const T *grad, const T *y, int64_t gi, int64_t yi)
{
    const float g = (float)grad[gi];
    return y && (float)y[yi] <= 0.0f ? 0.0f : g;
}

// Fixed point relative to `top`: T = round(a I8_FIX / top), off by at most top 2^-24; the product and the factor are
// formed in 64 bits.
__device__ __forceinline__ int gd_fix(float a, double inv) { return (int)__builtin_rint((double)a * inv); }

// For dL/dx: a_mn = g_mn * col_scale_n, fixed point relative to the row's largest magnitude.  One wave a row.
template <typename T>
__global__ void __launch_bounds__(256)
grad_row_digits_kernel(const T *__restrict__ grad, int64_t g_stride, const T *__restrict__ y, int64_t y_stride,
                       const float *__restrict__ col_scale, int M, int N, int8_t *__restrict__ digits, int64_t stride,
                       int64_t plane, float *__restrict__ row_top)
{
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= M) return;
    uint32_t top_bits = 0;
    for (int n = lane; n < N; n += 64) {
        const float a = gd_grad(grad, y, row * g_stride + n, row * y_stride + n) * col_scale[n];
        const uint32_t m = __float_as_uint(a) & 0x7fffffffu;
        top_bits = m > top_bits ? m : top_bits;
    }
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t m = __shfl_xor(top_bits, o);
        top_bits = m > top_bits ? m : top_bits;
    }
    const bool finite = top_bits < 0x7f800000u;
    const float top = __uint_as_float(top_bits);
    const double inv = !finite || top_bits == 0 ? 0.0 : (double)I8_FIX / (double)top;
    if (lane == 0) row_top[row] = finite ? top : __builtin_nanf("");
    int8_t *d = digits + row * stride;
    for (int n = lane * 4; n < (int)stride; n += 256) {
        uint32_t w[3] = {0, 0, 0};
        for (int j = 0; j < 4; ++j) {
            if (n + j < N && inv != 0.0) {
                const float a = gd_grad(grad, y, row * g_stride + n + j, row * y_stride + n + j) * col_scale[n + j];
                int d0, d1, d2;
                i8_digits(gd_fix(a, inv), d0, d1, d2);
                w[0] |= (uint32_t)(d0 & 255) << (8 * j);
                w[1] |= (uint32_t)(d1 & 255) << (8 * j);
                w[2] |= (uint32_t)(d2 & 255) << (8 * j);
            }
        }
        for (int p = 0; p < 3; ++p) *(uint32_t *)(d + p * plane + n) = w[p];
    }
}

int frcnn_i8_grad_row_digits(const void *grad, int type, int64_t grad_stride, const void *y, int64_t y_stride,
                             const float *col_scale, int M, int N, int8_t *digits, int64_t stride, int64_t plane,
                             float *row_top, hipStream_t stream)
{
#define GR_LAUNCH(T)                                                                                                    \
    hipLaunchKernelGGL((grad_row_digits_kernel<T>), dim3((M + 3) / 4), dim3(256), 0, stream, (const T *)grad, grad_stride, \
                       (const T *)y, y_stride, col_scale, M, N, digits, stride, plane, row_top)
    if (type == FRCNN_F32) GR_LAUNCH(float);
    else if (type == FRCNN_BF16) GR_LAUNCH(__bf16);
    else GR_LAUNCH(_Float16);
#undef GR_LAUNCH
    FRCNN_CHECK_LAUNCH("grad_row_digits");
    return FRCNN_OK;
}

// For dL/dw: a_mn = g_mn * row_scale_m, fixed point relative to the COLUMN's largest magnitude, written transposed
// (n, m).  First pass: largest magnitude and plain sum (dL/dbias) of every column over GC_ROWS rows; second pass: the
// column's magnitude from those partials, the digits, and the sum of the partials in row order (the same bits every
// run).
#define GC_ROWS 256
template <typename T>
__global__ void __launch_bounds__(256)
grad_col_partials_kernel(const T *__restrict__ grad, int64_t g_stride, const T *__restrict__ y, int64_t y_stride,
                         const float *__restrict__ row_scale, int M, int N, uint32_t *__restrict__ part_top,
                         float *__restrict__ part_sum)
{
    __shared__ uint32_t tops[4][64];
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = blockIdx.x * 64 + lane;
    const int64_t m0 = (int64_t)blockIdx.y * GC_ROWS;
    uint32_t top = 0;
    float sum = 0.0f;
    if (n < N) {
        for (int i = wave; i < GC_ROWS; i += 4) {
            const int64_t m = m0 + i;
            if (m >= M) break;
            const float g = gd_grad(grad, y, m * g_stride + n, m * y_stride + n);
            const uint32_t b = __float_as_uint(g * row_scale[m]) & 0x7fffffffu;
            top = b > top ? b : top;
            sum += g;
        }
    }
    tops[wave][lane] = top;
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && n < N) {
        for (int w = 1; w < 4; ++w) {
            top = tops[w][lane] > top ? tops[w][lane] : top;
            sum += sums[w][lane];
        }
        part_top[(int64_t)blockIdx.y * N + n] = top;
        part_sum[(int64_t)blockIdx.y * N + n] = sum;
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
grad_col_digits_kernel(const T *__restrict__ grad, int64_t g_stride, const T *__restrict__ y, int64_t y_stride,
                       const float *__restrict__ row_scale, int M, int N, int8_t *__restrict__ digits, int64_t stride,
                       int64_t plane, float *__restrict__ col_top, float *__restrict__ col_sum,
                       const uint32_t *__restrict__ part_top, const float *__restrict__ part_sum, int n_part)
{
    __shared__ int8_t tile[3][64][68]; // [digit][n][m]
    __shared__ double inv_s[64];
    const int64_t m0 = (int64_t)blockIdx.y * 64;
    const int n0 = blockIdx.x * 64;
    if (threadIdx.x < 64) {
        const int n = n0 + threadIdx.x;
        uint32_t top = 0;
        float sum = 0.0f;
        if (n < N) {
            for (int p = 0; p < n_part; ++p) {
                const uint32_t b = part_top[(int64_t)p * N + n];
                top = b > top ? b : top;
                sum += part_sum[(int64_t)p * N + n];
            }
        }
        const bool finite = top < 0x7f800000u;
        inv_s[threadIdx.x] = !finite || top == 0 ? 0.0 : (double)I8_FIX / (double)__uint_as_float(top);
        if (blockIdx.y == 0 && n < N) {
            col_top[n] = finite ? __uint_as_float(top) : __builtin_nanf("");
            if (col_sum) col_sum[n] = sum;
        }
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = n0 + lane;
    const double inv = inv_s[lane];
    for (int i = wave; i < 64; i += 4) {
        const int64_t m = m0 + i;
        int d0 = 0, d1 = 0, d2 = 0;
        if (m < M && n < N && inv != 0.0)
            i8_digits(gd_fix(gd_grad(grad, y, m * g_stride + n, m * y_stride + n) * row_scale[m], inv), d0, d1, d2);
        tile[0][lane][i] = (int8_t)d0;
        tile[1][lane][i] = (int8_t)d1;
        tile[2][lane][i] = (int8_t)d2;
    }
    __syncthreads();
    const int tn = threadIdx.x >> 2, tm = (threadIdx.x & 3) * 16;
    if (n0 + tn >= N || m0 + tm >= stride) return;
    for (int p = 0; p < 3; ++p) {
        uint32_t w[4];
        for (int j = 0; j < 4; ++j) w[j] = *(const uint32_t *)&tile[p][tn][tm + 4 * j];
        *(uint4 *)(digits + p * plane + (int64_t)(n0 + tn) * stride + m0 + tm) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

size_t frcnn_i8_grad_col_partials(int M, int N)
{
    return (size_t)((M + GC_ROWS - 1) / GC_ROWS) * (size_t)N * 8;
}

int frcnn_i8_grad_col_digits(const void *grad, int type, int64_t grad_stride, const void *y, int64_t y_stride,
                             const float *row_scale, int M, int N, int8_t *digits, int64_t stride, int64_t plane,
                             float *col_top, float *col_sum, void *partials, hipStream_t stream)
{
    const int n_part = (M + GC_ROWS - 1) / GC_ROWS;
    uint32_t *part_top = (uint32_t *)partials;
    float *part_sum = (float *)partials + (size_t)n_part * N;
#define GC_LAUNCH(T)                                                                                                   \
    hipLaunchKernelGGL((grad_col_partials_kernel<T>), dim3((N + 63) / 64, n_part), dim3(256), 0, stream, (const T *)grad, \
                       grad_stride, (const T *)y, y_stride, row_scale, M, N, part_top, part_sum);                      \
    hipLaunchKernelGGL((grad_col_digits_kernel<T>), dim3((N + 63) / 64, (M + 63) / 64), dim3(256), 0, stream,          \
                       (const T *)grad, grad_stride, (const T *)y, y_stride, row_scale, M, N, digits, stride, plane,   \
                       col_top, col_sum, part_top, part_sum, n_part)
    if (type == FRCNN_F32) { GC_LAUNCH(float); }
    else if (type == FRCNN_BF16) { GC_LAUNCH(__bf16); }
    else { GC_LAUNCH(_Float16); }
#undef GC_LAUNCH
    FRCNN_CHECK_LAUNCH("grad_col_digits");
    return FRCNN_OK;
}
