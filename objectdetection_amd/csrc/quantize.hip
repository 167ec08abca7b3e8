// quantize.hip -- what turns rows of numbers into 8-bit integers for linear_i8.hip: the row quantiser, and for the
// training step the transposed codes and the pieces of the gradients.
#include "i8_common.h"

// One workgroup a row, the row held in registers between the maximum and the codes (V elements of 16 bytes a load,
// NV loads a thread), so that x is read once.
// Bound by HBM: 32,000 rows of 25,088 fp32 727 us (4.0 GB, 5.5 TB/s), 2,000 of 12,544 21.6 us (5.8 TB/s), 32,000 of 1,024
// bf16 18.8 us (5.2 TB/s); a copy of 4 GiB reaches 4.7 TB/s.
// Two workgroups' rows have to fit a CU, so that one loads while the other computes: registers are bounded to 64 (but for
// the longest rows, 32,000 of 50,176 fp32 1,540 us, 5.2 TB/s).
template <typename T, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS, NV > 7 ? 4 : 8)
quantize_rows_kernel(const I8Rows A, const I8Rows B, int K)
{
    constexpr int V = 16 / sizeof(T);
    __shared__ uint32_t red[THREADS / 64];
    const bool second = (int)blockIdx.x >= A.M;
    const int row = second ? blockIdx.x - A.M : blockIdx.x, t = threadIdx.x;
    if (!second && row >= i8_rows(A.n_rows, A.M)) return;
    const T *xr = (const T *)(second ? B.x : A.x) + (int64_t)row * (second ? B.x_stride : A.x_stride);
    const int64_t c_stride = second ? B.c_stride : A.c_stride;
    int8_t *cr = (second ? B.codes : A.codes) + (int64_t)row * c_stride;
    const int kf = K - K % V; // whole vectors up to here; the last K % V elements one a thread
    I8Vec<T, V> v[NV];
    T v_tail = kf + t < K && t < V ? xr[kf + t] : (T)0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * THREADS + t) * V;
        v[i] = I8Vec<T, V>{};
        if (k < kf) v[i] = i8_load<T, V>(xr + k);
    }
    uint32_t top_bits = qr_bits((float)v_tail);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) top_bits = qr_max(top_bits, qr_bits((float)v[i].v[j]));
    const QrRow q = qr_row(qr_block_max<THREADS>(top_bits, red));
    if (t == 0) (second ? B.scale : A.scale)[row] = q.scale;
    if (__builtin_expect(q.far, 0)) {
        v_tail = qr_lift(v_tail, q);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) v[i].v[j] = qr_lift(v[i].v[j], q);
    }
    const bool wide = (c_stride & 15) == 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * THREADS + t) * V;
        if (k >= kf) break;
        uint32_t p[V / 4];
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            int c[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = q.none ? 0 : qr_code((float)v[i].v[4 * j + e], q);
            p[j] = qr_pack(c[0], c[1], c[2], c[3]);
        }
        if (wide) __builtin_memcpy(__builtin_assume_aligned(cr + k, V), p, V);
        else __builtin_memcpy(cr + k, p, V);
    }
    // the tail, and with a stride that is a multiple of 16 zeros up to the next multiple, which belong to the row
    if (t < 16 && kf + t < (wide ? (K + 15) & ~15 : K))
        cr[kf + t] = (int8_t)(q.none || kf + t >= K ? 0 : qr_code((float)v_tail, q));
}

// Rows too long for the registers of a workgroup: the same in two passes over the row, the second out of the caches.
// 2,000 rows of 60,000 bf16 102 us (0.36 GB once, 3.5 TB/s), of 131,000 fp32 408 us (3.2 TB/s).
template <typename T>
__global__ void __launch_bounds__(1024, 8)
quantize_rows_long_kernel(const I8Rows A, int K)
{
    constexpr int V = 16 / sizeof(T), AHEAD = 4, STEP = 1024 * V * AHEAD;
    __shared__ uint32_t red[16];
    const int row = blockIdx.x, t = threadIdx.x;
    if (row >= i8_rows(A.n_rows, A.M)) return;
    const T *xr = (const T *)A.x + (int64_t)row * A.x_stride;
    int8_t *cr = A.codes + (int64_t)row * A.c_stride;
    const int kf = K - K % V; // whole vectors up to here; the last K % V elements one a thread
    auto load = [&](I8Vec<T, V>(&v)[AHEAD], int k0) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int k = k0 + (i * 1024 + t) * V;
            v[i] = I8Vec<T, V>{};
            if (k < kf) v[i] = i8_load<T, V>(xr + k);
        }
    };
    const T v_tail = kf + t < K && t < V ? xr[kf + t] : (T)0.0f;
    uint32_t top_bits = qr_bits((float)v_tail);
    for (int k0 = 0; k0 < kf; k0 += STEP) {
        I8Vec<T, V> v[AHEAD];
        load(v, k0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) top_bits = qr_max(top_bits, qr_bits((float)v[i].v[j]));
    }
    const QrRow q = qr_row(qr_block_max<1024>(top_bits, red));
    if (t == 0) A.scale[row] = q.scale;
    auto code = [&](T x) { return q.none ? 0 : qr_code((float)(q.far ? qr_lift(x, q) : x), q); };
    const bool wide = (A.c_stride & 15) == 0;
    for (int k0 = 0; k0 < kf; k0 += STEP) {
        I8Vec<T, V> v[AHEAD];
        load(v, k0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int k = k0 + (i * 1024 + t) * V;
            if (k >= kf) break;
            uint32_t p[V / 4];
#pragma unroll
            for (int j = 0; j < V / 4; ++j)
                p[j] = qr_pack(code(v[i].v[4 * j]), code(v[i].v[4 * j + 1]), code(v[i].v[4 * j + 2]), code(v[i].v[4 * j + 3]));
            if (wide) __builtin_memcpy(__builtin_assume_aligned(cr + k, V), p, V);
            else __builtin_memcpy(cr + k, p, V);
        }
    }
    if (t < 16 && kf + t < (wide ? (K + 15) & ~15 : K)) cr[kf + t] = (int8_t)(kf + t >= K ? 0 : code(v_tail));
}

// B: rows of a second matrix of the same type and length in the same launch (B.M = 0: none)
template <typename T> static int quantize_rows_t(const I8Rows &A, const I8Rows &B, int K, hipStream_t st)
{
    constexpr int V = 16 / sizeof(T);
    const int M = A.M + B.M;
#define QR_LAUNCH(THREADS, NV)                                                                            \
    if (K <= THREADS * NV * V) {                                                                          \
        hipLaunchKernelGGL((quantize_rows_kernel<T, THREADS, NV>), dim3(M), dim3(THREADS), 0, st, A, B, K); \
        FRCNN_CHECK_LAUNCH("quantize_rows");                                                              \
        return FRCNN_OK;                                                                                  \
    }
    // four loads a thread, or one where there are too few rows to fill the chip
    if (M >= 1024) {
        QR_LAUNCH(64, 4)
        QR_LAUNCH(128, 4)
        QR_LAUNCH(256, 4)
        QR_LAUNCH(512, 4)
    }
    QR_LAUNCH(64, 1)
    QR_LAUNCH(256, 1)
    QR_LAUNCH(1024, 1)
    QR_LAUNCH(1024, 4)
    if constexpr (V == 4) {
        QR_LAUNCH(1024, 7)  // what 64 registers hold
        QR_LAUNCH(1024, 16) // and 128, one workgroup a CU: 2,000 rows of 60,000 145 us, in two passes 176; in 16 bits it spills
    }
#undef QR_LAUNCH
    for (const I8Rows *r : {&A, &B}) {
        if (r->M == 0) continue;
        hipLaunchKernelGGL((quantize_rows_long_kernel<T>), dim3(r->M), dim3(1024), 0, st, *r, K);
        FRCNN_CHECK_LAUNCH("quantize_rows");
    }
    return FRCNN_OK;
}

int frcnn_i8_quantize(const I8Rows &A, const I8Rows &B, int K, hipStream_t st)
{
    if (B.M && B.type != A.type) { // two types: two launches
        const int rc = frcnn_i8_quantize(A, I8Rows{}, K, st);
        return rc == FRCNN_OK ? frcnn_i8_quantize(B, I8Rows{}, K, st) : rc;
    }
    if (A.type == FRCNN_F32) return quantize_rows_t<float>(A, B, K, st);
    if (A.type == FRCNN_BF16) return quantize_rows_t<__bf16>(A, B, K, st);
    return quantize_rows_t<_Float16>(A, B, K, st);
}

extern "C" int frcnn_quantize_rows_i8(const void *x, int x_type, int64_t x_stride, int M, int K, const int32_t *n_rows,
                                      int8_t *codes, int64_t codes_stride, float *scale, void *stream)
{
    FRCNN_REQUIRE(i8_type_ok(x_type), "quantize_rows: unknown element type %d", x_type);
    FRCNN_REQUIRE(M >= 0 && M <= I8_MAX_ROWS && K > 0 && K <= I8_MAX_ROW,
                  "quantize_rows: bad shape (%d, %d); at most %d rows of %d", M, K, I8_MAX_ROWS, I8_MAX_ROW);
    FRCNN_REQUIRE(codes_stride >= K && x_stride >= 0, "quantize_rows: bad strides");
    if (M == 0) return FRCNN_OK;
    FRCNN_REQUIRE(x && codes && scale, "quantize_rows: null pointer");
    FRCNN_REQUIRE((codes_stride & 15) != 0 || ((uintptr_t)codes & 15) == 0,
                  "quantize_rows: codes of a padded row stride have to be 16-byte aligned");
    return frcnn_i8_quantize(I8Rows{x, x_type, x_stride, M, n_rows, codes, codes_stride, scale}, I8Rows{}, K,
                             (hipStream_t)stream);
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

// ---- what the gradients' products are made from ----------------------------------------------------------------------
// g_mn = grad_mn, or 0 where a ReLU cut: where its output y_mn is below zero or +0 (y = NULL: no ReLU).  -0 stands for a
// positive number that the output's type rounds to zero; a NaN lets the gradient through, as torch's threshold backward does.
__device__ __forceinline__ bool gd_cut(float y) { return y <= 0.0f && __float_as_uint(y) != 0x80000000u; }
template <typename T> __device__ __forceinline__ float gd_grad(const T *grad, const T *y, int64_t gi, int64_t yi)
{
    const float g = (float)grad[gi];
    return y && gd_cut((float)y[yi]) ? 0.0f : g;
}

// Codes (rows, cols) -> fp16 (cols, rows), one 64 x 64 tile; a thread reads 16 codes of a row and writes 16 of a column.
__device__ __forceinline__ void gd_transpose(const int8_t *src, int64_t s_stride, int rows, int cols, _Float16 *dst,
                                             int64_t d_stride, int64_t r0, int64_t c0, int8_t (&tile)[64][68])
{
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
    I8Vec<_Float16, 16> h;
#pragma unroll
    for (int j = 0; j < 16; ++j) h.v[j] = (_Float16)(int16_t)tile[tc + j][tr];
    __builtin_memcpy(__builtin_assume_aligned(dst + (c0 + tr) * d_stride + r0 + tc, 32), &h, 32);
}

// For dL/dx: a_mn = g_mn * b_scale_n in pieces, scaled by the row's largest magnitude.  One wave a row, four neighbours a
// lane, up to NV of those held in registers; a longer row is read again (from the caches) for its pieces.  The largest is that
// of the products in fp32, the pieces are taken from the exact products.
template <typename T, int NV>
__device__ __forceinline__ void gd_row_pieces(const I8Grad &A, int64_t row)
{
    const int lane = threadIdx.x & 63, N = A.N;
    if (row >= A.M) return;
    const T *g = (const T *)A.grad + row * A.grad_stride, *z = A.y ? (const T *)A.y + row * A.y_stride : nullptr;
    struct Quad {
        float g[4], s[4];
    };
    auto load = [&](Quad &a, int n) {
        if (n + 4 <= N) {
            const I8Vec<T, 4> v = i8_load<T, 4>(g + n);
            const I8Vec<float, 4> c = i8_load<float, 4>(A.b_scale + n);
            I8Vec<T, 4> u = v;
            if (z) u = i8_load<T, 4>(z + n);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a.g[j] = z && gd_cut((float)u.v[j]) ? 0.0f : (float)v.v[j];
                a.s[j] = c.v[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a.g[j] = n + j < N ? gd_grad(g, z, n + j, n + j) : 0.0f;
                a.s[j] = n + j < N ? A.b_scale[n + j] : 0.0f;
            }
        }
    };
    Quad a[NV];
    uint32_t top_bits = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) load(a[i], (i * 64 + lane) * 4);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) top_bits = qr_max(top_bits, qr_bits(a[i].g[j] * a[i].s[j]));
    for (int n = (NV * 64 + lane) * 4; n < N; n += 256) {
        Quad t;
        load(t, n);
        for (int j = 0; j < 4; ++j) top_bits = qr_max(top_bits, qr_bits(t.g[j] * t.s[j]));
    }
    for (int o = 32; o > 0; o >>= 1) top_bits = qr_max(top_bits, __shfl_xor(top_bits, o));
    const bool finite = top_bits < 0x7f800000u;
    const float top = __uint_as_float(top_bits);
    const bool none = !finite || top_bits == 0;
    const double up = i8_pow2(i8_shift(top));
    if (lane == 0) A.row_top[row] = finite ? top : __builtin_nanf("");
    _Float16 *d = A.row_pieces + row * A.row_stride;
    const int64_t plane = A.M * A.row_stride;
    auto store = [&](const Quad &t, int n) {
        I8Vec<_Float16, 4> h[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) i8_pieces(none ? 0.0 : (double)t.g[j] * (double)t.s[j] * up, h[0].v[j], h[1].v[j]);
#pragma unroll
        for (int p = 0; p < 2; ++p) __builtin_memcpy(__builtin_assume_aligned(d + p * plane + n, 8), &h[p], 8);
    };
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * 64 + lane) * 4 < (int)A.row_stride) store(a[i], (i * 64 + lane) * 4);
    for (int n = (NV * 64 + lane) * 4; n < (int)A.row_stride; n += 256) {
        Quad t;
        load(t, n);
        store(t, n);
    }
}

// For dL/dw: a_mn = g_mn * a_scale_m in pieces, scaled by the COLUMN's largest magnitude, written transposed (n, m).
// First the largest magnitude and the plain sum (dL/dbias) of every column over GC_ROWS rows; then (grad_col_pieces_kernel)
// the column's magnitude from those partials, the pieces, and the sum of the partials in row order (the same bits every
// run).
#define GC_ROWS 64
template <typename T>
__device__ __forceinline__ void gd_col_partials(const I8Grad &A, int bx, int by, uint32_t (&tops)[4][64], float (&sums)[4][64])
{
    const T *grad = (const T *)A.grad, *y = (const T *)A.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = bx * 64 + lane, N = A.N;
    const int64_t m0 = (int64_t)by * GC_ROWS;
    uint32_t top = 0;
    float sum = 0.0f;
    if (n < N) {
        float g[GC_ROWS / 4], s[GC_ROWS / 4]; // all loads before the first use
#pragma unroll
        for (int i = 0; i < GC_ROWS / 4; ++i) {
            const int64_t m = m0 + i * 4 + wave;
            g[i] = m < A.M ? gd_grad(grad, y, m * A.grad_stride + n, m * A.y_stride + n) : 0.0f;
            s[i] = m < A.M ? A.a_scale[m] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < GC_ROWS / 4; ++i) {
            top = qr_max(top, qr_bits(g[i] * s[i]));
            sum += g[i];
        }
    }
    tops[wave][lane] = top;
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && n < N) {
        for (int w = 1; w < 4; ++w) {
            top = qr_max(top, tops[w][lane]);
            sum += sums[w][lane];
        }
        A.part_top[(int64_t)by * N + n] = top;
        A.part_sum[(int64_t)by * N + n] = sum;
    }
}

// All that depends on nothing but the call's inputs, in one launch: workgroups [0, b0) row pieces, [b0, b1) column
// partials, [b1, b2) b transposed, [b2, b3) a transposed.  2,048 x 25,088 x 1,024 fp32: 58 us, 0.25 GB at 4.3 TB/s.
template <typename T, int NV>
__global__ void __launch_bounds__(256)
grad_prepare_kernel(const I8Grad A, int b0, int b1, int b2)
{
    __shared__ union {
        int8_t tile[64][68];
        struct {
            uint32_t tops[4][64];
            float sums[4][64];
        };
    } s;
    int b = blockIdx.x;
    if (b < b0) {
        gd_row_pieces<T, NV>(A, (int64_t)b * 4 + (threadIdx.x >> 6));
    } else if (b < b1) {
        b -= b0;
        const int nx = (A.N + 63) / 64;
        gd_col_partials<T>(A, b % nx, b / nx, s.tops, s.sums);
    } else {
        const bool second = b >= b2;
        b -= second ? b2 : b1;
        const int nx = (A.K + 63) / 64;
        if (second) gd_transpose(A.a, A.a_stride, A.M, A.K, A.a_t, A.col_stride, (int64_t)(b / nx) * 64, (int64_t)(b % nx) * 64, s.tile);
        else gd_transpose(A.b, A.b_stride, A.N, A.K, A.b_t, A.row_stride, (int64_t)(b / nx) * 64, (int64_t)(b % nx) * 64, s.tile);
    }
}

// 2,048 x 1,024 fp32 14.0 us, 8,192 x 1,024 bf16 24.6 us: the column's partials, one after the other, are waited for first.
template <typename T>
__global__ void __launch_bounds__(256)
grad_col_pieces_kernel(const I8Grad A, int n_part)
{
    __shared__ __align__(16) _Float16 tile[2][64][68]; // [piece][n][m]
    __shared__ double ups[64];
    __shared__ uint32_t tops[4][64];
    __shared__ float sums[4][64];
    const T *grad = (const T *)A.grad, *y = (const T *)A.y;
    const int64_t m0 = (int64_t)blockIdx.y * 64;
    const int n0 = blockIdx.x * 64, N = A.N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = n0 + lane;
    { // the column's magnitude and sum: a quarter of the partials a wave, the quarters in order
        const int quarter = (n_part + 3) / 4, p0 = wave * quarter, p1 = p0 + quarter < n_part ? p0 + quarter : n_part;
        uint32_t top = 0;
        float sum = 0.0f;
        if (n < N) {
#pragma unroll 8
            for (int p = p0; p < p1; ++p) {
                top = qr_max(top, A.part_top[(int64_t)p * N + n]);
                sum += A.part_sum[(int64_t)p * N + n];
            }
        }
        tops[wave][lane] = top;
        sums[wave][lane] = sum;
    }
    __syncthreads();
    if (wave == 0) {
        uint32_t top = tops[0][lane];
        float sum = sums[0][lane];
        for (int w = 1; w < 4; ++w) {
            top = qr_max(top, tops[w][lane]);
            sum += sums[w][lane];
        }
        const bool finite = top < 0x7f800000u;
        ups[lane] = !finite || top == 0 ? 0.0 : i8_pow2(i8_shift(__uint_as_float(top)));
        if (blockIdx.y == 0 && n < N) {
            A.col_top[n] = finite ? __uint_as_float(top) : __builtin_nanf("");
            if (A.grad_bias) A.grad_bias[n] = sum;
        }
    }
    __syncthreads();
    const double up = ups[lane];
    double v[16]; // rows 16 wave .. 16 wave + 15 of the tile
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t m = m0 + wave * 16 + i;
        v[i] = m < A.M && n < N ? (double)gd_grad(grad, y, m * A.grad_stride + n, m * A.y_stride + n) * (double)A.a_scale[m] : 0.0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        I8Vec<_Float16, 4> h[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) i8_pieces(up != 0.0 ? v[4 * i + j] * up : 0.0, h[0].v[j], h[1].v[j]);
#pragma unroll
        for (int p = 0; p < 2; ++p) __builtin_memcpy(__builtin_assume_aligned(&tile[p][lane][wave * 16 + 4 * i], 8), &h[p], 8);
    }
    __syncthreads();
    const int tn = threadIdx.x >> 2, tm = (threadIdx.x & 3) * 16;
    if (n0 + tn >= N || m0 + tm >= A.col_stride) return;
    for (int p = 0; p < 2; ++p) {
        I8Vec<_Float16, 16> h;
        __builtin_memcpy(&h, __builtin_assume_aligned(&tile[p][tn][tm], 8), 32);
        __builtin_memcpy(__builtin_assume_aligned(A.col_pieces + ((int64_t)p * N + n0 + tn) * A.col_stride + m0 + tm, 32), &h, 32);
    }
}

int frcnn_i8_grad_parts(int M) { return (M + GC_ROWS - 1) / GC_ROWS; }

template <typename T> static int grad_prepare_t(const I8Grad &A, hipStream_t st)
{
    const int nx = (A.N + 63) / 64, kx = (A.K + 63) / 64, mx = (A.M + 63) / 64, parts = frcnn_i8_grad_parts(A.M);
    const int64_t b0 = A.row_pieces ? (A.M + 3) / 4 : 0, b1 = b0 + (A.part_top ? (int64_t)nx * parts : 0),
                  b2 = b1 + (A.b_t ? (int64_t)kx * nx : 0), b3 = b2 + (A.a_t ? (int64_t)kx * mx : 0);
    if (A.N <= 256)
        hipLaunchKernelGGL((grad_prepare_kernel<T, 1>), dim3((unsigned)b3), dim3(256), 0, st, A, (int)b0, (int)b1, (int)b2);
    else
        hipLaunchKernelGGL((grad_prepare_kernel<T, 4>), dim3((unsigned)b3), dim3(256), 0, st, A, (int)b0, (int)b1, (int)b2);
    FRCNN_CHECK_LAUNCH("grad_prepare");
    if (A.part_top) {
        hipLaunchKernelGGL((grad_col_pieces_kernel<T>), dim3(nx, mx), dim3(256), 0, st, A, parts);
        FRCNN_CHECK_LAUNCH("grad_col_pieces");
    }
    return FRCNN_OK;
}

int frcnn_i8_grad_prepare(const I8Grad &A, hipStream_t st)
{
    if (A.type == FRCNN_F32) return grad_prepare_t<float>(A, st);
    if (A.type == FRCNN_BF16) return grad_prepare_t<__bf16>(A, st);
    return grad_prepare_t<_Float16>(A, st);
}
