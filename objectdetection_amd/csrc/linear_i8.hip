// linear_i8.hip -- dense layers on 8-bit integers: out_mn = (sum_k a_mk b_nk) a_scale_m b_scale_n + bias_n, rows of a
// (RoIs) and rows of b (output channels) both contiguous in k, and the two gradient products, which are the same
// product on 24-bit fixed-point gradients (three 8-bit digits, three sums).
//
// The sums are exact: 32-bit integers cannot wrap below 2^17 products of two bytes.  Their order therefore does not
// matter, and splitting k over workgroups changes no bit.  The scales and the bias are applied in 64 bits and the
// result is rounded to fp32 (and from there to 16 bits): the sign a ReLU looks at is the sign of the exact expression.
#include "i8_common.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

#define LI_BK 64           // bytes of k per LDS stage: one matrix instruction deep
#define LI_STAGES 4
#define LI_OOB 0x70000000  // a byte offset beyond every tile: the buffer load returns zeros unread
#define LI_MAX_STRIDE 4000000 // 256 rows of it stay below LI_OOB

struct LiArgs {
    const int8_t *a, *b;
    int64_t a_stride, b_stride, a_plane; // bytes
    const int32_t *n_rows;               // device count of valid rows of a, or NULL
    int M, N, K;
    int tiles_m, tiles_n, k_split;       // k_split: bytes of k per split, a multiple of LI_BK
    const float *a_scale, *b_scale, *bias;
    int relu, out_type;
    void *out;
    int64_t out_stride;                  // elements
    void *partial;                       // per-split sums, or NULL
};

// One result from an exact sum: the scales and the bias in 64 bits, then fp32.
__device__ __forceinline__ float li_finish(double sum, double a_scale, double b_scale, double bias, int relu)
{
    const float z = (float)__builtin_fma(sum * a_scale, b_scale, bias);
    return relu && z < 0.0f ? 0.0f : z; // keeps NaN
}

// sum_p digit_p 2^(8 (2 - p)) of a fixed-point row, or the plain sum
template <int P> __device__ __forceinline__ double li_sum(int d0, int d1, int d2)
{
    const double t = (double)d0;
    return P == 1 ? t : __builtin_fma(t, 65536.0, __builtin_fma((double)d1, 256.0, (double)d2));
}

// Four neighbours (the first `count` of them) in out's type; the address is aligned to one element.
template <typename T> __device__ __forceinline__ void li_store(T *o, const float (&z)[4], int count)
{
    T h[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) h[r] = (T)z[r];
    if (count >= 4) {
        __builtin_memcpy(o, h, sizeof(h));
    } else {
        if (count > 0) o[0] = h[0];
        if (count > 1) o[1] = h[1];
        if (count > 2) o[2] = h[2];
    }
}

// A stage of LDS holds LI_BK = 64 bytes of k for the tile's rows of a (P planes) and of b.  The 16-byte slot of chunk c of
// row r is c ^ swizzle(r).  A 16-byte LDS read serves its lanes in four turns of sixteen, 0-3 with 12-15 and 20-27 first;
// with the lanes on sixteen rows by four chunks this swizzle puts each turn on all 64 banks once (no conflict counted;
// (r >> 2) & 3, which spreads lanes 0-15, doubles the cycles).
__device__ __forceinline__ int li_swz(int r) { return (-(r >> 2)) & 3; }

// Workgroups go to the eight XCDs in turn: neighbours in the tile order go to one XCD, eight tiles of m by all of n, so
// that its L2 sees a row of a and a row of b several times.
__device__ __forceinline__ void li_tile(int tiles_m, int tiles_n, int &tm, int &tn)
{
    const int tiles = tiles_m * tiles_n;
    const int xcd = blockIdx.x & 7, q = tiles >> 3, r = tiles & 7;
    const int l = xcd * q + (xcd < r ? xcd : r) + (blockIdx.x >> 3);
    const int group = l / (8 * tiles_n), rem = l - group * 8 * tiles_n;
    const int gm = tiles_m - group * 8 < 8 ? tiles_m - group * 8 : 8;
    tm = group * 8 + rem % gm;
    tn = rem / gm;
}

// One tile of BM x BN by waves of WM x WN.  k goes by in stages of 64 bytes: global -> LDS directly, LI_STAGES in the
// ring; LDS -> registers one stage ahead of the matrix instructions; so that a load has LI_STAGES - 1 stages to arrive.
template <int BM, int BN, int WM, int WN, int P>
__device__ __forceinline__ void linear_i8_tile(const LiArgs &A)
{
    constexpr int BK = LI_BK;
    constexpr int NW = (BM / WM) * (BN / WN);
    constexpr int TM = WM / 16, TN = WN / 16;
    constexpr int RPL = 1024 / BK, CPR = BK / 16; // rows a load of 64 x 16 bytes covers, chunks of a row
    constexpr int GA = BM / RPL / NW, GB = BN / RPL / NW; // loads a wave issues per stage (and plane)
    constexpr int LPS = GA * P + GB;
    constexpr int STAGE = (P * BM + BN) * BK;
    static_assert(GA * RPL * NW == BM && GB * RPL * NW == BN, "tile rows have to divide over the waves");
    __shared__ __align__(1024) int8_t s0[STAGE];
    __shared__ __align__(1024) int8_t s1[STAGE];
    __shared__ __align__(1024) int8_t s2[STAGE];
    __shared__ __align__(1024) int8_t s3[STAGE];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tile_m, tile_n;
    li_tile(A.tiles_m, A.tiles_n, tile_m, tile_n);
    const int M = i8_rows(A.n_rows, A.M);
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    if (m0 >= M) return;
    const int ks = blockIdx.y * A.k_split;
    const int ke = ks + A.k_split < A.K ? ks + A.k_split : A.K;
    const int rows_a = M - m0 < BM ? M - m0 : BM, rows_b = A.N - n0 < BN ? A.N - n0 : BN;
    const int kp = (A.K + 15) & ~15;

    __amdgpu_buffer_rsrc_t ra[P];
#pragma unroll
    for (int p = 0; p < P; ++p)
        ra[p] = __builtin_amdgcn_make_buffer_rsrc((void *)(A.a + p * A.a_plane + (int64_t)m0 * A.a_stride), 0,
                                                  (int)((rows_a - 1) * A.a_stride) + kp, 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(A.b + (int64_t)n0 * A.b_stride), 0, (int)((rows_b - 1) * A.b_stride) + kp, 0x00020000);
    int va[GA], vb[GB];
    // rows of one wave's loads are RPL apart, a multiple of the swizzle's period or not: the chunk is per load
    int ca[GA], cb[GB];
#pragma unroll
    for (int j = 0; j < GA; ++j) {
        const int r = (wave * GA + j) * RPL + lane / CPR;
        ca[j] = ((lane % CPR) ^ li_swz(r)) * 16;
        va[j] = r * (int)A.a_stride + ca[j];
    }
#pragma unroll
    for (int j = 0; j < GB; ++j) {
        const int r = (wave * GB + j) * RPL + lane / CPR;
        cb[j] = ((lane % CPR) ^ li_swz(r)) * 16;
        vb[j] = r * (int)A.b_stride + cb[j];
    }
    // Load i of a stage.  Chunks at and beyond the end of k are not read: their offset is beyond the buffer and the load
    // stores zeros.  A stage past the end is filled like any other, so that the loads in flight are the same in every step.
    auto fill1 = [&](int8_t *s, int k0, int i) {
        if (i < GA * P) {
            const int j = i % GA, p = i / GA;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra[p], (lds_void *)(s + (p * BM + (wave * GA + j) * RPL) * BK), 16,
                                                     k0 + ca[j] < ke ? va[j] : LI_OOB, k0, 0, 0);
        } else {
            const int j = i - GA * P;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void *)(s + (P * BM + (wave * GB + j) * RPL) * BK), 16,
                                                     k0 + cb[j] < ke ? vb[j] : LI_OOB, k0, 0, 0);
        }
    };
    auto fill = [&](int8_t *s, int k0) {
#pragma unroll
        for (int i = 0; i < LPS; ++i) fill1(s, k0, i);
    };
    // the last chunk of k may hold bytes of whatever follows the row: cleared in a's rows
    auto clear_tail = [&](int8_t *s, int k0) {
        for (int r = threadIdx.x; r < P * BM; r += NW * 64) {
            const int c = (A.K - k0) >> 4;
            int8_t *q = s + r * BK + ((c ^ li_swz(r % BM)) << 4);
            for (int j = A.K & 15; j < 16; ++j) q[j] = 0;
        }
        __syncthreads();
    };
    const int wm0 = (wave % (BM / WM)) * WM, wn0 = (wave / (BM / WM)) * WN;
    const int i16 = lane & 15, q4 = lane >> 4;
    i32x4 acc[P][TM][TN];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) acc[p][tm][tn] = (i32x4){0, 0, 0, 0};
    // b is the instruction's row operand: a lane's four results are neighbours in n
    const int frag = i16 * BK + ((q4 ^ li_swz(i16)) << 4);
    struct Frags {
        i32x4 a[P * TM], b[TN];
    };
    Frags f0, f1;
    auto read1 = [&](Frags &f, const int8_t *s, int i) {
        if (i < TN) f.b[i] = *(const i32x4 *)(s + (P * BM + wn0 + i * 16) * BK + frag);
        else f.a[i - TN] = *(const i32x4 *)(s + ((i - TN) / TM * BM + wm0 + (i - TN) % TM * 16) * BK + frag);
    };
    // One step multiplies the stage that `f` holds, reads the next one, `next`, into `g`, and refills the buffer `cur` that
    // `f` came from.  Behind the wait and the barrier the next stage is complete in every wave (the LI_STAGES - 2 later
    // ones may be in flight) and every wave has read the current one (lgkmcnt).  Reads and loads go out between the matrix
    // instructions, a few behind each group of TN.
    auto step = [&](const Frags &f, Frags &g, int8_t *cur, int8_t *next, int k0) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LPS * (LI_STAGES - 2)) : "memory");
        if (k0 + 2 * BK > A.K && k0 + BK < A.K && (A.K & 15)) clear_tail(next, k0 + BK);
        constexpr int G = P * TM, R = G > 1 ? (P * TM + TN + G - 2) / (G - 1) : P * TM + TN, L = (LPS + G - 1) / G;
#pragma unroll
        for (int t = 0; t < G; ++t) {
#pragma unroll
            for (int tn = 0; tn < TN; ++tn)
                acc[t / TM][t % TM][tn] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.b[tn], f.a[t], acc[t / TM][t % TM][tn], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = t * R; i < (t + 1) * R && i < P * TM + TN; ++i) read1(g, next, i);
#pragma unroll
            for (int i = t * L; i < (t + 1) * L && i < LPS; ++i) fill1(cur, k0 + LI_STAGES * BK, i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    fill(s0, ks);
    fill(s1, ks + BK);
    fill(s2, ks + 2 * BK);
    fill(s3, ks + 3 * BK);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LPS * (LI_STAGES - 1)) : "memory");
    if (ks + BK > A.K && (A.K & 15)) clear_tail(s0, ks);
#pragma unroll
    for (int i = 0; i < P * TM + TN; ++i) read1(f0, s0, i);
    for (int k0 = ks;;) {
        step(f0, f1, s0, s1, k0);
        if ((k0 += BK) >= ke) break;
        step(f1, f0, s1, s2, k0);
        if ((k0 += BK) >= ke) break;
        step(f0, f1, s2, s3, k0);
        if ((k0 += BK) >= ke) break;
        step(f1, f0, s3, s0, k0);
        if ((k0 += BK) >= ke) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the fills past the end, before the LDS is given back

    const int mw = m0 + wm0 + i16, nw = n0 + wn0 + q4 * 4;
    if (A.partial) {
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int m = mw + tm * 16;
            if (m >= M) continue;
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) {
                const int n = nw + tn * 16;
                const int64_t at = ((int64_t)blockIdx.y * A.M + m) * A.N + n;
                if (P == 1) {
                    int32_t *o = (int32_t *)A.partial + at;
                    if (n + 4 <= A.N) __builtin_memcpy(o, &acc[0][tm][tn], 16);
                    else
                        for (int r = 0; r < 4; ++r)
                            if (n + r < A.N) o[r] = acc[0][tm][tn][r];
                } else {
                    for (int r = 0; r < 4; ++r)
                        if (n + r < A.N)
                            ((int64_t *)A.partial)[at + r] = ((int64_t)acc[0][tm][tn][r] << 16) +
                                                             ((int64_t)acc[P > 1 ? 1 : 0][tm][tn][r] << 8) +
                                                             acc[P > 2 ? 2 : 0][tm][tn][r];
                }
            }
        }
        return;
    }
    double sa[TM];
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) {
        sa[tm] = mw + tm * 16 < M ? (double)A.a_scale[mw + tm * 16] : 0.0;
        if (P == 3) sa[tm] *= 1.0 / (double)I8_FIX;
    }
    auto write = [&](auto *out) {
#pragma unroll
        for (int tn = 0; tn < TN; ++tn) {
            const int n = nw + tn * 16;
            double sb[4], bias[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int nr = n + r < A.N ? n + r : A.N - 1;
                sb[r] = P == 1 ? (double)A.b_scale[nr] : 1.0;
                bias[r] = P == 1 && A.bias ? (double)A.bias[nr] : 0.0;
            }
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                const int m = mw + tm * 16;
                float z[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    z[r] = li_finish(li_sum<P>(acc[0][tm][tn][r], acc[P > 1 ? 1 : 0][tm][tn][r], acc[P > 2 ? 2 : 0][tm][tn][r]),
                                     sa[tm], sb[r], bias[r], A.relu);
                if (m < M) li_store(out + (int64_t)m * A.out_stride + n, z, A.N - n);
            }
        }
    };
    if (A.out_type == FRCNN_F32) write((float *)A.out);
    else if (A.out_type == FRCNN_BF16) write((__bf16 *)A.out);
    else write((_Float16 *)A.out);
}

// (The body is a device function: a kernel template with these builtins in it is dropped from the host pass.)
template <int BM, int BN, int WM, int WN, int P, int OCC>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * 64, OCC)
linear_i8_kernel(const LiArgs A)
{
    linear_i8_tile<BM, BN, WM, WN, P>(A);
}

// Joins the sums of a split k.
template <int P>
__global__ void __launch_bounds__(256)
linear_i8_join_kernel(const LiArgs A, int splits)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t MN = (int64_t)A.M * A.N;
    if (i >= MN) return;
    const int m = (int)(i / A.N), n = (int)(i - (int64_t)m * A.N);
    if (m >= i8_rows(A.n_rows, A.M)) return;
    double s;
    if (P == 1) {
        int32_t t = 0;
        for (int k = 0; k < splits; ++k) t += ((const int32_t *)A.partial)[k * MN + i];
        s = (double)t;
    } else {
        int64_t t = 0;
        for (int k = 0; k < splits; ++k) t += ((const int64_t *)A.partial)[k * MN + i];
        s = (double)t;
    }
    const float z = li_finish(s, (double)A.a_scale[m] * (P == 3 ? 1.0 / (double)I8_FIX : 1.0),
                              P == 1 ? (double)A.b_scale[n] : 1.0, P == 1 && A.bias ? (double)A.bias[n] : 0.0, A.relu);
    const int64_t at = (int64_t)m * A.out_stride + n;
    if (A.out_type == FRCNN_F32) ((float *)A.out)[at] = z;
    else if (A.out_type == FRCNN_BF16) ((__bf16 *)A.out)[at] = (__bf16)z;
    else ((_Float16 *)A.out)[at] = (_Float16)z;
}

static size_t up256(size_t v) { return (v + 255) / 256 * 256; }

struct LiPlan {
    int bm, bn, splits, k_split;
};

// Tile by the rows there are; k is split until about every CU has a workgroup, down to 512 bytes each.
static LiPlan li_plan(int M, int N, int K, int P)
{
    LiPlan p;
    p.bm = p.bn = 64;
    if (P == 1 && M <= 32) p.bm = 32;
    else if (P == 1 && (int64_t)((M + 255) / 256) * ((N + 255) / 256) >= 256) p.bm = p.bn = 256;
    else if (M > 64 && N > 64) p.bm = p.bn = 128;
    const int64_t tiles = (int64_t)((M + p.bm - 1) / p.bm) * ((N + p.bn - 1) / p.bn);
    const int steps = (K + LI_BK - 1) / LI_BK;
    int64_t want = tiles >= 256 ? 1 : 256 / tiles;
    const int most = steps / 8 > 0 ? steps / 8 : 1;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int per = (steps + (int)want - 1) / (int)want;
    p.k_split = per * LI_BK;
    p.splits = (steps + per - 1) / per;
    return p;
}

static size_t li_partial_bytes(const LiPlan &p, int M, int N, int P)
{
    return p.splits > 1 ? up256((size_t)p.splits * M * N * (P == 3 ? 8 : 4)) : 0;
}

template <int P> static int li_launch(LiArgs &A, const LiPlan &p, void *partial, hipStream_t st)
{
    A.tiles_m = (A.M + p.bm - 1) / p.bm;
    A.tiles_n = (A.N + p.bn - 1) / p.bn;
    A.k_split = p.k_split;
    A.partial = p.splits > 1 ? partial : nullptr;
    const int64_t tiles = (int64_t)A.tiles_m * A.tiles_n;
    FRCNN_REQUIRE(tiles < (1ll << 31), "linear_i8: too many tiles");
    const dim3 grid((unsigned)tiles, p.splits);
    if (p.bm == 256) {
        hipLaunchKernelGGL((linear_i8_kernel<256, 256, 64, 128, 1, 2>), grid, dim3(512), 0, st, A);
    } else if (p.bm == 128) {
        if (P == 1) hipLaunchKernelGGL((linear_i8_kernel<128, 128, 64, 64, 1, 2>), grid, dim3(256), 0, st, A);
        else hipLaunchKernelGGL((linear_i8_kernel<128, 128, 64, 32, 3, 2>), grid, dim3(512), 0, st, A);
    } else if (p.bm == 64) {
        hipLaunchKernelGGL((linear_i8_kernel<64, 64, 32, 32, P, 1>), grid, dim3(256), 0, st, A);
    } else {
        hipLaunchKernelGGL((linear_i8_kernel<32, 64, 32, 32, 1, 1>), grid, dim3(128), 0, st, A);
    }
    FRCNN_CHECK_LAUNCH("linear_i8");
    if (p.splits > 1) {
        const int64_t MN = (int64_t)A.M * A.N;
        hipLaunchKernelGGL((linear_i8_join_kernel<P>), dim3((unsigned)((MN + 255) / 256)), dim3(256), 0, st, A, p.splits);
        FRCNN_CHECK_LAUNCH("linear_i8_join");
    }
    return FRCNN_OK;
}

// ---- entry points ------------------------------------------------------------------------------------------------------
static int64_t li_stride(int K) { return ((int64_t)K + 15) / 16 * 16; }

// Rows that the kernel reads in place: 16-byte aligned, and not overlapping.  (The last chunk of a row may reach up to 15
// bytes beyond K; it is aligned like the row's start, so it lies in the same 16 bytes as the row's last element.)
static bool li_in_place(const void *p, int64_t stride, int K)
{
    return ((uintptr_t)p & 15) == 0 && (stride & 15) == 0 && stride >= K && stride <= LI_MAX_STRIDE;
}

static bool li_shape_ok(int M, int N, int K) { return M >= 0 && N > 0 && K > 0 && K <= I8_MAX_K && (int64_t)M * N < (1ll << 40); }

extern "C" size_t frcnn_matmul_i8_workspace_bytes(int M, int N, int K)
{
    if (!li_shape_ok(M, N, K) || M == 0) return 0;
    // rows of a and b copied to an aligned stride where the caller's are not, and the sums of a split k
    return up256((size_t)M * li_stride(K)) + up256((size_t)N * li_stride(K)) + li_partial_bytes(li_plan(M, N, K, 1), M, N, 1);
}

extern "C" int frcnn_matmul_i8(const int8_t *a, int64_t a_stride, const float *a_scale, const int8_t *b, int64_t b_stride,
                               const float *b_scale, const float *bias, int relu, int M, int N, int K,
                               const int32_t *n_rows, void *out, int out_type, int64_t out_stride, void *workspace,
                               size_t workspace_bytes, void *stream)
{
    FRCNN_REQUIRE(li_shape_ok(M, N, K), "matmul_i8: bad shape (%d, %d, %d); K is at most %d", M, N, K, I8_MAX_K);
    FRCNN_REQUIRE(i8_type_ok(out_type), "matmul_i8: unknown element type %d", out_type);
    FRCNN_REQUIRE(a_stride >= 0 && b_stride >= 0 && out_stride >= N, "matmul_i8: bad strides");
    if (M == 0) return FRCNN_OK;
    FRCNN_REQUIRE(a && a_scale && b && b_scale && out, "matmul_i8: null pointer");
    hipStream_t st = (hipStream_t)stream;
    const LiPlan p = li_plan(M, N, K, 1);
    char *ws = (char *)workspace;
    const size_t need = frcnn_matmul_i8_workspace_bytes(M, N, K);
    if (workspace_bytes < need || (need && !workspace)) {
        frcnn_set_error("matmul_i8: workspace too small (%zu < %zu)", workspace_bytes, need);
        return FRCNN_EWORKSPACE;
    }
    const int64_t ld = li_stride(K);
    LiArgs A = {};
    if (M == 1) a_stride = ld;
    if (li_in_place(a, a_stride, K)) {
        A.a = a;
        A.a_stride = a_stride;
    } else {
        int rc = frcnn_i8_pad_rows(a, a_stride, M, K, (int8_t *)ws, ld, st);
        if (rc != FRCNN_OK) return rc;
        A.a = (const int8_t *)ws;
        A.a_stride = ld;
    }
    ws += up256((size_t)M * ld);
    if (N == 1) b_stride = ld;
    if (li_in_place(b, b_stride, K)) {
        A.b = b;
        A.b_stride = b_stride;
    } else {
        int rc = frcnn_i8_pad_rows(b, b_stride, N, K, (int8_t *)ws, ld, st);
        if (rc != FRCNN_OK) return rc;
        A.b = (const int8_t *)ws;
        A.b_stride = ld;
    }
    ws += up256((size_t)N * ld);
    A.n_rows = n_rows;
    A.M = M; A.N = N; A.K = K;
    A.a_scale = a_scale; A.b_scale = b_scale; A.bias = bias;
    A.relu = relu; A.out_type = out_type; A.out = out; A.out_stride = out_stride;
    return li_launch<1>(A, p, ws, st);
}

extern "C" size_t frcnn_linear_i8_workspace_bytes(int M, int N, int K)
{
    if (!li_shape_ok(M, N, K) || M == 0) return 0;
    return up256((size_t)M * 4) + up256((size_t)M * li_stride(K)) + frcnn_matmul_i8_workspace_bytes(M, N, K);
}

extern "C" int frcnn_linear_i8(const void *x, int x_type, int64_t x_stride, const int8_t *b, int64_t b_stride,
                               const float *b_scale, const float *bias, int relu, int M, int N, int K,
                               const int32_t *n_rows, void *out, int out_type, int64_t out_stride, void *workspace,
                               size_t workspace_bytes, void *stream)
{
    FRCNN_REQUIRE(li_shape_ok(M, N, K), "linear_i8: bad shape (%d, %d, %d); K is at most %d", M, N, K, I8_MAX_K);
    if (M == 0) return FRCNN_OK;
    const size_t need = frcnn_linear_i8_workspace_bytes(M, N, K);
    if (workspace_bytes < need || !workspace) {
        frcnn_set_error("linear_i8: workspace too small (%zu < %zu)", workspace_bytes, need);
        return FRCNN_EWORKSPACE;
    }
    char *ws = (char *)workspace;
    float *a_scale = (float *)ws;
    int8_t *a = (int8_t *)(ws + up256((size_t)M * 4));
    char *rest = (char *)a + up256((size_t)M * li_stride(K));
    int rc = frcnn_quantize_rows_i8(x, x_type, x_stride, M, K, n_rows, a, li_stride(K), a_scale, stream);
    if (rc != FRCNN_OK) return rc;
    return frcnn_matmul_i8(a, li_stride(K), a_scale, b, b_stride, b_scale, bias, relu, M, N, K, n_rows, out, out_type,
                           out_stride, rest, workspace_bytes - (size_t)(rest - ws), stream);
}

// Workspace of the gradients: for dL/dx the digits (3, M, N), their magnitudes, b transposed (K, N) and the sums of a
// split; for dL/dw the digits (3, N, M), magnitudes, column partials, a transposed (K, M) and the sums of a split.
struct LiGrad {
    size_t digits, top, col_sum, partials, other, split, total;
    LiPlan plan;
};

static LiGrad li_grad_plan(int rows, int cols, int inner, size_t partials)
{ // a product (rows, cols) over `inner`
    LiGrad g;
    const size_t ld = (size_t)li_stride(inner);
    size_t off = 0;
    g.plan = li_plan(rows, cols, inner, 3);
    g.digits = off; off += up256(3 * (size_t)rows * ld);
    g.top = off; off += up256((size_t)rows * 4);
    g.col_sum = off; off += up256((size_t)rows * 4);
    g.partials = off; off += up256(partials);
    g.other = off; off += up256((size_t)cols * ld);
    g.split = off; off += li_partial_bytes(g.plan, rows, cols, 3);
    g.total = off;
    return g;
}

extern "C" size_t frcnn_linear_i8_backward_workspace_bytes(int M, int N, int K)
{
    if (M <= 0 || N <= 0 || K <= 0 || M > I8_MAX_K || N > I8_MAX_K || K > I8_MAX_K) return 0;
    const size_t x = li_grad_plan(M, K, N, 0).total, w = li_grad_plan(N, K, M, frcnn_i8_grad_col_partials(M, N)).total;
    return x > w ? x : w;
}

extern "C" int frcnn_linear_i8_backward(const void *grad, int grad_type, int64_t grad_stride, const void *y,
                                        int64_t y_stride, const int8_t *a, int64_t a_stride, const float *a_scale,
                                        const int8_t *b, int64_t b_stride, const float *b_scale, int M, int N, int K,
                                        void *grad_x, int grad_x_type, void *grad_w, int grad_w_type, float *grad_bias,
                                        void *workspace, size_t workspace_bytes, void *stream)
{
    FRCNN_REQUIRE(M > 0 && N > 0 && K > 0 && M <= I8_MAX_K && N <= I8_MAX_K && K <= I8_MAX_K,
                  "linear_i8_backward: bad shape (%d, %d, %d); each is at most %d", M, N, K, I8_MAX_K);
    FRCNN_REQUIRE(i8_type_ok(grad_type) && i8_type_ok(grad_x_type) && i8_type_ok(grad_w_type),
                  "linear_i8_backward: unknown element type");
    FRCNN_REQUIRE(grad && a && a_scale && b && b_scale, "linear_i8_backward: null pointer");
    FRCNN_REQUIRE(grad_stride >= 0 && y_stride >= 0 && a_stride >= 0 && b_stride >= 0, "linear_i8_backward: bad strides");
    const size_t need = frcnn_linear_i8_backward_workspace_bytes(M, N, K);
    if (workspace_bytes < need || !workspace) {
        frcnn_set_error("linear_i8_backward: workspace too small (%zu < %zu)", workspace_bytes, need);
        return FRCNN_EWORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
    if (grad_x) {
        const LiGrad g = li_grad_plan(M, K, N, 0);
        const int64_t ld = li_stride(N), plane = (int64_t)M * ld;
        int rc = frcnn_i8_grad_row_digits(grad, grad_type, grad_stride, y, y_stride, b_scale, M, N, (int8_t *)(ws + g.digits),
                                          ld, plane, (float *)(ws + g.top), st);
        if (rc != FRCNN_OK) return rc;
        rc = frcnn_i8_transpose(b, b_stride, N, K, (int8_t *)(ws + g.other), ld, st);
        if (rc != FRCNN_OK) return rc;
        LiArgs A = {};
        A.a = (const int8_t *)(ws + g.digits); A.a_stride = ld; A.a_plane = plane;
        A.b = (const int8_t *)(ws + g.other); A.b_stride = ld;
        A.M = M; A.N = K; A.K = N;
        A.a_scale = (const float *)(ws + g.top);
        A.out = grad_x; A.out_type = grad_x_type; A.out_stride = K;
        rc = li_launch<3>(A, g.plan, ws + g.split, st);
        if (rc != FRCNN_OK) return rc;
    }
    if (grad_w || grad_bias) { // the bias gradient is a by-product of the columns' magnitudes
        const LiGrad g = li_grad_plan(N, K, M, frcnn_i8_grad_col_partials(M, N));
        const int64_t ld = li_stride(M), plane = (int64_t)N * ld;
        int rc = frcnn_i8_grad_col_digits(grad, grad_type, grad_stride, y, y_stride, a_scale, M, N, (int8_t *)(ws + g.digits),
                                          ld, plane, (float *)(ws + g.top), grad_bias, ws + g.partials, st);
        if (rc != FRCNN_OK) return rc;
        if (!grad_w) return FRCNN_OK;
        rc = frcnn_i8_transpose(a, a_stride, M, K, (int8_t *)(ws + g.other), ld, st);
        if (rc != FRCNN_OK) return rc;
        LiArgs A = {};
        A.a = (const int8_t *)(ws + g.digits); A.a_stride = ld; A.a_plane = plane;
        A.b = (const int8_t *)(ws + g.other); A.b_stride = ld;
        A.M = N; A.N = K; A.K = M;
        A.a_scale = (const float *)(ws + g.top);
        A.out = grad_w; A.out_type = grad_w_type; A.out_stride = K;
        rc = li_launch<3>(A, g.plan, ws + g.split, st);
        if (rc != FRCNN_OK) return rc;
    }
    return FRCNN_OK;
}
