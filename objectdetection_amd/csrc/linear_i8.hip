// linear_i8.hip -- dense layers on 8-bit integers: out_mn = (sum_k a_mk b_nk) a_scale_m b_scale_n + bias_n, rows of a
// (RoIs) and rows of b (output channels) both contiguous in k, and the two gradient products, which go through the same
// tiles in fp16: a gradient's factor in two pieces (i8_pieces), a code as it is, sums in fp32 that are joined in 64 bits.
//
// The layer's sums are exact: 32-bit integers cannot wrap below 2^17 products of two bytes.  Their order therefore does
// not matter, and splitting k over workgroups changes no bit.  The gradients' sums have one fixed order for a size.  The scales and the bias are applied in 64 bits and the
// result is rounded to fp32 (and from there to 16 bits): the sign a ReLU looks at is the sign of the exact expression.
#include "i8_common.h"
#include <type_traits>

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

#define LI_BK 64           // bytes of k per LDS stage: one matrix instruction deep
#define LI_STAGES 4
#define LI_OOB 0x70000000  // a byte offset beyond every tile: the buffer load returns zeros unread
#define LI_MAX_STRIDE 4000000 // 256 rows of it stay below LI_OOB

struct LiArgs {
    const int8_t *a, *b;
    int64_t a_stride, b_stride, a_plane; // bytes
    const int32_t *n_rows;               // device count of valid rows of a, or NULL
    int M, N, K;                         // K: bytes of a row's k (two pieces: two a number, zeros up to a multiple of 32)
    int tiles_m, tiles_n, k_split;       // k_split: bytes of k per split, a multiple of LI_BK
    const float *a_scale, *b_scale, *bias;
    int out_type;
    float low;                           // ReLU: the largest fp32 number that out's type rounds to zero; none: NaN
    bool stream;                         // results stored past the caches
    void *out;
    int64_t out_stride;                  // elements
    void *partial;                       // sums of a split k, (splits, M, li_ld4(N)) int32 (P = 2: double), or NULL
    int splits;
    int n_group;                         // short rows: output channels of a workgroup
};

// Row length of a split's sums: quads of neighbours are stored whole
__host__ __device__ __forceinline__ int li_ld4(int N) { return (N + 3) & ~3; }

// One result from an exact sum: the scales' product is exact in 64 bits (24 bits each; sum times scale would take up to 55), so
// that sum, scales and bias are rounded once, to 64 bits, and keep the exact expression's sign; then fp32.
// Behind a ReLU a zero tells what it was: -0 for a positive result that the output's type rounds to zero (`low`: the largest
// number that it does; NaN without a ReLU, so that one comparison decides), +0 for what the ReLU cut off.  Both are equal to
// zero; the backward call reads the difference.
__device__ __forceinline__ float li_finish(double sum, double a_scale, double b_scale, double bias, float low)
{
    const double zd = __builtin_fma(sum, a_scale * b_scale, bias);
    const float z = (float)zd;
    // zd > 0 by its upper half: fp32 scales and biases leave nothing between 0 and 2^-1022
    const float zero = __double2hiint(zd) > 0 ? -0.0f : 0.0f;
    return z <= low ? zero : z; // keeps NaN
}

// P: planes of a.  1: bytes, whole-number sums.  2: the pieces of a gradient's factor, fp32 sums.
template <int P> struct LiAcc { typedef i32x4 type; };
template <> struct LiAcc<2> { typedef f32x4 type; };
__device__ __forceinline__ double li_sum(int s) { return (double)s; }
__device__ __forceinline__ double li_sum(float hi, float lo) { return __builtin_fma((double)lo, 1.0 / I8_LO, (double)hi); }

// One step of a tile, 64 bytes of k
__device__ __forceinline__ i32x4 li_mfma(i32x4 b, i32x4 a, i32x4 acc) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, acc, 0, 0, 0); }
__device__ __forceinline__ f32x4 li_mfma(i32x4 b, i32x4 a, f32x4 acc)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), acc, 0, 0, 0);
}

// What a row's sum is multiplied by: its scale, or the way back from i8_shift (NaN for a row that is not finite)
template <int P> __device__ __forceinline__ double li_row_scale(float s)
{
    return P == 1 || s != s ? (double)s : i8_pow2(-i8_shift(s));
}

// V neighbours (the first `count` of them) in out's type; the address is aligned to one element.  STREAM: past the caches;
// only where rows lie on 64 bytes, so that the 64 bytes which four lanes store are whole (pieces of 32 take twice as long).
template <bool STREAM = false, typename T, int V> __device__ __forceinline__ void li_store(T *o, const float (&z)[V], int count)
{
    typedef int words __attribute__((ext_vector_type(V * sizeof(T) / 4), aligned(sizeof(T))));
    T h[V];
#pragma unroll
    for (int r = 0; r < V; ++r) h[r] = (T)z[r];
    if (count >= V) {
        words q;
        __builtin_memcpy(&q, h, sizeof(h));
        if constexpr (STREAM && sizeof(h) == 16) __builtin_nontemporal_store(q, (words *)o);
        else *(words *)o = q;
    } else {
#pragma unroll
        for (int r = 0; r < V - 1; ++r)
            if (r < count) o[r] = h[r];
    }
}

__device__ __forceinline__ void li_store_as(const LiArgs &A, int64_t at, float z)
{
    if (A.out_type == FRCNN_F32) ((float *)A.out)[at] = z;
    else if (A.out_type == FRCNN_BF16) ((__bf16 *)A.out)[at] = (__bf16)z;
    else ((_Float16 *)A.out)[at] = (_Float16)z;
}

// A stage of LDS holds LI_BK = 64 bytes of k for the tile's rows of a (P planes) and of b.  The 16-byte slot of chunk c of
// row r is c ^ swizzle(r).  A 16-byte LDS read serves its lanes in four turns of sixteen, 0-3 with 12-15 and 20-27 first;
// with the lanes on sixteen rows by four chunks this swizzle puts each turn on all 64 banks once (no conflict counted;
// (r >> 2) & 3, which spreads lanes 0-15, doubles the cycles).
__device__ __forceinline__ int li_swz(int r) { return (-(r >> 2)) & 3; }

// Workgroups go to the eight XCDs in turn: neighbours in the tile order go to one XCD, eight tiles of m by all of n, so
// that its L2 sees a row of a and a row of b several times.
__device__ __forceinline__ void li_tile(int block, int tiles_m, int tiles_n, int &tm, int &tn)
{
    const int tiles = tiles_m * tiles_n;
    const int xcd = block & 7, q = tiles >> 3, r = tiles & 7;
    const int l = xcd * q + (xcd < r ? xcd : r) + (block >> 3);
    const int group = l / (8 * tiles_n), rem = l - group * 8 * tiles_n;
    const int gm = tiles_m - group * 8 < 8 ? tiles_m - group * 8 : 8;
    tm = group * 8 + rem % gm;
    tn = rem / gm;
}

// Many rows of a product are bound by the clock under load: 32,000 x 25,088 x 1,024 by 256 x 256 tiles takes 684-719 us
// (from card to card), 2.29-2.40 POPS, with the matrix pipes busy in 55 % of the cycles at 2.05 GHz (zeros for operands and no
// traffic: 447 us where this took 712).  At k = 1,024 (to bf16, 47-56 us) the stores and the 64-bit epilogue, which nothing overlaps with one
// workgroup a CU, take the larger part; 2,000 x 12,544 x 1,024 by 128 x 128 in two splits takes 38 us and 9 to join.
// Tried: 32 x 32 x 32 instructions 711 -> 744 us; 128 x 256 tiles in a ring of three stages, two workgroups a CU,
// 688 -> 874 us (45 -> 50 at k = 1,024); 128 x 128 a wave spills.
//
// One tile of BM x BN by waves of WM x WN.  k goes by in stages of 64 bytes: global -> LDS directly, LI_STAGES in the
// ring; LDS -> registers one stage ahead of the matrix instructions; so that a load has LI_STAGES - 1 stages to arrive.
template <int BM, int BN, int WM, int WN, int P>
__device__ __forceinline__ void linear_i8_tile(const LiArgs &A, int block, int split)
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
    li_tile(block, A.tiles_m, A.tiles_n, tile_m, tile_n);
    const int M = i8_rows(A.n_rows, A.M);
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    if (m0 >= M) return;
    const int ks = split * A.k_split;
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
    // A lane's results of one 16 x 16 tile are four neighbours in n.  For 16-bit results the rows of b are dealt out so that
    // those of two tiles make eight neighbours: 16 bytes a lane and 64 a row, as four of 32 bits are.
    const bool pairs = TN % 2 == 0 && A.out_type != FRCNN_F32 && A.splits == 1;
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
        const int n = pairs ? (r & ~31) + ((r >> 2) & 3) * 8 + ((r >> 4) & 1) * 4 + (r & 3) : r;
        vb[j] = n * (int)A.b_stride + cb[j];
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
    typedef typename LiAcc<P>::type Acc;
    Acc acc[P][TM][TN];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) acc[p][tm][tn] = (Acc){0, 0, 0, 0};
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
                acc[t / TM][t % TM][tn] = li_mfma(f.b[tn], f.a[t], acc[t / TM][t % TM][tn]);
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

    auto sum = [&](int tm, int tn, int r) {
        if constexpr (P == 1) return li_sum(acc[0][tm][tn][r]);
        else return li_sum(acc[0][tm][tn][r], acc[1][tm][tn][r]);
    };
    const int mw = m0 + wm0 + i16, nw = n0 + wn0 + q4 * 4;
    if (A.splits > 1) {
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int m = mw + tm * 16;
            if (m >= M) continue;
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) {
                const int n = nw + tn * 16;
                if (n >= A.N) continue;
                const int64_t at = ((int64_t)split * A.M + m) * li_ld4(A.N) + n;
                if constexpr (P == 1) {
                    *(i32x4 *)((int32_t *)A.partial + at) = acc[0][tm][tn];
                } else {
                    double v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = sum(tm, tn, r);
                    __builtin_memcpy(__builtin_assume_aligned((double *)A.partial + at, 16), v, 32);
                }
            }
        }
        return;
    }
    double sa[TM];
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) sa[tm] = mw + tm * 16 < M ? li_row_scale<P>(A.a_scale[mw + tm * 16]) : 0.0;
    auto write = [&](auto *out, auto stream) {
        constexpr int PT = sizeof(*out) == 2 && TN % 2 == 0 ? 2 : 1, V = 4 * PT; // tiles a store takes
#pragma unroll
        for (int tn = 0; tn < TN; tn += PT) {
            const int n = n0 + wn0 + tn * 16 + q4 * V;
            double sb[V], bias[V];
#pragma unroll
            for (int r = 0; r < V; ++r) {
                const int nr = n + r < A.N ? n + r : A.N - 1;
                sb[r] = P == 1 ? (double)A.b_scale[nr] : 1.0;
                bias[r] = P == 1 && A.bias ? (double)A.bias[nr] : 0.0;
            }
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                const int m = mw + tm * 16;
                float z[V];
#pragma unroll
                for (int r = 0; r < V; ++r) z[r] = li_finish(sum(tm, tn + r / 4, r % 4), sa[tm], sb[r], bias[r], A.low);
                if (m < M) li_store<decltype(stream)::value>(out + (int64_t)m * A.out_stride + n, z, A.N - n);
            }
        }
    };
    auto write_as = [&](auto *out) { // (two copies: a choice at each store is merged into plain stores)
        if (A.stream) write(out, std::true_type{});
        else write(out, std::false_type{});
    };
    if (A.out_type == FRCNN_F32) write_as((float *)A.out);
    else if (A.out_type == FRCNN_BF16) write_as((__bf16 *)A.out);
    else write_as((_Float16 *)A.out);
}

// (The body is a device function: a kernel template with these builtins in it is dropped from the host pass.)
template <int BM, int BN, int WM, int WN, int P, int OCC>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * 64, OCC)
linear_i8_kernel(const LiArgs A)
{
    linear_i8_tile<BM, BN, WM, WN, P>(A, blockIdx.x, blockIdx.y);
}

// Two fp16 products for each of the gradient's: 2,048 x 25,088 x 1,024 (both, 0.42 TFLOP) 390-440 us, 0.95-1.08 PFLOP/s, by
// 128 x 256 (the registers and the LDS of the layer's 256 x 256, whose matrix instructions take as long); 8,192 x 1,024 x
// 1,024 82 us, 0.84 PFLOP/s, by 64 x 128.  A large library product in fp16 reaches 1.15 PFLOP/s.
// Both gradients' products in one launch: the first `blocks` workgroups are A's (tiles of a split next to each other), the
// rest B's.
template <int BM, int BN, int WM, int WN, int OCC>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * 64, OCC)
linear_i8_grad_kernel(const LiArgs A, const LiArgs B, int blocks)
{
    const bool second = (int)blockIdx.x >= blocks;
    const LiArgs &R = second ? B : A;
    const int i = second ? blockIdx.x - blocks : blockIdx.x, tiles = R.tiles_m * R.tiles_n;
    linear_i8_tile<BM, BN, WM, WN, 2>(R, i % tiles, i / tiles);
}

// Joins the sums of a split k: a lane takes four neighbours.  2,000 x 1,024 of two splits 8.8 us, 2,048 x 1,024 of eight 16 us
// (4.7 TB/s): bound by the sums' way in.  (Letting the split that arrives last do this, behind a
// device-scope fence, was tried: the fence writes back the whole L2 and the product of 2,000 x 12,544 x 1,024 went from 44
// to 165 us.)
template <int P> __device__ __forceinline__ void linear_i8_join(const LiArgs &A, int64_t i)
{
    const int quads = li_ld4(A.N) / 4;
    const int m = (int)(i / quads), n = (int)(i % quads) * 4;
    if (m >= i8_rows(A.n_rows, A.M)) return;
    const int64_t step = (int64_t)A.M * quads;
    typedef typename std::conditional<P == 1, int64_t, double>::type Sum;
    Sum t[4] = {0, 0, 0, 0};
#pragma unroll 8
    for (int k = 0; k < A.splits; ++k) {
        if constexpr (P == 1) {
            const i32x4 v = ((const i32x4 *)A.partial)[k * step + i];
#pragma unroll
            for (int r = 0; r < 4; ++r) t[r] += v[r];
        } else {
            double v[4];
            __builtin_memcpy(v, __builtin_assume_aligned((const double *)A.partial + (k * step + i) * 4, 16), 32);
#pragma unroll
            for (int r = 0; r < 4; ++r) t[r] += v[r];
        }
    }
    const double a_scale = li_row_scale<P>(A.a_scale[m]);
    float z[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int nr = n + r < A.N ? n + r : A.N - 1;
        z[r] = li_finish((double)t[r], a_scale, P == 1 ? (double)A.b_scale[nr] : 1.0,
                         P == 1 && A.bias ? (double)A.bias[nr] : 0.0, A.low);
    }
    const int64_t at = (int64_t)m * A.out_stride + n;
    if (A.out_type == FRCNN_F32) li_store((float *)A.out + at, z, A.N - n);
    else if (A.out_type == FRCNN_BF16) li_store((__bf16 *)A.out + at, z, A.N - n);
    else li_store((_Float16 *)A.out + at, z, A.N - n);
}

__global__ void __launch_bounds__(64) linear_i8_join_kernel(const LiArgs A)
{
    linear_i8_join<1>(A, (int64_t)blockIdx.x * 64 + threadIdx.x);
}

__global__ void __launch_bounds__(64) linear_i8_grad_join_kernel(const LiArgs A, const LiArgs B, int blocks)
{
    const bool second = (int)blockIdx.x >= blocks;
    linear_i8_join<2>(second ? B : A, (int64_t)(second ? blockIdx.x - blocks : blockIdx.x) * 64 + threadIdx.x);
}

// ---- a few rows -----------------------------------------------------------------------------------------------------
// One launch from float rows (or codes) to the result: a workgroup takes LF_N output channels and all of k.  A thread owns
// the 16-byte chunks t, t + 1024, ... of k, of the weight rows and of x alike, so that it needs nothing of its neighbours but
// the row's maximum and the final sum; the weights, which are all there is to read, stay in its registers for every row of
// x.  Each workgroup quantises x for itself, out of the L2.  One row of 12,544 by 1,024 channels: 6.2 us for 12.9 MB
// (2.1 TB/s); a chain of load, maximum over the workgroup, codes and sum over the workgroup bounds it.
#define LF_THREADS 1024
#define LF_N 4
#define LF_CHUNKS 2 // of a thread: k up to 32,768

template <typename T>
__global__ void __launch_bounds__(LF_THREADS)
linear_i8_few_kernel(const T *__restrict__ x, int64_t x_stride, const float *__restrict__ x_scale, const LiArgs A)
{
    __shared__ uint32_t red[LF_THREADS / 64];
    __shared__ int sums[LF_THREADS / 64][LF_N];
    const int n0 = blockIdx.x * LF_N, t = threadIdx.x, K = A.K;
    const int kf = K & ~15, tail = kf + t < K && t < 16; // the last K % 16 elements: one a lane of the first wave
    i32x4 w[LF_N][LF_CHUNKS];
    int w_tail[LF_N];
#pragma unroll
    for (int r = 0; r < LF_N; ++r) {
        const int8_t *b = A.b + (int64_t)(n0 + r < A.N ? n0 + r : A.N - 1) * A.b_stride;
#pragma unroll
        for (int i = 0; i < LF_CHUNKS; ++i) {
            const int k = (i * LF_THREADS + t) * 16;
            w[r][i] = (i32x4){0, 0, 0, 0};
            if (k < kf) __builtin_memcpy(&w[r][i], b + k, 16);
        }
        w_tail[r] = tail ? b[kf + t] : 0;
    }
    const int M = i8_rows(A.n_rows, A.M);
#pragma unroll 1
    for (int m = 0; m < M; ++m) {
        i32x4 q[LF_CHUNKS];
        int q_tail = 0;
        float scale;
        const T *xr = x + m * x_stride;
        if constexpr (sizeof(T) == 1) {
#pragma unroll
            for (int i = 0; i < LF_CHUNKS; ++i) {
                const int k = (i * LF_THREADS + t) * 16;
                q[i] = (i32x4){0, 0, 0, 0};
                if (k < kf) __builtin_memcpy(&q[i], xr + k, 16);
            }
            if (tail) q_tail = xr[kf + t];
            scale = x_scale[m];
        } else {
            I8Vec<T, 16> v[LF_CHUNKS];
            uint32_t top_bits = 0;
            float v_tail = tail ? (float)xr[kf + t] : 0.0f;
#pragma unroll
            for (int i = 0; i < LF_CHUNKS; ++i) {
                const int k = (i * LF_THREADS + t) * 16;
                if (k < kf) v[i] = i8_load<T, 16>(xr + k);
            }
            top_bits = qr_bits(v_tail);
#pragma unroll
            for (int i = 0; i < LF_CHUNKS; ++i)
                if ((i * LF_THREADS + t) * 16 < kf)
#pragma unroll
                    for (int j = 0; j < 16; ++j) top_bits = qr_max(top_bits, qr_bits((float)v[i].v[j]));
            const QrRow row = qr_row(qr_block_max<LF_THREADS>(top_bits, red));
            scale = row.scale;
            if (__builtin_expect(row.far, 0)) {
                v_tail = qr_lift(v_tail, row);
#pragma unroll
                for (int i = 0; i < LF_CHUNKS; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[i].v[j] = qr_lift(v[i].v[j], row);
            }
            if (!row.none) q_tail = qr_code(v_tail, row);
#pragma unroll
            for (int i = 0; i < LF_CHUNKS; ++i) {
                q[i] = (i32x4){0, 0, 0, 0};
                if ((i * LF_THREADS + t) * 16 < kf && !row.none)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        q[i][j] = (int)qr_pack(qr_code((float)v[i].v[4 * j], row), qr_code((float)v[i].v[4 * j + 1], row),
                                               qr_code((float)v[i].v[4 * j + 2], row), qr_code((float)v[i].v[4 * j + 3], row));
            }
        }
        int sum[LF_N];
#pragma unroll
        for (int r = 0; r < LF_N; ++r) {
            sum[r] = q_tail * w_tail[r];
#pragma unroll
            for (int i = 0; i < LF_CHUNKS; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[r] = __builtin_amdgcn_sdot4(q[i][j], w[r][i][j], sum[r], false);
            for (int o = 32; o > 0; o >>= 1) sum[r] += __shfl_xor(sum[r], o);
        }
        if ((t & 63) == 0)
#pragma unroll
            for (int r = 0; r < LF_N; ++r) sums[t >> 6][r] = sum[r];
        __syncthreads();
        if (t < LF_N && n0 + t < A.N) {
            int total = 0;
            for (int v = 0; v < LF_THREADS / 64; ++v) total += sums[v][t];
            const int n = n0 + t;
            const float z = li_finish((double)total, (double)scale, (double)A.b_scale[n], A.bias ? (double)A.bias[n] : 0.0, A.low);
            li_store_as(A, m * A.out_stride + n, z);
        }
        __syncthreads(); // red and sums are the next row's
    }
}

// ---- short rows ------------------------------------------------------------------------------------------------------
// For k up to LR_K the codes of BM rows stay in LDS: one launch, x read once, no codes in memory.  First each wave quantises
// its BM / 8 rows, up to four at a time so that their chains of dependent operations overlap; then it multiplies all BM rows
// with 16 output channels of its own, whose weights it takes straight from the L2 into registers (no two waves of a workgroup
// want the same ones), LR_AHEAD steps ahead.  blockIdx.y: a group of output channels; with few rows the groups are what
// fills the chip, and each quantises for itself.  32,000 rows of 1,024 fp32 by 105 channels: 36.6 us, 145 MB at 4.0 TB/s;
// a workgroup reads and then multiplies, and two of them a CU overlap only in part.
#define LR_THREADS 512
#define LR_K 1024
#define LR_AHEAD 8

// 16-byte slot of chunk c in row r: rows lie a multiple of 256 bytes apart, the sixteen rows a matrix instruction reads
// differ in the slot instead
__device__ __forceinline__ int lr_slot(int c, int r) { return (c & ~15) | ((c ^ r) & 15); }

template <typename T, int BM>
__device__ __forceinline__ void linear_i8_short(const T *__restrict__ x, int64_t x_stride, const LiArgs &A)
{
    constexpr int NW = LR_THREADS / 64, TM = BM / 16, V = 16 / sizeof(T), D = LR_AHEAD;
    constexpr int ROWS = BM / NW < 4 ? BM / NW : 4;
    constexpr int NV = LR_K / (64 * V); // loads of a lane per row
    extern __shared__ __align__(1024) int8_t codes[]; // BM rows of kp bytes
    __shared__ float scales[BM];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int M = i8_rows(A.n_rows, A.M), K = A.K;
    const int m0 = blockIdx.x * BM;
    if (m0 >= M) return;
    const int rows = M - m0 < BM ? M - m0 : BM;
    const int kp = (K + 255) & ~255, steps = (K + 63) >> 6;
    const int kf = K - K % V, tail = kf + lane < K && lane < V; // whole vectors up to kf; the last K % V elements one a lane
    // rows wave, wave + NW, ...; a row behind the last is the last again: nothing of it is stored
#pragma unroll 1
    for (int batch = 0; batch < BM / (NW * ROWS) && batch * ROWS * NW + wave < rows; ++batch) {
        I8Vec<T, V> v[ROWS][NV];
        T v_tail[ROWS];
        uint32_t top_bits[ROWS];
#pragma unroll
        for (int g = 0; g < ROWS; ++g) {
            const int r = (batch * ROWS + g) * NW + wave;
            const T *xr = x + (int64_t)(m0 + (r < rows ? r : rows - 1)) * x_stride;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int k = (i * 64 + lane) * V;
                v[g][i] = I8Vec<T, V>{};
                if (k < kf) v[g][i] = i8_load<T, V>(xr + k);
            }
            v_tail[g] = tail ? xr[kf + lane] : (T)0.0f;
        }
#pragma unroll
        for (int g = 0; g < ROWS; ++g) {
            top_bits[g] = qr_bits((float)v_tail[g]);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) top_bits[g] = qr_max(top_bits[g], qr_bits((float)v[g][i].v[j]));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
#pragma unroll
            for (int g = 0; g < ROWS; ++g) top_bits[g] = qr_max(top_bits[g], __shfl_xor(top_bits[g], o));
#pragma unroll
        for (int g = 0; g < ROWS; ++g) {
            const int r = (batch * ROWS + g) * NW + wave;
            const QrRow q = qr_row(top_bits[g]);
            if (lane == 0) scales[r] = q.scale;
            if (__builtin_expect(q.far, 0)) {
                v_tail[g] = qr_lift(v_tail[g], q);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) v[g][i].v[j] = qr_lift(v[g][i].v[j], q);
            }
            int8_t *row = codes + r * kp;
            if (kf < steps * 64) { // zeros in the last step's 64 bytes, and codes over them
                const int k = (kf & ~63) + lane;
                row[lr_slot(k >> 4, r) * 16 + (k & 15)] = 0;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); // other lanes' codes stay behind these zeros; no instruction
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int k = (i * 64 + lane) * V;
                if (k < kf) {
                    uint32_t p[V / 4];
#pragma unroll
                    for (int j = 0; j < V / 4; ++j) {
                        int c[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[e] = q.none ? 0 : qr_code((float)v[g][i].v[4 * j + e], q);
                        p[j] = qr_pack(c[0], c[1], c[2], c[3]);
                    }
                    __builtin_memcpy(__builtin_assume_aligned(row + lr_slot(k >> 4, r) * 16 + (k & 15), V), p, V);
                }
            }
            if (tail)
                row[lr_slot((kf + lane) >> 4, r) * 16 + ((kf + lane) & 15)] = (int8_t)(q.none ? 0 : qr_code((float)v_tail[g], q));
        }
    }
    __syncthreads();
    const int i16 = lane & 15, q4 = lane >> 4;
    const int n_end = A.n_group * (blockIdx.y + 1) < A.N ? A.n_group * (blockIdx.y + 1) : A.N;
    const int full = K >> 6; // steps of 64 whole; K & 63: one more, cut
    double sa[TM];
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) sa[tm] = (double)scales[tm * 16 + i16];
    for (int n0 = A.n_group * blockIdx.y + wave * 16; n0 < n_end; n0 += NW * 16) {
        i32x4 fb[D], fl, acc[TM];
        const int8_t *b = A.b + (int64_t)(n0 + i16 < A.N ? n0 + i16 : A.N - 1) * A.b_stride + q4 * 16;
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) acc[tm] = (i32x4){0, 0, 0, 0};
        auto multiply = [&](const i32x4 &f, int step) {
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                const int r = tm * 16 + i16;
                const i32x4 fa = *(const i32x4 *)(codes + r * kp + lr_slot(step * 4 + q4, r) * 16);
                acc[tm] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, fa, acc[tm], 0, 0, 0);
            }
        };
        // The step that K ends in: a's codes are zeros behind K, so only what lies behind the last weight must not be
        // read: such an address is moved back, and the bytes are shifted to where they belong.
        if (K & 63) {
            const int8_t *end = A.b + (int64_t)(A.N - 1) * A.b_stride + K - 16, *p = b + full * 64;
            const int over = p > end ? (int)(p - end) : 0;
            uint64_t h[2];
            __builtin_memcpy(h, p - over, 16);
            const int bits = (over & 7) * 8;
            uint64_t lo = over & 8 ? h[1] : h[0], hi = over & 8 ? 0 : h[1];
            lo = bits ? lo >> bits | hi << (64 - bits) : lo;
            hi >>= bits;
            if (over >= 16) lo = hi = 0;
            fl = (i32x4){(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
        }
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (d < full) __builtin_memcpy(&fb[d], b + d * 64, 16);
        for (int s = 0; s < full; s += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                if (s + d < full) multiply(fb[d], s + d);
                if (s + d + D < full) __builtin_memcpy(&fb[d], b + (s + d + D) * 64, 16);
            }
        }
        if (K & 63) multiply(fl, full);
        auto write = [&](auto *out) {
            const int n = n0 + q4 * 4;
            double sb[4], bias[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int nr = n + r < A.N ? n + r : A.N - 1;
                sb[r] = (double)A.b_scale[nr];
                bias[r] = A.bias ? (double)A.bias[nr] : 0.0;
            }
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                const int m = m0 + tm * 16 + i16;
                float z[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) z[r] = li_finish((double)acc[tm][r], sa[tm], sb[r], bias[r], A.low);
                if (m < M) li_store(out + (int64_t)m * A.out_stride + n, z, n_end - n);
            }
        };
        if (A.out_type == FRCNN_F32) write((float *)A.out);
        else if (A.out_type == FRCNN_BF16) write((__bf16 *)A.out);
        else write((_Float16 *)A.out);
    }
}

template <typename T, int BM>
__global__ void __launch_bounds__(LR_THREADS, 4)
linear_i8_short_kernel(const T *__restrict__ x, int64_t x_stride, const LiArgs A)
{
    linear_i8_short<T, BM>(x, x_stride, A);
}

static size_t up256(size_t v) { return (v + 255) / 256 * 256; }

struct LiPlan {
    int bm, bn, splits, k_split;
    int64_t tiles;
};

// k in `want` parts, as many as come out even, down to `least` stages each; not at all up to `whole` stages.
// LI_SMALL: the tiles of 64.  One launch fewer is worth a few stages one after the other: 99 rows of 2,048 by 1,024 channels
// whole : in four parts 12.3 : 11.3 us on the GPU, 13.2 : 17.1 us a call; both gradients of 512 x 2,048 x 1,000 whole : in two
// parts 39.5 : 42.2 us on the GPU, of 512 x 1,024 x 1,024 32.3 : 31.8.
#define LI_SMALL 16, 32
static LiPlan li_split(int bm, int bn, int M, int N, int K, int64_t want, int least = 8, int whole = 0)
{
    LiPlan p;
    p.bm = bm;
    p.bn = bn;
    p.tiles = (int64_t)((M + bm - 1) / bm) * ((N + bn - 1) / bn);
    const int steps = (K + LI_BK - 1) / LI_BK;
    const int most = steps <= whole || steps < least ? 1 : steps / least;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int per = (steps + (int)want - 1) / (int)want;
    p.k_split = per * LI_BK;
    p.splits = (steps + per - 1) / per;
    return p;
}

// Up to 256 rows: 64 x 64 tiles (32 x 64 up to 32 rows), k split over the CUs; they need half as many splits as larger ones
// (product and join of 99 rows of 12,544, calls replayed in a graph, 13.2 us : 18.7).  Above, 128 x 128 or 256 x 256 by an estimate of the time, in ns:
//   256 x 256, one workgroup a CU: 870 a stage with the whole chip at it (there the clock gives way: 2.3 POPS), 700 at least;
//   128 x 128: 320 a stage for each workgroup of a CU (1.6 POPS);
//   and for a split k the sums' way out and back, at 8 TB/s, and a launch.
// us, 256 : 128, by 1,024 channels: 2,000 rows of 12,544 49 : 44, 4,000 70 : 66, 6,000 90 : 113; of 25,088 2,048 rows 67 : 75,
// 4,000 102 : 123, 6,000 146 : 233; of 6,272 13,000 rows 82 : 124, 20,000 164 : 160; 32,000 rows of 1,024 (to 16 bits) 45 : 61.
static LiPlan li_plan(int M, int N, int K)
{
    if (M <= 256 || N <= 64) {
        const int bm = M <= 32 ? 32 : 64;
        const int64_t tiles = (int64_t)((M + bm - 1) / bm) * ((N + 63) / 64);
        return li_split(bm, 64, M, N, K, 256 / tiles, LI_SMALL);
    }
    LiPlan best = {};
    double least = 0.0;
    for (int side = 128; side <= 256; side *= 2) {
        const int64_t tiles = (int64_t)((M + side - 1) / side) * ((N + side - 1) / side);
        for (int64_t want = 256 / tiles > 1 ? 256 / tiles : 1; want; want = want > 1 ? 1 : 0) {
            const LiPlan p = li_split(side, side, M, N, K, want);
            const int64_t blocks = tiles * p.splits, rounds = (blocks + 255) / 256;
            const double stages = (double)(p.k_split / LI_BK), share = rounds > 1 ? 1.0 : (double)blocks / 256.0;
            double ns = side == 256 ? rounds * (stages * (share * 870.0 > 700.0 ? share * 870.0 : 700.0) + 7000.0)
                                    : rounds * stages * 320.0 + 5000.0;
            if (p.splits > 1) ns += 4000.0 + (2.0 * p.splits + 1.0) * M * N * 4.0 / 8000.0;
            if (best.splits == 0 || ns < least) {
                best = p;
                least = ns;
            }
        }
    }
    return best;
}

// The gradients' tiles: of the same size for both products, so that one launch takes them.  128 x 256 where the two of them
// have 512 such tiles, else 64 x 128.  A whole backward call, us, large : small tiles, M x N x K: 2,048 x 1,024 x 25,088
// 464 : 536, 256 x 1,024 x 25,088 114 : 124, 512 x 1,024 x 12,544 99 : 107, 8,192 x 256 x 4,096 159 : 169; with fewer tiles
// 8,192 x 1,024 x 1,024 144 : 143, 2,048 x 1,024 x 1,024 92 : 58; and with one row of tiles only, 128 x 1,024 x 25,088,
// 110 : 96.
static bool li_grad_large(int M, int N, int K)
{
    return M >= 256 && ((int64_t)((M + 127) / 128) + (N + 127) / 128) * ((K + 255) / 256) >= 512;
}

static LiPlan li_grad_plan(int rows, int cols, int inner, bool large)
{
    if (large) return li_split(128, 256, rows, cols, inner, 256 / ((int64_t)((rows + 127) / 128) * ((cols + 255) / 256)));
    const int bn = cols > 64 ? 128 : 64;
    const int64_t tiles = (int64_t)((rows + 63) / 64) * ((cols + bn - 1) / bn);
    return li_split(64, bn, rows, cols, inner, 256 / tiles, LI_SMALL);
}

static size_t li_split_bytes(const LiPlan &p, int M, int N, int bytes)
{
    return p.splits > 1 ? up256((size_t)p.splits * M * li_ld4(N) * bytes) : 0;
}

static void li_apply(LiArgs &A, const LiPlan &p, void *split)
{
    A.tiles_m = (A.M + p.bm - 1) / p.bm;
    A.tiles_n = (A.N + p.bn - 1) / p.bn;
    A.k_split = p.k_split;
    A.splits = p.splits;
    A.partial = split;
}

static int64_t li_join_blocks(const LiArgs &A) { return ((int64_t)A.M * (li_ld4(A.N) / 4) + 63) / 64; }

static int li_launch(LiArgs &A, const LiPlan &p, void *split, hipStream_t st)
{
    li_apply(A, p, split);
    FRCNN_REQUIRE(p.tiles < (1ll << 31), "linear_i8: too many tiles");
    const dim3 grid((unsigned)p.tiles, p.splits);
    if (p.bm == 256) hipLaunchKernelGGL((linear_i8_kernel<256, 256, 64, 128, 1, 2>), grid, dim3(512), 0, st, A);
    else if (p.bm == 128) hipLaunchKernelGGL((linear_i8_kernel<128, 128, 64, 64, 1, 2>), grid, dim3(256), 0, st, A);
    else if (p.bm == 64) hipLaunchKernelGGL((linear_i8_kernel<64, 64, 32, 32, 1, 1>), grid, dim3(256), 0, st, A);
    else hipLaunchKernelGGL((linear_i8_kernel<32, 64, 32, 32, 1, 1>), grid, dim3(128), 0, st, A);
    FRCNN_CHECK_LAUNCH("linear_i8");
    if (p.splits > 1) {
        hipLaunchKernelGGL(linear_i8_join_kernel, dim3((unsigned)li_join_blocks(A)), dim3(64), 0, st, A);
        FRCNN_CHECK_LAUNCH("linear_i8_join");
    }
    return FRCNN_OK;
}

// A, and B where B.out is not NULL
static int li_grad_launch(const LiArgs &A, const LiArgs &B, int bn, hipStream_t st)
{
    const int64_t a = A.out ? (int64_t)A.tiles_m * A.tiles_n * A.splits : 0, b = B.out ? (int64_t)B.tiles_m * B.tiles_n * B.splits : 0;
    if (bn == 256)
        hipLaunchKernelGGL((linear_i8_grad_kernel<128, 256, 64, 64, 2>), dim3((unsigned)(a + b)), dim3(512), 0, st, A, B, (int)a);
    else if (bn == 128)
        hipLaunchKernelGGL((linear_i8_grad_kernel<64, 128, 32, 64, 2>), dim3((unsigned)(a + b)), dim3(256), 0, st, A, B, (int)a);
    else
        hipLaunchKernelGGL((linear_i8_grad_kernel<64, 64, 32, 32, 1>), dim3((unsigned)(a + b)), dim3(256), 0, st, A, B, (int)a);
    FRCNN_CHECK_LAUNCH("linear_i8_grad");
    const int64_t ja = A.out && A.splits > 1 ? li_join_blocks(A) : 0, jb = B.out && B.splits > 1 ? li_join_blocks(B) : 0;
    if (ja + jb) {
        hipLaunchKernelGGL(linear_i8_grad_join_kernel, dim3((unsigned)(ja + jb)), dim3(64), 0, st, A, B, (int)ja);
        FRCNN_CHECK_LAUNCH("linear_i8_grad_join");
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

static bool li_shape_ok(int M, int N, int K)
{
    return M >= 0 && M <= I8_MAX_ROWS && N > 0 && N <= I8_MAX_ROWS && K > 0 && K <= I8_MAX_K;
}
static bool li_ws_ok(const void *ws) { return ((uintptr_t)ws & 255) == 0; }

// The few-rows form.  1,024 channels, rows of 12,544, calls replayed in a graph: 1 / 2 / 3 / 4 rows 5.9 / 9.0 / 12.1 / 15.6 us
// against 14.8 (five rows) by tiles and three launches, which cost the host 6 us more than one.
static bool lf_takes(int M, int K) { return M <= 4 && K <= LF_THREADS * LF_CHUNKS * 16; }

// The short-rows form (K >= 16: the last weight is read by a 16-byte load).  It reads the weights once per BM rows, so it
// gives way to quantiser and tiles where rows and channels are both many.  us against us, on the GPU (a call of three launches
// also costs the host 6 us more): rows of 1,024 by 105 channels 8.9 : 11.2 (500 rows), 9.2 : 13.8 (2,000), 36.6 : 40.7
// (32,000); by 256 10.6 : 16.5 (2,000), 24.6 : 21.7 (8,000); by 1,024 10.4 : 15.0 (500), 15.4 : 15.6 (1,000), 19.3 : 17.1
// (2,000); 32,000 rows of 512 by 256 27.4 : 29.8.
static bool lr_takes(int M, int N, int K)
{
    return K <= LR_K && K >= 16 && M > 2 && (N <= 128 || (N <= 256 && K <= 512) || (int64_t)M * N <= (1 << 20));
}

template <typename T>
static int lf_launch(const LiArgs &A, const T *x, int64_t x_stride, const float *x_scale, hipStream_t st)
{
    hipLaunchKernelGGL((linear_i8_few_kernel<T>), dim3((A.N + LF_N - 1) / LF_N), dim3(LF_THREADS), 0, st, x, x_stride, x_scale, A);
    FRCNN_CHECK_LAUNCH("linear_i8_few");
    return FRCNN_OK;
}

template <typename T, int BM> static int lr_launch(LiArgs A, const T *x, int64_t x_stride, hipStream_t st)
{
    const int tiles = (A.M + BM - 1) / BM;
    int groups = tiles >= 256 ? 1 : 256 / tiles;
    const int most = (A.N + LR_THREADS / 4 - 1) / (LR_THREADS / 4); // 16 channels a wave
    if (groups > most) groups = most;
    A.n_group = ((A.N + groups - 1) / groups + 3) & ~3;
    const size_t lds = (size_t)BM * ((A.K + 255) & ~255);
    static size_t granted[FRCNN_MAX_DEVICES];
    if (frcnn_reserve_dynamic_lds((const void *)linear_i8_short_kernel<T, BM>, lds, granted) != hipSuccess) {
        frcnn_set_error("linear_i8_short: %zu bytes of LDS refused", lds);
        return FRCNN_ELAUNCH;
    }
    hipLaunchKernelGGL((linear_i8_short_kernel<T, BM>), dim3(tiles, (A.N + A.n_group - 1) / A.n_group), dim3(LR_THREADS), lds,
                       st, x, x_stride, A);
    FRCNN_CHECK_LAUNCH("linear_i8_short");
    return FRCNN_OK;
}

// 64 rows a workgroup where those fill the chip, 16 where they do not
template <typename T> static int lr_run(const LiArgs &A, const T *x, int64_t x_stride, hipStream_t st)
{
    const int64_t full = (int64_t)((A.M + 63) / 64) * ((A.N + LR_THREADS / 4 - 1) / (LR_THREADS / 4));
    return full >= 256 ? lr_launch<T, 64>(A, x, x_stride, st) : lr_launch<T, 16>(A, x, x_stride, st);
}

// A row of codes brought to an aligned stride where it is not read in place; *p and *stride become what is read.
static int li_in_rows(const int8_t **p, int64_t *stride, int rows, int K, char *copy, hipStream_t st)
{
    const int64_t ld = li_stride(K);
    if (rows == 1) *stride = ld;
    if (li_in_place(*p, *stride, K)) return FRCNN_OK;
    const int rc = frcnn_i8_pad_rows(*p, *stride, rows, K, (int8_t *)copy, ld, st);
    *p = (const int8_t *)copy;
    *stride = ld;
    return rc;
}

static LiArgs li_args(const int8_t *a, int64_t a_stride, const float *a_scale, const int8_t *b, int64_t b_stride,
                      const float *b_scale, const float *bias, int relu, int M, int N, int K, const int32_t *n_rows, void *out,
                      int out_type, int64_t out_stride)
{
    LiArgs A = {};
    A.a = a; A.a_stride = a_stride; A.a_scale = a_scale;
    A.b = b; A.b_stride = b_stride; A.b_scale = b_scale;
    A.bias = bias;
    A.M = M; A.N = N; A.K = K; A.n_rows = n_rows;
    A.out = out; A.out_type = out_type; A.out_stride = out_stride;
    A.low = !relu ? __builtin_nanf("") : out_type == FRCNN_F16 ? 0x1p-25f : out_type == FRCNN_BF16 ? 0x1p-134f : 0.0f;
    A.stream = (((uintptr_t)out | (uint64_t)out_stride * i8_type_bytes(out_type)) & 63) == 0;
    return A;
}

// Workspace: [sums of a split k][codes of b on an aligned stride][codes of a on an aligned stride][a's scales]
static size_t li_ws_b(int M, int N, int K) { return li_split_bytes(li_plan(M, N, K), M, N, 4); }
static size_t li_ws_a(int M, int N, int K) { return li_ws_b(M, N, K) + up256((size_t)N * li_stride(K)); }
static size_t li_ws_scale(int M, int N, int K) { return li_ws_a(M, N, K) + up256((size_t)M * li_stride(K)); }

extern "C" size_t frcnn_matmul_i8_workspace_bytes(int M, int N, int K)
{
    return !li_shape_ok(M, N, K) || M == 0 || lf_takes(M, K) ? 0 : li_ws_scale(M, N, K);
}

extern "C" int frcnn_matmul_i8(const int8_t *a, int64_t a_stride, const float *a_scale, const int8_t *b, int64_t b_stride,
                               const float *b_scale, const float *bias, int relu, int M, int N, int K,
                               const int32_t *n_rows, void *out, int out_type, int64_t out_stride, void *workspace,
                               size_t workspace_bytes, void *stream)
{
    FRCNN_REQUIRE(li_shape_ok(M, N, K), "matmul_i8: bad shape (%d, %d, %d); K is at most %d, M and N %d", M, N, K,
                  I8_MAX_K, I8_MAX_ROWS);
    FRCNN_REQUIRE(i8_type_ok(out_type), "matmul_i8: unknown element type %d", out_type);
    FRCNN_REQUIRE(a_stride >= 0 && b_stride >= 0 && out_stride >= N, "matmul_i8: bad strides");
    if (M == 0) return FRCNN_OK;
    FRCNN_REQUIRE(a && a_scale && b && b_scale && out, "matmul_i8: null pointer");
    hipStream_t st = (hipStream_t)stream;
    LiArgs A = li_args(a, a_stride, a_scale, b, b_stride, b_scale, bias, relu, M, N, K, n_rows, out, out_type, out_stride);
    if (lf_takes(M, K)) return lf_launch(A, a, a_stride, a_scale, st);
    const size_t need = li_ws_scale(M, N, K);
    FRCNN_REQUIRE(li_ws_ok(workspace), "matmul_i8: the workspace has to be 256-byte aligned");
    if (workspace_bytes < need || !workspace) {
        frcnn_set_error("matmul_i8: workspace too small (%zu < %zu)", workspace_bytes, need);
        return FRCNN_EWORKSPACE;
    }
    const LiPlan p = li_plan(M, N, K);
    char *ws = (char *)workspace;
    int rc = li_in_rows(&A.a, &A.a_stride, M, K, ws + li_ws_a(M, N, K), st);
    if (rc == FRCNN_OK) rc = li_in_rows(&A.b, &A.b_stride, N, K, ws + li_ws_b(M, N, K), st);
    return rc == FRCNN_OK ? li_launch(A, p, ws, st) : rc;
}

extern "C" size_t frcnn_linear_i8_workspace_bytes(int M, int N, int K)
{
    return !li_shape_ok(M, N, K) || M == 0 || lf_takes(M, K) || lr_takes(M, N, K) ? 0 : li_ws_scale(M, N, K) + up256((size_t)M * 4);
}

extern "C" int frcnn_linear_i8(const void *x, int x_type, int64_t x_stride, const int8_t *b, int64_t b_stride,
                               const float *b_scale, const float *bias, int relu, int M, int N, int K,
                               const int32_t *n_rows, void *out, int out_type, int64_t out_stride, void *workspace,
                               size_t workspace_bytes, void *stream)
{
    FRCNN_REQUIRE(li_shape_ok(M, N, K), "linear_i8: bad shape (%d, %d, %d); K is at most %d, M and N %d", M, N, K,
                  I8_MAX_K, I8_MAX_ROWS);
    FRCNN_REQUIRE(i8_type_ok(x_type) && i8_type_ok(out_type), "linear_i8: unknown element type");
    FRCNN_REQUIRE(x_stride >= 0 && b_stride >= 0 && out_stride >= N, "linear_i8: bad strides");
    if (M == 0) return FRCNN_OK;
    FRCNN_REQUIRE(x && b && b_scale && out, "linear_i8: null pointer");
    hipStream_t st = (hipStream_t)stream;
    LiArgs A = li_args(nullptr, li_stride(K), nullptr, b, b_stride, b_scale, bias, relu, M, N, K, n_rows, out, out_type,
                       out_stride);
    if (lr_takes(M, N, K)) {
        if (x_type == FRCNN_F32) return lr_run(A, (const float *)x, x_stride, st);
        if (x_type == FRCNN_BF16) return lr_run(A, (const __bf16 *)x, x_stride, st);
        return lr_run(A, (const _Float16 *)x, x_stride, st);
    }
    if (lf_takes(M, K)) {
        if (x_type == FRCNN_F32) return lf_launch(A, (const float *)x, x_stride, nullptr, st);
        if (x_type == FRCNN_BF16) return lf_launch(A, (const __bf16 *)x, x_stride, nullptr, st);
        return lf_launch(A, (const _Float16 *)x, x_stride, nullptr, st);
    }
    const size_t need = frcnn_linear_i8_workspace_bytes(M, N, K);
    FRCNN_REQUIRE(li_ws_ok(workspace), "linear_i8: the workspace has to be 256-byte aligned");
    if (workspace_bytes < need || !workspace) {
        frcnn_set_error("linear_i8: workspace too small (%zu < %zu)", workspace_bytes, need);
        return FRCNN_EWORKSPACE;
    }
    const LiPlan p = li_plan(M, N, K);
    char *ws = (char *)workspace;
    int8_t *codes = (int8_t *)(ws + li_ws_a(M, N, K));
    float *scale = (float *)(ws + li_ws_scale(M, N, K));
    A.a = codes;
    A.a_scale = scale;
    int rc = frcnn_i8_quantize(I8Rows{x, x_type, x_stride, M, n_rows, codes, li_stride(K), scale}, I8Rows{}, K, st);
    if (rc == FRCNN_OK) rc = li_in_rows(&A.b, &A.b_stride, N, K, ws + li_ws_b(M, N, K), st);
    return rc == FRCNN_OK ? li_launch(A, p, ws, st) : rc;
}

// ---- training ----------------------------------------------------------------------------------------------------------
// Codes and scales of both operands lie one behind the other in the caller's `saved`: a (M, ld), a_scale, b (N, ld), b_scale.
struct LiSaved {
    size_t a, a_scale, b, b_scale, total;
};
static LiSaved li_saved(int M, int N, int K)
{
    LiSaved s;
    s.a = 0;
    s.a_scale = s.a + up256((size_t)M * li_stride(K));
    s.b = s.a_scale + up256((size_t)M * 4);
    s.b_scale = s.b + up256((size_t)N * li_stride(K));
    s.total = s.b_scale + up256((size_t)N * 4);
    return s;
}

extern "C" size_t frcnn_linear_i8_train_saved_bytes(int M, int N, int K)
{
    return !li_shape_ok(M, N, K) || M == 0 ? 0 : li_saved(M, N, K).total;
}

extern "C" size_t frcnn_linear_i8_train_workspace_bytes(int M, int N, int K)
{
    return !li_shape_ok(M, N, K) || M == 0 || lf_takes(M, K) ? 0 : li_ws_b(M, N, K);
}

extern "C" int frcnn_linear_i8_train(const void *x, int x_type, int64_t x_stride, const void *w, int w_type,
                                     int64_t w_stride, const float *bias, int relu, int M, int N, int K, void *out,
                                     int out_type, int64_t out_stride, void *saved, size_t saved_bytes, void *workspace,
                                     size_t workspace_bytes, void *stream)
{
    FRCNN_REQUIRE(li_shape_ok(M, N, K) && M > 0, "linear_i8_train: bad shape (%d, %d, %d); K is at most %d, M and N %d", M, N, K,
                  I8_MAX_K, I8_MAX_ROWS);
    FRCNN_REQUIRE(i8_type_ok(x_type) && i8_type_ok(w_type) && i8_type_ok(out_type), "linear_i8_train: unknown element type");
    FRCNN_REQUIRE(x_stride >= 0 && w_stride >= 0 && out_stride >= N, "linear_i8_train: bad strides");
    FRCNN_REQUIRE(x && w && out, "linear_i8_train: null pointer");
    const LiSaved l = li_saved(M, N, K);
    const size_t need = frcnn_linear_i8_train_workspace_bytes(M, N, K);
    FRCNN_REQUIRE(li_ws_ok(workspace) && li_ws_ok(saved), "linear_i8_train: saved and workspace have to be 256-byte aligned");
    FRCNN_REQUIRE(M + N <= I8_MAX_ROWS, "linear_i8_train: M + N (%d) is at most %d", M + N, I8_MAX_ROWS);
    if (!saved || saved_bytes < l.total || workspace_bytes < need || (need && !workspace)) {
        frcnn_set_error("linear_i8_train: saved (%zu of %zu bytes) or workspace (%zu of %zu) too small", saved_bytes, l.total,
                        workspace_bytes, need);
        return FRCNN_EWORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    const int64_t ld = li_stride(K);
    char *s = (char *)saved;
    const I8Rows a = {x, x_type, x_stride, M, nullptr, (int8_t *)(s + l.a), ld, (float *)(s + l.a_scale)};
    const I8Rows b = {w, w_type, w_stride, N, nullptr, (int8_t *)(s + l.b), ld, (float *)(s + l.b_scale)};
    const int rc = frcnn_i8_quantize(a, b, K, st);
    if (rc != FRCNN_OK) return rc;
    LiArgs A = li_args(a.codes, ld, a.scale, b.codes, ld, b.scale, bias, relu, M, N, K, nullptr, out, out_type, out_stride);
    if (lf_takes(M, K)) return lf_launch(A, a.codes, ld, a.scale, st);
    return li_launch(A, li_plan(M, N, K), workspace, st);
}

// Workspace of the gradients, part by part
struct LiGrad {
    size_t x_split, x_pieces, x_top, b_t, w_split, w_pieces, w_top, a_t, part_top, part_sum, total;
    LiPlan x, w;
};

static LiGrad li_grad(int M, int N, int K)
{
    LiGrad g;
    const size_t ldn = (size_t)li_stride(N), ldm = (size_t)li_stride(M), parts = (size_t)frcnn_i8_grad_parts(M) * N * 4;
    size_t off = 0;
    const bool large = li_grad_large(M, N, K);
    g.x = li_grad_plan(M, K, 2 * (int)ldn, large);
    g.w = li_grad_plan(N, K, 2 * (int)ldm, large);
    g.x_split = off; off += li_split_bytes(g.x, M, K, 8);
    g.x_pieces = off; off += up256(2 * 2 * (size_t)M * ldn);
    g.x_top = off; off += up256((size_t)M * 4);
    g.b_t = off; off += up256(2 * (size_t)K * ldn);
    g.w_split = off; off += li_split_bytes(g.w, N, K, 8);
    g.w_pieces = off; off += up256(2 * 2 * (size_t)N * ldm);
    g.w_top = off; off += up256((size_t)N * 4);
    g.a_t = off; off += up256(2 * (size_t)K * ldm);
    g.part_top = off; off += up256(parts);
    g.part_sum = off; off += up256(parts);
    g.total = off;
    return g;
}

// out (rows, cols) from pieces (2, rows, ld) and codes (cols, ld), both fp16
static LiArgs li_grad_args(const _Float16 *pieces, const float *top, const _Float16 *codes, int rows, int cols, int64_t ld,
                           void *out, int out_type)
{
    LiArgs A = li_args((const int8_t *)pieces, 2 * ld, top, (const int8_t *)codes, 2 * ld, nullptr, nullptr, 0, rows, cols,
                       2 * (int)ld, nullptr, out, out_type, cols);
    A.a_plane = 2 * ld * rows;
    return A;
}

extern "C" size_t frcnn_linear_i8_backward_workspace_bytes(int M, int N, int K)
{
    if (M <= 0 || N <= 0 || K <= 0 || M > I8_MAX_K || N > I8_MAX_K || K > I8_MAX_K) return 0;
    return li_grad(M, N, K).total;
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
    FRCNN_REQUIRE(grad && b && b_scale && ((a && a_scale) || (!grad_w && !grad_bias)), "linear_i8_backward: null pointer");
    FRCNN_REQUIRE(grad_stride >= 0 && y_stride >= 0 && a_stride >= 0 && b_stride >= 0, "linear_i8_backward: bad strides");
    const LiGrad l = li_grad(M, N, K);
    FRCNN_REQUIRE(li_ws_ok(workspace), "linear_i8_backward: the workspace has to be 256-byte aligned");
    if (workspace_bytes < l.total || !workspace) {
        frcnn_set_error("linear_i8_backward: workspace too small (%zu < %zu)", workspace_bytes, l.total);
        return FRCNN_EWORKSPACE;
    }
    if (!grad_x && !grad_w && !grad_bias) return FRCNN_OK;
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
    const int64_t ldn = li_stride(N), ldm = li_stride(M);
    I8Grad g = {};
    g.grad = grad; g.type = grad_type; g.grad_stride = grad_stride;
    g.y = y; g.y_stride = y_stride;
    g.a = a; g.a_stride = a_stride; g.a_scale = a_scale;
    g.b = b; g.b_stride = b_stride; g.b_scale = b_scale;
    g.M = M; g.N = N; g.K = K;
    g.row_stride = ldn; g.col_stride = ldm;
    LiArgs X = {}, W = {};
    if (grad_x) {
        g.row_pieces = (_Float16 *)(ws + l.x_pieces);
        g.row_top = (float *)(ws + l.x_top);
        g.b_t = (_Float16 *)(ws + l.b_t);
        X = li_grad_args(g.row_pieces, g.row_top, g.b_t, M, K, ldn, grad_x, grad_x_type);
        li_apply(X, l.x, ws + l.x_split);
    }
    if (grad_w || grad_bias) { // the bias gradient is a by-product of the columns' magnitudes
        g.col_pieces = (_Float16 *)(ws + l.w_pieces);
        g.col_top = (float *)(ws + l.w_top);
        g.part_top = (uint32_t *)(ws + l.part_top);
        g.part_sum = (float *)(ws + l.part_sum);
        g.grad_bias = grad_bias;
    }
    if (grad_w) {
        g.a_t = (_Float16 *)(ws + l.a_t);
        W = li_grad_args(g.col_pieces, g.col_top, g.a_t, N, K, ldm, grad_w, grad_w_type);
        li_apply(W, l.w, ws + l.w_split);
    }
    const int rc = frcnn_i8_grad_prepare(g, st);
    return rc != FRCNN_OK || (!grad_x && !grad_w) ? rc : li_grad_launch(X, W, l.x.bn, st);
}
