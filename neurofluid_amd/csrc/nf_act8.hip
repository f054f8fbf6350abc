// nf_act8.hip — activations kept in 8 bits between forward and backward, and the weight gradient that reads them.
//
// Form: e4m3 codes with one power-of-two scale for every 32 features of a row.  2^k is the smallest power that brings the block's largest finite
// magnitude to 448 (e4m3's largest) or less, k >= -110; code = x / 2^k rounded to nearest even (the division is exact).  So nothing saturates (but magnitudes above
// 1.875 2^127), a
// value is off by at most 2^-4 of itself or 2^-10 2^k, and whatever is not finite becomes NaN, in its own place only.  Codes are rows of
// Kp = 32 ceil(K / 32) bytes (zeros behind K); scales (k + 127, a byte) lie block by block, [Kp / 32][64 ceil(rows / 64)], so that the reader of
// a column of blocks finds eight rows' scales in eight adjacent bytes.
#include "nf_common.h"

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

#define A8_ROWS 64            // rows of a pack tile, of a scale row's padding and of a gradient slab

__device__ __forceinline__ float a8_cv(float v) { return v; }
struct A8Bf16 { unsigned short u; };
struct A8F16 { unsigned short u; };
__device__ __forceinline__ float a8_cv(A8Bf16 v) { return __uint_as_float((unsigned)v.u << 16); }
__device__ __forceinline__ float a8_cv(A8F16 v) { return (float)__builtin_bit_cast(_Float16, v.u); }
__device__ __forceinline__ void a8_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void a8_st(A8Bf16* p, float v) { p->u = __builtin_bit_cast(unsigned short, (__bf16)v); }
__device__ __forceinline__ void a8_st(A8F16* p, float v) { p->u = __builtin_bit_cast(unsigned short, (_Float16)v); }

// ------------------------------------------------------------------------------------------------
// pack / unpack: a thread holds 8 adjacent features, four neighbours a block; a workgroup 64 rows x 128 features.  One pass, bound by memory:
// 63 001 x 2 432 fp32, 613 MB in and 158 MB out, 171 us (4.5 TB/s), and 133 us back (5.8 TB/s: the codes are still in the caches).
// ------------------------------------------------------------------------------------------------
template <typename T, bool VEC> __device__ __forceinline__ void a8_load8(const T* p, int left, float (&v)[8])
{
    if (VEC && left >= 8) {
        alignas(16) T e[8];
        if (sizeof(T) == 4) { *(uint4*)e = ((const uint4*)p)[0]; *(uint4*)(e + 4) = ((const uint4*)p)[sizeof(T) == 4 ? 1 : 0]; }
        else *(uint4*)e = *(const uint4*)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = a8_cv(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? a8_cv(p[i]) : 0.f;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_act8_pack(const T* __restrict__ x, long long xs, int rows, int K, int Kp, int Rp, uint8_t* __restrict__ codes,
                                                   uint8_t* __restrict__ scales)
{
    __shared__ uint8_t sc[4][A8_ROWS];
    const int c = blockIdx.x * 128 + (threadIdx.x & 15) * 8, r0 = blockIdx.y * A8_ROWS, blk = (threadIdx.x & 15) >> 2;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const int lr = it * 16 + (threadIdx.x >> 4), r = r0 + lr;
        float v[8];
        const bool in = r < rows && c < K;
        if (in) a8_load8<T, VEC>(x + (long long)r * xs + c, K - c, v);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
        unsigned top = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned u = __float_as_uint(v[i]) & 0x7fffffffu;
            if (u < 0x7f800000u) top = max(top, u);
            else v[i] = __uint_as_float(0x7fc00000u);
        }
        top = max(top, (unsigned)__shfl_xor((int)top, 1));
        top = max(top, (unsigned)__shfl_xor((int)top, 2));
        // beyond 1.875 2^127 the code's value would be 2^128, which is infinite: such magnitudes are taken as 1.875 2^127 (6 % less at the most)
        if (top > 0x7f700000u) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((__float_as_uint(v[i]) & 0x7fffffffu) < 0x7f800000u) v[i] = fminf(fmaxf(v[i], -__uint_as_float(0x7f700000u)), __uint_as_float(0x7f700000u));
        }
        // top = 1.f 2^e: k = e - 8 while 1.f <= 1.75 (448 = 1.75 2^8), else e - 7
        const int k = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -110);
        const float inv = __uint_as_float((unsigned)(127 - k) << 23);
        if (r < rows && c < Kp) {
            int lo = 0, hi = 0;
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
            *(int2*)(codes + (long long)r * Kp + c) = make_int2(lo, hi);
        }
        if ((threadIdx.x & 3) == 0) sc[blk][lr] = (uint8_t)(k + 127);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int b = threadIdx.x >> 4, w = threadIdx.x & 15, gb = blockIdx.x * 4 + b;
        if (gb < Kp / 32) *(unsigned*)(scales + (long long)gb * Rp + r0 + 4 * w) = *(const unsigned*)&sc[b][4 * w];
    }
}

// A thread writes 16 bytes, next to its neighbours' (8 features of 16 bits, 4 of 32: with 8 of 32 a store's lanes lie 32 bytes apart, 240 us
// for 63 001 x 2 432 in fp32 instead of 206).  past: from 64 MB on stores go around the caches, which hold the codes then (133 us).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_act8_unpack(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int K, int Kp, int Rp,
                                                     T* __restrict__ out, long long os, int past)
{
    constexpr int PER = 16 / sizeof(T), LANES = 128 / PER;
    const int c = blockIdx.x * 128 + (threadIdx.x % LANES) * PER, r0 = blockIdx.y * A8_ROWS;
    if (c >= K) return;
#pragma unroll
    for (int it = 0; it < A8_ROWS * LANES / 256; ++it) {
        const int r = r0 + it * (256 / LANES) + threadIdx.x / LANES;
        if (r >= rows) break;
        unsigned w[PER / 4];
        if (PER == 8) *(uint2*)w = *(const uint2*)(codes + (long long)r * Kp + c);
        else w[0] = *(const unsigned*)(codes + (long long)r * Kp + c);
        const float s = __uint_as_float((unsigned)scales[(long long)(c >> 5) * Rp + r] << 23);
        alignas(16) T e[PER];
#pragma unroll
        for (int i = 0; i < PER / 4; ++i) {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
            a8_st(&e[4 * i], a.x * s); a8_st(&e[4 * i + 1], a.y * s); a8_st(&e[4 * i + 2], b.x * s); a8_st(&e[4 * i + 3], b.y * s);
        }
        T* o = out + (long long)r * os + c;
        typedef unsigned W4 __attribute__((ext_vector_type(4)));
        if (VEC && K - c >= PER) {
            if (past) __builtin_nontemporal_store(*(const W4*)e, (W4*)o);
            else *(W4*)o = *(const W4*)e;
        }
        else {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (c + i < K) o[i] = e[i];
        }
    }
}

static size_t a8_kp(int K) { return ((size_t)K + 31) / 32 * 32; }
static size_t a8_rp(int rows) { return ((size_t)rows + A8_ROWS - 1) / A8_ROWS * A8_ROWS; }

extern "C" size_t nf_act8_code_bytes(int rows, int K) { return rows > 0 && K > 0 ? (size_t)rows * a8_kp(K) : 0; }
extern "C" size_t nf_act8_scale_bytes(int rows, int K) { return rows > 0 && K > 0 ? a8_rp(rows) * (a8_kp(K) / 32) : 0; }

#define A8_MAX (1 << 30)
#define A8_GRID(rows, K) dim3((unsigned)((a8_kp(K) + 127) / 128), (unsigned)(a8_rp(rows) / A8_ROWS))

extern "C" int nf_act8_pack(int dtype, const void* x, int64_t x_stride, int rows, int K, uint8_t* codes, uint8_t* scales, nf_stream_t stream)
{
    NF_CHECK_ARG(dtype >= 0 && dtype <= 2, "dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    NF_CHECK_ARG(rows >= 0 && K >= 0 && rows <= A8_MAX && K <= A8_MAX, "bad sizes");
    if (rows == 0 || K == 0) return NF_OK;
    NF_CHECK_ARG(x && codes && scales, "null pointer");
    NF_CHECK_ARG((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "codes and scales must be 16-byte aligned");
    const int es = dtype == 0 ? 4 : 2;
    const bool vec = (uintptr_t)x % 16 == 0 && x_stride * es % 16 == 0;
    // a launch's grid has at most 65 535 tiles of rows: longer tensors go in pieces
    const int step = 65535 * A8_ROWS;
    for (int r0 = 0; r0 < rows; r0 += step) {
        const int n = rows - r0 < step ? rows - r0 : step;
        const dim3 grid = A8_GRID(n, K);
        const int Kp = (int)a8_kp(K), Rp = (int)a8_rp(rows);
#define A8_PACK(T)                                                                                                                       \
    do {                                                                                                                                 \
        const T* p = (const T*)x + (int64_t)r0 * x_stride;                                                                               \
        if (vec) hipLaunchKernelGGL((k_act8_pack<T, true>), grid, dim3(256), 0, (hipStream_t)stream, p, (long long)x_stride, n, K, Kp, Rp, \
                                    codes + (size_t)r0 * Kp, scales + r0);                                                               \
        else hipLaunchKernelGGL((k_act8_pack<T, false>), grid, dim3(256), 0, (hipStream_t)stream, p, (long long)x_stride, n, K, Kp, Rp,    \
                                codes + (size_t)r0 * Kp, scales + r0);                                                                   \
    } while (0)
        if (dtype == 0) A8_PACK(float);
        else if (dtype == 1) A8_PACK(A8Bf16);
        else A8_PACK(A8F16);
#undef A8_PACK
        NF_CHECK_LAUNCH();
    }
    return NF_OK;
}

extern "C" int nf_act8_unpack(int dtype, const uint8_t* codes, const uint8_t* scales, int rows, int K, void* out, int64_t out_stride, nf_stream_t stream)
{
    NF_CHECK_ARG(dtype >= 0 && dtype <= 2, "dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    NF_CHECK_ARG(rows >= 0 && K >= 0 && rows <= A8_MAX && K <= A8_MAX && out_stride >= 0, "bad sizes");
    if (rows == 0 || K == 0) return NF_OK;
    NF_CHECK_ARG(out && codes && scales, "null pointer");
    NF_CHECK_ARG((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "codes and scales must be 16-byte aligned");
    const int es = dtype == 0 ? 4 : 2;
    const bool vec = (uintptr_t)out % 16 == 0 && out_stride * es % 16 == 0;
    const int past = (long long)rows * K * es >= 64ll << 20;
    const int step = 65535 * A8_ROWS;
    for (int r0 = 0; r0 < rows; r0 += step) {
        const int n = rows - r0 < step ? rows - r0 : step;
        const dim3 grid = A8_GRID(n, K);
        const int Kp = (int)a8_kp(K), Rp = (int)a8_rp(rows);
#define A8_UNPACK(T)                                                                                                                         \
    do {                                                                                                                                     \
        T* p = (T*)out + (int64_t)r0 * out_stride;                                                                                           \
        if (vec) hipLaunchKernelGGL((k_act8_unpack<T, true>), grid, dim3(256), 0, (hipStream_t)stream, codes + (size_t)r0 * Kp, scales + r0, n, \
                                    K, Kp, Rp, p, (long long)out_stride, past);                                                                    \
        else hipLaunchKernelGGL((k_act8_unpack<T, false>), grid, dim3(256), 0, (hipStream_t)stream, codes + (size_t)r0 * Kp, scales + r0, n,   \
                                K, Kp, Rp, p, (long long)out_stride, past);                                                                        \
    } while (0)
        if (dtype == 0) A8_UNPACK(float);
        else if (dtype == 1) A8_UNPACK(A8Bf16);
        else A8_UNPACK(A8F16);
#undef A8_UNPACK
        NF_CHECK_LAUNCH();
    }
    return NF_OK;
}

// ------------------------------------------------------------------------------------------------
// weight gradients from the codes:  dW[m][k] = sum_r dy[r][m] x^[r][k],   db[m] = sum_r dy[r][m]
//
// A code with its scale has four significant bits: it is a bf16 number, exactly.  dy is written as a sum of bf16 numbers, exactly too: one for
// bf16, two for fp16 (11 bits), three for fp32 (24 bits; each the truncation of what is left, so that no rounding can overflow; only what lies below 2^-133, bf16's smallest
// number, is lost).  So 1 / 2 / 3 bf16 matrix instructions with fp32 accumulation give every product exactly, at 16 / 8 / 5.3 times the fp32 matrix rate: the result is that
// of an fp32 product of dy with the unpacked values, up to the order of the sums.
//
// Both operands lie along the outputs, and the reduction runs over the rows: a wave loads 8 rows, a lane C adjacent columns of them, and 8 rows of
// one column are the 16 bytes that a lane feeds the matrix instruction: the transposition happens in the packing.  Column j of lane p goes to
// LDS place 64 j + p, so that both the writes and the reads run through whole bank rows; which column a matrix row stands for is then settled
// where the result is stored.
//
// Tile: (64 C) x (64 C) outputs a workgroup, each of 4 waves a quarter, 32 rows a slab, two slabs in LDS: while one is multiplied the next is
// packed into the other and the one after that is on its way in registers; one barrier a slab.  C = 4 (256 x 256: 64 matrix instructions a
// slab and plane for 32 fragment reads) from 32 such tiles on, else C = 2 (two workgroups a CU).  C = 4 against 2, us a call with the second launch, bf16:
// 32 768 rows, 64 tiles 270 / 400, 32 tiles 155 / 207, 16 tiles 99 / 122, 8 tiles 65 / 73; 6001 rows, 32 tiles 54 / 56, 16 tiles 45 / 45; 63 001 rows, one
// tile 43 / 36.  (fp32: 633 / 832, 339 / 432, 202 / 242, 125 / 139; 94 / 94, 68 / 60; 62 / 52.  For many rows the border could lie lower.)  The
// rows are split into slices, whose partial tiles a second launch adds in a fixed order.
//
// What bounds it: 32 768 rows, 2 048 x 2 048, bf16: 294 us = 935 TFLOP/s (the library's 8192^3 bf16 product reaches 1 093), the matrix unit busy 47 % of
// the cycles at the clock that its power leaves, 28 % of a wave's cycles waiting (fragments out of LDS: 96 KB a slab and workgroup).
// 63 001 rows, 256 x 256, fp32 (three planes): 48 us for 81 MB of operands (each read by two tiles) and 24.8 GFLOP in bf16.  Neither bound is
// near (16 us, 23 us): 124 slices of four tiles leave a workgroup 16 slabs, of which the first and the last three run unoverlapped.
// By dy's type, us a call with the second launch: 63 001 rows 256 x 256 fp32 52, fp16 64, bf16 45; 32 768 rows 2 048 x 2 048 fp32 703, fp16 1 155,
// bf16 319.  fp16 with its two planes takes longer than fp32 with three; why is not known.
// ------------------------------------------------------------------------------------------------
#define A8_MAX_JOBS 16
#define A8_SLAB 32

struct A8Job { long long out; int dy_col, M, x_col, K, db, tile0, tiles_k; };     // db: offset of the column sums in the slice's record, -1: none
struct A8Jobs { int n, ntiles; A8Job j[A8_MAX_JOBS]; };

struct A8Args {
    const void* dy; long long dys; const uint8_t* codes; const uint8_t* scales;
    int rows, Kp, Rp, rows_per_slice, nslices;
    float* out;                            // slice s at out + s * total: the jobs' tiles, then their column sums
    float* bias;                           // the same for one slice: the column sums go here
    long long total;
};

template <bool B> struct A8Bool { static constexpr bool value = B; };

template <typename T> struct A8Planes { static constexpr int n = 3; };
template <> struct A8Planes<A8F16> { static constexpr int n = 2; };
template <> struct A8Planes<A8Bf16> { static constexpr int n = 1; };

// v = h + (what is returned), h = v with its low 16 bits cleared.  A NaN leaves NaN, an infinity (FIRST: no rest is one) nothing.
template <bool FIRST> __device__ __forceinline__ float a8_rest(float v)
{
    const float h = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    return FIRST && h == v ? 0.f : v - h;
}
// the upper halves of two words: (low: a, high: b)
__device__ __forceinline__ unsigned a8_hi2(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }

template <typename T, int C, bool VEC>
__global__ void __launch_bounds__(256, C == 4 ? 1 : 2) k_act8_wgrad(A8Args a, A8Jobs J)
{
    constexpr int NP = A8Planes<T>::n, TILE = 64 * C, NB = C;        // NB: 32-blocks of a wave in either direction
    __shared__ uint4 sA[2][NP][4][TILE];
    __shared__ uint4 sB[2][4][TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave & 1, wk = wave >> 1;
    // consecutive tiles of a slice share operand columns: they go to one XCD (workgroups go round the eight of them)
    int id = blockIdx.x;
    {
        const int n = gridDim.x, x = id & 7, q = n >> 3, rem = n & 7;
        id = x * q + min(x, rem) + (id >> 3);
    }
    const int slice = id / J.ntiles, tile = id - slice * J.ntiles;
    int ji = 0;
    while (ji + 1 < J.n && tile >= J.j[ji + 1].tile0) ++ji;
    const A8Job job = J.j[ji];
    const int tm = (tile - job.tile0) / job.tiles_k, tk = (tile - job.tile0) - tm * job.tiles_k;
    const int m0 = tm * TILE, k0 = tk * TILE;
    const int rb = slice * a.rows_per_slice, re = min(a.rows, rb + a.rows_per_slice);
    // columns of this lane; beyond the job's they are read from inside it (the results are not stored)
    const int cm = m0 + C * lane, ckl = min(k0 + C * lane, (job.K + 31) / 32 * 32 - C);
    const bool with_bias = job.db >= 0 && tk == 0, vec = VEC && job.dy_col % C == 0;
    const bool inside = vec && cm + C <= job.M;
    const T* dyp = (const T*)a.dy + job.dy_col;
    const uint8_t* xp = a.codes + job.x_col;
    const uint8_t* sp = a.scales + (long long)((job.x_col + ckl) >> 5) * a.Rp;
    f32x16 acc[NB][NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    float bsum[C] = {};

    struct alignas(sizeof(T) * C) Row { T v[C]; };
    struct Regs { Row d[8]; unsigned x[8]; uint2 s; };
    // Any slab: rows behind the slice are not read, columns behind the job are read from inside it.
    auto fetch_part = [&](Regs& g, int r0) {
        const int r = r0 + 8 * wave;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long long rr = min(r + i, re - 1);
            const T* p = dyp + rr * a.dys;
            if (inside) g.d[i] = *(const Row*)(p + cm);
            else {
#pragma unroll
                for (int c = 0; c < C; ++c) g.d[i].v[c] = p[min(cm + c, job.M - 1)];
            }
            if (C == 4) g.x[i] = *(const unsigned*)(xp + rr * a.Kp + ckl);
            else g.x[i] = *(const unsigned short*)(xp + rr * a.Kp + ckl);
        }
        g.s = *(const uint2*)(sp + min(r, a.Rp - 8));      // (rows are padded to 64)
    };
    // A whole slab of a tile inside its job, row by row from uniform bases.  (Behind the slice's last eight rows: those again, never used.)
    const unsigned off_d = (unsigned)cm * sizeof(T), off_x = (unsigned)ckl;
    const long long step_d = a.dys * (long long)sizeof(T);
    struct Bases { const char* d; const char* x; };
    auto bases = [&](int r0) {
        const int r = min(r0 + 8 * wave, re - 8);
        return Bases{(const char*)dyp + r * step_d, (const char*)xp + (long long)r * a.Kp};
    };
    auto fetch_row = [&](Regs& g, int i, Bases& p) {
        g.d[i] = *(const Row*)(p.d + off_d);
        if (C == 4) g.x[i] = *(const unsigned*)(p.x + off_x);
        else g.x[i] = *(const unsigned short*)(p.x + off_x);
        p.d += step_d;
        p.x += a.Kp;
    };
    // Packing a slab, in C * NP pieces for dy (a column's plane each) and 2 C for the codes (four rows of two features, a feature).
    constexpr int PIECES = C * NP + 2 * C;
    float v[8];          // what is left of the column
    unsigned e[8];       // two features as bf16 pairs
    auto pack = [&](const Regs& g, int buf, int piece, int left, auto full, auto bias) {
        const bool cut = !decltype(full)::value && left < 8;
        if (piece < C * NP) {
            const int c = piece / NP, p = piece % NP;
            if (NP == 1 && !decltype(bias)::value && !cut) {         // bf16: the halves as they are
                const unsigned sel = (c & 1) ? 0x07060302u : 0x05040100u;
                unsigned w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = ((const unsigned*)g.d[i].v)[c / 2];
                sA[buf][0][wave][64 * c + lane] = make_uint4(__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel),
                                                             __builtin_amdgcn_perm(w[5], w[4], sel), __builtin_amdgcn_perm(w[7], w[6], sel));
                return;
            }
            if (p == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = a8_cv(g.d[i].v[c]);
                if (cut)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = i < left ? v[i] : 0.f;
                if (decltype(bias)::value) bsum[c] += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            }
            sA[buf][p][wave][64 * c + lane] = make_uint4(a8_hi2(v[0], v[1]), a8_hi2(v[2], v[3]), a8_hi2(v[4], v[5]), a8_hi2(v[6], v[7]));
            if (p + 1 < NP)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = p == 0 ? a8_rest<true>(v[i]) : a8_rest<false>(v[i]);
        } else {
            const int h = (piece - C * NP) / 4, f = (piece - C * NP) % 4;
            if (f < 2) {
#pragma unroll
                for (int i = 4 * f; i < 4 * f + 4; ++i) {
                    const float s = __uint_as_float(((i < 4 ? g.s.x >> (8 * i) : g.s.y >> (8 * i - 32)) & 0xffu) << 23);
                    const unsigned w = cut && i >= left ? 0u : g.x[i];
                    e[i] = h ? __builtin_bit_cast(unsigned, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true))
                             : __builtin_bit_cast(unsigned, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
                }
            } else {
                const unsigned sel = f == 3 ? 0x07060302u : 0x05040100u;
                sB[buf][wave][64 * (2 * h + f - 2) + lane] = make_uint4(__builtin_amdgcn_perm(e[1], e[0], sel), __builtin_amdgcn_perm(e[3], e[2], sel),
                                                                        __builtin_amdgcn_perm(e[5], e[4], sel), __builtin_amdgcn_perm(e[7], e[6], sel));
            }
        }
    };
    bf16x8 fa[2][NP][NB], fb[2][NB];
    auto fragments = [&](int ks, int buf) {
        const int o = 2 * ks + (lane >> 5), l = lane & 31;
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[ks][j] = __builtin_bit_cast(bf16x8, sB[buf][o][64 * j + 32 * wk + l]);
#pragma unroll
        for (int p = NP - 1; p >= 0; --p)
#pragma unroll
            for (int i = 0; i < NB; ++i) fa[ks][p][i] = __builtin_bit_cast(bf16x8, sA[buf][p][o][64 * i + 32 * wm + l]);
    };
    constexpr int PRODUCTS = 2 * NP * NB * NB;
    auto product = [&](int n) {          // the small parts first
        const int j = n % NB, i = n / NB % NB, p = NP - 1 - n / (NB * NB) % NP, ks = n / (NB * NB * NP);
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[ks][p][i], fb[ks][j], acc[i][j], 0, 0, 0);
    };
    // Slab n is multiplied while n + 1 is packed from one set of registers and n + 2, n + 3 are on their way (the other set, then the same): a load
    // has two slabs' time.  A wave issues in order, so everything else goes in pieces between the matrix instructions, in whose shadow it runs:
    // the packing with the slab's first half, the loads with the second, whose fragments were read during the first; the next slab's first
    // fragments are read during the second half, which is why the barrier lies between the two.
    auto step = [&](Regs& g, int r0, int buf, auto bias) {
        fragments(1, buf);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
#pragma unroll
            for (int n = PRODUCTS / 2 * q / PIECES; n < PRODUCTS / 2 * (q + 1) / PIECES; ++n) product(n);
            pack(g, buf ^ 1, q, 8, A8Bool<true>(), bias);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        fragments(0, buf ^ 1);
        Bases p = bases(r0 + 3 * A8_SLAB);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
#pragma unroll
            for (int n = PRODUCTS / 2 * q / 8; n < PRODUCTS / 2 * (q + 1) / 8; ++n) product(PRODUCTS / 2 + n);
            fetch_row(g, q, p);
            if (q == 7) g.s = *(const uint2*)(sp + min(r0 + 3 * A8_SLAB + 8 * wave, a.Rp - 8));
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto run = [&](auto whole, auto bias) {
        Regs g0, g1;
        auto pack_part = [&](const Regs& g, int r0, int buf) {
#pragma unroll
            for (int q = 0; q < PIECES; ++q) pack(g, buf, q, re - (r0 + 8 * wave), A8Bool<false>(), bias);
        };
        fetch_part(g0, rb);
        fetch_part(g1, rb + A8_SLAB);
        pack_part(g0, rb, 0);
        fetch_part(g0, rb + 2 * A8_SLAB);
        __syncthreads();
        int r0 = rb;
        if (decltype(whole)::value) {
            fragments(0, 0);
            for (; r0 + 3 * A8_SLAB <= re; r0 += 2 * A8_SLAB) {              // (both packed slabs exist)
                step(g1, r0, 0, bias);
                step(g0, r0 + A8_SLAB, 1, bias);
            }
            fetch_part(g1, r0 + A8_SLAB);
            fetch_part(g0, r0 + 2 * A8_SLAB);
        }
        // what is left: up to three slabs, or the whole slice of a tile that its job does not fill
        for (int buf = 0; r0 < re; r0 += A8_SLAB, buf ^= 1) {
            if (r0 + A8_SLAB < re) {
                if (buf) pack_part(g0, r0 + A8_SLAB, 0);
                else pack_part(g1, r0 + A8_SLAB, 1);
                if (buf) fetch_part(g0, r0 + 3 * A8_SLAB);
                else fetch_part(g1, r0 + 3 * A8_SLAB);
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                fragments(ks, buf);
#pragma unroll
                for (int n = 0; n < PRODUCTS / 2; ++n) product(ks * (PRODUCTS / 2) + n);
            }
            __syncthreads();
        }
    };
    if (rb < re) {
        const bool whole = vec && m0 + TILE <= job.M;
        if (whole && with_bias) run(A8Bool<true>(), A8Bool<true>());
        else if (whole) run(A8Bool<true>(), A8Bool<false>());
        else run(A8Bool<false>(), A8Bool<true>());
    }
    // place 64 j + p of a tile is column C p + j: a lane holds C adjacent features of its rows
    float* out = a.out + slice * a.total + job.out;
    const int k = k0 + C * (32 * wk + (lane & 31));
    const bool quads = job.K % C == 0 && (uintptr_t)out % (4 * C) == 0;
    typedef float Out __attribute__((ext_vector_type(C)));
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int m = m0 + C * (32 * wm + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) + i;
            if (m >= job.M || k >= job.K) continue;
            float* o = out + (long long)m * job.K + k;
            if (quads) {
                Out w;
#pragma unroll
                for (int j = 0; j < NB; ++j) w[j] = acc[i][j][r];
                *(Out*)o = w;
            } else {
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    if (k + j < job.K) o[j] = acc[i][j][r];
            }
        }
    if (with_bias) {
        float* sb = (float*)&sB[0][0][0];
#pragma unroll
        for (int c = 0; c < C; ++c) sb[wave * TILE + C * lane + c] = bsum[c];
        __syncthreads();
        for (int c = tid; c < TILE && m0 + c < job.M; c += 256)
            a.bias[slice * a.total + job.db + m0 + c] = (sb[c] + sb[TILE + c]) + (sb[2 * TILE + c] + sb[3 * TILE + c]);
    }
}

// Slices added in a fixed order: a thread a quarter of them for four numbers, then the four quarters.  Record: [weights (n_w) | biases].
// (124 slices of 65 792 numbers, 33 MB: 10 us; 4 of 4.2 million, 84 MB: 14 us.)
__global__ void __launch_bounds__(256) k_act8_fold(const float* __restrict__ part, long long n, long long n_w, long long n_all, int nslices, float* __restrict__ dw,
                                                   float* __restrict__ db)
{
    __shared__ float4 s4[3][64];
    const int c = threadIdx.x & 63, g = threadIdx.x >> 6;
    const long long i = ((long long)blockIdx.x * 64 + c) * 4;
    const int per = (nslices + 3) / 4, s0 = g * per, s1 = min(nslices, s0 + per);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n) {
#pragma unroll 8
        for (int s = s0; s < s1; ++s) {
            const float4 e = *(const float4*)(part + s * n + i);        // (records are whole quads long)
            v.x += e.x; v.y += e.y; v.z += e.z; v.w += e.w;
        }
    }
    if (g > 0) s4[g - 1][c] = v;
    __syncthreads();
    if (g == 0 && i < n) {
        const float4 b = s4[0][c], d = s4[1][c], e = s4[2][c];
        const float o[4] = {(v.x + b.x) + (d.x + e.x), (v.y + b.y) + (d.y + e.y), (v.z + b.z) + (d.z + e.z), (v.w + b.w) + (d.w + e.w)};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i + k < n_w) dw[i + k] = o[k];
            else if (i + k < n_all) db[i + k - n_w] = o[k];
        }
    }
}

struct A8Plan { A8Jobs J; int C, nslices, rows_per_slice; long long n_w, n_b, record; };

static void a8_tiles(int njobs, const nf_act8_job_t* jobs, int C, A8Plan* p)
{
    const int tile = 64 * C;
    int tiles = 0;
    long long out = 0, bias = 0;
    for (int i = 0; i < njobs; ++i) {
        const nf_act8_job_t& s = jobs[i];
        A8Job& j = p->J.j[i];
        j.dy_col = s.dy_col; j.M = s.M; j.x_col = s.x_col; j.K = s.K; j.out = out;
        j.db = s.bias ? (int)bias : -1;
        j.tile0 = tiles; j.tiles_k = (s.K + tile - 1) / tile;
        tiles += ((s.M + tile - 1) / tile) * j.tiles_k;
        out += (long long)s.M * s.K;
        if (s.bias) bias += s.M;
    }
    p->J.n = njobs; p->J.ntiles = tiles; p->C = C;
    p->n_w = out; p->n_b = bias; p->record = (out + bias + 3) / 4 * 4;
}

static A8Plan a8_plan(int rows, int njobs, const nf_act8_job_t* jobs)
{
    A8Plan p;
    const int slabs = (rows + A8_SLAB - 1) / A8_SLAB;
    a8_tiles(njobs, jobs, 4, &p);
    int want = 256;
    if (p.J.ntiles < 32) { a8_tiles(njobs, jobs, 2, &p); want = 512; }
    int s = want / p.J.ntiles;
    if (s > slabs / 8) s = slabs / 8;
    if (s < 1) s = 1;
    const int per = (slabs + s - 1) / s;
    p.nslices = per > 0 ? (slabs + per - 1) / per : 1;
    p.rows_per_slice = per * A8_SLAB;
    return p;
}

static int a8_jobs_ok(const char* who, int rows, int dy_cols, int x_cols, int njobs, const nf_act8_job_t* jobs)
{
    const char* bad = nullptr;
    if (njobs < 1 || njobs > A8_MAX_JOBS || !jobs) bad = "1 to 16 jobs";
    else if (rows < 0 || rows > A8_MAX || dy_cols < 1 || dy_cols > A8_MAX || x_cols < 1 || x_cols > A8_MAX) bad = "bad sizes";
    else {
        long long outputs = 0, tiles = 0;
        for (int i = 0; i < njobs; ++i) {
            const nf_act8_job_t& j = jobs[i];
            if (j.M < 1 || j.K < 1 || j.dy_col < 0 || j.x_col < 0 || j.dy_col > dy_cols - j.M || j.x_col > x_cols - j.K) bad = "a job leaves its operands";
            else if (j.x_col % 32) bad = "a job's first feature must begin a block of 32";
            else tiles += ((long long)j.M + 127) / 128 * (((long long)j.K + 127) / 128);          // (of the smaller kind)
            outputs += j.M;
        }
        if (!bad && outputs > A8_MAX) bad = "the jobs have too many outputs";
        if (!bad && tiles > 0x7fffffffLL) bad = "too many tiles";
    }
    if (bad) { nf_set_error("%s: %s", who, bad); return NF_EINVAL; }
    return NF_OK;
}

extern "C" size_t nf_act8_wgrad_workspace_floats(int rows, int dy_cols, int x_cols, int njobs, const nf_act8_job_t* jobs)
{
    if (a8_jobs_ok(__func__, rows, dy_cols, x_cols, njobs, jobs)) return 0;
    const A8Plan p = a8_plan(rows, njobs, jobs);
    return p.nslices > 1 ? (size_t)p.nslices * (size_t)p.record : 0;
}

extern "C" int nf_act8_wgrad(int dtype, const void* dy, int64_t dy_stride, int dy_cols, const uint8_t* codes, const uint8_t* scales, int x_cols, int rows,
                             int njobs, const nf_act8_job_t* jobs, float* workspace, float* dweights, float* dbias, nf_stream_t stream)
{
    NF_CHECK_ARG(dtype >= 0 && dtype <= 2, "dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    const int rc = a8_jobs_ok(__func__, rows, dy_cols, x_cols, njobs, jobs);
    if (rc) return rc;
    const A8Plan p = a8_plan(rows, njobs, jobs);
    NF_CHECK_ARG(dweights && (p.n_b == 0 || dbias) && (rows == 0 || (dy && codes && scales)), "null pointer");
    NF_CHECK_ARG(p.nslices == 1 || (workspace && (uintptr_t)workspace % 16 == 0), "null or unaligned workspace (nf_act8_wgrad_workspace_floats)");
    NF_CHECK_ARG((long long)p.nslices * p.J.ntiles <= 0x7fffffffLL && p.record / 256 < 0x7fffffffLL, "too many tiles");
    A8Args a = {};
    a.dy = dy; a.dys = dy_stride; a.codes = codes; a.scales = scales;
    a.rows = rows; a.Kp = (int)a8_kp(x_cols); a.Rp = (int)a8_rp(rows); a.nslices = p.nslices; a.rows_per_slice = p.rows_per_slice;
    a.total = p.record;
    a.out = p.nslices > 1 ? workspace : dweights;
    a.bias = p.nslices > 1 ? workspace + p.n_w : dbias;
    const int es = dtype == 0 ? 4 : 2;
    const bool vec = (uintptr_t)dy % (p.C * es) == 0 && dy_stride % p.C == 0;
    const dim3 grid((unsigned)(p.nslices * p.J.ntiles));
    hipStream_t st = (hipStream_t)stream;
#define A8_GO(T, C_)                                                                                       \
    do {                                                                                                   \
        if (vec) hipLaunchKernelGGL((k_act8_wgrad<T, C_, true>), grid, dim3(256), 0, st, a, p.J);           \
        else hipLaunchKernelGGL((k_act8_wgrad<T, C_, false>), grid, dim3(256), 0, st, a, p.J);              \
    } while (0)
#define A8_GO_C(T) do { if (p.C == 4) A8_GO(T, 4); else A8_GO(T, 2); } while (0)
    if (dtype == 0) A8_GO_C(float);
    else if (dtype == 1) A8_GO_C(A8Bf16);
    else A8_GO_C(A8F16);
#undef A8_GO_C
#undef A8_GO
    NF_CHECK_LAUNCH();
    if (p.nslices > 1) {
        hipLaunchKernelGGL(k_act8_fold, dim3((unsigned)((p.record + 255) / 256)), dim3(256), 0, st, (const float*)workspace, p.record, p.n_w, p.n_w + p.n_b, p.nslices,
                           dweights, p.n_b ? dbias : nullptr);
        NF_CHECK_LAUNCH();
    }
    return NF_OK;
}
