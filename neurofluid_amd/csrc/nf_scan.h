// nf_scan.h — kernels of the gated linear recurrence (one instantiation per storage type: nf_scan_f32 / _bf16 / _f16.hip).
//
//   h_t = A_t h_{t-1} + x_t,   A_t = gate_t or exp(gate_t)                                  (forward; reverse: t runs downwards)
//   u_t = A_t (g_t + u_{t+1}), dx_t = g_t + u_{t+1}, dA_t = dx_t h_{t-1} (log gate: times A_t), dh0 = u_0      (backward)
//
// A stretch of steps acts on the state that enters it as  h -> P h + H  (P = the product of its gates, H = what it gives from a zero
// state), and two stretches compose: (P1, H1) then (P2, H2) = (P1 P2, P2 H1 + H2).  The time axis is cut into one stretch of
// NF_SCAN_TPT steps per thread: a thread reduces its stretch to (P, H) in registers, the stretches of a tile are composed across lanes (shuffles) and
// waves (LDS), and with the state that really enters it every thread then runs its steps once more, one after the other, in fp32 — so
// a state is rounded only where it is stored, and the products P only carry states from one stretch to the next.  The order of every
// sum is fixed by the sizes: results repeat bit for bit.  The backward recomputes the states of a tile from x and
// the state at the tile's start (kept by the forward in fp32: 1 / tile of a tensor) instead of reading h back, which would be as many
// bytes but rounded to the storage type.
//
// Lanes: CG channel groups of VEC adjacent channels x 64 / CG stretches; NW waves share a tile (1: four independent chains per
// workgroup, no barrier).  A row of a tile is CG * VEC adjacent channels: 128 B of 16-bit and 256 B of 32-bit data for CG = 32, VEC = 2.
#pragma once
#include "nf_common.h"

#define NF_SCAN_TPT 8
#define NF_SCAN_WG 256

struct NfScanArgs {
    const void* gate; const void* x; const void* g;
    const float* h0; const float* g_last;
    void* h; float* h_last; float* states;
    void* dgate; float* dgate_part; void* dx; float* dh0;
    const int* sid;                      // packed: the sequence of every row (-1: none), else NULL
    float* agg;                          // [chain][chunk][2][D]: (P, H) of a chunk (write when only_agg)
    const float* carry;                  // [chain][chunk][D]: the state that enters a chunk, or NULL (one chunk)
    long long gate_sb, gate_st, x_sb, x_st, g_sb, g_st;      // strides of a batch / a step, in elements
    int B, T, D, nblk, nchunk, tiles_per_chunk, ntiles;
    int gate32, shared, log_gate, reverse, only_agg;
};

struct NfF32 { typedef float st; static __device__ __forceinline__ float cv(st v) { return v; } static __device__ __forceinline__ st pk(float v) { return v; } };
struct NfBf16 {
    typedef unsigned short st;
    static __device__ __forceinline__ float cv(st v) { return __uint_as_float((unsigned)v << 16); }
    static __device__ __forceinline__ st pk(float v) { return __builtin_bit_cast(st, (__bf16)v); }       // nearest even
};
struct NfF16 {
    typedef unsigned short st;
    static __device__ __forceinline__ float cv(st v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ st pk(float v) { return __builtin_bit_cast(st, (_Float16)v); }
};

template <typename E, int VEC> struct NfVec { typedef typename E::st type __attribute__((ext_vector_type(VEC))); };
template <typename E> struct NfVec<E, 1> { typedef typename E::st type; };
template <typename E> __device__ __forceinline__ float nf_el(const typename NfVec<E, 1>::type& v, int) { return E::cv(v); }
template <typename E> __device__ __forceinline__ float nf_el(const typename NfVec<E, 2>::type& v, int k) { return E::cv(v[k]); }

// One thread's stretch of a tensor as it lies in memory.
template <typename E, int VEC> struct NfStretch {
    typename NfVec<E, VEC>::type r[NF_SCAN_TPT];
    // p: the row of processed step 0 at this thread's channels; step = the signed stride between processed steps
    __device__ __forceinline__ void load(const typename E::st* p, long long step, int j0, int T)
    {
        typedef typename NfVec<E, VEC>::type V;
        if (j0 + NF_SCAN_TPT <= T) {
            const typename E::st* q = p + j0 * step;
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i) { r[i] = *(const V*)q; q += step; }
        } else {
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i) r[i] = *(const V*)(p + (long long)min(j0 + i, T - 1) * step);
        }
    }
    __device__ __forceinline__ float at(int i, int k) const { return nf_el<E>(r[i], k); }
};

// The gate comes in the storage type or in fp32, per channel or one per step: both are uniform branches.
template <typename E, int VEC> struct NfGateStretch {
    unsigned r[NF_SCAN_TPT * VEC];       // fp32: a word per channel; else the row's VEC elements packed in word VEC * i
    __device__ __forceinline__ void load(const NfScanArgs& a, const char* p, long long step, int j0, int T)
    {
        const bool full = j0 + NF_SCAN_TPT <= T;
        if (sizeof(typename E::st) == 4 || a.gate32) {
            const float* f = (const float*)p;
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i) {
                const float* q = f + (long long)(full ? j0 + i : min(j0 + i, T - 1)) * step;
                if (a.shared || VEC == 1) r[VEC * i] = __float_as_uint(q[0]);
                else { const float2 v = *(const float2*)q; r[VEC * i] = __float_as_uint(v.x); r[VEC * i + VEC - 1] = __float_as_uint(v.y); }
            }
        } else {
            const unsigned short* f = (const unsigned short*)p;
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i) {
                const unsigned short* q = f + (long long)(full ? j0 + i : min(j0 + i, T - 1)) * step;
                r[VEC * i] = (a.shared || VEC == 1) ? *q : *(const unsigned*)q;
            }
        }
    }
    // gates of step i as factors
    __device__ __forceinline__ void get(const NfScanArgs& a, float (&A)[NF_SCAN_TPT][VEC]) const
    {
#pragma unroll
        for (int i = 0; i < NF_SCAN_TPT; ++i) {
            if (sizeof(typename E::st) == 4 || a.gate32) {
                A[i][0] = __uint_as_float(r[VEC * i]);
                if (VEC == 2) A[i][VEC - 1] = a.shared ? A[i][0] : __uint_as_float(r[VEC * i + VEC - 1]);
            } else {
                A[i][0] = E::cv((typename E::st)(r[VEC * i] & 0xffffu));
                if (VEC == 2) A[i][VEC - 1] = a.shared ? A[i][0] : E::cv((typename E::st)(r[VEC * i] >> 16));
            }
        }
        if (a.log_gate) {
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i) {
                A[i][0] = expf(A[i][0]);
                if (VEC == 2) A[i][VEC - 1] = a.shared ? A[i][0] : expf(A[i][VEC - 1]);
            }
        }
    }
};

template <typename E, int VEC> __device__ __forceinline__ void nf_put(typename E::st* p, const float (&v)[VEC])
{
    if (VEC == 1) p[0] = E::pk(v[0]);
    else {
        typename NfVec<E, 2>::type w;
        w[0] = E::pk(v[0]); w[1] = E::pk(v[VEC - 1]);
        *(typename NfVec<E, 2>::type*)p = w;
    }
}

// Which steps of a stretch start / end a sequence and which belong to none (bit i), for packed rows.
struct NfMarks { unsigned start, end, none; };
__device__ __forceinline__ NfMarks nf_scan_marks(const int* sid, int j0, int T, int reverse)
{
    NfMarks m = {0u, 0u, 0u};
    auto at = [&](int j) { return (j < 0 || j >= T) ? -2 : sid[reverse ? T - 1 - j : j]; };
    int prev = at(j0 - 1), cur = at(j0);
#pragma unroll
    for (int i = 0; i < NF_SCAN_TPT; ++i) {
        const int next = at(j0 + i + 1);
        if (cur < 0) m.none |= 1u << i;
        else {
            if (cur != prev) m.start |= 1u << i;
            if (cur != next) m.end |= 1u << i;
        }
        prev = cur; cur = next;
    }
    return m;
}

template <int VEC> struct NfAgg {
    float P[VEC], H[VEC];
    int closed;             // a sequence begins inside: nothing of the entering state comes out
    __device__ __forceinline__ void after(const NfAgg& p)      // this stretch behind stretch p
    {
        if (closed) return;
#pragma unroll
        for (int k = 0; k < VEC; ++k) { H[k] = fmaf(P[k], p.H[k], H[k]); P[k] *= p.P[k]; }
        closed = p.closed;
    }
    __device__ __forceinline__ void apply(float (&c)[VEC]) const
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k) c[k] = closed ? H[k] : fmaf(P[k], c[k], H[k]);
    }
    __device__ __forceinline__ void one() { closed = 0; for (int k = 0; k < VEC; ++k) { P[k] = 1.f; H[k] = 0.f; } }
};

// Composition over the stretches of a tile in processing order (DIR = 0: upwards, 1: downwards): `a` becomes the composition of
// everything of this WAVE in front of this lane's stretch, `total` of the whole wave (valid in every lane of the last stretch's channel).
template <int VEC, int CG, int DIR> __device__ __forceinline__ void nf_wave_scan(NfAgg<VEC>& a, NfAgg<VEC>& total, int tg, int packed)
{
    constexpr int TG = 64 / CG;
    auto shift = [&](float v, int d) { return DIR ? __shfl_down(v, d) : __shfl_up(v, d); };
    auto shifti = [&](int v, int d) { return DIR ? __shfl_down(v, d) : __shfl_up(v, d); };
    const int pos = DIR ? TG - 1 - tg : tg;
#pragma unroll
    for (int s = 1; s < TG; s *= 2) {
        NfAgg<VEC> p;
#pragma unroll
        for (int k = 0; k < VEC; ++k) { p.P[k] = shift(a.P[k], s * CG); p.H[k] = shift(a.H[k], s * CG); }
        p.closed = packed ? shifti(a.closed, s * CG) : 0;
        if (pos >= s) a.after(p);
    }
    const int cg = (threadIdx.x & 63) % CG, last = (DIR ? 0 : TG - 1) * CG + cg;
    total.closed = packed ? __shfl(a.closed, last) : 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) { total.P[k] = __shfl(a.P[k], last); total.H[k] = __shfl(a.H[k], last); }
    NfAgg<VEC> e;
#pragma unroll
    for (int k = 0; k < VEC; ++k) { e.P[k] = shift(a.P[k], CG); e.H[k] = shift(a.H[k], CG); }
    e.closed = packed ? shifti(a.closed, CG) : 0;
    if (pos == 0) e.one();
    a = e;
}

// LDS exchange of the waves' totals; two buffers, so that one barrier a tile is enough (a wave can be at most one tile ahead).
template <int VEC, int CG, int NW> struct NfScanLds {
    float P[2][NW][CG * VEC], H[2][NW][CG * VEC];
    int closed[2][NW];
};

template <int VEC, int CG, int NW> __device__ __forceinline__ void nf_lds_put(NfScanLds<VEC, CG, NW>& s, int buf, int w, int lane, const NfAgg<VEC>& t)
{
    if (lane < CG) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) { s.P[buf][w][lane * VEC + k] = t.P[k]; s.H[buf][w][lane * VEC + k] = t.H[k]; }
        if (lane == 0) s.closed[buf][w] = t.closed;
    }
}

template <int VEC, int CG, int NW> __device__ __forceinline__ NfAgg<VEC> nf_lds_get(const NfScanLds<VEC, CG, NW>& s, int buf, int w, int cg)
{
    NfAgg<VEC> t;
#pragma unroll
    for (int k = 0; k < VEC; ++k) { t.P[k] = s.P[buf][w][cg * VEC + k]; t.H[k] = s.H[buf][w][cg * VEC + k]; }
    t.closed = s.closed[buf][w];
    return t;
}

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
template <typename E, int VEC, int CG, int NW>
__global__ void __launch_bounds__(NF_SCAN_WG) k_scan_fwd(NfScanArgs a)
{
    constexpr int TG = 64 / CG, TS = NW * TG * NF_SCAN_TPT;
    typedef typename E::st st;
    __shared__ NfScanLds<VEC, CG, NW> lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cg = lane % CG, tg = lane / CG;
    long long unit = NW == 1 ? (long long)blockIdx.x * 4 + wave : (long long)blockIdx.x;
    if (unit >= (long long)a.B * a.nblk * a.nchunk) return;        // (NW = 1 only: no barrier below)
    const int blk = (int)(unit % a.nblk);
    unit /= a.nblk;
    const int chunk = (int)(unit % a.nchunk), b = (int)(unit / a.nchunk);
    const int w = NW == 1 ? 0 : wave;
    const int ch = (blk * CG + cg) * VEC;
    const bool live = ch < a.D;
    const int chl = live ? ch : 0;
    const int T = a.T, rev = a.reverse, packed = a.sid != nullptr;
    const long long sg = rev ? -1 : 1, t_first = rev ? T - 1 : 0;
    const long long gstep = sg * a.gate_st, xstep = sg * a.x_st, hstep = sg * a.D;
    const int gsize = (sizeof(st) == 4 || a.gate32) ? 4 : 2;
    const char* gp = (const char*)a.gate + ((long long)b * a.gate_sb + t_first * a.gate_st + (a.shared ? 0 : chl)) * gsize;
    const st* xp = (const st*)a.x + (long long)b * a.x_sb + t_first * a.x_st + chl;
    st* hp = (st*)a.h + ((long long)b * T + t_first) * a.D + chl;
    const int tile0 = chunk * a.tiles_per_chunk, tile1 = min(a.ntiles, tile0 + a.tiles_per_chunk);
    float c[VEC], Pc[VEC];               // the state that enters the tile; only_agg: the product of the chunk so far
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        Pc[k] = 1.f;
        c[k] = a.only_agg ? 0.f : a.carry ? a.carry[((long long)b * a.nchunk + chunk) * a.D + chl + k]
                                          : (a.h0 && !packed) ? a.h0[(long long)b * a.D + chl + k] : 0.f;
    }
    NfStretch<E, VEC> xs;
    NfGateStretch<E, VEC> gs;
    const int off = (w * TG + tg) * NF_SCAN_TPT;
    gs.load(a, gp, gstep, tile0 * TS + off, T);
    xs.load(xp, xstep, tile0 * TS + off, T);
    int buf = 0;
    for (int tile = tile0; tile < tile1; ++tile, buf ^= 1) {
        const int j0 = tile * TS + off;
        float A[NF_SCAN_TPT][VEC], x[NF_SCAN_TPT][VEC];
        gs.get(a, A);
#pragma unroll
        for (int i = 0; i < NF_SCAN_TPT; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[i][k] = xs.at(i, k);
        if (tile + 1 < tile1) {          // the next tile is on its way while this one is worked on
            gs.load(a, gp, gstep, j0 + TS, T);
            xs.load(xp, xstep, j0 + TS, T);
        }
        NfMarks m = {0u, 0u, 0u};
        if (packed) m = nf_scan_marks(a.sid, j0, T, rev);
        else if (j0 < T && j0 + NF_SCAN_TPT >= T) m.end = 1u << (T - 1 - j0);
        unsigned idle = m.none;
        if (j0 + NF_SCAN_TPT > T) idle |= j0 >= T ? ~0u : ~0u << (T - j0);
        if (idle) {
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i)
                if (idle >> i & 1u)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) { A[i][k] = 1.f; x[i][k] = 0.f; }
        }
        if (m.start && a.h0) {           // the first step of a sequence: its initial state goes in with x, nothing comes from before
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i)
                if (m.start >> i & 1u) {
                    const int s = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) x[i][k] = fmaf(A[i][k], a.h0[(long long)s * a.D + chl + k], x[i][k]);
                }
        }
        NfAgg<VEC> me, tot;
        me.one();
        if (m.start) {
            me.closed = 1;
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) me.H[k] = (m.start >> i & 1u) ? x[i][k] : fmaf(A[i][k], me.H[k], x[i][k]);
        } else {
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) { me.H[k] = fmaf(A[i][k], me.H[k], x[i][k]); me.P[k] *= A[i][k]; }
        }
        nf_wave_scan<VEC, CG, 0>(me, tot, tg, packed);
        if (a.states && !a.only_agg && w == 0 && tg == 0 && live)
#pragma unroll
            for (int k = 0; k < VEC; ++k) a.states[((long long)b * a.ntiles + tile) * a.D + ch + k] = c[k];
        float s[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[k] = c[k];
        if (NW > 1) {
            nf_lds_put<VEC, CG, NW>(lds, buf, w, lane, tot);
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NW; ++v) {
                const NfAgg<VEC> o = nf_lds_get<VEC, CG, NW>(lds, buf, v, cg);
                if (v == w)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) s[k] = c[k];
                o.apply(c);
#pragma unroll
                for (int k = 0; k < VEC; ++k) Pc[k] *= o.P[k];
            }
        } else {
            tot.apply(c);
#pragma unroll
            for (int k = 0; k < VEC; ++k) Pc[k] *= tot.P[k];
        }
        if (a.only_agg) continue;
        me.apply(s);
        if (j0 < T) {
            st* q = hp + j0 * hstep;
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) s[k] = (m.start >> i & 1u) ? x[i][k] : fmaf(A[i][k], s[k], x[i][k]);
                if (live && j0 + i < T) {
                    if (m.none >> i & 1u) { const float z[VEC] = {}; nf_put<E, VEC>(q, z); }
                    else nf_put<E, VEC>(q, s);
                    if (m.end >> i & 1u) {
                        const int q_ = packed ? a.sid[rev ? T - 1 - (j0 + i) : j0 + i] : b;      // the final state is the last step's, to the bit
#pragma unroll
                        for (int k = 0; k < VEC; ++k) a.h_last[(long long)q_ * a.D + ch + k] = s[k];
                    }
                }
                q += hstep;
            }
        }
    }
    if (a.only_agg && w == 0 && tg == 0 && live) {
        float* o = a.agg + ((long long)b * a.nchunk + chunk) * 2 * a.D + ch;
#pragma unroll
        for (int k = 0; k < VEC; ++k) { o[k] = Pc[k]; o[a.D + k] = c[k]; }
    }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
template <typename E, int VEC, int CG, int NW>
__global__ void __launch_bounds__(NF_SCAN_WG) k_scan_bwd(NfScanArgs a)
{
    constexpr int TG = 64 / CG, TS = NW * TG * NF_SCAN_TPT;
    typedef typename E::st st;
    __shared__ NfScanLds<VEC, CG, NW> lds_f, lds_r;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cg = lane % CG, tg = lane / CG;
    long long unit = NW == 1 ? (long long)blockIdx.x * 4 + wave : (long long)blockIdx.x;
    if (unit >= (long long)a.B * a.nblk * a.nchunk) return;
    const int blk = (int)(unit % a.nblk);
    unit /= a.nblk;
    const int chunk = (int)(unit % a.nchunk), b = (int)(unit / a.nchunk);
    const int w = NW == 1 ? 0 : wave;
    const int ch = (blk * CG + cg) * VEC;
    const bool live = ch < a.D;
    const int chl = live ? ch : 0;
    const int T = a.T, rev = a.reverse, packed = a.sid != nullptr;
    const long long sg = rev ? -1 : 1, t_first = rev ? T - 1 : 0;
    const long long gstep = sg * a.gate_st, xstep = sg * a.x_st, dstep = sg * a.D, ystep = sg * a.g_st;
    const int gsize = (sizeof(st) == 4 || a.gate32) ? 4 : 2;
    const char* gp = (const char*)a.gate + ((long long)b * a.gate_sb + t_first * a.gate_st + (a.shared ? 0 : chl)) * gsize;
    const st* xp = (const st*)a.x + (long long)b * a.x_sb + t_first * a.x_st + chl;
    const st* yp = a.g ? (const st*)a.g + (long long)b * a.g_sb + t_first * a.g_st + chl : nullptr;
    const long long orow = (long long)b * T + t_first;
    const int tile0 = chunk * a.tiles_per_chunk, tile1 = min(a.ntiles, tile0 + a.tiles_per_chunk);
    float u[VEC], Pc[VEC];               // u: the gradient that enters the tile from behind
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        Pc[k] = 1.f;
        u[k] = a.only_agg ? 0.f : a.carry ? a.carry[((long long)b * a.nchunk + chunk) * a.D + chl + k]
                                          : (a.g_last && !packed) ? a.g_last[(long long)b * a.D + chl + k] : 0.f;
    }
    NfStretch<E, VEC> xs, ys;
    NfGateStretch<E, VEC> gs;
    float cn[VEC];                       // the state at the (next) tile's start
    const int off = (w * TG + tg) * NF_SCAN_TPT;
    auto fetch = [&](int tile) {
        const int j0 = tile * TS + off;
        gs.load(a, gp, gstep, j0, T);
        if (yp) ys.load(yp, ystep, j0, T);
        if (!a.only_agg) {
            xs.load(xp, xstep, j0, T);
#pragma unroll
            for (int k = 0; k < VEC; ++k) cn[k] = a.states[((long long)b * a.ntiles + tile) * a.D + chl + k];
        }
    };
    fetch(tile1 - 1);
    int buf = 0;
    for (int tile = tile1 - 1; tile >= tile0; --tile, buf ^= 1) {
        const int j0 = tile * TS + off;
        float A[NF_SCAN_TPT][VEC], x[NF_SCAN_TPT][VEC], y[NF_SCAN_TPT][VEC], c[VEC];
        gs.get(a, A);
#pragma unroll
        for (int k = 0; k < VEC; ++k) c[k] = a.only_agg ? 0.f : cn[k];
#pragma unroll
        for (int i = 0; i < NF_SCAN_TPT; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) { x[i][k] = a.only_agg ? 0.f : xs.at(i, k); y[i][k] = yp ? ys.at(i, k) : 0.f; }
        if (tile > tile0) fetch(tile - 1);
        NfMarks m = {0u, 0u, 0u};
        if (packed) m = nf_scan_marks(a.sid, j0, T, rev);
        unsigned idle = m.none;
        if (j0 + NF_SCAN_TPT > T) idle |= j0 >= T ? ~0u : ~0u << (T - j0);
        if (idle) {
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i)
                if (idle >> i & 1u)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) { A[i][k] = 1.f; x[i][k] = 0.f; y[i][k] = 0.f; }
        }
        if (m.end && a.g_last) {         // the last step of a sequence takes the gradient of its final state
#pragma unroll
            for (int i = 0; i < NF_SCAN_TPT; ++i)
                if (m.end >> i & 1u) {
                    const int s = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) y[i][k] += a.g_last[(long long)s * a.D + chl + k];
                }
        }
        // backwards: the stretch as u -> P u + H
        NfAgg<VEC> rv, rtot;
        rv.one();
        if (m.end) rv.closed = 1;
#pragma unroll
        for (int i = NF_SCAN_TPT - 1; i >= 0; --i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                rv.H[k] = A[i][k] * (((m.end >> i & 1u) ? 0.f : rv.H[k]) + y[i][k]);
                rv.P[k] *= A[i][k];
            }
        // forwards: the stretch as c -> P c + H, started anew where a sequence begins
        NfAgg<VEC> fw, ftot;
        float hs0[NF_SCAN_TPT][VEC];     // the initial state of a sequence that begins at step i
        if (!a.only_agg) {
            fw.one();
            if (m.start) {
                fw.closed = 1;
#pragma unroll
                for (int i = 0; i < NF_SCAN_TPT; ++i) {
                    int s = 0;
                    if (m.start >> i & 1u) s = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        hs0[i][k] = ((m.start >> i & 1u) && a.h0) ? a.h0[(long long)s * a.D + chl + k] : 0.f;
                        fw.H[k] = fmaf(A[i][k], (m.start >> i & 1u) ? hs0[i][k] : fw.H[k], x[i][k]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < NF_SCAN_TPT; ++i)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) { fw.H[k] = fmaf(A[i][k], fw.H[k], x[i][k]); fw.P[k] *= A[i][k]; hs0[i][k] = 0.f; }
            }
            nf_wave_scan<VEC, CG, 0>(fw, ftot, tg, packed);
        }
        nf_wave_scan<VEC, CG, 1>(rv, rtot, tg, packed);
        float su[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) su[k] = u[k];
        if (NW > 1) {
            nf_lds_put<VEC, CG, NW>(lds_r, buf, w, lane, rtot);
            if (!a.only_agg) nf_lds_put<VEC, CG, NW>(lds_f, buf, w, lane, ftot);
            __syncthreads();
#pragma unroll
            for (int v = NW - 1; v >= 0; --v) {
                const NfAgg<VEC> o = nf_lds_get<VEC, CG, NW>(lds_r, buf, v, cg);
                if (v == w)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) su[k] = u[k];
                o.apply(u);
#pragma unroll
                for (int k = 0; k < VEC; ++k) Pc[k] *= o.P[k];
            }
            if (!a.only_agg)
#pragma unroll
                for (int v = 0; v < NW - 1; ++v)
                    if (v < w) nf_lds_get<VEC, CG, NW>(lds_f, buf, v, cg).apply(c);
        } else {
            rtot.apply(u);
#pragma unroll
            for (int k = 0; k < VEC; ++k) Pc[k] *= rtot.P[k];
        }
        if (a.only_agg) continue;
        fw.apply(c);
        rv.apply(su);
        // the states in front of every step, then the gradients from the last step to the first
        float hb[NF_SCAN_TPT][VEC];
#pragma unroll
        for (int i = 0; i < NF_SCAN_TPT; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                if (m.start >> i & 1u) c[k] = hs0[i][k];
                hb[i][k] = c[k];
                c[k] = fmaf(A[i][k], c[k], x[i][k]);
            }
        float dsum[NF_SCAN_TPT];
#pragma unroll
        for (int i = NF_SCAN_TPT - 1; i >= 0; --i) {
            float dx[VEC], dg[VEC];
            dsum[i] = 0.f;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                dx[k] = ((m.end >> i & 1u) ? 0.f : su[k]) + y[i][k];
                su[k] = A[i][k] * dx[k];
                dg[k] = (a.log_gate ? su[k] : dx[k]) * hb[i][k];
            }
            if (m.none >> i & 1u)
#pragma unroll
                for (int k = 0; k < VEC; ++k) dx[k] = dg[k] = 0.f;
            const int j = j0 + i;
            if (live && j < T) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) dsum[i] += dg[k];
                if (a.dx) nf_put<E, VEC>((st*)a.dx + orow * a.D + ch + j * dstep, dx);
                if (!a.shared && a.dgate) {
                    const long long o = orow * a.D + ch + j * dstep;
                    if (sizeof(st) == 4 || a.gate32) nf_put<NfF32, VEC>((float*)a.dgate + o, dg);
                    else nf_put<E, VEC>((st*)a.dgate + o, dg);
                }
                if ((m.start >> i & 1u) && a.dh0) {
                    const int q_ = a.sid[rev ? T - 1 - j : j];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) a.dh0[(long long)q_ * a.D + ch + k] = su[k];
                }
            }
        }
        if (a.shared && a.dgate) {
            // sum over the channels of the block: halves of the steps change sides at every level, so that a lane ends with the sums of
            // TPT / CG steps (or a share of one) after TPT - 1 shuffles and a few
            int first = 0;
#pragma unroll
            for (int mm = CG / 2, n = NF_SCAN_TPT; mm >= 1; mm /= 2) {
                if (n > 1) {
                    const bool up = cg & mm;
                    n /= 2;
#pragma unroll
                    for (int i = 0; i < NF_SCAN_TPT / 2; ++i)
                        if (i < n) {
                            const float keep = up ? dsum[i + n] : dsum[i], send = up ? dsum[i] : dsum[i + n];
                            dsum[i] = keep + __shfl_xor(send, mm);
                        }
                    first += up ? n : 0;
                } else dsum[0] += __shfl_xor(dsum[0], mm);
            }
            constexpr int N = CG >= NF_SCAN_TPT ? 1 : NF_SCAN_TPT / CG, REST = CG >= NF_SCAN_TPT ? CG / NF_SCAN_TPT : 1;
            if (cg % REST == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int j = j0 + first + i;
                    if (j < T) {
                        const long long o = orow + sg * j;
                        if (a.nblk > 1) a.dgate_part[(long long)blk * a.B * T + o] = dsum[i];
                        else if (sizeof(st) == 4 || a.gate32) ((float*)a.dgate)[o] = dsum[i];
                        else ((st*)a.dgate)[o] = E::pk(dsum[i]);
                    }
                }
            }
        }
    }
    if (w == 0 && tg == 0 && live) {
        if (a.only_agg) {
            float* o = a.agg + ((long long)b * a.nchunk + chunk) * 2 * a.D + ch;
#pragma unroll
            for (int k = 0; k < VEC; ++k) { o[k] = Pc[k]; o[a.D + k] = u[k]; }
        } else if (!packed && chunk == 0 && a.dh0)
#pragma unroll
            for (int k = 0; k < VEC; ++k) a.dh0[(long long)b * a.D + ch + k] = u[k];
    }
}

template <typename E> int nf_scan_launch(const NfScanArgs& a, int vec, int cg, int nw, int backward, hipStream_t st)
{
    const long long units = (long long)a.B * a.nblk * a.nchunk;
    const dim3 grid((unsigned)(nw == 1 ? (units + 3) / 4 : units));
#define NF_SCAN_GO(V, C, W)                                                                                       \
    if (vec == V && cg == C && nw == W) {                                                                         \
        if (backward) hipLaunchKernelGGL((k_scan_bwd<E, V, C, W>), grid, dim3(NF_SCAN_WG), 0, st, a);              \
        else hipLaunchKernelGGL((k_scan_fwd<E, V, C, W>), grid, dim3(NF_SCAN_WG), 0, st, a);                       \
        return 1;                                                                                                 \
    }
#define NF_SCAN_GO_W(V, C) NF_SCAN_GO(V, C, 1) NF_SCAN_GO(V, C, 4)
    NF_SCAN_GO_W(2, 32) NF_SCAN_GO_W(2, 16) NF_SCAN_GO_W(2, 8) NF_SCAN_GO_W(2, 2)
    NF_SCAN_GO_W(1, 32) NF_SCAN_GO_W(1, 16) NF_SCAN_GO_W(1, 8) NF_SCAN_GO_W(1, 2)
#undef NF_SCAN_GO_W
#undef NF_SCAN_GO
    return 0;
}
int nf_scan_launch_f32(const NfScanArgs& a, int vec, int cg, int nw, int backward, hipStream_t st);
int nf_scan_launch_bf16(const NfScanArgs& a, int vec, int cg, int nw, int backward, hipStream_t st);
int nf_scan_launch_f16(const NfScanArgs& a, int vec, int cg, int nw, int backward, hipStream_t st);
