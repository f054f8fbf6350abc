// nf_scan.h — kernels of the gated linear recurrence (one instantiation per storage type: nf_scan_f32 / _bf16 / _f16.hip).
//
//   h_t = A_t h_{t-1} + x_t,   A_t = gate_t or exp(gate_t)                                  (forward; reverse: t runs downwards)
//   u_t = A_t (g_t + u_{t+1}), dx_t = g_t + u_{t+1}, dA_t = dx_t h_{t-1} (log gate: times A_t), dh0 = u_0      (backward)
//
// A stretch of steps acts on the state that enters it as  h -> P h + H  (P = the product of its gates, H = what it gives from a zero
// state), and two stretches compose: (P1, H1) then (P2, H2) = (P1 P2, P2 H1 + H2).  The time axis is cut into one stretch of TPT steps per
// thread: a thread reduces its stretch to (P, H) in registers, the stretches of a tile are composed across lanes (shuffles) and
// waves (LDS), and with the state that really enters it every thread then runs its steps once more, one after the other, in fp32 — so
// a state is rounded only where it is stored, and the products P only carry states from one stretch to the next.  The order of every
// sum is fixed by the sizes: results repeat bit for bit.  The backward recomputes the states of a tile from x and
// the state at the tile's start (kept by the forward in fp32: 1 / tile of a tensor) instead of reading h back, which would be as many
// bytes but rounded to the storage type.
//
// Lanes: CG channel groups of VEC adjacent channels x 64 / CG stretches; NW waves share a tile.
//
// A (sequence, block of channels) is a chain; its tiles follow one another.
//   many chains (CHAIN = false): NW waves walk a whole chain (NW = 1: four independent chains a workgroup, no barrier);
//   few chains (CHAIN = true): a workgroup takes ONE tile.  It publishes the tile's (P, H), collects those of the tiles in front of it and goes on
//     with the state they make: every tensor is still read and written once.  The collection has a fixed shape, whatever the order of
//     arrival: tiles in groups of 16, groups in sets of 16; a group's last tile publishes the group's (P, H), a set's last tile the state behind it;
//     a tile composes the set's state, the groups of its set and the tiles of its group in front of it, at most 31 entries.
//     Tiles are handed out by a counter, those of every chain in order, so a tile waits only for workgroups that already run (each
//     publishes its own (P, H) before it waits for anything), and every wait ends.  An entry is one 64-bit word, written and read
//     by relaxed device-scope atomics: it is there or it is not, no fence is needed.  The words are set to "empty" by a launch in front.
#pragma once
#include "nf_common.h"

#define NF_SCAN_WG 256
#define NF_SCAN_MAX_STEPS (1 << 30)
#define NF_SCAN_MAX_CHANNELS (1 << 20)
#define NF_SCAN_FAN 16                               // tiles a group, groups a set
#define NF_SCAN_EMPTY 0xffffffffffffffffull
#define NF_SCAN_CLOSED 0xfffffffeu                   // in P's place: a sequence begins inside, nothing of the entering state comes out

struct NfScanArgs {
    const void* gate; const void* x; const void* g;
    const float* h0; const float* g_last;
    void* h; float* h_last; float* states;
    void* dgate; float* dgate_part; void* dx; float* dh0;
    const int* sid;                      // packed: the sequence of every row (-1: none), else NULL
    unsigned long long* ws_tile; unsigned long long* ws_group; unsigned long long* ws_set;      // [k][chain][CG * VEC]
    int* ticket;
    long long gate_sb, x_sb, g_sb;       // strides of a batch, in bytes
    int gate_st, x_st, g_st;             // strides of a step, in bytes (a tile's rows span less than 2^31)
    int B, T, D, nblk, ntiles;
    int gate32, shared, log_gate, reverse;
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

// Where the rows of a tile lie: uniform base, 32-bit offsets.  jl = step within the tile in processing order.
template <int TS> struct NfRows {
    int rev, last;                       // last: the tile's last step that exists
    __device__ __forceinline__ NfRows(int tile, int T, int reverse) : rev(reverse), last(min(TS, T - tile * TS) - 1) {}
    __device__ __forceinline__ long long first(int tile, int T) const { return rev ? (long long)T - TS - (long long)tile * TS : (long long)tile * TS; }
    __device__ __forceinline__ unsigned at(int jl) const { return (unsigned)(rev ? TS - 1 - jl : jl); }
};

// One thread's stretch of a tensor as it lies in memory.
template <typename E, int VEC, int TPT> struct NfStretch {
    typename NfVec<E, VEC>::type r[TPT];
    template <int TS> __device__ __forceinline__ void load(const char* base, unsigned lane_off, int step, int jl, const NfRows<TS>& rows)
    {
        typedef typename NfVec<E, VEC>::type V;
        if (rows.last == TS - 1) {
            const unsigned o = rows.at(jl) * (unsigned)step + lane_off;
            const int s = rows.rev ? -step : step;
#pragma unroll
            for (int i = 0; i < TPT; ++i) r[i] = *(const V*)(base + (unsigned)(o + i * s));
        } else {
#pragma unroll
            for (int i = 0; i < TPT; ++i) r[i] = *(const V*)(base + (unsigned)(rows.at(min(jl + i, rows.last)) * (unsigned)step + lane_off));
        }
    }
    __device__ __forceinline__ float at(int i, int k) const { return E::cv(r[i][k]); }
};

// The gate comes in the storage type or in fp32, per channel or one per step: both are uniform branches.
template <typename E, int VEC, int TPT> struct NfGateStretch {
    unsigned r[TPT * VEC];               // fp32: a word per channel; else the row's VEC elements packed from word VEC * i on
    template <typename W, int TS>
    __device__ __forceinline__ void load_as(const char* base, unsigned lane_off, int step, int jl, const NfRows<TS>& rows)
    {
        constexpr int N = (sizeof(W) + 3) / 4;
        const bool full = rows.last == TS - 1;
        const unsigned o = rows.at(jl) * (unsigned)step + lane_off;
        const int s = rows.rev ? -step : step;
#pragma unroll
        for (int i = 0; i < TPT; ++i) {
            const unsigned oo = full ? (unsigned)(o + i * s) : rows.at(min(jl + i, rows.last)) * (unsigned)step + lane_off;
            const W v = *(const W*)(base + oo);
            if constexpr (sizeof(W) < 4) r[VEC * i] = (unsigned)v;
            else if constexpr (N == 1) r[VEC * i] = __builtin_bit_cast(unsigned, v);
            else
#pragma unroll
                for (int k = 0; k < N; ++k) r[VEC * i + k] = v[k];
        }
    }
    template <int TS> __device__ __forceinline__ void load(const NfScanArgs& a, const char* base, unsigned lane_off, int jl, const NfRows<TS>& rows)
    {
        typedef unsigned W32 __attribute__((ext_vector_type(VEC)));
        typedef unsigned W16 __attribute__((ext_vector_type(VEC >= 4 ? VEC / 2 : 2)));
        if (sizeof(typename E::st) == 4 || a.gate32) {
            if (a.shared || VEC == 1) load_as<unsigned>(base, lane_off, a.gate_st, jl, rows);
            else load_as<W32>(base, lane_off, a.gate_st, jl, rows);
        } else {
            if (a.shared || VEC == 1) load_as<unsigned short>(base, lane_off, a.gate_st, jl, rows);
            else if (VEC == 2) load_as<unsigned>(base, lane_off, a.gate_st, jl, rows);
            else load_as<W16>(base, lane_off, a.gate_st, jl, rows);
        }
    }
    __device__ __forceinline__ void get(const NfScanArgs& a, float (&A)[TPT][VEC]) const
    {
#pragma unroll
        for (int i = 0; i < TPT; ++i) {
            if (sizeof(typename E::st) == 4 || a.gate32) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) A[i][k] = __uint_as_float(r[VEC * i + (a.shared ? 0 : k)]);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const unsigned w = r[VEC * i + (a.shared ? 0 : k / 2)];
                    A[i][k] = E::cv((typename E::st)((k & 1) && !a.shared ? w >> 16 : w & 0xffffu));
                }
            }
        }
        if (a.log_gate) {
#pragma unroll
            for (int i = 0; i < TPT; ++i) {
                if (a.shared) {
                    const float e = expf(A[i][0]);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) A[i][k] = e;
                } else
#pragma unroll
                    for (int k = 0; k < VEC; ++k) A[i][k] = expf(A[i][k]);
            }
        }
    }
};

template <typename E, int VEC> __device__ __forceinline__ void nf_put(char* p, const float (&v)[VEC])
{
    typename NfVec<E, VEC>::type w;
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[k] = E::pk(v[k]);
    *(typename NfVec<E, VEC>::type*)p = w;
}

// Which steps of a stretch start / end a sequence and which belong to none (bit i), for packed rows.
struct NfMarks { unsigned start, end, none; };
template <int TPT> __device__ __forceinline__ NfMarks nf_scan_marks(const int* sid, int j0, int T, int reverse)
{
    NfMarks m = {0u, 0u, 0u};
    auto at = [&](int j) { return (j < 0 || j >= T) ? -2 : sid[reverse ? T - 1 - j : j]; };
    int s[TPT + 2];
#pragma unroll
    for (int i = 0; i < TPT + 2; ++i) s[i] = at(j0 - 1 + i);
#pragma unroll
    for (int i = 0; i < TPT; ++i) {
        if (s[i + 1] < 0) m.none |= 1u << i;
        else {
            if (s[i + 1] != s[i]) m.start |= 1u << i;
            if (s[i + 1] != s[i + 2]) m.end |= 1u << i;
        }
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
    __device__ __forceinline__ void one()
    {
        closed = 0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) { P[k] = 1.f; H[k] = 0.f; }
    }
};

// Composition over the stretches of a wave in processing order (DIR = 0: upwards, 1: downwards): `a` becomes the composition of
// everything in front of this lane's stretch, `total` that of the whole wave (in every lane).
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
    __device__ __forceinline__ void put(int buf, int w, int lane, const NfAgg<VEC>& t)
    {
        if (lane < CG) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) { P[buf][w][lane * VEC + k] = t.P[k]; H[buf][w][lane * VEC + k] = t.H[k]; }
            if (lane == 0) closed[buf][w] = t.closed;
        }
    }
    __device__ __forceinline__ NfAgg<VEC> get(int buf, int w, int cg) const
    {
        NfAgg<VEC> t;
#pragma unroll
        for (int k = 0; k < VEC; ++k) { t.P[k] = P[buf][w][cg * VEC + k]; t.H[k] = H[buf][w][cg * VEC + k]; }
        t.closed = closed[buf][w];
        return t;
    }
};

// ---- the chain's exchange --------------------------------------------------------------------------
template <int VEC> __device__ __forceinline__ void nf_publish(unsigned long long* p, const NfAgg<VEC>& t)
{
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        const unsigned P = t.closed ? NF_SCAN_CLOSED : t.P[k] != t.P[k] ? 0x7fc00000u : __float_as_uint(t.P[k]);      // (a NaN never looks like a mark)
        __hip_atomic_store(p + k, (unsigned long long)__float_as_uint(t.H[k]) << 32 | P, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
template <int VEC> struct NfEntry {
    unsigned long long w[VEC];
    __device__ __forceinline__ void ask(const unsigned long long* p)
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[k] = __hip_atomic_load(p + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __device__ __forceinline__ NfAgg<VEC> wait(const unsigned long long* p)
    {
        NfAgg<VEC> t;
        t.closed = 0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            while (w[k] == NF_SCAN_EMPTY) w[k] = __hip_atomic_load(p + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            t.P[k] = __uint_as_float((unsigned)w[k]); t.H[k] = __uint_as_float((unsigned)(w[k] >> 32));
            t.closed |= (unsigned)w[k] == NF_SCAN_CLOSED;
        }
        return t;
    }
};

// The state that enters tile k of a chain (one wave's work; c = the chain's initial state), and the publications that tile k owes: `own` is its (P, H).
template <int VEC, int CG> __device__ __forceinline__ void nf_chain(const NfScanArgs& a, int k, int chain, int nchains, int cg, int tg,
                                                                    const NfAgg<VEC>& own, int packed, float (&c)[VEC])
{
    constexpr int TG = 64 / CG, CH = CG * VEC, PER = (NF_SCAN_FAN - 1 + TG - 1) / TG;
    const int grp = k / NF_SCAN_FAN, set = grp / NF_SCAN_FAN, nt = k % NF_SCAN_FAN, ng = grp % NF_SCAN_FAN;
    auto word = [&](unsigned long long* ws, int idx) { return ws + ((long long)idx * nchains + chain) * CH + cg * VEC; };
    if (k + 1 < a.ntiles && tg == 0) nf_publish<VEC>(word(a.ws_tile, k), own);
    NfEntry<VEC> et[PER], eg[PER], es;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = tg * PER + i;
        if (e < nt) et[i].ask(word(a.ws_tile, grp * NF_SCAN_FAN + e));
        if (e < ng) eg[i].ask(word(a.ws_group, set * NF_SCAN_FAN + e));
    }
    if (set > 0) es.ask(word(a.ws_set, set - 1));
    NfAgg<VEC> t, tot;
    t.one();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = tg * PER + i;
        if (e < nt) { NfAgg<VEC> n = et[i].wait(word(a.ws_tile, grp * NF_SCAN_FAN + e)); if (i > 0) n.after(t); t = n; }
    }
    nf_wave_scan<VEC, CG, 0>(t, tot, tg, packed);
    const NfAgg<VEC> tiles = tot;
    if (nt == NF_SCAN_FAN - 1 && k + 1 < a.ntiles && tg == 0) {
        NfAgg<VEC> g = own;
        g.after(tiles);
        nf_publish<VEC>(word(a.ws_group, grp), g);
    }
    t.one();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = tg * PER + i;
        if (e < ng) { NfAgg<VEC> n = eg[i].wait(word(a.ws_group, set * NF_SCAN_FAN + e)); if (i > 0) n.after(t); t = n; }
    }
    nf_wave_scan<VEC, CG, 0>(t, tot, tg, packed);
    if (set > 0) {
        const NfAgg<VEC> s = es.wait(word(a.ws_set, set - 1));
#pragma unroll
        for (int i = 0; i < VEC; ++i) c[i] = s.H[i];
    }
    tot.apply(c);
    tiles.apply(c);
    if (nt == NF_SCAN_FAN - 1 && ng == NF_SCAN_FAN - 1 && k + 1 < a.ntiles && tg == 0) {
        float o[VEC];
        NfAgg<VEC> s;
        s.one();
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = c[i];
        own.apply(o);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s.H[i] = o[i];
        nf_publish<VEC>(word(a.ws_set, set), s);
    }
}

// A workgroup's place: the chain, and for CHAIN its tile by ticket.
struct NfPlace { int blk, b, k, w; bool ok; };
template <int NW, bool CHAIN> __device__ __forceinline__ NfPlace nf_place(const NfScanArgs& a)
{
    __shared__ int s_ticket;
    NfPlace p;
    const int nchains = a.B * a.nblk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int chain;
    if (CHAIN) {
        if (threadIdx.x == 0) s_ticket = __hip_atomic_fetch_add(a.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        const int t = __builtin_amdgcn_readfirstlane(s_ticket);
        chain = t % nchains;
        p.k = t / nchains;
    } else {
        chain = NW == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
        p.k = 0;
    }
    p.ok = chain < nchains;
    p.blk = chain % a.nblk;
    p.b = chain / a.nblk;
    p.w = NW == 1 ? 0 : wave;
    return p;
}

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
template <typename E, int VEC, int CG, int TPT, int NW, bool CHAIN>
__global__ void __launch_bounds__(NW == 1 ? NF_SCAN_WG : 64 * NW) k_scan_fwd(NfScanArgs a)
{
    constexpr int TG = 64 / CG, TS = NW * TG * TPT, ES = sizeof(typename E::st);
    __shared__ NfScanLds<VEC, CG, NW> lds;
    __shared__ float s_c[CHAIN ? CG * VEC : 1];
    const NfPlace pl = nf_place<NW, CHAIN>(a);
    if (!pl.ok) return;                                  // (NW = 1 only: no barrier below)
    const int lane = threadIdx.x & 63, cg = lane % CG, tg = lane / CG, w = pl.w, b = pl.b;
    const int ch = (pl.blk * CG + cg) * VEC;
    const bool live = ch < a.D;
    const int chl = live ? ch : 0;
    const int T = a.T, rev = a.reverse, packed = a.sid != nullptr;
    const int gs = (ES == 4 || a.gate32) ? 4 : 2, hstep = a.D * ES;
    const char* gbase = (const char*)a.gate + b * a.gate_sb;
    const char* xbase = (const char*)a.x + b * a.x_sb;
    char* hbase = (char*)a.h + (long long)b * T * hstep;
    const unsigned goff = a.shared ? 0u : (unsigned)(chl * gs), xoff = (unsigned)(chl * ES);
    const int jl = (w * TG + tg) * TPT;
    float c[VEC];                        // the state that enters the tile
#pragma unroll
    for (int k = 0; k < VEC; ++k) c[k] = (a.h0 && !packed) ? a.h0[(long long)b * a.D + chl + k] : 0.f;
    int buf = 0;
    for (int tile = pl.k; tile < (CHAIN ? pl.k + 1 : a.ntiles); ++tile, buf ^= 1) {
        const NfRows<TS> rows(tile, T, rev);
        const long long row0 = rows.first(tile, T);
        NfStretch<E, VEC, TPT> xs;
        NfGateStretch<E, VEC, TPT> gt;
        gt.load(a, gbase + row0 * a.gate_st, goff, jl, rows);
        xs.load(xbase + row0 * a.x_st, xoff, a.x_st, jl, rows);
        const int j0 = tile * TS + jl;
        NfMarks m = {0u, 0u, 0u};
        if (packed) m = nf_scan_marks<TPT>(a.sid, j0, T, rev);
        else if (j0 < T && j0 + TPT >= T) m.end = 1u << (T - 1 - j0);
        float A[TPT][VEC], x[TPT][VEC];
        gt.get(a, A);
#pragma unroll
        for (int i = 0; i < TPT; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[i][k] = xs.at(i, k);
        unsigned idle = m.none;
        if (j0 + TPT > T) idle |= j0 >= T ? ~0u : ~0u << (T - j0);
        if (idle) {
#pragma unroll
            for (int i = 0; i < TPT; ++i)
                if (idle >> i & 1u)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) { A[i][k] = 1.f; x[i][k] = 0.f; }
        }
        if (packed && m.start && a.h0) { // the first step of a sequence: its initial state goes in with x, nothing comes from before
#pragma unroll
            for (int i = 0; i < TPT; ++i)
                if (m.start >> i & 1u) {
                    const int s = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) x[i][k] = fmaf(A[i][k], a.h0[(long long)s * a.D + chl + k], x[i][k]);
                }
        }
        NfAgg<VEC> me, tot;
        me.one();
        if (packed && m.start) {
            me.closed = 1;
#pragma unroll
            for (int i = 0; i < TPT; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) me.H[k] = (m.start >> i & 1u) ? x[i][k] : fmaf(A[i][k], me.H[k], x[i][k]);
        } else {
#pragma unroll
            for (int i = 0; i < TPT; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) { me.H[k] = fmaf(A[i][k], me.H[k], x[i][k]); me.P[k] *= A[i][k]; }
        }
        nf_wave_scan<VEC, CG, 0>(me, tot, tg, packed);
        if (NW > 1) {
            lds.put(buf, w, lane, tot);
            __syncthreads();
        }
        if (CHAIN) {
            if (w == 0) {
                NfAgg<VEC> own = lds.get(buf, 0, cg);
#pragma unroll
                for (int v = 1; v < NW; ++v) { NfAgg<VEC> n = lds.get(buf, v, cg); n.after(own); own = n; }
                nf_chain<VEC, CG>(a, tile, pl.b * a.nblk + pl.blk, a.B * a.nblk, cg, tg, own, packed, c);
                if (tg == 0)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) s_c[cg * VEC + k] = c[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < VEC; ++k) c[k] = s_c[cg * VEC + k];
        }
        if (a.states && w == 0 && tg == 0 && live)
#pragma unroll
            for (int k = 0; k < VEC; ++k) a.states[((long long)b * a.ntiles + tile) * a.D + ch + k] = c[k];
        float s[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[k] = c[k];
        if (NW > 1) {
#pragma unroll
            for (int v = 0; v < NW; ++v) {
                if (v == w)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) s[k] = c[k];
                if (!CHAIN || v < w) lds.get(buf, v, cg).apply(c);
            }
        } else tot.apply(c);
        me.apply(s);
        if (j0 < T) {
            char* hb = hbase + row0 * hstep;
#pragma unroll
            for (int i = 0; i < TPT; ++i) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) s[k] = (packed && (m.start >> i & 1u)) ? x[i][k] : fmaf(A[i][k], s[k], x[i][k]);
                if (live && j0 + i < T) {
                    char* q = hb + (unsigned)(rows.at(jl + i) * (unsigned)hstep + xoff);
                    if (m.none >> i & 1u) { const float z[VEC] = {}; nf_put<E, VEC>(q, z); }
                    else nf_put<E, VEC>(q, s);
                    if (m.end >> i & 1u) {       // the final state is the last step's, to the bit
                        const int q_ = packed ? a.sid[rev ? T - 1 - (j0 + i) : j0 + i] : b;
#pragma unroll
                        for (int k = 0; k < VEC; ++k) a.h_last[(long long)q_ * a.D + ch + k] = s[k];
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
template <typename E, int VEC, int CG, int TPT, int NW, bool CHAIN>
__global__ void __launch_bounds__(NW == 1 ? NF_SCAN_WG : 64 * NW) k_scan_bwd(NfScanArgs a)
{
    constexpr int TG = 64 / CG, TS = NW * TG * TPT, ES = sizeof(typename E::st);
    __shared__ NfScanLds<VEC, CG, NW> lds_f, lds_r;
    __shared__ float s_c[CHAIN ? CG * VEC : 1];
    const NfPlace pl = nf_place<NW, CHAIN>(a);
    if (!pl.ok) return;
    const int lane = threadIdx.x & 63, cg = lane % CG, tg = lane / CG, w = pl.w, b = pl.b;
    const int ch = (pl.blk * CG + cg) * VEC;
    const bool live = ch < a.D;
    const int chl = live ? ch : 0;
    const int T = a.T, rev = a.reverse, packed = a.sid != nullptr;
    const int gs = (ES == 4 || a.gate32) ? 4 : 2, hstep = a.D * ES, gstep = a.D * gs;
    const char* gbase = (const char*)a.gate + b * a.gate_sb;
    const char* xbase = (const char*)a.x + b * a.x_sb;
    const char* ybase = a.g ? (const char*)a.g + b * a.g_sb : nullptr;
    const unsigned goff = a.shared ? 0u : (unsigned)(chl * gs), xoff = (unsigned)(chl * ES);
    const int jl = (w * TG + tg) * TPT;
    float u[VEC];                        // the gradient that enters the tile from behind
#pragma unroll
    for (int k = 0; k < VEC; ++k) u[k] = (a.g_last && !packed) ? a.g_last[(long long)b * a.D + chl + k] : 0.f;
    int buf = 0;
    for (int it = pl.k; it < (CHAIN ? pl.k + 1 : a.ntiles); ++it, buf ^= 1) {
        const int tile = a.ntiles - 1 - it;
        const NfRows<TS> rows(tile, T, rev);
        const long long row0 = rows.first(tile, T);
        NfStretch<E, VEC, TPT> xs, ys;
        NfGateStretch<E, VEC, TPT> gt;
        gt.load(a, gbase + row0 * a.gate_st, goff, jl, rows);
        if (ybase) ys.load(ybase + row0 * a.g_st, xoff, a.g_st, jl, rows);
        xs.load(xbase + row0 * a.x_st, xoff, a.x_st, jl, rows);
        float c[VEC];                    // the state that enters the tile in front
#pragma unroll
        for (int k = 0; k < VEC; ++k) c[k] = a.states[((long long)b * a.ntiles + tile) * a.D + chl + k];
        const int j0 = tile * TS + jl;
        NfMarks m = {0u, 0u, 0u};
        if (packed) m = nf_scan_marks<TPT>(a.sid, j0, T, rev);
        float A[TPT][VEC], x[TPT][VEC], y[TPT][VEC];
        gt.get(a, A);
#pragma unroll
        for (int i = 0; i < TPT; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) { x[i][k] = xs.at(i, k); y[i][k] = ybase ? ys.at(i, k) : 0.f; }
        unsigned idle = m.none;
        if (j0 + TPT > T) idle |= j0 >= T ? ~0u : ~0u << (T - j0);
        if (idle) {
#pragma unroll
            for (int i = 0; i < TPT; ++i)
                if (idle >> i & 1u)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) { A[i][k] = 1.f; x[i][k] = 0.f; y[i][k] = 0.f; }
        }
        if (packed && m.end && a.g_last) {       // the last step of a sequence takes the gradient of its final state
#pragma unroll
            for (int i = 0; i < TPT; ++i)
                if (m.end >> i & 1u) {
                    const int s = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) y[i][k] += a.g_last[(long long)s * a.D + chl + k];
                }
        }
        // backwards: the stretch as u -> P u + H
        NfAgg<VEC> rv, rtot, fw, ftot;
        rv.one();
        rv.closed = packed && m.end;
#pragma unroll
        for (int i = TPT - 1; i >= 0; --i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                rv.H[k] = A[i][k] * (((packed && (m.end >> i & 1u)) ? 0.f : rv.H[k]) + y[i][k]);
                rv.P[k] *= A[i][k];
            }
        // forwards: the stretch as c -> P c + H, started anew where a sequence begins
        fw.one();
        if (packed && m.start) {
            fw.closed = 1;
#pragma unroll
            for (int i = 0; i < TPT; ++i) {
                int s = 0;
                if (m.start >> i & 1u) s = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float h0 = ((m.start >> i & 1u) && a.h0) ? a.h0[(long long)s * a.D + chl + k] : 0.f;
                    fw.H[k] = fmaf(A[i][k], (m.start >> i & 1u) ? h0 : fw.H[k], x[i][k]);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) fw.P[k] = rv.P[k];
#pragma unroll
            for (int i = 0; i < TPT; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) fw.H[k] = fmaf(A[i][k], fw.H[k], x[i][k]);
        }
        nf_wave_scan<VEC, CG, 1>(rv, rtot, tg, packed);
        nf_wave_scan<VEC, CG, 0>(fw, ftot, tg, packed);
        if (NW > 1) {
            lds_r.put(buf, w, lane, rtot);
            lds_f.put(buf, w, lane, ftot);
            __syncthreads();
        }
        if (CHAIN) {
            if (w == 0) {
                NfAgg<VEC> own = lds_r.get(buf, NW - 1, cg);
#pragma unroll
                for (int v = NW - 2; v >= 0; --v) { NfAgg<VEC> n = lds_r.get(buf, v, cg); n.after(own); own = n; }
                nf_chain<VEC, CG>(a, it, pl.b * a.nblk + pl.blk, a.B * a.nblk, cg, tg, own, packed, u);
                if (tg == 0)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) s_c[cg * VEC + k] = u[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < VEC; ++k) u[k] = s_c[cg * VEC + k];
        }
        float su[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) su[k] = u[k];
        if (NW > 1) {
#pragma unroll
            for (int v = NW - 1; v >= 0; --v) {
                if (v == w)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) su[k] = u[k];
                lds_r.get(buf, v, cg).apply(u);
            }
#pragma unroll
            for (int v = 0; v < NW - 1; ++v)
                if (v < w) lds_f.get(buf, v, cg).apply(c);
        } else rtot.apply(u);
        fw.apply(c);
        rv.apply(su);
        // the states in front of every step, then the gradients from the last step to the first
        float hb[TPT][VEC];
#pragma unroll
        for (int i = 0; i < TPT; ++i) {
            if (packed && (m.start >> i & 1u)) {
                const int s = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
#pragma unroll
                for (int k = 0; k < VEC; ++k) c[k] = a.h0 ? a.h0[(long long)s * a.D + chl + k] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) { hb[i][k] = c[k]; c[k] = fmaf(A[i][k], c[k], x[i][k]); }
        }
        const long long orow = (long long)b * T + row0;
        float dsum[TPT];
#pragma unroll
        for (int i = TPT - 1; i >= 0; --i) {
            float dx[VEC], dg[VEC];
            dsum[i] = 0.f;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                dx[k] = ((packed && (m.end >> i & 1u)) ? 0.f : su[k]) + y[i][k];
                su[k] = A[i][k] * dx[k];
                dg[k] = (a.log_gate ? su[k] : dx[k]) * hb[i][k];
            }
            if (m.none >> i & 1u)
#pragma unroll
                for (int k = 0; k < VEC; ++k) dx[k] = dg[k] = 0.f;
            if (live && j0 + i < T) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) dsum[i] += dg[k];
                if (a.dx) nf_put<E, VEC>((char*)a.dx + orow * hstep + (unsigned)(rows.at(jl + i) * (unsigned)hstep + xoff), dx);
                if (!a.shared && a.dgate) {
                    char* q = (char*)a.dgate + orow * gstep + (unsigned)(rows.at(jl + i) * (unsigned)gstep + goff);
                    if (ES == 4 || a.gate32) nf_put<NfF32, VEC>(q, dg);
                    else nf_put<E, VEC>(q, dg);
                }
                if (packed && (m.start >> i & 1u) && a.dh0) {
                    const int q_ = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
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
            for (int mm = CG / 2, n = TPT; mm >= 1; mm /= 2) {
                if (n > 1) {
                    const bool up = cg & mm;
                    n /= 2;
#pragma unroll
                    for (int i = 0; i < TPT / 2; ++i)
                        if (i < n) {
                            const float keep = up ? dsum[i + n] : dsum[i], send = up ? dsum[i] : dsum[i + n];
                            dsum[i] = keep + __shfl_xor(send, mm);
                        }
                    first += up ? n : 0;
                } else dsum[0] += __shfl_xor(dsum[0], mm);
            }
            constexpr int N = CG >= TPT ? 1 : TPT / CG, REST = CG >= TPT ? CG / TPT : 1;
            if (cg % REST == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (j0 + first + i < T) {
                        const long long o = orow + rows.at(jl + first + i);
                        if (a.nblk > 1) a.dgate_part[(long long)pl.blk * a.B * T + o] = dsum[i];
                        else if (ES == 4 || a.gate32) ((float*)a.dgate)[o] = dsum[i];
                        else ((typename E::st*)a.dgate)[o] = E::pk(dsum[i]);
                    }
            }
        }
        if (!packed && it == a.ntiles - 1 && a.dh0 && w == 0 && tg == 0 && live)
#pragma unroll
            for (int k = 0; k < VEC; ++k) a.dh0[(long long)b * a.D + ch + k] = u[k];
    }
}

// (VEC, CG) -> steps a thread; nw: 1, 4 (whole chains) or -NF_SCAN_CW (a tile a workgroup, chained)
#define NF_SCAN_CW 4
#define NF_SCAN_TPT(vec) ((vec) == 4 ? 4 : 8)
template <typename E> int nf_scan_launch(const NfScanArgs& a, int vec, int cg, int nw, int backward, hipStream_t st)
{
    const long long chains = (long long)a.B * a.nblk;
#define NF_SCAN_GO(V, C, W, CH, GRID)                                                                                                            \
    if (vec == V && cg == C && nw == (CH ? -W : W)) {                                                                                           \
        if (backward) hipLaunchKernelGGL((k_scan_bwd<E, V, C, NF_SCAN_TPT(V), W, CH>), dim3((unsigned)(GRID)), dim3(W == 1 ? NF_SCAN_WG : 64 * W), 0, st, a); \
        else hipLaunchKernelGGL((k_scan_fwd<E, V, C, NF_SCAN_TPT(V), W, CH>), dim3((unsigned)(GRID)), dim3(W == 1 ? NF_SCAN_WG : 64 * W), 0, st, a);          \
        return 1;                                                                                                                               \
    }
#define NF_SCAN_GO_W(V, C) NF_SCAN_GO(V, C, 1, false, (chains + 3) / 4) NF_SCAN_GO(V, C, 4, false, chains) NF_SCAN_GO(V, C, NF_SCAN_CW, true, chains * a.ntiles)
    NF_SCAN_GO_W(4, 16) NF_SCAN_GO_W(4, 8) NF_SCAN_GO_W(4, 4) NF_SCAN_GO_W(4, 1)
    NF_SCAN_GO_W(2, 32) NF_SCAN_GO_W(2, 8) NF_SCAN_GO_W(2, 2)
    NF_SCAN_GO_W(1, 32) NF_SCAN_GO_W(1, 8) NF_SCAN_GO_W(1, 2)
#undef NF_SCAN_GO_W
#undef NF_SCAN_GO
    return 0;
}
int nf_scan_launch_f32(const NfScanArgs& a, int vec, int cg, int nw, int backward, hipStream_t st);
int nf_scan_launch_bf16(const NfScanArgs& a, int vec, int cg, int nw, int backward, hipStream_t st);
int nf_scan_launch_f16(const NfScanArgs& a, int vec, int cg, int nw, int backward, hipStream_t st);
