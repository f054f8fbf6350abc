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
//   very many, or short ones (NF_SCAN_WAVE): a wave walks a whole chain, four independent ones a workgroup, no barrier;
//   many (NF_SCAN_WALK): a workgroup walks a whole chain;
//   few (NF_SCAN_CHAIN): a workgroup takes ONE tile.  It publishes the tile's (P, H), collects those of the tiles in front of it and goes on
//     with the state they make: every tensor is still read and written once.  The collection has a fixed shape, whatever the order of
//     arrival: tiles in groups of 16, groups in sets of 16; a group's last tile publishes the group's (P, H), a set's last tile the state behind it;
//     a tile composes the set's state, the groups of its set and the tiles of its group in front of it, at most 31 entries.
//     Tiles are handed out by a counter per chain, in order, so a tile waits only for workgroups that already run (each
//     publishes its own (P, H) before it waits for anything), and every wait ends.  An entry is one 64-bit word, written and read
//     by relaxed device-scope atomics: it is there or it is not, no fence is needed.  The words are set to "empty" by a launch in front.
//
// What bounds them: a step costs two or three products for each value read, so memory does wherever the arithmetic keeps up.  A pass reads and
// writes every tensor once (bytes below, over the time; a large copy on the same card moves 5.2 TB/s).
//   walk: 8 x 2048 x 2048 bf16, fp32 gates, 268 MB forward 52 us (5.2 TB/s), 470 MB backward 88 us (5.3 TB/s);
//   wave: 4096 x 192 x 32 fp32, 205 MB forward 33 us (6.3 TB/s: part of it comes from the last-level cache), 309 MB backward 48 us;
//     256 x 512 x 1024 fp16, 805 MB forward 161 us (5.0 TB/s), 1.3 GB backward 291 us (4.6 TB/s);
//     40 000 x 192 x 4 fp32, 277 MB 59 us (4.7 TB/s): four channels a lane share a gate, so exp and the exchange across 64 lanes weigh on
//     few values, and waves wait for their turn to issue (61 % of their cycles) more than for memory (26 %);
//   chain: 4 x 4096 x 1024 bf16, 101 MB forward 30 us (3.4 TB/s); 65 537 x 256 fp16, 101 MB forward 40 us (2.5 TB/s), 168 MB backward 58 us (2.9 TB/s):
//     a tile's entry reaches the others through memory, group by group and set by set, and a workgroup has no loads under way while it waits for
//     them (a wave waits 74 % of its cycles).
#pragma once
#include "nf_common.h"

#define NF_SCAN_WAVE 0
#define NF_SCAN_CHAIN 1
#define NF_SCAN_WALK 2
#define NF_SCAN_WG 256
#define NF_SCAN_MAX_STEPS (1 << 30)
#define NF_SCAN_MAX_CHANNELS (1 << 20)
#define NF_SCAN_FAN 16                               // tiles a group, groups a set
#define NF_SCAN_EMPTY 0xffffffffffffffffull
#define NF_SCAN_LINE 32                              // ints between two chains' counters: a cache line (one counter for all took 15 ns a tile)
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
    int gate_st, x_st, g_st;             // strides of a step, in bytes (a tile's rows span less than 2^32)
    int B, T, D, nblk, ntiles;
    int gate32, shared, log_gate, reverse;
    int chain0;                          // NF_SCAN_WAVE: the launch's first chain
    int past;                            // x is too large for the caches: stores go around them
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
            unsigned o = rows.at(jl) * (unsigned)step + lane_off;
            const int s = rows.rev ? -step : step;
#pragma unroll
            for (int i = 0; i < TPT; ++i) { r[i] = *(const V*)(base + o); o += s; }
        } else {
#pragma unroll
            for (int i = 0; i < TPT; ++i) r[i] = *(const V*)(base + (unsigned)(rows.at(min(jl + i, rows.last)) * (unsigned)step + lane_off));
        }
    }
    __device__ __forceinline__ void clear(unsigned idle)
    {
#pragma unroll
        for (int i = 0; i < TPT; ++i)
            if (idle >> i & 1u)
#pragma unroll
                for (int k = 0; k < VEC; ++k) r[i][k] = 0;
    }
    __device__ __forceinline__ float at(int i, int k) const { return E::cv(r[i][k]); }
};

// The gate as factors.  It comes in the storage type or in fp32 (a uniform branch), per channel or one per step (SHARED).
template <typename W, int N, int TPT, int TS>
__device__ __forceinline__ void nf_gate_words(unsigned (&r)[TPT][N], const char* base, unsigned lane_off, int step, int jl, const NfRows<TS>& rows)
{
    const bool full = rows.last == TS - 1;
    unsigned o = rows.at(jl) * (unsigned)step + lane_off;
    const int s = rows.rev ? -step : step;
#pragma unroll
    for (int i = 0; i < TPT; ++i) {
        const W v = *(const W*)(base + (full ? o : (unsigned)(rows.at(min(jl + i, rows.last)) * (unsigned)step + lane_off)));
        o += s;
        if constexpr (sizeof(W) < 4) r[i][0] = (unsigned)v;
        else if constexpr (sizeof(W) == 4) r[i][0] = __builtin_bit_cast(unsigned, v);
        else
#pragma unroll
            for (int k = 0; k < (int)(sizeof(W) / 4); ++k) r[i][k] = v[k];
    }
}
template <typename E, int VEC, int TPT, bool SHARED> struct NfGateStretch {
    static constexpr int N = SHARED ? 1 : VEC;
    unsigned r[TPT][N];                  // fp32: a word per channel; else packed from word 0 on
    template <int TS> __device__ __forceinline__ void load(const NfScanArgs& a, const char* base, unsigned lane_off, int jl, const NfRows<TS>& rows)
    {
        typedef unsigned W32 __attribute__((ext_vector_type(N >= 2 ? N : 2)));
        typedef unsigned W16 __attribute__((ext_vector_type(N >= 4 ? N / 2 : 2)));
        if (sizeof(typename E::st) == 4 || a.gate32) {
            if constexpr (N == 1) nf_gate_words<unsigned>(r, base, lane_off, a.gate_st, jl, rows);
            else nf_gate_words<W32>(r, base, lane_off, a.gate_st, jl, rows);
        } else {
            if constexpr (N == 1) nf_gate_words<unsigned short>(r, base, lane_off, a.gate_st, jl, rows);
            else if constexpr (N == 2) nf_gate_words<unsigned>(r, base, lane_off, a.gate_st, jl, rows);
            else nf_gate_words<W16>(r, base, lane_off, a.gate_st, jl, rows);
        }
    }
    __device__ __forceinline__ void get(const NfScanArgs& a, float (&A)[TPT][N]) const
    {
        if (sizeof(typename E::st) == 4 || a.gate32) {
#pragma unroll
            for (int i = 0; i < TPT; ++i)
#pragma unroll
                for (int k = 0; k < N; ++k) A[i][k] = __uint_as_float(r[i][k]);
        } else {
#pragma unroll
            for (int i = 0; i < TPT; ++i)
#pragma unroll
                for (int k = 0; k < N; ++k) A[i][k] = E::cv((typename E::st)((k & 1) ? r[i][k / 2] >> 16 : r[i][k / 2] & 0xffffu));
        }
        if (a.log_gate) {
#pragma unroll
            for (int i = 0; i < TPT; ++i)
#pragma unroll
                for (int k = 0; k < N; ++k) A[i][k] = expf(A[i][k]);
        }
    }
};

// past: around the caches (uniform), for rows of whole cache lines of a tensor that they would not hold anyway
template <typename E, int VEC> __device__ __forceinline__ void nf_put(char* p, const float (&v)[VEC], bool past)
{
    typename NfVec<E, VEC>::type w;
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[k] = E::pk(v[k]);
    if (past) {          // (between the empty statements: the two stores would be made one, and that an ordinary one)
        asm volatile("");
        __builtin_nontemporal_store(w, (typename NfVec<E, VEC>::type*)p);
        asm volatile("");
    } else *(typename NfVec<E, VEC>::type*)p = w;
}

// Which steps of a stretch start / end a sequence and which belong to none (bit i), for packed rows.
struct NfMarks { unsigned start, end, none; };
template <int TPT> __device__ __forceinline__ NfMarks nf_scan_marks(const int* sid, int j0, int T, int reverse)
{
    NfMarks m = {0u, 0u, 0u};
    int s[TPT + 2];
#pragma unroll
    for (int i = 0; i < TPT + 2; ++i) {
        const int j = min(max(j0 - 1 + i, 0), T - 1);
        s[i] = sid[reverse ? T - 1 - j : j];
    }
#pragma unroll
    for (int i = 0; i < TPT + 2; ++i) s[i] = (j0 - 1 + i < 0 || j0 - 1 + i >= T) ? -2 : s[i];
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

// What a zero state adds to a stretch is nothing, however large its product of gates has become (H is what the stretch gives from zero).
__device__ __forceinline__ float nf_carry(float P, float c, float H) { return fmaf(c == 0.f ? 0.f : P, c, H); }
// A product of gates: behind a gate of zero nothing of the entering state is left, also where the other factor has overflowed.  (Gates that are not
// finite themselves show in H.)  v_mul_legacy_f32: 0 times anything = 0.  As LLVM's intrinsic, not as inline assembly: its result goes to row
// exchanges and comes from exp, and the compiler sets the wait states between those and an instruction only where it knows what that is.
extern "C" __device__ __attribute__((const)) float nf_gates(float p, float q) __asm("llvm.amdgcn.fmul.legacy");

// (P, H) of a stretch: N products (1: one gate for all channels), VEC states.
template <int VEC, int N, bool PACKED> struct NfAgg {
    float P[N], H[VEC];
    int closed;             // a sequence begins inside: nothing of the entering state comes out
    __device__ __forceinline__ bool shut() const { return PACKED && closed; }
    __device__ __forceinline__ void after(const NfAgg& p)      // this stretch behind stretch p
    {
        if (shut()) return;
#pragma unroll
        for (int k = 0; k < VEC; ++k) H[k] = nf_carry(P[N == 1 ? 0 : k], p.H[k], H[k]);
#pragma unroll
        for (int k = 0; k < N; ++k) P[k] = nf_gates(P[k], p.P[k]);
        if (PACKED) closed = p.closed;
    }
    __device__ __forceinline__ void apply(float (&c)[VEC]) const
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k) c[k] = shut() ? H[k] : nf_carry(P[N == 1 ? 0 : k], c[k], H[k]);
    }
    __device__ __forceinline__ void one()
    {
        closed = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) P[k] = 1.f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) H[k] = 0.f;
    }
};

// f(value) for every value of a stretch that lanes exchange
template <int VEC, int N, bool PACKED, typename F> __device__ __forceinline__ NfAgg<VEC, N, PACKED> nf_map(const NfAgg<VEC, N, PACKED>& a, F f)
{
    NfAgg<VEC, N, PACKED> r;
#pragma unroll
    for (int k = 0; k < N; ++k) r.P[k] = __int_as_float(f(__float_as_int(a.P[k])));
#pragma unroll
    for (int k = 0; k < VEC; ++k) r.H[k] = __int_as_float(f(__float_as_int(a.H[k])));
    r.closed = PACKED ? f(a.closed) : 0;
    return r;
}
template <int VEC, int N, bool PACKED> __device__ __forceinline__ void nf_take(NfAgg<VEC, N, PACKED>& a, bool take, const NfAgg<VEC, N, PACKED>& b)
{
#pragma unroll
    for (int k = 0; k < N; ++k) a.P[k] = take ? b.P[k] : a.P[k];
#pragma unroll
    for (int k = 0; k < VEC; ++k) a.H[k] = take ? b.H[k] : a.H[k];
    if (PACKED) a.closed = take ? b.closed : a.closed;
}

// Composition over the stretches of a wave in processing order (DIR = 0: upwards, 1: downwards): `a` becomes the composition of
// everything in front of this lane's stretch, `total` that of the whole wave (in every lane).
template <int CG, int DIR, int VEC, int N, bool PACKED>
__device__ __forceinline__ void nf_wave_scan(NfAgg<VEC, N, PACKED>& a, NfAgg<VEC, N, PACKED>& total, int tg)
{
    typedef NfAgg<VEC, N, PACKED> Agg;
    constexpr int TG = 64 / CG;
    const int lane = threadIdx.x & 63;
    if constexpr (TG == 4) {
        // four rows of 16 lanes: the row exchanges of the vector unit (no trip through LDS).  Pairs of rows, then halves.
        auto lo16 = [](int v) { return (int)__builtin_amdgcn_permlane16_swap(v, v, false, false)[0]; };       // rows 0 0 2 2
        auto hi16 = [](int v) { return (int)__builtin_amdgcn_permlane16_swap(v, v, false, false)[1]; };       // rows 1 1 3 3
        auto lo32 = [](int v) { return (int)__builtin_amdgcn_permlane32_swap(v, v, false, false)[0]; };
        auto hi32 = [](int v) { return (int)__builtin_amdgcn_permlane32_swap(v, v, false, false)[1]; };
        const Agg even = nf_map(a, lo16), odd = nf_map(a, hi16);
        const Agg first = DIR ? odd : even;
        Agg pair = DIR ? even : odd;
        pair.after(first);
        const Agg low = nf_map(pair, lo32), high = nf_map(pair, hi32);
        const Agg half = DIR ? high : low;
        total = DIR ? low : high;
        total.after(half);
        a.one();
        nf_take(a, ((tg & 1) != 0) != (DIR != 0), first);       // the second row of a pair
        Agg e = a;
        e.after(half);
        nf_take(a, (tg >= 2) != (DIR != 0), e);                 // the second half
    } else {
        const int pos = DIR ? TG - 1 - tg : tg;
        auto from = [](int v, int l) { return __builtin_amdgcn_ds_bpermute(4 * l, v); };
#pragma unroll
        for (int s = 1; s < TG; s *= 2) {
            const int l = lane + (DIR ? s * CG : -s * CG);
            const Agg p = nf_map(a, [&](int v) { return from(v, l); });
            if (pos >= s) a.after(p);
        }
        const int last = (DIR ? 0 : TG - 1) * CG + lane % CG;
        total = nf_map(a, [&](int v) { return from(v, last); });
        const int l = lane + (DIR ? CG : -CG);
        a = nf_map(a, [&](int v) { return from(v, l); });
        Agg e;
        e.one();
        nf_take(a, pos == 0, e);
    }
}

// LDS exchange of the waves' totals
template <int VEC, int N, int CG, int NW, bool PACKED> struct NfScanLds {
    typedef NfAgg<VEC, N, PACKED> Agg;
    float P[NW][CG * N], H[NW][CG * VEC];
    int closed[NW];
    __device__ __forceinline__ void put(int w, int lane, const Agg& t)
    {
        if (lane < CG) {
#pragma unroll
            for (int k = 0; k < N; ++k) P[w][lane * N + k] = t.P[k];
#pragma unroll
            for (int k = 0; k < VEC; ++k) H[w][lane * VEC + k] = t.H[k];
            if (PACKED && lane == 0) closed[w] = t.closed;
        }
    }
    __device__ __forceinline__ Agg get(int w, int cg) const
    {
        Agg t;
#pragma unroll
        for (int k = 0; k < N; ++k) t.P[k] = P[w][cg * N + k];
#pragma unroll
        for (int k = 0; k < VEC; ++k) t.H[k] = H[w][cg * VEC + k];
        t.closed = PACKED ? closed[w] : 0;
        return t;
    }
};

// ---- the chain's exchange --------------------------------------------------------------------------
template <int VEC, int N, bool PACKED> __device__ __forceinline__ void nf_publish(unsigned long long* p, const NfAgg<VEC, N, PACKED>& t)
{
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        const float f = t.P[N == 1 ? 0 : k];
        const unsigned P = t.shut() ? NF_SCAN_CLOSED : f != f ? 0x7fc00000u : __float_as_uint(f);      // (a NaN never looks like a mark)
        __hip_atomic_store(p + k, (unsigned long long)__float_as_uint(t.H[k]) << 32 | P, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
template <int VEC, int N, bool PACKED> struct NfEntry {
    unsigned long long w[VEC];
    __device__ __forceinline__ void ask(const unsigned long long* p)
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[k] = __hip_atomic_load(p + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __device__ __forceinline__ bool missing() const
    {
        bool m = false;
#pragma unroll
        for (int k = 0; k < VEC; ++k) m |= w[k] == NF_SCAN_EMPTY;
        return m;
    }
    __device__ __forceinline__ NfAgg<VEC, N, PACKED> wait(const unsigned long long* p)
    {
        // Polls go past the caches to memory that every XCD shares, so one lane polls one word for all that wait, and they read again
        // when it is there (an entry's words are stored together: most often once).
        for (unsigned long long m = __ballot(missing()); m != 0; m = __ballot(missing())) {
            if ((int)(threadIdx.x & 63) == __ffsll((long long)m) - 1) {
                int k = 0;
#pragma unroll
                for (int i = VEC - 1; i > 0; --i)
                    if (w[i] == NF_SCAN_EMPTY) k = i;
                while (__hip_atomic_load(p + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == NF_SCAN_EMPTY) __builtin_amdgcn_s_sleep(6);
            }
            if (missing()) ask(p);
        }
        NfAgg<VEC, N, PACKED> t;
        t.closed = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) t.P[k] = __uint_as_float((unsigned)w[k]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) t.H[k] = __uint_as_float((unsigned)(w[k] >> 32));
        if (PACKED) t.closed = (unsigned)w[0] == NF_SCAN_CLOSED;
        return t;
    }
};

// Ordered composition over the lanes that are CG apart, in every lane.
template <int CG, int VEC, int N, bool PACKED> __device__ __forceinline__ void nf_wave_total(NfAgg<VEC, N, PACKED>& a)
{
    typedef NfAgg<VEC, N, PACKED> Agg;
#pragma unroll
    for (int s = CG; s < 64; s *= 2) {
        Agg lo = nf_map(a, [&](int v) { return __shfl_xor(v, s); }), hi = a;
        nf_take(hi, !(threadIdx.x & s), lo);
        nf_take(lo, !(threadIdx.x & s), a);
        hi.after(lo);
        a = hi;
    }
}

// What enters tile k of a chain, left in LDS.  Waves take 8 channel groups each, so that a lane has two entries to fetch at the
// most (fewer a wave: more waves that poll; 44 us against 46 for 65 536 steps x 256 channels, fp32):
// role 0: the tiles of k's group in front of it, and the publications that tile k owes; role 1: the groups of its set, and the set's state.
template <int VEC, int N, int CG, bool PACKED> struct NfChainLds {
    NfScanLds<VEC, N, CG, 2, PACKED> part;
    float set[CG * VEC];
};
template <int VEC, int CG> __device__ __forceinline__ unsigned long long* nf_chain_word(const NfScanArgs& a, unsigned long long* ws, int idx, int chain, int cg)
{
    return ws + ((long long)idx * (a.B * a.nblk) + chain) * (CG * VEC) + cg * VEC;
}
template <int VEC, int N, int CG, int NW, int DIR, bool PACKED>
__device__ __forceinline__ void nf_chain_collect(const NfScanArgs& a, int w, int k, int chain, const NfScanLds<VEC, N, CG, NW, PACKED>& waves,
                                                 NfChainLds<VEC, N, CG, PACKED>& lds)
{
    typedef NfAgg<VEC, N, PACKED> Agg;
    constexpr int CQ = CG <= 8 ? CG : 8, SUBS = CG / CQ, TQ = 64 / CQ, PER = (NF_SCAN_FAN - 1 + TQ - 1) / TQ;
    const int role = w / (NW / 2), sub = w % (NW / 2);
    if (sub >= SUBS) return;
    const int lane = threadIdx.x & 63, cg = sub * CQ + lane % CQ, tq = lane / CQ;
    const int grp = k / NF_SCAN_FAN, set = grp / NF_SCAN_FAN, nt = k % NF_SCAN_FAN, ng = grp % NF_SCAN_FAN;
    Agg own;
    if (role == 0 && tq == 0 && k + 1 < a.ntiles) {
        own = waves.get(DIR ? NW - 1 : 0, cg);
#pragma unroll
        for (int v = 1; v < NW; ++v) { Agg n = waves.get(DIR ? NW - 1 - v : v, cg); n.after(own); own = n; }
        nf_publish(nf_chain_word<VEC, CG>(a, a.ws_tile, k, chain, cg), own);
    }
    const int n = role == 0 ? nt : ng, first = role == 0 ? grp * NF_SCAN_FAN : set * NF_SCAN_FAN;
    unsigned long long* ws = role == 0 ? a.ws_tile : a.ws_group;
    NfEntry<VEC, N, PACKED> et[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (tq * PER + i < n) et[i].ask(nf_chain_word<VEC, CG>(a, ws, first + tq * PER + i, chain, cg));
    Agg t;
    t.one();
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (tq * PER + i < n) {
            Agg e = et[i].wait(nf_chain_word<VEC, CG>(a, ws, first + tq * PER + i, chain, cg));
            if (i > 0) e.after(t);
            t = e;
        }
    nf_wave_total<CQ>(t);
    if (tq == 0) {
        if (role == 0 && nt == NF_SCAN_FAN - 1 && k + 1 < a.ntiles) {
            own.after(t);
            nf_publish(nf_chain_word<VEC, CG>(a, a.ws_group, grp, chain, cg), own);
        }
        lds.part.put(role, cg, t);
        if (role == 1 && set > 0) {
            const unsigned long long* p = nf_chain_word<VEC, CG>(a, a.ws_set, set - 1, chain, cg);
            NfEntry<VEC, N, PACKED> e;
            e.ask(p);
            const Agg s = e.wait(p);
#pragma unroll
            for (int i = 0; i < VEC; ++i) lds.set[cg * VEC + i] = s.H[i];
        }
    }
}
// Behind a barrier: c becomes the state that enters tile k; a set's last tile publishes the state behind it.
template <int VEC, int N, int CG, int NW, int DIR, bool PACKED>
__device__ __forceinline__ void nf_chain_enter(const NfScanArgs& a, int k, int chain, int cg, bool publisher, const NfScanLds<VEC, N, CG, NW, PACKED>& waves,
                                               const NfChainLds<VEC, N, CG, PACKED>& lds, float (&c)[VEC])
{
    const int set = k / (NF_SCAN_FAN * NF_SCAN_FAN);
    if (set > 0)
#pragma unroll
        for (int i = 0; i < VEC; ++i) c[i] = lds.set[cg * VEC + i];
    lds.part.get(1, cg).apply(c);
    lds.part.get(0, cg).apply(c);
    if (publisher && (k + 1) % (NF_SCAN_FAN * NF_SCAN_FAN) == 0 && k + 1 < a.ntiles) {
        NfAgg<VEC, N, PACKED> s;
        s.one();
#pragma unroll
        for (int i = 0; i < VEC; ++i) s.H[i] = c[i];
        for (int v = 0; v < NW; ++v) waves.get(DIR ? NW - 1 - v : v, cg).apply(s.H);
        nf_publish(nf_chain_word<VEC, CG>(a, a.ws_set, set, chain, cg), s);
    }
}

// A wave's place: its chain, and for NF_SCAN_CHAIN the workgroup's tile by ticket.
struct NfPlace { int blk, b, k, w, chain; bool ok; };
template <int MODE> __device__ __forceinline__ NfPlace nf_place(const NfScanArgs& a)
{
    __shared__ int s_ticket;
    NfPlace p;
    const int nchains = a.B * a.nblk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (MODE == NF_SCAN_CHAIN) {
        p.chain = blockIdx.x % nchains;
        if (threadIdx.x == 0) s_ticket = __hip_atomic_fetch_add(a.ticket + p.chain * NF_SCAN_LINE, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        p.k = __builtin_amdgcn_readfirstlane(s_ticket);
        p.w = wave;
    } else if (MODE == NF_SCAN_WALK) {
        p.chain = blockIdx.x;
        p.k = 0;
        p.w = wave;
    } else {
        p.chain = a.chain0 + blockIdx.x * (NF_SCAN_WG / 64) + wave;
        p.k = p.w = 0;
    }
    p.ok = p.chain < nchains;
    p.blk = p.chain % a.nblk;
    p.b = p.chain / a.nblk;
    return p;
}

template <bool B> struct NfBool { static constexpr bool value = B; };

// Steps of a stretch that are not the tensor's (bit i).
template <int TPT> __device__ __forceinline__ unsigned nf_beyond(int j0, int T) { return j0 + TPT <= T ? 0u : j0 >= T ? ~0u : ~0u << (T - j0); }

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
template <typename E, int VEC, int CG, int TPT, int NW, int MODE, bool PACKED, bool SHARED>
__global__ void __launch_bounds__(MODE == NF_SCAN_WAVE ? NF_SCAN_WG : 64 * NW, MODE == NF_SCAN_CHAIN && sizeof(typename E::st) == 2 ? 4 : 1) k_scan_fwd(NfScanArgs a)
{
    constexpr int TG = 64 / CG, TS = NW * TG * TPT, ES = sizeof(typename E::st), N = SHARED ? 1 : VEC;
    typedef NfAgg<VEC, N, PACKED> Agg;
    constexpr bool CHAIN = MODE == NF_SCAN_CHAIN, WAVE = MODE == NF_SCAN_WAVE;
    __shared__ NfScanLds<VEC, N, CG, NW, PACKED> lds_[CHAIN ? 1 : 2];     // two for a walk: one barrier a tile is enough, a wave is at most one tile ahead
    __shared__ NfChainLds<VEC, N, CG, PACKED> s_chain;
    const NfPlace pl = nf_place<MODE>(a);
    if (!pl.ok) return;                                  // (whole chains by waves only: no barrier below)
    const int lane = threadIdx.x & 63, cg = lane % CG, tg = lane / CG, w = pl.w, b = pl.b;
    const int ch = (pl.blk * CG + cg) * VEC;
    const bool live = ch < a.D;
    const int chl = live ? ch : 0;
    const int T = a.T, rev = a.reverse;
    const bool past = CG * VEC * ES >= 128 && a.past;
    const int gs = (ES == 4 || a.gate32) ? 4 : 2, hstep = a.D * ES;
    const char* gbase = (const char*)a.gate + b * a.gate_sb;
    const char* xbase = (const char*)a.x + b * a.x_sb;
    char* hbase = (char*)a.h + (long long)b * T * hstep;
    const unsigned goff = SHARED ? 0u : (unsigned)(chl * gs), xoff = (unsigned)(chl * ES);
    const int jl = (w * TG + tg) * TPT;
    float c[VEC];                        // the state that enters the tile
#pragma unroll
    for (int k = 0; k < VEC; ++k) c[k] = 0.f;
    if (a.h0 && !PACKED)
#pragma unroll
        for (int k = 0; k < VEC; ++k) c[k] = a.h0[(long long)b * a.D + chl + k];
    auto initial = [&](int j, float (&s)[VEC]) {         // the state in front of step j, the first of its sequence
        const int q = a.sid[rev ? T - 1 - j : j];
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[k] = a.h0 ? a.h0[(long long)q * a.D + chl + k] : 0.f;
    };
    for (int tile = pl.k; tile < (CHAIN ? pl.k + 1 : a.ntiles); ++tile) {
        const NfRows<TS> rows(tile, T, rev);
        const long long row0 = rows.first(tile, T);
        NfStretch<E, VEC, TPT> x;
        NfGateStretch<E, VEC, TPT, SHARED> gt;
        gt.load(a, gbase + row0 * a.gate_st, goff, jl, rows);
        x.load(xbase + row0 * a.x_st, xoff, a.x_st, jl, rows);
        const int j0 = tile * TS + jl;
        const bool edge = tile == a.ntiles - 1;          // (uniform) the last tile: steps that do not exist, the final state
        NfMarks m = {0u, 0u, 0u};
        if (PACKED) m = nf_scan_marks<TPT>(a.sid, j0, T, rev);
        const bool plain = PACKED ? !__any(m.start | m.end | m.none) : !edge;      // (uniform) a wave whose steps are all inside one sequence
        float A[TPT][N];
        gt.get(a, A);
        if (!plain) {
            const unsigned idle = m.none | nf_beyond<TPT>(j0, T);
            x.clear(idle);
#pragma unroll
            for (int i = 0; i < TPT; ++i)
                if (idle >> i & 1u)
#pragma unroll
                    for (int k = 0; k < N; ++k) A[i][k] = 1.f;
        }
        Agg me, tot;
        me.one();
        if (PACKED && m.start) {
            me.closed = 1;
#pragma unroll
            for (int i = 0; i < TPT; ++i) {
                if (m.start >> i & 1u) initial(j0 + i, me.H);
#pragma unroll
                for (int k = 0; k < VEC; ++k) me.H[k] = fmaf(A[i][N == 1 ? 0 : k], me.H[k], x.at(i, k));
            }
        } else {
#pragma unroll
            for (int i = 0; i < TPT; ++i) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) me.H[k] = fmaf(A[i][N == 1 ? 0 : k], me.H[k], x.at(i, k));
#pragma unroll
                for (int k = 0; k < N; ++k) me.P[k] = i == 0 ? A[i][k] : nf_gates(me.P[k], A[i][k]);
            }
        }
        nf_wave_scan<CG, 0>(me, tot, tg);
        float s[VEC];
        auto& lds = lds_[CHAIN ? 0 : tile & 1];
        if constexpr (!WAVE) {
            lds.put(w, lane, tot);
            __syncthreads();
        }
        if constexpr (CHAIN) {
            nf_chain_collect<VEC, N, CG, NW, 0, PACKED>(a, w, tile, pl.chain, lds, s_chain);
            __syncthreads();
            nf_chain_enter<VEC, N, CG, NW, 0, PACKED>(a, tile, pl.chain, cg, w == 0 && tg == 0, lds, s_chain, c);
        }
        if (a.states && w == 0 && tg == 0 && live)
#pragma unroll
            for (int k = 0; k < VEC; ++k) a.states[((long long)b * a.ntiles + tile) * a.D + ch + k] = c[k];
        if constexpr (!WAVE) {
#pragma unroll
            for (int v = 0; v < NW; ++v) {
                if (v == w)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) s[k] = c[k];
                if (!CHAIN || v < w) lds.get(v, cg).apply(c);
            }
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) s[k] = c[k];
            tot.apply(c);
        }
        me.apply(s);
        char* hb = hbase + row0 * hstep;
        unsigned ho = rows.at(jl) * (unsigned)hstep + xoff;
        const int hs = rev ? -hstep : hstep;
        if (plain) {
            if (live) {
#pragma unroll
                for (int i = 0; i < TPT; ++i) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) s[k] = fmaf(A[i][N == 1 ? 0 : k], s[k], x.at(i, k));
                    nf_put<E, VEC>(hb + ho, s, past);
                    ho += hs;
                }
            }
        } else if (live) {
#pragma unroll
            for (int i = 0; i < TPT; ++i) {
                if (PACKED && (m.start >> i & 1u)) initial(j0 + i, s);
#pragma unroll
                for (int k = 0; k < VEC; ++k) s[k] = fmaf(A[i][N == 1 ? 0 : k], s[k], x.at(i, k));
                if (j0 + i < T) {
                    if (PACKED && (m.none >> i & 1u)) { const float z[VEC] = {}; nf_put<E, VEC>(hb + ho, z, past); }
                    else nf_put<E, VEC>(hb + ho, s, past);
                    if (PACKED ? m.end >> i & 1u : j0 + i == T - 1) {        // the final state is the last step's, to the bit
                        const int q = PACKED ? a.sid[rev ? T - 1 - (j0 + i) : j0 + i] : b;
#pragma unroll
                        for (int k = 0; k < VEC; ++k) a.h_last[(long long)q * a.D + ch + k] = s[k];
                    }
                }
                ho += hs;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
template <typename E, int VEC, int CG, int TPT, int NW, int MODE, bool PACKED, bool SHARED>
__global__ void __launch_bounds__(MODE == NF_SCAN_WAVE ? NF_SCAN_WG : 64 * NW) k_scan_bwd(NfScanArgs a)
{
    constexpr int TG = 64 / CG, TS = NW * TG * TPT, ES = sizeof(typename E::st), N = SHARED ? 1 : VEC;
    typedef NfAgg<VEC, N, PACKED> Agg;
    constexpr bool CHAIN = MODE == NF_SCAN_CHAIN, WAVE = MODE == NF_SCAN_WAVE;
    __shared__ NfScanLds<VEC, N, CG, NW, PACKED> lds_f_[CHAIN ? 1 : 2], lds_r_[CHAIN ? 1 : 2];
    __shared__ NfChainLds<VEC, N, CG, PACKED> s_chain;
    const NfPlace pl = nf_place<MODE>(a);
    if (!pl.ok) return;
    const int lane = threadIdx.x & 63, cg = lane % CG, tg = lane / CG, w = pl.w, b = pl.b;
    const int ch = (pl.blk * CG + cg) * VEC;
    const bool live = ch < a.D;
    const int chl = live ? ch : 0;
    const int T = a.T, rev = a.reverse;
    const bool past = CG * VEC * ES >= 128 && a.past;
    const int gs = (ES == 4 || a.gate32) ? 4 : 2, hstep = a.D * ES, gstep = a.D * gs;
    const char* gbase = (const char*)a.gate + b * a.gate_sb;
    const char* xbase = (const char*)a.x + b * a.x_sb;
    const char* ybase = a.g ? (const char*)a.g + b * a.g_sb : nullptr;
    const unsigned goff = SHARED ? 0u : (unsigned)(chl * gs), xoff = (unsigned)(chl * ES);
    const int jl = (w * TG + tg) * TPT;
    float u[VEC];                        // the gradient that enters the tile from behind
#pragma unroll
    for (int k = 0; k < VEC; ++k) u[k] = 0.f;
    if (a.g_last && !PACKED)
#pragma unroll
        for (int k = 0; k < VEC; ++k) u[k] = a.g_last[(long long)b * a.D + chl + k];
    auto of_sequence = [&](const float* p, int j, float (&s)[VEC]) {         // the row of p that belongs to step j's sequence, or zeros
        const int q = a.sid[rev ? T - 1 - j : j];
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[k] = p ? p[(long long)q * a.D + chl + k] : 0.f;
    };
    for (int it = pl.k; it < (CHAIN ? pl.k + 1 : a.ntiles); ++it) {
        const int tile = a.ntiles - 1 - it;
        const NfRows<TS> rows(tile, T, rev);
        const long long row0 = rows.first(tile, T);
        NfStretch<E, VEC, TPT> x, y;
        NfGateStretch<E, VEC, TPT, SHARED> gt;
        gt.load(a, gbase + row0 * a.gate_st, goff, jl, rows);
        if (ybase) y.load(ybase + row0 * a.g_st, xoff, a.g_st, jl, rows);
        else y.clear(~0u);
        x.load(xbase + row0 * a.x_st, xoff, a.x_st, jl, rows);
        float c[VEC];                    // the state that enters the tile in front
#pragma unroll
        for (int k = 0; k < VEC; ++k) c[k] = a.states[((long long)b * a.ntiles + tile) * a.D + chl + k];
        const int j0 = tile * TS + jl;
        NfMarks m = {0u, 0u, 0u};
        if (PACKED) m = nf_scan_marks<TPT>(a.sid, j0, T, rev);
        const bool plain = PACKED ? !__any(m.start | m.end | m.none) : it != 0;    // (uniform) a wave whose steps are all inside one sequence
        float A[TPT][N];
        gt.get(a, A);
        if (!plain) {
            const unsigned idle = m.none | nf_beyond<TPT>(j0, T);
            x.clear(idle);
            y.clear(idle);
#pragma unroll
            for (int i = 0; i < TPT; ++i)
                if (idle >> i & 1u)
#pragma unroll
                    for (int k = 0; k < N; ++k) A[i][k] = 1.f;
        }
        Agg rv, rtot, fw, ftot;
        auto reduce = [&](auto marked) {
            constexpr bool MARKED = decltype(marked)::value;
            // backwards: the stretch as u -> P u + H (what enters the last step of a sequence is the gradient of its final state)
            rv.one();
            if (MARKED) rv.closed = m.end != 0u;
#pragma unroll
            for (int i = TPT - 1; i >= 0; --i) {
                if (MARKED && (m.end >> i & 1u)) of_sequence(a.g_last, j0 + i, rv.H);
#pragma unroll
                for (int k = 0; k < VEC; ++k) rv.H[k] = A[i][N == 1 ? 0 : k] * (rv.H[k] + y.at(i, k));
#pragma unroll
                for (int k = 0; k < N; ++k) rv.P[k] = i == TPT - 1 ? A[i][k] : nf_gates(rv.P[k], A[i][k]);
            }
            // forwards: the stretch as c -> P c + H, started anew where a sequence begins
            fw.one();
            if (MARKED) fw.closed = m.start != 0u;
#pragma unroll
            for (int k = 0; k < N; ++k) fw.P[k] = rv.P[k];
#pragma unroll
            for (int i = 0; i < TPT; ++i) {
                if (MARKED && (m.start >> i & 1u)) of_sequence(a.h0, j0 + i, fw.H);
#pragma unroll
                for (int k = 0; k < VEC; ++k) fw.H[k] = fmaf(A[i][N == 1 ? 0 : k], fw.H[k], x.at(i, k));
            }
        };
        if (PACKED && !plain) reduce(NfBool<true>());
        else reduce(NfBool<false>());
        nf_wave_scan<CG, 1>(rv, rtot, tg);
        nf_wave_scan<CG, 0>(fw, ftot, tg);
        float su[VEC];
        auto& lds_r = lds_r_[CHAIN ? 0 : it & 1];
        auto& lds_f = lds_f_[CHAIN ? 0 : it & 1];
        if constexpr (!WAVE) {
            lds_r.put(w, lane, rtot);
            lds_f.put(w, lane, ftot);
            __syncthreads();
        }
        if constexpr (CHAIN) {
            nf_chain_collect<VEC, N, CG, NW, 1, PACKED>(a, w, it, pl.chain, lds_r, s_chain);
            __syncthreads();
            nf_chain_enter<VEC, N, CG, NW, 1, PACKED>(a, it, pl.chain, cg, w == 0 && tg == 0, lds_r, s_chain, u);
        }
        if constexpr (!WAVE) {
#pragma unroll
            for (int v = 0; v < NW - 1; ++v)
                if (v < w) lds_f.get(v, cg).apply(c);
#pragma unroll
            for (int v = NW - 1; v >= 0; --v) {
                if (v == w)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) su[k] = u[k];
                if (!CHAIN || v > w) lds_r.get(v, cg).apply(u);
            }
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) su[k] = u[k];
            rtot.apply(u);
        }
        fw.apply(c);
        rv.apply(su);
        const long long orow = (long long)b * T + row0;
        float dsum[TPT];
        auto finish = [&](auto exact) {
            constexpr bool PLAIN = decltype(exact)::value, MARKED = PACKED && !PLAIN;
            // the states in front of every step, then the gradients from the last step to the first
            float hb[TPT][VEC];
#pragma unroll
            for (int i = 0; i < TPT; ++i) {
                if (MARKED && (m.start >> i & 1u)) of_sequence(a.h0, j0 + i, c);
#pragma unroll
                for (int k = 0; k < VEC; ++k) { hb[i][k] = c[k]; c[k] = fmaf(A[i][N == 1 ? 0 : k], c[k], x.at(i, k)); }
            }
            char* xq = (char*)a.dx + orow * hstep;
            char* gq = (char*)a.dgate + orow * gstep;
            unsigned xo = rows.at(jl + TPT - 1) * (unsigned)hstep + xoff, go = rows.at(jl + TPT - 1) * (unsigned)gstep + goff;
#pragma unroll
            for (int i = TPT - 1; i >= 0; --i) {
                float dx[VEC], dg[VEC];
                if (MARKED && (m.end >> i & 1u)) of_sequence(a.g_last, j0 + i, su);
                dsum[i] = 0.f;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    dx[k] = su[k] + y.at(i, k);
                    su[k] = A[i][N == 1 ? 0 : k] * dx[k];
                    dg[k] = (a.log_gate ? su[k] : dx[k]) * hb[i][k];
                }
                if (MARKED && (m.none >> i & 1u))
#pragma unroll
                    for (int k = 0; k < VEC; ++k) dx[k] = dg[k] = 0.f;
                if (live && (PLAIN || j0 + i < T)) {
                    if (SHARED)
#pragma unroll
                        for (int k = 0; k < VEC; ++k) dsum[i] += dg[k];
                    if (a.dx) nf_put<E, VEC>(xq + xo, dx, past);
                    if (!SHARED && a.dgate) {
                        if (ES == 4 || a.gate32) nf_put<NfF32, VEC>(gq + go, dg, past);
                        else nf_put<E, VEC>(gq + go, dg, past);
                    }
                    if (MARKED && (m.start >> i & 1u) && a.dh0) {
                        const int q = a.sid[rev ? T - 1 - (j0 + i) : j0 + i];
#pragma unroll
                        for (int k = 0; k < VEC; ++k) a.dh0[(long long)q * a.D + ch + k] = su[k];
                    }
                }
                xo -= rev ? -hstep : hstep;
                go -= rev ? -gstep : gstep;
            }
        };
        if (plain) finish(NfBool<true>());
        else finish(NfBool<false>());
        if (SHARED && a.dgate) {
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
            constexpr int NS = CG >= TPT ? 1 : TPT / CG, REST = CG >= TPT ? CG / TPT : 1;
            if (cg % REST == 0) {
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (j0 + first + i < T) {
                        const long long o = orow + rows.at(jl + first + i);
                        if (a.nblk > 1) a.dgate_part[(long long)pl.blk * a.B * T + o] = dsum[i];
                        else if (ES == 4 || a.gate32) ((float*)a.dgate)[o] = dsum[i];
                        else ((typename E::st*)a.dgate)[o] = E::pk(dsum[i]);
                    }
            }
        }
        // the tile's first stretch ends with dh0
        if (!PACKED && it == a.ntiles - 1 && a.dh0 && w == 0 && tg == 0 && live)
#pragma unroll
            for (int k = 0; k < VEC; ++k) a.dh0[(long long)b * a.D + ch + k] = su[k];
    }
}

// Steps a thread and waves a tile: 16 values of a tensor a thread for a wave on its own, else 32 on eight waves (fewer tiles, half the exchange a
// step: 65 536 steps x 256 channels, fp32, chained forward 46 us against 76; fp16 41 against 63).
#define NF_SCAN_TPT(vec, mode) (((vec) == 4 ? 4 : 8) * ((mode) == NF_SCAN_WAVE ? 1 : 2))
#define NF_SCAN_NW(mode) ((mode) == NF_SCAN_WAVE ? 1 : 8)
// (a launch has fewer than 2^32 threads: more chains than NF_SCAN_SLICE by waves take several launches, the other modes are refused)
#define NF_SCAN_SLICE (1 << 25)
#define NF_SCAN_MAX_TILES ((1 << 23) - 1)
template <typename E> int nf_scan_launch(const NfScanArgs& a, int vec, int cg, int mode, int backward, hipStream_t st)
{
    const long long all = (long long)a.B * a.nblk, chains = mode == NF_SCAN_WAVE && all - a.chain0 > NF_SCAN_SLICE ? NF_SCAN_SLICE : all - a.chain0;
    const dim3 grid((unsigned)(mode == NF_SCAN_WAVE ? (chains + NF_SCAN_WG / 64 - 1) / (NF_SCAN_WG / 64) : mode == NF_SCAN_WALK ? chains : chains * a.ntiles));
    const int packed = a.sid != nullptr;
#define NF_SCAN_GO(V, C, M, PK, SH)                                                                                                                          \
    if (vec == V && cg == C && mode == M && packed == PK && a.shared == SH) {                                                                               \
        constexpr int NW = NF_SCAN_NW(M), TH = M == NF_SCAN_WAVE ? NF_SCAN_WG : 64 * NW, TPT = NF_SCAN_TPT(V, M);                                             \
        if (backward) hipLaunchKernelGGL((k_scan_bwd<E, V, C, TPT, NW, M, PK, SH>), grid, dim3(TH), 0, st, a);                                               \
        else hipLaunchKernelGGL((k_scan_fwd<E, V, C, TPT, NW, M, PK, SH>), grid, dim3(TH), 0, st, a);                                                        \
        return 1;                                                                                                                                           \
    }
#define NF_SCAN_GO_S(V, C, SH) NF_SCAN_GO(V, C, NF_SCAN_WAVE, false, SH) NF_SCAN_GO(V, C, NF_SCAN_WALK, false, SH) NF_SCAN_GO(V, C, NF_SCAN_CHAIN, false, SH) NF_SCAN_GO(V, C, NF_SCAN_CHAIN, true, SH)
#define NF_SCAN_GO_C(V, C) NF_SCAN_GO_S(V, C, false) NF_SCAN_GO_S(V, C, true)
    NF_SCAN_GO_C(4, 16) NF_SCAN_GO_C(4, 8) NF_SCAN_GO_C(4, 4) NF_SCAN_GO_C(4, 1)
    NF_SCAN_GO_C(2, 32) NF_SCAN_GO_C(2, 8) NF_SCAN_GO_C(2, 2)
    NF_SCAN_GO_C(1, 32) NF_SCAN_GO_C(1, 8) NF_SCAN_GO_C(1, 2)
#undef NF_SCAN_GO_C
#undef NF_SCAN_GO_S
#undef NF_SCAN_GO
    return 0;
}
int nf_scan_launch_f32(const NfScanArgs& a, int vec, int cg, int mode, int backward, hipStream_t st);
int nf_scan_launch_bf16(const NfScanArgs& a, int vec, int cg, int mode, int backward, hipStream_t st);
int nf_scan_launch_f16(const NfScanArgs& a, int vec, int cg, int mode, int backward, hipStream_t st);
