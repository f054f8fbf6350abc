// nf_scan.hip — entry points of the gated linear recurrence (kernels: nf_scan.h).
#include "nf_scan.h"
#include <math.h>

static int scan_tile(const nf_scan_t* s) { return NF_SCAN_NW(s->mode) * (64 / s->cg) * NF_SCAN_TPT(s->vec, s->mode); }
static long long scan_blocks(const nf_scan_t* s) { return (s->D + s->cg * s->vec - 1) / (s->cg * s->vec); }

static int scan_check(const nf_scan_t* s, const char* who)
{
    if (!s) { nf_set_error("%s: null descriptor", who); return NF_EINVAL; }
    if (s->dtype < 0 || s->dtype > 2) { nf_set_error("%s: dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)", who); return NF_EINVAL; }
    if (s->B < 0 || s->T < 0 || s->D < 1 || s->T > NF_SCAN_MAX_STEPS || s->D > NF_SCAN_MAX_CHANNELS) { nf_set_error("%s: bad sizes", who); return NF_EINVAL; }
    if (s->row_splits && (s->B != 1 || s->n_seq < 0)) { nf_set_error("%s: packed rows come as one batch", who); return NF_EINVAL; }
    return NF_OK;
}

static bool scan_plan_ok(const nf_scan_t* s)
{
    const bool lanes = s->vec == 4 ? (s->cg == 16 || s->cg == 8 || s->cg == 4 || s->cg == 1) : ((s->vec == 2 || s->vec == 1) && (s->cg == 32 || s->cg == 8 || s->cg == 2));
    return lanes && s->mode >= 0 && s->mode <= 2 && (s->mode == NF_SCAN_CHAIN || !s->row_splits) && s->D % s->vec == 0;
}

// elements that every row which (base, strides) reaches can be read at a time: 4, 2 or 1
static int scan_vec(const void* p, int64_t sb, int64_t st, int size)
{
    int v = 4;
    while (v > 1 && ((uintptr_t)p % (v * size) || sb % v || st % v)) v /= 2;
    return v;
}

// Figures: forward / backward, us, as timed with this plan and with others forced.
// Lanes: as many channels a block as D has, a cache line's 64 of 16 bits or 32 of 32 bits at the most (65 536 steps x 256 channels, fp32:
// 47 / 69 with 32, 58 / 77 with 64; fp16 46 / 65 with 64, 45 / 69 with 32).  Fewer channels, 40 000 x 192 fp32, one gate a step: four channels a lane,
// D = 4 65 / 94 with one lane (four 77 / 107, eight 117 / 193), 16 199 / 288 with four (eight 219 / 304, one 283 / 448).  One or two channels a
// lane (rows that are not aligned for more), lanes across: D = 1 42 / 58 with two (eight 43 / 85, 32 130 / 315), 3 52 / 105 with eight (two 101 / 196,
// 32 126 / 359); 32 of them pay from many channels on: D = 34 (two a lane) 532 / 746 against 669 / 904 with eight, but 18 374 / 589 against
// 320 / 443 and 9 (one a lane) 240 / 429 against 230 / 307: between 8 and 16 groups eight lanes would be the better choice.
// Modes: thousands of chains, or chains of few steps, take a wave each; from 8 192 channels on a workgroup each (2048 steps, bf16: 16 384
// channels 40 / 72 against 47 / 87 chained and 176 / 291 by waves, 8 192 32 / 53 against 33 / 54; 4 096 channels and 4096 steps 51 / 90 against
// 36 / 55); fewer ones are chained.  From 4 096 chains on by waves: 4 096 x 192 x 32 fp32 35 / 50 against 41 / 100 by workgroups, though
// 4 096 x 1024 x 32 226 / 344 against 204 / 312.  Chains of one or two tiles gain nothing from being chained, and a tile that they do not
// fill costs more than waves: 64 x 400 x 64 fp32 14 / 17 against 8 / 12 by workgroups, 700 x 192 x 32 13 / 25 by workgroups against 12 / 18
// by waves, 2000 x 600 x 1 27 / 41 against 12 / 16.
extern "C" int nf_scan_plan(nf_scan_t* s, size_t* state_floats)
{
    const int rc = scan_check(s, __func__);
    if (rc) return rc;
    const int es = s->dtype == 0 ? 4 : 2, gs = (s->dtype == 0 || s->gate32) ? 4 : 2;
    int v = scan_vec(s->x, s->x_sb, s->x_st, es);
    if (!s->shared) { const int vg = scan_vec(s->gate, s->gate_sb, s->gate_st, gs); v = vg < v ? vg : v; }
    while (s->D % v) v /= 2;
    s->vec = v;
    if (v == 4) s->cg = s->D <= 4 ? 1 : s->D <= 16 ? 4 : s->D <= 32 || s->dtype == 0 ? 8 : 16;
    else s->cg = s->D <= 2 * v ? 2 : s->D <= 8 * v ? 8 : 32;
    const long long chains = (long long)s->B * scan_blocks(s);
    s->mode = NF_SCAN_WAVE;
    if (s->row_splits) s->mode = NF_SCAN_CHAIN;
    else if (chains < 4096 && s->T > 2 * scan_tile(s)) s->mode = chains * s->cg * s->vec >= 8192 ? NF_SCAN_WALK : NF_SCAN_CHAIN;
    const int tile = scan_tile(s);
    if (state_floats) *state_floats = (size_t)s->B * ((s->T + tile - 1) / tile) * s->D;
    return NF_OK;
}

// workspace, in 8-byte words: [tile | group | set entries | counters] of the chained kernels, then the per-block sums of a shared gate's gradient
struct ScanWs {
    size_t tile, group, set, counters, part;
    size_t entries() const { return tile + group + set; }
    size_t words() const { return entries() + counters + (part + 1) / 2; }
};
static ScanWs scan_workspace(const nf_scan_t* s, int backward)
{
    ScanWs w = {0, 0, 0, 0, 0};
    if (s->mode == NF_SCAN_CHAIN) {
        const int tile = scan_tile(s);
        const size_t per = (size_t)s->B * scan_blocks(s) * s->cg * s->vec, nt = (s->T + tile - 1) / tile;
        w.tile = nt * per;
        w.group = (nt + NF_SCAN_FAN - 1) / NF_SCAN_FAN * per;
        w.set = (nt + NF_SCAN_FAN * NF_SCAN_FAN - 1) / (NF_SCAN_FAN * NF_SCAN_FAN) * per;
        w.counters = (size_t)s->B * scan_blocks(s) * NF_SCAN_LINE / 2;
    }
    if (backward && s->shared && s->dgate && scan_blocks(s) > 1) w.part = (size_t)scan_blocks(s) * s->B * s->T;
    return w;
}

extern "C" size_t nf_scan_workspace_bytes(const nf_scan_t* s, int backward)
{
    if (scan_check(s, __func__) || !scan_plan_ok(s)) return 0;
    return 8 * scan_workspace(s, backward).words();
}

// What has to be there before the tiles run, in one launch (any part may be absent; as three launches: 164 us for
// 50 001 packed rows of 200 channels with gradients instead of 157).
//  - The sequence of every packed row (-1: before the first or behind the last), by bisection of the splits.
//  - The final states of empty sequences are their initial ones (and their gradients pass through).  Splits are clamped to [0, T], so that bad ones
//    give bad numbers but no access out of range.
//  - The chain's entries are set to "empty", the counters of tiles to 0 (by a kernel: a memset node in a captured graph has given wrong results).
struct NfFront {
    const int64_t* rs; int n_seq, T, D;
    int* sid;                                            // rows, or NULL
    const float* src; float* dst;                        // empty sequences: from src (NULL: zeros), or dst NULL
    unsigned long long* words; size_t entries, n;        // the workspace's
};
__global__ void __launch_bounds__(256) k_scan_front(NfFront a)
{
    const size_t first = (size_t)blockIdx.x * 256 + threadIdx.x, step = (size_t)gridDim.x * 256;
    for (size_t i = first; i < a.n; i += step) a.words[i] = i < a.entries ? NF_SCAN_EMPTY : 0ull;
    if (a.sid)
        for (size_t r = first; r < (size_t)a.T; r += step) {
            int lo = 0, hi = a.n_seq;            // the number of k in [1, n_seq] with rs[k] <= r
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (a.rs[mid + 1] <= (int64_t)r) lo = mid + 1;
                else hi = mid;
            }
            a.sid[r] = (lo < a.n_seq && a.rs[lo] <= (int64_t)r) ? lo : -1;
        }
    if (a.dst)
        for (size_t e = first; e < (size_t)a.n_seq * a.D; e += step) {
            const int s = (int)(e / a.D);
            const int64_t b0 = min(max(a.rs[s], (int64_t)0), (int64_t)a.T), b1 = min(max(a.rs[s + 1], (int64_t)0), (int64_t)a.T);
            if (b0 >= b1) a.dst[e] = a.src ? a.src[e] : 0.f;
        }
}
static int scan_front(const NfFront& f, hipStream_t st)
{
    size_t n = f.n;
    if (f.sid && (size_t)f.T > n) n = f.T;
    if (f.dst && (size_t)f.n_seq * f.D > n) n = (size_t)f.n_seq * f.D;
    if (n == 0) return NF_OK;
    const size_t blocks = (n + 255) / 256;
    hipLaunchKernelGGL(k_scan_front, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, f);
    NF_CHECK_LAUNCH();
    return NF_OK;
}

__global__ void __launch_bounds__(256) k_scan_fold(const float* __restrict__ part, int nblk, long long n, int type, void* __restrict__ out)
{
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    for (int b = 0; b < nblk; ++b) s += part[b * n + i];
    if (type == 0) ((float*)out)[i] = s;
    else if (type == 1) ((unsigned short*)out)[i] = NfBf16::pk(s);
    else ((unsigned short*)out)[i] = NfF16::pk(s);
}

static int scan_go(const nf_scan_t* s, const NfScanArgs& a, int backward, hipStream_t st)
{
    if (s->dtype == 0) return nf_scan_launch_f32(a, s->vec, s->cg, s->mode, backward, st);
    if (s->dtype == 1) return nf_scan_launch_bf16(a, s->vec, s->cg, s->mode, backward, st);
    return nf_scan_launch_f16(a, s->vec, s->cg, s->mode, backward, st);
}

static int scan_run(const nf_scan_t* s, int backward, hipStream_t st, const char* who)
{
    const int rc = scan_check(s, who);
    if (rc) return rc;
    if (!scan_plan_ok(s)) { nf_set_error("%s: no plan (nf_scan_plan)", who); return NF_EINVAL; }
    const bool packed = s->row_splits != nullptr;
    const int n_state = packed ? s->n_seq : s->B;
    const float* init = backward ? s->g_last : s->h0;
    float* fin = backward ? s->dh0 : s->h_last;
    if (!backward && !fin && n_state > 0) { nf_set_error("%s: null h_last", who); return NF_EINVAL; }
    NfFront front = {};
    if (packed) {
        front.rs = s->row_splits; front.n_seq = s->n_seq; front.T = s->T; front.D = s->D;
        front.src = init; front.dst = fin;
    }
    if (s->B == 0 || s->T == 0) return scan_front(front, st);        // (dense with T = 0: the caller copies the state)
    if (!s->gate || !s->x || (backward ? !s->states : !s->h)) { nf_set_error("%s: null pointer", who); return NF_EINVAL; }
    if (packed && !s->sid) { nf_set_error("%s: packed rows need the row buffer (sid)", who); return NF_EINVAL; }
    const int es = s->dtype == 0 ? 4 : 2, gs = (s->dtype == 0 || s->gate32) ? 4 : 2;
    if (scan_vec(s->x, s->x_sb, s->x_st, es) < s->vec || (!s->shared && scan_vec(s->gate, s->gate_sb, s->gate_st, gs) < s->vec) ||
        (backward && s->g && scan_vec(s->g, s->g_sb, s->g_st, es) < s->vec) || (!backward && (uintptr_t)s->h % (s->vec * es)) ||
        (backward && ((uintptr_t)s->dx % (s->vec * es) || (!s->shared && (uintptr_t)s->dgate % (s->vec * gs))))) {
        nf_set_error("%s: the plan reads %d elements at a time, a tensor is not aligned for it", who, s->vec);
        return NF_EINVAL;
    }
    NfScanArgs a = {};
    a.gate = s->gate; a.x = s->x; a.g = s->g; a.h0 = s->h0; a.g_last = s->g_last; a.h = s->h; a.h_last = s->h_last; a.states = s->states;
    a.dgate = s->dgate; a.dx = s->dx; a.dh0 = s->dh0; a.sid = packed ? s->sid : nullptr;
    const int tile = scan_tile(s);
    const int64_t far = 0xffffffffll / tile / 4;         // (a tile's rows: unsigned 32-bit offsets)
    const int64_t gate_st = s->T > 1 ? s->gate_st : 0, x_st = s->T > 1 ? s->x_st : 0, g_st = s->T > 1 ? s->g_st : 0;
    if (gate_st < 0 || x_st < 0 || g_st < 0 || gate_st > far || x_st > far || g_st > far ||
        (s->T > 1 && s->D > far)) {
        nf_set_error("%s: steps of a tensor lie too far apart (copy it)", who);
        return NF_EINVAL;
    }
    a.gate_sb = s->gate_sb * gs; a.x_sb = s->x_sb * es; a.g_sb = s->g_sb * es;
    a.gate_st = (int)(gate_st * gs); a.x_st = (int)(x_st * es); a.g_st = (int)(g_st * es);
    a.B = s->B; a.T = s->T; a.D = s->D;
    a.nblk = (int)scan_blocks(s);
    a.ntiles = (s->T + tile - 1) / tile;
    a.gate32 = s->gate32 != 0; a.shared = s->shared != 0; a.log_gate = s->log_gate != 0; a.reverse = s->reverse != 0;
    // From 64 MB a tensor on (a quarter of the last-level cache) what is written would only push out what is still to be read: 8 x 2048 x 2048
    // bf16 forward 51 us against 62, 4096 x 192 x 32 fp32 backward 48 against 53.  Below, the caller finds h there.
    a.past = (long long)s->B * s->T * s->D * es >= 64ll << 20;
    const long long chains = (long long)a.B * a.nblk;
    if (chains > 0x7ffffff0LL || (s->mode != NF_SCAN_WAVE && chains * (s->mode == NF_SCAN_CHAIN ? a.ntiles : 1) > NF_SCAN_MAX_TILES)) { nf_set_error("%s: too many chains", who); return NF_EINVAL; }
    const ScanWs ws = scan_workspace(s, backward);
    const size_t n_part = ws.part;
    if (s->workspace_bytes < 8 * ws.words() || (ws.words() && (!s->workspace || (uintptr_t)s->workspace % 8))) {
        nf_set_error("%s: workspace too small or unaligned (nf_scan_workspace_bytes)", who);
        return NF_EINVAL;
    }
    unsigned long long* words = (unsigned long long*)s->workspace;
    a.ws_tile = words; a.ws_group = words + ws.tile; a.ws_set = a.ws_group + ws.group; a.ticket = (int*)(words + ws.entries());
    a.dgate_part = n_part ? (float*)(words + ws.entries() + ws.counters) : nullptr;
    if (packed && !backward) front.sid = s->sid;
    front.words = words; front.entries = ws.entries(); front.n = ws.entries() + ws.counters;
    const int rf = scan_front(front, st);
    if (rf) return rf;
    for (long long c = 0; c < chains; c += s->mode == NF_SCAN_WAVE ? NF_SCAN_SLICE : chains) {
        a.chain0 = (int)c;
        if (!scan_go(s, a, backward, st)) { nf_set_error("%s: no kernel for the plan", who); return NF_EINVAL; }
        NF_CHECK_LAUNCH();
    }
    if (n_part) {
        const long long n = (long long)s->B * s->T;
        hipLaunchKernelGGL(k_scan_fold, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (const float*)a.dgate_part, a.nblk, n,
                           a.gate32 ? 0 : s->dtype, s->dgate);
        NF_CHECK_LAUNCH();
    }
    return NF_OK;
}

extern "C" int nf_scan_fwd(const nf_scan_t* s, nf_stream_t stream) { return scan_run(s, 0, (hipStream_t)stream, __func__); }
extern "C" int nf_scan_bwd(const nf_scan_t* s, nf_stream_t stream) { return scan_run(s, 1, (hipStream_t)stream, __func__); }

// ------------------------------------------------------------------------------------------------
// one step: next = A state + x, h = next rounded to the storage type.  Reads gate, x and state, writes both: bandwidth, or the launch
// (160 000 x 64 bf16, 144 MB: 21.9 us, 6.6 TB/s; 1 024 x 32 fp32: 2.9 us).
// ------------------------------------------------------------------------------------------------
struct NfStepArgs {
    const void* gate; const void* x; const float* state; float* next; void* h;
    long long n; int D, gate32, shared, log_gate; long long gate_s, x_s, state_s, next_s;
};

template <typename E, int V> __global__ void __launch_bounds__(256) k_scan_step(NfStepArgs a)
{
    typedef typename E::st st;
    const long long e = ((long long)blockIdx.x * 256 + threadIdx.x) * V;
    if (e >= a.n) return;
    const long long r = e / a.D;
    const int d = (int)(e - r * a.D);
    typedef st SV __attribute__((ext_vector_type(V)));
    typedef float FV __attribute__((ext_vector_type(V)));
    float A[V];
    if (a.shared) {
        float g0;
        if (sizeof(st) == 4 || a.gate32) g0 = ((const float*)a.gate)[r * a.gate_s];
        else g0 = E::cv(((const st*)a.gate)[r * a.gate_s]);
        if (a.log_gate) g0 = expf(g0);
#pragma unroll
        for (int k = 0; k < V; ++k) A[k] = g0;
    } else {
        if (sizeof(st) == 4 || a.gate32) {
            const FV v = *(const FV*)((const float*)a.gate + r * a.gate_s + d);
#pragma unroll
            for (int k = 0; k < V; ++k) A[k] = v[k];
        } else {
            const SV v = *(const SV*)((const st*)a.gate + r * a.gate_s + d);
#pragma unroll
            for (int k = 0; k < V; ++k) A[k] = E::cv(v[k]);
        }
        if (a.log_gate)
#pragma unroll
            for (int k = 0; k < V; ++k) A[k] = expf(A[k]);
    }
    const SV xv = *(const SV*)((const st*)a.x + r * a.x_s + d);
    const FV sv = *(const FV*)(a.state + r * a.state_s + d);
    FV o;
    SV h;
#pragma unroll
    for (int k = 0; k < V; ++k) { o[k] = fmaf(A[k], sv[k], E::cv(xv[k])); h[k] = E::pk(o[k]); }
    *(FV*)(a.next + r * a.next_s + d) = o;
    *(SV*)((st*)a.h + e) = h;
}

extern "C" int nf_scan_step(int dtype, int gate32, int shared, int log_gate, int rows, int D, const void* gate, int64_t gate_stride, const void* x,
                            int64_t x_stride, const float* state, int64_t state_stride, float* next, int64_t next_stride, void* h, nf_stream_t stream)
{
    NF_CHECK_ARG(dtype >= 0 && dtype <= 2, "dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    NF_CHECK_ARG(rows >= 0 && D >= 1, "bad sizes");
    if (rows == 0) return NF_OK;
    NF_CHECK_ARG(gate && x && state && next && h, "null pointer");
    NfStepArgs a = {gate, x, state, next, h, (long long)rows * D, D, gate32 != 0, shared != 0, log_gate != 0, gate_stride, x_stride, state_stride, next_stride};
    const int es = dtype == 0 ? 4 : 2, gs = (dtype == 0 || gate32) ? 4 : 2;
    // four elements a thread where every row allows it: 16-byte accesses of the fp32 state
    const bool v4 = D % 4 == 0 && (uintptr_t)x % (4 * es) == 0 && x_stride % 4 == 0 && (uintptr_t)state % 16 == 0 && state_stride % 4 == 0 &&
                    (uintptr_t)next % 16 == 0 && next_stride % 4 == 0 && (uintptr_t)h % (4 * es) == 0 &&
                    (shared || ((uintptr_t)gate % (4 * gs) == 0 && gate_stride % 4 == 0));
    const long long threads = a.n / (v4 ? 4 : 1);
    NF_CHECK_ARG(threads <= 0xffffff00LL, "too many elements");         // (a launch has fewer than 2^32 threads)
    const dim3 grid((unsigned)((threads + 255) / 256));
    hipStream_t st = (hipStream_t)stream;
#define NF_STEP(E)                                                                                     \
    do {                                                                                               \
        if (v4) hipLaunchKernelGGL((k_scan_step<E, 4>), grid, dim3(256), 0, st, a);                     \
        else hipLaunchKernelGGL((k_scan_step<E, 1>), grid, dim3(256), 0, st, a);                        \
    } while (0)
    if (dtype == 0) NF_STEP(NfF32);
    else if (dtype == 1) NF_STEP(NfBf16);
    else NF_STEP(NfF16);
#undef NF_STEP
    NF_CHECK_LAUNCH();
    return NF_OK;
}
