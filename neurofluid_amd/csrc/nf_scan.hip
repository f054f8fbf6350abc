// nf_scan.hip — entry points of the gated linear recurrence (kernels: nf_scan.h).
//
// Where the parallelism comes from.  A (sequence, block of channels) is a chain; its tiles follow one another.
//   many chains: one workgroup (NW = 4 waves on a tile) or one wave (NW = 1, four chains a workgroup) walks a whole chain, each
//     tensor is read and written once;
//   few chains: the time axis is cut into chunks of whole tiles.  One launch reduces every chunk to (P, H), a small one carries the states
//     through the chunks in order, a third runs the chunks from the states that enter them.  The gate and the input are read twice.
#include "nf_scan.h"
#include <math.h>

static int scan_tile(int cg, int nw) { return nw * (64 / cg) * NF_SCAN_TPT; }

// Chunks a chain is cut into: enough workgroups for four per CU.
static int scan_chunks(const nf_scan_t* s)
{
    const int tile = scan_tile(s->cg, s->nw), ntiles = (s->T + tile - 1) / tile;
    const long long units = (long long)s->B * ((s->D + s->cg * s->vec - 1) / (s->cg * s->vec));
    if (s->nw == 1 || ntiles <= 4 || units >= 512) return 1;
    const long long want = (1024 + units - 1) / units;
    const int per = (int)((ntiles + want - 1) / want);
    return (ntiles + per - 1) / per;
}

static int scan_check(const nf_scan_t* s, const char* who)
{
    if (!s) { nf_set_error("%s: null descriptor", who); return NF_EINVAL; }
    if (s->dtype < 0 || s->dtype > 2) { nf_set_error("%s: dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)", who); return NF_EINVAL; }
    if (s->B < 0 || s->T < 0 || s->D < 1) { nf_set_error("%s: bad sizes", who); return NF_EINVAL; }
    if (s->row_splits && (s->B != 1 || s->n_seq < 0)) { nf_set_error("%s: packed rows come as one batch", who); return NF_EINVAL; }
    return NF_OK;
}

static bool scan_plan_ok(const nf_scan_t* s)
{
    return (s->vec == 1 || s->vec == 2) && (s->cg == 32 || s->cg == 16 || s->cg == 8 || s->cg == 2) && (s->nw == 1 || s->nw == 4) &&
           (s->vec == 1 || s->D % 2 == 0);
}

// true if every row that (base, strides) reaches can be read two elements at a time
static bool scan_pairs(const void* p, int64_t sb, int64_t st, int size) { return (uintptr_t)p % (2 * size) == 0 && sb % 2 == 0 && st % 2 == 0; }

extern "C" int nf_scan_plan(nf_scan_t* s, size_t* state_floats)
{
    const int rc = scan_check(s, __func__);
    if (rc) return rc;
    const int es = s->dtype == 0 ? 4 : 2, gs = (s->dtype == 0 || s->gate32) ? 4 : 2;
    s->vec = (s->D % 2 == 0 && scan_pairs(s->x, s->x_sb, s->x_st, es) && (s->shared || scan_pairs(s->gate, s->gate_sb, s->gate_st, gs))) ? 2 : 1;
    s->cg = 32;
    const int cgs[3] = {2, 8, 16};
    for (int i = 2; i >= 0; --i)
        if (cgs[i] * s->vec >= s->D) s->cg = cgs[i];
    const int nblk = (s->D + s->cg * s->vec - 1) / (s->cg * s->vec);
    const int t1 = scan_tile(s->cg, 1);
    s->nw = (!s->row_splits && ((long long)s->B * nblk >= 4096 || s->T <= 2 * t1)) ? 1 : 4;
    const int tile = scan_tile(s->cg, s->nw);
    if (state_floats) *state_floats = (size_t)s->B * ((s->T + tile - 1) / tile) * s->D;
    return NF_OK;
}

// workspace: [agg | carry] when the time axis is cut, then the per-block sums of a shared gate's gradient
static void scan_workspace(const nf_scan_t* s, int backward, size_t* agg, size_t* carry, size_t* part)
{
    const int nchunk = scan_chunks(s), nblk = (s->D + s->cg * s->vec - 1) / (s->cg * s->vec);
    *agg = nchunk > 1 ? (size_t)s->B * nchunk * 2 * s->D : 0;
    *carry = nchunk > 1 ? (size_t)s->B * nchunk * s->D : 0;
    *part = (backward && s->shared && s->dgate && nblk > 1) ? (size_t)nblk * s->B * s->T : 0;
}

extern "C" size_t nf_scan_workspace_floats(const nf_scan_t* s, int backward)
{
    if (scan_check(s, __func__) || !scan_plan_ok(s)) return 0;
    size_t a, c, p;
    scan_workspace(s, backward, &a, &c, &p);
    return a + c + p;
}

// The sequence of every packed row (-1: before the first or behind the last), by bisection of the splits; the final states of empty
// sequences are their initial ones (and their gradients pass through): written here.  Splits are clamped to [0, T], so that bad ones give bad
// numbers but no access out of range.
__global__ void __launch_bounds__(256) k_scan_rows(const int64_t* __restrict__ rs, int n_seq, int T, int* __restrict__ sid)
{
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (r >= T) return;
    int lo = 0, hi = n_seq;              // the number of k in [1, n_seq] with rs[k] <= r
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (rs[mid + 1] <= r) lo = mid + 1;
        else hi = mid;
    }
    sid[r] = (lo < n_seq && rs[lo] <= r) ? lo : -1;
}

__global__ void __launch_bounds__(256) k_scan_empty(const int64_t* __restrict__ rs, int n_seq, int T, int D, const float* __restrict__ src,
                                                    float* __restrict__ dst)
{
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= (long long)n_seq * D) return;
    const int s = (int)(e / D);
    const int64_t a = min(max(rs[s], (int64_t)0), (int64_t)T), b = min(max(rs[s + 1], (int64_t)0), (int64_t)T);
    if (a >= b) dst[e] = src ? src[e] : 0.f;
}

// The states that enter the chunks, in order.  One thread per channel of a chain; the loads do not depend on the state.
__global__ void __launch_bounds__(64) k_scan_carry(const float* __restrict__ agg, const float* __restrict__ init, const int* __restrict__ sid, int B,
                                                   int D, int T, int nchunk, int steps, int reverse, int backward, float* __restrict__ carry)
{
    const int d = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (d >= D) return;
    float c = init ? init[(long long)b * D + d] : 0.f;
    auto at = [&](int j) { return (j < 0 || j >= T) ? -2 : sid[reverse ? T - 1 - j : j]; };
#pragma unroll 8
    for (int i = 0; i < nchunk; ++i) {
        const int k = backward ? nchunk - 1 - i : i;
        const long long o = (long long)b * nchunk + k;
        const float P = agg[o * 2 * D + d], H = agg[(o * 2 + 1) * D + d];
        carry[o * D + d] = c;
        bool closed = false;
        if (sid) {                       // does a sequence begin (backwards: end) inside the chunk?
            const int j0 = k * steps, j1 = min(T, j0 + steps) - 1;
            closed = backward ? at(j1 + 1) != at(j0) : at(j0 - 1) != at(j1);
        }
        c = closed ? H : fmaf(P, c, H);
    }
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
    if (s->dtype == 0) return nf_scan_launch_f32(a, s->vec, s->cg, s->nw, backward, st);
    if (s->dtype == 1) return nf_scan_launch_bf16(a, s->vec, s->cg, s->nw, backward, st);
    return nf_scan_launch_f16(a, s->vec, s->cg, s->nw, backward, st);
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
    if (packed && s->n_seq > 0 && fin) {
        const long long n = (long long)s->n_seq * s->D;
        hipLaunchKernelGGL(k_scan_empty, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, s->row_splits, s->n_seq, s->T, s->D, init, fin);
        NF_CHECK_LAUNCH();
    }
    if (s->B == 0 || s->T == 0) return NF_OK;        // (dense with T = 0: the caller copies the state)
    if (!s->gate || !s->x || (backward ? !s->states : !s->h)) { nf_set_error("%s: null pointer", who); return NF_EINVAL; }
    if (packed && !s->sid) { nf_set_error("%s: packed rows need the row buffer (sid)", who); return NF_EINVAL; }
    const int es = s->dtype == 0 ? 4 : 2, gs = (s->dtype == 0 || s->gate32) ? 4 : 2;
    if (s->vec == 2 && !(scan_pairs(s->x, s->x_sb, s->x_st, es) && (s->shared || scan_pairs(s->gate, s->gate_sb, s->gate_st, gs)) &&
                         (!backward || !s->g || scan_pairs(s->g, s->g_sb, s->g_st, es)))) {
        nf_set_error("%s: the plan reads two elements at a time, a tensor is not aligned for it", who);
        return NF_EINVAL;
    }
    NfScanArgs a = {};
    a.gate = s->gate; a.x = s->x; a.g = s->g; a.h0 = s->h0; a.g_last = s->g_last; a.h = s->h; a.h_last = s->h_last; a.states = s->states;
    a.dgate = s->dgate; a.dx = s->dx; a.dh0 = s->dh0; a.sid = packed ? s->sid : nullptr;
    a.gate_sb = s->gate_sb; a.gate_st = s->gate_st; a.x_sb = s->x_sb; a.x_st = s->x_st; a.g_sb = s->g_sb; a.g_st = s->g_st;
    a.B = s->B; a.T = s->T; a.D = s->D;
    const int tile = scan_tile(s->cg, s->nw);
    a.nblk = (s->D + s->cg * s->vec - 1) / (s->cg * s->vec);
    a.ntiles = (s->T + tile - 1) / tile;
    a.nchunk = scan_chunks(s);
    a.tiles_per_chunk = (a.ntiles + a.nchunk - 1) / a.nchunk;
    a.gate32 = s->gate32 != 0; a.shared = s->shared != 0; a.log_gate = s->log_gate != 0; a.reverse = s->reverse != 0;
    if ((long long)a.B * a.nblk * a.nchunk > 0x7fffffffLL) { nf_set_error("%s: too many chains", who); return NF_EINVAL; }
    size_t n_agg, n_carry, n_part;
    scan_workspace(s, backward, &n_agg, &n_carry, &n_part);
    if (s->workspace_floats < n_agg + n_carry + n_part || (n_agg + n_carry + n_part && !s->workspace)) {
        nf_set_error("%s: workspace too small (nf_scan_workspace_floats)", who);
        return NF_EINVAL;
    }
    float* agg = s->workspace;
    float* carry = agg + n_agg;
    a.dgate_part = n_part ? carry + n_carry : nullptr;
    if (packed && !backward) {
        hipLaunchKernelGGL(k_scan_rows, dim3((unsigned)((s->T + 255) / 256)), dim3(256), 0, st, s->row_splits, s->n_seq, s->T, s->sid);
        NF_CHECK_LAUNCH();
    }
    if (a.nchunk > 1) {
        NfScanArgs r = a;
        r.only_agg = 1; r.agg = agg;
        if (!scan_go(s, r, backward, st)) { nf_set_error("%s: no kernel for the plan", who); return NF_EINVAL; }
        NF_CHECK_LAUNCH();
        hipLaunchKernelGGL(k_scan_carry, dim3((s->D + 63) / 64, s->B), dim3(64), 0, st, (const float*)agg, packed ? (const float*)nullptr : init, a.sid, s->B,
                           s->D, s->T, a.nchunk, a.tiles_per_chunk * tile, a.reverse, backward, carry);
        NF_CHECK_LAUNCH();
        a.carry = carry;
    }
    if (!scan_go(s, a, backward, st)) { nf_set_error("%s: no kernel for the plan", who); return NF_EINVAL; }
    NF_CHECK_LAUNCH();
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
// one step: next = A state + x, h = next rounded to the storage type.  Reads gate, x and state, writes both: bandwidth, or the launch.
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
    NF_CHECK_ARG((threads + 255) / 256 <= 0x7fffffffLL, "too many elements");
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
