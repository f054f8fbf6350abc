// nf_scan_f32.hip — the recurrence's kernels (nf_scan.h) for f32 storage.
#include "nf_scan.h"

int nf_scan_launch_f32(const NfScanArgs& a, int vec, int cg, int mode, int backward, hipStream_t st) { return nf_scan_launch<NfF32>(a, vec, cg, mode, backward, st); }
