// nf_scan_bf16.hip — the recurrence's kernels (nf_scan.h) for bf16 storage.
#include "nf_scan.h"

int nf_scan_launch_bf16(const NfScanArgs& a, int vec, int cg, int mode, int backward, hipStream_t st) { return nf_scan_launch<NfBf16>(a, vec, cg, mode, backward, st); }
