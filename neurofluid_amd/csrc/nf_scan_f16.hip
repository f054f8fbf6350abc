// nf_scan_f16.hip — the recurrence's kernels (nf_scan.h) for f16 storage.
#include "nf_scan.h"

int nf_scan_launch_f16(const NfScanArgs& a, int vec, int cg, int mode, int backward, hipStream_t st) { return nf_scan_launch<NfF16>(a, vec, cg, mode, backward, st); }
