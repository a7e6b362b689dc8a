#include "smm_scan.cuh"
namespace smm {
bool scan_umma_fits(const ScanParams&, int) { return false; }
int scan_umma_launch(ScanParams&, cudaStream_t) { return SMM_ERR_UNSUPPORTED; }
int umma_seg_len(long long tokens, int, int, int) { return static_cast<int>(tokens > 0 ? tokens : 1); }
}
