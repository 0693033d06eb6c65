// selective_scan_f16.cu — the selective scan's kernels for __half.
#include "selective_scan.cuh"

template int mk::scan::run_type<__half>(const mk_scan_args*, const mk::Device*, const mk::scan::Plan&, bool, cudaStream_t);
