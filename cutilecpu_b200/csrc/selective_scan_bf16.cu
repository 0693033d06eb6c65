// selective_scan_bf16.cu — the selective scan's kernels for __nv_bfloat16.
#include "selective_scan.cuh"

template int mk::scan::run_type<__nv_bfloat16>(const mk_scan_args*, const mk::Device*, const mk::scan::Plan&, bool, cudaStream_t);
