// selective_scan_f32.cu — the selective scan's kernels for float.
#include "selective_scan.cuh"

template int mk::scan::run_type<float>(const mk_scan_args*, const mk::Device*, const mk::scan::Plan&, bool, cudaStream_t);
