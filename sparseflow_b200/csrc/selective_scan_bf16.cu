// bf16 instantiations of the selective scan kernels.
#include "selective_scan.cuh"

namespace sf {
template sf_status scan_forward<__nv_bfloat16>(const ScanArgs&, int, bool, dim3, cudaStream_t);
template sf_status scan_backward<__nv_bfloat16>(const ScanArgs&, int, bool, dim3, cudaStream_t);
}  // namespace sf
