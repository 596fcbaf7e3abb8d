// Affine layer norm, backward pass for fp16 rows (a translation unit of its own: the shapes' kernels take a
// minute to compile for each type).
#include "layer_norm_backward.cuh"

namespace ctu {
namespace norm {

template cudaError_t backward_as<__half>(const AffineArgs &, const WaitLimit &, cudaStream_t);

}  // namespace norm
}  // namespace ctu
