// Block norms: adjoints of the first gradients (see block_norm.cuh).
#include "block_norm.cuh"

namespace ictc {
namespace block_norm {

cudaError_t launch_second(const BlockArgs& a, const Shape& s, int grid, int bytes, int lmax, int layout, bool branch,
                       cudaStream_t stream) {
  return launch_mode<kSecond>(a, s, grid, bytes, lmax, layout, branch, stream);
}

}  // namespace block_norm
}  // namespace ictc
