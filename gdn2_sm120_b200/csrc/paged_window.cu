// Attention of drafted tokens over a paged cache with a window and sinks: the kernels of tree attention, in which a sequence's
// tiles between the sinks and the window are passed over.
#include "paged_tree.cuh"

namespace gdn2 {
namespace paged {

int launch_tree_window(const TreeParams& p, int dtype, cudaStream_t stream) {
  return dtype == GDN2_BF16 ? launch_tree_dim<__nv_bfloat16, true>(p, stream) : launch_tree_dim<__half, true>(p, stream);
}

}  // namespace paged
}  // namespace gdn2
