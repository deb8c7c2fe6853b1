// Attention of drafted tokens over a paged cache with a window and sinks: the kernels of tree attention, in which a sequence's
// tiles between the sinks and the window are passed over.
//
// Decoding 64 sequences of up to 16384 tokens, a window of 4096 and 4 sinks, 32 / 8 heads: 172 us, 6.25 TB/s of what the window
// holds; with a NaN among the values of every token and cached place 8 us more, since only tokens that were taken out of a tile are
// looked at again.  Trees of 24 drafts of 8 sequences, a window of 1000 and 64 sinks, pages of 16: 30 us and 8 for the join, a chain of
// drafts 22; without a window over as many tokens 21: latency, with two tiles of 128 tokens a CTA.  What a row sees of the tile
// at the window's edge follows from its place; the bytes of a tree's mask are loaded all at once (eight at a time 41 us).
#include "paged_tree.cuh"

namespace gdn2 {
namespace paged {

int launch_tree_window(const TreeParams& p, int dtype, cudaStream_t stream) {
  return dtype == GDN2_BF16 ? launch_tree_dim<__nv_bfloat16, true>(p, stream) : launch_tree_dim<__half, true>(p, stream);
}

}  // namespace paged
}  // namespace gdn2
