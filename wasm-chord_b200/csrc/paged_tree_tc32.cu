// Paged attention of trees of new tokens on the tensor cores, f32 activations over any cache (paged_attn_tc32.cuh).
#include "paged_attn_tc32.cuh"

namespace wcb {
namespace paged {

cudaError_t launch_tree_tc32(const AttendArgs& a, int cache, cudaStream_t s) { return run_tc32_cache<true>(a, cache, s); }

}  // namespace paged
}  // namespace wcb
