// Paged attention of trees of new tokens on the tensor cores, 16-bit activations and cache (paged_attn_tc.cuh).
#include "paged_attn_tc.cuh"

namespace wcb {
namespace paged {

cudaError_t launch_tree_tc(const AttendArgs& a, int act, cudaStream_t s) { return run_tc_act<true>(a, act, s); }

}  // namespace paged
}  // namespace wcb
