// Paged attention of trees of new tokens, 16-bit activations and cache (paged_attn.cuh).
#include "paged_attn.cuh"

namespace wcb {
namespace paged {

cudaError_t launch_tree_16(const AttendArgs& a, int act, int rows, cudaStream_t s) {
  return act == E_F16 ? run_attend_rows<__half, __half, true>(a, rows, s)
                      : run_attend_rows<__nv_bfloat16, __nv_bfloat16, true>(a, rows, s);
}

}  // namespace paged
}  // namespace wcb
