// Paged attention, f32 activations over any cache (paged_attn.cuh).
#include "paged_attn.cuh"

namespace wcb {
namespace paged {

cudaError_t launch_attend_32(const AttendArgs& a, int cache, int rows, cudaStream_t s) {
  return cache == E_F16    ? run_attend_rows<float, __half>(a, rows, s)
         : cache == E_BF16 ? run_attend_rows<float, __nv_bfloat16>(a, rows, s)
                           : run_attend_rows<float, float>(a, rows, s);
}

}  // namespace paged
}  // namespace wcb
