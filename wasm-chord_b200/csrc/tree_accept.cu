// The way down a tree of drafted tokens: from the first new token on to the child that holds the
// token sampled at its parent, as long as there is one.
//
// next[p] = the lowest i with parent[i] = p and token[i] = sampled[p]; the way is 0, next[0], next[next[0]] ..
// Bound by latency: 12 bytes a node. One CTA a sequence finds next[] of all nodes at once in shared
// memory, one thread walks it; so the loads of a tree are three dependent ones, not three for each level. A
// sequence of more than NODES tokens is searched level by level instead. One tree of 26 tokens 2.9 us, 256 of 32 to 128 tokens 3.3 us
// (GPU time in a graph), of which a launch is two.
#include "paged_common.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int AC_THREADS = 128;
constexpr int NODES = 4096;

__global__ void __launch_bounds__(AC_THREADS) accept_kernel(const __grid_constant__ AcceptArgs a) {
  __shared__ int next[NODES];
  __shared__ int s_count, s_child;
  const int tid = threadIdx.x, s = blockIdx.x;
  const Seq q = read_seq(a.batch, s);
  if (!q.sound && tid == 0) report(a.batch, ST_BAD_ROWS);
  const int32_t* parent = a.parent + q.r0;
  const int32_t* token = a.token + q.r0;
  const int32_t* sampled = a.sampled + q.r0;
  int32_t* path = a.path + int64_t(s) * a.max_path;
  int32_t* tokens = a.tokens + int64_t(s) * a.max_path;
  const int n = q.n;
  bool bad = false;
  if (n <= NODES) {
    for (int i = tid; i < n; i += AC_THREADS) next[i] = n;
    __syncthreads();
    for (int i = tid; i < n; i += AC_THREADS) {
      if (i == 0) continue;
      const int p = __ldg(parent + i);
      if (p < -1 || p >= i) bad = true;
      else if (p >= 0) {
        const int t = __ldg(sampled + p);
        if (t >= 0 && t == __ldg(token + i)) atomicMin(&next[p], i);
      }
    }
    __syncthreads();
    if (tid == 0) {
      int c = 0, at = 0;
      for (; at < n && c < a.max_path; ++c) {
        const int to = next[at];
        next[at] = -1 - c;  // (a node's place on the way, for the others)
        path[c] = at;
        at = to;
      }
      s_count = c;
    }
    __syncthreads();
    for (int i = tid; i < n; i += AC_THREADS)
      if (next[i] < 0) tokens[-1 - next[i]] = __ldg(sampled + i);
  } else {
    for (int i = 1 + tid; i < n; i += AC_THREADS) {
      const int p = __ldg(parent + i);
      bad |= p < -1 || p >= i;
    }
    int c = 0, at = 0;
    while (at < n && c < a.max_path) {
      const int t = __ldg(sampled + at);
      if (tid == 0) {
        path[c] = at;
        tokens[c] = t;
        s_child = n;
      }
      ++c;
      __syncthreads();
      if (t >= 0) {
        for (int i = at + 1 + tid; i < n; i += AC_THREADS)
          if (__ldg(parent + i) == at && __ldg(token + i) == t) {
            atomicMin(&s_child, i);
            break;
          }
      }
      __syncthreads();
      at = s_child;
      __syncthreads();
    }
    if (tid == 0) s_count = c;
    __syncthreads();
  }
  const int count = s_count;
  for (int i = count + tid; i < a.max_path; i += AC_THREADS) path[i] = tokens[i] = -1;
  if (tid == 0) a.count[s] = count;
  if (__syncthreads_or(bad) && tid == 0) report(a.batch, ST_BAD_TREE);
}

}  // namespace

cudaError_t launch_accept(const AcceptArgs& a, cudaStream_t s) {
  accept_kernel<<<a.batch.n_seqs, AC_THREADS, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace paged
}  // namespace wcb
