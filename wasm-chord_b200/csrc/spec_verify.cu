// Verification of drafted tokens against the target's probabilities.
//
// Token i is accepted while u_i q(x_i) < p(x_i) (the product of two 24-bit
// numbers is exact in 64 bits). At the first token turned down the next one is
// drawn from r_j = max(p_j - q_j, 0), after the last accepted one from p: the
// lowest j with r_0 + .. + r_j > u S. The target's row of each sequence is read, and the draft's where a token was
// turned down (where nothing is left of the target above the draft, the target's again): memory bound for
// large batches, latency bound for one sequence. A cluster of C CTAs shares one sequence's row in C slices: each
// sums its slice by chunks of 256 (64-bit sums, which keep the order of the
// chunks), the CTAs exchange their sums through distributed shared memory, and
// the one whose slice holds u S searches its chunks, then the chunk again.
//
// 192 sequences of 100003, a token turned down in 66 % of them (127 MB): 36 us, 54 % of the copy rate: each CTA has three
// steps that wait for one another (the count, the sums, the search), the loads of one row are
// too few to fill them, and 384 CTAs leave some SMs with three and others with two. One sequence of 32000: 5.7 us.
#include <cooperative_groups.h>

#include "paged_common.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int VF_THREADS = 512;
constexpr int VF_WARPS = VF_THREADS / 32;
constexpr int CHUNK = 256;  // probabilities of one warp's round
constexpr int MAX_CLUSTER = 8;

__device__ __forceinline__ float clean(float p) { return p > 0.0f && p <= FLT_MAX ? p : 0.0f; }

// r_j; `certain`: the draft's probabilities are 1 at that token and 0 elsewhere
__device__ __forceinline__ double rest(const float* p, const float* q, int certain, int j) {
  const float pj = clean(__ldg(p + j));
  const float qj = q ? clean(__ldg(q + j)) : (j == certain ? 1.0f : 0.0f);
  return pj > qj ? double(pj) - double(qj) : 0.0;
}

__global__ void __launch_bounds__(VF_THREADS, 3) verify_kernel(const __grid_constant__ VerifyArgs a, int chunks_per_cta) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int s = blockIdx.x / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ double chunk_sum[];  // [chunks_per_cta]
  __shared__ double s_sum[2][MAX_CLUSTER];
  __shared__ double s_warp[VF_WARPS];
  __shared__ int s_count;

  // every CTA of the cluster runs before any writes into another's shared memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // how many drafted tokens are accepted
  int len = a.draft_len ? __ldg(a.draft_len + s) : a.max_draft;
  len = max(0, min(len, a.max_draft));
  const float* tp = a.target + s * a.t_seq;
  const float* dp = a.draft_probs ? a.draft_probs + s * a.d_seq : nullptr;
  if (warp == 0) {
    int count = len;
    uint32_t bad = 0;
    for (int i0 = 0; i0 < len; i0 += 32) {
      const int i = i0 + lane;
      bool ok = true;
      if (i < len) {
        const int x = __ldg(a.draft + int64_t(s) * a.max_draft + i);
        if (x < 0 || x >= a.vocab) {
          ok = false;
          bad = ST_BAD_TOKEN;
        } else {
          const float p = clean(__ldg(tp + i * a.t_row + x));
          const float q = dp ? clean(__ldg(dp + i * a.d_row + x)) : 1.0f;
          const float u = __ldg(a.u_accept + int64_t(s) * a.max_draft + i);
          ok = double(u) * double(q) < double(p);
        }
      }
      const unsigned no = __ballot_sync(0xffffffffu, !ok);
      if (no) {
        count = i0 + __ffs(int(no)) - 1;
        break;
      }
    }
    if (bad && rank == 0 && a.status) atomicOr(a.status, bad);
    if (lane == 0) s_count = count;
  }
  __syncthreads();
  const int count = s_count;
  const float* p = tp + count * a.t_row;
  const float* q = nullptr;
  int certain = -1;
  if (count < len) {
    if (dp) q = dp + count * a.d_row;
    else certain = __ldg(a.draft + int64_t(s) * a.max_draft + count);
  }

  const int n_chunks = (a.vocab + CHUNK - 1) / CHUNK;
  const int first = rank * chunks_per_cta, mine = max(0, min(chunks_per_cta, n_chunks - first));
  double total = 0.0, before = 0.0, own = 0.0;
  int round = 0;
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  for (;; ++round) {
    // slice's chunk sums
    double acc = 0.0;
    for (int c = warp; c < mine; c += VF_WARPS) {
      const int j0 = (first + c) * CHUNK + lane;
      double v = 0.0;
      if (j0 - lane + CHUNK <= a.vocab) {
        float pj[CHUNK / 32], qj[CHUNK / 32];
#pragma unroll
        for (int e = 0; e < CHUNK / 32; ++e) pj[e] = __ldg(p + j0 + 32 * e);
        if (q) {
#pragma unroll
          for (int e = 0; e < CHUNK / 32; ++e) qj[e] = __ldg(q + j0 + 32 * e);
        } else {
#pragma unroll
          for (int e = 0; e < CHUNK / 32; ++e) qj[e] = j0 + 32 * e == certain ? 1.0f : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < CHUNK / 32; ++e) {
          const float x = clean(pj[e]), y = clean(qj[e]);
          v += x > y ? double(x) - double(y) : 0.0;
        }
      } else {
        for (int j = j0; j < a.vocab; j += 32) v += rest(p, q, certain, j);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) chunk_sum[c] = v;
      acc += v;
    }
    if (lane == 0) s_warp[warp] = acc;
    __syncthreads();
    if (tid < C) {  // the slice's sum to every CTA of the cluster
      double sum = 0.0;
      for (int w = 0; w < VF_WARPS; ++w) sum += s_warp[w];
      cluster.map_shared_rank(&s_sum[round][0], tid)[rank] = sum;
    }
    cluster.sync();
    total = before = 0.0;
    for (int r = 0; r < C; ++r) {
      if (r < rank) before += s_sum[round][r];
      total += s_sum[round][r];
    }
    own = s_sum[round][rank];
    if (total > 0.0 || round == 1 || count == len) break;
    q = nullptr;  // nothing is left of the target: draw from the target itself
    certain = -1;
  }

  int32_t* out = a.tokens + int64_t(s) * (a.max_draft + 1);
  if (rank == 0) {
    for (int i = tid; i <= a.max_draft; i += VF_THREADS) {
      if (i < count) out[i] = __ldg(a.draft + int64_t(s) * a.max_draft + i);
      else if (i > count || !(total > 0.0)) out[i] = -1;
    }
    if (tid == 0) {
      a.accepted[s] = count;
      if (!(total > 0.0) && a.status) atomicOr(a.status, uint32_t(ST_BAD_PROBS));
    }
  }
  if (!(total > 0.0) || own <= 0.0) return;
  float u = __ldg(a.u_sample + s);
  u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
  const double goal = double(u) * total;
  // the CTA whose slice passes the goal; sums grow with the rank, so exactly one does:
  // the first with before + own > goal (the last with anything in it, should rounding leave none)
  double upto = 0.0;
  int owner = -1, last = 0;
  for (int r = 0; r < C; ++r) {
    const double v = s_sum[round][r];
    upto += v;
    if (v > 0.0) last = r;
    if (owner < 0 && upto > goal) owner = r;
  }
  if (owner < 0) owner = last;
  if (owner != rank || warp != 0) return;
  // first warp: the chunk, then the token in it
  double run = before;
  int chunk = -1, some = 0;
  double base = 0.0;
  for (int c0 = 0; c0 < mine && chunk < 0; c0 += 32) {
    const int c = c0 + lane;
    const double v = c < mine ? chunk_sum[c] : 0.0;
    double inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    const unsigned has = __ballot_sync(0xffffffffu, v > 0.0), hit = __ballot_sync(0xffffffffu, v > 0.0 && run + inc > goal);
    const int pick = hit ? __ffs(int(hit)) - 1 : (has ? 31 - __clz(int(has)) : -1);
    if (pick >= 0) {
      some = c0 + pick;
      base = run + __shfl_sync(0xffffffffu, inc - v, pick);
    }
    if (hit) chunk = some;
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (chunk < 0) chunk = some;
  run = base;
  int token = -1, any = -1;
  for (int e = 0; e < CHUNK / 32 && token < 0; ++e) {
    const int j = (first + chunk) * CHUNK + 32 * e + lane;
    const double v = j < a.vocab ? rest(p, q, certain, j) : 0.0;
    double inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    const unsigned has = __ballot_sync(0xffffffffu, v > 0.0), hit = __ballot_sync(0xffffffffu, v > 0.0 && run + inc > goal);
    if (hit) token = j - lane + __ffs(int(hit)) - 1;
    if (has) any = j - lane + 31 - __clz(int(has));
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) out[count] = token >= 0 ? token : any;
}

}  // namespace

cudaError_t launch_verify(const VerifyArgs& a, cudaStream_t s) {
  // CTAs of a sequence: until there are two for each SM, with slices of at least 2048 probabilities.
  // (192 sequences of 100003: 2 CTAs 36.3 us, 1: 46, 3: 40, 4: 39)
  int c = 1;
  while (c < MAX_CLUSTER && a.n_seqs * c < 2 * SMS && a.vocab / (2 * c) >= 2048) c *= 2;
  const int n_chunks = (a.vocab + CHUNK - 1) / CHUNK;
  const int per = (n_chunks + c - 1) / c;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.n_seqs) * unsigned(c));
  cfg.blockDim = dim3(VF_THREADS);
  cfg.dynamicSmemBytes = sizeof(double) * size_t(per);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(c);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, verify_kernel, a, per);
}

}  // namespace paged
}  // namespace wcb
