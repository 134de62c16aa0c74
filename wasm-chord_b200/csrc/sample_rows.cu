// Tokens from rows of logits: temperature, top-k, top-p, min-p, a draw from a given random number.
//
// With m a row's largest logit, token j weighs e_j = exp((l_j - m) / T). In the order of falling logits (ties: the
// lowest index first) top-k keeps the first k, top-p of those the ones before which less than p of their sum
// lies, min-p those with e_j >= min_p; each is a beginning of the same order, so all that is left is one too: the
// logits above a threshold, and of those at it the ones up to some index. The token is the lowest index at
// which the sum of the kept e in the order of indices exceeds u times the sum of all.
//
// Sums are whole numbers: e_j is rounded to steps of 2^-43 (of the largest, which is 1), so that sums of up to 2^20
// of them fit in 64 bits and come out the same in any order. e itself is computed in 64 bits, 2^-44 of its value:
// e = 2^(n / 64) (1 + s + s^2 / 2 + s^3 / 6 + s^4 / 24), n the nearest whole number to y = 64 log2(e) (l - m) / T,
// s = (y - n) ln(2) / 64.
//
// Split: a cluster of C CTAs takes a row, each a slice of its indices. The order is never made: the
// thresholds are found digit by digit (8 bits of the logits' order-preserving bits at a time), counting (top-k) or
// summing (top-p) the tokens of each digit in shared memory; the CTAs read each other's counts through
// distributed shared memory.
#include <cooperative_groups.h>

#include <atomic>
#include <climits>

#include "paged_common.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int SR_THREADS = 512;
constexpr int SR_WARPS = SR_THREADS / 32;
constexpr int SR_CLUSTER = 8;
constexpr int SR_CACHE = 200 * 1024;  // bytes of a slice in shared memory at most
constexpr int FIX = 43;  // bits after the point

// order-preserving bits; 0: no candidate (NaN, -infinity)
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l >= -FLT_MAX)) return 0;
  const uint32_t b = __float_as_uint(l + 0.0f);  // (-0 is 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// What is left after a filter: keys above `key`, and those at it up to index `last`.
struct Kept {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool has(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};
__device__ __forceinline__ Kept stricter(const Kept& a, const Kept& b) {
  return a.key != b.key ? (a.key > b.key ? a : b) : (a.last < b.last ? a : b);
}

struct Weights {
  double top, rate;  // the largest logit; 64 log2(e) / T
  const double* table;
  // a logit of at most `top`
  __device__ __forceinline__ double of(float l) const {
    if (double(l) == top) return 1.0;  // (infinities too)
    const double y = (double(l) - top) * rate;
    if (!(y >= -60.0 * 64.0)) return 0.0;  // (far below a step)
    const double big = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double z = y + big;
    const int n = __double2loint(z);
    const double s = (y - (z - big)) * (0.69314718055994530942 / 64.0);
    const double p = table[n & 63] * (1.0 + s * (1.0 + s * (0.5 + s * (1.0 / 6.0 + s * (1.0 / 24.0)))));
    return __hiloint2double(__double2hiint(p) + ((n >> 6) << 20), __double2loint(p));
  }
};
__device__ __forceinline__ unsigned long long fixed(double e) {
  const double one = 512.0;  // its last bit is 2^-43
  return static_cast<unsigned long long>(__double_as_longlong(e + one) - __double_as_longlong(one));
}

struct SampleShared {
  double table[64];
  unsigned count[2][256], lo[2][256], hi[2][256];  // of a digit: tokens, the two halves of their sum
  unsigned long long sum[2][SR_CLUSTER];
  int num[2][SR_CLUSTER];
  unsigned long long warp_sum[SR_WARPS];
  int warp_num[SR_WARPS];
  unsigned long long pick_before;
  unsigned pick_bin, pick_count;
  int found;
};

// CACHED: the slice fits into shared memory; else it is read again and again
template <typename T, bool CACHED>
__global__ void __launch_bounds__(SR_THREADS, 2) sample_kernel(const __grid_constant__ SampleArgs a, int per) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ float cache[];
  __shared__ SampleShared sh;
  const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
  const int first = rank * per, mine = max(0, min(per, a.vocab - first));
  if (tid < 64) sh.table[tid] = exp2(double(tid) / 64.0);
  // every CTA of the cluster runs before any writes into another's shared memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  auto logit = [&](int i) {
    if constexpr (CACHED) return cache[i];
    else return to_f32(logits[first + i]);
  };

  int swap = 0;  // which of the exchanged arrays is in use: what the others may still be reading is the other one
  // a number of each CTA's threads, summed (or the largest) over the cluster
  auto block_sum = [&](unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sh.warp_sum[warp] = v;
    __syncthreads();
    unsigned long long all = 0;
#pragma unroll
    for (int w = 0; w < SR_WARPS; ++w) all += sh.warp_sum[w];
    return all;
  };
  auto exchange = [&](unsigned long long v) {  // to sh.sum[swap][] of every CTA
    swap ^= 1;
    if (tid < C) cluster.map_shared_rank(&sh.sum[swap][0], tid)[rank] = v;
    cluster.sync();
  };

  // the slice, and the row's largest key
  uint32_t best = 0;
  for (int i = tid; i < mine; i += SR_THREADS) {
    const float l = to_f32(logits[first + i]);
    if constexpr (CACHED) cache[i] = l;
    best = max(best, key_of(l));
  }
  best = __reduce_max_sync(0xffffffffu, best);
  if (lane == 0) sh.warp_num[warp] = int(best);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SR_WARPS; ++w) best = max(best, uint32_t(sh.warp_num[w]));
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  exchange(best);
  for (int r = 0; r < C; ++r) best = max(best, uint32_t(sh.sum[swap][r]));

  float* probs = a.probs ? a.probs + row * a.probs_stride + first : nullptr;
  if (best == 0) {  // no candidates
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.status) atomicOr(a.status, uint32_t(ST_BAD_PROBS));
    }
    if (probs)
      for (int i = tid; i < mine; i += SR_THREADS) probs[i] = 0.0f;
    return;
  }
  const uint32_t best_bits = best & 0x80000000u ? best & 0x7fffffffu : ~best;
  const float temp = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  const bool greedy = !(temp > 0.0f);
  Weights w{double(__uint_as_float(best_bits)), greedy ? 0.0 : 64.0 * 1.4426950408889634074 / double(temp), sh.table};
  int top_k = a.top_k ? __ldg(a.top_k + row) : 0;
  float top_p = a.top_p ? __ldg(a.top_p + row) : 1.0f, min_p = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  if (greedy) {
    top_k = 1;
    top_p = 1.0f;
    min_p = 0.0f;
  }
  Kept kept{1u, INT_MAX};  // every candidate

  // How many of the tokens at `key` a CTA's slice has, and where its n-th one is (n from 0; -1: it has fewer)
  auto nth_at = [&](uint32_t key, int n) {
    // the index of the n-th token at `key` of the row
    int cnt = 0;
    const int part = (mine + SR_WARPS - 1) / SR_WARPS, from = min(mine, warp * part), to = min(mine, from + part);
    for (int i = from + lane; i < to; i += 32) cnt += key_of(logit(i)) == key;
    cnt = __reduce_add_sync(0xffffffffu, unsigned(cnt));
    __syncthreads();
    if (lane == 0) sh.warp_num[warp] = cnt;
    __syncthreads();
    int all = 0, before = 0;
    for (int x = 0; x < SR_WARPS; ++x) {
      if (x < warp) before += sh.warp_num[x];
      all += sh.warp_num[x];
    }
    exchange(all);
    for (int r = 0; r < rank; ++r) before += int(sh.sum[swap][r]);
    __syncthreads();
    if (n >= before && n < before + cnt) {  // in this warp's part
      int left = n - before;
      for (int i0 = from; i0 < to; i0 += 32) {
        const int i = i0 + lane;
        unsigned at = __ballot_sync(0xffffffffu, i < to && key_of(logit(i)) == key);
        const int c = __popc(at);
        if (left < c) {
          for (; left > 0; --left) at &= at - 1;
          if (lane < C) cluster.map_shared_rank(&sh.found, lane)[0] = first + i0 + __ffs(int(at)) - 1;
          break;
        }
        left -= c;
      }
    }
    cluster.sync();
    return sh.found;
  };

  // The end of the kept tokens in the order of falling logits, among those of `in`: by count (the goal-th one), or by weight: the first
  // with which the sum reaches goal.
  auto select = [&](const Kept& in, bool by_weight, double goal) {
    uint32_t prefix = 0;
    unsigned long long before = 0;  // count or weight of the digits above
    unsigned inside = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      const int b = (shift >> 3) & 1;
      __syncthreads();
      if (tid < 256) sh.count[b][tid] = sh.lo[b][tid] = sh.hi[b][tid] = 0;
      __syncthreads();
      for (int i = tid; i < mine; i += SR_THREADS) {
        const uint32_t k = key_of(logit(i));
        if (!in.has(k, first + i) || (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
        const unsigned d = (k >> shift) & 255u;
        atomicAdd(&sh.count[b][d], 1u);
        if (by_weight) {
          const unsigned long long f = fixed(w.of(logit(i)));
          const unsigned lo = unsigned(f), old = atomicAdd(&sh.lo[b][d], lo);
          atomicAdd(&sh.hi[b][d], unsigned(f >> 32) + (old + lo < old ? 1u : 0u));
        }
      }
      cluster.sync();
      unsigned cnt = 0;
      unsigned long long mass = 0;
      if (tid < 256) {
        const int d = 255 - tid;  // from the top
        for (int r = 0; r < C; ++r) {
          cnt += cluster.map_shared_rank(&sh.count[b][0], r)[d];
          if (by_weight) mass += (static_cast<unsigned long long>(cluster.map_shared_rank(&sh.hi[b][0], r)[d]) << 32) + cluster.map_shared_rank(&sh.lo[b][0], r)[d];
        }
        if (!by_weight) mass = cnt;
        unsigned long long inc = mass;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += t;
        }
        if (lane == 31) sh.warp_sum[warp] = inc;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        unsigned long long base = before;
        for (int x = 0; x < warp; ++x) base += sh.warp_sum[x];
        const unsigned long long upto = base + inc, prev = upto - mass;
        if (double(upto) >= goal && double(prev) < goal) {  // one digit: the goal is above zero and below the sum of all
          sh.pick_bin = unsigned(d);
          sh.pick_count = cnt;
          sh.pick_before = prev;
        }
      }
      __syncthreads();
      prefix |= sh.pick_bin << shift;
      before = sh.pick_before;
      inside = sh.pick_count;
    }
    // tokens at one key: how many of them
    unsigned take = inside;
    if (by_weight) {
      const double e = double(fixed(w.of(__uint_as_float(prefix & 0x80000000u ? prefix & 0x7fffffffu : ~prefix))));
      const double need = ceil((goal - double(before)) / e);
      take = need >= double(inside) || !(e > 0.0) ? inside : need > 1.0 ? unsigned(need) : 1u;
    } else {
      take = unsigned(goal) - unsigned(before);
    }
    __syncthreads();
    Kept out{prefix, INT_MAX};
    if (take < inside) out.last = nth_at(prefix, int(take) - 1);
    return out;
  };

  if (top_k > 0 && top_k < a.vocab) {
    unsigned n = 0;
    for (int i = tid; i < mine; i += SR_THREADS) n += key_of(logit(i)) != 0;
    __syncthreads();
    exchange(block_sum(n));
    unsigned long long all = 0;
    for (int r = 0; r < C; ++r) all += sh.sum[swap][r];
    if (static_cast<unsigned long long>(top_k) < all) kept = select(kept, false, double(top_k));
  }
  if (top_p < 1.0f) {
    unsigned long long v = 0;
    for (int i = tid; i < mine; i += SR_THREADS)
      if (kept.has(key_of(logit(i)), first + i)) v += fixed(w.of(logit(i)));
    __syncthreads();
    exchange(block_sum(v));
    unsigned long long all = 0;
    for (int r = 0; r < C; ++r) all += sh.sum[swap][r];
    kept = stricter(kept, select(kept, true, fmax(1.0, double(fmaxf(top_p, 0.0f)) * double(all))));
  }
  const double floor_e = min_p > 0.0f ? fmin(double(min_p), 1.0) : 0.0;

  // the sum of what is kept, by warps (each a part of the slice)
  const int part = (mine + SR_WARPS - 1) / SR_WARPS, from = min(mine, warp * part), to = min(mine, from + part);
  auto weight = [&](int i) {
    const float l = logit(i);
    if (!kept.has(key_of(l), first + i)) return 0.0;
    const double e = w.of(l);
    return e >= floor_e ? e : 0.0;
  };
  unsigned long long v = 0;
  for (int i = from + lane; i < to; i += 32) v += fixed(weight(i));
  __syncthreads();
  const unsigned long long own = block_sum(v);
  exchange(own);
  unsigned long long all = 0, before = 0;
  for (int r = 0; r < C; ++r) {
    if (r < rank) before += sh.sum[swap][r];
    all += sh.sum[swap][r];
  }
  if (probs) {
    const double inv = 1.0 / (double(all) * (1.0 / double(1ull << FIX)));
    for (int i = tid; i < mine; i += SR_THREADS) probs[i] = float(weight(i) * inv);
  }
  float u = __ldg(a.u + row);
  u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
  const double goal = double(u) * double(all);
  // the CTA, then the warp, whose sum passes the goal (the sum of all does)
  if (!(double(before) <= goal && double(before + own) > goal)) return;
  unsigned long long base = before;
  for (int x = 0; x < warp; ++x) base += sh.warp_sum[x];
  if (!(double(base) <= goal && double(base + sh.warp_sum[warp]) > goal)) return;
  for (int i0 = from; i0 < to; i0 += 32) {
    const int i = i0 + lane;
    const unsigned long long f = i < to ? fixed(weight(i)) : 0;
    unsigned long long inc = f;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, double(base + inc) > goal);
    if (hit) {
      if (lane == 0) a.tokens[row] = first + i0 + __ffs(int(hit)) - 1;
      break;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
}

template <typename T, bool CACHED>
cudaError_t run_sample(const SampleArgs& a, int c, int per, size_t shared, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  if (CACHED) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!(done.load(std::memory_order_acquire) & bit)) {
      e = cudaFuncSetAttribute(sample_kernel<T, CACHED>, cudaFuncAttributeMaxDynamicSharedMemorySize, SR_CACHE);
      if (e != cudaSuccess) return e;
      done.fetch_or(bit, std::memory_order_release);
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.n_rows) * unsigned(c));
  cfg.blockDim = dim3(SR_THREADS);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(c);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, CACHED>, a, per);
}

template <typename T>
cudaError_t run_sample(const SampleArgs& a, cudaStream_t s) {
  // CTAs of a row: until there are two for each SM, with slices of at least 1024 logits; more where the slices do not fit
  int c = 1;
  while (c < SR_CLUSTER && ((a.n_rows * c < 2 * SMS && a.vocab / (2 * c) >= 1024) || static_cast<long long>(a.vocab + c - 1) / c * 4 > SR_CACHE / 2)) c *= 2;
  const int per = (a.vocab + c - 1) / c;
  if (per <= SR_CACHE / 4) return run_sample<T, true>(a, c, per, size_t(per) * 4, s);
  return run_sample<T, false>(a, c, per, 0, s);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int kind, cudaStream_t s) {
  return kind == E_F16 ? run_sample<__half>(a, s) : kind == E_BF16 ? run_sample<__nv_bfloat16>(a, s) : run_sample<float>(a, s);
}

}  // namespace paged
}  // namespace wcb
