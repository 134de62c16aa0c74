// Tokens from rows of logits: temperature, top-k, top-p, min-p, a draw from a given random number.
//
// With m a row's largest logit, token j weighs e_j = exp((l_j - m) / T). In the order of falling logits (ties: the
// lowest index first) top-k keeps the first k, top-p of those the ones before which less than p of their sum
// lies, min-p those with e_j >= min_p; each is a beginning of the same order, so all that is left is one too: the
// logits above a threshold, and of those at it the ones up to some index. The token is the lowest index at
// which the sum of the kept e in the order of indices exceeds u times the sum of all.
//
// Sums are whole numbers: e_j is rounded to steps of 2^-43 (of the largest, which is 1), so that sums of up to 2^20
// of them fit in 64 bits and come out the same in any order. e itself is computed in 64 bits, to 2^-45 of its value: with
// y = log2(e) (l - m) / T and n the nearest whole number to y, e = 2^n 2^(y - n), the latter by its Chebyshev interpolation
// of degree 9 on [-1/2, 1/2].
//
// Split: a cluster of C CTAs takes a row, each a slice of its indices that stays in shared memory. The order is never
// made. Bins of (m - l) / T, counted, tell in which of them top-k ends, and, since a bin's width bounds its weights, between
// which two top-p does. One pass over the slice then computes each weight that is wanted once: tokens above the bins in question are
// summed, by chunks of 256 indices, for the draw; those in them, a few hundred, are gathered into every CTA, which finds the
// ends by itself, digit by digit (10 bits of the logits' order-preserving bits at a time, counting or summing the tokens of each digit), and adds what
// is kept of its own to its chunks. Where there are too many of them (many equal logits, say), the digits of the whole
// row are gone through, over all CTAs. What they exchange goes through distributed shared memory.
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
constexpr int SR_CACHE = 190 * 1024;     // bytes of a slice in shared memory at most
constexpr int SR_CACHE_TWO = 82 * 1024;  // so that an SM holds two
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
  double top, rate;  // the largest logit; log2(e) / T
  // a logit of at most `top`
  __device__ __forceinline__ double of(float l) const {
    if (double(l) == top) return 1.0;  // (infinities too)
    const double d = double(l) - top;
    constexpr double BIG = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double z = fma(d, rate, BIG);
    if (!(z >= BIG - 60.0)) return 0.0;  // far below a step (and where infinities are the largest)
    const double f = fma(d, rate, BIG - z);
    double p = 1.0205905413765595794e-7;
    p = fma(p, f, 1.325964524488711024e-6);
    p = fma(p, f, 1.5252672924850736404e-5);
    p = fma(p, f, 1.5403433751251008921e-4);
    p = fma(p, f, 1.3333558200794592645e-3);
    p = fma(p, f, 9.6181291939343133551e-3);
    p = fma(p, f, 5.5504108664651672007e-2);
    p = fma(p, f, 0.2402265069564033974);
    p = fma(p, f, 0.69314718055994615897);
    p = fma(p, f, 1.0000000000000134868);
    return __hiloint2double(__double2hiint(p) + (__double2loint(z) << 20), __double2loint(p));
  }
};
__device__ __forceinline__ unsigned long long fixed(double e) {
  const double one = 512.0;  // its last bit is 2^-43
  return static_cast<unsigned long long>(__double_as_longlong(e + one) - __double_as_longlong(one));
}

constexpr int BINS = 2048;
constexpr float REACH = 20.0f;    // the bins' width is REACH / BINS; what lies farther from the largest logit is in the last one
constexpr float SLACK = 2e-5f;    // of a bin's weights: its ends are rounded, and sums of 32 bits
constexpr int DIGITS = 1024;
constexpr int LIST = 2048;        // tokens that a row's list holds
constexpr int CHUNK = 256;        // logits of one warp's round

struct SampleShared {
  union {
    unsigned bins[BINS];
    struct {
      uint32_t key[LIST];
      int at[LIST];
    } list;
  };
  unsigned count[DIGITS];  // of a digit: tokens, the two halves of their sum
  union {
    struct {
      unsigned lo[DIGITS], hi[DIGITS];
    };
    int mine[LIST];  // this CTA's part of the list, until it is gathered
  };
  unsigned long long sum[2][3][SR_CLUSTER];  // exchanged
  unsigned long long warp_sum[3][SR_WARPS];
  float warp_low[SR_WARPS], warp_up[SR_WARPS];
  unsigned long long pick_before;
  unsigned pick, pick_count;
  int first, last;  // bins between which top-p ends
  int found, listed;
};

// CACHED: the slice fits into shared memory; else it is read again and again
template <typename T, bool CACHED>
__global__ void __launch_bounds__(SR_THREADS, 2) sample_kernel(const __grid_constant__ SampleArgs a, int per) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ __align__(16) unsigned long long chunk_sum[];  // of each CHUNK of the slice; then the slice
  __shared__ SampleShared sh;
  const int start = rank * per, mine = max(0, min(per, a.vocab - start));
  const int chunks = (mine + CHUNK - 1) / CHUNK;
  const T* logits = static_cast<const T*>(a.logits) + row * a.stride + start;
  // the slice lies in shared memory as far behind a multiple of 16 bytes as in memory
  constexpr int V = 16 / int(sizeof(T));
  T* cache = reinterpret_cast<T*>(chunk_sum + ((per + CHUNK - 1) / CHUNK + 1) / 2 * 2) + int((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  // every CTA of the cluster runs before any writes into another's shared memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  auto logit = [&](int i) {
    if constexpr (CACHED) return to_f32(cache[i]);
    else return to_f32(logits[i]);
  };

  // A number of each CTA to all CTAs of the cluster (three at a time). What others may still read of the exchange before is the
  // other half of sh.sum.
  int swap = 0;
  auto exchange = [&](int i, unsigned long long v) {  // every thread the same v
    if (tid < C) cluster.map_shared_rank(&sh.sum[swap][i][0], tid)[rank] = v;
  };
  auto block_sum = [&](int i, unsigned long long v) {  // (a barrier follows)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sh.warp_sum[i][warp] = v;
  };
  auto of_warps = [&](int i) {
    unsigned long long all = 0;
#pragma unroll
    for (int w = 0; w < SR_WARPS; ++w) all += sh.warp_sum[i][w];
    return all;
  };
  auto of_cluster = [&](int i, int upto) {
    unsigned long long all = 0;
    for (int r = 0; r < upto; ++r) all += sh.sum[swap][i][r];
    return all;
  };

  // the slice, and the row's largest key with the lowest index that has it
  uint32_t best = 0;
  int best_at = 0;
  auto look = [&](float l, int i) {
    const uint32_t k = key_of(l);
    if (k > best || (k == best && i < best_at)) {
      best = k;
      best_at = i;
    }
  };
  {
    const int head = min(mine, int((16 - (reinterpret_cast<uintptr_t>(logits) & 15)) & 15) / int(sizeof(T)));
    const int words = (mine - head) / V, tail = head + words * V;
    for (int i = tid; i < head + (mine - tail); i += SR_THREADS) {
      const int at = i < head ? i : tail + i - head;
      const T x = logits[at];
      if constexpr (CACHED) cache[at] = x;
      look(to_f32(x), at);
    }
    const uint4* from = reinterpret_cast<const uint4*>(logits + head);
    for (int i0 = tid; i0 < words; i0 += 4 * SR_THREADS) {
      uint4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j * SR_THREADS < words) x[j] = __ldg(from + i0 + j * SR_THREADS);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * SR_THREADS;
        if (i < words) {
          if constexpr (CACHED) *reinterpret_cast<uint4*>(cache + head + i * V) = x[j];
          alignas(16) T e[V];
          *reinterpret_cast<uint4*>(e) = x[j];
#pragma unroll
          for (int q = 0; q < V; ++q) look(to_f32(e[q]), head + i * V + q);
        }
      }
    }
    // larger keys first, then lower indices
    unsigned long long v = (static_cast<unsigned long long>(best) << 32) | uint32_t(~(start + best_at));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long x = __shfl_xor_sync(0xffffffffu, v, o);
      v = x > v ? x : v;
    }
    if (lane == 0) sh.warp_sum[0][warp] = v;
    for (int i = tid; i < BINS; i += SR_THREADS) sh.bins[i] = 0;
    if (tid == 0) {
      sh.first = sh.last = BINS - 1;
      sh.listed = 0;
      sh.pick = BINS;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SR_WARPS; ++w) v = sh.warp_sum[0][w] > v ? sh.warp_sum[0][w] : v;
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    exchange(0, v);
    cluster.sync();
    for (int r = 0; r < C; ++r) v = sh.sum[swap][0][r] > v ? sh.sum[swap][0][r] : v;
    best = uint32_t(v >> 32);
    best_at = int(~uint32_t(v));
  }
  float* probs = a.probs ? a.probs + row * a.probs_stride + start : nullptr;
  const float temp = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  if (best == 0 || !(temp > 0.0f)) {  // no candidates, or the largest logit's token
    if (rank == 0 && tid == 0) {
      a.tokens[row] = best == 0 ? -1 : best_at;
      if (best == 0 && a.status) atomicOr(a.status, uint32_t(ST_BAD_PROBS));
    }
    if (probs)
      for (int i = tid; i < mine; i += SR_THREADS) probs[i] = best != 0 && start + i == best_at ? 1.0f : 0.0f;
    return;
  }
  const float top = __uint_as_float(best & 0x80000000u ? best & 0x7fffffffu : ~best);
  const Weights w{double(top), 1.4426950408889634074 / double(temp)};
  const int top_k = a.top_k ? __ldg(a.top_k + row) : 0;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : 1.0f, min_p = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  const bool by_k = top_k > 0 && top_k < a.vocab, by_p = top_p < 1.0f;
  const double least = min_p > 0.0f ? fmin(double(min_p), 1.0) : 0.0;
  const float per_bin = float(BINS) / REACH / temp;
  // (infinite logits: all others are in the last bin; a temperature without end: all in the first)
  auto bin_of = [&](float l) { return l == top ? 0 : int(fminf((top - l) * per_bin, float(BINS - 1))); };
  // the last bin in which min-p leaves something
  const int least_bin = least > 0.0 ? int(fminf(-logf(float(least)) * (float(BINS) / REACH) * (1.0f + SLACK), float(BINS - 1))) + 1 : BINS;

  // What is kept: `kept`, of bins up to max_bin. Bins below sure are kept whole.
  Kept kept{1u, INT_MAX};
  int max_bin = BINS - 1, sure = BINS;
  auto weight = [&](int i) {
    const float l = logit(i);
    const uint32_t k = key_of(l);
    const int b = bin_of(l);
    if (!k || b > max_bin || b > least_bin || !(b < sure || kept.has(k, start + i))) return 0.0;
    const double e = w.of(l);
    return e >= least ? e : 0.0;
  };

  // Digits, counted (and summed) here or over all CTAs: the first from the top with which they reach the goal, into sh.pick ..
  auto pick = [&](bool over_all, bool by_weight, unsigned long long before, double goal) {
    static_assert(DIGITS == 2 * SR_THREADS, "two digits a thread");
    const int d = DIGITS - 2 - 2 * tid;  // the thread's second one
    unsigned cnt[2] = {0, 0};
    unsigned long long mass[2] = {0, 0};
    for (int r = over_all ? 0 : rank; r < (over_all ? C : rank + 1); ++r) {
      const uint2 n = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.count, r) + d);
      cnt[0] += n.y;
      cnt[1] += n.x;
      if (by_weight) {
        const uint2 lo = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.lo, r) + d);
        const uint2 hi = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.hi, r) + d);
        mass[0] += (static_cast<unsigned long long>(hi.y) << 32) + lo.y;
        mass[1] += (static_cast<unsigned long long>(hi.x) << 32) + lo.x;
      }
    }
    if (!by_weight) {
      mass[0] = cnt[0];
      mass[1] = cnt[1];
    }
    const unsigned long long own = mass[0] + mass[1];
    unsigned long long inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) sh.warp_sum[0][warp] = inc;
    __syncthreads();
    unsigned long long prev = before + inc - own;
    for (int x = 0; x < warp; ++x) prev += sh.warp_sum[0][x];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (double(prev) < goal && double(prev + mass[j]) >= goal) {  // one digit: the goal lies above what is before and not above all
        sh.pick = unsigned(d + 1 - j);
        sh.pick_count = cnt[j];
        sh.pick_before = prev;
      }
      prev += mass[j];
    }
    __syncthreads();
  };

  // Among keys that each() goes through, `bits` of them not known to be the same (the others: prefix), the one with which, from the largest
  // on, the count or the sum of `before` and theirs reaches the goal; in sh.pick_before what comes before it, in sh.pick_count how many there are.
  auto select = [&](auto&& each, bool over_all, uint32_t prefix, int bits, bool by_weight, unsigned long long before, double goal) {
    for (int known = 32 - bits; known < 32;) {
      const int shift = max(0, 32 - known - 10);
      const uint32_t above = known ? ~0u << (32 - known) : 0u;
      if (over_all) cluster.sync();  // the counts before were read
      else __syncthreads();
      for (int i = tid; i < DIGITS; i += SR_THREADS) sh.count[i] = sh.lo[i] = sh.hi[i] = 0;
      __syncthreads();
      each([&](uint32_t k, float l) {
        if ((k & above) != prefix) return;
        const unsigned d = (k & ~above) >> shift;
        atomicAdd(&sh.count[d], 1u);
        if (by_weight) {
          const unsigned long long f = fixed(w.of(l));
          const unsigned lo = unsigned(f), old = atomicAdd(&sh.lo[d], lo);
          atomicAdd(&sh.hi[d], unsigned(f >> 32) + (old + lo < old ? 1u : 0u));
        }
      });
      if (over_all) cluster.sync();
      else __syncthreads();
      pick(over_all, by_weight, before, goal);
      prefix |= sh.pick << shift;
      before = sh.pick_before;
      known = 32 - shift;
    }
    return prefix;
  };
  // of the tokens at that key, how many it takes
  auto take_of = [&](uint32_t key, bool by_weight, double goal) {
    const double left = goal - double(sh.pick_before);
    if (!by_weight) return unsigned(left);
    const double e = double(fixed(w.of(__uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key))));
    const double need = ceil(left / e);
    return need >= double(sh.pick_count) || !(e > 0.0) ? sh.pick_count : need > 1.0 ? unsigned(need) : 1u;
  };

  // ---- bins: where top-k and top-p end ----
  int k_bin = BINS, above_k = 0;  // top-k's bin, tokens above it
  bool whole = true;              // all of that bin is kept
  int first = BINS, last = -1;    // top-p ends in these bins
  const double p = fmax(double(top_p), 0.0);
  if (by_k || by_p) {
    for (int i = tid; i < mine; i += SR_THREADS) {
      const float l = logit(i);
      if (key_of(l)) atomicAdd(&sh.bins[bin_of(l)], 1u);
    }
    cluster.sync();
    constexpr int PER = BINS / SR_THREADS;
    static_assert(PER == 4, "four bins a thread");
    unsigned cnt[PER] = {0, 0, 0, 0};
    for (int r = 0; r < C; ++r) {
      const uint4 n = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.bins, r) + PER * tid);
      cnt[0] += n.x;
      cnt[1] += n.y;
      cnt[2] += n.z;
      cnt[3] += n.w;
    }
    if (by_k) {
      const unsigned own = cnt[0] + cnt[1] + cnt[2] + cnt[3];
      unsigned inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      if (lane == 31) sh.warp_sum[0][warp] = inc;
      __syncthreads();
      unsigned prev = inc - own;
      for (int x = 0; x < warp; ++x) prev += unsigned(sh.warp_sum[0][x]);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (prev < unsigned(top_k) && prev + cnt[j] >= unsigned(top_k)) {
          sh.pick = unsigned(PER * tid + j);
          sh.pick_before = prev;
          sh.pick_count = cnt[j];
        }
        prev += cnt[j];
      }
      __syncthreads();
      k_bin = int(sh.pick);  // BINS: there are fewer tokens
      if (k_bin < BINS) {
        above_k = int(sh.pick_before);
        whole = above_k + int(sh.pick_count) == top_k;
        max_bin = k_bin;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (PER * tid + j > k_bin) cnt[j] = 0;
          if (PER * tid + j == k_bin) cnt[j] = unsigned(top_k - above_k);
        }
      }
    }
    if (by_p) {
      // lower and upper bounds of the weights up to and with each bin, and of those after it
      float low[PER], up[PER], low_inc = 0.0f, up_inc = 0.0f;
      const float width = REACH / float(BINS) * 1.44269504f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int b = PER * tid + j;
        up[j] = float(cnt[j]) * exp2f(-width * float(b)) * (1.0f + SLACK);
        low[j] = b == BINS - 1 ? 0.0f : float(cnt[j]) * exp2f(-width * float(b + 1)) * (1.0f - SLACK);
        low_inc += low[j];
        up_inc += up[j];
      }
      float low_sum = low_inc, up_sum = up_inc;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float x = __shfl_up_sync(0xffffffffu, low_sum, o), y = __shfl_up_sync(0xffffffffu, up_sum, o);
        if (lane >= o) {
          low_sum += x;
          up_sum += y;
        }
      }
      if (lane == 31) {
        sh.warp_low[warp] = low_sum;
        sh.warp_up[warp] = up_sum;
      }
      __syncthreads();
      float low_all = 0.0f, up_all = 0.0f, l = low_sum - low_inc, u = up_sum - up_inc;
#pragma unroll
      for (int x = 0; x < SR_WARPS; ++x) {
        if (x < warp) {
          l += sh.warp_low[x];
          u += sh.warp_up[x];
        }
        low_all += sh.warp_low[x];
        up_all += sh.warp_up[x];
      }
      // the end is in the first bin at which (sum so far) (1 - p) >= p (sum after it)
      const float q = float(p), q1 = float(1.0 - p);
      int may = BINS - 1, must = BINS - 1;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        l += low[j];
        u += up[j];
        if (u * q1 * (1.0f + SLACK) >= q * fmaxf(low_all - l, 0.0f) * (1.0f - SLACK)) may = min(may, PER * tid + j);
        if (l * q1 * (1.0f - SLACK) >= q * fmaxf(up_all - u, 0.0f) * (1.0f + SLACK) + SLACK * up_all) must = min(must, PER * tid + j);
      }
      may = int(__reduce_min_sync(0xffffffffu, unsigned(may)));
      must = int(__reduce_min_sync(0xffffffffu, unsigned(must)));
      if (lane == 0) {
        atomicMin(&sh.first, may);
        atomicMin(&sh.last, must);
      }
      __syncthreads();
      last = min(sh.last, max_bin);
      first = min(sh.first, last);
    }
    sure = by_p ? first : whole ? max_bin + 1 : k_bin;
  }

  // ---- one pass: weights, sums of the sure tokens by chunks, the others listed ----
  unsigned long long sum_above = 0, sum_between = 0;  // above top-p's bins; between them and top-k's end
  for (int c = warp; c < chunks; c += SR_WARPS) {
    unsigned long long v = 0;
#pragma unroll 4
    for (int e = 0; e < CHUNK / 32; ++e) {
      const int i = c * CHUNK + 32 * e + lane;
      if (i >= mine) continue;
      const float l = logit(i);
      const int b = bin_of(l);
      if (!key_of(l) || b > max_bin) continue;
      if ((b >= first && b <= last) || (b == k_bin && !whole)) {
        const int at = atomicAdd(&sh.listed, 1);
        if (at < LIST) sh.mine[at] = i;
      } else if (by_p || b <= least_bin) {
        const double x = w.of(l);
        const unsigned long long f = fixed(x);
        if (b < sure && x >= least) v += f;
        if (b < first) sum_above += f;
        else sum_between += f;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) chunk_sum[c] = v;
  }

  if (by_p || !whole) {
    block_sum(0, sum_above);
    block_sum(1, sum_between);
    __syncthreads();
    const int listed = sh.listed;
    swap ^= 1;
    exchange(0, of_warps(0));
    exchange(1, of_warps(1));
    exchange(2, listed);
    cluster.sync();
    sum_above = of_cluster(0, C);
    sum_between = of_cluster(1, C);
    const unsigned long long total = of_cluster(2, C);
    bool fits = total <= LIST;
    if (fits) {
      // the lists to every CTA, one behind the other
      const int before = int(of_cluster(2, rank)), n = int(total);
      for (int j = tid; j < listed; j += SR_THREADS) {
        const int i = sh.mine[j];
        const uint32_t k = key_of(logit(i));
        for (int r = 0; r < C; ++r) {
          cluster.map_shared_rank(sh.list.key, r)[before + j] = k;
          cluster.map_shared_rank(sh.list.at, r)[before + j] = start + i;
        }
      }
      cluster.sync();
      auto value = [](uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); };
      auto each_listed = [&](int from, int to, auto&& f) {
        for (int j = tid; j < n; j += SR_THREADS) {
          const uint32_t k = sh.list.key[j];
          const float l = value(k);
          const int b = bin_of(l);
          if (b >= from && b <= to && (b != k_bin || kept.has(k, sh.list.at[j]))) f(k, l);
        }
      };
      // the end among those of bins from .. to
      auto end_in = [&](int from, int to, bool by_weight, unsigned long long done, double goal) {
        // bits that are not the same in all of them
        uint32_t all1 = ~0u, any1 = 0;
        each_listed(from, to, [&](uint32_t k, float) {
          all1 &= k;
          any1 |= k;
        });
        all1 = __reduce_and_sync(0xffffffffu, all1);
        any1 = __reduce_or_sync(0xffffffffu, any1);
        __syncthreads();
        if (lane == 0) sh.warp_sum[0][warp] = (static_cast<unsigned long long>(all1) << 32) | any1;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < SR_WARPS; ++x) {
          all1 &= uint32_t(sh.warp_sum[0][x] >> 32);
          any1 |= uint32_t(sh.warp_sum[0][x]);
        }
        const int bits = max(1, 32 - __clz(int(all1 ^ any1)));
        const uint32_t key = select([&](auto&& f) { each_listed(from, to, f); }, false, bits == 32 ? 0u : any1 & (~0u << bits), bits, by_weight, done, goal);
        const unsigned take = take_of(key, by_weight, goal);
        Kept end{key, INT_MAX};
        if (take < sh.pick_count) {  // equal logits: those of the lowest indices, which are the largest when turned round
          end.last = int(~select(
              [&](auto&& f) {
                for (int j = tid; j < n; j += SR_THREADS)
                  if (sh.list.key[j] == key && kept.has(key, sh.list.at[j])) f(~uint32_t(sh.list.at[j]), 0.0f);
              },
              false, ~0u << 20, 20, false, 0, double(take)));
        }
        return end;
      };
      if (!whole) kept = end_in(k_bin, k_bin, false, above_k, double(top_k));
      if (by_p) {
        unsigned long long v = 0, in_bins = 0;
        each_listed(0, BINS - 1, [&](uint32_t, float l) { v += fixed(w.of(l)); });
        if (k_bin > last) each_listed(first, last, [&](uint32_t, float l) { in_bins += fixed(w.of(l)); });
        __syncthreads();
        block_sum(0, v);
        block_sum(1, in_bins);
        __syncthreads();
        v = of_warps(0);
        in_bins = k_bin > last ? of_warps(1) : v;
        const double goal = fmax(1.0, p * double(sum_above + sum_between + v));
        if (double(sum_above) < goal && double(sum_above + in_bins) >= goal)
          kept = stricter(kept, end_in(first, last, true, sum_above, goal));
        else
          fits = false;
      }
      if (fits) {  // what is kept of the CTA's own to its chunks
        __syncthreads();
        for (int j = before + tid; j < before + listed; j += SR_THREADS) {
          const uint32_t k = sh.list.key[j];
          const int at = sh.list.at[j];
          if (!kept.has(k, at)) continue;
          const double x = w.of(value(k));
          if (x >= least) atomicAdd(&chunk_sum[(at - start) / CHUNK], fixed(x));
        }
        __syncthreads();
      }
    }
    if (!fits) {
      // the whole row, digit by digit, then its chunks again
      kept = Kept{1u, INT_MAX};
      max_bin = BINS - 1;
      sure = 0;
      auto each_of_slice = [&](auto&& f) {
        for (int i = tid; i < mine; i += SR_THREADS) {
          const float l = logit(i);
          const uint32_t k = key_of(l);
          if (k && kept.has(k, start + i)) f(k, l);
        }
      };
      auto end_of_row = [&](bool by_weight, double goal) {
        const uint32_t key = select(each_of_slice, true, 0u, 32, by_weight, 0, goal);
        const unsigned take = take_of(key, by_weight, goal);
        Kept end{key, INT_MAX};
        if (take < sh.pick_count)
          end.last = int(~select(
              [&](auto&& f) {
                for (int i = tid; i < mine; i += SR_THREADS)
                  if (key_of(logit(i)) == key && kept.has(key, start + i)) f(~uint32_t(start + i), 0.0f);
              },
              true, ~0u << 20, 20, false, 0, double(take)));
        return end;
      };
      if (k_bin < BINS) kept = end_of_row(false, double(top_k));
      if (by_p) {
        unsigned long long v = 0;
        each_of_slice([&](uint32_t, float l) { v += fixed(w.of(l)); });
        __syncthreads();
        block_sum(0, v);
        __syncthreads();
        swap ^= 1;
        exchange(0, of_warps(0));
        cluster.sync();
        kept = stricter(kept, end_of_row(true, fmax(1.0, p * double(of_cluster(0, C)))));
      }
      for (int c = warp; c < chunks; c += SR_WARPS) {
        unsigned long long v = 0;
#pragma unroll 4
        for (int e = 0; e < CHUNK / 32; ++e) {
          const int i = c * CHUNK + 32 * e + lane;
          if (i < mine) v += fixed(weight(i));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) chunk_sum[c] = v;
      }
    }
  }

  // ---- the draw ----
  __syncthreads();
  unsigned long long acc = 0;
  for (int c = tid; c < chunks; c += SR_THREADS) acc += chunk_sum[c];
  block_sum(0, acc);
  __syncthreads();
  swap ^= 1;
  exchange(0, of_warps(0));
  cluster.sync();
  const unsigned long long before = of_cluster(0, rank), own = sh.sum[swap][0][rank], all = of_cluster(0, C);
  float u = __ldg(a.u + row);
  u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
  const double goal = double(u) * double(all);
  // the CTA whose slice passes the goal (the sum of all does), in it the chunk, in it the token
  if (warp == 0 && double(before) <= goal && double(before + own) > goal) {
    unsigned long long base = before;
    int chunk = -1;
    for (int c0 = 0; chunk < 0; c0 += 32) {
      const unsigned long long v = c0 + lane < chunks ? chunk_sum[c0 + lane] : 0;
      unsigned long long inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, double(base + inc) > goal);
      const int at = hit ? __ffs(int(hit)) - 1 : 31;
      if (hit) chunk = c0 + at;
      base += __shfl_sync(0xffffffffu, hit ? inc - v : inc, at);
    }
    for (int e = 0; e < CHUNK / 32; ++e) {
      const int i = chunk * CHUNK + 32 * e + lane;
      unsigned long long inc = i < mine ? fixed(weight(i)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, double(base + inc) > goal);
      if (hit) {
        if (lane == 0) a.tokens[row] = start + chunk * CHUNK + 32 * e + __ffs(int(hit)) - 1;
        break;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  if (probs) {
    const double inv = 1.0 / (double(all) * (1.0 / double(1ull << FIX)));
    for (int i = tid; i < mine; i += SR_THREADS) probs[i] = float(weight(i) * inv);
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
  // bytes of a CTA's chunk sums, and of its slice (which may begin up to 16 bytes late)
  auto slice = [&](int c) { return (a.vocab + c - 1) / c; };
  auto sums = [&](int c) { return sizeof(unsigned long long) * size_t(((slice(c) + CHUNK - 1) / CHUNK + 1) / 2 * 2); };
  auto bytes = [&](int c) { return sums(c) + size_t(slice(c)) * sizeof(T) + 16; };
  // CTAs of a row: until there are two for each SM, with slices of at least 1024 logits; more where an SM does not hold two slices
  int c = 1;
  while (c < SR_CLUSTER && ((a.n_rows * c < 2 * SMS && a.vocab / (2 * c) >= 1024) || bytes(c) > size_t(SR_CACHE_TWO))) c *= 2;
  if (bytes(c) <= size_t(SR_CACHE)) return run_sample<T, true>(a, c, slice(c), bytes(c), s);
  return run_sample<T, false>(a, c, slice(c), sums(c), s);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int kind, cudaStream_t s) {
  return kind == E_F16 ? run_sample<__half>(a, s) : kind == E_BF16 ? run_sample<__nv_bfloat16>(a, s) : run_sample<float>(a, s);
}

}  // namespace paged
}  // namespace wcb
