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
constexpr int SR_CACHE = 176 * 1024;     // bytes of a slice in shared memory at most
constexpr int SR_CACHE_TWO = 66 * 1024;  // so that an SM holds two
constexpr int FIX = 43;                  // bits after the point
constexpr int BINS = 2048;
constexpr float REACH = 20.0f;  // the bins' width is REACH / BINS; what lies farther from the largest logit is in the last one
constexpr float SLACK = 2e-5f;  // of a bin's weights: its ends are rounded, and sums of 32 bits
constexpr float BIN0 = 8388608.0f;  // 2^23: bins as floats, BIN0 + number, so that adding BIN0 rounds to a whole one
constexpr int DIGITS = 1024;
constexpr int LIST = 4096;  // tokens that a row's list holds, an equal part for each CTA
constexpr int CHUNK = 256;  // logits of one warp's round, 8 a lane

// order-preserving bits of a number (-0 is 0)
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// What a filter leaves: logits above `at`, and those at it up to index `last`.
struct Cut {
  float at;
  int last;
  __device__ __forceinline__ bool has(float l, int i) const { return l > at || (l == at && i <= last); }
};
__device__ __forceinline__ Cut stricter(const Cut& a, const Cut& b) {
  return a.at != b.at ? (a.at > b.at ? a : b) : (a.last < b.last ? a : b);
}

struct Weights {
  double top, rate;  // the largest logit; log2(e) / T
  // a logit of at most `top` and at least 60 / rate below it. (Without branches: several of them are computed side by side.)
  __device__ __forceinline__ double of(float l) const {
    constexpr double BIG = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double d = double(fminf(l, FLT_MAX)) - top;
    const double z = fma(d, rate, BIG);
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
    p = fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(z) << 20), __double2loint(p));
  }
};
__device__ __forceinline__ unsigned long long fixed(double e) {
  const double one = 512.0;  // its last bit is 2^-43
  return static_cast<unsigned long long>(__double_as_longlong(e + one) - __double_as_longlong(one));
}

struct SampleShared {
  uint2 list[LIST];  // logit, index
  unsigned count[DIGITS], hi[DIGITS];  // of a digit: tokens, the halves of their sum
  union {
    unsigned lo[DIGITS];
    unsigned bins[BINS / 2];  // two counts of 16 bits in a word
  };
  unsigned long long sum[2][3][SR_CLUSTER];  // exchanged
  unsigned long long warp_sum[3][SR_WARPS];
  float warp_low[SR_WARPS], warp_up[SR_WARPS];
  unsigned long long pick_before;
  unsigned pick, pick_count;
  int first, last;  // bins between which top-p ends
  int listed;
};

// Places of a slice in shared memory: as far behind a multiple of 16 bytes as in memory, filled up with -infinity to whole chunks.
template <typename T>
__host__ __device__ constexpr int places(int per) {
  return (per + 16 / int(sizeof(T)) - 1 + CHUNK - 1) / CHUNK * CHUNK;
}

// CACHED: the slice fits into shared memory; else it is read again and again
template <typename T, bool CACHED>
__global__ void __launch_bounds__(SR_THREADS, 2) sample_kernel(const __grid_constant__ SampleArgs a, int per) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ __align__(16) unsigned long long chunk_sum[];  // of each chunk of the slice; then the slice
  __shared__ SampleShared sh;
  constexpr int V = 16 / int(sizeof(T));
  const int begin = rank * per, mine = max(0, min(per, a.vocab - begin));
  const T* slice = static_cast<const T*>(a.logits) + row * a.stride + begin;
  const int shift = int((reinterpret_cast<uintptr_t>(slice) & 15) / sizeof(T));
  const int chunks = mine > 0 ? (shift + mine + CHUNK - 1) / CHUNK : 0;
  const int start = begin - shift;  // index of place 0
  T* cache = reinterpret_cast<T*>(chunk_sum + (places<T>(per) / CHUNK + 1) / 2 * 2);
  // every CTA of the cluster runs before any writes into another's shared memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  auto logit = [&](int at) {
    if constexpr (CACHED) return to_f32(cache[at]);
    else return at >= shift && at < shift + mine ? to_f32(slice[at - shift]) : -INFINITY;
  };
  // a lane's 8 logits of a chunk, and where they lie
  auto place = [&](int c, int j) { return c * CHUNK + (sizeof(T) == 4 ? 128 * (j / 4) + 4 * lane + j % 4 : 8 * lane + j); };
  auto eight = [&](int c, float (&l)[8]) {
    if constexpr (CACHED) {
      alignas(16) T e[8];
#pragma unroll
      for (int j = 0; j < 8; j += V) *reinterpret_cast<uint4*>(e + j) = *reinterpret_cast<const uint4*>(cache + place(c, j));
#pragma unroll
      for (int j = 0; j < 8; ++j) l[j] = to_f32(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) l[j] = logit(place(c, j));
    }
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
  auto block_max = [&](unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long x = __shfl_xor_sync(0xffffffffu, v, o);
      v = x > v ? x : v;
    }
    if (lane == 0) sh.warp_sum[0][warp] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SR_WARPS; ++w) v = sh.warp_sum[0][w] > v ? sh.warp_sum[0][w] : v;
    return v;
  };

  // ---- the slice, and the row's largest logit ----
  float top = -INFINITY;
  {
    const int head = shift ? min(mine, V - shift) : 0, words = (mine - head) / V, tail = head + words * V;
    for (int i = tid; i < head + (mine - tail); i += SR_THREADS) {
      const int at = i < head ? i : tail + i - head;
      const T x = slice[at];
      if constexpr (CACHED) cache[shift + at] = x;
      top = fmaxf(top, to_f32(x));  // (the number, where the other is NaN)
    }
    if constexpr (CACHED) {
      for (int at = tid; at < shift + chunks * CHUNK - (shift + mine); at += SR_THREADS)
        cache[at < shift ? at : mine + at] = from_f32<T>(-INFINITY);
    }
    const uint4* from = reinterpret_cast<const uint4*>(slice + head);
    constexpr int AHEAD = 8;
    for (int i0 = tid; i0 < words; i0 += AHEAD * SR_THREADS) {
      uint4 x[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (i0 + j * SR_THREADS < words) x[j] = __ldg(from + i0 + j * SR_THREADS);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int i = i0 + j * SR_THREADS;
        if (i < words) {
          if constexpr (CACHED) *reinterpret_cast<uint4*>(cache + shift + head + i * V) = x[j];
          alignas(16) T e[V];
          *reinterpret_cast<uint4*>(e) = x[j];
#pragma unroll
          for (int q = 0; q < V; ++q) top = fmaxf(top, to_f32(e[q]));
        }
      }
    }
    for (int i = tid; i < BINS / 2; i += SR_THREADS) sh.bins[i] = 0;
    if (tid == 0) {
      sh.first = sh.last = BINS - 1;
      sh.listed = 0;
      sh.pick = BINS;
    }
    const unsigned long long v = block_max(key_of(top));
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    exchange(0, v);
    cluster.sync();
    unsigned long long best = v;
    for (int r = 0; r < C; ++r) best = sh.sum[swap][0][r] > best ? sh.sum[swap][0][r] : best;
    top = value_of(uint32_t(best));
  }
  float* probs = a.probs ? a.probs + row * a.probs_stride + start : nullptr;
  const bool some = top > -INFINITY;
  const float temp = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  if (!some || !(temp > 0.0f)) {  // no candidates, or the largest logit's token: the lowest index that has it
    int at = INT_MAX;
    if (some)
      for (int c = warp; c < chunks; c += SR_WARPS) {
        float l[8];
        eight(c, l);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (l[j] == top) at = min(at, start + place(c, j));
      }
    __syncthreads();
    const unsigned long long v = block_max(~uint32_t(at));
    swap ^= 1;
    exchange(0, v);
    cluster.sync();
    unsigned long long lowest = v;
    for (int r = 0; r < C; ++r) lowest = sh.sum[swap][0][r] > lowest ? sh.sum[swap][0][r] : lowest;
    const int token = some ? int(~uint32_t(lowest)) : -1;
    if (rank == 0 && tid == 0) {
      a.tokens[row] = token;
      if (!some && a.status) atomicOr(a.status, uint32_t(ST_BAD_PROBS));
    }
    if (probs)
      for (int i = shift + tid; i < shift + mine; i += SR_THREADS) probs[i] = start + i == token ? 1.0f : 0.0f;
    return;
  }
  const float ceiling = fminf(top, FLT_MAX);
  const Weights w{double(ceiling), 1.4426950408889634074 / double(temp)};
  const int top_k = a.top_k ? __ldg(a.top_k + row) : 0;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : 1.0f, min_p = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  const bool by_k = top_k > 0 && top_k < a.vocab, by_p = top_p < 1.0f;
  const double least = min_p > 0.0f ? fmin(double(min_p), 1.0) : 0.0;
  // candidates (NaN is none): where there are infinities, only they; weights below 2^-59 count as none
  const float lowest = top > FLT_MAX ? INFINITY : -FLT_MAX;
  const float faint = fmaxf(lowest, ceiling - 41.0f * temp);
  // A logit's bin, as BIN0 + number: one that is larger is in the same bin or an earlier one.
  const float per_bin = fminf(float(BINS) / REACH / temp, 1e30f), of_top = ceiling * per_bin;
  auto bin_of = [&](float l) { return fminf(fmaf(-l, per_bin, of_top), float(BINS - 1)) + BIN0; };
  auto number = [](float bin) { return int(__float_as_uint(bin) & (BINS - 1)); };
  // (16 bits count a slice's; of_top's rounding is to be far below a bin)
  const bool binned = per < 65536 && top <= FLT_MAX && fabsf(of_top) <= 65536.0f;

  // What is kept: bins up to sure (as bin_of gives them), and what cut has; of both, what min-p leaves.
  float sure = 2.0f * BIN0;  // all
  Cut cut{INFINITY, -1};     // none
  auto keeps = [&](float l, int at) { return l >= faint && (bin_of(l) <= sure || cut.has(l, start + at)); };

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
      if (mass[j] > 0 && double(prev) < goal && double(prev + mass[j]) >= goal) {  // one digit: the goal lies above what is before and not above all
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
      const int low = max(0, 32 - known - 10);
      const uint32_t above = known ? ~0u << (32 - known) : 0u;
      if (over_all) cluster.sync();  // the counts before were read
      else __syncthreads();
      for (int i = tid; i < DIGITS; i += SR_THREADS) sh.count[i] = sh.lo[i] = sh.hi[i] = 0;
      __syncthreads();
      each([&](uint32_t k, unsigned long long f) {
        if ((k & above) != prefix) return;
        const unsigned d = (k & ~above) >> low;
        atomicAdd(&sh.count[d], 1u);
        if (by_weight) {
          const unsigned x = unsigned(f), old = atomicAdd(&sh.lo[d], x);
          atomicAdd(&sh.hi[d], unsigned(f >> 32) + (old + x < old ? 1u : 0u));
        }
      });
      if (over_all) cluster.sync();
      else __syncthreads();
      pick(over_all, by_weight, before, goal);
      prefix |= sh.pick << low;
      before = sh.pick_before;
      known = 32 - low;
    }
    return prefix;
  };
  // of the tokens at that key, how many it takes
  auto take_of = [&](uint32_t key, bool by_weight, double goal) {
    const double left = goal - double(sh.pick_before);
    if (!by_weight) return unsigned(left);
    const double need = ceil(left / double(fixed(w.of(value_of(key)))));
    return need >= double(sh.pick_count) ? sh.pick_count : need > 1.0 ? unsigned(need) : 1u;
  };

  // ---- bins: where top-k and top-p end ----
  int k_bin = BINS, above_k = 0;  // top-k's bin, tokens above it
  bool whole = true;              // all of that bin is kept
  int first = BINS, last = -1;    // top-p ends in these bins
  const double p = fmax(double(top_p), 0.0);
  if ((by_k || by_p) && binned) {
    for (int c = warp; c < chunks; c += SR_WARPS) {
      float l[8];
      eight(c, l);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int b = number(bin_of(l[j]));
        if (l[j] >= lowest) atomicAdd(&sh.bins[b >> 1], 1u << (16 * (b & 1)));
      }
    }
    cluster.sync();
    constexpr int PER = BINS / SR_THREADS;
    static_assert(PER == 4, "four bins a thread");
    unsigned cnt[PER] = {0, 0, 0, 0};
    for (int r = 0; r < C; ++r) {
      const uint2 n = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.bins, r) + 2 * tid);
      cnt[0] += n.x & 0xffffu;
      cnt[1] += n.x >> 16;
      cnt[2] += n.y & 0xffffu;
      cnt[3] += n.y >> 16;
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
        const int b = PER * tid + j;  // logits of b - 1/2 to b + 1/2 widths
        up[j] = float(cnt[j]) * exp2f(-width * fmaxf(float(b) - 0.5f, 0.0f)) * (1.0f + SLACK);
        low[j] = b == BINS - 1 ? 0.0f : float(cnt[j]) * exp2f(-width * (float(b) + 0.5f)) * (1.0f - SLACK);
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
      last = min(sh.last, k_bin);
      first = min(sh.first, last);
    }
    const int end = by_p ? first : whole ? min(k_bin + 1, BINS) : k_bin;  // bins before it are kept whole
    sure = BIN0 + float(end - 1);
  }

  // ---- one pass: weights, sums of the sure tokens by chunks, the others listed ----
  const bool lists = (by_p || !whole) && binned;
  const int room = LIST / C;
  unsigned long long sum_all = 0, sum_above = 0;  // of what is not listed; of that, above top-p's bins
  if (binned || !(by_k || by_p)) {
    uint2* list = sh.list + rank * room;
    const float k_at = BIN0 + float(k_bin), k_end = by_k && k_bin < BINS ? k_at : 2.0f * BIN0;
    const float list_from = by_p ? BIN0 + float(first) : k_at, list_to = by_p ? BIN0 + float(last) : whole ? 0.0f : k_at;
    const float k_list = !whole ? k_at : 0.0f;
    // the last bin whose weights are wanted: of the sure ones, those that min-p may leave; with top-p all
    const float least_bin = least > 0.0 ? fminf(BIN0 + ceilf(-logf(float(least)) * (float(BINS) / REACH) * (1.0f + SLACK)) + 2.0f, 2.0f * BIN0) : 2.0f * BIN0;
    const float wanted = !binned ? 2.0f * BIN0 : by_p ? k_end : fminf(sure, least_bin);
    for (int c = warp; c < chunks; c += SR_WARPS) {
      unsigned long long v = 0;
      float l[8];
      eight(c, l);
#pragma unroll
      for (int half = 0; half < 8; half += 4) {
        bool on[4], sures[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = l[half + j], b = bin_of(x);
          bool listed = false;
          if (lists) listed = x >= lowest && ((b >= list_from && b <= list_to) || b == k_list);
          if (listed) {
            const int at = atomicAdd(&sh.listed, 1);
            if (at < room) list[at] = make_uint2(__float_as_uint(x), unsigned(start + place(c, half + j)));
          }
          on[j] = x >= faint && b <= wanted && !listed;
          sures[j] = b <= sure;
        }
        if (__any_sync(0xffffffffu, on[0] || on[1] || on[2] || on[3])) {
          double x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = w.of(l[half + j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned long long f = on[j] ? fixed(x[j]) : 0;
            sum_all += f;
            if (sures[j]) {
              if (least > 0.0) {  // (for all threads alike)
                sum_above += f;
                if (x[j] >= least) v += f;
              } else {
                v += f;
              }
            }
          }
        }
      }
      if (!(least > 0.0)) sum_above += v;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) chunk_sum[c] = v;
    }
  }

  bool fits = binned || !(by_k || by_p);
  if (lists) {
    block_sum(0, sum_above);
    block_sum(1, sum_all);
    __syncthreads();
    // sums and lists to every CTA
    const int listed = min(sh.listed, room);
    swap ^= 1;
    exchange(0, of_warps(0));
    exchange(1, of_warps(1));
    exchange(2, sh.listed);
    for (int j = tid; j < listed; j += SR_THREADS) {
      const uint2 x = sh.list[rank * room + j];
      for (int r = 1; r < C; ++r) cluster.map_shared_rank(sh.list, (rank + r) % C)[rank * room + j] = x;
    }
    cluster.sync();
    sum_above = of_cluster(0, C);
    sum_all = of_cluster(1, C);
    int n = 0;
    for (int r = 0; r < C; ++r) {
      n += int(sh.sum[swap][2][r]);
      fits = fits && sh.sum[swap][2][r] <= unsigned(room);
    }
    if (fits) {
      struct Item {
        float l;
        int at, bin;
        unsigned long long weight;
      };
      auto item = [&](int j) {
        int r = 0;
        for (; j >= int(sh.sum[swap][2][r]); ++r) j -= int(sh.sum[swap][2][r]);
        const uint2 x = sh.list[r * room + j];
        const float l = __uint_as_float(x.x);
        return Item{l, int(x.y), number(bin_of(l)), l >= faint ? fixed(w.of(l)) : 0};
      };
      const Item own = tid < n ? item(tid) : Item{0.0f, 0, 0, 0};
      auto each_listed = [&](auto&& f) {
        if (tid < n && (own.bin != k_bin || whole || cut.has(own.l, own.at))) f(own);
        for (int j = tid + SR_THREADS; j < n; j += SR_THREADS) {
          const Item x = item(j);
          if (x.bin != k_bin || whole || cut.has(x.l, x.at)) f(x);
        }
      };
      // the end among those of bins from .. to; same: the bits that are in all of their keys, and those that are in any
      auto end_in = [&](int from, int to, unsigned long long same, bool by_weight, unsigned long long done, double goal) {
        const uint32_t any1 = uint32_t(same);
        const int bits = max(1, 32 - __clz(int(uint32_t(same >> 32) ^ any1)));
        const uint32_t key = select(
            [&](auto&& f) {
              each_listed([&](const Item& x) {
                if (x.bin >= from && x.bin <= to) f(key_of(x.l), x.weight);
              });
            },
            false, bits == 32 ? 0u : any1 & (~0u << bits), bits, by_weight, done, goal);
        const unsigned take = take_of(key, by_weight, goal);
        Cut end{value_of(key), INT_MAX};
        if (take < sh.pick_count)  // equal logits: those of the lowest indices, which are the largest when turned round
          end.last = int(~select(
              [&](auto&& f) {
                each_listed([&](const Item& x) {
                  if (x.l == end.at) f(~uint32_t(x.at), 0ull);
                });
              },
              false, ~0u << 20, 20, false, 0, double(take)));
        return end;
      };
      // the sum of the listed, of those in bins from .. to, and the bits of the latter's keys
      unsigned long long sum_listed = 0, sum_in = 0, same = 0;
      auto look_at = [&](int from, int to) {
        unsigned long long v = 0, in = 0;
        uint32_t all1 = ~0u, any1 = 0;
        each_listed([&](const Item& x) {
          v += x.weight;
          if (x.bin >= from && x.bin <= to) {
            in += x.weight;
            all1 &= key_of(x.l);
            any1 |= key_of(x.l);
          }
        });
        all1 = __reduce_and_sync(0xffffffffu, all1);
        any1 = __reduce_or_sync(0xffffffffu, any1);
        __syncthreads();
        block_sum(0, v);
        block_sum(1, in);
        if (lane == 0) sh.warp_sum[2][warp] = (static_cast<unsigned long long>(all1) << 32) | any1;
        __syncthreads();
        sum_listed = of_warps(0);
        sum_in = of_warps(1);
#pragma unroll
        for (int x = 0; x < SR_WARPS; ++x) {
          all1 &= uint32_t(sh.warp_sum[2][x] >> 32);
          any1 |= uint32_t(sh.warp_sum[2][x]);
        }
        same = (static_cast<unsigned long long>(all1) << 32) | any1;
      };
      if (!whole) {
        cut = Cut{-INFINITY, -1};
        look_at(k_bin, k_bin);
        const Cut end = end_in(k_bin, k_bin, same, false, above_k, double(top_k));
        __syncthreads();
        cut = end;
      }
      if (by_p) {
        look_at(first, last);
        const double goal = fmax(1.0, p * double(sum_all + sum_listed));
        fits = double(sum_above) < goal && double(sum_above + sum_in) >= goal;
        if (fits) {
          const Cut end = end_in(first, last, same, true, sum_above, goal);
          cut = whole ? end : stricter(cut, end);
        }
      }
      if (fits) {  // what is kept of the CTA's own to its chunks
        each_listed([&](const Item& x) {
          const int at = x.at - start;
          if (at >= shift && at < shift + mine && cut.has(x.l, x.at) && x.l >= faint && (!(least > 0.0) || w.of(x.l) >= least))
            atomicAdd(&chunk_sum[at / CHUNK], x.weight);
        });
      }
    }
  }
  // the weights of four logits that are kept, 32 places apart; a whole warp
  auto weights = [&](int at, double (&x)[4]) {
    float l[4];
    bool on[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      l[j] = logit(at + 32 * j);
      on[j] = keeps(l[j], at + 32 * j);
      x[j] = 0.0;
    }
    if (__any_sync(0xffffffffu, on[0] || on[1] || on[2] || on[3])) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double e = w.of(l[j]);
        x[j] = on[j] && e >= least ? e : 0.0;
      }
    }
  };
  if (!fits) {
    // the whole row, digit by digit, then its chunks
    cut = Cut{-INFINITY, -1};
    auto each_of_slice = [&](auto&& f) {
      for (int at = shift + tid; at < shift + mine; at += SR_THREADS) {
        const float l = logit(at);
        if (l >= lowest && cut.has(l, start + at)) f(l);
      }
    };
    // the sum of a number over all CTAs' threads
    auto sum_of_all = [&](unsigned long long v) {
      __syncthreads();
      block_sum(0, v);
      __syncthreads();
      swap ^= 1;
      exchange(0, of_warps(0));
      cluster.sync();
      return of_cluster(0, C);
    };
    auto weight = [&](float l) { return l >= faint ? fixed(w.of(l)) : 0ull; };
    auto end_of_row = [&](bool by_weight, double goal) {
      const uint32_t key = select(
          [&](auto&& f) {
            each_of_slice([&](float l) { f(key_of(l), by_weight ? weight(l) : 0ull); });
          },
          true, 0u, 32, by_weight, 0, goal);
      const unsigned take = take_of(key, by_weight, goal);
      Cut end{value_of(key), INT_MAX};
      if (take < sh.pick_count)
        end.last = int(~select(
            [&](auto&& f) {
              for (int at = shift + tid; at < shift + mine; at += SR_THREADS)
                if (logit(at) == end.at && cut.has(end.at, start + at)) f(~uint32_t(start + at), 0ull);
            },
            true, ~0u << 20, 20, false, 0, double(take)));
      return end;
    };
    if (by_k) {
      unsigned long long v = 0;
      each_of_slice([&](float) { ++v; });
      if (static_cast<unsigned long long>(top_k) < sum_of_all(v)) cut = end_of_row(false, double(top_k));
    }
    if (by_p) {
      unsigned long long v = 0;
      each_of_slice([&](float l) { v += weight(l); });
      const double goal = fmax(1.0, p * double(sum_of_all(v)));
      cut = stricter(cut, end_of_row(true, goal));
    }
    sure = NAN;  // no bins: all is the cut's
    __syncthreads();
    for (int c = warp; c < chunks; c += SR_WARPS) {
      unsigned long long v = 0;
      for (int half = 0; half < CHUNK; half += 128) {
        double x[4];
        weights(c * CHUNK + half + lane, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) v += fixed(x[j]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) chunk_sum[c] = v;
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
      const int at = chunk * CHUNK + 32 * e + lane;
      const float l = logit(at);
      double x = keeps(l, at) ? w.of(l) : 0.0;
      if (x < least) x = 0.0;
      unsigned long long inc = fixed(x);
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
    for (int c = warp; c < chunks; c += SR_WARPS) {
      for (int half = 0; half < CHUNK; half += 128) {
        const int at = c * CHUNK + half + lane;
        double x[4];
        weights(at, x);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at + 32 * j >= shift && at + 32 * j < shift + mine) probs[at + 32 * j] = float(x[j] * inv);
      }
    }
  }
}

template <typename T, bool CACHED>
cudaError_t run_sample(const SampleArgs& a, int c, int per, size_t shared, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (!(done.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(sample_kernel<T, CACHED>, cudaFuncAttributeMaxDynamicSharedMemorySize, SR_CACHE);
    if (e != cudaSuccess) return e;
    done.fetch_or(bit, std::memory_order_release);
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
  // bytes of a CTA's chunk sums, and of its slice with them
  auto slice = [&](int c) { return (a.vocab + c - 1) / c; };
  auto sums = [&](int c) { return sizeof(unsigned long long) * size_t((places<T>(slice(c)) / CHUNK + 1) / 2 * 2); };
  auto bytes = [&](int c) { return sums(c) + size_t(places<T>(slice(c))) * sizeof(T); };
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
