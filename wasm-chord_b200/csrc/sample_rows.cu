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
//
// Measured: one row of 32000, f32, top-k 40 and top-p 0.9: 15 us, latency (8 CTAs; of 26000 clocks the loads and the largest logit take 3000, bins
// 9000, the pass 1000, the lists 9000, the draw 3000: a barrier of the cluster costs 1200). 416 rows of 32000, bf16, eight kinds of
// settings: 49 us (rows without filters alone 35, with top-p 0.95 73, greedy 12; 27 MB, floor 4 us). 192 rows of 100003, f32, with probabilities: 116 us
// (154 MB, floor 23 us). What bounds many rows: instructions (issue 57 %), integer ones first (bins, masks, 64-bit sums: that pipe 40 %), with
// shared-memory atomics (9 clocks for 32 logits) for the bins, then barriers between short steps; the 64-bit units, 15 operations a
// weight at 3.3 clocks a warp, are busy for 11 to 17 %, and bound only rows without filters. Tried: a table of 64
// powers instead of the longer polynomial (bank conflicts took what it saved), conversions to 64 bits by integer operations (no
// difference), 256 threads a CTA (66 to 76 us), lists of up to 512 tokens sorted (14000 clocks; digits 8000).
#include <cooperative_groups.h>

#include <atomic>
#include <climits>
#include <type_traits>

#include "paged_common.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int SR_THREADS = 512;
constexpr int SR_WARPS = SR_THREADS / 32;
constexpr int SR_CLUSTER = 8;
constexpr int SR_CACHE = 66 * 1024;  // bytes of a slice in shared memory at most: an SM holds two
constexpr int FIX = 43;              // bits after the point
constexpr int BINS = 2048;
constexpr float REACH = 20.0f;  // the bins' width is REACH / BINS; what lies farther from the largest logit is in the last one
constexpr float SLACK = 2e-5f;  // of a bin's weights: its ends are rounded, and sums of 32 bits
constexpr float BIN0 = 8388608.0f;  // 2^23: bins as floats, BIN0 + number, so that adding BIN0 rounds to a whole one
constexpr int DIGITS = 1024;
constexpr int CONTROL = 256;  // threads that go through bins, digits and lists: what they do is no less for being shared by more
constexpr int LIST = 4096;  // tokens that a row's list holds, an equal part for each CTA
constexpr int CHUNK = 256;  // logits of one warp's round, 8 a lane
constexpr int COSTED = 2048;  // rows of a call that are put in order

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

// the sum over a warp of whole numbers below 2^50
__device__ __forceinline__ unsigned long long warp_sum50(unsigned long long v) {
  const unsigned lo = __reduce_add_sync(0xffffffffu, unsigned(v) & 0x1ffffffu);
  const unsigned hi = __reduce_add_sync(0xffffffffu, unsigned(v >> 25));
  return (static_cast<unsigned long long>(hi) << 25) + lo;
}

struct SampleShared {
  uint2 list[LIST];  // logit, index
  unsigned count[DIGITS];  // of a digit: tokens, the halves of their sum
  union {
    struct {
      unsigned lo[DIGITS], hi[DIGITS];
    };
    unsigned bins[BINS];  // or, packed, two counts of 16 bits in each of half as many words
  };
  unsigned long long sum[2][3][SR_CLUSTER];  // exchanged
  unsigned long long warp_sum[3][SR_WARPS];
  float warp_low[CONTROL / 32], warp_up[CONTROL / 32];
  unsigned long long pick_before;
  unsigned pick, pick_count;
  uint32_t found;
  int k_bin, above_k, whole;  // top-k's bin (BINS: there are fewer tokens), tokens above it, whether all of it is kept
  int first, last;            // bins between which top-p ends
  int listed, fits, row;
  Cut end;
  unsigned long long kinds[COSTED / 32];
};

// Places of a slice in shared memory: as far behind a multiple of 16 bytes as in memory, filled up with -infinity to whole chunks.
template <typename T>
__host__ __device__ constexpr int places(int per) {
  return (per + 16 / int(sizeof(T)) - 1 + CHUNK - 1) / CHUNK * CHUNK;
}

// CACHED: the slice fits into shared memory; else it is read again and again
template <typename T, bool CACHED>
__global__ void __launch_bounds__(SR_THREADS, 2) sample_kernel(const __grid_constant__ SampleArgs a, int per, bool by_cost) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ __align__(16) unsigned long long chunk_sum[];  // of each chunk of the slice; then the slice
  __shared__ SampleShared sh;
  // every CTA of the cluster runs before any writes into another's shared memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  int row = blockIdx.x / C;
  if (by_cost) {
    // Of more rows than run at once the dear ones come first, so that none of them begins last: the row that has this place
    // in the order of (kind, row). Counts of the four kinds in 16 bits each, by 32 rows.
    constexpr int STRIPS = COSTED / SR_THREADS;
    int kind[STRIPS];
    unsigned same[STRIPS];
#pragma unroll
    for (int j = 0; j < STRIPS; ++j) {
      const int r = j * SR_THREADS + tid;
      kind[j] = 4;
      if (r < a.n_rows) {
        const int k = a.top_k ? __ldg(a.top_k + r) : 0;
        const bool warm = !a.temperature || __ldg(a.temperature + r) > 0.0f, p = a.top_p && __ldg(a.top_p + r) < 1.0f;
        kind[j] = !warm ? 3 : p && (k <= 0 || k > 256) ? 0 : k > 0 ? 1 : 2;
      }
      unsigned long long counts = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned mask = __ballot_sync(0xffffffffu, kind[j] == q);
        if (kind[j] == q) same[j] = mask;
        counts |= static_cast<unsigned long long>(__popc(mask)) << (16 * q);
      }
      if (lane == 0) sh.kinds[j * SR_WARPS + warp] = counts;
    }
    __syncthreads();
    if (warp == 0) {  // what comes before each 32 rows, kind by kind
      constexpr int PER = STRIPS * SR_WARPS / 32;
      unsigned long long mine[PER], sum = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        mine[j] = sh.kinds[PER * lane + j];
        sum += mine[j];
      }
      unsigned long long inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      const unsigned long long all = __shfl_sync(0xffffffffu, inc, 31);
      unsigned long long before = inc - sum + (all << 16) + (all << 32) + (all << 48);  // (kinds before this one)
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        sh.kinds[PER * lane + j] = before;
        before += mine[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < STRIPS; ++j)
      if (kind[j] < 4 && int((sh.kinds[j * SR_WARPS + warp] >> (16 * kind[j])) & 0xffffu) + __popc(same[j] & ((1u << lane) - 1u)) == row) sh.row = j * SR_THREADS + tid;
    __syncthreads();
    row = sh.row;
  }
  constexpr int V = 16 / int(sizeof(T));
  const int begin = rank * per, mine = max(0, min(per, a.vocab - begin));
  const T* slice = static_cast<const T*>(a.logits) + row * a.stride + begin;
  const int shift = int((reinterpret_cast<uintptr_t>(slice) & 15) / sizeof(T));
  const int chunks = mine > 0 ? (shift + mine + CHUNK - 1) / CHUNK : 0;
  const int start = begin - shift;  // index of place 0
  T* cache = reinterpret_cast<T*>(chunk_sum + (places<T>(per) / CHUNK + 1) / 2 * 2);
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
    } else if (c * CHUNK >= shift && (c + 1) * CHUNK <= shift + mine) {
      alignas(16) T e[8];
#pragma unroll
      for (int j = 0; j < 8; j += V) *reinterpret_cast<uint4*>(e + j) = __ldg(reinterpret_cast<const uint4*>(slice - shift + place(c, j)));
#pragma unroll
      for (int j = 0; j < 8; ++j) l[j] = to_f32(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) l[j] = logit(place(c, j));
    }
  };

  // Numbers of each thread, summed by CTA, to all CTAs of the cluster (three at a time). What others may still read of the exchange before is
  // the other half of sh.sum.
  int swap = 0;
  auto block_sum = [&](int i, unsigned long long v) {  // (a barrier follows)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sh.warp_sum[i][warp] = v;
  };
  auto of_warps = [&](int i) {  // one warp
    unsigned long long v = lane < SR_WARPS ? sh.warp_sum[i][lane] : 0;
#pragma unroll
    for (int o = SR_WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto exchange = [&](int i, unsigned long long v) {  // one warp, every lane the same v
    if (lane < C) cluster.map_shared_rank(&sh.sum[swap][i][0], lane)[rank] = v;
  };
  auto of_cluster = [&](int i, int upto) {
    unsigned long long all = 0;
    for (int r = 0; r < upto; ++r) all += sh.sum[swap][i][r];
    return all;
  };
  auto control_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(CONTROL) : "memory"); };
  // the largest of a number (above zero) over all CTAs' threads
  auto max_of_all = [&](uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0) sh.warp_sum[0][warp] = v;
    __syncthreads();
    if (warp == 0) exchange(0, __reduce_max_sync(0xffffffffu, lane < SR_WARPS ? uint32_t(sh.warp_sum[0][lane]) : 0u));
    cluster.sync();
    uint32_t best = 0;
    for (int r = 0; r < C; ++r) best = max(best, uint32_t(sh.sum[swap][0][r]));
    return best;
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
    for (int i = tid; i < BINS; i += SR_THREADS) sh.bins[i] = 0;
    if (tid == 0) {
      sh.first = sh.last = BINS - 1;
      sh.listed = 0;
      sh.k_bin = BINS;
      sh.whole = 1;
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    top = value_of(max_of_all(key_of(top)));
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
    swap ^= 1;
    const int first_at = int(~max_of_all(~uint32_t(at))), token = some ? first_at : -1;
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
  // (of_top's rounding is to be far below a bin)
  const bool binned = top <= FLT_MAX && fabsf(of_top) <= 65536.0f;

  // What is kept: bins up to sure (as bin_of gives them), and what cut has; of both, what min-p leaves.
  float sure = 2.0f * BIN0;  // all
  Cut cut{INFINITY, -1};     // none
  auto keeps = [&](float l, int at) { return l >= faint && (bin_of(l) <= sure || cut.has(l, start + at)); };

  // Digits, counted (and summed) here or over all CTAs: the first from the top with which they reach the goal, into sh.pick ..; the
  // control threads.
  auto pick = [&](bool over_all, bool by_weight, unsigned long long before, unsigned long long goal) {
    constexpr int PER = DIGITS / CONTROL;
    const int d = DIGITS - PER - PER * tid;  // the thread's last one
    unsigned cnt[PER];
    unsigned long long mass[PER], own = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      cnt[j] = 0;
      mass[j] = 0;
    }
    for (int r = over_all ? 0 : rank; r < (over_all ? C : rank + 1); ++r) {
#pragma unroll
      for (int j = 0; j < PER; j += 4) {
        const uint4 n = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.count, r) + d + j);
#pragma unroll
        for (int q = 0; q < 4; ++q) cnt[j + q] += (&n.x)[q];
        if (by_weight) {
          const uint4 lo = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.lo, r) + d + j);
          const uint4 hi = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.hi, r) + d + j);
#pragma unroll
          for (int q = 0; q < 4; ++q) mass[j + q] += (static_cast<unsigned long long>((&hi.x)[q]) << 32) + (&lo.x)[q];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (!by_weight) mass[j] = cnt[j];
      own += mass[j];
    }
    unsigned long long inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) sh.warp_sum[0][warp] = inc;
    control_sync();
    unsigned long long prev = before + inc - own;
    for (int x = 0; x < warp; ++x) prev += sh.warp_sum[0][x];
    if (own > 0 && prev < goal && prev + own >= goal) {  // one thread: the goal lies above what is before and not above all
#pragma unroll
      for (int j = PER - 1; j >= 0; --j) {
        if (prev < goal && prev + mass[j] >= goal) {
          sh.pick = unsigned(d + j);
          sh.pick_count = cnt[j];
          sh.pick_before = prev;
        }
        prev += mass[j];
      }
    }
    control_sync();
  };
  // Among keys that each() goes through, `bits` of them not known to be the same (the others: prefix), the one with which, from the largest
  // on, the count or the sum of `before` and theirs reaches the goal; in sh.pick_before what comes before it, in sh.pick_count how many there
  // are. Over all CTAs every thread, else the control threads.
  auto select = [&](auto over_all, auto&& each, uint32_t prefix, int bits, bool by_weight, unsigned long long before, unsigned long long goal) {
    constexpr bool ALL = decltype(over_all)::value;
    for (int known = 32 - bits; known < 32;) {
      const int low = max(0, 32 - known - 10);
      const uint32_t above = known ? ~0u << (32 - known) : 0u;
      if constexpr (ALL) cluster.sync();  // the counts before were read
      else control_sync();
      for (int i = 4 * tid; i < DIGITS; i += 4 * (ALL ? SR_THREADS : CONTROL))
        *reinterpret_cast<uint4*>(sh.count + i) = *reinterpret_cast<uint4*>(sh.lo + i) = *reinterpret_cast<uint4*>(sh.hi + i) = make_uint4(0, 0, 0, 0);
      if constexpr (ALL) __syncthreads();
      else control_sync();
      each([&](uint32_t k, unsigned long long f) {
        if ((k & above) != prefix) return;
        const unsigned d = (k & ~above) >> low;
        atomicAdd(&sh.count[d], 1u);
        if (by_weight) {
          const unsigned x = unsigned(f), old = atomicAdd(&sh.lo[d], x);
          atomicAdd(&sh.hi[d], unsigned(f >> 32) + (old + x < old ? 1u : 0u));
        }
      });
      if constexpr (ALL) {
        cluster.sync();
        if (tid < CONTROL) pick(true, by_weight, before, goal);
        __syncthreads();
      } else {
        control_sync();
        pick(false, by_weight, before, goal);
      }
      prefix |= sh.pick << low;
      before = sh.pick_before;
      known = 32 - low;
      if (!ALL && known < 32 && sh.pick_count == 1) {  // only one has these digits
        each([&](uint32_t k, unsigned long long) {
          if ((k & (~0u << low)) == prefix) sh.found = k;
        });
        control_sync();
        prefix = sh.found;
        break;
      }
    }
    return prefix;
  };
  // of the tokens at that key, how many it takes
  auto take_of = [&](uint32_t key, bool by_weight, unsigned long long goal) {
    const unsigned long long left = goal - sh.pick_before;
    if (!by_weight) return unsigned(left);
    const unsigned long long e = fixed(w.of(value_of(key)));
    return unsigned(min(static_cast<unsigned long long>(sh.pick_count), (left + e - 1) / e));
  };
  // top-p's goal
  auto goal_of = [&](unsigned long long sum) { return max(1ull, static_cast<unsigned long long>(ceil(fmax(double(top_p), 0.0) * double(sum)))); };

  // ---- bins: where top-k and top-p end ----
  int k_bin = BINS, above_k = 0;
  bool whole = true;
  int first = BINS, last = -1;
  if ((by_k || by_p) && binned) {
    // (one CTA reads the counts of many: 16 bits a count there)
    const bool packed = C >= 4 && per < 65536;
    int far = 0;  // in the last bin
    for (int c = warp; c < chunks; c += SR_WARPS) {
      float l[8];
      eight(c, l);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float b = bin_of(l[j]);
        if (b < BIN0 + float(BINS - 1)) atomicAdd(&sh.bins[packed ? number(b) >> 1 : number(b)], packed && (number(b) & 1) ? 0x10000u : 1u);
        else far += l[j] >= lowest ? 1 : 0;
      }
    }
    far = int(__reduce_add_sync(0xffffffffu, unsigned(far)));
    if (lane == 0 && far) atomicAdd(&sh.bins[packed ? BINS / 2 - 1 : BINS - 1], packed ? unsigned(far) << 16 : unsigned(far));
    cluster.sync();
    if (tid < CONTROL) {
      constexpr int PER = BINS / CONTROL, WORDS = PER / 4;
      static_assert(PER == 8, "a 16-byte word of packed counts a thread");
      unsigned cnt[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) cnt[j] = 0;
      // (the loads of eight, or four, CTAs are on their way together)
      if (packed) {
        uint4 theirs[SR_CLUSTER];
#pragma unroll
        for (int r = 0; r < SR_CLUSTER; ++r) theirs[r] = r < C ? reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.bins, r))[tid] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < SR_CLUSTER; ++r)
#pragma unroll
          for (int j = 0; j < PER; j += 2) {
            cnt[j] += (&theirs[r].x)[j / 2] & 0xffffu;
            cnt[j + 1] += (&theirs[r].x)[j / 2] >> 16;
          }
      } else {
#pragma unroll
        for (int r0 = 0; r0 < SR_CLUSTER; r0 += 4) {
          if (r0 >= C) break;
          uint4 theirs[4][WORDS];
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int q = 0; q < WORDS; ++q)
              theirs[r][q] = r0 + r < C ? reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.bins, r0 + r))[WORDS * tid + q] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < PER; ++j) cnt[j] += (&theirs[r][j / 4].x)[j % 4];
        }
      }
      if (by_k) {
        unsigned own = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) own += cnt[j];
        unsigned inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned t = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += t;
        }
        if (lane == 31) sh.warp_sum[0][warp] = inc;
        control_sync();
        unsigned prev = inc - own;
        for (int x = 0; x < warp; ++x) prev += unsigned(sh.warp_sum[0][x]);
        if (prev < unsigned(top_k) && prev + own >= unsigned(top_k)) {
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            if (prev < unsigned(top_k) && prev + cnt[j] >= unsigned(top_k)) {
              sh.k_bin = PER * tid + j;
              sh.above_k = int(prev);
              sh.whole = prev + cnt[j] == unsigned(top_k);
            }
            prev += cnt[j];
          }
        }
        control_sync();
        if (by_p && sh.k_bin < BINS) {
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            if (PER * tid + j > sh.k_bin) cnt[j] = 0;
            if (PER * tid + j == sh.k_bin) cnt[j] = unsigned(top_k - sh.above_k);
          }
        }
      }
      if (by_p) {
        // lower and upper bounds of the weights up to and with each bin, and of those after it
        constexpr float STEP = REACH / float(BINS) * 1.44269504f;
        const float half = exp2f(-0.5f * STEP), unit = half * half;
        float at = exp2f(-STEP * float(PER * tid)), low_inc = 0.0f, up_inc = 0.0f;
        float low[PER], up[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {  // logits of b - 1/2 to b + 1/2 widths
          up[j] = float(cnt[j]) * (at / half);
          low[j] = PER * tid + j == BINS - 1 ? 0.0f : float(cnt[j]) * (at * half);
          at *= unit;
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
        control_sync();
        float low_all = 0.0f, up_all = 0.0f, l = low_sum - low_inc, u = up_sum - up_inc;
#pragma unroll
        for (int x = 0; x < CONTROL / 32; ++x) {
          if (x < warp) {
            l += sh.warp_low[x];
            u += sh.warp_up[x];
          }
          low_all += sh.warp_low[x];
          up_all += sh.warp_up[x];
        }
        // the end is in the first bin at which (sum so far) (1 - p) >= p (sum after it)
        const float q = fmaxf(top_p, 0.0f), q1 = 1.0f - q;
        unsigned may = BINS - 1, must = BINS - 1;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          l += low[j];
          u += up[j];
          if (u * q1 * (1.0f + SLACK) >= q * fmaxf(low_all - l, 0.0f) * (1.0f - SLACK)) may = min(may, unsigned(PER * tid + j));
          if (l * q1 * (1.0f - SLACK) >= q * fmaxf(up_all - u, 0.0f) * (1.0f + SLACK) + SLACK * up_all) must = min(must, unsigned(PER * tid + j));
        }
        may = __reduce_min_sync(0xffffffffu, may);
        must = __reduce_min_sync(0xffffffffu, must);
        if (lane == 0) {
          atomicMin(&sh.first, int(may));
          atomicMin(&sh.last, int(must));
        }
      }
    }
    __syncthreads();
    k_bin = sh.k_bin;
    above_k = sh.above_k;
    whole = sh.whole != 0;
    if (by_p) {
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
    auto enlist = [&](float x, int at) {
      const int n = atomicAdd(&sh.listed, 1);
      if (n < room) list[n] = make_uint2(__float_as_uint(x), unsigned(start + at));
    };
    // what the integer units do for each logit is the bound beside the 64-bit ones, so rows without filters, and with top-p alone, have loops of their own
    if (!by_k && !by_p && !(least > 0.0)) {
      for (int c = warp; c < chunks; c += SR_WARPS) {
        unsigned long long v = 0;
        float l[8];
        eight(c, l);
#pragma unroll
        for (int half = 0; half < 8; half += 4) {
          double x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = w.of(l[half + j]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (l[half + j] >= faint) v += fixed(x[j]);
        }
        v = warp_sum50(v);
        if (lane == 0) chunk_sum[c] = v;
      }
    } else if (by_p && !by_k && !(least > 0.0)) {
      for (int c = warp; c < chunks; c += SR_WARPS) {
        unsigned long long v = 0;
        float l[8];
        eight(c, l);
#pragma unroll
        for (int half = 0; half < 8; half += 4) {
          float b[4];
          double x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            b[j] = bin_of(l[half + j]);
            x[j] = w.of(l[half + j]);
          }
          bool some = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool listed = b[j] >= list_from && b[j] <= list_to;
            some |= listed;
            if (l[half + j] >= faint && !listed) {
              const unsigned long long f = fixed(x[j]);
              sum_all += f;
              if (b[j] < list_from) v += f;
            }
          }
          if (some) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (b[j] >= list_from && b[j] <= list_to && l[half + j] >= lowest) enlist(l[half + j], place(c, half + j));
          }
        }
        sum_above += v;
        v = warp_sum50(v);
        if (lane == 0) chunk_sum[c] = v;
      }
    } else {
      // (past the last bin of interest nothing is done: nearly everywhere, with top-k. The last bin of all has no end: if it is of interest, what
      // is passed over is no candidate, or, where nothing is listed, weighs nothing. So too without bins: there of_top may be rounded by any
      // number of them)
      const float furthest = fmaxf(wanted, fmaxf(list_to, k_list));
      const bool ends = binned && furthest < BIN0 + float(BINS - 1);
      const float slope = ends ? per_bin : 1.0f, base = ends ? of_top : 0.0f;
      const float reach = ends ? furthest - BIN0 + 1.0f : lists ? -lowest : -faint;
      for (int c = warp; c < chunks; c += SR_WARPS) {
        unsigned long long v = 0;
        float l[8];
        eight(c, l);
#pragma unroll
        for (int half = 0; half < 8; half += 4) {
          bool near = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) near |= !(fmaf(-l[half + j], slope, base) > reach);
          if (!__any_sync(0xffffffffu, near)) continue;
          bool on[4], sures[4], listed[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = l[half + j], b = bin_of(x);
            listed[j] = lists && x >= lowest && ((b >= list_from && b <= list_to) || b == k_list);
            on[j] = x >= faint && b <= wanted && !listed[j];
            sures[j] = b <= sure;
          }
          if (listed[0] || listed[1] || listed[2] || listed[3]) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (listed[j]) enlist(l[half + j], place(c, half + j));
          }
          if (__any_sync(0xffffffffu, on[0] || on[1] || on[2] || on[3])) {
            double x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = w.of(l[half + j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const unsigned long long f = on[j] ? fixed(x[j]) : 0;
              sum_all += f;
              if (sures[j]) sum_above += f;
              if (sures[j] && x[j] >= least) v += f;
            }
          }
        }
        v = warp_sum50(v);
        if (lane == 0) chunk_sum[c] = v;
      }
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
    if (warp < 2) exchange(warp, of_warps(warp));
    if (warp == 2) exchange(2, sh.listed);
    for (int j = tid; j < listed; j += SR_THREADS) {
      const uint2 x = sh.list[rank * room + j];
      for (int r = 1; r < C; ++r) cluster.map_shared_rank(sh.list, (rank + r) % C)[rank * room + j] = x;
    }
    cluster.sync();
    if (tid < CONTROL) {
      sum_above = of_cluster(0, C);
      sum_all = of_cluster(1, C);
      int n = 0;
      for (int r = 0; r < C; ++r) {
        n += int(sh.sum[swap][2][r]);
        fits = fits && sh.sum[swap][2][r] <= unsigned(room);
      }
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
      if (fits && n <= 32) {
        // few: sorted, a lane each (every warp by itself). Both ends are places in that order.
        const Item own = lane < n ? item(lane) : Item{-INFINITY, INT_MAX, BINS, 0};
        float l = own.l;
        int at = own.at;
        unsigned long long f = own.weight;
#pragma unroll
        for (int k = 2; k <= 32; k *= 2)
#pragma unroll
          for (int j = k / 2; j > 0; j /= 2) {
            const float ol = __shfl_xor_sync(0xffffffffu, l, j);
            const int oat = __shfl_xor_sync(0xffffffffu, at, j);
            const unsigned long long of = __shfl_xor_sync(0xffffffffu, f, j);
            // the larger logit, or of equal ones the lower index, to the front (to the back in every other run)
            const bool mine_first = l > ol || (l == ol && at < oat), front = ((lane & j) == 0) == ((lane & k) == 0);
            if (mine_first != front) {
              l = ol;
              at = oat;
              f = of;
            }
          }
        const int bin = number(bin_of(l));
        const int in_p = __popc(__ballot_sync(0xffffffffu, lane < n && bin <= last)), above = __popc(__ballot_sync(0xffffffffu, lane < n && bin < k_bin));
        int end = whole ? n : above + (top_k - above_k);  // what top-k leaves of the list
        if (by_p) {
          unsigned long long inc = f;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
          }
          const unsigned long long sum_listed = __shfl_sync(0xffffffffu, inc, max(end - 1, 0));
          const unsigned long long goal = goal_of(sum_all + (end > 0 ? sum_listed : 0));
          // the first with which the sum reaches the goal
          const unsigned reached = __ballot_sync(0xffffffffu, lane < min(in_p, end) && sum_above + inc >= goal);
          fits = sum_above < goal && reached != 0;
          end = fits ? __ffs(int(reached)) : 1;
        }
        cut = Cut{__shfl_sync(0xffffffffu, l, end - 1), __shfl_sync(0xffffffffu, at, end - 1)};
      } else if (fits) {
        const Item own = tid < n ? item(tid) : Item{0.0f, 0, 0, 0};
        auto each_listed = [&](auto&& f) {
          if (tid < n && (own.bin != k_bin || whole || cut.has(own.l, own.at))) f(own);
          for (int j = tid + CONTROL; j < n; j += CONTROL) {
            const Item x = item(j);
            if (x.bin != k_bin || whole || cut.has(x.l, x.at)) f(x);
          }
        };
        // the end among those of bins from .. to; same: the bits that are in all of their keys, and those that are in any
        auto end_in = [&](int from, int to, unsigned long long same, bool by_weight, unsigned long long done, unsigned long long goal) {
          const uint32_t any1 = uint32_t(same);
          const int bits = max(1, 32 - __clz(int(uint32_t(same >> 32) ^ any1)));
          const uint32_t key = select(
              std::false_type(),
              [&](auto&& f) {
                each_listed([&](const Item& x) {
                  if (x.bin >= from && x.bin <= to) f(key_of(x.l), x.weight);
                });
              },
              bits == 32 ? 0u : any1 & (~0u << bits), bits, by_weight, done, goal);
          const unsigned take = take_of(key, by_weight, goal);
          Cut end{value_of(key), INT_MAX};
          if (take < sh.pick_count)  // equal logits: those of the lowest indices, which are the largest when turned round
            end.last = int(~select(
                std::false_type(),
                [&](auto&& f) {
                  each_listed([&](const Item& x) {
                    if (x.l == end.at) f(~uint32_t(x.at), 0ull);
                  });
                },
                ~0u << 20, 20, false, 0, take));
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
          control_sync();
          block_sum(0, v);
          block_sum(1, in);
          if (lane == 0) sh.warp_sum[2][warp] = (static_cast<unsigned long long>(all1) << 32) | any1;
          control_sync();
          sum_listed = sum_in = 0;
#pragma unroll
          for (int x = 0; x < CONTROL / 32; ++x) {
            sum_listed += sh.warp_sum[0][x];
            sum_in += sh.warp_sum[1][x];
            all1 &= uint32_t(sh.warp_sum[2][x] >> 32);
            any1 |= uint32_t(sh.warp_sum[2][x]);
          }
          same = (static_cast<unsigned long long>(all1) << 32) | any1;
        };
        if (!whole) {
          cut = Cut{-INFINITY, -1};
          look_at(k_bin, k_bin);
          cut = end_in(k_bin, k_bin, same, false, above_k, top_k);
        }
        if (by_p) {
          look_at(first, last);
          const unsigned long long goal = goal_of(sum_all + sum_listed);
          fits = sum_above < goal && sum_above + sum_in >= goal;
          if (fits) {
            const Cut end = end_in(first, last, same, true, sum_above, goal);
            cut = whole ? end : stricter(cut, end);
          }
        }
      }
      if (tid == 0) {
        sh.fits = fits;
        sh.end = cut;
      }
    }
    __syncthreads();
    fits = sh.fits != 0;
    cut = sh.end;
    if (fits) {  // what is kept of the CTA's own to its chunks
      for (int j = tid; j < listed; j += SR_THREADS) {
        const uint2 x = sh.list[rank * room + j];
        const float l = __uint_as_float(x.x);
        if (!cut.has(l, int(x.y)) || l < faint) continue;
        const double e = w.of(l);
        if (e >= least) atomicAdd(&chunk_sum[(int(x.y) - start) / CHUNK], fixed(e));
      }
    }
  }
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
      if (warp == 0) exchange(0, of_warps(0));
      cluster.sync();
      return of_cluster(0, C);
    };
    auto weight = [&](float l) { return l >= faint ? fixed(w.of(l)) : 0ull; };
    auto end_of_row = [&](bool by_weight, unsigned long long goal) {
      const uint32_t key = select(
          std::true_type(),
          [&](auto&& f) {
            each_of_slice([&](float l) { f(key_of(l), by_weight ? weight(l) : 0ull); });
          },
          0u, 32, by_weight, 0, goal);
      const unsigned take = take_of(key, by_weight, goal);
      Cut end{value_of(key), INT_MAX};
      if (take < sh.pick_count)
        end.last = int(~select(
            std::true_type(),
            [&](auto&& f) {
              for (int at = shift + tid; at < shift + mine; at += SR_THREADS)
                if (logit(at) == end.at && cut.has(end.at, start + at)) f(~uint32_t(start + at), 0ull);
            },
            ~0u << 20, 20, false, 0, take));
      return end;
    };
    if (by_k) {
      unsigned long long v = 0;
      each_of_slice([&](float) { ++v; });
      if (static_cast<unsigned long long>(top_k) < sum_of_all(v)) cut = end_of_row(false, top_k);
    }
    if (by_p) {
      unsigned long long v = 0;
      each_of_slice([&](float l) { v += weight(l); });
      cut = stricter(cut, end_of_row(true, goal_of(sum_of_all(v))));
    }
    sure = NAN;  // no bins: all is the cut's
    __syncthreads();
    for (int c = warp; c < chunks; c += SR_WARPS) {
      unsigned long long v = 0;
      float l[8];
      eight(c, l);
#pragma unroll 1
      for (int j = 0; j < 8; ++j)
        if (keeps(l[j], place(c, j))) {
          const double e = w.of(l[j]);
          if (e >= least) v += fixed(e);
        }
      v = warp_sum50(v);
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
  if (warp == 0) exchange(0, of_warps(0));
  cluster.sync();
  const unsigned long long before = of_cluster(0, rank), own = sh.sum[swap][0][rank], all = of_cluster(0, C);
  float u = __ldg(a.u + row);
  u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
  const unsigned long long goal = static_cast<unsigned long long>(double(u) * double(all)) + 1;  // the sum that exceeds u times all
  // the CTA whose slice reaches the goal (the sum of all does), in it the chunk, in it the token
  if (warp == 0 && before < goal && before + own >= goal) {
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
      const unsigned hit = __ballot_sync(0xffffffffu, base + inc >= goal);
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
      const unsigned hit = __ballot_sync(0xffffffffu, base + inc >= goal);
      if (hit) {
        if (lane == 0) a.tokens[row] = start + chunk * CHUNK + 32 * e + __ffs(int(hit)) - 1;
        break;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  if (probs) {
    const double inv = 1.0 / (double(all) * (1.0 / double(1ull << FIX)));
    // 16 bytes at a time where the rows allow it
    const bool wide = (reinterpret_cast<uintptr_t>(probs) & 15) == 0;
    for (int c = warp; c < chunks; c += SR_WARPS) {
      const bool inside = c * CHUNK >= shift && (c + 1) * CHUNK <= shift + mine;
      float l[8];
      eight(c, l);
#pragma unroll
      for (int half = 0; half < 8; half += 4) {
        bool on[4];
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) on[j] = keeps(l[half + j], place(c, half + j));
        if (__any_sync(0xffffffffu, on[0] || on[1] || on[2] || on[3])) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const double e = w.of(l[half + j]);
            y[j] = on[j] && e >= least ? float(e * inv) : 0.0f;
          }
        }
        float* to = probs + place(c, half);
        if (wide && inside) {
          *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (inside || (place(c, half + j) >= shift && place(c, half + j) < shift + mine)) to[j] = y[j];
        }
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
  // (eight kinds of settings: 416 rows of 32000, bf16, 49 us, in their own order 65; 192 of 100003, two CTAs a row, 115 and 132)
  const bool by_cost = a.n_rows * c > 2 * SMS && a.n_rows <= COSTED && (a.temperature || a.top_k || a.top_p);
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, CACHED>, a, per, by_cost);
}

template <typename T>
cudaError_t run_sample(const SampleArgs& a, cudaStream_t s) {
  // CTAs of a row: until there are two for each SM, with slices of at least 1024 logits. What a CTA does beside its logits
  // costs as much as some ten thousand of them, so that many rows are not cut further to fit into shared memory: (192 rows of 100003, f32,
  // top-p 0.95) 2 CTAs that read their slices again 107 us, 8 with slices in shared memory 167, 4 of either kind 129 to 170.
  int c = 1;
  while (c < SR_CLUSTER && a.n_rows * c < 2 * SMS && a.vocab / (2 * c) >= 1024) c *= 2;
  const int per = (a.vocab + c - 1) / c;
  const size_t sums = sizeof(unsigned long long) * size_t((places<T>(per) / CHUNK + 1) / 2 * 2), slice = size_t(places<T>(per)) * sizeof(T);
  if (sums + slice <= size_t(SR_CACHE)) return run_sample<T, true>(a, c, per, sums + slice, s);
  return run_sample<T, false>(a, c, per, sums, s);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int kind, cudaStream_t s) {
  return kind == E_F16 ? run_sample<__half>(a, s) : kind == E_BF16 ? run_sample<__nv_bfloat16>(a, s) : run_sample<float>(a, s);
}

}  // namespace paged
}  // namespace wcb
