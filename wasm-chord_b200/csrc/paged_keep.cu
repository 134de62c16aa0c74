// The accepted tokens of a tree move to the slots behind their sequence's context, in every layer: slot
// context + i takes the key and value of slot context + path[i].
//
// path ascends, so path[i] >= i: what a move overwrites was read by an earlier one or is not wanted. A thread
// owns 16 bytes of a token in one layer's keys or values and moves them for i = 0, 1 .., several at a time,
// all loads before the first store; no thread reads what another writes. A CTA finds the moves of its sequence (those
// with path[i] > i) once, then each of its threads goes through them.
//
// Bound by latency: lengths (and path), page table and the tokens are three loads that wait for one another. One sequence in 22 layers
// 3.5 us; 32 sequences in 80 layers of 8 heads of 128, bf16, 54 tokens moved (35 MB) 11 to 14 us, 40 to 50 % of the copy rate: a CTA
// for each layer's keys or values (16.4 us) made the lookups as often. Paths of up to 32 tokens (214 moved, 140 MB) 35 us, 61 %.
#include "paged_common.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int KP_THREADS = 128;
constexpr int KP_MOVES = 128;  // moves that are looked up at a time
constexpr int KP_AHEAD = 8;    // loads of a thread before its stores

// The moves of this CTA's words, WIDE of them at a time: all loads before the first store
template <int WIDE>
__device__ __forceinline__ void move_words(const KeepArgs& a, const int64_t* of, const int64_t* to, int moves, int words, int per_head, int items) {
  constexpr int AHEAD = KP_AHEAD / WIDE;
  const int step = gridDim.y * KP_THREADS;
  for (int it = blockIdx.y * KP_THREADS + threadIdx.x; it < items; it += WIDE * step) {
    uint8_t* base[WIDE];
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      const int at = min(it + i * step, items - 1), pool = at / words, w = at % words;
      base[i] = static_cast<uint8_t*>(a.pools[pool]) + (w / per_head) * a.pool.head_stride * a.size + (w % per_head) * 16;
    }
    for (int m0 = 0; m0 < moves; m0 += AHEAD) {
      uint4 x[WIDE][AHEAD];
#pragma unroll
      for (int i = 0; i < WIDE; ++i)
#pragma unroll
        for (int m = 0; m < AHEAD; ++m)
          if (m0 + m < moves && it + i * step < items) x[i][m] = *reinterpret_cast<const uint4*>(base[i] + of[m0 + m]);
#pragma unroll
      for (int i = 0; i < WIDE; ++i)
#pragma unroll
        for (int m = 0; m < AHEAD; ++m)
          if (m0 + m < moves && it + i * step < items) *reinterpret_cast<uint4*>(base[i] + to[m0 + m]) = x[i][m];
    }
  }
}

__global__ void __launch_bounds__(KP_THREADS) keep_kernel(const __grid_constant__ KeepArgs a) {
  __shared__ int64_t s_of[KP_MOVES], s_to[KP_MOVES];
  __shared__ int s_moves[KP_THREADS / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, s = blockIdx.x;
  const bool says = blockIdx.y == 0;  // one CTA of a sequence reports
  // (a thread's first entry of the path, and the one before it, with the lengths: not after them)
  const int32_t* path = a.path + int64_t(s) * a.max_path;
  const int first = tid < a.max_path ? __ldg(path + tid) : 0, first_before = tid > 0 && tid < a.max_path ? __ldg(path + tid - 1) : -1;
  const int given = __ldg(a.count + s);
  const Seq q = read_seq(a.batch, s);
  if (!q.sound && says && tid == 0) report(a.batch, ST_BAD_ROWS);
  const int count = q.n > 0 ? min(max(given, 0), a.max_path) : 0;
  // a path that does not ascend, or leaves the new tokens, is not followed
  bool bad = false;
  for (int i = tid; i < count; i += KP_THREADS) {
    const int p = i == tid ? first : __ldg(path + i), before = i == tid ? first_before : __ldg(path + i - 1);
    bad |= p <= before || p >= q.n;
  }
  if (__syncthreads_or(bad)) {
    if (says && tid == 0) report(a.batch, ST_BAD_TREE);
    return;
  }
  const int context = q.kv - q.n, table = table_tokens(a.pool, a.batch);
  const int per_head = a.pool.head_dim * a.size / 16;
  const int words = a.pool.n_kv * per_head;  // 16-byte words of a token in one layer's keys or values
  const int items = words * 2 * a.n_layers;
  uint32_t wrong = 0;
  auto slot = [&](int pos) -> int64_t {
    if (pos < 0) {
      wrong |= ST_BAD_LEN;
      return -1;
    }
    const int page = pos < table ? __ldg(a.batch.page_table + int64_t(s) * a.batch.max_pages + pos / a.pool.page_size) : -1;
    if (page < 0 || page >= a.pool.n_pages) {
      wrong |= ST_BAD_PAGE;
      return -1;
    }
    return (page * a.pool.page_stride + int64_t(pos % a.pool.page_size) * a.pool.token_stride) * a.size;
  };
  for (int i0 = 0; i0 < count; i0 += KP_MOVES) {
    // the moves, in their order
    const int i = i0 + tid;
    int64_t of = -1, to = -1;
    if (i < count) {
      const int p = i == tid ? first : __ldg(path + i);
      if (p > i) {
        of = slot(context + p);
        to = slot(context + i);
      }
    }
    const bool move = of >= 0 && to >= 0;
    const unsigned some = __ballot_sync(0xffffffffu, move);
    if (lane == 0) s_moves[warp] = __popc(some);
    __syncthreads();
    int at = __popc(some & ((1u << lane) - 1u)), moves = 0;
#pragma unroll
    for (int w = 0; w < KP_THREADS / 32; ++w) {
      if (w < warp) at += s_moves[w];
      moves += s_moves[w];
    }
    if (move) {
      s_of[at] = of;
      s_to[at] = to;
    }
    __syncthreads();
    // KP_AHEAD loads of a thread are on their way together: of one word where there are many moves, else of several
    if (moves > 4) move_words<1>(a, s_of, s_to, moves, words, per_head, items);
    else if (moves > 2) move_words<2>(a, s_of, s_to, moves, words, per_head, items);
    else if (moves > 0) move_words<4>(a, s_of, s_to, moves, words, per_head, items);
    __syncthreads();  // the moves are done with
  }
  if (says) report(a.batch, wrong);
}

}  // namespace

cudaError_t launch_keep(const KeepArgs& a, cudaStream_t s) {
  const int words = a.pool.n_kv * a.pool.head_dim * a.size / 16;
  const long long items = static_cast<long long>(words) * 2 * a.n_layers;
  // one word of each thread, up to some CTAs an SM; then more of a thread, so that the lookups are made once for them. (Three CTAs run on an
  // SM, by 154 registers a thread; a fourth that begins as the first end is worth its lookups.)
  long long y = (items + KP_THREADS - 1) / KP_THREADS;
  // (CTAs an SM 3 / 4 / 8. 32 sequences, 80 layers, 8 heads of 128, bf16, paths of up to 8 tokens 16.7 / 13.8 / 14.5 us; 64 in 32 layers 13.3 / 11.1 /
  // 11.6; 9 in 80 5.5 / 6.5 / 8.7; 24 in 80, up to 32 tokens 32 / 28 / 25.5)
  const long long most = (a.max_path <= 16 ? 4 : 8) * SMS / a.batch.n_seqs;
  if (y > most) y = most < 1 ? 1 : most;
  keep_kernel<<<dim3(a.batch.n_seqs, unsigned(y)), KP_THREADS, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace paged
}  // namespace wcb
