// Attention of new tokens over a paged cache: the kernel for few rows and for
// f32 activations (mma.sync; the products of a decode step are far from the
// tensor cores' rate, its bytes are the bound).
//
// o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys a token sees, in one
// pass over K and V with a running maximum m and sum l (both f32):
//   m' = max(m, s_j), l' = l 2^(m - m') + 2^(s_j - m'), o' = o 2^(m - m') + 2^(s_j - m') v_j,
// s in units of log2. Rows of a key head: the rep query heads that share it, of
// every new token (row = token * rep + head), in blocks of 16 WM rows.
//
// Split: a unit is (sequence, key head, row block); its keys are TK-key tiles.
// All tiles of all units lie on one line, cut into one equal part per CTA, so
// that ragged lengths leave no CTA idle and one long sequence fills the GPU. A CTA
// finds its place from the lengths on the device (nothing is planned on the
// host, so a captured call follows the lengths of its replay). A unit that is
// cut leaves (o, m, l) pieces in the workspace, at most two a CTA; the CTA that
// finishes last joins them in their order, so results do not depend on timing.
//
// Tile: 4 warps, WM along rows and WN = 4 / WM along the tile's keys; K and V
// arrive by 16-byte cp.async through STAGES buffers; the page of every key is
// looked up one tile earlier into shared memory. Keys that do not exist (past
// the end, a page outside the pool) are filled with zeros, never read. Where
// some rows of a block see a key and others do not, V is first searched
// for infinities and NaN: 0 * inf must not reach the rows that do not see it.
//
// 16-bit types: m16n8k16. P is kept as a sum of two 16-bit numbers for WM = 1
// (the tensor cores idle there anyway), rounded once for larger WM. f32
// activations: m16n8k8 in tf32 with q and p (and an f32 cache's k and v) split
// into two tf32 numbers each, which keeps 21 bits; an f16 or bf16 cache is exact
// in tf32.
#pragma once
#include <type_traits>

#include "device_common.cuh"
#include "paged_common.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int AT_THREADS = 128;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  // 0 source bytes: the 16 bytes are zeros and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32_of(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
// x = hi + lo in tf32. An infinity or NaN stays in hi alone (inf - inf would make a NaN of it).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = tf32_of(x);
  const float l = x - __uint_as_float(hi);
  lo = fabsf(x) <= FLT_MAX ? tf32_of(l) : 0u;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two consecutive elements of a 32-bit word as f32
template <typename CT>
__device__ __forceinline__ float2 pair_f32(uint32_t w);
template <>
__device__ __forceinline__ float2 pair_f32<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 pair_f32<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- the line of tiles ------------------------------------------------------

// Keys of rows [r0, r1) of a sequence's key head: lo <= key < hi (in the cache's
// table), first and last token's positions.
struct Block {
  int lo, hi, pos0, pos1, tile0, tiles;
};
__device__ __forceinline__ Block row_block(const AttendArgs& a, const Seq& q, int rows, int rb, int M, int TK, int table) {
  Block b;
  const int r0 = rb * M, r1 = min(rows, r0 + M);
  b.pos0 = q.kv - q.n + r0 / a.rep;
  b.pos1 = q.kv - q.n + (r1 - 1) / a.rep;
  b.hi = min(b.pos1 + 1, table);
  b.lo = a.window > 0 ? max(0, b.pos0 - a.window + 1) : 0;
  b.tile0 = b.lo / TK;
  // rows that see nothing still have their zeros written
  b.tiles = b.hi > b.lo ? (b.hi + TK - 1) / TK - b.tile0 : 1;
  return b;
}
__device__ __forceinline__ int seq_rows(const AttendArgs& a, const Seq& q) {
  const long long r = static_cast<long long>(q.n) * a.rep;
  return r > a.row_lo && r <= a.row_hi ? int(r) : 0;
}
// Tiles of one key head of a sequence; a whole warp, its lanes over the row blocks (a chunk
// of a few thousand tokens has dozens, and every CTA of a call counts them).
__device__ __forceinline__ long long head_tiles(const AttendArgs& a, const Seq& q, int rows, int M, int TK, int table) {
  long long n = 0;
  for (int rb = threadIdx.x & 31; rb * M < rows; rb += 32) n += row_block(a, q, rows, rb, M, TK, table).tiles;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}
// The same for 32 sequences, one of each lane: those of one or two row blocks by their lane, the
// others one after the other by the warp.
__device__ __forceinline__ long long lane_tiles(const AttendArgs& a, const Seq& q, int M, int TK, int table) {
  const int rows = seq_rows(a, q);
  long long n = 0;
  if (rows > 0 && rows <= 2 * M) {
    n = row_block(a, q, rows, 0, M, TK, table).tiles;
    if (rows > M) n += row_block(a, q, rows, 1, M, TK, table).tiles;
  }
  for (unsigned left = __ballot_sync(0xffffffffu, rows > 2 * M); left; left &= left - 1) {
    const int src = __ffs(int(left)) - 1;
    Seq w;
    w.n = __shfl_sync(0xffffffffu, q.n, src);
    w.kv = __shfl_sync(0xffffffffu, q.kv, src);
    w.r0 = 0;
    w.sound = true;
    const long long sum = head_tiles(a, w, __shfl_sync(0xffffffffu, rows, src), M, TK, table);
    if (int(threadIdx.x & 31) == src) n = sum;
  }
  return n;
}
// Row block of line position `at` in a key head whose tiles begin at unit0 (moved to the block's
// first tile); a whole warp.
__device__ __forceinline__ int find_block(const AttendArgs& a, const Seq& q, int rows, int M, int TK, int table, long long at, long long& unit0) {
  const int lane = threadIdx.x & 31;
  for (int rb0 = 0;; rb0 += 32) {
    const int rb = rb0 + lane;
    const long long n = rb * M < rows ? row_block(a, q, rows, rb, M, TK, table).tiles : 0;
    long long inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && at < unit0 + inc);
    if (hit || (rb0 + 32) * M >= rows) {  // (the position is in the head, so there is a hit)
      const int src = hit ? __ffs(int(hit)) - 1 : 0;
      unit0 += __shfl_sync(0xffffffffu, inc - n, src);
      return rb0 + src;
    }
    unit0 += __shfl_sync(0xffffffffu, inc, 31);
  }
}

// Where on the line this CTA works.
struct Place {
  long long begin, end, per;  // tiles [begin, end); per: tiles of a CTA
  long long seq_begin;        // first tile of sequence `seq`
  int seq;
};

// All THREADS threads (whole warps). Blocks of THREADS sequences are summed; the one that holds the
// CTA's first tile is found by a scan.
template <int THREADS>
__device__ __forceinline__ Place find_place(const AttendArgs& a, int M, int TK, long long* s_warp, long long* s_out) {
  constexpr int NW = THREADS / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int table = table_tokens(a.pool, a.batch);
  const int n = a.batch.n_seqs;
  Place pl;
  long long total = 0;
  bool unsound = false;
  for (int s0 = 0; s0 < n; s0 += THREADS) {
    Seq q{0, 0, 0, true};
    if (s0 + tid < n) q = read_seq(a.batch, s0 + tid);
    unsound |= !q.sound;
    total += lane_tiles(a, q, M, TK, table) * a.pool.n_kv;
  }
  if (unsound && blockIdx.x == 0) report(a.batch, ST_BAD_ROWS);
  long long inc = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) s_warp[warp] = inc;
  if (tid == 0) s_out[0] = -1;
  __syncthreads();
  long long all = 0, before = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += s_warp[w];
    all += s_warp[w];
  }
  pl.per = (all + gridDim.x - 1) / gridDim.x;
  if (pl.per < 1) pl.per = 1;
  pl.begin = pl.per * blockIdx.x;
  pl.end = min(all, pl.begin + pl.per);
  pl.seq = 0;
  pl.seq_begin = 0;
  if (pl.begin >= pl.end) {
    pl.begin = pl.end = 0;
    return pl;  // no work; uniform over the CTA
  }
  if (n <= THREADS) {
    const long long first = before + inc - total;
    if (total > 0 && first <= pl.begin && pl.begin < first + total) {
      s_out[0] = tid;
      s_out[1] = first;
    }
    __syncthreads();
  } else {
    long long base = 0;
    for (int s0 = 0; s0 < n; s0 += THREADS) {
      const int s = s0 + tid;
      Seq q{0, 0, 0, true};
      if (s < n) q = read_seq(a.batch, s);
      const long long v = lane_tiles(a, q, M, TK, table) * a.pool.n_kv;
      inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      __syncthreads();  // the last round's sums are read
      if (lane == 31) s_warp[warp] = inc;
      __syncthreads();
      before = 0;
      long long sum = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        if (w < warp) before += s_warp[w];
        sum += s_warp[w];
      }
      const long long first = base + before + inc - v;
      if (v > 0 && first <= pl.begin && pl.begin < first + v) {
        s_out[0] = s;
        s_out[1] = first;
      }
      __syncthreads();
      base += sum;
      if (s_out[0] >= 0) break;
    }
  }
  pl.seq = int(s_out[0]);
  pl.seq_begin = s_out[1];
  return pl;
}

// ---- the kernel -------------------------------------------------------------

template <typename AT, typename CT, int HD, int WM>
struct AttnCfg {
  static constexpr bool F32A = std::is_same<AT, float>::value;
  static constexpr bool F32C = std::is_same<CT, float>::value;
  static constexpr int WN = 4 / WM;
  static constexpr int TK = F32C ? 32 : 64;  // keys of a tile
  static constexpr int KW = TK / WN;         // keys of a warp
  static constexpr int M = 16 * WM;
  static constexpr int ROW = HD * int(sizeof(CT)) + 16;  // bytes of a staged row: 16 more than a multiple of 128
  static constexpr int STAGE = 2 * TK * ROW;
  static constexpr int STAGES = 3;
  static constexpr int QBYTES = F32A ? M * HD * 8 : 0;  // q as tf32 pairs in fragment order
  static constexpr int OPITCH = HD + 4;                 // floats; joining the warps' results
  static constexpr int JOIN = WN > 1 ? 4 * 16 * OPITCH * 4 + 4 * 16 * 8 : 0;
  static constexpr int RING = STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN;
  static constexpr int OFFS = (STAGES + 1) * TK * 8 + (STAGES + 1) * 2 * 4;
  static constexpr int SMEM = RING + QBYTES + OFFS;
  static constexpr bool TWO_P = !F32A && WM == 1;
};

template <typename AT, typename CT, int HD, int WM>
__global__ void __launch_bounds__(AT_THREADS) attend_kernel(const __grid_constant__ AttendArgs a) {
  using L = AttnCfg<AT, CT, HD, WM>;
  constexpr int TK = L::TK, KW = L::KW, M = L::M, WN = L::WN, ROW = L::ROW, S = L::STAGES;
  constexpr bool F32A = L::F32A, F32C = L::F32C;
  constexpr int NT = KW / 8;   // 8-key column blocks of a warp
  constexpr int ND = HD / 8;   // 8-dim column blocks of the output
  constexpr int CH = HD * int(sizeof(CT)) / 16;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t sm[];
  uint4* qfrag = reinterpret_cast<uint4*>(sm + L::RING);
  long long* offs = reinterpret_cast<long long*>(sm + L::RING + L::QBYTES);  // [S + 1][TK]: element offset of a key's row, -1 = none
  unsigned* holes = reinterpret_cast<unsigned*>(offs + (S + 1) * TK);        // [S + 1][TK / 32]: keys below the end without a page
  __shared__ long long s_scan[8], s_place[2];
  __shared__ int s_last;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp % WM, wn = warp / WM;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t sbase = smem_u32(sm);
  const int table = table_tokens(a.pool, a.batch);
  const Place pl = find_place<AT_THREADS>(a, M, TK, s_scan, s_place);
  if (pl.begin >= pl.end) return;

  // walk to the unit of the first tile
  int s = pl.seq, kvh = 0, rb = 0;
  Seq sq = read_seq(a.batch, s);
  int rows = seq_rows(a, sq);
  long long at = pl.begin;       // line position
  long long unit0;               // line position of the unit's first tile
  Block blk;
  {
    const long long ht = head_tiles(a, sq, rows, M, TK, table);
    kvh = int((at - pl.seq_begin) / ht);
    unit0 = pl.seq_begin + kvh * ht;
    rb = find_block(a, sq, rows, M, TK, table, at, unit0);
    blk = row_block(a, sq, rows, rb, M, TK, table);
  }

  while (true) {
    const int ta = int(at - unit0), tb = int(min(static_cast<long long>(blk.tiles), pl.end - unit0));
    const int r0 = rb * M, rn = min(M, rows - r0);  // rows of the block
    const CT* kbase = static_cast<const CT*>(a.pool.k) + kvh * a.pool.head_stride;
    const CT* vbase = static_cast<const CT*>(a.pool.v) + kvh * a.pool.head_stride;

    // the page of every key of tile i, into ring slot i % (S + 1)
    auto look_up = [&](int i) {
      if (tid < TK) {
        const int key = (blk.tile0 + i) * TK + tid;
        long long off = -1;
        bool hole = false;
        if (key >= blk.lo && key < blk.hi) {
          const int page = __ldg(a.batch.page_table + int64_t(s) * a.batch.max_pages + key / a.pool.page_size);
          if (page >= 0 && page < a.pool.n_pages)
            off = page * a.pool.page_stride + int64_t(key % a.pool.page_size) * a.pool.token_stride;
          else hole = true;
        }
        offs[(i % (S + 1)) * TK + tid] = off;
        const unsigned any = __ballot_sync(0xffffffffu, hole);
        if (lane == 0) holes[(i % (S + 1)) * (TK / 32) + warp] = any;
      }
    };
    auto request = [&](int i) {
      const uint32_t dst = sbase + uint32_t((i % S) * L::STAGE);
#pragma unroll
      for (int c = tid; c < TK * CH; c += AT_THREADS) {
        const int key = c / CH, ch = c % CH;
        const long long off = offs[(i % (S + 1)) * TK + key];
        const int64_t e = (off < 0 ? 0 : off) + ch * (16 / int(sizeof(CT)));
        const uint32_t d = dst + uint32_t(key * ROW + ch * 16);
        cp16(d, kbase + e, off >= 0);
        cp16(d + TK * ROW, vbase + e, off >= 0);
      }
    };

    __syncthreads();  // the ring and offs of the last unit are done with
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (ta + i < tb) look_up(ta + i);

    // queries of the block. Row r of the block: token (r0 + r) / rep, head (r0 + r) % rep
    auto q_row = [&](int r) -> const AT* {
      const int gr = r0 + r;
      return static_cast<const AT*>(a.q) + (sq.r0 + gr / a.rep) * a.q_stride + (kvh * a.rep + gr % a.rep) * HD;
    };
    uint32_t qf[F32A ? 1 : HD / 16][4];
    if constexpr (!F32A) {
      const int ra = 16 * wm + g, rc = ra + 8;
      const AT* pa = q_row(min(ra, rn - 1));
      const AT* pc = q_row(min(rc, rn - 1));
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        qf[k][0] = __ldg(reinterpret_cast<const uint32_t*>(pa + 16 * k + 2 * t));
        qf[k][1] = __ldg(reinterpret_cast<const uint32_t*>(pc + 16 * k + 2 * t));
        qf[k][2] = __ldg(reinterpret_cast<const uint32_t*>(pa + 16 * k + 8 + 2 * t));
        qf[k][3] = __ldg(reinterpret_cast<const uint32_t*>(pc + 16 * k + 8 + 2 * t));
      }
    } else {
      // fragment order [m-tile][k-step][hi | lo][lane]: k index t is dim 2t (16-bit cache) or t,
      // k index t + 4 is dim 2t + 1 or t + 4, as the K fragments hold them
      for (int i = tid; i < WM * (HD / 8) * 32; i += AT_THREADS) {
        const int ln = i & 31, k = (i >> 5) % (HD / 8), m = (i >> 5) / (HD / 8);
        const int gg = ln >> 2, tt = ln & 3;
        const float* pa = reinterpret_cast<const float*>(q_row(min(16 * m + gg, rn - 1))) + 8 * k;
        const float* pc = reinterpret_cast<const float*>(q_row(min(16 * m + gg + 8, rn - 1))) + 8 * k;
        const int d0 = F32C ? tt : 2 * tt, d1 = F32C ? tt + 4 : 2 * tt + 1;
        uint4 hi, lo;
        split_tf32(__ldg(pa + d0), hi.x, lo.x);
        split_tf32(__ldg(pc + d0), hi.y, lo.y);
        split_tf32(__ldg(pa + d1), hi.z, lo.z);
        split_tf32(__ldg(pc + d1), hi.w, lo.w);
        qfrag[((m * (HD / 8) + k) * 2) * 32 + ln] = hi;
        qfrag[((m * (HD / 8) + k) * 2 + 1) * 32 + ln] = lo;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S - 1; ++i) {
      if (ta + i < tb) request(ta + i);
      cp_commit();
    }

    float o[ND][4];
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    float mx[2] = {-INFINITY, -INFINITY}, ls[2] = {0.0f, 0.0f};
    // positions of this thread's two rows (rows past the block see what its last row sees; nothing of theirs is kept)
    int pos[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) pos[h] = sq.kv - sq.n + (r0 + min(16 * wm + g + 8 * h, rn - 1)) / a.rep;

    bool hole_seen = false;
    for (int i = ta; i < tb; ++i) {
      cp_wait<S - 2>();
      __syncthreads();
      // offs of tile i + S - 1 were written before this barrier; its stage was read before it
      if (i + S - 1 < tb) request(i + S - 1);
      cp_commit();
      if (i + S < tb) look_up(i + S);  // into the place of tile i - 1, which every warp has left
      const int key0 = (blk.tile0 + i) * TK;
      const uint32_t ks = sbase + uint32_t((i % S) * L::STAGE), vs = ks + TK * ROW;
      const int kw0 = wn * KW;  // this warp's keys in the tile
      unsigned gaps = 0;
#pragma unroll
      for (int w = 0; w < TK / 32; ++w) gaps |= holes[(i % (S + 1)) * (TK / 32) + w];
      const bool hole = gaps != 0;
      hole_seen |= hole;
      // some key of the tile is not seen by every row
      const bool ragged = key0 + TK > min(blk.hi, blk.pos0 + 1) || key0 < blk.lo ||
                          (a.window > 0 && key0 < blk.pos1 - a.window + 1) || hole;

      // S = Q K^T
      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.0f;
      if constexpr (!F32A) {
        // one ldmatrix.x4: keys 8n .. +8 of two k-steps' halves: (dims 0-7, 8-15, 16-23, 24-31)
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t b[4];
            ldsm4(b, ks + uint32_t((kw0 + 8 * n + (lane & 7)) * ROW + (32 * k + 8 * (lane >> 3)) * 2));
            mma16(sc[n], qf[2 * k], b[0], b[1], AT());
            mma16(sc[n], qf[2 * k + 1], b[2], b[3], AT());
          }
        }
      } else if constexpr (!F32C) {
#pragma unroll 2
        for (int k = 0; k < HD / 32; ++k) {
          uint32_t qh[4][4], ql[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 h = qfrag[((wm * (HD / 8) + 4 * k + j) * 2) * 32 + lane];
            const uint4 l = qfrag[((wm * (HD / 8) + 4 * k + j) * 2 + 1) * 32 + lane];
            qh[j][0] = h.x; qh[j][1] = h.y; qh[j][2] = h.z; qh[j][3] = h.w;
            ql[j][0] = l.x; ql[j][1] = l.y; ql[j][2] = l.z; ql[j][3] = l.w;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t b[4];
            ldsm4(b, ks + uint32_t((kw0 + 8 * n + (lane & 7)) * ROW + (32 * k + 8 * (lane >> 3)) * 2));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = pair_f32<CT>(b[j]);
              mma8(sc[n], qh[j], __float_as_uint(f.x), __float_as_uint(f.y));
              mma8(sc[n], ql[j], __float_as_uint(f.x), __float_as_uint(f.y));
            }
          }
        }
      } else {
#pragma unroll 2
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t qh[2][4], ql[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 h = qfrag[((wm * (HD / 8) + 2 * k + j) * 2) * 32 + lane];
            const uint4 l = qfrag[((wm * (HD / 8) + 2 * k + j) * 2 + 1) * 32 + lane];
            qh[j][0] = h.x; qh[j][1] = h.y; qh[j][2] = h.z; qh[j][3] = h.w;
            ql[j][0] = l.x; ql[j][1] = l.y; ql[j][2] = l.z; ql[j][3] = l.w;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t b[4];
            ldsm4(b, ks + uint32_t((kw0 + 8 * n + (lane & 7)) * ROW + (16 * k + 4 * (lane >> 3)) * 4));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t h0, l0, h1, l1;
              split_tf32(__uint_as_float(b[2 * j]), h0, l0);
              split_tf32(__uint_as_float(b[2 * j + 1]), h1, l1);
              mma8(sc[n], qh[j], h0, h1);
              mma8(sc[n], qh[j], l0, l1);
              mma8(sc[n], ql[j], h0, h1);
            }
          }
        }
      }

      // scale, masks, running maximum
      float top[2] = {mx[0], mx[1]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = sc[n][e] * a.scale_log2;
          if (ragged) {
            const int kk = kw0 + 8 * n + 2 * t + (e & 1), key = key0 + kk, p = pos[e >> 1];
            const bool seen = key <= p && key < blk.hi && key >= blk.lo && (a.window <= 0 || key > p - a.window) &&
                              (!hole || offs[(i % (S + 1)) * TK + kk] >= 0);
            if (!seen) v = -INFINITY;
          }
          sc[n][e] = v;
          top[e >> 1] = fmaxf(top[e >> 1], v);
        }
      }
      float fac[2], use[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        use[h] = top[h] == -INFINITY ? 0.0f : top[h];
        fac[h] = fast_exp2(mx[h] - use[h]);
        mx[h] = top[h];
        ls[h] *= fac[h];
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[n][e] = fast_exp2(sc[n][e] - use[e >> 1]);
          ls[e >> 1] += sc[n][e];
        }
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= fac[e >> 1];

      // keys that some rows see and others do not: an infinity or NaN among their values is added
      // to the rows that see it, and taken out of the tile
      if (ragged && (blk.pos1 > blk.pos0)) {
        bool odd = false;
        CT* vt = reinterpret_cast<CT*>(sm + (i % S) * L::STAGE + TK * ROW);
        for (int c = tid; c < TK * HD; c += AT_THREADS) {
          const float v = to_f32(vt[(c / HD) * (ROW / int(sizeof(CT))) + c % HD]);
          odd |= !(fabsf(v) <= FLT_MAX);
        }
        if (__syncthreads_or(odd)) {
          for (int kk = kw0; kk < kw0 + KW; ++kk) {
            const int key = key0 + kk;
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float v = to_f32(vt[kk * (ROW / int(sizeof(CT))) + 8 * n + 2 * t + (e & 1)]);
                const int p = pos[e >> 1];
                if (!(fabsf(v) <= FLT_MAX) && key <= p && (a.window <= 0 || key > p - a.window)) o[n][e] += v;
              }
          }
          __syncthreads();
          for (int c = tid; c < TK * HD; c += AT_THREADS) {
            CT* x = vt + (c / HD) * (ROW / int(sizeof(CT))) + c % HD;
            if (!(fabsf(to_f32(*x)) <= FLT_MAX)) *x = from_f32<CT>(0.0f);
          }
          __syncthreads();
        }
      }

      // O += P V
      if constexpr (!F32A) {
#pragma unroll
        for (int k = 0; k < KW / 16; ++k) {
          uint32_t ph[4], pl2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = sc[2 * k + (j >> 1)][(j & 1) * 2], y = sc[2 * k + (j >> 1)][(j & 1) * 2 + 1];
            ph[j] = pack2<AT>(x, y);
            if constexpr (L::TWO_P) {
              const float2 f = pair_f32<AT>(ph[j]);
              pl2[j] = pack2<AT>(x - f.x, y - f.y);
            }
          }
          // one ldmatrix.x4.trans: 16 keys x 16 dims
#pragma unroll
          for (int n = 0; n < ND / 2; ++n) {
            uint32_t b[4];
            ldsm4t(b, vs + uint32_t((kw0 + 16 * k + (lane & 15)) * ROW + (16 * n + 8 * (lane >> 4)) * 2));
            mma16(o[2 * n], ph, b[0], b[1], AT());
            mma16(o[2 * n + 1], ph, b[2], b[3], AT());
            if constexpr (L::TWO_P) {
              mma16(o[2 * n], pl2, b[0], b[1], AT());
              mma16(o[2 * n + 1], pl2, b[2], b[3], AT());
            }
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < NT; ++k) {  // 8 keys: key 2t is k index t, key 2t + 1 is t + 4
          uint32_t ph[4], pw[4];
          split_tf32(sc[k][0], ph[0], pw[0]);
          split_tf32(sc[k][2], ph[1], pw[1]);
          split_tf32(sc[k][1], ph[2], pw[2]);
          split_tf32(sc[k][3], ph[3], pw[3]);
          if constexpr (!F32C) {
#pragma unroll
            for (int n = 0; n < ND / 4; ++n) {  // 8 keys x 32 dims
              uint32_t b[4];
              ldsm4t(b, vs + uint32_t((kw0 + 8 * k + (lane & 7)) * ROW + (32 * n + 8 * (lane >> 3)) * 2));
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 f = pair_f32<CT>(b[j]);
                mma8(o[4 * n + j], ph, __float_as_uint(f.x), __float_as_uint(f.y));
                mma8(o[4 * n + j], pw, __float_as_uint(f.x), __float_as_uint(f.y));
              }
            }
          } else {
#pragma unroll
            for (int n = 0; n < ND; ++n) {
              const float f0 = ldsf(vs + uint32_t((kw0 + 8 * k + 2 * t) * ROW + (8 * n + g) * 4));
              const float f1 = ldsf(vs + uint32_t((kw0 + 8 * k + 2 * t + 1) * ROW + (8 * n + g) * 4));
              uint32_t h0, l0, h1, l1;
              split_tf32(f0, h0, l0);
              split_tf32(f1, h1, l1);
              mma8(o[n], ph, h0, h1);
              mma8(o[n], ph, l0, l1);
              mma8(o[n], pw, h0, h1);
            }
          }
        }
      }
    }
    cp_wait<0>();
    if (hole_seen && tid == 0) report(a.batch, ST_BAD_PAGE);
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // the four lanes of a row
      ls[h] += __shfl_xor_sync(0xffffffffu, ls[h], 1);
      ls[h] += __shfl_xor_sync(0xffffffffu, ls[h], 2);
    }
    if (tid == 0 && blk.pos1 >= table) report(a.batch, ST_BAD_PAGE);
    if (tid == 0 && blk.pos0 < 0) report(a.batch, ST_BAD_LEN);

    const bool whole = ta == 0 && tb == blk.tiles;
    float* piece = a.part + (size_t(blockIdx.x) * 2 + (ta == 0 ? 1 : 0)) * size_t(M) * (HD + 2);  // [M][HD], then [M][2]
    auto put = [&](int r, int d, float x, float y, float m, float l) {  // two results of row r
      if (whole) {
        const int gr = r0 + r;
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        AT* dst = static_cast<AT*>(a.out) + (sq.r0 + gr / a.rep) * a.out_stride + (kvh * a.rep + gr % a.rep) * HD + d;
        const bool some = inv != 0.0f || l != l;
        x = some ? x * inv : 0.0f;
        y = some ? y * inv : 0.0f;
        if constexpr (F32A) *reinterpret_cast<float2*>(dst) = make_float2(x, y);
        else *reinterpret_cast<uint32_t*>(dst) = pack2<AT>(x, y);
        if (d == 0 && a.lse)
          a.lse[int64_t(sq.r0 + gr / a.rep) * a.n_heads + kvh * a.rep + gr % a.rep] =
              some ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
      } else {
        *reinterpret_cast<float2*>(piece + size_t(r) * HD + d) = make_float2(x, y);
        if (d == 0) *reinterpret_cast<float2*>(piece + size_t(M) * HD + 2 * r) = make_float2(m, l);
      }
    };
    if constexpr (WN == 1) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * wm + g + 8 * h;
        if (r < rn)
#pragma unroll
          for (int n = 0; n < ND; ++n) put(r, 8 * n + 2 * t, o[n][2 * h], o[n][2 * h + 1], mx[h], ls[h]);
      }
    } else {
      // the WN warps of a row tile, joined through shared memory (the ring is empty)
      float* os = reinterpret_cast<float*>(sm);
      float2* ml = reinterpret_cast<float2*>(sm + 4 * 16 * L::OPITCH * 4);
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = warp * 16 + g + 8 * h;
#pragma unroll
        for (int n = 0; n < ND; ++n)
          *reinterpret_cast<float2*>(os + r * L::OPITCH + 8 * n + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if (t == 0) ml[r] = make_float2(mx[h], ls[h]);
      }
      __syncthreads();
      for (int c = tid; c < rn * (HD / 2); c += AT_THREADS) {
        const int r = c / (HD / 2), d = 2 * (c % (HD / 2));
        const int w0 = r / 16, rr = r % 16;  // warps w0, w0 + WM, ..
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < WN; ++j) m = fmaxf(m, ml[(w0 + j * WM) * 16 + rr].x);
        const float u = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
        for (int j = 0; j < WN; ++j) {
          const int w = (w0 + j * WM) * 16 + rr;
          const float2 q = ml[w];
          const float f = fast_exp2(q.x - u);
          const float2 v = *reinterpret_cast<const float2*>(os + w * L::OPITCH + d);
          l += f * q.y;
          x += f * v.x;
          y += f * v.y;
        }
        put(r, d, x, y, m, l);
      }
    }

    if (!whole) {
      // the last of the unit's CTAs joins its pieces, in their order
      const long long u1 = unit0 + blk.tiles - 1;
      const int c0 = int(unit0 / pl.per), c1 = int(u1 / pl.per);
      __threadfence();
      __syncthreads();
      if (tid == 0) s_last = atomicInc(reinterpret_cast<unsigned*>(a.tickets) + c0, unsigned(c1 - c0)) == unsigned(c1 - c0);
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int c = tid; c < rn * (HD / 4); c += AT_THREADS) {
          const int r = c / (HD / 4), d = 4 * (c % (HD / 4));
          float m = -INFINITY;
          for (int p = c0; p <= c1; ++p) {
            const float* pc = a.part + (size_t(p) * 2 + (p == c0 ? 1 : 0)) * size_t(M) * (HD + 2);
            m = fmaxf(m, __ldcg(reinterpret_cast<const float2*>(pc + size_t(M) * HD + 2 * r)).x);
          }
          const float u = m == -INFINITY ? 0.0f : m;
          float l = 0.0f;
          float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int p = c0; p <= c1; ++p) {
            const float* pc = a.part + (size_t(p) * 2 + (p == c0 ? 1 : 0)) * size_t(M) * (HD + 2);
            const float2 q = __ldcg(reinterpret_cast<const float2*>(pc + size_t(M) * HD + 2 * r));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(pc + size_t(r) * HD + d));
            const float f = fast_exp2(q.x - u);
            l += f * q.y;
            x.x += f * v.x;
            x.y += f * v.y;
            x.z += f * v.z;
            x.w += f * v.w;
          }
          const int gr = r0 + r;
          const bool some = l > 0.0f || l != l;
          const float inv = some ? 1.0f / l : 0.0f;
          const int64_t tok = sq.r0 + gr / a.rep;
          const int hh = kvh * a.rep + gr % a.rep;
          AT* dst = static_cast<AT*>(a.out) + tok * a.out_stride + hh * HD + d;
          const float v0 = some ? x.x * inv : 0.0f, v1 = some ? x.y * inv : 0.0f;
          const float v2 = some ? x.z * inv : 0.0f, v3 = some ? x.w * inv : 0.0f;
          if constexpr (F32A) *reinterpret_cast<float4*>(dst) = make_float4(v0, v1, v2, v3);
          else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<AT>(v0, v1), pack2<AT>(v2, v3));
          if (d == 0 && a.lse) a.lse[tok * a.n_heads + hh] = some ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
        }
      }
    }

    at = unit0 + tb;
    if (at >= pl.end) break;
    // next unit
    unit0 += blk.tiles;
    ++rb;
    if (rb * M >= rows) {
      rb = 0;
      if (++kvh == a.pool.n_kv) {
        kvh = 0;
        do {
          ++s;  // there are tiles left, so a sequence with rows follows
          sq = read_seq(a.batch, s);
          rows = seq_rows(a, sq);
        } while (rows == 0);
      }
    }
    blk = row_block(a, sq, rows, rb, M, TK, table);
  }
}

template <typename AT, typename CT, int HD, int WM>
cudaError_t run_attend(const AttendArgs& a, cudaStream_t st) {
  using L = AttnCfg<AT, CT, HD, WM>;
  static_assert(L::SMEM <= 227 * 1024, "shared memory");
  // the limit is a property of the kernel on the current device: set on every call (no
  // state that a second device or thread could find half made)
  cudaError_t e = cudaFuncSetAttribute(attend_kernel<AT, CT, HD, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  if (e != cudaSuccess) return e;
  attend_kernel<AT, CT, HD, WM><<<ATTEND_CTAS, AT_THREADS, L::SMEM, st>>>(a);
  return cudaGetLastError();
}

template <typename AT, typename CT>
cudaError_t run_attend_rows(const AttendArgs& a, int rows, cudaStream_t st) {
  if (a.pool.head_dim == 64)
    return rows == 16 ? run_attend<AT, CT, 64, 1>(a, st) : rows == 32 ? run_attend<AT, CT, 64, 2>(a, st) : run_attend<AT, CT, 64, 4>(a, st);
  return rows == 16 ? run_attend<AT, CT, 128, 1>(a, st) : rows == 32 ? run_attend<AT, CT, 128, 2>(a, st) : run_attend<AT, CT, 128, 4>(a, st);
}

}  // namespace
}  // namespace paged
}  // namespace wcb
