// Attention of new tokens over a paged cache: the kernel for few rows (mma.sync;
// the products of a decode step are far from the tensor cores' rate, its bytes are
// the bound).
//
// o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys a token sees, in one
// pass over K and V with a running maximum m and sum l (both f32):
//   m' = max(m, s_j), l' = l 2^(m - m') + 2^(s_j - m'), o' = o 2^(m - m') + 2^(s_j - m') v_j,
// s in units of log2. Rows of a key head: the rep query heads that share it, of
// every new token (row = token * rep + head), in blocks of 8 NB rows.
//
// Split: a unit is (sequence, key head, row block); its keys are TK-key tiles.
// All tiles of all units lie on one line, cut into one equal part per CTA, so
// that ragged lengths leave no CTA idle and one long sequence fills the GPU; a unit
// counts V tiles more than it has, for its queries, its start and its end. A CTA finds
// its place from the lengths on the device (nothing is planned on the host, so a
// captured call follows the lengths of its replay). A unit that is cut (those of a few
// tiles are not) leaves (o, m, l) pieces in the workspace, at most two a CTA; the CTA
// that finishes last joins them in their order, so results do not depend on timing.
//
// Products: transposed, S^T = K Q^T and O^T = V^T P^T, so that keys and dims fill the 16 rows of an
// mma and the few rows of a decode step its 8 columns (8 rows a key head at most need
// half the products, registers and exponentials of the other way round). The 4 warps share
// a tile's keys, each with its own m, l and O, joined at a unit's end. m moves only where some
// score passes it by 2^8 (sums in f32 and P have room for that; 2^15 where P is f16, and m then lies 2^7 below the
// largest score), by one vote a tile.
//
// Tile: K and V
// arrive in rows of 128-byte panels, swizzled, through STAGES buffers: whole tiles by
// TMA in boxes of gcd(page_size, TK) tokens, which never cross a page; tiles that
// begin or end inside, and pools whose gcd is below 8, by 16-byte cp.async, which
// leaves out single keys. The page of every key is looked up one tile
// earlier. Keys that do not exist (past the end, a page outside the pool) are
// zeros, never read. Where some rows of a block see a key and others do not, V is first searched
// for infinities and NaN: 0 * inf must not reach the rows that do not see it.
//
// 16-bit types: m16n8k16. P is kept as a sum of two 16-bit numbers for NB = 1
// (the tensor cores idle there anyway), rounded once for larger NB. f32
// activations: m16n8k8 in tf32 with q and p (and an f32 cache's k and v) split
// into two tf32 numbers each, which keeps 21 bits; an f16 or bf16 cache is exact
// in tf32. The tensor cores cut their sums off instead of rounding them, so long sums are
// kept short: small products have accumulators of their own, and a tile's P V is summed
// by itself and added to O by an ordinary multiply-add.
//
// Measured, single tokens over f16: 64 sequences of up to 8191 keys, 64/8 heads of 128
// (1.1 GB), 182 us run after run, 93 % of the copy rate; one of 131071 keys (537 MB) 96 us, 86 %, the rest is the
// launch, the first loads and the join; 16 sequences of 1 to 6 tokens over 500 to 2304
// keys, 32/32 heads (349 MB), 66 us, 81 %; one sequence of 320 keys 8 us, all of it latency.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
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
// The same for a cache's numbers, with hi cut off instead of rounded: 21 bits as well (lo has a bit more to hold), numbers
// near FLT_MAX do not become infinite, so that a value that is not seen is 0 times a number, and the mask is the
// cheaper instruction (64 sequences of up to 4191 keys, 64/8 heads of 128, f32 over f32: 470 -> 418 us).
__device__ __forceinline__ void split_tf32_cut(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  const float l = x - __uint_as_float(hi);
  lo = fabsf(x) <= FLT_MAX ? tf32_of(l) : 0u;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded wait for one phase of an mbarrier: until so many ns have passed (or 2^24 polls), or until `gone`, where there is
// one, says that another thread has given up.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, uint64_t ns, const volatile int* gone = nullptr) {
  const uint32_t addr = smem_u32(bar);
  uint64_t start = 0;
  for (uint32_t it = 0; it < (1u << 24); ++it) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(addr), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 63) == 63) {
      uint64_t now;
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
      if (start == 0) start = now;
      if (now - start > ns || (gone && *gone)) return false;
    }
  }
  return false;
}
constexpr uint64_t DRAIN_NS = 10000000;  // for copies and products still on their way when a CTA gives up

// an 8 x 8 block of 16-bit values, a row (2t, 2t + 1) in lane 4 g + t, transposed
__device__ __forceinline__ uint32_t transposed8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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

// ---- tiles by TMA ------------------------------------------------------------

// box of tokens of one head: a 128-byte panel of dims from x on, tokens from `slot` of `page`
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int head, int slot, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(head), "r"(slot), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

// Tensor map of the pool's keys or values: (dim, head, token, page), boxes of 128 bytes of dims x
// `box` tokens, 128-byte swizzle. False where the pool cannot be described (strides of 2^40 bytes and more).
template <typename CT>
bool make_map(CUtensorMap* map, const Pool& p, const void* base, int box) {
  static const PFN_cuTensorMapEncodeTiled encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled>(f);
  }();
  if (!encode) return false;
  constexpr CUtensorMapDataType kind = sizeof(CT) == 4                          ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : std::is_same<CT, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint64_t dims[4] = {cuuint64_t(p.head_dim), cuuint64_t(p.n_kv), cuuint64_t(p.page_size), cuuint64_t(p.n_pages)};
  // a dimension of one may have any stride: one that the encoder takes
  const cuuint64_t least = cuuint64_t(p.head_dim) * sizeof(CT);
  const cuuint64_t strides[3] = {p.n_kv > 1 ? cuuint64_t(p.head_stride) * sizeof(CT) : least,
                                 p.page_size > 1 ? cuuint64_t(p.token_stride) * sizeof(CT) : least,
                                 p.n_pages > 1 ? cuuint64_t(p.page_stride) * sizeof(CT) : least};
  for (cuuint64_t s : strides)
    if (s >= (cuuint64_t(1) << 40)) return false;
  const cuuint32_t boxes[4] = {128 / sizeof(CT), 1, cuuint32_t(box), 1}, steps[4] = {1, 1, 1, 1};
  return encode(map, kind, 4, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Both maps; the box's tokens, or 0 where tiles of TK keys cannot come by TMA: a box starts on a
// group of 8 rows (1024 bytes, the swizzle's period) and stays in one page.
template <typename CT>
int make_maps(CUtensorMap* k, CUtensorMap* v, const Pool& p, int TK) {
  int box = TK;
  while (p.page_size % box) box /= 2;
  return box >= 8 && make_map<CT>(k, p, p.k, box) && make_map<CT>(v, p, p.v, box) ? box : 0;
}

// ---- the line of tiles ------------------------------------------------------

// row / rep and row % rep: rep_inv is above 2^40 / rep by at most 1, which is exact as long as the product fits in 64 bits,
// up to 2^24 tokens (the most a call takes)
__device__ __forceinline__ int token_of(const AttendArgs& a, int row) { return int((uint64_t(uint32_t(row)) * a.rep_inv) >> 40); }
__device__ __forceinline__ int head_of(const AttendArgs& a, int row) { return row - token_of(a, row) * a.rep; }

// Keys of rows [r0, r1) of a sequence's key head: lo <= key < hi (in the cache's
// table), first and last token's positions.
struct Block {
  int lo, hi, pos0, pos1, tile0, tiles;
};
__device__ __forceinline__ Block row_block(const AttendArgs& a, const Seq& q, int rows, int rb, int M, int TK, int table) {
  Block b;
  const int r0 = rb * M, r1 = min(rows, r0 + M);
  b.pos0 = q.kv - q.n + token_of(a, r0);
  b.pos1 = q.kv - q.n + token_of(a, r1 - 1);
  b.hi = min(b.pos1 + 1, table);
  b.lo = a.window > 0 ? min(max(0, b.pos0 - a.window + 1), max(0, b.hi)) : 0;  // (no tile past the table: its end counts in 32 bits)
  b.tile0 = b.lo / TK;
  // rows that see nothing still have their zeros written
  b.tiles = b.hi > b.lo ? (b.hi + TK - 1) / TK - b.tile0 : 1;
  return b;
}
__device__ __forceinline__ int seq_rows(const AttendArgs& a, const Seq& q) {
  const long long r = static_cast<long long>(q.n) * a.rep;
  return r > a.row_lo && r <= a.row_hi ? int(r) : 0;
}
// Places on the line of one key head of a sequence, its tiles and V for each unit; a whole warp, its lanes over the row blocks (a chunk
// of a few thousand tokens has dozens, and every CTA of a call counts them).
__device__ __forceinline__ long long head_tiles(const AttendArgs& a, const Seq& q, int rows, int M, int TK, int V, int table) {
  long long n = 0;
  for (int rb = threadIdx.x & 31; rb * M < rows; rb += 32) n += row_block(a, q, rows, rb, M, TK, table).tiles + V;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}
// The same for 32 sequences, one of each lane: those of one or two row blocks by their lane, the
// others one after the other by the warp.
__device__ __forceinline__ long long lane_tiles(const AttendArgs& a, const Seq& q, int M, int TK, int V, int table) {
  const int rows = seq_rows(a, q);
  long long n = 0;
  if (rows > 0 && rows <= 2 * M) {
    n = row_block(a, q, rows, 0, M, TK, table).tiles + V;
    if (rows > M) n += row_block(a, q, rows, 1, M, TK, table).tiles + V;
  }
  for (unsigned left = __ballot_sync(0xffffffffu, rows > 2 * M); left; left &= left - 1) {
    const int src = __ffs(int(left)) - 1;
    Seq w;
    w.n = __shfl_sync(0xffffffffu, q.n, src);
    w.kv = __shfl_sync(0xffffffffu, q.kv, src);
    w.r0 = 0;
    w.sound = true;
    const long long sum = head_tiles(a, w, __shfl_sync(0xffffffffu, rows, src), M, TK, V, table);
    if (int(threadIdx.x & 31) == src) n = sum;
  }
  return n;
}
// Row block of line position `at` in a key head whose tiles begin at unit0 (moved to the block's
// first tile); a whole warp.
__device__ __forceinline__ int find_block(const AttendArgs& a, const Seq& q, int rows, int M, int TK, int V, int table, long long at, long long& unit0) {
  const int lane = threadIdx.x & 31;
  for (int rb0 = 0;; rb0 += 32) {
    const int rb = rb0 + lane;
    const long long n = rb * M < rows ? row_block(a, q, rows, rb, M, TK, table).tiles + V : 0;
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

// All THREADS threads (whole warps). THREADS sequences at a time are counted, neighbours by different
// warps (a long chunk keeps a warp busy), and their tiles summed up; the sequence that holds the CTA's
// first tile is found by a scan.
template <int THREADS>
struct PlaceShared {
  long long count[THREADS];
  long long warp[THREADS / 32];
  long long found[2];
};
template <int THREADS>
__device__ __forceinline__ Place find_place(const AttendArgs& a, int M, int TK, int V, PlaceShared<THREADS>& sh) {
  constexpr int NW = THREADS / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int table = table_tokens(a.pool, a.batch);
  const int n = a.batch.n_seqs;
  Place pl;
  bool unsound = false;
  // sh.count of sequences s0 .. s0 + THREADS - 1, this thread's sum up to its own, the sum of all
  auto count = [&](int s0, long long& mine, long long& upto, long long& all) {
    const int slot = lane * NW + warp, s = s0 + slot;
    Seq q{0, 0, 0, true};
    if (s < n) q = read_seq(a.batch, s);
    unsound |= !q.sound;
    sh.count[slot] = lane_tiles(a, q, M, TK, V, table) * a.pool.n_kv;
    __syncthreads();
    mine = sh.count[tid];
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) sh.warp[warp] = inc;
    __syncthreads();
    long long before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) before += sh.warp[w];
      all += sh.warp[w];
    }
    upto = before + inc;
  };
  if (tid == 0) sh.found[0] = -1;
  long long mine, upto, sum, all = 0;
  for (int s0 = 0; s0 < n; s0 += THREADS) {
    if (s0) __syncthreads();
    count(s0, mine, upto, sum);
    all += sum;
  }
  if (unsound && blockIdx.x == 0) report(a.batch, ST_BAD_ROWS);
  pl.per = all < 0x7fffffff ? (int(all) + int(gridDim.x) - 1) / int(gridDim.x) : (all + gridDim.x - 1) / gridDim.x;
  if (pl.per < 1) pl.per = 1;
  pl.begin = pl.per * blockIdx.x;
  pl.end = min(all, pl.begin + pl.per);
  pl.seq = 0;
  pl.seq_begin = 0;
  if (pl.begin >= pl.end) {
    pl.begin = pl.end = 0;
    return pl;  // no work; uniform over the CTA
  }
  long long base = 0;
  for (int s0 = 0;; s0 += THREADS) {
    if (n > THREADS) {  // (else the one count still stands)
      __syncthreads();
      count(s0, mine, upto, sum);
    }
    const long long first = base + upto - mine;
    if (mine > 0 && first <= pl.begin && pl.begin < first + mine) {
      sh.found[0] = s0 + tid;
      sh.found[1] = first;
    }
    __syncthreads();
    base += sum;
    if (sh.found[0] >= 0 || s0 + THREADS >= n) break;
  }
  pl.seq = int(sh.found[0]);
  pl.seq_begin = sh.found[1];
  return pl;
}
// (64-bit division is long; nearly every call's counts fit in 32)
__device__ __forceinline__ int quotient(long long x, long long y) {
  return x < 0x7fffffff && y < 0x7fffffff ? int(x) / int(y) : int(x / y);
}

// ---- the kernel -------------------------------------------------------------

constexpr float SLACK = 8.0f;  // how far (in powers of two) a score may pass the maximum before it moves
// What O and l are scaled by lies below the maximum by so much where P is held in f16, which ends at 2^-24: weights down
// to 2^-31 of the largest count (2^-24 dropped 1.8e-3 of the weight at 60000 keys 2^-25 below one key, and l counted it).
// P stays below 2^15. bf16 and tf32 have f32's exponents and need none.
template <typename T>
constexpr float LIFT = std::is_same<T, __half>::value ? 7.0f : 0.0f;

template <typename AT, typename CT, int HD, int NB>
struct AttnCfg {
  static constexpr bool F32A = std::is_same<AT, float>::value;
  static constexpr bool F32C = std::is_same<CT, float>::value;
  static constexpr int TK = 64;       // keys of a tile
  static constexpr int V = 2;         // what a unit costs beside its tiles, in tiles (0: the drafts of 66 us take 71, the 182 us 189)
  static constexpr int SNAP = 2;      // units of so few tiles are not cut
  static constexpr int KW = TK / 4;   // keys of a warp: the rows of one mma
  static constexpr int M = 8 * NB;    // rows of a block
  static constexpr int PANELS = HD * int(sizeof(CT)) / 128;
  static constexpr int PANEL = TK * 128;            // bytes: TK rows of 128
  static constexpr int STAGE = 2 * PANELS * PANEL;  // K, then V
  static constexpr int STAGES = STAGE > 16384 ? 2 : 3;
  static constexpr int QBYTES = F32A ? NB * (HD / 8) * 512 : 0;  // q as tf32 pairs in fragment order
  static constexpr int OPITCH = HD + 4;                          // floats; joining the warps' results
  static constexpr int JOIN = 4 * M * OPITCH * 4 + 4 * M * 8;
  static constexpr int RING = STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN;
  static constexpr int OFFS = (STAGES + 1) * TK * 8 + (STAGES + 1) * 2 * 4;
  static constexpr int SMEM = RING + QBYTES + OFFS + 1024;  // + alignment to the swizzle's period
  static constexpr bool TWO_P = !F32A && NB == 1;
  // CTAs of an SM: what shared memory holds, as far as the registers of the rows go
  static constexpr int FIT = 227 * 1024 / (SMEM + 2048);
  static constexpr int WANT = NB == 1 ? (HD == 64 ? 4 : 3) : 2;
  static constexpr int PER_SM = FIT < 1 ? 1 : FIT < WANT ? FIT : WANT;
};

template <typename AT, typename CT, int HD, int NB>
__global__ void __launch_bounds__(AT_THREADS, (AttnCfg<AT, CT, HD, NB>::PER_SM))
attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
              const __grid_constant__ CUtensorMap vmap, int box) {
  using L = AttnCfg<AT, CT, HD, NB>;
  constexpr int TK = L::TK, KW = L::KW, M = L::M, S = L::STAGES, V = L::V, SNAP = L::SNAP;
  constexpr bool F32A = L::F32A, F32C = L::F32C;
  constexpr int MB = HD / 16;                    // 16-dim blocks of the output
  constexpr int CH = HD * int(sizeof(CT)) / 16;  // 16-byte chunks of a row
  constexpr int VT = L::PANELS * L::PANEL;       // bytes from a stage's K to its V
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint4* qfrag = reinterpret_cast<uint4*>(sm + L::RING);
  long long* offs = reinterpret_cast<long long*>(sm + L::RING + L::QBYTES);  // [S + 1][TK]: a key's page or row offset, -1 = none
  unsigned* holes = reinterpret_cast<unsigned*>(offs + (S + 1) * TK);        // [S + 1][2]: keys below the end without a page
  __shared__ PlaceShared<AT_THREADS> s_place;
  __shared__ int s_last;
  __shared__ uint64_t s_full[S];  // a stage's bytes are there (tiles by TMA)
  __shared__ int s_late[2];       // a tile did not come

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t sbase = smem_u32(sm);
  const int table = table_tokens(a.pool, a.batch);
  const Place pl = find_place<AT_THREADS>(a, M, TK, V, s_place);
  if (pl.begin >= pl.end) return;
  if (tid == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&s_full[i], 1);
    s_late[0] = s_late[1] = 0;
    mbar_fence_init();
  }
  uint32_t phase = 0;  // bit i: of s_full[i]

  // byte offset of 16-byte chunk c of row r in a stage's K or V; elements by row and dim
  auto chunk_at = [](int r, int c) { return uint32_t((c >> 3) * L::PANEL + r * 128 + (((c & 7) ^ (r & 7)) << 4)); };
  auto elem_at = [&](int r, int d) {
    constexpr int V = 16 / int(sizeof(CT));
    return chunk_at(r, d / V) + uint32_t(d % V) * uint32_t(sizeof(CT));
  };
  // ldmatrix of this warp's 16 keys, two chunks: what a lane adds for its row and chunk (the swizzle's
  // xor leaves bits 1 and 2 of the chunk apart). K: the matrices go keys first, V (transposed): chunks first
  const int kw0 = warp * KW;
  const uint32_t lane_k = uint32_t(kw0 + (lane & 15)) * 128 + (uint32_t((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t lane_v = uint32_t(kw0 + (lane & 7) + 8 * (lane >> 4)) * 128 + (uint32_t(((lane >> 3) & 1) ^ (lane & 7)) << 4);

  // walk to the unit of the first tile
  int s = pl.seq, kvh = 0, rb = 0;
  Seq sq = read_seq(a.batch, s);
  int rows = seq_rows(a, sq);
  long long unit0;  // the unit's first place on the line: V, then its tiles
  Block blk;
  if (rows <= M) {  // one block a head
    blk = row_block(a, sq, rows, 0, M, TK, table);
    kvh = quotient(pl.begin - pl.seq_begin, blk.tiles + V);
    unit0 = pl.seq_begin + static_cast<long long>(kvh) * (blk.tiles + V);
  } else {
    const long long ht = head_tiles(a, sq, rows, M, TK, V, table);
    kvh = quotient(pl.begin - pl.seq_begin, ht);
    unit0 = pl.seq_begin + kvh * ht;
    rb = find_block(a, sq, rows, M, TK, V, table, pl.begin, unit0);
    blk = row_block(a, sq, rows, rb, M, TK, table);
  }

  auto next_unit = [&] {
    unit0 += blk.tiles + V;
    if (unit0 >= pl.end) return false;
    ++rb;
    if (rb * M >= rows) {
      rb = 0;
      if (++kvh == a.pool.n_kv) {
        kvh = 0;
        do {
          ++s;  // there are units left, so a sequence with rows follows
          sq = read_seq(a.batch, s);
          rows = seq_rows(a, sq);
        } while (rows == 0);
      }
    }
    blk = row_block(a, sq, rows, rb, M, TK, table);
    return true;
  };
  // a small unit is the part's that it begins in
  if (blk.tiles <= SNAP && unit0 < pl.begin && !next_unit()) return;

  while (true) {
    const int ta = blk.tiles <= SNAP ? 0 : int(max(0LL, pl.begin - unit0 - V));
    const int tb = blk.tiles <= SNAP ? blk.tiles : int(min(static_cast<long long>(blk.tiles), pl.end - unit0 - V));
    if (tb <= ta) break;  // the part ends before the unit's first tile
    const int r0 = rb * M, rn = min(M, rows - r0);  // rows of the block
    const CT* kbase = static_cast<const CT*>(a.pool.k) + kvh * a.pool.head_stride;
    const CT* vbase = static_cast<const CT*>(a.pool.v) + kvh * a.pool.head_stride;

    // every key of tile i exists (its page may still be missing): it comes by TMA
    auto whole_tile = [&](int i) { return box > 0 && (blk.tile0 + i) * TK >= blk.lo && (blk.tile0 + i + 1) * TK <= blk.hi; };
    // the page of every key of tile i (an element offset where the tile comes by cp.async), into ring slot i % (S + 1)
    auto look_up = [&](int i) {
      if (tid < TK) {
        const int key = (blk.tile0 + i) * TK + tid;
        long long off = -1;
        bool hole = false;
        if (key >= blk.lo && key < blk.hi) {
          const int page = __ldg(a.batch.page_table + int64_t(s) * a.batch.max_pages + key / a.pool.page_size);
          if (page >= 0 && page < a.pool.n_pages)
            off = whole_tile(i) ? page : page * a.pool.page_stride + int64_t(key % a.pool.page_size) * a.pool.token_stride;
          else hole = true;
        }
        offs[(i % (S + 1)) * TK + tid] = off;
        const unsigned any = __ballot_sync(0xffffffffu, hole);
        if (lane == 0) holes[(i % (S + 1)) * 2 + warp] = any;
      }
    };
    auto request = [&](int i) {
      const uint32_t dst = sbase + uint32_t((i % S) * L::STAGE);
      const long long* ro = offs + (i % (S + 1)) * TK;
      if (whole_tile(i)) {
        if (tid == 0) mbar_expect_tx(&s_full[i % S], L::STAGE + a.withheld);
        if (tid < TK && tid % box == 0) {
          const long long page = ro[tid];
          const int at_page = page < 0 ? a.pool.n_pages : int(page);  // a page that is not there: past the last one, zeros
          const int slot = ((blk.tile0 + i) * TK + tid) % a.pool.page_size;
#pragma unroll
          for (int p = 0; p < L::PANELS; ++p) {
            tma_load(dst + p * L::PANEL + tid * 128, &kmap, p * (128 / int(sizeof(CT))), kvh, slot, at_page, &s_full[i % S]);
            tma_load(dst + VT + p * L::PANEL + tid * 128, &vmap, p * (128 / int(sizeof(CT))), kvh, slot, at_page, &s_full[i % S]);
          }
        }
        return;
      }
#pragma unroll 8
      for (int c = tid; c < TK * CH; c += AT_THREADS) {
        const int key = c / CH, ch = c % CH;
        const long long off = ro[key];
        const int64_t e = (off < 0 ? 0 : off) + ch * (16 / int(sizeof(CT)));
        const uint32_t d = dst + chunk_at(key, ch);
        cp16(d, kbase + e, off >= 0);
        cp16(d + VT, vbase + e, off >= 0);
      }
    };

    fence_proxy_async();  // (results went through the ring's memory)
    __syncthreads();  // the ring and offs of the last unit are done with
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (ta + i < tb) look_up(ta + i);

    // queries of the block. Row r of the block: token (r0 + r) / rep, head (r0 + r) % rep
    auto q_row = [&](int r) -> const AT* {
      const int gr = r0 + r;
      return static_cast<const AT*>(a.q) + (sq.r0 + token_of(a, gr)) * a.q_stride + (kvh * a.rep + head_of(a, gr)) * HD;
    };
    uint32_t qf[F32A ? 1 : NB][F32A ? 1 : HD / 16][2];
    if constexpr (!F32A) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const AT* p = q_row(min(8 * nb + g, rn - 1));
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          qf[nb][k][0] = __ldg(reinterpret_cast<const uint32_t*>(p + 16 * k + 2 * t));
          qf[nb][k][1] = __ldg(reinterpret_cast<const uint32_t*>(p + 16 * k + 8 + 2 * t));
        }
      }
    } else {
      // fragment order [nb][k-step][lane]: (hi, hi, lo, lo) of k indices t and t + 4, which are dims 2t and
      // 2t + 1 (16-bit cache) or t and t + 4, as the K fragments hold them
      for (int i = tid; i < NB * (HD / 8) * 32; i += AT_THREADS) {
        const int ln = i & 31, k = (i >> 5) % (HD / 8), nb = (i >> 5) / (HD / 8);
        const int tt = ln & 3;
        const float* p = reinterpret_cast<const float*>(q_row(min(8 * nb + (ln >> 2), rn - 1))) + 8 * k;
        uint4 f;
        split_tf32(__ldg(p + (F32C ? tt : 2 * tt)), f.x, f.z);
        split_tf32(__ldg(p + (F32C ? tt + 4 : 2 * tt + 1)), f.y, f.w);
        qfrag[i] = f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S - 1; ++i) {
      if (ta + i < tb) request(ta + i);
      cp_commit();
    }

    float o[MB][NB][4];  // (dim g, row 2t), (dim g, row 2t + 1), (dim g + 8, ..)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mb][nb][e] = 0.0f;
    // this lane's rows 2t and 2t + 1 of each 8: the maximum (the same in every lane of a row), the lane's part of the sum, the
    // position (rows past the block see what its last row sees; nothing of theirs is kept)
    float mx[NB][2], ls[NB][2];
    int pos[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[nb][h] = -INFINITY;
        ls[nb][h] = 0.0f;
        pos[nb][h] = sq.kv - sq.n + token_of(a, r0 + min(8 * nb + 2 * t + h, rn - 1));
      }

    bool hole_seen = false;
    for (int i = ta; i < tb; ++i) {
      if (whole_tile(i)) {
        if (!bar_wait(&s_full[i % S], (phase >> (i % S)) & 1, a.wait_ns)) s_late[i & 1] = 1;
      } else {
        cp_wait<S - 2>();
        fence_proxy_async();  // the stage may be TMA's next
      }
      __syncthreads();
      const bool late = s_late[i & 1] != 0;  // (the next tile's flag is another, so that every thread reads the same)
      // offs of tile i + S - 1 were written before this barrier; its stage was read before it
      if (i + S - 1 < tb) request(i + S - 1);
      cp_commit();
      if (i + S < tb) look_up(i + S);  // into the place of tile i - 1, which every warp has left
      const int key0 = (blk.tile0 + i) * TK;
      const uint32_t ks = sbase + uint32_t((i % S) * L::STAGE), vs = ks + VT;
      const bool hole = (holes[(i % (S + 1)) * 2] | holes[(i % (S + 1)) * 2 + 1]) != 0;
      hole_seen |= hole;
      // some key of the tile is not seen by every row
      const bool ragged = key0 + TK > min(blk.hi, blk.pos0 + 1) || key0 < blk.lo ||
                          (a.window > 0 && key0 < blk.pos1 - a.window + 1) || hole;

      // S^T = K Q^T: (key g, row 2t), (key g, row 2t + 1), (key g + 8, ..)
      float sc[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[nb][e] = 0.0f;
      if constexpr (!F32A) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t x[4];
          ldsm4(x, ks + uint32_t((k >> 2) * L::PANEL) + (lane_k ^ uint32_t((k & 3) * 32)));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma16(sc[nb], x, qf[nb][k][0], qf[nb][k][1], AT());
        }
      } else {
        float sl[NB][4];  // the small products
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) sl[nb][e] = 0.0f;
        if constexpr (!F32C) {
#pragma unroll 4
          for (int k = 0; k < HD / 16; ++k) {  // two k-steps of 8 dims
            uint32_t x[4];
            ldsm4(x, ks + uint32_t((k >> 2) * L::PANEL) + (lane_k ^ uint32_t((k & 3) * 32)));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 u = pair_f32<CT>(x[2 * j]), v = pair_f32<CT>(x[2 * j + 1]);
              const uint32_t f[4] = {__float_as_uint(u.x), __float_as_uint(v.x), __float_as_uint(u.y), __float_as_uint(v.y)};
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                const uint4 q = qfrag[(nb * (HD / 8) + 2 * k + j) * 32 + lane];
                mma8(sc[nb], f, q.x, q.y);
                mma8(sl[nb], f, q.z, q.w);
              }
            }
          }
        } else {
#pragma unroll 4
          for (int k = 0; k < HD / 8; ++k) {
            uint32_t x[4], h[4], l[4];
            ldsm4(x, ks + uint32_t((k >> 2) * L::PANEL) + (lane_k ^ uint32_t((k & 3) * 32)));
#pragma unroll
            for (int j = 0; j < 4; ++j) split_tf32_cut(__uint_as_float(x[j]), h[j], l[j]);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              const uint4 q = qfrag[(nb * (HD / 8) + k) * 32 + lane];
              mma8(sc[nb], h, q.x, q.y);
              mma8(sl[nb], l, q.x, q.y);
              mma8(sl[nb], h, q.z, q.w);
            }
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nb][e] += sl[nb][e];
      }

      // scale, masks, maximum
      bool grow = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = sc[nb][e] * a.scale_log2;
          if (ragged) {
            const int kk = kw0 + g + 8 * (e >> 1), key = key0 + kk, p = pos[nb][e & 1];
            const bool seen = key <= p && key < blk.hi && key >= blk.lo && (a.window <= 0 || key > p - a.window) &&
                              (!hole || offs[(i % (S + 1)) * TK + kk] >= 0);
            if (!seen) v = -INFINITY;
          }
          sc[nb][e] = v;
          grow |= v > mx[nb][e & 1] + (SLACK + LIFT<AT>);
        }
      }
      const bool moved = __any_sync(0xffffffffu, grow);
      float fac[NB][2];
      if (moved) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float top = fmaxf(mx[nb][h], fmaxf(sc[nb][h], sc[nb][h + 2]) - LIFT<AT>);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            fac[nb][h] = mx[nb][h] == top ? 1.0f : fast_exp2(mx[nb][h] - top);
            mx[nb][h] = top;
            ls[nb][h] *= fac[nb][h];
          }
        // O takes its factor here: a maximum moves in the first tile and rarely after it
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mb][nb][e] *= fac[nb][e & 1];
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float m = mx[nb][e & 1];
          sc[nb][e] = fast_exp2(sc[nb][e] - (m == -INFINITY ? 0.0f : m));
          ls[nb][e & 1] += sc[nb][e];
        }

      // keys that some rows see and others do not: an infinity or NaN among their values is added
      // to the rows that see it, and taken out of the tile
      if (ragged && blk.pos1 > blk.pos0) {
        bool odd = false;
        uint8_t* vt = sm + (i % S) * L::STAGE + VT;
        auto val = [&](int r, int d) -> CT& { return *reinterpret_cast<CT*>(vt + elem_at(r, d)); };
        for (int c = tid; c < TK * HD; c += AT_THREADS) odd |= !(fabsf(to_f32(val(c / HD, c % HD))) <= FLT_MAX);
        if (__syncthreads_or(odd)) {
          for (int kk = kw0; kk < kw0 + KW; ++kk) {
            const int key = key0 + kk;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float v = to_f32(val(kk, 16 * mb + g + 8 * (e >> 1)));
                  const int p = pos[nb][e & 1];
                  if (!(fabsf(v) <= FLT_MAX) && key <= p && (a.window <= 0 || key > p - a.window)) o[mb][nb][e] += v;
                }
          }
          __syncthreads();
          for (int c = tid; c < TK * HD; c += AT_THREADS) {
            CT& x = val(c / HD, c % HD);
            if (!(fabsf(to_f32(x)) <= FLT_MAX)) x = from_f32<CT>(0.0f);
          }
          fence_proxy_async();
          __syncthreads();
        }
      }

      if (late) {
        // give up, once the copies on their way have landed: those of this tile and of the ones requested after it
        for (int j = i; j < tb && j < i + S; ++j)
          if (whole_tile(j)) bar_wait(&s_full[j % S], (phase >> (j % S)) & 1, DRAIN_NS);
        cp_wait<0>();
        if (tid == 0) report(a.batch, ST_ABORTED);
        return;
      }
      if (whole_tile(i)) phase ^= 1u << (i % S);

      // O^T += V^T P^T
      if constexpr (!F32A) {
        uint32_t ph[NB][2], pw[NB][2];  // keys 2t, 2t + 1 (and + 8) of row g: S^T's blocks transposed
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float x = sc[nb][2 * h], y = sc[nb][2 * h + 1];
            const uint32_t w = pack2<AT>(x, y);
            ph[nb][h] = transposed8(w);
            if constexpr (L::TWO_P) {
              const float2 f = pair_f32<AT>(w);
              pw[nb][h] = transposed8(pack2<AT>(x - f.x, y - f.y));
            }
          }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          uint32_t x[4];
          ldsm4t(x, vs + uint32_t((mb >> 2) * L::PANEL) + (lane_v ^ uint32_t((mb & 3) * 32)));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            mma16(o[mb][nb], x, ph[nb][0], ph[nb][1], AT());
            if constexpr (L::TWO_P) mma16(o[mb][nb], x, pw[nb][0], pw[nb][1], AT());
          }
        }
      } else {
        // two k-steps of 8 keys. k index t and t + 4: keys 2t and 2t + 1 (16-bit cache) or t and t + 4. P's values
        // for them lie in other lanes: of key k and row g in lane 4 k + g / 2
        uint32_t ph[2][NB][2], pw[2][NB][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = F32C ? t + 4 * h : 2 * t + h;
              const float x = __shfl_sync(0xffffffffu, sc[nb][2 * j], 4 * key + (g >> 1));
              const float y = __shfl_sync(0xffffffffu, sc[nb][2 * j + 1], 4 * key + (g >> 1));
              split_tf32((g & 1) ? y : x, ph[j][nb][h], pw[j][nb][h]);
            }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          float x[NB][4];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[nb][e] = 0.0f;
          if constexpr (!F32C) {
            uint32_t w[4];
            ldsm4t(w, vs + uint32_t((mb >> 2) * L::PANEL) + (lane_v ^ uint32_t((mb & 3) * 32)));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 u = pair_f32<CT>(w[2 * j]), v = pair_f32<CT>(w[2 * j + 1]);
              const uint32_t f[4] = {__float_as_uint(u.x), __float_as_uint(v.x), __float_as_uint(u.y), __float_as_uint(v.y)};
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                mma8(x[nb], f, pw[j][nb][0], pw[j][nb][1]);
                mma8(x[nb], f, ph[j][nb][0], ph[j][nb][1]);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t h[4], l[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)  // (dim g, key t), (dim g + 8, key t), (.., key t + 4)
                split_tf32_cut(ldsf(vs + elem_at(kw0 + 8 * j + t + 4 * (e >> 1), 16 * mb + g + 8 * (e & 1))), h[e], l[e]);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                mma8(x[nb], l, ph[j][nb][0], ph[j][nb][1]);
                mma8(x[nb], h, pw[j][nb][0], pw[j][nb][1]);
                mma8(x[nb], h, ph[j][nb][0], ph[j][nb][1]);
              }
            }
          }
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mb][nb][e] += x[nb][e];
        }
      }
    }
    cp_wait<0>();
    if (hole_seen && tid == 0) report(a.batch, ST_BAD_PAGE);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) ls[nb][h] += __shfl_xor_sync(0xffffffffu, ls[nb][h], d);
    if (tid == 0 && blk.pos1 >= table) report(a.batch, ST_BAD_PAGE);
    if (tid == 0 && blk.pos0 < 0) report(a.batch, ST_BAD_LEN);

    // four results of row r from dim d on, l and m of the row
    auto finish = [&](int r, int d, float4 x, float m, float l) {
      const int gr = r0 + r;
      const bool some = l > 0.0f || l != l;
      const float inv = some ? 1.0f / l : 0.0f;
      const int64_t tok = sq.r0 + token_of(a, gr);
      const int hh = kvh * a.rep + head_of(a, gr);
      AT* dst = static_cast<AT*>(a.out) + tok * a.out_stride + hh * HD + d;
      const float v0 = some ? x.x * inv : 0.0f, v1 = some ? x.y * inv : 0.0f;
      const float v2 = some ? x.z * inv : 0.0f, v3 = some ? x.w * inv : 0.0f;
      if constexpr (F32A) *reinterpret_cast<float4*>(dst) = make_float4(v0, v1, v2, v3);
      else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<AT>(v0, v1), pack2<AT>(v2, v3));
      if (d == 0 && a.lse) a.lse[tok * a.n_heads + hh] = some ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
    };

    // the four warps' results, joined through shared memory (the ring is empty)
    const bool whole = ta == 0 && tb == blk.tiles;
    float* piece = a.part + (size_t(blockIdx.x) * 2 + (ta == 0 ? 1 : 0)) * size_t(M) * (HD + 2);  // [M][HD], then [M][2]
    {
      float* os = reinterpret_cast<float*>(sm);
      float2* ml = reinterpret_cast<float2*>(sm + 4 * M * L::OPITCH * 4);
      __syncthreads();
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
            os[(warp * M + 8 * nb + 2 * t + (e & 1)) * L::OPITCH + 16 * mb + g + 8 * (e >> 1)] = o[mb][nb][e];
        if (g == 0) {
          ml[warp * M + 8 * nb + 2 * t] = make_float2(mx[nb][0], ls[nb][0]);
          ml[warp * M + 8 * nb + 2 * t + 1] = make_float2(mx[nb][1], ls[nb][1]);
        }
      }
      __syncthreads();
      for (int c = tid; c < rn * (HD / 4); c += AT_THREADS) {
        const int r = c / (HD / 4), d = 4 * (c % (HD / 4));
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w * M + r].x);
        const float u = m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 q = ml[w * M + r];
          const float f = fast_exp2(q.x - u);
          const float4 v = *reinterpret_cast<const float4*>(os + (w * M + r) * L::OPITCH + d);
          l += f * q.y;
          x.x += f * v.x;
          x.y += f * v.y;
          x.z += f * v.z;
          x.w += f * v.w;
        }
        if (whole) finish(r, d, x, m, l);
        else {
          *reinterpret_cast<float4*>(piece + size_t(r) * HD + d) = x;
          if (d == 0) *reinterpret_cast<float2*>(piece + size_t(M) * HD + 2 * r) = make_float2(m, l);
        }
      }
    }

    if (!whole) {
      // The last of the unit's CTAs joins its pieces, in their order. More than GROUP pieces: the last of
      // every `step` of them joins those into the first one's, the last of all the groups (one sequence
      // of 131071 keys, 75 pieces: in one go 98.1 us, by groups 95.6).
      constexpr int GROUP = 8;
      const int c0 = quotient(unit0 + V, pl.per), c1 = quotient(unit0 + V + blk.tiles - 1, pl.per);
      auto part = [&](int p) { return a.part + (size_t(p) * 2 + (p == c0 ? 1 : 0)) * size_t(M) * (HD + 2); };
      // whether this CTA is the last of n at a counter (which is left at zero)
      auto last = [&](int ticket, int n) {
        __threadfence();
        __syncthreads();
        if (tid == 0) s_last = n == 1 || atomicInc(reinterpret_cast<unsigned*>(a.tickets) + ticket, unsigned(n - 1)) == unsigned(n - 1);
        __syncthreads();
        const bool is = s_last;
        if (is) __threadfence();
        return is;
      };
      // pieces from, from + step .. of up to `to`; into the first, or the output
      auto join = [&](int from, int to, int step, bool out) {
        for (int c = tid; c < rn * (HD / 4); c += AT_THREADS) {
          const int r = c / (HD / 4), d = 4 * (c % (HD / 4));
          // eight at a time: their loads are on the way together
          float m = -INFINITY, l = 0.0f;
          float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int p0 = from; p0 <= to; p0 += 8 * step) {
            float2 q[8];
            float4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float* pc = part(p0 + j * step <= to ? p0 + j * step : p0);
              q[j] = __ldcg(reinterpret_cast<const float2*>(pc + size_t(M) * HD + 2 * r));
              v[j] = __ldcg(reinterpret_cast<const float4*>(pc + size_t(r) * HD + d));
            }
            float nm = m;
#pragma unroll
            for (int j = 0; j < 8; ++j) nm = fmaxf(nm, q[j].x);
            const float u = nm == -INFINITY ? 0.0f : nm, f0 = fast_exp2(m - u);
            m = nm;
            l *= f0;
            x = make_float4(x.x * f0, x.y * f0, x.z * f0, x.w * f0);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (p0 + j * step <= to) {
                const float f = fast_exp2(q[j].x - u);
                l += f * q[j].y;
                x.x += f * v[j].x;
                x.y += f * v[j].y;
                x.z += f * v[j].z;
                x.w += f * v[j].w;
              }
          }
          if (out) {
            finish(r, d, x, m, l);
          } else {
            float* to_piece = part(from);
            __syncwarp(HD == 128 ? 0xffffffffu : 0xffffu << (lane & 16));  // a row's threads have read its m and l before one writes them
            *reinterpret_cast<float4*>(to_piece + size_t(r) * HD + d) = x;
            if (d == 0) *reinterpret_cast<float2*>(to_piece + size_t(M) * HD + 2 * r) = make_float2(m, l);
          }
        }
      };
      const int n = c1 - c0 + 1;
      if (n <= GROUP) {
        if (last(c0, n)) join(c0, c1, 1, true);
      } else {
        // counters: a group's is its first CTA's; that of the groups is c0 + 1's, a CTA that no other unit begins in
        const int step = n <= 16 * GROUP ? GROUP : 4 * GROUP;
        const int me = c0 + (int(blockIdx.x) - c0) / step * step, end = min(c1, me + step - 1);
        if (last(me, end - me + 1)) {
          if (end > me) join(me, end, 1, false);
          if (last(c0 + 1, (n + step - 1) / step)) join(c0, c1, step, true);
        }
      }
    }

    if (!next_unit()) break;
  }
}

// The shared-memory limit is a property of a kernel on a device: set the first time a device runs it. Two threads may
// both find it unset and both set it; neither launches before it is.
template <typename K>
cudaError_t allow_shared(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

template <typename AT, typename CT, int HD, int NB>
cudaError_t run_attend(const AttendArgs& a, cudaStream_t st) {
  using L = AttnCfg<AT, CT, HD, NB>;
  static_assert(L::SMEM <= 227 * 1024, "shared memory");
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_shared(attend_kernel<AT, CT, HD, NB>, L::SMEM, done);
  if (e != cudaSuccess) return e;
  CUtensorMap km{}, vm{};
  const int box = make_maps<CT>(&km, &vm, a.pool, L::TK);
  attend_kernel<AT, CT, HD, NB><<<SMS * L::PER_SM, AT_THREADS, L::SMEM, st>>>(a, km, vm, box);
  return cudaGetLastError();
}

template <typename AT, typename CT>
cudaError_t run_attend_rows(const AttendArgs& a, int rows, cudaStream_t st) {
  if (a.pool.head_dim == 64)
    return rows == 8 ? run_attend<AT, CT, 64, 1>(a, st) : rows == 16 ? run_attend<AT, CT, 64, 2>(a, st) : run_attend<AT, CT, 64, 4>(a, st);
  return rows == 8 ? run_attend<AT, CT, 128, 1>(a, st) : rows == 16 ? run_attend<AT, CT, 128, 2>(a, st) : run_attend<AT, CT, 128, 4>(a, st);
}

}  // namespace
}  // namespace paged
}  // namespace wcb
