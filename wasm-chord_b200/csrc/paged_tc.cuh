// What the two tensor-core attention kernels share (paged_attn_tc.cuh: 16-bit
// activations, paged_attn_tc32.cuh: f32 activations): tcgen05 descriptors and instructions, bounded
// waits, the walk over a CTA's units.
#pragma once
#include "paged_attn.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int TC_TK = 128;
constexpr int TILE_PANEL = 128 * 128;  // bytes of 128 rows x 64 dims
constexpr int HOLE_RING = 8;   // tiles: the loaders are at most 4 ahead of the softmax
constexpr int ODD_RING = 16;   // units, likewise

__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
  // 128-byte swizzle, rows of 128 bytes, 8-row groups 1024 bytes apart
  return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_nmajor(uint32_t addr) {
  // the same tile read along its keys: 64-dim panels apart by TILE_PANEL, 8-key groups by 1024 bytes
  return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(TILE_PANEL >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
template <typename T>
constexpr uint32_t idesc(int n, bool b_nmajor) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (b_nmajor ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}

// two f32 operations in one instruction
__device__ __forceinline__ uint64_t pack_f32x2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

struct TcShared {
  uint64_t full[8], empty[8];  // ring slots
  uint64_t q_full[2], s_full[2][2], p_full[2][2], o_done[2][2];  // [row tile][half of the keys]
  uint64_t offs_full, piece_full[2], last_full[2];
  uint64_t drained[2];           // all products of a row tile are done
  uint64_t wait_ns;
  uint32_t tmem;
  int abort;                     // a wait ran out: everybody leaves
  uint32_t holes[HOLE_RING][4];  // keys of a tile without a page
  int odd[ODD_RING];             // by item: a ragged tile has infinities or NaN among its values
  int last[2];
};

// A role's wait; one that gives up takes the others with it.
__device__ __forceinline__ bool tc_wait(TcShared* sh, uint64_t* bar, uint32_t parity) {
  if (bar_wait(bar, parity, sh->wait_ns, &sh->abort)) return true;
  *reinterpret_cast<volatile int*>(&sh->abort) = 1;
  return false;
}

// the same for a whole warp, which goes on or leaves together
__device__ __forceinline__ bool tc_wait_warp(TcShared* sh, uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, tc_wait(sh, bar, parity));
}

// The units of this CTA, walked by every role by itself.
template <int M, int V, bool TREE>  // rows of a block: one or two tiles of 128; what a unit costs beside its tiles, in tiles
struct Walk {
  Place pl;
  long long unit0;  // the unit's first place on the line: V, then its tiles
  int s, kvh, rb, rows, table;
  Seq sq;
  Block blk;
  int ta, tb;  // tiles of the current unit

  // a whole warp; false: the part ends before its first tile
  __device__ __forceinline__ bool start(const AttendArgs& a, const Place& p) {
    pl = p;
    table = table_tokens(a.pool, a.batch);
    s = pl.seq;
    sq = read_seq(a.batch, s);
    rows = seq_rows(a, sq);
    const long long ht = head_tiles<TREE>(a, sq, rows, M, TC_TK, V, table);
    kvh = quotient(pl.begin - pl.seq_begin, ht);
    unit0 = pl.seq_begin + kvh * ht;
    rb = find_block<TREE>(a, sq, rows, M, TC_TK, V, table, pl.begin, unit0);
    blk = row_block<TREE>(a, sq, rows, rb, M, TC_TK, table);
    return cut() || next(a);
  }
  // units of no more tiles than they cost otherwise are not cut: they are the part's that they begin in
  __device__ __forceinline__ bool cut() {
    if (blk.tiles <= V) {
      ta = 0;
      tb = unit0 >= pl.begin ? blk.tiles : 0;
    } else {
      ta = int(max(0LL, pl.begin - unit0 - V));
      tb = int(min(static_cast<long long>(blk.tiles), pl.end - unit0 - V));
    }
    return tb > ta;
  }
  __device__ __forceinline__ bool next(const AttendArgs& a) {
    unit0 += blk.tiles + V;
    if (unit0 >= pl.end) return false;
    ++rb;
    if (rb * M >= rows) {
      rb = 0;
      if (++kvh == a.pool.n_kv) {
        kvh = 0;
        do {
          ++s;
          sq = read_seq(a.batch, s);
          rows = seq_rows(a, sq);
        } while (rows == 0);
      }
    }
    blk = row_block<TREE>(a, sq, rows, rb, M, TC_TK, table);
    return cut();
  }
  // tiles [ta, end) that rows 128 w .. of the block need (those after end see nothing); at least
  // one, so that rows without a key are written too; 0: there are no such rows
  __device__ __forceinline__ int end_of(const AttendArgs& a, int w) const {
    const int r0 = rb * M + 128 * w;
    if (r0 >= rows) return ta;
    if constexpr (TREE) return tb;
    const int r1 = min(rows, r0 + 128);
    const int hi = min(sq.kv - sq.n + token_of(a, r1 - 1) + 1, table);
    const int t = (max(hi, 0) + TC_TK - 1) / TC_TK - blk.tile0;
    return max(min(t, tb), ta + 1);
  }
  // some key of the tile is seen by some rows of the block and not by others, or by none
  __device__ __forceinline__ bool ragged(const AttendArgs& a, int i) const {
    const int key0 = (blk.tile0 + i) * TC_TK;
    return key0 + TC_TK > min(blk.hi, blk.pos0 + 1) || key0 < blk.lo || (a.window > 0 && key0 < blk.pos1 - a.window + 1);
  }
  __device__ __forceinline__ long long key_offset(const AttendArgs& a, int key, bool& hole) const {
    hole = false;
    if (key < blk.lo || key >= blk.hi) return -1;
    const int page = __ldg(a.batch.page_table + int64_t(s) * a.batch.max_pages + key / a.pool.page_size);
    if (page < 0 || page >= a.pool.n_pages) {
      hole = true;
      return -1;
    }
    return page * a.pool.page_stride + int64_t(key % a.pool.page_size) * a.pool.token_stride;
  }
};

// What a row sees: of a chain the keys [lo, hi); of a tree those of its context [lo, context) and, below hi, the new tokens that its mask names.
template <bool TREE>
struct Sight {
  int lo, hi, context;
  const uint32_t* bits;
  __device__ __forceinline__ Sight(const AttendArgs& a, const Seq& q, int token, int table) {
    const int first = q.kv - q.n;
    if constexpr (TREE) {
      context = first;
      hi = min(q.kv, table);
      lo = a.window > 0 ? max(0, first + tree_depth(a, q, token) - a.window + 1) : 0;
      bits = a.mask + int64_t(q.r0 + token) * a.mask_words;
    } else {
      hi = min(first + token + 1, table);
      lo = a.window > 0 ? max(0, first + token - a.window + 1) : 0;
    }
  }
  // bit c: key + c is seen
  __device__ __forceinline__ uint32_t of32(const AttendArgs& a, int key) const {
    auto below = [&](int to) {  // keys below `to`
      const int n = max(0, min(32, to - key));
      return n >= 32 ? 0xffffffffu : (1u << n) - 1u;
    };
    if constexpr (TREE) {
      const int at = key - context, w = at >> 5;
      auto word = [&](int i) { return i >= 0 && i < a.mask_words ? __ldg(bits + i) : 0u; };
      return ((below(context) & ~below(lo)) | (~below(context) & __funnelshift_r(word(w), word(w + 1), at & 31))) & below(hi);
    } else {
      return below(hi) & ~below(lo);
    }
  }
  __device__ __forceinline__ bool has(const AttendArgs& a, int key) const {
    if constexpr (TREE) {
      if (key >= context) return key < hi && tree_bit(a, bits, key - context);
      return key >= lo && key < hi;
    } else {
      return key >= lo && key < hi;
    }
  }
  // the first key from `key` on that may be seen
  __device__ __forceinline__ int from(int key) const { return TREE ? key : max(key, lo); }
};

// byte offset of 16-byte chunk ch of row r in a swizzled tile
__device__ __forceinline__ uint32_t tile_at(int r, int ch) {
  return uint32_t((ch >> 3) * TILE_PANEL + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
}

template <typename T>
__device__ __forceinline__ bool finite16(uint32_t w) {  // both halves
  constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return (w & E) != E && ((w >> 16) & E) != E;
}

}  // namespace
}  // namespace paged
}  // namespace wcb
