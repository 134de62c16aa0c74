// Attention of many new rows over a paged cache on the 5th-generation tensor
// cores, 16-bit activations and cache (the formulas and the line of tiles:
// paged_attn.cuh; here M = 256 rows and TK = 128 keys).
//
// One CTA per SM holds two tiles of 128 rows (row = token * rep + head), each with
// a warpgroup for its softmax (one thread a row: no shuffles) and a thread that
// issues its products; both share the K and V tiles that four loader warps bring
// into a ring of tiles in shared memory: by TMA, in boxes of gcd(page_size, 128) tokens,
// which never cross a page. The values of ragged tiles (the diagonal, the ends) and pools
// whose gcd is below 8 come by 16-byte cp.async, which can leave out single keys (measured:
// 2100 clocks for a 32 KB tile, against the 2048 that a tile of keys takes the tensor
// cores). Per tile of keys:
//   S = Q K^T      tcgen05.mma, both operands from shared memory, S in TMEM (f32)
//   P = 2^(S - m)  read from TMEM, rounded to 16 bits, written back over S
//   O += P V       tcgen05.mma, P from TMEM, V as it lies ([key][dim]: N-major)
// S is made in two halves of 64 keys, each with its own barriers, so that one half's
// products run while the other's exponentials do (S in one piece: every tile
// waited for its own two products, 2.64 ms against 2.42 at the size below; a half
// costs more shared-memory reads of Q, so that the products of a tile of 128 keys
// take 2560 clocks of the SM instead of 2048).
// The running maximum is taken anew only where a half's sum of exponentials shows
// that it has to be (O in TMEM is rescaled then; sums in f32 and P in 16 bits have
// room for the factor): one vote on the sum instead of 64 comparisons a row.
// TMEM: S0 | S1 | O0 | O1, 512 columns at head_dim 128.
//
// 2047 new tokens over 32767 keys, 64/8 heads of 128, bf16: 2.3 ms with new inputs from call to call, 925 TFLOP/s (55 % of
// the measured cuBLAS rate); 1.98 ms at best, run after run. What bounds it: the
// chain within a half, S to registers, exponentials, P back, products, none of which is near its limit by itself (tensor
// pipe 47 %, exponentials 49 %, issue 36 % busy): 1250 clocks a half with both row tiles; without the
// exponentials 600, and the products' 2560 clocks become the bound. Part of the exponentials by a polynomial on the
// multiply-add units (a quarter, an eighth) gained nothing. About 120 bytes of registers spill. Short units: 11
// sequences of 204 tokens 72 us (82 with units that are cut in two for one tile).
// P is rounded once to the 16-bit type: kept in two parts, as for few rows, P V would be two products, and a bf16 output would
// still be off by its own rounding (relative error 1.7e-3 in place of 2.3e-3 at the size above).
#include "paged_tc.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int TC_THREADS = 448;  // 2 softmax warpgroups, 4 loader warps, 2 issuing warps
constexpr int TC_M = 256;
// A half's sum of exponentials may grow to this before the maximum is taken anew, and m then lies so many powers of two below
// it. f16: sums of P up to 2^15, and weights down to 2^-32 of the largest count (P in f16 ends at 2^-24); bf16 has f32's range.
template <typename T>
constexpr float GROWTH = std::is_same<T, __half>::value ? 32768.0f : 8192.0f;
template <typename T>
constexpr float BELOW = std::is_same<T, __half>::value ? 8.0f : 0.0f;
constexpr int UNIT = 3;  // a unit's queries, start and end take about as long as so many tiles of keys

template <int HD>
struct TcCfg {
  static constexpr int PANELS = HD / 64;
  static constexpr int TILE = PANELS * TILE_PANEL;  // bytes of 128 rows x HD
  static constexpr int SLOTS = HD == 128 ? 4 : 6;   // K and V tiles in the ring
  static constexpr int Q = 0;                       // two tiles of queries
  static constexpr int RING = 2 * TILE;
  static constexpr int OFFS = RING + SLOTS * TILE;  // [2][128] row offsets (64 bits)
  static constexpr int BARS = OFFS + 2 * 128 * 8;
  static constexpr int SMEM = BARS + 512 + 1024;    // + alignment to 1024
};

template <typename T, int HD>
__global__ void __launch_bounds__(TC_THREADS, 1)
attend_tc_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap, int box) {
  using L = TcCfg<HD>;
  constexpr int NS = L::SLOTS, CH = HD / 8;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ TcShared sh;
  __shared__ PlaceShared<TC_THREADS> s_place;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sbase = smem_u32(sm);

  const Place pl = find_place<TC_THREADS>(a, TC_M, TC_TK, UNIT, s_place);
  if (pl.begin >= pl.end) return;  // the whole CTA; nothing is held yet
  Walk<TC_M, UNIT> wk;
  if (!wk.start(a, pl)) return;    // likewise

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh.full[i], 4);
      mbar_init(&sh.empty[i], 2);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh.q_full[w], 128);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sh.s_full[w][b], 1);
        mbar_init(&sh.p_full[w][b], 4);
        mbar_init(&sh.o_done[w][b], 1);
      }
      mbar_init(&sh.piece_full[w], 128);
      mbar_init(&sh.last_full[w], 1);
    }
    mbar_init(&sh.offs_full, 128);
    for (int w = 0; w < 2; ++w) mbar_init(&sh.drained[w], 1);
    sh.abort = 0;
    sh.wait_ns = a.wait_ns;
    mbar_fence_init();
  }
  if (tid < ODD_RING) sh.odd[tid] = 0;
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp >= 12) {
    // ---- issuing warps: products of row tile w --------------------------------
    // The whole warp walks the loops, so that addresses and descriptors are uniform values; one
    // lane, always the same, issues.
    const int w = __shfl_sync(0xffffffffu, warp - 12, 0);
    {
      // elect.sync instead of lane == 0: the compiler then keeps descriptors in uniform registers
      // (8 products issue in 600 clocks instead of 940)
      uint32_t elected;
      asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(elected));
      const bool one = elected != 0;
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t ts = tm + 128 * w, to = tm + 256 + 128 * w;
      const uint64_t qd = desc_kmajor(sbase + L::Q + w * L::TILE);
      const uint64_t kd = desc_kmajor(sbase + L::RING), vd = desc_nmajor(sbase + L::RING);
      constexpr uint32_t ID_S = idesc<T>(64, false), ID_O = idesc<T>(HD, true);
      uint32_t slot = 0, phase = 0;  // of the next ring tile
      uint32_t it = 0, t = 0;        // units, and tiles of keys so far
      auto step = [&] {
        if (++slot == NS) {
          slot = 0;
          phase ^= 1;
        }
      };
      // S of half b of the K tile in ring slot ks
      auto product_s = [&](uint32_t ks, int b) {
        tc_fence_after();
        const uint64_t kb = kd + uint64_t(ks * (L::TILE >> 4) + b * (64 * 128 >> 4));
        if (one) {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const uint32_t o = ((k / 4) * TILE_PANEL + (k % 4) * 32) >> 4;
            mma_ss(ts + 64 * b, qd + o, kb + o, ID_S, k > 0);
          }
          tc_commit(&sh.s_full[w][b]);
          if (b) tc_commit(&sh.empty[ks]);
        }
        __syncwarp();
      };
      bool ok = true;
      do {
        const int end = wk.end_of(a, w);
        if (end > wk.ta) {
          ok = tc_wait_warp(&sh, &sh.q_full[w], it & 1) && tc_wait_warp(&sh, &sh.full[slot], phase);
          if (!ok) break;
          product_s(slot, 0);
          product_s(slot, 1);
          ++it;
        }
        for (int i = wk.ta; i < wk.tb && ok; ++i) {
          if (i < end) {  // K of this tile is used up
            step();
            const uint32_t vs = slot;
            const uint64_t vb = vd + uint64_t(vs * (L::TILE >> 4));
            ok = tc_wait_warp(&sh, &sh.full[slot], phase);
            step();
            const bool more = i + 1 < end;
            if (more) ok = ok && tc_wait_warp(&sh, &sh.full[slot], phase);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              ok = ok && tc_wait_warp(&sh, &sh.p_full[w][b], t & 1);
              if (!ok) break;
              tc_fence_after();
              if (one) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_ts(to, ts + 64 * b + 8 * k, vb + (4 * b + k) * (2048 >> 4), ID_O, i > wk.ta || b > 0 || k > 0);
                tc_commit(&sh.o_done[w][b]);
                if (b) tc_commit(&sh.empty[vs]);
              }
              __syncwarp();
              if (more) {  // the next S lies over this P: its product has to be done
                ok = tc_wait_warp(&sh, &sh.o_done[w][b], t & 1);
                if (!ok) break;
                product_s(slot, b);
              }
            }
            ++t;
          } else {  // rows of this tile see none of these keys
            ok = tc_wait_warp(&sh, &sh.full[slot], phase);
            if (!ok) break;
            if (one) bar_arrive(&sh.empty[slot]);
            step();
            ok = tc_wait_warp(&sh, &sh.full[slot], phase);
            if (!ok) break;
            if (one) bar_arrive(&sh.empty[slot]);
            step();
          }
        }
      } while (ok && wk.next(a));
      // the memory of S, P and O is given back after the last product, whether or not the roles came to their ends
      if (one) tc_commit(&sh.drained[w]);
      __syncwarp();
      bar_wait(&sh.drained[w], 0, DRAIN_NS);
    }
  } else if (warp >= 8) {
    // ---- loaders --------------------------------------------------------------
    const int lt = tid - 256;
    long long* offs = reinterpret_cast<long long*>(sm + L::OFFS);
    uint32_t n = 0, tiles = 0, item = 0, by_copy = 0;
    uint32_t issued = 0;  // ring tiles up to the last that came by TMA
    bool ok = true, holes_seen = false;
    // the page of this thread's key of tile i; -1: none
    auto page_of = [&](int i) {
      const int key = (wk.blk.tile0 + i) * TC_TK + lt;
      return key + max(box - 1, 0) >= wk.blk.lo && key < wk.blk.hi  // (a box that begins before the first key)
                 ? __ldg(a.batch.page_table + int64_t(wk.s) * a.batch.max_pages + key / a.pool.page_size)
                 : -1;
    };
    auto room = [&](uint32_t m) {
      return m < NS || tc_wait_warp(&sh, &sh.empty[m % NS], ((m / NS) - 1) & 1);
    };
    do {
      if (lt == 0) sh.odd[(item + ODD_RING / 2) % ODD_RING] = 0;
      const bool many = wk.blk.pos1 > wk.blk.pos0;
      int next = page_of(wk.ta);
      for (int i = wk.ta; i < wk.tb && ok; ++i, ++tiles, n += 2) {
        const int page = next;
        if (i + 1 < wk.tb) next = page_of(i + 1);  // its latency passes while this tile waits for room
        const int key = (wk.blk.tile0 + i) * TC_TK + lt, slot = key % a.pool.page_size;
        const bool in = key >= wk.blk.lo && key < wk.blk.hi, there = in && page >= 0 && page < a.pool.n_pages;
        const unsigned hb = __ballot_sync(0xffffffffu, in && !there);
        if (lane == 0) sh.holes[tiles % HOLE_RING][warp - 8] = hb;
        holes_seen |= hb != 0;
        const bool ragged = wk.ragged(a, i);
        // a ragged tile's keys may be there whole, they are masked; its values have to be looked at
        const int by_tma = box == 0 ? 0 : ragged ? 1 : 2;
        if (by_tma > 0) {
#pragma unroll 1
          for (int kvi = 0; kvi < by_tma && ok; ++kvi) {
            ok = room(n + kvi);
            if (!ok) break;
            uint64_t* bar = &sh.full[(n + kvi) % NS];
            issued = n + kvi + 1;
            if (lane == 0) {  // warp 8's arrival brings the bytes to wait for
              if (warp == 8) mbar_expect_tx(bar, L::TILE + a.withheld);
              else bar_arrive(bar);
            }
            if (lt % box == 0) {
              const uint32_t dst = sbase + L::RING + ((n + kvi) % NS) * L::TILE + lt * 128;
#pragma unroll
              for (int p = 0; p < L::PANELS; ++p)  // a page that is not there: past the last one, zeros
                tma_load(dst + p * TILE_PANEL, kvi ? &vmap : &kmap, 64 * p, wk.kvh, slot, page >= 0 && page < a.pool.n_pages ? page : a.pool.n_pages, bar);
            }
          }
          if (by_tma == 2) continue;
          if (!ok) break;
        }
        offs[(by_copy & 1) * 128 + lt] = there ? page * a.pool.page_stride + int64_t(slot) * a.pool.token_stride : -1;
        bar_arrive(&sh.offs_full);
        ok = tc_wait_warp(&sh, &sh.offs_full, by_copy & 1);
        const long long* ro = offs + (by_copy & 1) * 128;
        ++by_copy;
#pragma unroll 1
        for (int kvi = by_tma; kvi < 2 && ok; ++kvi) {
          ok = room(n + kvi);
          if (!ok) break;
          const T* base = static_cast<const T*>(kvi ? a.pool.v : a.pool.k) + wk.kvh * a.pool.head_stride;
          const uint32_t dst = sbase + L::RING + ((n + kvi) % NS) * L::TILE;
#pragma unroll 8
          for (int c = lt; c < 128 * CH; c += 128) {
            const int r = c / CH, ch = c % CH;
            const long long o = ro[r];
            cp16(dst + tile_at(r, ch), base + (o < 0 ? 0 : o) + ch * 8, o >= 0);
          }
          cp_commit();
        }
        if (!ok) break;
#pragma unroll 1
        for (int kvi = by_tma; kvi < 2; ++kvi) {
          if (kvi == 0) cp_wait<1>();
          else cp_wait<0>();
          // keys that some rows see and others do not: infinities and NaN are taken out of their values
          if (kvi && many && ragged) {
            uint8_t* t = sm + L::RING + ((n + 1) % NS) * L::TILE;
            bool odd = false;
            for (int c = lt; c < 128 * CH; c += 128) {  // the chunks this thread copied
              uint4* x = reinterpret_cast<uint4*>(t + tile_at(c / CH, c % CH));
              const uint4 v = *x;
              if (!(finite16<T>(v.x) && finite16<T>(v.y) && finite16<T>(v.z) && finite16<T>(v.w))) {
                odd = true;
                alignas(16) T e[8];
                *reinterpret_cast<uint4*>(e) = v;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  if (!(fabsf(to_f32(e[j])) <= FLT_MAX)) e[j] = from_f32<T>(0.0f);
                *x = *reinterpret_cast<const uint4*>(e);
              }
            }
            if (odd) sh.odd[item % ODD_RING] = 1;
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) bar_arrive(&sh.full[(n + kvi) % NS]);
        }
      }
      ++item;
    } while (ok && wk.next(a));
    cp_wait<0>();
    // nor does the CTA leave before its boxes have landed: those of the last tiles, if a role gave up
    for (uint32_t m = n > NS ? n - NS : 0; m < issued; ++m) bar_wait(&sh.full[m % NS], (m / NS) & 1, DRAIN_NS);
    if (holes_seen && lane == 0) report(a.batch, ST_BAD_PAGE);
  } else {
    // ---- softmax of row tile w: thread = row ----------------------------------
    const int w = warp >> 2, row = tid & 127;
    const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + 128 * w, to = tmem + lanes + 256 + 128 * w;
    uint32_t tiles = 0, t = 0, item = 0, cuts = 0;  // tiles of the ring, tiles of keys with rows, units, units cut
    bool ok = true;
    // the row tile's queries, and at a unit's end its results on their way out
    uint8_t* qt = sm + L::Q + w * L::TILE;
    constexpr int RPI = 32 / CH;             // rows that a warp moves at once
    const int r32 = 32 * (warp & 3);         // its first row
    do {
      const int r0 = wk.rb * TC_M + 128 * w, rn = min(128, wk.rows - r0);
      const int end = wk.end_of(a, w);
      if (end > wk.ta) {
        // queries into shared memory: a warp its own 32 rows, whole rows at a time; rows that are not there are zeros
        const int gr = r0 + min(row, rn - 1);
        // a row's places in q and out, in its thread; other lanes ask for them
        const long long q_at = (wk.sq.r0 + token_of(a, gr)) * a.q_stride + (wk.kvh * a.rep + head_of(a, gr)) * HD;
        const long long o_at = (wk.sq.r0 + token_of(a, gr)) * a.out_stride + (wk.kvh * a.rep + head_of(a, gr)) * HD;
        {
          uint4 x[32 / RPI];
#pragma unroll
          for (int j = 0; j < 32 / RPI; ++j) {
            const int r = RPI * j + lane / CH;
            const long long from = __shfl_sync(0xffffffffu, q_at, r);
            x[j] = r32 + r < rn ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + from) + lane % CH) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int j = 0; j < 32 / RPI; ++j) *reinterpret_cast<uint4*>(qt + tile_at(r32 + RPI * j + lane / CH, lane % CH)) = x[j];
        }
        fence_proxy_async();
        bar_arrive(&sh.q_full[w]);

        const int pos = wk.sq.kv - wk.sq.n + token_of(a, gr);
        const int khi = min(pos + 1, wk.table), klo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        float m = -INFINITY, l = 0.0f;  // m: the maximum that O and l are scaled by
        for (int i = wk.ta; i < end && ok; ++i) {
          const uint32_t* holes = sh.holes[(tiles + (i - wk.ta)) % HOLE_RING];
          const bool cut = wk.ragged(a, i);
#pragma unroll 1
          for (int b = 0; b < 2; ++b) {
            ok = tc_wait_warp(&sh, &sh.s_full[w][b], t & 1);
            if (!ok) break;
            tc_fence_after();
            const int key0 = (wk.blk.tile0 + i) * TC_TK + 64 * b;
            // bit c: key key0 + c is seen; mask: some row of the warp does not see all of them
            uint32_t seen[2];
            bool mask = false;
            if (cut || (holes[2 * b] | holes[2 * b + 1]) != 0) {
              const int lo = max(0, min(64, klo - key0)), hi = max(0, min(64, khi - key0));
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const int b0 = max(0, min(32, lo - 32 * q)), b1 = max(0, min(32, hi - 32 * q));
                const uint32_t below1 = b1 >= 32 ? 0xffffffffu : (1u << b1) - 1u, below0 = b0 >= 32 ? 0xffffffffu : (1u << b0) - 1u;
                seen[q] = below1 & ~below0 & ~holes[2 * b + q];
              }
              mask = __any_sync(0xffffffffu, (seen[0] & seen[1]) != 0xffffffffu);
            }
            // the row's 64 products in registers: TMEM is read once
            uint32_t v[64];
#pragma unroll
            for (int q = 0; q < 2; ++q) tmem_ld32(ts + 64 * b + 32 * q, *reinterpret_cast<uint32_t(*)[32]>(v + 32 * q));
            tmem_wait_ld();
            if (mask) {
              const uint32_t none = a.scale_log2 < 0.0f ? 0x7f800000u : 0xff800000u;  // -infinity once scaled
#pragma unroll
              for (int e = 0; e < 64; ++e)
                if (!((seen[e / 32] >> (e % 32)) & 1)) v[e] = none;
            }
            const uint64_t scale2 = pack_f32x2(a.scale_log2, a.scale_log2);
            uint64_t sum[2];
            auto exponentials = [&] {  // P, into S's place, and its sum
              const float use = m == -INFINITY ? 0.0f : m;
              const uint64_t use2 = pack_f32x2(-use, -use);
              sum[0] = sum[1] = 0;
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  float x, y;
                  const uint64_t z = fma_f32x2(pack_f32x2(__uint_as_float(v[32 * q + 2 * e]), __uint_as_float(v[32 * q + 2 * e + 1])), scale2, use2);
                  unpack_f32x2(z, x, y);
                  x = fast_exp2(x);
                  y = fast_exp2(y);
                  sum[e & 1] = add_f32x2(sum[e & 1], pack_f32x2(x, y));
                  p[e] = pack2<T>(x, y);
                }
                tmem_st16(ts + 64 * b + 16 * q, p);
              }
            };
            auto total = [&] {
              float x0, y0, x1, y1;
              unpack_f32x2(sum[0], x0, y0);
              unpack_f32x2(sum[1], x1, y1);
              return (x0 + y0) + (x1 + y1);
            };
            // Most halves need no maximum: the last one still serves as long as the sum shows that no
            // exponential left the range of f16 and of a sound sum; a row's sum is wanted anyway.
            // A row decides by its own sum alone, so that its result does not depend on what its neighbours see.
            float part = 0.0f;
            bool moves = m == -INFINITY;
            if (!__all_sync(0xffffffffu, moves)) {
              exponentials();
              part = total();
              moves = moves || !(part <= GROWTH<T>);
            }
            const bool again = __any_sync(0xffffffffu, moves);
            if (again) {
              float top;
              if (a.scale_log2 >= 0.0f) {
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 64; e += 8)
#pragma unroll
                  for (int j = 0; j < 4; ++j) x[j] = max3(x[j], __uint_as_float(v[e + 2 * j]), __uint_as_float(v[e + 2 * j + 1]));
                top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * a.scale_log2;
              } else {  // a negative scale turns the order round
                float x = INFINITY;
#pragma unroll
                for (int e = 0; e < 64; ++e) x = fminf(x, __uint_as_float(v[e]));
                top = x * a.scale_log2;
              }
              const float nm = moves ? fmaxf(m, top - BELOW<T>) : m;
              if (__any_sync(0xffffffffu, nm > m)) {
                const float f = m == nm ? 1.0f : fast_exp2(m - (nm == -INFINITY ? 0.0f : nm));
                if (i > wk.ta || b) {  // after the last product
                  ok = tc_wait_warp(&sh, &sh.o_done[w][1 - b], (b ? t : t - 1) & 1);
                  if (!ok) break;
                  tc_fence_after();
#pragma unroll 1
                  for (int q = 0; q < HD / 16; ++q) {
                    uint32_t o[16];
                    tmem_ld16(to + 16 * q, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_st16(to + 16 * q, o);
                  }
                }
                l *= f;
                m = nm;
              }
              tmem_wait_st();  // the first P lies in the same columns: two stores have no order of their own
              exponentials();
              part = total();
            }
            l += part;
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.p_full[w][b]);
          }
          ++t;
        }
        if (ok) ok = tc_wait_warp(&sh, &sh.o_done[w][1], (t - 1) & 1);
        if (!ok) break;
        tc_fence_after();

        // results: normalised, or a piece [HD][256] + m [256] + l [256]
        const bool whole = wk.ta == 0 && wk.tb == wk.blk.tiles;
        constexpr size_t PIECE = size_t(TC_M) * (HD + 2);
        float* piece = a.part + (size_t(blockIdx.x) * 2 + (wk.ta == 0 ? 1 : 0)) * PIECE + 128 * w + row;
        const bool odd = *reinterpret_cast<volatile int*>(&sh.odd[item % ODD_RING]) != 0;
        const int64_t tok = wk.sq.r0 + token_of(a, gr);
        const int hh = wk.kvh * a.rep + head_of(a, gr);
        const bool some = (l > 0.0f && m > -INFINITY) || l != l;
        const float inv = some ? 1.0f / l : 0.0f;
        // rows leave through shared memory, each warp its own: a thread's row by itself would be 32 lines a store
        auto stage = [&](const float (&x)[32], int q) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint4 y;
            y.x = pack2<T>(x[8 * c], x[8 * c + 1]);
            y.y = pack2<T>(x[8 * c + 2], x[8 * c + 3]);
            y.z = pack2<T>(x[8 * c + 4], x[8 * c + 5]);
            y.w = pack2<T>(x[8 * c + 6], x[8 * c + 7]);
            *reinterpret_cast<uint4*>(qt + tile_at(row, 4 * q + c)) = y;
          }
        };
        auto send = [&] {
          __syncwarp();
#pragma unroll 4
          for (int j = 0; j < 32 / RPI; ++j) {
            const int r = RPI * j + lane / CH;
            const long long to_at = __shfl_sync(0xffffffffu, o_at, r);
            if (r32 + r < rn)
              *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to_at + 8 * (lane % CH)) = *reinterpret_cast<const uint4*>(qt + tile_at(r32 + r, lane % CH));
          }
          __syncwarp();
        };
#pragma unroll 1
        for (int q = 0; q < HD / 32; ++q) {
          uint32_t v[32];
          tmem_ld32(to + 32 * q, v);
          tmem_wait_ld();
          if (odd) {
            // infinities and NaN that were taken out of ragged tiles, for the rows that see them
#pragma unroll 1
            for (int i = wk.ta; i < end; ++i) {
              if (!wk.ragged(a, i)) continue;
              const int k0 = (wk.blk.tile0 + i) * TC_TK;
#pragma unroll 1
              for (int key = max(k0, klo); key < min(k0 + TC_TK, khi); ++key) {
                bool hole;
                const long long off = wk.key_offset(a, key, hole);
                if (off < 0) continue;
                const T* vp = static_cast<const T*>(a.pool.v) + wk.kvh * a.pool.head_stride + off + 32 * q;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float x = to_f32(vp[e]);
                  if (!(fabsf(x) <= FLT_MAX)) v[e] = __float_as_uint(__uint_as_float(v[e]) + x);
                }
              }
            }
          }
          if (whole) {
            float x[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = some ? __uint_as_float(v[e]) * inv : 0.0f;
            stage(x, q);
          } else if (row < rn) {
#pragma unroll
            for (int e = 0; e < 32; ++e) piece[size_t(32 * q + e) * TC_M] = __uint_as_float(v[e]);
          }
        }
        tc_fence_before();
        if (whole) send();
        if (row < rn) {
          if (whole) {
            if (a.lse) a.lse[tok * a.n_heads + hh] = some ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
          } else {
            piece[size_t(HD) * TC_M] = m;
            piece[size_t(HD + 1) * TC_M] = l;
          }
        }
        if (row == 0 && w == 0) {
          uint32_t bits = 0;
          if (wk.blk.pos1 >= wk.table) bits |= ST_BAD_PAGE;
          if (wk.blk.pos0 < 0) bits |= ST_BAD_LEN;
          report(a.batch, bits);
        }
        if (!whole) {
          // the last of the unit's CTAs joins this tile's pieces, in their order
          const int c0 = quotient(wk.unit0 + UNIT, wk.pl.per), c1 = quotient(wk.unit0 + UNIT + wk.blk.tiles - 1, wk.pl.per);
          __threadfence();
          bar_arrive(&sh.piece_full[w]);
          ok = tc_wait_warp(&sh, &sh.piece_full[w], cuts & 1);
          if (!ok) break;
          if (row == 0) {
            sh.last[w] = atomicInc(reinterpret_cast<unsigned*>(a.tickets) + TC_TICKETS + 2 * c0 + w, unsigned(c1 - c0)) == unsigned(c1 - c0);
            bar_arrive(&sh.last_full[w]);
          }
          ok = tc_wait_warp(&sh, &sh.last_full[w], cuts & 1);
          if (!ok) break;
          ++cuts;
          if (sh.last[w]) {
            __threadfence();
            auto part = [&](int p) { return a.part + (size_t(p) * 2 + (p == c0 ? 1 : 0)) * PIECE + 128 * w + row; };
            float jm = -INFINITY, jl = 0.0f;
            if (row < rn)
              for (int p = c0; p <= c1; ++p) jm = fmaxf(jm, __ldcg(part(p) + size_t(HD) * TC_M));
            const float u = jm == -INFINITY ? 0.0f : jm;
            if (row < rn)
              for (int p = c0; p <= c1; ++p) jl += fast_exp2(__ldcg(part(p) + size_t(HD) * TC_M) - u) * __ldcg(part(p) + size_t(HD + 1) * TC_M);
            const bool any = jl > 0.0f || jl != jl;
            const float jinv = any ? 1.0f / jl : 0.0f;
#pragma unroll 1
            for (int q = 0; q < HD / 32; ++q) {
              float x[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = 0.0f;
              if (row < rn) {
#pragma unroll 2
                for (int p = c0; p <= c1; ++p) {
                  const float* pp = part(p);
                  const float f = fast_exp2(__ldcg(pp + size_t(HD) * TC_M) - u);
#pragma unroll
                  for (int e = 0; e < 32; ++e) x[e] = fmaf(f, __ldcg(pp + size_t(32 * q + e) * TC_M), x[e]);
                }
              }
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = any ? x[e] * jinv : 0.0f;
              stage(x, q);
            }
            send();
            if (a.lse && row < rn) a.lse[tok * a.n_heads + hh] = any ? (jm + log2f(jl)) * 0.69314718055994531f : -INFINITY;
          }
        }
      }
      tiles += uint32_t(wk.tb - wk.ta);
      ++item;
    } while (ok && wk.next(a));
    tmem_wait_ld();
    tmem_wait_st();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && sh.abort) report(a.batch, ST_ABORTED);
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <typename T, int HD>
cudaError_t run_tc(const AttendArgs& a, cudaStream_t s) {
  using L = TcCfg<HD>;
  static_assert(L::SMEM + sizeof(TcShared) + sizeof(PlaceShared<TC_THREADS>) <= 227 * 1024, "shared memory");
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_shared(attend_tc_kernel<T, HD>, L::SMEM, done);
  if (e != cudaSuccess) return e;
  CUtensorMap km{}, vm{};
  const int box = make_maps<T>(&km, &vm, a.pool, TC_TK);
  attend_tc_kernel<T, HD><<<TC_CTAS, TC_THREADS, L::SMEM, s>>>(a, km, vm, box);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attend_tc(const AttendArgs& a, int act, cudaStream_t s) {
  if (act == E_F16) return a.pool.head_dim == 64 ? run_tc<__half, 64>(a, s) : run_tc<__half, 128>(a, s);
  return a.pool.head_dim == 64 ? run_tc<__nv_bfloat16, 64>(a, s) : run_tc<__nv_bfloat16, 128>(a, s);
}

}  // namespace paged
}  // namespace wcb
