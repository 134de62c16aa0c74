// Attention of many new rows over a paged cache on the 5th-generation tensor
// cores, f32 activations over a cache of any type (the formulas and the line of tiles:
// paged_attn.cuh; the 16-bit kernel this one is built like: paged_attn_tc.cuh).
//
// f32 numbers go to the tensor cores as sums of two f16 numbers, x = 2^e (hi + lo), 22 bits: the
// exponents are a row's (q) or 8 keys' (k and v), so that the largest of them lies below 2^14 and
// what is lost of the others is below 2^-38 of it. 8 keys whose largest numbers are farther apart than 2^16 stay out of the products:
// each row that sees one adds it in ordinary f32 arithmetic, so that a large key or value, of a later token for instance,
// takes no bits from what other rows see. P is split with an exponent of each row's own for 64 keys, that of
// the largest weight times the size of its values among the keys that the row sees. An f16 cache needs no
// splitting; a bf16 cache is widened and split like an f32 one (its range is f32's).
//   S  = Qlo Khi + Qhi Klo + Qhi Khi             (two products over an f16 cache)
//   O' = Plo Vhi + Phi Vlo + Phi Vhi             (one half of 64 keys)
//   O  = O 2^(m - m') + O' 2^e                   in registers, by ordinary f32 arithmetic
// The last line is why this is not the 16-bit kernel with more products: sums in TMEM over a long
// sequence are cut off at every step, which f32 outputs would show; over 64 keys they are not. TMEM: S of each
// row tile in two halves of 64 keys, over which Phi and Plo are written (16 columns in place of 16), and two O' of each
// row tile, one of them being added to O while the products of the next are made.
//
// Keys and values of an f32 cache are loaded, scaled and split by eight loader warps (each 8 keys
// of a half, so a group's exponent is one warp's affair); those of an f16 cache come by TMA where
// the tile is whole. head_dim 64: two row tiles of 128 rows; 128: one (Q in two parts and a
// ring of K and V in two parts fill the shared memory).
//
// 46 sequences of 919 tokens, 32/4 heads of 64, f32 cache: 1.19 ms, 134 TFLOP/s of the formula's
// products, 402 of those made (24 % of the measured cuBLAS rate); one of 2048 tokens over 16384 keys
// 1.12 ms, 234 and 694 TFLOP/s (42 %). The rows' own exponents of P and the search for keys that are far apart are 1 to
// 7 % of that (an exponent for each key instead, read by a second way through the softmax: 10 %); a call all of whose
// keys are far apart takes a hundred times as long. What bounds it: the
// instructions of the splitting, in the softmax (P) and in the loaders (K and V), about 500 bytes of registers that
// spill in each kernel, and at few tiles a unit's start and end.
#pragma once
#include "paged_tc.cuh"

namespace wcb {
namespace paged {
namespace {

template <typename CT, int HD>
struct Tc32Cfg {
  static constexpr bool F32C = !std::is_same<CT, __half>::value;  // f32, or bf16 widened to it: not exact in f16
  static constexpr int RT = HD == 64 ? 2 : 1;       // row tiles
  static constexpr int M = 128 * RT;
  static constexpr int LW = F32C ? 8 : 4;           // loader warps: those of an f32 cache have the splitting to do
  static constexpr int WGS = RT + LW / 4 + 1;       // softmax warpgroups, loaders, issuing warps
  static constexpr int THREADS = 128 * WGS;
  static constexpr int PART = HD / 64 * TILE_PANEL;  // bytes of 128 rows x HD in f16
  static constexpr int SLOT = (F32C ? 2 : 1) * PART;
  static constexpr int SLOTS = F32C ? (HD == 64 ? 4 : 2) : (HD == 64 ? 6 : 4);
  static constexpr int Q = 0;                        // [row tile][hi, lo]
  static constexpr int RING = RT * 2 * PART;
  static constexpr int OFFS = RING + SLOTS * SLOT;   // [2][128] row offsets (f16 cache)
  static constexpr int SMEM = OFFS + 2 * 128 * 8 + 1024;
  // registers of a thread by role; together no more than the launch's (two row tiles, f32: softmax 168 and loaders 48 took
  // a tenth more for 2048 tokens over 16384 keys; 152 and 64 more than either at short units)
  static constexpr int LAUNCH = 65536 / THREADS / 8 * 8;
  static constexpr int R_MMA = 40, R_LOAD = F32C ? (RT == 2 ? 56 : 96) : 80;
  static constexpr int R_SOFT = RT == 2 ? (F32C ? 160 : 192) : 240;
  static_assert(RT * R_SOFT + LW / 4 * R_LOAD + R_MMA <= WGS * LAUNCH, "register split");
};

constexpr int EXP_RING = 8;  // tiles
constexpr int UNIT = 2;      // a unit's queries, start and end take about as long as so many tiles of keys

constexpr float WIDE = 1.0f / 65536;  // 8 keys whose numbers are farther apart than this do not share an exponent

struct Tc32Shared : TcShared {
  // of 8 keys: their numbers are so many times (a power of two, of values its exponent too) what the tile holds (read four at a time)
  alignas(16) float kfac[EXP_RING][16];
  alignas(16) float vfac[EXP_RING][16];
  alignas(16) float vexp[EXP_RING][16];
  alignas(8) uint32_t apart[HOLE_RING][4];  // keys that the products leave out for that
};

__device__ __forceinline__ float pow2(int e) { return __int_as_float((max(-126, min(127, e)) + 127) << 23); }
// the exponent that brings numbers up to `top` below 2^14; `none` where there are only zeros
__device__ __forceinline__ int group_exp(float top, int none) {
  const int e = int(__float_as_uint(top) >> 23) - 127;  // top in [2^e, 2^(e + 1)); below 2^-126: -127
  return top > 0.0f ? max(-126, min(120, e - 13)) : none;
}
// (two f32 operations in one instruction)
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// two finite numbers as two f16 each
__device__ __forceinline__ void split_f16(uint64_t z, uint32_t& hi, uint32_t& lo) {
  float x, y;
  unpack_f32x2(z, x, y);
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  unpack_f32x2(add_f32x2(z, pack_f32x2(-f.x, -f.y)), x, y);
  lo = pack2<__half>(x, y);
}

template <typename CT, int HD, bool TREE>
__global__ void __launch_bounds__((Tc32Cfg<CT, HD>::THREADS), 1)
attend_tc32_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, int box) {
  using L = Tc32Cfg<CT, HD>;
  constexpr bool F32C = L::F32C;
  constexpr int NS = L::SLOTS, RT = L::RT, M = L::M, MMA_WARP = 4 * RT + L::LW;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ Tc32Shared sh;
  __shared__ PlaceShared<L::THREADS> s_place;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sbase = smem_u32(sm);

  const Place pl = find_place<L::THREADS, TREE>(a, M, TC_TK, UNIT, s_place);
  if (pl.begin >= pl.end) return;  // the whole CTA; nothing is held yet
  Walk<M, UNIT, TREE> wk;
  if (!wk.start(a, pl)) return;    // likewise

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh.full[i], L::LW);
      mbar_init(&sh.empty[i], RT);
    }
    for (int w = 0; w < RT; ++w) {
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
    for (int w = 0; w < RT; ++w) mbar_init(&sh.drained[w], 1);
    sh.abort = 0;
    sh.wait_ns = a.wait_ns;
    mbar_fence_init();
  }
  if (tid < ODD_RING) sh.odd[tid] = 0;
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp >= MMA_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::R_MMA));
    // ---- issuing warps (paged_attn_tc.cuh says how) ------------------------------
    const int w = __shfl_sync(0xffffffffu, warp - MMA_WARP, 0);
    if (w < RT) {
      uint32_t elected;
      asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(elected));
      const bool one = elected != 0;
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t ts = tm + 128 * w, to = tm + 256 + 128 * w;  // (one row tile: O' of 128 columns at 256 and 384)
      const uint64_t qd = desc_kmajor(sbase + L::Q + w * 2 * L::PART);
      const uint64_t kd = desc_kmajor(sbase + L::RING), vd = desc_nmajor(sbase + L::RING);
      constexpr uint32_t ID_S = idesc<__half>(64, false), ID_O = idesc<__half>(HD, true);
      constexpr uint32_t LO = L::PART >> 4;  // from a tile's hi to its lo, in descriptors
      uint32_t slot = 0, phase = 0;          // of the next ring tile
      uint32_t it = 0, t = 0;                // units, and tiles of keys so far
      auto step = [&] {
        if (++slot == NS) {
          slot = 0;
          phase ^= 1;
        }
      };
      auto product_s = [&](uint32_t ks, int b) {
        tc_fence_after();
        const uint64_t kb = kd + uint64_t(ks * (L::SLOT >> 4) + b * (64 * 128 >> 4));
        if (one) {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const uint32_t o = ((k / 4) * TILE_PANEL + (k % 4) * 32) >> 4;
            mma_ss(ts + 64 * b, qd + LO + o, kb + o, ID_S, k > 0);
            if (F32C) mma_ss(ts + 64 * b, qd + o, kb + LO + o, ID_S, 1);
          }
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const uint32_t o = ((k / 4) * TILE_PANEL + (k % 4) * 32) >> 4;
            mma_ss(ts + 64 * b, qd + o, kb + o, ID_S, 1);
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
            const uint64_t vb = vd + uint64_t(vs * (L::SLOT >> 4));
            ok = tc_wait_warp(&sh, &sh.full[slot], phase);
            step();
            const bool more = i + 1 < end;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              ok = ok && tc_wait_warp(&sh, &sh.p_full[w][b], t & 1);
              if (!ok) break;
              tc_fence_after();
              if (one) {
                const uint32_t od = to + HD * b;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const uint64_t v = vb + (4 * b + k) * (2048 >> 4);
                  mma_ts(od, ts + 64 * b + 16 * k + 8, v, ID_O, k > 0);
                  if (F32C) mma_ts(od, ts + 64 * b + 16 * k, v + LO, ID_O, 1);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_ts(od, ts + 64 * b + 16 * k, vb + (4 * b + k) * (2048 >> 4), ID_O, 1);
                tc_commit(&sh.o_done[w][b]);
                if (b) tc_commit(&sh.empty[vs]);
              }
              __syncwarp();
              if (more) {  // the next S lies over this P: its product has to be done
                if (b == 0) ok = tc_wait_warp(&sh, &sh.full[slot], phase);
                ok = ok && tc_wait_warp(&sh, &sh.o_done[w][b], t & 1);
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
  } else if (warp >= 4 * RT) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::R_LOAD));
    // ---- loaders --------------------------------------------------------------
    const int lt = tid - 128 * RT, lw = warp - 4 * RT;
    long long* offs = reinterpret_cast<long long*>(sm + L::OFFS);
    uint32_t n = 0, tiles = 0, item = 0, by_copy = 0;
    uint32_t issued = 0;  // ring tiles up to the last that came by TMA
    bool ok = true, holes_seen = false;
    // this thread's key of a tile. f32: 8 keys of each half are one warp's (lanes 0 .. 7, 8 .. 15; the others have none)
    const int my_key = F32C ? 64 * ((lane >> 3) & 1) + 8 * lw + (lane & 7) : lt;
    auto page_of = [&](int i) {
      const int key = (wk.blk.tile0 + i) * TC_TK + my_key;
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
        if (i + 1 < wk.tb) next = page_of(i + 1);
        const int key = (wk.blk.tile0 + i) * TC_TK + my_key, at_slot = key % a.pool.page_size;
        const bool in = key >= wk.blk.lo && key < wk.blk.hi, there = in && page >= 0 && page < a.pool.n_pages;
        const unsigned hb = __ballot_sync(0xffffffffu, in && !there) & (F32C ? 0xffffu : 0xffffffffu);
        if (lane == 0) {
          if (F32C) {
            uint8_t* h = reinterpret_cast<uint8_t*>(sh.holes[tiles % HOLE_RING]);  // by 8 keys
            h[lw] = uint8_t(hb);
            h[8 + lw] = uint8_t(hb >> 8);
            uint8_t* x = reinterpret_cast<uint8_t*>(sh.apart[tiles % HOLE_RING]);
            x[lw] = x[8 + lw] = 0;
          } else {
            sh.holes[tiles % HOLE_RING][lw] = hb;
          }
        }
        holes_seen |= hb != 0;
        const long long off = there ? page * a.pool.page_stride + int64_t(at_slot) * a.pool.token_stride : -1;
        if constexpr (F32C) {
          constexpr int LPR = HD / 8;        // lanes of a row (8 numbers each): 8 or 16
          constexpr int RPI = 32 / LPR;      // rows of an iteration
          constexpr int IT = 2 * 8 / RPI;    // 16-byte words of a lane: two of each of its rows
          const int sub = lane % LPR, rr = lane / LPR;
          const CT* base[2] = {static_cast<const CT*>(a.pool.k) + wk.kvh * a.pool.head_stride + 8 * sub,
                                  static_cast<const CT*>(a.pool.v) + wk.kvh * a.pool.head_stride + 8 * sub};
          // K's halves, V's halves: the next one is on its way while one is split. (A rolled loop, like all that is long here:
          // the roles' code together has to stay in the instruction cache. Unrolled, the kernel took 1.81 ms where
          // it took 1.50 ms at 46 sequences of 919 new tokens, 32/4 heads of 64.)
          float4 y[IT], ahead[IT];
          auto load = [&](int u) {
            const CT* from = u < 2 ? base[0] : base[1];
#pragma unroll
            for (int j = 0; j < IT; j += 2) {
              const long long o = __shfl_sync(0xffffffffu, off, 8 * (u & 1) + RPI * (j / 2) + rr);
              if constexpr (std::is_same<CT, float>::value) {
                ahead[j] = o >= 0 ? __ldg(reinterpret_cast<const float4*>(from + o)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                ahead[j + 1] = o >= 0 ? __ldg(reinterpret_cast<const float4*>(from + o) + 1) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              } else {
                const uint4 w = o >= 0 ? __ldg(reinterpret_cast<const uint4*>(from + o)) : make_uint4(0, 0, 0, 0);
                auto widen = [](uint32_t x, uint32_t y) {  // (a bf16 is the upper half of its f32)
                  return make_float4(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u), __uint_as_float(y << 16), __uint_as_float(y & 0xffff0000u));
                };
                ahead[j] = widen(w.x, w.y);
                ahead[j + 1] = widen(w.z, w.w);
              }
            }
          };
#pragma unroll 1
          for (int u = -1; u < 4; ++u) {
            const int kvi = u >> 1, b = u & 1;
#pragma unroll
            for (int j = 0; j < IT; ++j) y[j] = ahead[j];
            if (u < 3) load(u + 1);
            if (u < 0) continue;
            if (b == 0) {
              ok = ok && room(n + kvi);
              if (!ok) break;
            }
            // the largest of 8 numbers each, of all 8 keys, and the smallest of the former that is not zero
            float top = 0.0f, low = INFINITY, t8[IT / 2];
            uint64_t zero = 0;  // NaN where a number is not finite
#pragma unroll
            for (int j = 0; j < IT; ++j) {
              const float t = fmaxf(fmaxf(fabsf(y[j].x), fabsf(y[j].y)), fmaxf(fabsf(y[j].z), fabsf(y[j].w)));
              t8[j / 2] = j % 2 ? fmaxf(t8[j / 2], t) : t;
              zero = fma_f32x2(pack_f32x2(y[j].x, y[j].y), 0, zero);
              zero = fma_f32x2(pack_f32x2(y[j].z, y[j].w), 0, zero);
            }
            float z0, z1;
            unpack_f32x2(zero, z0, z1);
            const bool bad = __any_sync(0xffffffffu, z0 != z0 || z1 != z1);
            if (bad) {
              // infinities and NaN take no part in the exponent; a value's is added to O at the end, to the
              // rows that see it
              bool odd = false;
#pragma unroll
              for (int j = 0; j < IT; ++j) {
                if (j % 2 == 0) t8[j / 2] = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float& v = (&y[j].x)[e];
                  if (fabsf(v) <= FLT_MAX) {
                    t8[j / 2] = fmaxf(t8[j / 2], fabsf(v));
                  } else if (kvi) {
                    odd = true;
                    v = 0.0f;
                  }
                }
              }
              if (odd) sh.odd[item % ODD_RING] = 1;
            }
#pragma unroll
            for (int j = 0; j < IT / 2; ++j) {
              top = fmaxf(top, t8[j]);
              if (t8[j] > 0.0f) low = fminf(low, t8[j]);
            }
            // (the bits of numbers that are not negative are in their order)
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
            low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(low)));
            const int none = kvi ? -126 : 0;  // zeros among values never make the largest exponent
            const int ge = group_exp(top, none);
            // Farther apart than WIDE, a key against the others? (The first look takes 8 numbers by themselves, which is cheap; a key's
            // own small ones lose nothing that shows beside its large ones.)
            if (low < top * WIDE) {
              low = INFINITY;
#pragma unroll
              for (int j = 0; j < IT / 2; ++j) {
                float t = t8[j];
#pragma unroll
                for (int d = LPR / 2; d > 0; d >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
                if (t > 0.0f) low = fminf(low, t);
              }
              low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(low)));
            }
            if (lane == 0) {
              const int at = 8 * b + lw, r = tiles % EXP_RING;
              if (kvi) {
                sh.vfac[r][at] = pow2(ge);
                sh.vexp[r][at] = float(ge);
              } else {
                sh.kfac[r][at] = pow2(ge);
              }
              if (low < top * WIDE) {
                // what is large in one key, seen or not, would take the others' bits: the rows that see
                // these keys add them by themselves (those without a page are left out already)
                uint8_t* h = reinterpret_cast<uint8_t*>(sh.holes[tiles % HOLE_RING]) + at;
                uint8_t* x = reinterpret_cast<uint8_t*>(sh.apart[tiles % HOLE_RING]) + at;
                *x |= uint8_t(~*h);
                *h = 0xff;
              }
            }
            const uint64_t f = pack_f32x2(pow2(-ge), pow2(-ge));
            uint8_t* dst = sm + L::RING + ((n + kvi) % NS) * L::SLOT;
#pragma unroll
            for (int j = 0; j < IT; j += 2) {
              uint4 h, l;
              split_f16(mul_f32x2(pack_f32x2(y[j].x, y[j].y), f), h.x, l.x);
              split_f16(mul_f32x2(pack_f32x2(y[j].z, y[j].w), f), h.y, l.y);
              split_f16(mul_f32x2(pack_f32x2(y[j + 1].x, y[j + 1].y), f), h.z, l.z);
              split_f16(mul_f32x2(pack_f32x2(y[j + 1].z, y[j + 1].w), f), h.w, l.w);
              if (bad) {  // an infinity or NaN stays in hi alone
                if (!finite16<__half>(h.x) || !finite16<__half>(h.y) || !finite16<__half>(h.z) || !finite16<__half>(h.w)) l = make_uint4(0, 0, 0, 0);
              }
              const uint32_t o = tile_at(64 * b + 8 * lw + RPI * (j / 2) + rr, sub);
              *reinterpret_cast<uint4*>(dst + o) = h;
              *reinterpret_cast<uint4*>(dst + L::PART + o) = l;
            }
            if (b == 1) {
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) bar_arrive(&sh.full[(n + kvi) % NS]);
            }
          }
        } else {
          constexpr int CH = HD / 8;
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
              if (lane == 0) {  // the first warp's arrival brings the bytes to wait for
                if (lw == 0) mbar_expect_tx(bar, L::SLOT + a.withheld);
                else bar_arrive(bar);
              }
              if (lt % box == 0) {
                const uint32_t dst = sbase + L::RING + ((n + kvi) % NS) * L::SLOT + lt * 128;
#pragma unroll
                for (int p = 0; p < HD / 64; ++p)  // a page that is not there: past the last one, zeros
                  tma_load(dst + p * TILE_PANEL, kvi ? &vmap : &kmap, 64 * p, wk.kvh, at_slot, page >= 0 && page < a.pool.n_pages ? page : a.pool.n_pages, bar);
              }
            }
            if (by_tma == 2) continue;
            if (!ok) break;
          }
          offs[(by_copy & 1) * 128 + lt] = off;
          bar_arrive(&sh.offs_full);
          ok = tc_wait_warp(&sh, &sh.offs_full, by_copy & 1);
          const long long* ro = offs + (by_copy & 1) * 128;
          ++by_copy;
#pragma unroll 1
          for (int kvi = by_tma; kvi < 2 && ok; ++kvi) {
            ok = room(n + kvi);
            if (!ok) break;
            const __half* base = static_cast<const __half*>(kvi ? a.pool.v : a.pool.k) + wk.kvh * a.pool.head_stride;
            const uint32_t dst = sbase + L::RING + ((n + kvi) % NS) * L::SLOT;
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
              uint8_t* t = sm + L::RING + ((n + 1) % NS) * L::SLOT;
              bool odd = false;
              for (int c = lt; c < 128 * CH; c += 128) {  // the chunks this thread copied
                uint4* x = reinterpret_cast<uint4*>(t + tile_at(c / CH, c % CH));
                const uint4 v = *x;
                if (!(finite16<__half>(v.x) && finite16<__half>(v.y) && finite16<__half>(v.z) && finite16<__half>(v.w))) {
                  odd = true;
                  alignas(16) __half e[8];
                  *reinterpret_cast<uint4*>(e) = v;
#pragma unroll
                  for (int j = 0; j < 8; ++j)
                    if (!(fabsf(to_f32(e[j])) <= FLT_MAX)) e[j] = from_f32<__half>(0.0f);
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
      }
      ++item;
    } while (ok && wk.next(a));
    cp_wait<0>();
    // nor does the CTA leave before its boxes have landed: those of the last tiles, if a role gave up
    for (uint32_t m = n > NS ? n - NS : 0; m < issued; ++m) bar_wait(&sh.full[m % NS], (m / NS) & 1, DRAIN_NS);
    if (holes_seen && lane == 0) report(a.batch, ST_BAD_PAGE);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::R_SOFT));
    // ---- softmax of row tile w: thread = row ----------------------------------
    const int w = warp >> 2, row = tid & 127;
    const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + 128 * w, to = tmem + lanes + 256 + 128 * w;
    uint32_t tiles = 0, t = 0, item = 0, cuts = 0;  // tiles of the ring, tiles of keys with rows, units, units cut
    bool ok = true;
    // the row tile's queries (two f16 parts), and at a unit's end its results on their way out
    uint8_t* qt = sm + L::Q + w * 2 * L::PART;
    constexpr int LPR = HD / 4, RPI = 32 / LPR;  // lanes of a row, rows that a warp moves at once
    const int r32 = 32 * (warp & 3);             // its first row
    do {
      const int r0 = wk.rb * M + 128 * w, rn = min(128, wk.rows - r0);
      const int end = wk.end_of(a, w);
      if (end > wk.ta) {
        // the queries, scaled and split: a warp its own 32 rows, whole rows at a time; rows that are not there are zeros
        const int gr = r0 + min(row, rn - 1);
        float qinv = 1.0f;
        // a row's places in q and out, in its thread; other lanes ask for them
        const long long q_at = (wk.sq.r0 + token_of(a, gr)) * a.q_stride + (wk.kvh * a.rep + head_of(a, gr)) * HD;
        const long long o_at = (wk.sq.r0 + token_of(a, gr)) * a.out_stride + (wk.kvh * a.rep + head_of(a, gr)) * HD;
#pragma unroll 1
        for (int j0 = 0; j0 < 32 / RPI; j0 += 8) {
          float4 x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = RPI * (j0 + j) + lane / LPR;
            const long long from = __shfl_sync(0xffffffffu, q_at, r);
            x[j] = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + from) + lane % LPR);  // (of the last row where there is none)
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (r32 + RPI * (j0 + j) + lane / LPR >= rn) x[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            // (a row with an infinity or NaN gives NaN)
            float top = fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w)));
#pragma unroll
            for (int d = LPR / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const int ge = group_exp(top, 0);
            const float f = copysignf(pow2(-ge), a.scale_log2), back = pow2(ge);  // (a negative scale turns the queries)
#pragma unroll
            for (int i = 0; i < RPI; ++i) {
              const float v = __shfl_sync(0xffffffffu, back, i * LPR);
              if (lane == RPI * (j0 + j) + i) qinv = v;
            }
            uint2 h, l;
            split_f16(mul_f32x2(pack_f32x2(x[j].x, x[j].y), pack_f32x2(f, f)), h.x, l.x);
            split_f16(mul_f32x2(pack_f32x2(x[j].z, x[j].w), pack_f32x2(f, f)), h.y, l.y);
            const uint32_t o = tile_at(r32 + RPI * (j0 + j) + lane / LPR, (lane % LPR) >> 1) + 8 * (lane & 1);
            *reinterpret_cast<uint2*>(qt + o) = h;
            *reinterpret_cast<uint2*>(qt + L::PART + o) = l;
          }
        }
        fence_proxy_async();
        bar_arrive(&sh.q_full[w]);

        const Sight<TREE> sight(a, wk.sq, token_of(a, gr), wk.table);
        float m = -INFINITY, l = 0.0f;  // m: the maximum that O and l are scaled by
        float o[HD];
#pragma unroll
        for (int d = 0; d < HD; ++d) o[d] = 0.0f;
        const float scale = fabsf(a.scale_log2);
        float due = 0.0f;  // factor of the half whose O' is not added yet
        auto add_half = [&](int b) {
#pragma unroll
          for (int q = 0; q < HD / 16; ++q) {
            uint32_t x[16];
            tmem_ld16(to + HD * b + 16 * q, x);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; e += 2)
              unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), pack_f32x2(due, due), pack_f32x2(o[16 * q + e], o[16 * q + e + 1])),
                           o[16 * q + e], o[16 * q + e + 1]);
          }
        };
        auto rescale = [&](float top) {
          if (__any_sync(0xffffffffu, top > m + SLACK)) {
            // (a row by itself: not by what its neighbours see). Over an f16 cache a whole number, so that m - lift is exact
            const float nm = top > m + SLACK ? (F32C ? top : ceilf(top)) : m;
            const float f = m == nm ? 1.0f : fast_exp2(m - (nm == -INFINITY ? 0.0f : nm));
#pragma unroll
            for (int d = 0; d < HD; ++d) o[d] *= f;
            due *= f;
            l *= f;
            m = nm;
          }
        };
        for (int i = wk.ta; i < end && ok; ++i) {
          const uint32_t rt = tiles + (i - wk.ta);  // ring tile pair
          const uint32_t* holes = sh.holes[rt % HOLE_RING];
          const bool cut = wk.ragged(a, i);
          if constexpr (F32C) {
            // the values' factors, after S: the loaders are in this tile then, and the slot's barrier in this phase or past it (a row
            // tile that sees few keys would else be here two phases early, where the parity is the same)
            ok = tc_wait_warp(&sh, &sh.s_full[w][0], t & 1) && tc_wait_warp(&sh, &sh.full[(2 * rt + 1) % NS], ((2 * rt + 1) / NS) & 1);
            if (!ok) break;
            // keys that the products leave out: q k and p v by ordinary arithmetic, one key after another (rare, and
            // short code rather than fast)
            const uint64_t* apart = reinterpret_cast<const uint64_t*>(sh.apart[rt % HOLE_RING]);
            if ((apart[0] | apart[1]) != 0) {
#pragma unroll 1
              for (int b = 0; b < 2; ++b)
#pragma unroll 1
                for (uint64_t left = apart[b]; left; left &= left - 1) {
                  const int key = (wk.blk.tile0 + i) * TC_TK + 64 * b + __ffsll(static_cast<long long>(left)) - 1;
                  bool hole;
                  const long long off = wk.key_offset(a, key, hole);
                  if (off < 0) continue;
                  const CT* kp = static_cast<const CT*>(a.pool.k) + wk.kvh * a.pool.head_stride + off;
                  const CT* vp = static_cast<const CT*>(a.pool.v) + wk.kvh * a.pool.head_stride + off;
                  const float* qp = static_cast<const float*>(a.q) + q_at;
                  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
                  for (int d = 0; d < HD; d += 8) {
                    float x[8], y[8];
                    load_vec<float, 8>(qp + d, x);
                    load_vec<CT, 8>(kp + d, y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum[e & 3] = fmaf(x[e], y[e], sum[e & 3]);
                  }
                  const float x = sight.has(a, key) ? ((sum[0] + sum[1]) + (sum[2] + sum[3])) * a.scale_log2 : -INFINITY;
                  rescale(x);
                  const float p = fast_exp2(x - (m == -INFINITY ? 0.0f : m));
                  l += p;
#pragma unroll
                  for (int d = 0; d < HD; d += 8) {
                    float y[8];
                    load_vec<CT, 8>(vp + d, y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[d + e] = fmaf(p, fabsf(y[e]) <= FLT_MAX ? y[e] : 0.0f, o[d + e]);  // (the others are added at the unit's end)
                  }
                }
            }
          }
#pragma unroll 1
          for (int b = 0; b < 2; ++b) {
            if (!F32C || b) ok = tc_wait_warp(&sh, &sh.s_full[w][b], t & 1);
            if (!ok) break;
            tc_fence_after();
            const int key0 = (wk.blk.tile0 + i) * TC_TK + 64 * b;
            const uint32_t sa = ts + 64 * b;
            uint32_t v[2][16];
            tmem_ld16(sa, v[0]);
            // factors of the products: of 8 keys, or of all; never zero, or a masked product's infinity would become NaN
            float kf[8];
            auto factor = [&](float f) { return fmaxf(scale * qinv * f, 1e-37f); };
            if constexpr (F32C) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float4 ke = *reinterpret_cast<const float4*>(&sh.kfac[rt % EXP_RING][8 * b + 4 * q]);
#pragma unroll
                for (int j = 0; j < 4; ++j) kf[4 * q + j] = factor((&ke.x)[j]);
              }
            } else {
              kf[0] = factor(1.0f);
            }
            // which of the keys this row sees; whether some row of the warp does not see all of them
            uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
            bool mask = false;
            if (cut || (holes[2 * b] | holes[2 * b + 1]) != 0) {
#pragma unroll
              for (int q = 0; q < 2; ++q) seen[q] = sight.of32(a, key0 + 32 * q) & ~holes[2 * b + q];
              mask = __any_sync(0xffffffffu, (seen[0] & seen[1]) != 0xffffffffu);
            }
            // S is read twice, 16 keys at a time: for the maxima, then for P, whose two parts take the 16 columns' place
            auto keys = [&](int c, uint32_t (&x)[16]) {  // columns 16 c .. of S, the next ones on their way
              tmem_wait_ld();
              if (mask) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  if (!((seen[c >> 1] >> (16 * (c & 1) + e)) & 1)) x[e] = 0xff800000u;  // -infinity
              }
            };
            // the largest score, and the largest of a score and its values' exponent, of what the row sees
            float top = -INFINITY, top_v = -INFINITY;
            float ve[8];
            if constexpr (F32C) {
#pragma unroll
              for (int q = 0; q < 2; ++q)
                *reinterpret_cast<float4*>(ve + 4 * q) = *reinterpret_cast<const float4*>(&sh.vexp[rt % EXP_RING][8 * b + 4 * q]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t (&x)[16] = v[c & 1];
              keys(c, x);
              tmem_ld16(sa + (c < 3 ? 16 * (c + 1) : 0), v[(c + 1) & 1]);  // (after the last: the first again)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float f = kf[F32C ? 2 * c + q : 0];
                auto at = [&](int e) { return __uint_as_float(x[8 * q + e]); };
                const float t = max3(max3(at(0), at(1), at(2)), max3(at(3), at(4), at(5)), fmaxf(at(6), at(7))) * f;
                top = fmaxf(top, t);
                if constexpr (F32C) top_v = fmaxf(top_v, t + ve[2 * c + q]);
              }
            }
            rescale(top);
            const float use = m == -INFINITY ? 0.0f : m;
            // P goes to the products times 2^lift, which brings the row's largest weight (times the size of its values) near
            // 2^14: two f16 numbers end at 2^-24, 2^-38 of that. Only what the row sees counts, and with its weight.
            int lift = 14 - int(fminf(fmaxf(ceilf((F32C ? top_v : top) - use), -112.0f), 140.0f));
            if (!F32C && fabsf(use) > 8388608.0f) lift = 0;  // (scores that are whole numbers at best)
            float vf[8];  // of P
            if constexpr (F32C) {
              const float up = pow2(lift);
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float4 x = *reinterpret_cast<const float4*>(&sh.vfac[rt % EXP_RING][8 * b + 4 * q]);
#pragma unroll
                for (int j = 0; j < 4; ++j) vf[4 * q + j] = fminf((&x.x)[j] * up, 0x1p126f);  // (finite, for weights of zero)
              }
            }
            const float from = F32C ? use : use - float(lift);  // (exact: whole numbers below 2^24)
            uint64_t s2[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t (&x)[16] = v[c & 1];
              keys(c, x);
              if (c < 3) tmem_ld16(sa + 16 * (c + 1), v[(c + 1) & 1]);
              uint32_t p[8], r[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int gq = F32C ? 2 * c + e / 4 : 0;
                float y0, y1;
                unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), pack_f32x2(kf[gq], kf[gq]), pack_f32x2(-from, -from)), y0, y1);
                uint64_t z = pack_f32x2(fast_exp2(y0), fast_exp2(y1));
                s2[e & 1] = add_f32x2(s2[e & 1], z);
                if (F32C) z = mul_f32x2(z, pack_f32x2(vf[gq], vf[gq]));
                split_f16(z, p[e], r[e]);
              }
              tmem_st8(sa + 16 * c, p);
              tmem_st8(sa + 16 * c + 8, r);
            }
            {
              float x0, y0, x1, y1;
              unpack_f32x2(s2[0], x0, y0);
              unpack_f32x2(s2[1], x1, y1);
              l += ((x0 + y0) + (x1 + y1)) * (F32C ? 1.0f : pow2(-lift));
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.p_full[w][b]);
            // the half before this one
            if (i > wk.ta || b) {
              ok = tc_wait_warp(&sh, &sh.o_done[w][1 - b], (b ? t : t - 1) & 1);
              if (!ok) break;
              tc_fence_after();
              add_half(1 - b);
              tc_fence_before();
            }
            due = pow2(-lift);
          }
          ++t;
        }
        if (ok) ok = tc_wait_warp(&sh, &sh.o_done[w][1], (t - 1) & 1);
        if (!ok) break;
        tc_fence_after();
        add_half(1);
        tc_fence_before();

        // infinities and NaN that were taken out of the values, for the rows that see them
        if (*reinterpret_cast<volatile int*>(&sh.odd[item % ODD_RING]) != 0) {
#pragma unroll 1
          for (int i = wk.ta; i < end; ++i) {
            if (!F32C && !wk.ragged(a, i)) continue;
            const int k0 = (wk.blk.tile0 + i) * TC_TK;
#pragma unroll 1
            for (int key = sight.from(k0); key < min(k0 + TC_TK, sight.hi); ++key) {
              if (TREE && !sight.has(a, key)) continue;
              bool hole;
              const long long off = wk.key_offset(a, key, hole);
              if (off < 0) continue;
              const CT* vp = static_cast<const CT*>(a.pool.v) + wk.kvh * a.pool.head_stride + off;
#pragma unroll
              for (int d = 0; d < HD; ++d) {
                const float x = to_f32(vp[d]);
                if (!(fabsf(x) <= FLT_MAX)) o[d] += x;
              }
            }
          }
        }
        // results: normalised, or a piece [HD / 4][M][4] + m [M] + l [M]
        const bool whole = wk.ta == 0 && wk.tb == wk.blk.tiles;
        const int64_t tok = wk.sq.r0 + token_of(a, gr);
        const int hh = wk.kvh * a.rep + head_of(a, gr);
        constexpr size_t PIECE = size_t(M) * (HD + 2);
        const int pr = 128 * w + row;  // the row in a piece
        // rows leave through shared memory, each warp its own: a thread's row by itself would be 32 lines a store
        auto send = [&] {
          const bool some = (l > 0.0f && m > -INFINITY) || l != l;
          const float inv = some ? 1.0f / l : 0.0f;
#pragma unroll
          for (int c = 0; c < HD / 4; ++c) {
            float4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) (&y.x)[e] = some ? o[4 * c + e] * inv : 0.0f;
            *reinterpret_cast<float4*>(qt + (c / (HD / 8)) * L::PART + tile_at(row, c % (HD / 8))) = y;
          }
          __syncwarp();
#pragma unroll 4
          for (int j = 0; j < 32 / RPI; ++j) {
            const int r = RPI * j + lane / LPR, c = lane % LPR;
            const long long to_at = __shfl_sync(0xffffffffu, o_at, r);
            if (r32 + r < rn)
              *reinterpret_cast<float4*>(static_cast<float*>(a.out) + to_at + 4 * c) =
                  *reinterpret_cast<const float4*>(qt + (c / (HD / 8)) * L::PART + tile_at(r32 + r, c % (HD / 8)));
          }
          __syncwarp();
          if (a.lse && row < rn) a.lse[tok * a.n_heads + hh] = some ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
        };
        if (whole) {
          send();
        } else if (row < rn) {
          float* piece = a.part + (size_t(blockIdx.x) * 2 + (wk.ta == 0 ? 1 : 0)) * PIECE;
#pragma unroll
          for (int d = 0; d < HD; d += 4) reinterpret_cast<float4*>(piece)[size_t(d / 4) * M + pr] = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
          piece[size_t(HD) * M + pr] = m;
          piece[size_t(HD + 1) * M + pr] = l;
        }
        if (row == 0 && w == 0) {
          uint32_t bits = 0;
          if (wk.blk.pos1 >= wk.table) bits |= ST_BAD_PAGE;
          if ((TREE ? wk.sq.kv - wk.sq.n : wk.blk.pos0) < 0) bits |= ST_BAD_LEN;
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
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int d = 0; d < HD; ++d) o[d] = 0.0f;
            if (row < rn) {
              auto part = [&](int p) { return a.part + (size_t(p) * 2 + (p == c0 ? 1 : 0)) * PIECE; };
              for (int p = c0; p <= c1; ++p) m = fmaxf(m, __ldcg(part(p) + size_t(HD) * M + pr));
              const float u = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
              for (int p = c0; p <= c1; ++p) {
                const float* pp = part(p);
                const float f = fast_exp2(__ldcg(pp + size_t(HD) * M + pr) - u);
                l += f * __ldcg(pp + size_t(HD + 1) * M + pr);
#pragma unroll
                for (int d = 0; d < HD; d += 4) {
                  const float4 y = __ldcg(reinterpret_cast<const float4*>(pp) + size_t(d / 4) * M + pr);
                  o[d] = fmaf(f, y.x, o[d]);
                  o[d + 1] = fmaf(f, y.y, o[d + 1]);
                  o[d + 2] = fmaf(f, y.z, o[d + 2]);
                  o[d + 3] = fmaf(f, y.w, o[d + 3]);
                }
              }
            }
            send();
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
  if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <typename CT, int HD, bool TREE>
cudaError_t run_tc32(const AttendArgs& a, cudaStream_t s) {
  using L = Tc32Cfg<CT, HD>;
  static_assert(L::SMEM + sizeof(Tc32Shared) + sizeof(PlaceShared<L::THREADS>) <= 227 * 1024, "shared memory");
  // the register split draws on what the kernel is launched with (looked up until it is known: a call that fails, for want
  // of a device for instance, says why and leaves nothing behind)
  static std::atomic<int> regs{0};
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes at;
    const cudaError_t found = cudaFuncGetAttributes(&at, attend_tc32_kernel<CT, HD, TREE>);
    if (found != cudaSuccess) return found;
    regs.store(at.numRegs, std::memory_order_relaxed);
  }
  if (L::WGS * regs.load(std::memory_order_relaxed) < L::RT * L::R_SOFT + L::LW / 4 * L::R_LOAD + L::R_MMA) return cudaErrorInvalidKernelImage;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_shared(attend_tc32_kernel<CT, HD, TREE>, L::SMEM, done);
  if (e != cudaSuccess) return e;
  CUtensorMap km{}, vm{};
  int box = 0;
  if constexpr (!L::F32C) box = make_maps<CT>(&km, &vm, a.pool, TC_TK);
  attend_tc32_kernel<CT, HD, TREE><<<TC_CTAS, L::THREADS, L::SMEM, s>>>(a, km, vm, box);
  return cudaGetLastError();
}

template <bool TREE>
cudaError_t run_tc32_cache(const AttendArgs& a, int cache, cudaStream_t s) {
  if (cache == E_F16) return a.pool.head_dim == 64 ? run_tc32<__half, 64, TREE>(a, s) : run_tc32<__half, 128, TREE>(a, s);
  if (cache == E_BF16) return a.pool.head_dim == 64 ? run_tc32<__nv_bfloat16, 64, TREE>(a, s) : run_tc32<__nv_bfloat16, 128, TREE>(a, s);
  return a.pool.head_dim == 64 ? run_tc32<float, 64, TREE>(a, s) : run_tc32<float, 128, TREE>(a, s);
}

}  // namespace
}  // namespace paged
}  // namespace wcb
