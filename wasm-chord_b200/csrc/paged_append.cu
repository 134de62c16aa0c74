// Append: per-head norm, rotation by position, store to pages.
//
// x' = x / sqrt(mean(x^2) + eps) * w for each query and key head (optional), then
// pair i of the head turns by position * inv_freq[i]:
//   (a, b) -> (a cos - b sin, a sin + b cos).
// Memory bound: q, k and v are read once and written once; a call for a few
// tokens is bound by its launch and two dependent loads. One CTA takes one token
// (a few tokens: part of one token's heads, blockIdx.y). A thread takes two runs of 8
// elements of one head, half a head (or half the rotated part) apart, so that a head's sum
// of squares is a shuffle over head_dim / 16 lanes, pairs of either kind lie in one thread and
// neighbouring threads in neighbouring 16 bytes. The token's cosines and
// sines are computed once by the first rot / 2 threads into shared memory:
// position * inv_freq / 2 pi is reduced to a fraction of a turn in 64 bits (in
// 32 bits a position of 10^6 is off by up to 0.06 rad), its sine and cosine taken
// in 32.
//
// 7700 tokens of 32/32 heads of 128, f16 (380 MB): 67 us, 87 % of the copy rate. What carries it are many
// small CTAs on an SM, which hide each other's lookups: 4 of 256 threads 83 us, 8 73 us, 12 of 128 67 us;
// requesting the rows before the lookups (88 us and more) or four tokens a CTA (91 us) cost registers
// and with them CTAs.
#include "paged_common.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int AP_THREADS = 128;
constexpr int AP_PER_SM = 12;

template <typename AT, typename CT>
__global__ void __launch_bounds__(AP_THREADS, AP_PER_SM) append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ int s_seq;
  __shared__ float2 s_turn[64];
  const int tid = threadIdx.x, row = blockIdx.x;
  const int hd = a.pool.head_dim, nkv = a.pool.n_kv;
  if (tid == 0) s_seq = -1;
  __syncthreads();
  // the row's sequence: q_start does not descend, so at most one s has it
  uint32_t bad = 0;
  for (int s = tid; s < a.batch.n_seqs; s += AP_THREADS) {
    const Seq q = read_seq(a.batch, s);
    if (!q.sound) bad |= ST_BAD_ROWS;
    if (q.n > 0 && row >= q.r0 && row < q.r0 + q.n) s_seq = s;
  }
  if (bad && row == 0 && blockIdx.y == 0) report(a.batch, bad);
  __syncthreads();
  const int s = s_seq;
  if (s < 0) return;  // a row of no sequence
  const Seq sq = read_seq(a.batch, s);
  const int pos = sq.kv - sq.n + (row - sq.r0);
  // where the token's key and value go: -1 = nowhere
  int64_t slot = -1;
  bad = 0;
  if (pos < 0) bad = ST_BAD_LEN;
  else if (pos >= table_tokens(a.pool, a.batch)) bad = ST_BAD_PAGE;
  else {
    const int page = __ldg(a.batch.page_table + int64_t(s) * a.batch.max_pages + pos / a.pool.page_size);
    if (page < 0 || page >= a.pool.n_pages) bad = ST_BAD_PAGE;
    else slot = page * a.pool.page_stride + int64_t(pos % a.pool.page_size) * a.pool.token_stride;
  }
  if (bad && tid == 0 && blockIdx.y == 0) report(a.batch, bad);
  if (tid < a.rot / 2) {
    const double turn = double(pos) * a.turns[tid];
    const float f = float(2.0 * (turn - rint(turn)));  // half turns in [-1, 1]
    float sn, cs;
    sincospif(f, &sn, &cs);
    s_turn[tid] = make_float2(cs, sn);
  }
  __syncthreads();

  const int lph = hd / 16;  // threads of a head
  const int items = (a.n_heads + 2 * nkv) * lph;
  const int rounds = (items + AP_THREADS - 1) / AP_THREADS;
  for (int r = blockIdx.y; r < rounds; r += gridDim.y) {
    const int it = r * AP_THREADS + tid;
    const bool on = it < items;
    const int hh = on ? it / lph : 0, sub = it % lph;
    const bool is_q = hh < a.n_heads, is_k = !is_q && hh < a.n_heads + nkv;
    const int head = is_q ? hh : is_k ? hh - a.n_heads : hh - a.n_heads - nkv;
    // the two runs: of the rotated part where pairs are halves, of the rest of such a head, of a whole head
    int c0 = 8 * sub, c1 = c0 + hd / 2;
    bool turn0 = false, turn1 = false;
    if (a.halves) {
      if (8 * sub < a.rot / 2) {
        c1 = c0 + a.rot / 2;
        turn0 = turn1 = is_q || is_k;
      } else {
        c0 = a.rot + 8 * sub - a.rot / 2;
        c1 = c0 + (hd - a.rot) / 2;
      }
    } else {
      turn0 = (is_q || is_k) && c0 < a.rot;
      turn1 = (is_q || is_k) && c1 < a.rot;
    }
    const AT* src = is_q ? static_cast<const AT*>(a.q) + row * a.q_stride
                  : is_k ? static_cast<const AT*>(a.k) + row * a.k_stride
                         : static_cast<const AT*>(a.v) + row * a.v_stride;
    float x[8], y[8];
    if (on) {
      load_vec<AT, 8>(src + head * hd + c0, x);
      load_vec<AT, 8>(src + head * hd + c1, y);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.0f;
    }
    const float* w = is_q ? a.q_norm : a.k_norm;
    if (a.q_norm || a.k_norm) {  // uniform: every lane takes part in the shuffles
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[e] * x[e] + y[e] * y[e];
      for (int o = lph / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (on && (is_q || is_k) && w) {
        const float inv = rsqrtf(sum / float(hd) + a.eps);
        float wx[8], wy[8];
        load_vec<float, 8>(w + c0, wx);
        load_vec<float, 8>(w + c1, wy);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = x[e] * inv * wx[e];
          y[e] = y[e] * inv * wy[e];
        }
      }
    }
    if (!on) continue;
    if (a.halves) {
      if (turn0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 t = s_turn[8 * sub + e];
          const float p = x[e], q = y[e];
          x[e] = p * t.x - q * t.y;
          y[e] = p * t.y + q * t.x;
        }
      }
    } else {
      auto turn = [&](float (&z)[8], int c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 t = s_turn[c / 2 + e];
          const float p = z[2 * e], q = z[2 * e + 1];
          z[2 * e] = p * t.x - q * t.y;
          z[2 * e + 1] = p * t.y + q * t.x;
        }
      };
      if (turn0) turn(x, c0);
      if (turn1) turn(y, c1);
    }
    if (is_q) {
      AT* dst = static_cast<AT*>(a.q_out) + row * a.q_out_stride + head * hd;
      store_vec<AT, 8>(dst + c0, x);
      store_vec<AT, 8>(dst + c1, y);
    } else if (slot >= 0) {
      CT* dst = static_cast<CT*>(is_k ? a.pool.k : a.pool.v) + slot + head * a.pool.head_stride;
      store_vec<CT, 8>(dst + c0, x);
      store_vec<CT, 8>(dst + c1, y);
    }
  }
}

template <typename AT, typename CT>
cudaError_t run_append(const AppendArgs& a, cudaStream_t s) {
  const int n = a.batch.n_tokens;
  const int items = (a.n_heads + 2 * a.pool.n_kv) * (a.pool.head_dim / 16);
  const int rounds = (items + AP_THREADS - 1) / AP_THREADS;
  // few tokens: a token's heads over several CTAs
  const int y = n >= 2 * SMS ? 1 : (rounds < 2 * SMS / n ? rounds : 2 * SMS / n);
  append_kernel<AT, CT><<<dim3(n, y < 1 ? 1 : y), AP_THREADS, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, int act, int cache, cudaStream_t s) {
  if (act == E_F16) return run_append<__half, __half>(a, s);
  if (act == E_BF16) return run_append<__nv_bfloat16, __nv_bfloat16>(a, s);
  if (cache == E_F16) return run_append<float, __half>(a, s);
  if (cache == E_BF16) return run_append<float, __nv_bfloat16>(a, s);
  return run_append<float, float>(a, s);
}

}  // namespace paged
}  // namespace wcb
