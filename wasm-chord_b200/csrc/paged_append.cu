// Append: per-head norm, rotation by position, store to pages.
//
// x' = x / sqrt(mean(x^2) + eps) * w for each query and key head (optional), then
// pair i of the head turns by position * inv_freq[i]:
//   (a, b) -> (a cos - b sin, a sin + b cos).
// Memory bound: q, k and v are read once and written once; a call for a few
// tokens is bound by its launch and two dependent loads. One CTA takes one token
// (a few tokens: part of one token's heads, blockIdx.y). A thread takes 8 pairs
// (16 elements) of one head, so that a head's sum of squares is a shuffle over
// head_dim / 16 lanes and every access is 16 bytes wide. The token's cosines and
// sines are computed once by the first rot / 2 threads into shared memory:
// position * inv_freq / 2 pi is reduced to a fraction of a turn in 64 bits (in
// 32 bits a position of 10^6 is off by up to 0.06 rad), its sine and cosine taken
// in 32.
#include "paged_common.cuh"

namespace wcb {
namespace paged {
namespace {

constexpr int AP_THREADS = 256;

template <typename AT, typename CT>
__global__ void __launch_bounds__(AP_THREADS) append_kernel(const __grid_constant__ AppendArgs a) {
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
    // the 16 elements: two runs of 8, apart by half the rotated part where pairs are halves
    int c0 = 16 * sub, c1 = 16 * sub + 8;
    const bool turned = (is_q || is_k) && (a.halves ? 8 * sub < a.rot / 2 : 16 * sub < a.rot);
    if (a.halves && turned) {
      c0 = 8 * sub;
      c1 = 8 * sub + a.rot / 2;
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
    if (turned) {
      if (a.halves) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 t = s_turn[8 * sub + e];
          const float p = x[e], q = y[e];
          x[e] = p * t.x - q * t.y;
          y[e] = p * t.y + q * t.x;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 t = s_turn[8 * sub + e], u = s_turn[8 * sub + 4 + e];
          const float p = x[2 * e], q = x[2 * e + 1];
          x[2 * e] = p * t.x - q * t.y;
          x[2 * e + 1] = p * t.y + q * t.x;
          const float g = y[2 * e], h = y[2 * e + 1];
          y[2 * e] = g * u.x - h * u.y;
          y[2 * e + 1] = g * u.y + h * u.x;
        }
      }
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
  const int items = (a.n_heads + 2 * a.pool.n_kv) * (a.pool.head_dim / 16);
  const int rounds = (items + AP_THREADS - 1) / AP_THREADS;
  // few tokens: a token's heads over several CTAs
  const int y = a.batch.n_tokens >= 296 ? 1 : (rounds < 296 / a.batch.n_tokens ? rounds : 296 / a.batch.n_tokens);
  append_kernel<AT, CT><<<dim3(a.batch.n_tokens, y < 1 ? 1 : y), AP_THREADS, 0, s>>>(a);
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
