// Entry points of the paged serving operators (include/wcb.h): argument checks,
// the choice of kernels, workspace layout. Every check that needs no GPU comes
// before the first CUDA call.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <string>

#include "../../include/wcb.h"
#include "paged.h"

extern "C" __attribute__((visibility("hidden"))) void wcb_internal_set_last_error(const char* msg);

namespace {

using namespace wcb::paged;

uint32_t fail(uint32_t code, const char* msg) {
  wcb_internal_set_last_error(msg);
  return code;
}
uint32_t bad(const char* msg) { return fail(WCB_ERR_INVALID_ARGUMENT, msg); }

uint32_t cuda_result(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return WCB_OK;
  try {
    const std::string m = std::string("Backend error: ") + what + ": " + cudaGetErrorString(e);
    wcb_internal_set_last_error(m.c_str());
  } catch (...) {
  }
  return e == cudaErrorMemoryAllocation ? WCB_ERR_OOM : WCB_ERR_BACKEND_UNSUPPORTED;
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
int size_of(uint32_t dtype) { return dtype == WCB_KV_F32 ? 4 : 2; }

// strides that the kernels' 64-bit element offsets can take
constexpr uint64_t MAX_STRIDE = uint64_t(1) << 40;

uint32_t check_pool(const wcb_paged_kv* kv, Pool* out) {
  if (!kv) return bad("Invalid argument: null pointer");
  if (kv->struct_size < sizeof(wcb_paged_kv)) return bad("Invalid argument: wcb_paged_kv.struct_size");
  if (kv->dtype > WCB_KV_BF16) return bad("Unsupported data type: the paged cache is F32, F16 or BF16");
  if (!kv->k || !kv->v) return bad("Invalid argument: null pointer");
  if (kv->head_dim != 64 && kv->head_dim != 128) return bad("Invalid tensor shape: need head_dim 64|128");
  if (kv->n_kv_heads == 0 || kv->n_kv_heads > 1024 || kv->page_size == 0 || kv->page_size > (1u << 30) ||
      kv->n_pages == 0 || kv->n_pages > unsigned(INT_MAX))
    return bad("Invalid tensor shape: need 1 <= n_kv_heads <= 1024, 1 <= page_size <= 2^30, 1 <= n_pages < 2^31");
  if (off16(kv->k) || off16(kv->v)) return bad("Invalid argument: k and v must be 16-byte aligned");
  uint64_t ps = kv->page_stride, ts = kv->token_stride, hs = kv->head_stride;
  if (ps == 0 && ts == 0 && hs == 0) {
    hs = kv->head_dim;
    ts = hs * kv->n_kv_heads;
    ps = ts * kv->page_size;
  }
  const uint64_t unit = 16 / uint64_t(size_of(kv->dtype));
  if (ps % unit || ts % unit || hs % unit || ps > MAX_STRIDE || ts > MAX_STRIDE || hs > MAX_STRIDE)
    return bad("Invalid argument: page, token and head strides must be multiples of 16 bytes, at most 2^40 elements");
  if ((kv->n_pages > 1 && ps == 0) || (kv->page_size > 1 && ts == 0) || (kv->n_kv_heads > 1 && hs == 0))
    return bad("Invalid argument: a stride of 0 (leave all three 0 for the layout without gaps)");
  out->k = kv->k;
  out->v = kv->v;
  out->page_stride = int64_t(ps);
  out->token_stride = int64_t(ts);
  out->head_stride = int64_t(hs);
  out->page_size = int(kv->page_size);
  out->n_pages = int(kv->n_pages);
  out->n_kv = int(kv->n_kv_heads);
  out->head_dim = int(kv->head_dim);
  return WCB_OK;
}

uint32_t check_batch(const wcb_paged_batch* b, Batch* out) {
  if (!b) return bad("Invalid argument: null pointer");
  if (b->struct_size < sizeof(wcb_paged_batch)) return bad("Invalid argument: wcb_paged_batch.struct_size");
  if (b->reserved != 0) return bad("Invalid argument: wcb_paged_batch.reserved must be 0");
  if (b->n_seqs == 0 || b->n_seqs > 65536 || b->n_tokens == 0 || b->n_tokens > (1u << 24) || b->max_q_len == 0 ||
      b->max_q_len > b->n_tokens || b->max_pages == 0 || b->max_pages > unsigned(INT_MAX))
    return bad("Invalid tensor shape: need 1 <= n_seqs <= 65536, 1 <= max_q_len <= n_tokens <= 2^24, max_pages >= 1");
  if (!b->q_start || !b->kv_len || !b->page_table) return bad("Invalid argument: null pointer");
  if ((reinterpret_cast<uintptr_t>(b->q_start) | reinterpret_cast<uintptr_t>(b->kv_len) |
       reinterpret_cast<uintptr_t>(b->page_table) | reinterpret_cast<uintptr_t>(b->status)) & 3)
    return bad("Invalid argument: q_start, kv_len, page_table and status must be 4-byte aligned");
  out->q_start = b->q_start;
  out->kv_len = b->kv_len;
  out->page_table = b->page_table;
  out->status = b->status;
  out->n_seqs = int(b->n_seqs);
  out->n_tokens = int(b->n_tokens);
  out->max_pages = int(b->max_pages);
  return WCB_OK;
}

uint32_t check_types(uint32_t dtype, uint32_t cache) {
  if (dtype == WCB_KV_F32 || ((dtype == WCB_KV_F16 || dtype == WCB_KV_BF16) && cache == dtype)) return WCB_OK;
  return bad("Unsupported data type: F32 activations take any cache, F16 and BF16 ones a cache of their own type");
}

// rows of tokens: base address, stride between tokens, elements of a token
uint32_t check_rows(const void* p, uint64_t stride, uint64_t width, uint32_t dtype) {
  if (!p) return bad("Invalid argument: null pointer");
  if (off16(p) || stride % (16 / uint64_t(size_of(dtype))))
    return bad("Invalid argument: rows must start at multiples of 16 bytes");
  if (stride < width || stride > MAX_STRIDE) return bad("Invalid argument: a row stride is shorter than the row");
  return WCB_OK;
}

// Which kernels a call runs, from what the host knows: the longest sequence's rows
// (new tokens * rep), the number of sequences. Sequences of more than TC_MIN rows go to a tensor-core
// kernel, the others of the batch to the mma.sync kernel. Its row block is the smallest that holds the longest
// sequence's rows, so that no product is spent on rows that are not there. A call that would make no more than
// TC_UNITS blocks of 32 rows in all stays with the mma.sync kernel: cut into many parts, its small blocks are
// joined sooner than blocks of 256.
// Measured (us, tensor cores / mma.sync; 32/4 heads of 64, f16, 4096 keys): 1 sequence of 64 rows (8 blocks) 41 / 21, of
// 256 (32) 45 / 29, of 512 (64) 33 / 40, of 1024 28 / 64; 32 sequences of 40 rows (256) 70 / 114, of 256 87 / 423;
// f32 over f32: 1 of 128 rows 41 / 34, of 256 47 / 52, 32 of 40 185 / 290; f32 over bf16: 16 of 612 rows 56 / 92;
// 64/8 heads of 128, bf16: 1 of 64 rows (16) 46 / 32, of 128 (32) 47 / 45, of 256 (64) 53 / 61.
constexpr uint64_t TC_MIN = 32, TC_UNITS = 32;
struct Plan {
  int rows;     // row block of the mma.sync kernel, 0: not run
  bool tc;
  int split;    // sequences of more rows are the tensor-core kernel's
};
Plan plan(uint64_t n_seqs, uint64_t n_kv, uint64_t max_rows) {
  Plan p{};
  p.tc = max_rows > TC_MIN && n_seqs * n_kv * ((max_rows + 31) / 32) > TC_UNITS;
  p.split = p.tc ? (n_seqs == 1 ? 0 : int(TC_MIN)) : INT_MAX;
  const uint64_t r = p.tc ? (n_seqs == 1 ? 0 : TC_MIN) : max_rows;
  p.rows = r == 0 ? 0 : r <= 8 ? 8 : r <= 16 ? 16 : 32;
  return p;
}

// the kernels of a call run one after the other and share the pieces' memory
size_t workspace_bytes(const Plan& p, int head_dim) {
  const size_t row = sizeof(float) * 2 * size_t(head_dim + 2);
  const size_t x = size_t(ATTEND_CTAS) * size_t(p.rows) * row, y = p.tc ? size_t(TC_CTAS) * TC_ROWS * row : 0;
  return TICKET_BYTES + (x > y ? x : y);
}

}  // namespace

extern "C" {

uint32_t wcb_rope_init(wcb_rope* r, uint32_t rot_dim, double theta, uint32_t halves) {
  if (!r) return bad("Invalid argument: null pointer");
  if (rot_dim % 16 || rot_dim > 128 || halves > 1 || !(theta > 0.0) || std::isinf(theta))
    return bad("Invalid argument: need rot_dim a multiple of 16 up to 128, theta > 0, halves 0|1");
  r->struct_size = sizeof(wcb_rope);
  r->rot_dim = rot_dim;
  r->halves = halves;
  r->reserved = 0;
  for (uint32_t i = 0; i < 64; ++i)
    r->inv_freq[i] = i < rot_dim / 2 ? std::pow(theta, -2.0 * double(i) / double(rot_dim)) : 0.0;
  return WCB_OK;
}

uint32_t wcb_paged_append_dev(const wcb_paged_kv* kv, const wcb_paged_batch* batch, const wcb_rope* rope,
                              const void* q, const void* k, const void* v, void* q_out, uint32_t dtype,
                              uint32_t n_heads, uint64_t q_stride, uint64_t k_stride, uint64_t v_stride,
                              uint64_t q_out_stride, const float* q_norm, const float* k_norm, float eps, void* stream) {
  AppendArgs a;
  uint32_t rc = check_pool(kv, &a.pool);
  if (rc == WCB_OK) rc = check_batch(batch, &a.batch);
  if (rc == WCB_OK) rc = check_types(dtype, kv->dtype);
  if (rc != WCB_OK) return rc;
  if (rope) {
    if (rope->struct_size < sizeof(wcb_rope)) return bad("Invalid argument: wcb_rope.struct_size");
    if (rope->rot_dim % 16 || rope->rot_dim > kv->head_dim || rope->halves > 1 || rope->reserved != 0)
      return bad("Invalid argument: need rot_dim a multiple of 16 up to head_dim, halves 0|1, reserved 0");
  }
  if (n_heads > 4096) return bad("Invalid tensor shape: n_heads <= 4096");
  if ((n_heads == 0) != (q == nullptr)) return bad("Invalid argument: q without heads, or heads without q");
  const uint64_t hd = kv->head_dim;
  if (n_heads) {
    rc = check_rows(q, q_stride, n_heads * hd, dtype);
    if (rc == WCB_OK) rc = check_rows(q_out, q_out_stride, n_heads * hd, dtype);
    if (rc == WCB_OK && q == q_out && q_stride != q_out_stride)
      rc = bad("Invalid argument: q_out over q needs q's stride");
  }
  if (rc == WCB_OK) rc = check_rows(k, k_stride, kv->n_kv_heads * hd, dtype);
  if (rc == WCB_OK) rc = check_rows(v, v_stride, kv->n_kv_heads * hd, dtype);
  if (rc != WCB_OK) return rc;
  if (off16(q_norm) || off16(k_norm)) return bad("Invalid argument: q_norm and k_norm must be 16-byte aligned");
  if ((q_norm || k_norm) && !(eps >= 0.0f)) return bad("Invalid argument: eps must not be negative");
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.q_stride = int64_t(q_stride);
  a.k_stride = int64_t(k_stride);
  a.v_stride = int64_t(v_stride);
  a.q_out_stride = int64_t(q_out_stride);
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = eps;
  a.n_heads = int(n_heads);
  a.rot = rope ? int(rope->rot_dim) : 0;
  a.halves = rope ? int(rope->halves) : 0;
  for (int i = 0; i < 64; ++i) a.turns[i] = i < a.rot / 2 ? rope->inv_freq[i] * 0.15915494309189533577 : 0.0;
  return cuda_result(launch_append(a, int(dtype), int(kv->dtype), static_cast<cudaStream_t>(stream)), "paged append");
}

uint32_t wcb_paged_attention_workspace(const wcb_paged_kv* kv, const wcb_paged_batch* batch, uint32_t n_heads,
                                       size_t* bytes) {
  if (!bytes) return bad("Invalid argument: null pointer");
  Pool pool;
  Batch b;
  uint32_t rc = check_pool(kv, &pool);
  if (rc == WCB_OK) rc = check_batch(batch, &b);
  if (rc != WCB_OK) return rc;
  if (n_heads == 0 || n_heads > 4096 || n_heads % kv->n_kv_heads || n_heads / kv->n_kv_heads > 64)
    return bad("Invalid tensor shape: need n_heads % n_kv_heads == 0 (<= 64 per kv head)");
  const uint64_t rows = uint64_t(batch->max_q_len) * (n_heads / kv->n_kv_heads);
  *bytes = workspace_bytes(plan(batch->n_seqs, kv->n_kv_heads, rows), pool.head_dim);
  return WCB_OK;
}

uint32_t wcb_paged_attention_dev(const wcb_paged_kv* kv, const wcb_paged_batch* batch, const void* q, void* out,
                                 uint32_t dtype, uint32_t n_heads, uint64_t q_stride, uint64_t out_stride,
                                 void* workspace, size_t workspace_bytes_given, float scale, uint32_t window,
                                 float* lse, void* stream) {
  AttendArgs a;
  size_t need = 0;
  uint32_t rc = wcb_paged_attention_workspace(kv, batch, n_heads, &need);
  if (rc == WCB_OK) rc = check_pool(kv, &a.pool);
  if (rc == WCB_OK) rc = check_batch(batch, &a.batch);
  if (rc == WCB_OK) rc = check_types(dtype, kv->dtype);
  if (rc == WCB_OK) rc = check_rows(q, q_stride, uint64_t(n_heads) * kv->head_dim, dtype);
  if (rc == WCB_OK) rc = check_rows(out, out_stride, uint64_t(n_heads) * kv->head_dim, dtype);
  if (rc != WCB_OK) return rc;
  if (!workspace || off16(workspace) || workspace_bytes_given < need)
    return bad("Invalid argument: the workspace is missing, not 16-byte aligned or smaller than "
               "wcb_paged_attention_workspace says");
  if (reinterpret_cast<uintptr_t>(lse) & 3) return bad("Invalid argument: lse must be 4-byte aligned");
  if (!std::isfinite(scale)) return bad("Invalid argument: scale must be finite");
  if (window > (1u << 30)) return bad("Invalid argument: window <= 2^30");
  if (q == out) return bad("Invalid argument: out must not be q");
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.q_stride = int64_t(q_stride);
  a.out_stride = int64_t(out_stride);
  a.scale_log2 = float((scale != 0.0f ? double(scale) : 1.0 / std::sqrt(double(kv->head_dim))) * 1.4426950408889634074);
  a.n_heads = int(n_heads);
  a.rep = int(n_heads / kv->n_kv_heads);
  a.rep_inv = (uint64_t(1) << 40) / uint64_t(a.rep) + 1;
  a.window = int(window);
  a.tickets = static_cast<int*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + TICKET_BYTES);
  // test hook for the bounded waits (unset in normal use, read once): tiles wait for bytes that do not come
  static const bool withhold = std::getenv("WCB_TEST_WITHHOLD_COPY") != nullptr;
  a.withheld = withhold ? 16 : 0;
  a.wait_ns = withhold ? 20000000ull : 2000000000ull;
  const Plan p = plan(batch->n_seqs, kv->n_kv_heads, uint64_t(batch->max_q_len) * uint64_t(a.rep));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (p.tc) {
    a.row_lo = p.split;
    a.row_hi = INT_MAX;
    e = dtype == WCB_KV_F32 ? launch_attend_tc32(a, int(kv->dtype), s) : launch_attend_tc(a, int(dtype), s);
  }
  if (p.rows && e == cudaSuccess) {
    a.row_lo = 0;
    a.row_hi = p.split;
    e = dtype == WCB_KV_F32 ? launch_attend_32(a, int(kv->dtype), p.rows, s) : launch_attend_16(a, int(dtype), p.rows, s);
  }
  return cuda_result(e, "paged attention");
}

uint32_t wcb_spec_verify_dev(const int32_t* draft, const int32_t* draft_len, const float* target,
                             const float* draft_probs, const float* u_accept, const float* u_sample, uint32_t n_seqs,
                             uint32_t max_draft, uint32_t vocab, int32_t* tokens, int32_t* accepted,
                             uint64_t target_seq_stride, uint64_t target_row_stride, uint64_t draft_seq_stride,
                             uint64_t draft_row_stride, uint32_t* status, void* stream) {
  if (!target || !u_sample || !tokens || !accepted || (max_draft && (!draft || !u_accept)))
    return bad("Invalid argument: null pointer");
  if (n_seqs == 0 || n_seqs > (1u << 20) || max_draft > 1024 || vocab == 0 || vocab > (1u << 20))
    return bad("Invalid tensor shape: need 1 <= n_seqs <= 2^20, max_draft <= 1024, 1 <= vocab <= 2^20");
  if ((reinterpret_cast<uintptr_t>(draft) | reinterpret_cast<uintptr_t>(draft_len) | reinterpret_cast<uintptr_t>(target) |
       reinterpret_cast<uintptr_t>(draft_probs) | reinterpret_cast<uintptr_t>(u_accept) |
       reinterpret_cast<uintptr_t>(u_sample) | reinterpret_cast<uintptr_t>(tokens) |
       reinterpret_cast<uintptr_t>(accepted) | reinterpret_cast<uintptr_t>(status)) & 3)
    return bad("Invalid argument: pointers must be 4-byte aligned");
  const uint64_t t_row = target_row_stride ? target_row_stride : vocab;
  const uint64_t d_row = draft_row_stride ? draft_row_stride : vocab;
  const uint64_t t_seq = target_seq_stride ? target_seq_stride : t_row * (max_draft + 1);
  const uint64_t d_seq = draft_seq_stride ? draft_seq_stride : d_row * max_draft;
  if (t_row < vocab || d_row < vocab || t_row > MAX_STRIDE || d_row > MAX_STRIDE || t_seq > MAX_STRIDE || d_seq > MAX_STRIDE)
    return bad("Invalid argument: a row stride is shorter than the vocabulary, or a stride is above 2^40");
  VerifyArgs a;
  a.draft = draft;
  a.draft_len = draft_len;
  a.target = target;
  a.draft_probs = max_draft ? draft_probs : nullptr;
  a.u_accept = u_accept;
  a.u_sample = u_sample;
  a.n_seqs = int(n_seqs);
  a.max_draft = int(max_draft);
  a.vocab = int(vocab);
  a.tokens = tokens;
  a.accepted = accepted;
  a.t_seq = int64_t(t_seq);
  a.t_row = int64_t(t_row);
  a.d_seq = int64_t(d_seq);
  a.d_row = int64_t(d_row);
  a.status = status;
  return cuda_result(launch_verify(a, static_cast<cudaStream_t>(stream)), "draft verification");
}

}  // extern "C"
