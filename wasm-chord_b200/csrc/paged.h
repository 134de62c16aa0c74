// Paged serving operators (append, attend, verify): the kernels' arguments and
// launchers. The checked entry points are in paged.cpp.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace wcb {
namespace paged {

enum { E_F32 = 0, E_F16 = 1, E_BF16 = 2 };  // element types (WCB_KV_*)
enum { ST_BAD_PAGE = 1, ST_BAD_ROWS = 2, ST_BAD_LEN = 4, ST_BAD_TOKEN = 8, ST_BAD_PROBS = 16, ST_ABORTED = 32 };

// pool and batch as the kernels see them (wcb_paged_kv, wcb_paged_batch)
struct Pool {
  void* k;
  void* v;
  int64_t page_stride, token_stride, head_stride;
  int page_size, n_pages, n_kv, head_dim;
};

struct Batch {
  const int32_t* q_start;
  const int32_t* kv_len;
  const int32_t* page_table;
  uint32_t* status;
  int n_seqs, n_tokens, max_pages;
};

struct AppendArgs {
  Pool pool;
  Batch batch;
  const void *q, *k, *v;
  void* q_out;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  const float *q_norm, *k_norm;
  float eps;
  int n_heads, rot, halves;
  double turns[64];  // inv_freq / 2 pi
};

struct AttendArgs {
  Pool pool;
  Batch batch;
  const void* q;
  void* out;
  float* lse;
  int64_t q_stride, out_stride;
  float scale_log2;  // scale * log2(e)
  int n_heads, rep;  // rep: query heads of a key head
  uint64_t rep_inv;  // 2^40 / rep, rounded up: rows are divided by rep in many places
  int window;        // 0: none
  int row_lo, row_hi;  // sequences with row_lo < rows (new tokens * rep) <= row_hi are this launch's
  int* tickets;      // one per CTA, zero between calls
  float* part;       // partial results, two pieces per CTA
  uint64_t wait_ns;  // a wait for a copy or a product ends after so long
  uint32_t withheld; // bytes that a tile by TMA waits for and that do not come (test hook; 0)
};

struct VerifyArgs {
  const int32_t *draft, *draft_len;
  const float *target, *draft_probs, *u_accept, *u_sample;
  int n_seqs, max_draft, vocab;
  int32_t *tokens, *accepted;
  int64_t t_seq, t_row, d_seq, d_row;
  uint32_t* status;
};

// Work of an attention call is cut into equal parts, one per CTA; a part leaves at most two
// partial results.
constexpr int SMS = 148;
constexpr int ATTEND_CTAS = 4 * SMS;  // most CTAs of the mma.sync kernel
constexpr int TC_CTAS = SMS;      // parts of the tensor-core kernel: one CTA on each SM
constexpr int TC_ROWS = 256;      // rows of its CTA
constexpr int TC_TICKETS = 640;   // its first ticket, two a CTA
constexpr size_t TICKET_BYTES = 4096;

cudaError_t launch_append(const AppendArgs& a, int act, int cache, cudaStream_t s);
cudaError_t launch_attend_16(const AttendArgs& a, int act, int rows, cudaStream_t s);
cudaError_t launch_attend_32(const AttendArgs& a, int cache, int rows, cudaStream_t s);
cudaError_t launch_attend_tc(const AttendArgs& a, int act, cudaStream_t s);
cudaError_t launch_attend_tc32(const AttendArgs& a, int cache, cudaStream_t s);
cudaError_t launch_verify(const VerifyArgs& a, cudaStream_t s);

}  // namespace paged
}  // namespace wcb
