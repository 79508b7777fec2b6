// kvq.cu — C entry points of the quantised paged key-value cache on the device.
#include <climits>

#include "internal.h"
#include "kvq.cuh"

using namespace bitnet;

namespace {

std::string sz(size_t v) { return std::to_string(v); }

// The calling thread's current device, put back when the call returns.
struct DeviceScope {
  int before = -1;
  explicit DeviceScope(int device) {
    cudaGetDevice(&before);
    if (before != device)
      cudaSetDevice(device);
    else
      before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
};

int check_format(int kv_dtype, size_t head_dim) {
  if (kv_dtype != BITNET_KV_I8 && kv_dtype != BITNET_KV_I4) return config_error("kv_dtype must be I8 or I4");
  if (head_dim == 0 || head_dim % 2 != 0 || head_dim > (size_t)kKvqMaxHd)
    return config_error("head_dim of a quantised cache must be even and at most " + sz(kKvqMaxHd) + ", got " +
                        sz(head_dim));
  return BITNET_OK;
}

int check_pages(const bitnet_cuda_kv_pages* p, KvqView* c) {
  if (!p) return shape_error("non-null cache description", "null");
  BN_TRY(check_format(p->kv_dtype, p->head_dim));
  if (!p->pool || !p->page_table) return shape_error("non-null pool and page_table", "null");
  if ((uintptr_t)p->pool % 16) return shape_error("a 16-byte aligned pool", "a pool at " + sz((uintptr_t)p->pool % 16) + " mod 16");
  if ((uintptr_t)p->page_table % 4) return shape_error("a 4-byte aligned page_table", "an unaligned one");
  if (!p->pages || !p->seqs || !p->pages_per_seq || !p->kv_heads)
    return shape_error("pages, seqs, pages_per_seq and kv_heads > 0", "0");
  if (p->pages > INT_MAX || p->seqs > INT_MAX || p->pages_per_seq > INT_MAX / kPage || p->kv_heads > 65535)
    return shape_error("pages, seqs and positions below 2^31, kv_heads below 2^16", "more");
  c->pool = (uint8_t*)p->pool;
  c->table = p->page_table;
  c->pages = (int)p->pages;
  c->seqs = (int)p->seqs;
  c->per_seq = (int)p->pages_per_seq;
  c->kv_heads = (int)p->kv_heads;
  c->hd = (int)p->head_dim;
  c->i4 = p->kv_dtype == BITNET_KV_I4;
  return BITNET_OK;
}

int check_matrix(const void* p, size_t ld, size_t width, int bf16, const char* what) {
  if (!p) return shape_error(std::string("non-null ") + what, "null");
  if ((uintptr_t)p % (bf16 ? 2 : 4)) return shape_error(std::string(what) + " aligned to its elements", "an unaligned address");
  if (ld < width) return shape_error(std::string("row stride of ") + what + " >= " + sz(width), sz(ld));
  return BITNET_OK;
}

int check_words(const void* p, const char* what) {
  if (!p) return shape_error(std::string("non-null ") + what, "null");
  if ((uintptr_t)p % 4) return shape_error(std::string("4-byte aligned ") + what, "an unaligned address");
  return BITNET_OK;
}

// Checked last: every other refusal is the same with and without a GPU.
int check_ctx(const bitnet_cuda_ctx* ctx) { return ctx ? BITNET_OK : shape_error("non-null context", "null"); }

int check_rows(size_t rows, const KvqView& c) {
  // up to 32 lanes a row, kind and head; the grid's first dimension bounds their blocks
  if (rows > (size_t)INT_MAX / (2 * (size_t)c.kv_heads))
    return shape_error("rows * 2 * kv_heads < 2^31", "rows = " + sz(rows));
  return BITNET_OK;
}

int check_attend(const KvqView& c, const void* q, size_t ldq, int bf16, size_t rows, size_t n_heads, size_t max_len,
                 void* out, size_t ldo, float* lse, void* workspace, size_t workspace_bytes, int32_t* status,
                 KvqAttend* a, int* bound) {
  if (n_heads == 0 || n_heads % c.kv_heads != 0)
    return shape_error("n_heads a multiple of kv_heads (" + sz(c.kv_heads) + ")", sz(n_heads));
  // the kernels' 32-bit row numbers go on by up to a grid, or a CTA's tokens, behind the last row
  if (n_heads * (size_t)c.hd > (size_t)INT_MAX || rows > (size_t)INT_MAX - 1024)
    return shape_error("n_heads * head_dim below 2^31, rows below 2^31 - 1024", "more");
  const size_t width = n_heads * (size_t)c.hd;
  BN_TRY(check_matrix(q, ldq, width, bf16, "q"));
  BN_TRY(check_matrix(out, ldo, width, bf16, "out"));
  if (lse) BN_TRY(check_words(lse, "lse"));
  BN_TRY(check_words(status, "status"));
  if (max_len > (size_t)c.per_seq * kPage)
    return shape_error("max_len <= pages_per_seq * 16 (" + sz((size_t)c.per_seq * kPage) + ")", sz(max_len));
  const size_t need = kvq_attend_space((int)n_heads, c.kv_heads, c.hd);
  if (!workspace || (uintptr_t)workspace % 16) return shape_error("a 16-byte aligned workspace", workspace ? "an unaligned one" : "null");
  if (workspace_bytes < need) return shape_error("a workspace of " + sz(need) + " bytes", sz(workspace_bytes));
  a->q = q;
  a->out = out;
  a->ldq = ldq;
  a->ldo = ldo;
  a->bf16 = bf16 != 0;
  a->nh = (int)n_heads;
  a->lse = lse;
  a->status = status;
  a->space = workspace;
  *bound = (int)max_len;
  return BITNET_OK;
}

}  // namespace

extern "C" {

int bitnet_cuda_kv_block_bytes(int kv_dtype, size_t head_dim, size_t* bytes) {
  if (!bytes) return shape_error("non-null bytes", "null");
  BN_TRY(check_format(kv_dtype, head_dim));
  *bytes = (size_t)kvq_block_bytes((int)head_dim, kv_dtype == BITNET_KV_I4);
  return BITNET_OK;
}

int bitnet_cuda_kv_store_device(bitnet_cuda_ctx* ctx, const bitnet_cuda_kv_pages* cache, const void* k, size_t ldk,
                                const void* v, size_t ldv, int x_is_bf16, size_t rows, const int32_t* row_seq,
                                const int32_t* row_pos, const float* rope_cos, const float* rope_sin,
                                size_t rope_len, int32_t* status, void* stream) {
  KvqView c;
  BN_TRY(check_pages(cache, &c));
  if (rows == 0) return check_ctx(ctx);
  BN_TRY(check_rows(rows, c));
  const size_t width = (size_t)c.kv_heads * c.hd;
  BN_TRY(check_matrix(k, ldk, width, x_is_bf16, "k"));
  BN_TRY(check_matrix(v, ldv, width, x_is_bf16, "v"));
  BN_TRY(check_words(row_seq, "row_seq"));
  BN_TRY(check_words(row_pos, "row_pos"));
  BN_TRY(check_words(status, "status"));
  if ((rope_cos == nullptr) != (rope_sin == nullptr)) return shape_error("rope_cos and rope_sin, both or neither", "one of them");
  if (rope_cos) {
    BN_TRY(check_words(rope_cos, "rope_cos"));
    BN_TRY(check_words(rope_sin, "rope_sin"));
    if (rope_len == 0 || rope_len > (size_t)INT_MAX) return shape_error("0 < rope_len < 2^31", sz(rope_len));
  }
  KvqStore s;
  s.k = k;
  s.v = v;
  s.ldk = ldk;
  s.ldv = ldv;
  s.bf16 = x_is_bf16 != 0;
  s.rows = (int)rows;
  s.row_seq = row_seq;
  s.row_pos = row_pos;
  s.rope_cos = rope_cos;
  s.rope_sin = rope_sin;
  s.rope_len = (int)rope_len;
  s.status = status;
  BN_TRY(check_ctx(ctx));
  DeviceScope on(ctx->device);
  launch_kvq_store(c, s, stream ? (cudaStream_t)stream : ctx->stream);
  BN_CUDA(cudaGetLastError());
  return BITNET_OK;
}

int bitnet_cuda_kv_load_device(bitnet_cuda_ctx* ctx, const bitnet_cuda_kv_pages* cache, size_t rows,
                               const int32_t* row_seq, const int32_t* row_pos, void* k, size_t ldk, void* v,
                               size_t ldv, int out_is_bf16, int32_t* status, void* stream) {
  KvqView c;
  BN_TRY(check_pages(cache, &c));
  if (rows == 0) return check_ctx(ctx);
  BN_TRY(check_rows(rows, c));
  const size_t width = (size_t)c.kv_heads * c.hd;
  BN_TRY(check_matrix(k, ldk, width, out_is_bf16, "k"));
  BN_TRY(check_matrix(v, ldv, width, out_is_bf16, "v"));
  BN_TRY(check_words(row_seq, "row_seq"));
  BN_TRY(check_words(row_pos, "row_pos"));
  BN_TRY(check_words(status, "status"));
  BN_TRY(check_ctx(ctx));
  DeviceScope on(ctx->device);
  launch_kvq_load(c, (int)rows, row_seq, row_pos, k, ldk, v, ldv, out_is_bf16 != 0, status,
                  stream ? (cudaStream_t)stream : ctx->stream);
  BN_CUDA(cudaGetLastError());
  return BITNET_OK;
}

int bitnet_cuda_kv_attention_workspace(const bitnet_cuda_kv_pages* cache, size_t n_heads, size_t* bytes) {
  if (!bytes) return shape_error("non-null bytes", "null");
  KvqView c;
  BN_TRY(check_pages(cache, &c));
  if (n_heads == 0 || n_heads % c.kv_heads != 0 || n_heads > (size_t)INT_MAX)
    return shape_error("n_heads a multiple of kv_heads (" + sz(c.kv_heads) + ")", sz(n_heads));
  *bytes = kvq_attend_space((int)n_heads, c.kv_heads, c.hd);
  return BITNET_OK;
}

int bitnet_cuda_kv_attention_device(bitnet_cuda_ctx* ctx, const bitnet_cuda_kv_pages* cache, const void* q, size_t ldq,
                                    int x_is_bf16, size_t rows, size_t n_heads, const int32_t* row_seq,
                                    const int32_t* row_len, size_t max_len, void* out, size_t ldo, float* lse,
                                    void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  KvqView c;
  BN_TRY(check_pages(cache, &c));
  if (rows == 0) return check_ctx(ctx);
  KvqAttend a;
  int bound = 0;
  BN_TRY(check_attend(c, q, ldq, x_is_bf16, rows, n_heads, max_len, out, ldo, lse, workspace, workspace_bytes, status,
                      &a, &bound));
  BN_TRY(check_words(row_seq, "row_seq"));
  BN_TRY(check_words(row_len, "row_len"));
  KvqRows r;
  r.rows = (int)rows;
  r.row_seq = row_seq;
  r.row_len = row_len;
  BN_TRY(check_ctx(ctx));
  DeviceScope on(ctx->device);
  launch_kvq_attend(c, r, a, bound, stream ? (cudaStream_t)stream : ctx->stream);
  BN_CUDA(cudaGetLastError());
  return BITNET_OK;
}

int bitnet_cuda_kv_prompt_attention_device(bitnet_cuda_ctx* ctx, const bitnet_cuda_kv_pages* cache, const void* q,
                                           size_t ldq, int x_is_bf16, size_t rows, size_t n_heads, size_t n_seqs,
                                           const int32_t* seq_ids, const int32_t* cu_rows, const int32_t* starts,
                                           size_t max_len, void* out, size_t ldo, float* lse, void* workspace,
                                           size_t workspace_bytes, int32_t* status, void* stream) {
  KvqView c;
  BN_TRY(check_pages(cache, &c));
  if (rows == 0 || n_seqs == 0) return check_ctx(ctx);
  KvqAttend a;
  int bound = 0;
  BN_TRY(check_attend(c, q, ldq, x_is_bf16, rows, n_heads, max_len, out, ldo, lse, workspace, workspace_bytes, status,
                      &a, &bound));
  if (n_seqs >= (size_t)1 << 30) return shape_error("n_seqs below 2^30", sz(n_seqs));
  BN_TRY(check_words(seq_ids, "seq_ids"));
  BN_TRY(check_words(cu_rows, "cu_rows"));
  BN_TRY(check_words(starts, "starts"));
  KvqRows r;
  r.rows = (int)rows;
  r.runs = (int)n_seqs;
  r.seq_ids = seq_ids;
  r.cu = cu_rows;
  r.starts = starts;
  BN_TRY(check_ctx(ctx));
  DeviceScope on(ctx->device);
  launch_kvq_attend(c, r, a, bound, stream ? (cudaStream_t)stream : ctx->stream);
  BN_CUDA(cudaGetLastError());
  return BITNET_OK;
}

}  // extern "C"
