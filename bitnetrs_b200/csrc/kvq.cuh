// kvq.cuh — the quantised paged key-value cache: its layout and the launchers
// of the kernels that write it, read it back and attend over it.
//
// A page holds 16 positions.  What one page holds of one kv head is a block:
//   K codes [16][hd], V codes [16][hd], K parameters, V parameters
// with the parameters of a kind as f32 arrays of 16: scale (I8), or scale and
// zero (I4).  The codes of a row are hd bytes (I8, two's complement) or hd/2
// bytes (I4, dimension 2j in the low half of byte j).  A row's value is
// code * scale (I8) or zero + code * scale (I4).  Codes of a row are
// contiguous, so a lane fetches what it multiplies with a few wide loads; the
// parameters of 16 positions are one or two 64-byte lines behind them.
#pragma once

#include "kernels.cuh"

namespace bitnet {

struct KvqView {
  uint8_t* pool = nullptr;         // [pages][kv_heads] blocks
  const int32_t* table = nullptr;  // [seqs][per_seq] page of positions [16j, 16j + 16)
  int pages = 0, seqs = 0, per_seq = 0, kv_heads = 0, hd = 0;
  int i4 = 0;
};
constexpr int kKvqMaxHd = 256;

__host__ __device__ inline int kvq_row_bytes(int hd, int i4) { return i4 ? hd / 2 : hd; }
__host__ __device__ inline int kvq_block_bytes(int hd, int i4) {
  return 2 * kPage * kvq_row_bytes(hd, i4) + 2 * kPage * 4 * (i4 ? 2 : 1);
}
// The blocks of one layer of a model's cache.
KvqView kvq_layer(const KvGeom& g, const int32_t* table, int seqs, int layer);

// Rows of K and V into the cache: row r goes to position row_pos[r] of
// sequence row_seq[r] (a negative position skips the row; without the arrays
// row r is position r of sequence 0).  With rope_cos/sin
// [rope_len][hd/2] K is rotated first, and `q` (optional, nh heads of f32 a
// row) is rotated into q_out [rows][nh*hd].  status gets kStatusNonFinite for
// a value that is not finite and kStatusBadContext for a row with no place.
struct KvqStore {
  const void *k = nullptr, *v = nullptr;
  size_t ldk = 0, ldv = 0;
  int bf16 = 0;
  int rows = 0;
  const int32_t *row_seq = nullptr, *row_pos = nullptr;
  const float *rope_cos = nullptr, *rope_sin = nullptr;
  int rope_len = 0;
  const float* q = nullptr;
  size_t ldq = 0;
  int nh = 0;
  float* q_out = nullptr;
  int32_t* status = nullptr;
};
void launch_kvq_store(const KvqView& c, const KvqStore& s, cudaStream_t st);
// Rows of positions back to f32 or bf16 (rows as above; a row with no place is left alone).
void launch_kvq_load(const KvqView& c, int rows, const int32_t* row_seq, const int32_t* row_pos, void* k, size_t ldk,
                     void* v, size_t ldv, int bf16, int32_t* status, cudaStream_t st);

// Which positions a query row sees: the first `len` of sequence `seq`.  Either
// listed per row (row_seq, row_len + len_bias), or given by runs of
// consecutive positions: rows [cu[i], cu[i+1]) belong to sequence seq_ids[i]
// and stand at positions starts[i], starts[i] + 1, ...; rows outside every
// run are left alone.
struct KvqRows {
  int rows = 0;
  const int32_t *row_seq = nullptr, *row_len = nullptr;
  int len_bias = 0;
  int runs = 0;
  const int32_t *seq_ids = nullptr, *cu = nullptr, *starts = nullptr;
};
struct KvqAttend {
  const void* q = nullptr;  // [rows] of nh * hd, row stride ldq
  void* out = nullptr;      // the same, row stride ldo
  size_t ldq = 0, ldo = 0;
  int bf16 = 0;  // q and out are bf16 (else f32)
  int nh = 0;
  float* lse = nullptr;  // optional [rows][nh]
  int32_t* status = nullptr;
  void* space = nullptr;  // kvq_attend_space bytes
};
size_t kvq_attend_space(int nh, int kv_heads, int hd);
// `max_len` bounds the rows' lengths (a row that says more is cut there and reported).
void launch_kvq_attend(const KvqView& c, const KvqRows& r, const KvqAttend& a, int max_len, cudaStream_t st);
// Runs of rows on the tensor cores, 128 / (heads a unit) tokens a CTA
// (kernels_kvq_prompt.cu); launch_kvq_attend chooses it.
bool kvq_prompt_pays(const KvqView& c, const KvqRows& r, int nh, bool bf16);
void launch_kvq_prompt(const KvqView& c, const KvqRows& r, const KvqAttend& a, int max_len, cudaStream_t st);
const char* kvq_attend_kernel_name(const KvqView& c, const KvqRows& r, int nh, bool bf16);

}  // namespace bitnet
