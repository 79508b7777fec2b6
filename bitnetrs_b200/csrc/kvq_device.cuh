// kvq_device.cuh — device helpers shared by the kernels of the quantised cache.
#pragma once

#include <atomic>

#include "async.cuh"
#include "kvq.cuh"

namespace bitnet {
namespace {

// The block of (position, head) of a sequence; null when the sequence, the
// position or the page that the table names lies outside the cache.
__device__ __forceinline__ uint8_t* block_of(const KvqView& c, int seq, int pos, int head) {
  if ((unsigned)seq >= (unsigned)c.seqs || pos < 0 || pos / kPage >= c.per_seq) return nullptr;
  const int page = c.table[(size_t)seq * c.per_seq + pos / kPage];
  if ((unsigned)page >= (unsigned)c.pages) return nullptr;
  return c.pool + ((size_t)page * c.kv_heads + head) * kvq_block_bytes(c.hd, c.i4);
}
// Parameters of a kind (0 K, 1 V): 16 scales, then for I4 16 zeros.
__device__ __forceinline__ float* block_params(uint8_t* block, int hd, int i4, int kind) {
  return (float*)(block + 2 * kPage * kvq_row_bytes(hd, i4)) + kind * kPage * (i4 ? 2 : 1);
}

__device__ __forceinline__ float load_elem(const void* x, size_t i, int bf16) {
  return bf16 ? bf16_bits_to_f32(((const uint16_t*)x)[i]) : ((const float*)x)[i];
}
__device__ __forceinline__ void store_elem(void* x, size_t i, int bf16, float v) {
  if (bf16)
    ((uint16_t*)x)[i] = f32_to_bf16_bits(v);
  else
    ((float*)x)[i] = v;
}
__device__ __forceinline__ float code_at(const uint8_t* codes, int d, int i4) {
  return i4 ? (float)((codes[d >> 1] >> ((d & 1) * 4)) & 15) : (float)(int8_t)codes[d];
}

// A unit: the query heads of one row that share a kv head, up to kMaxHeads of them.
constexpr int kMaxHeads = 8;
struct Units {
  int per_row, per_kv, heads;  // units a row, units a kv head, heads a unit
};
__host__ __device__ inline Units units_of(int nh, int kv_heads) {
  const int group = nh / kv_heads;
  Units u;
  u.per_kv = (group + kMaxHeads - 1) / kMaxHeads;
  u.heads = (group + u.per_kv - 1) / u.per_kv;
  u.per_row = kv_heads * u.per_kv;
  return u;
}
// The query heads of unit u: [first, first + n).
__device__ __forceinline__ void unit_heads(const Units& us, int nh, int kv_heads, int u, int* kvh, int* first, int* n) {
  const int group = nh / kv_heads, part = u % us.per_kv;
  *kvh = u / us.per_kv;
  *first = *kvh * group + part * us.heads;
  *n = min(us.heads, group - part * us.heads);
}

// One head's joined result (m in units of log2): output and log-sum-exp.
__device__ __forceinline__ float lse_of(float m, float l) {
  return l > 0.0f || isnan(l) ? __fmul_rn(__fadd_rn(m, log2f(l)), 0.69314718055994530942f) : -INFINITY;
}

// How far a score may exceed the running maximum before the sums are rescaled
// (log2): rescaling then all but stops after a unit's first pages.
constexpr float kSlack = 6.0f;

__device__ __forceinline__ void tma_bytes(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
               "l"((uint64_t)src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float f16_lo(uint32_t h) {
  float r;
  asm("{ .reg .f16 a, b; mov.b32 {a, b}, %1; cvt.f32.f16 %0, a; }\n" : "=f"(r) : "r"(h));
  return r;
}
__device__ __forceinline__ float f16_hi(uint32_t h) {
  float r;
  asm("{ .reg .f16 a, b; mov.b32 {a, b}, %1; cvt.f32.f16 %0, b; }\n" : "=f"(r) : "r"(h));
  return r;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {  // within 2^-22; results below 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
// x as two fp16 terms, the larger in the low half.
__device__ __forceinline__ uint32_t two_terms(float x) {
  const uint32_t h = pack_f16(x, 0.0f);
  return pack_f16(f16_lo(h), __fsub_rn(x, f16_lo(h)));
}
// (x & mask) ^ bits in one instruction
__device__ __forceinline__ uint32_t and_xor(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;\n" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
  return r;
}
// Four signed bytes of w as fp16 pairs: elements (0, 2) and (1, 3).  A byte with
// its sign flipped, below the bits of 1024, is 1152 + c.
__device__ __forceinline__ void bytes_f16(uint32_t w, uint32_t* even, uint32_t* odd) {
  *even = add_f16x2(and_xor(w, 0x00ff00ffu, 0x64806480u), 0xe480e480u);
  *odd = add_f16x2(and_xor(w >> 8, 0x00ff00ffu, 0x64806480u), 0xe480e480u);
}
// Eight nibbles c of w as fp16 pairs (c - 7.5) / 512: x[i] = elements (i, i + 4).
// With codes on both sides of 0, and zero + 7.5 scale for the zero, neither of
// the two sums that make an I4 value's product outgrows it.  A nibble alone in
// its 16 bits is the subnormal c / 2^24 (or c / 2^20), so one product and sum,
// both exact, widens a pair.
constexpr float kNibbleMid = 7.5f, kNibbleUnit = 1.0f / 512;
__device__ __forceinline__ void nibbles_f16(uint32_t w, uint32_t* x) {
  constexpr uint32_t kLow = 0x78007800u, kHigh = 0x68006800u, kMid = 0xa380a380u;  // 2^15, 2^11, -7.5 / 512
  const uint32_t v = w >> 8;
  x[0] = fma_f16x2(w & 0x000f000fu, kLow, kMid);
  x[1] = fma_f16x2(w & 0x00f000f0u, kHigh, kMid);
  x[2] = fma_f16x2(v & 0x000f000fu, kLow, kMid);
  x[3] = fma_f16x2(v & 0x00f000f0u, kHigh, kMid);
}
}  // namespace
// Lets a kernel have its dynamic shared memory, once a device and kernel: the
// call costs the host a tenth of a small attention.
inline void allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess) done.fetch_or(bit);
}

}  // namespace bitnet
