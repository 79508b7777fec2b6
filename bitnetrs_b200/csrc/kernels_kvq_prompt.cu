// kernels_kvq_prompt.cu — causal attention of prompts over the quantised paged
// cache on the 5th-generation tensor cores.
//
// A CTA holds 128 rows, the heads of one unit for 128 / heads consecutive
// tokens of a sequence (row = token * heads + head), and goes through the keys
// in tiles of 64 with one pass of the softmax:
//   S[row][key] = Q . K codes        tcgen05.mma, M 128, N 64
//   O[row][dim] += W . V codes       tcgen05.mma, M 128, N head_dim
// The pages of a tile come as they lie (one bulk copy each) and three warps
// widen their codes to fp16, in which they are exact, into tiles of 128-byte
// lines (128-byte swizzle).  One image serves both products: keys by
// dimensions, the contraction along a line for S and across the lines for O.
// The scale of a K row multiplies its column of S, the scale of a V row the
// weight of its key; an I4 zero enters S times the sum of q, and the output as
// a sum of its own.
//
// Q is fp16, multiplied by a power of two a row so that its largest element is
// near 2^14: bf16 is exact there.  An f32 row is the sum of two such terms, as
// the weights W are for both types, each product being two on the same sums.
// Weights of one term (2^-11) move a result by some 2e-4, which a tenth and more
// of the bf16 outputs show; the second term costs bf16 rows 309 against 268 us
// (the 4 ragged prompts below, I4).
//
// Warps 0-3 weigh: a thread reads its row of S, writes W over it as the A
// operand of the second product, and rescales its row of O only when a score
// passes the row's maximum by kSlack (log2) or a weight times its scale of V
// grows too much.  A row's weights have a power of two of their own, by the
// largest such product that the row has had (not by scales alone: a key that
// the row does not see, or gives no weight, must not push the others below what
// fp16 holds); it is folded into the maximum, so that it divides out of the
// result.  The largest is between 2^-2 and 2^9 then (up to 2^15 with the slack),
// so what two terms of fp16 lose of a smaller one is below 2^-23 of it.  While
// the scales of a tile are within 2^6 of one another they tell that by
// themselves; else a row's products are looked at.  Warps 4-6 widen the next
// tile's K and this tile's V.  Warp 7 issues the products, and fetches pages
// kStages tiles ahead (their numbers one tile before that).  They meet at
// mbarriers only:
//   keys_ready    K widened, and its keys' parameters staged    3 warps
//   scores_full   S computed (K's tile is free)                 commit
//   weights_ready W written                                     4 warps
//   values_ready  V widened                                     3 warps
//   output_full   O summed (V's tile, W and S are free)         commit
// The first three have several barriers a kind, in turn: with one, a phase that
// a warp has yet to look at could be followed by the next.  A wait for a
// phase must begin after the phase before has ended and before the next one can
// end.  Every warp waits for each phase in turn, but for output_full the warps
// that weigh: before they arrive with the weights of tile j, O of tile j cannot
// be complete, and O of tile j - 1 (one buffer of S) or j - 2 (two) is, for S of
// tile j was issued after it.
// Two CTAs share an SM, so each has half of its tensor memory.  With a second S
// the next tile's scores are computed while a tile is weighed, K's widening
// running a tile ahead of V's.  Heads of up to 64 have room for it beside O and
// Q (its first term).  Heads of 96 and 128 have it where Q is one term and the
// codes are small enough that Q fits into shared memory beside four tiles of
// pages.  With two tiles, as I8 would have, pages come too late: 275 against
// 267 us for 4 ragged prompts, 4500 rows in all of 32 heads of 128 over 8 (bf16)
// behind up to 1900 positions; I4 gains, 281 to 265 us, and heads of 64 232 to
// 195 us (all with weights of one term).  Those prompts take 310 us over I4, 294
// over I8, 242 with heads of 64 and 489 as f32 rows; 1024 f32 rows of 20 heads
// over 5 (I8) take 52 us.
//
// What bounds it: the handshakes of a tile, S, weights, O, one after the other,
// with half of the SM's issue slots in use and three tenths of the tensor cores'
// time.  Not faster were (weights of one term): the weights by eight warps (305
// to 325 us), rows spread over four lanes so that a key's parameters serve four of
// them (307 to 324 us), and f32 sums brought to the output 32 or 64 dimensions at
// a time (470 to 509 us).
//
// Every wait is bounded; a CTA that gives up records it, waits (bounded) for
// its copies and products and frees its tensor memory.
#include "kvq_device.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace bitnet {

namespace {

constexpr int kPromptRows = 128, kPromptThreads = 256, kWiden = 96, kKeys = 64, kTilePages = kKeys / kPage;
constexpr uint32_t kTmemCols = 256;
// f32 rows: tiles that are summed in tensor memory.  With 8 the error is 0.5 to 1.6
// times that of f32 matrix products, with 4 it is 0.3 to 1.1 times and 1024 rows
// take 72 against 64 us (cold caches).
constexpr int kSumTiles = 8;

template <int HD, bool I4, bool TWO>
struct PromptTile {
  static constexpr int kRow = I4 ? HD / 2 : HD;  // bytes of a row's codes
  static constexpr int kBlock = 2 * kPage * kRow + (I4 ? 256 : 128);
  static constexpr int kAtoms = (HD + 63) / 64;  // 64 elements of fp16 are a 128-byte line
  static constexpr int kOperand = kAtoms * kKeys * 128;
  static constexpr bool kTwoS = HD <= 64 || (I4 && !TWO);  // two buffers of scores
  static constexpr bool kSharedQ = HD > 64 && kTwoS;       // Q (its one term) in shared memory
  static constexpr uint32_t kTmemS = HD, kTmemQ = HD + (kTwoS ? 2 : 1) * kKeys;  // O begins at 0
  static_assert(kTmemQ + (kSharedQ ? 0 : HD / 2) <= kTmemCols, "half of an SM's tensor memory");
  static constexpr int kQ = TWO || kSharedQ ? kAtoms * kPromptRows * 128 : 0;  // Q's second term, or Q
  static constexpr int kRaw = kTilePages * kBlock;
  static constexpr int kStages = TWO && HD > 64 && !I4 ? 2 : 4;  // tiles of pages
  static constexpr int kLag = kTwoS ? 1 : 0;                     // tiles by which V is widened behind K
  static constexpr int kTurns = kTwoS ? 4 : 2;                   // tiles whose parameters, or K's barrier, are kept apart
  static constexpr int kSmem = 1024 + 2 * kOperand + kQ + kStages * kRaw;
};

// Shared-memory operand of 128-byte lines, 128-byte swizzle, groups of 8 lines
// 1024 bytes apart; `lead` is the distance between two runs of 64 elements
// where the lines lie across the contraction.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | (uint64_t)((lead >> 4) & 0x3fffu) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// fp16 operands, f32 sums, M = 128; B's lines along (0) or across (1) the contraction.
__device__ __forceinline__ constexpr uint32_t product(int n, int across) {
  return (1u << 4) | ((uint32_t)across << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kPromptRows >> 4) << 24);
}
__device__ __forceinline__ void mma_tmem_a(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_smem_a(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
      : "memory");
}
// One lane of a whole warp, known as such to the compiler: operands of what it
// issues stay in uniform registers.
__device__ __forceinline__ bool elected() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(is));
  return is != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
// 16 columns of this warp's 32 lanes (without the wait).
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(at), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// 32 bytes at a time: a thread's accesses are a row from its neighbours', so each is a line of its own.
__device__ __forceinline__ void load_f32x8(const float* p, float* x) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store_f32x8(float* p, const float* x) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
               "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}

// Two f32 operations in one instruction, on neighbouring registers; each rounds
// as the plain one does.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The order in which 8 neighbouring dimensions of I4 codes are widened: pairs (i, i + 4).
template <bool I4>
__device__ __forceinline__ constexpr int widened(int i) {
  return I4 ? i / 2 + (i % 2) * 4 : i;
}

// 16 bytes of codes to fp16, 16-byte pieces p[0 ..].
template <bool I4>
__device__ __forceinline__ void widen(const uint4& raw, uint4* p) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (I4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t x[4];
      nibbles_f16(w[i], x);
      p[i] = make_uint4(x[0], x[1], x[2], x[3]);
    }
  } else {
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a byte with its sign flipped, below the bits of 1024, is 1152 + c
      const uint32_t u = w[i] ^ 0x80808080u;
      x[2 * i] = add_f16x2(__byte_perm(u, 0x64646464u, 0x4140), 0xe480e480u);
      x[2 * i + 1] = add_f16x2(__byte_perm(u, 0x64646464u, 0x4342), 0xe480e480u);
    }
    p[0] = make_uint4(x[0], x[1], x[2], x[3]);
    p[1] = make_uint4(x[4], x[5], x[6], x[7]);
  }
}

template <int HD, bool I4, bool TWO>
__global__ void __launch_bounds__(kPromptThreads, 2)
    kvq_prompt_kernel(KvqView c, KvqRows R, KvqAttend a, int max_len, int wide_q, int wide_out) {
  using T = PromptTile<HD, I4, TWO>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t pages_full[T::kStages];
  __shared__ __align__(8) uint64_t keys_ready[T::kTurns], scores_full[2], weights_ready[2], values_ready, output_full, drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up, found_run, found_tile;
  __shared__ __align__(16) float par[T::kTurns][4][kKeys];  // of a tile's keys: K scale and zero, V scale and zero
  __shared__ float pair_a[2][kPromptRows], pair_b[2][kPromptRows], pair_c[2][kPromptRows];
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  // in the prologue two threads share a row of Q, half of it each
  const int half = warp >> 2, row = (warp & 3) * 32 + lane;
  const Units us = units_of(a.nh, c.kv_heads);
  const int tokens_cta = kPromptRows / us.heads;

  // which tile: all units of the last tokens of the first run, then of those before them, and so on
  if (warp == 0) {
    int left = blockIdx.x / us.per_row, run = -1;
    for (int r0 = 0; r0 < R.runs && run < 0; r0 += 32) {
      int n = 0;
      if (r0 + lane < R.runs) {
        const int lo = max(R.cu[r0 + lane], 0), hi = min(R.cu[r0 + lane + 1], R.rows);
        n = hi > lo ? (hi - lo + tokens_cta - 1) / tokens_cta : 0;
      }
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, left < upto);
      if (hit) {
        const int at = __ffs(hit) - 1;
        run = r0 + at;
        const int n_at = __shfl_sync(0xffffffffu, n, at), upto_at = __shfl_sync(0xffffffffu, upto, at);
        left = n_at - 1 - (left - (upto_at - n_at));
      } else {
        left -= __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (lane == 0) {
      found_run = run;
      found_tile = left;
      gave_up = 0;
      for (int i = 0; i < T::kStages; ++i) mbar_init(smem_u32(&pages_full[i]), 1);
      for (int i = 0; i < T::kTurns; ++i) mbar_init(smem_u32(&keys_ready[i]), kWiden / 32);
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_u32(&scores_full[i]), 1);
        mbar_init(smem_u32(&weights_ready[i]), 4);
      }
      mbar_init(smem_u32(&values_ready), kWiden / 32);
      mbar_init(smem_u32(&output_full), 1);
      mbar_init(smem_u32(&drained), 1);
      asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
  }
  __syncthreads();
  const int run = found_run;
  if (run < 0) return;
  const int first_row = max(R.cu[run], 0), rows_run = min(R.cu[run + 1], R.rows) - first_row;
  const int token0 = found_tile * tokens_cta, tokens = min(tokens_cta, rows_run - token0);
  int kvh, h0, heads;
  unit_heads(us, a.nh, c.kv_heads, blockIdx.x % us.per_row, &kvh, &h0, &heads);
  const int seq = R.seq_ids[run];
  // positions that are seen: by the CTA's last token, and by this thread's row
  const long long start64 = (long long)R.starts[run] + (first_row - R.cu[run]) + token0;
  const int start = (int)min(max(start64, -(1LL << 30)), (long long)INT_MAX - 2 * kPromptRows);
  int seen = start + tokens;
  const int token = row / us.heads, head = row % us.heads;
  int limit_pos = start + token + 1;
  bool bad_place = (unsigned)seq >= (unsigned)c.seqs;
  if (bad_place) seen = 0;
  if (seen > max_len) {
    bad_place = true;
    seen = max_len;
  }
  if (bad_place && tid == 0) atomicOr(a.status, kStatusBadContext);
  limit_pos = min(limit_pos, seen);
  const bool live_row = token < tokens && head < heads;
  const size_t out_row = (size_t)(first_row + token0 + token);
  const size_t out_at = out_row * a.ldo + (size_t)(h0 + head) * HD;
  if (seen <= 0) {
    if (live_row && warp < 4) {
      for (int i = 0; i < HD; ++i) store_elem(a.out, out_at + i, a.bf16, 0.0f);
      if (a.lse) a.lse[out_row * a.nh + h0 + head] = -INFINITY;
    }
    return;
  }
  const int tiles = (seen + kKeys - 1) / kKeys;

  uint8_t* const base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *const k_tile = base, *const v_tile = base + T::kOperand, *const q_tile = base + 2 * T::kOperand;
  uint8_t* const raws = base + 2 * T::kOperand + T::kQ;
  if (warp == 7) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  // one tile's pages, by warp 7; next_page is the lane's page of the tile after the last one asked for
  int next_page = 0;
  auto look_up = [&](int j) {
    const int at = j * kTilePages + lane;
    next_page = 0;
    if (lane < kTilePages && at * kPage < seen) next_page = c.table[(size_t)seq * c.per_seq + at];
  };
  auto fetch = [&](int j) {
    const int stage = j % T::kStages, pages = min(kTilePages, (seen + kPage - 1) / kPage - j * kTilePages);
    const uint32_t bar = smem_u32(&pages_full[stage]);
    if ((unsigned)next_page >= (unsigned)c.pages) {  // looked at here, where it is used: the load has had a tile's time
      atomicOr(a.status, kStatusBadContext);
      next_page = 0;
    }
    const int page = next_page;
    if (lane == 0) mbar_expect_tx(bar, pages * T::kBlock);
    __syncwarp();
    if (lane < pages)
      tma_bytes(smem_u32(raws + stage * T::kRaw + lane * T::kBlock),
                c.pool + ((size_t)page * c.kv_heads + kvh) * T::kBlock, T::kBlock, bar);
    look_up(j + 1);
  };
  if (warp == 7) {
    look_up(0);
    for (int j = 0; j < min(tiles, T::kStages); ++j) fetch(j);
  }

  // q: the row's largest element, its sum, and whether all are finite, from the two threads' halves
  const size_t q_at = out_row * a.ldq + (size_t)(h0 + head) * HD + half * (HD / 2);
  auto load_q = [&](int i, float* x) {  // dimensions i .. i + 7 of the half
    if (!live_row) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = 0.0f;
    } else if (wide_q && !a.bf16) {
      const float4 u = *(const float4*)((const float*)a.q + q_at + i), v = *(const float4*)((const float*)a.q + q_at + i + 4);
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else if (wide_q) {
      const uint4 u = *(const uint4*)((const uint16_t*)a.q + q_at + i);
      x[0] = bf_lo(u.x), x[1] = bf_hi(u.x), x[2] = bf_lo(u.y), x[3] = bf_hi(u.y);
      x[4] = bf_lo(u.z), x[5] = bf_hi(u.z), x[6] = bf_lo(u.w), x[7] = bf_hi(u.w);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = load_elem(a.q, q_at + i + k, a.bf16);
    }
  };
  float top = 0.0f, qsum = 0.0f, odd = 0.0f;
#pragma unroll 2
  for (int i = 0; i < HD / 2; i += 8) {
    float x[8];
    load_q(i, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      top = fmaxf(top, fabsf(x[k]));
      qsum = __fadd_rn(qsum, x[k]);
      odd = __fmaf_rn(x[k], 0.0f, odd);  // NaN when an element is not finite
    }
  }
  pair_a[half][row] = top;
  pair_b[half][row] = qsum;
  pair_c[half][row] = odd;
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  const uint32_t tlane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  top = fmaxf(pair_a[0][row], pair_a[1][row]);
  qsum = __fadd_rn(pair_b[0][row], pair_b[1][row]);
  odd = __fadd_rn(pair_c[0][row], pair_c[1][row]);
  // 2^14 / 2^floor(log2 top), the exponents kept within what a float and its inverse can hold
  const int e = min(max((int)(__float_as_uint(top) >> 23), 20), 254);
  const float up = __uint_as_float((uint32_t)(268 - e) << 23), down = __uint_as_float((uint32_t)(e - 14) << 23);
  constexpr float kUnit = I4 ? kNibbleUnit : 1.0f;  // of the widened codes
  const float qs = __fadd_rn(__fmul_rn(__fdiv_rn(1.4426950408889634f / kUnit, __fsqrt_rn((float)HD)), down), odd);
  qsum = __fmul_rn(qsum, __fmul_rn(up, kUnit));
#pragma unroll 1
  for (int i = 0; i < HD / 2; i += 16) {
    uint32_t hi[8];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float x[8];
      load_q(i + 8 * g, x);
      uint32_t lo[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float u = __fmul_rn(x[widened<I4>(2 * k)], up), v = __fmul_rn(x[widened<I4>(2 * k + 1)], up);
        hi[4 * g + k] = pack_f16(u, v);
        if (TWO) lo[k] = pack_f16(__fsub_rn(u, f16_lo(hi[4 * g + k])), __fsub_rn(v, f16_hi(hi[4 * g + k])));
      }
      if (TWO || T::kSharedQ) {
        const int d = half * (HD / 2) + i + 8 * g, piece = (d % 64) / 8;
        const uint32_t* x16 = TWO ? lo : hi + 4 * g;
        *(uint4*)(q_tile + d / 64 * (kPromptRows * 128) + row * 128 + ((piece ^ (row & 7)) << 4)) =
            make_uint4(x16[0], x16[1], x16[2], x16[3]);
      }
    }
    __syncwarp();
    if (!T::kSharedQ) tmem_st8(tlane + T::kTmemQ + half * (HD / 4) + i / 2, hi);
  }
  tmem_wait_st();

  // the codes of K (0) or V (1) of the tile in `j`'s buffer, widened into an operand
  auto widen_tile = [&](int j, int kind, uint8_t* dst) {
    constexpr int kPieces = T::kRow / 16, kOut = I4 ? 4 : 2;  // 16-byte pieces of a row, and what each becomes
    const uint8_t* raw = raws + j % T::kStages * T::kRaw;
#pragma unroll
    for (int i = 0; i < (kKeys * kPieces + kWiden - 1) / kWiden; ++i) {
      const int at = i * kWiden + (tid - 128);
      if (kKeys * kPieces % kWiden != 0 && at >= kKeys * kPieces) break;
      const int key = at / kPieces, piece = at % kPieces;
      uint4 p[4], u = *(const uint4*)(raw + key / kPage * T::kBlock + (kind * kPage + key % kPage) * T::kRow + piece * 16);
      // lanes whose pieces go to the second 64 elements write the halves of their output the other way round: eight
      // lanes then write to eight places of a line, not to four
      const bool turn = HD > 64 && piece >= kPieces / 2;
      if (turn) u = make_uint4(u.z, u.w, u.x, u.y);
      widen<I4>(u, p);
#pragma unroll
      for (int k = 0; k < kOut; ++k) {
        const int to = piece * kOut + (turn ? k ^ (kOut / 2) : k);  // 16-byte piece of the widened row
        *(uint4*)(dst + to / 8 * (kKeys * 128) + key * 128 + (((to % 8) ^ (key & 7)) << 4)) = p[k];
      }
    }
  };
  auto stage_params = [&](int j) {
    const int key = tid - 128;
    if (key < kKeys) {
      const float* p = (const float*)(raws + j % T::kStages * T::kRaw + key / kPage * T::kBlock + 2 * kPage * T::kRow) + key % kPage;
      // behind the context the bytes may be anything
      const bool live = j * kKeys + key < seen;
      par[j % T::kTurns][0][key] = live ? p[0] : 0.0f;
      par[j % T::kTurns][1][key] = I4 && live ? __fmaf_rn(kNibbleMid, p[0], p[kPage]) : 0.0f;
      par[j % T::kTurns][2][key] = live ? p[I4 ? 2 * kPage : kPage] : 0.0f;
      par[j % T::kTurns][3][key] = I4 && live ? __fmaf_rn(kNibbleMid, p[2 * kPage], p[3 * kPage]) : 0.0f;
    }
  };
  auto scores_at = [&](int j) -> uint32_t { return T::kTmemS + (T::kTwoS && (j & 1) ? kKeys : 0); };
  // The second terms first: the sums are cut, not rounded, to f32, each time by
  // what they have grown to.  (2^-25 of the result an addition on average, eight
  // of them a tile: f32 rows bring the sums out every kSumTiles tiles, bf16 rows
  // have nowhere to bring them to and are off by 2^-22 a tile, 2^-13 at 32768 keys.)
  auto issue_scores = [&](int j) {
    const uint32_t d = tmem + scores_at(j);
    auto k_at = [&](int k) { return operand(smem_u32(k_tile) + k / 4 * (kKeys * 128) + k % 4 * 32, 16); };
    if (TWO || T::kSharedQ)
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
        mma_smem_a(d, operand(smem_u32(q_tile) + k / 4 * (kPromptRows * 128) + k % 4 * 32, 16), k_at(k),
                   product(kKeys, 0), k > 0);
    if (!T::kSharedQ)
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
        mma_tmem_a(d, tmem + T::kTmemQ + 8 * k, k_at(k), product(kKeys, 0), TWO || k > 0);
    mma_commit(smem_u32(&scores_full[j & 1]));
  };
  auto issue_output = [&](int j) {
    const uint32_t w = tmem + scores_at(j);
    const bool adds = TWO ? j % kSumTiles != 0 : j > 0;
    auto v_at = [&](int k) { return operand(smem_u32(v_tile) + k * 2048, kKeys * 128); };
#pragma unroll
    for (int k = 0; k < kKeys / 16; ++k) mma_tmem_a(tmem, w + 32 + 8 * k, v_at(k), product(HD, 1), adds || k > 0);
#pragma unroll
    for (int k = 0; k < kKeys / 16; ++k) mma_tmem_a(tmem, w + 8 * k, v_at(k), product(HD, 1), true);
    mma_commit(smem_u32(&output_full));
  };
  // One arrival a warp, after its writes to shared memory (for the products) or to tensor memory.
  auto arrive = [&](uint64_t& bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bar));
  };
  auto wait = [&](uint64_t& bar, int phase) {
    const bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar), phase & 1, &gave_up));
    if (!ok) give_up(&gave_up, a.status);
    return ok;
  };
  // Q is in place
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  tmem_wait_st();
  before_sync();
  __syncthreads();
  after_sync();

  // m: a maximum of the row's scores (in the units of the products times their
  // scales) at most kSlack / qs below the true one; mq: m * qs less the power
  // of two of the row's weights
  float m = -INFINITY, mq = -INFINITY, limit = -INFINITY, l = 0.0f, zsum = 0.0f;
  if (warp == 7) {
    // ---- products ----
    // scores of tile j into the buffer that held the weights of tile j - 2 (two buffers) or j - 1
    auto scores = [&](int j) {
      constexpr int kBack = T::kTwoS ? 2 : 1;
      if (!wait(keys_ready[j % T::kTurns], j / T::kTurns) || (j >= kBack && !wait(output_full, j - kBack))) return false;
      after_sync();
      if (elected()) issue_scores(j);
      __syncwarp();
      return true;
    };
    bool ok = scores(0);
    for (int j = 0; j < tiles && ok; ++j) {
      if (T::kTwoS && j + 1 < tiles && !scores(j + 1)) break;
      if (!wait(values_ready, j)) break;
      if (j + T::kStages < tiles) fetch(j + T::kStages);  // the tile's codes have been widened
      if (!wait(weights_ready[j & 1], j / 2)) break;
      after_sync();
      if (elected()) issue_output(j);
      __syncwarp();
      if (!T::kTwoS && j + 1 < tiles) ok = scores(j + 1);
    }
  } else if (warp >= 4) {
    // ---- widening ----
    for (int j = 0; j < tiles + T::kLag; ++j) {
      if (j < tiles) {
        if (!wait(pages_full[j % T::kStages], j / T::kStages) || (j > 0 && !wait(scores_full[(j - 1) & 1], (j - 1) / 2))) break;
        stage_params(j);
        widen_tile(j, 0, k_tile);
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        arrive(keys_ready[j % T::kTurns]);
      }
      const int v = j - T::kLag;
      if (v >= 0) {
        if (v > 0 && !wait(output_full, v - 1)) break;
        widen_tile(v, 1, v_tile);
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        arrive(values_ready);
      }
    }
  } else {
    // ---- weighing ----
    int ev = limit_pos > 0 ? 100 : -100;  // the row's weights are multiplied by 2^ev
    float cap = 0.0f;                     // 2^(9 - the largest ev of the warp's rows)
    float most = 0.0f;  // of the row's largest weight (relative to m) times scale of V: what it is at least
    float kept = 1.0f;  // what m's growth has left of the sums that are in the output's place
    // What a key's weight is multiplied with: the scale of V.  A zero (I4) goes into a sum of its own, in 32 bits; it
    // counts 2^24 times less, so that it cannot overflow there (a scale that much smaller is lost in 32 bits anyway).
    auto size_of = [&](const float(*p)[kKeys], int key) {
      return I4 ? fmaxf(p[2][key], __fmul_rn(fabsf(p[3][key]), 0x1p-24f)) : p[2][key];
    };
    // 16 elements of the row's output, in the order in which they lie in o
    auto load_sums = [&](int i, float* o) {
      const float* p = (const float*)a.out + out_at + i;
      float x[16];
      if (wide_out == 2) {
        load_f32x8(p, x);
        load_f32x8(p + 8, x + 8);
      } else if (wide_out) {
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
          const float4 u = *(const float4*)(p + k);
          x[k] = u.x, x[k + 1] = u.y, x[k + 2] = u.z, x[k + 3] = u.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = p[k];
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) o[k] = __fmaf_rn(x[k / 8 * 8 + widened<I4>(k % 8)], kept, o[k]);
    };
    auto store_out = [&](int i, const float* o) {
      float x[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k / 8 * 8 + widened<I4>(k % 8)] = o[k];
      if (!TWO && wide_out) {
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
          uint32_t u[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(x[k + 2 * n], x[k + 2 * n + 1]);
            u[n] = *(const uint32_t*)&p;
          }
          *(uint4*)((uint16_t*)a.out + out_at + i + k) = make_uint4(u[0], u[1], u[2], u[3]);
        }
      } else if (wide_out == 2) {
        store_f32x8((float*)a.out + out_at + i, x);
        store_f32x8((float*)a.out + out_at + i + 8, x + 8);
      } else if (wide_out) {
#pragma unroll
        for (int k = 0; k < 16; k += 4)
          *(float4*)((float*)a.out + out_at + i + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) store_elem(a.out, out_at + i + k, !TWO, x[k]);
      }
    };
    for (int j = 0; j < tiles; ++j) {
      if (!wait(keys_ready[j % T::kTurns], j / T::kTurns) || !wait(scores_full[j & 1], j / 2)) break;
      after_sync();
      const uint32_t s_at = tlane + scores_at(j);
      float s[kKeys];
#pragma unroll
      for (int i = 0; i < kKeys; i += 16) tmem_ld16(s_at + i, (uint32_t*)s + i);
      tmem_wait_ld();
      const float(*pj)[kKeys] = par[j % T::kTurns];
      const int key0 = j * kKeys;
#pragma unroll
      for (int i = 0; i < kKeys; i += 4) {
        const ulonglong2 ks = *(const ulonglong2*)&pj[0][i];
        uint64_t u = pair(s[i], s[i + 1]), v = pair(s[i + 2], s[i + 3]);
        if constexpr (I4) {
          const ulonglong2 kz = *(const ulonglong2*)&pj[1][i];
          u = fma2(u, ks.x, mul2(pair(qsum, qsum), kz.x));
          v = fma2(v, ks.y, mul2(pair(qsum, qsum), kz.y));
        } else {
          u = mul2(u, ks.x);
          v = mul2(v, ks.y);
        }
        const float2 x = unpair(u), y = unpair(v);
        s[i] = x.x, s[i + 1] = x.y, s[i + 2] = y.x, s[i + 3] = y.y;
      }
      if (TWO && j > 0 && j % kSumTiles == 0) {  // the sums so far, to the output's place
        if (!wait(output_full, j - 1)) break;
        after_sync();
#pragma unroll 1
        for (int i = 0; i < HD; i += 16) {
          float o[16];
          __syncwarp();
          tmem_ld16(tlane + i, (uint32_t*)o);
          tmem_wait_ld();
          if (live_row) {
            if (j > kSumTiles) load_sums(i, o);
            store_out(i, o);
          }
        }
        __syncwarp();
        kept = 1.0f;
      }
      const bool masked = key0 + kKeys > min(start + 1, seen);  // keys that the CTA's first token does not see, or no one does
      if (masked) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (key0 + i >= limit_pos) s[i] = -INFINITY;
      }
      float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kKeys; i += 2) tops[i / 2 % 4] = max3(tops[i / 2 % 4], s[i], s[i + 1]);
      const float top_s = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      // a score above the slack, or a scale of V that some row's 2^ev takes above 2^9
      const float size_a = size_of(pj, lane), size_b = size_of(pj, lane + 32), vtop = fmaxf(size_a, size_b);
      if (__any_sync(0xffffffffu, top_s > limit || vtop > cap)) {
        const float m_new = fmaxf(m, top_s), m_at = __fmul_rn(m_new, qs);
        // the tile's largest and least size, as bits (not numbers: 0)
        const uint32_t high = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(vtop, 0.0f)));
        const uint32_t low = __reduce_min_sync(
            0xffffffffu, __float_as_uint(fminf(fmaxf(size_a, 0.0f), fmaxf(size_b, 0.0f))));
        if (m == -INFINITY) {
          if (limit_pos > 0) ev = min(max(131 - (int)(high >> 23), -100), 100);  // the largest scale near 2^4
        } else {
          most = __fmul_rn(most, exp2_approx(__fsub_rn(__fmul_rn(m, qs), m_at)));
        }
        // a key with the largest score so far has a weight of 1
        if (top_s >= m) most = fmaxf(most, __uint_as_float(low));
        const float unit = __int_as_float((127 + ev) << 23);
        const bool fits = __fmul_rn(__uint_as_float(high), unit) <= 512.0f && __fmul_rn(most, unit) >= 0.25f;
        if (__any_sync(0xffffffffu, !fits && limit_pos > 0)) {
#pragma unroll
          for (int i = 0; i < kKeys; ++i)  // (a product that is not a number is passed over)
            most = fmaxf(most, __fmul_rn(exp2_approx(__fmaf_rn(s[i], qs, -m_at)), size_of(pj, i)));
          const float now = __fmul_rn(most, unit);
          if (!(now >= 0.25f && now <= 512.0f) && limit_pos > 0)
            ev = min(max(129 - (int)(__float_as_uint(most) >> 23), -100), 100);  // near 2^2 (no product yet: as large as it may be)
        }
        cap = __int_as_float((136 - __reduce_max_sync(0xffffffffu, ev)) << 23);
        m = m_new;
        const float nq = __fsub_rn(m_at, (float)ev);
        const float step = __fsub_rn(mq, nq), keep = mq == nq || m == -INFINITY ? 1.0f : exp2_approx(step);
        mq = nq;
        limit = __fadd_rn(m, __fdiv_rn(kSlack, qs));
        if (step < -100.0f) {  // values that grow so far leave nothing of the outputs before them, but their weights count
          const float half_step = exp2_approx(__fmul_rn(0.5f, step));
          l = __fmul_rn(__fmul_rn(l, half_step), half_step);
        } else {
          l = __fmul_rn(l, keep);
        }
        zsum = __fmul_rn(zsum, keep);
        kept = __fmul_rn(kept, keep);
        if ((TWO ? j % kSumTiles != 0 : j > 0) && __any_sync(0xffffffffu, keep != 1.0f)) {
          if (!wait(output_full, j - 1)) break;
          after_sync();
#pragma unroll 1
          for (int i = 0; i < HD; i += 16) {
            float o[16];
            tmem_ld16(tlane + i, (uint32_t*)o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __fmul_rn(o[k], keep);
            tmem_st16(tlane + i, (const uint32_t*)o);
          }
        }
      }
      // weights, over the scores; a key that the row does not see weighs nothing, whatever its scale
      uint64_t l_tile = 0, z_tile = 0;  // a tile's sums by themselves: a long context's would lose their small terms
      auto weigh = [&](auto some_hidden) {
#pragma unroll
        for (int i = 0; i < kKeys; i += 16) {
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int n = 0; n < 16; n += 4) {
            const ulonglong2 vs = *(const ulonglong2*)&pj[2][i + n];
            ulonglong2 vz = make_ulonglong2(0, 0);
            if constexpr (I4) vz = *(const ulonglong2*)&pj[3][i + n];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int at = i + n + 2 * k;
              const float2 x = unpair(fma2(pair(s[at], s[at + 1]), pair(qs, qs), pair(-mq, -mq)));
              const uint64_t w = pair(exp2_approx(x.x), exp2_approx(x.y));
              l_tile = add2(l_tile, w);
              uint64_t scale = k ? vs.y : vs.x, zero = k ? vz.y : vz.x;
              if constexpr (decltype(some_hidden)::value) {
                const bool h0 = key0 + at >= limit_pos, h1 = key0 + at + 1 >= limit_pos;
                const float2 a = unpair(scale), b = unpair(zero);
                scale = pair(h0 ? 0.0f : a.x, h1 ? 0.0f : a.y);
                zero = pair(h0 ? 0.0f : b.x, h1 ? 0.0f : b.y);
              }
              if constexpr (I4) z_tile = fma2(w, zero, z_tile);
              const uint64_t p = mul2(w, scale);
              const float2 f = unpair(p);
              const uint32_t h = pack_f16(f.x, f.y);
              hi[n / 2 + k] = h;
              const float2 r = unpair(add2(p, pair(-f16_lo(h), -f16_hi(h))));
              lo[n / 2 + k] = pack_f16(r.x, r.y);
            }
          }
          tmem_st8(s_at + i / 2, hi);
          tmem_st8(s_at + 32 + i / 2, lo);
        }
      };
      if (masked)
        weigh(std::true_type{});
      else
        weigh(std::false_type{});
      const float2 lt = unpair(l_tile), zt = unpair(z_tile);
      l = __fadd_rn(l, __fadd_rn(lt.x, lt.y));
      if (I4) zsum = __fadd_rn(zsum, __fadd_rn(zt.x, zt.y));
      tmem_wait_st();
      before_sync();
      // the last wait below must not take the phase before the last for its own; that one cannot end
      // before this arrival, and the one before it has ended
      if (T::kTwoS && j > 0 && j == tiles - 1 && !wait(output_full, j - 1)) break;
      arrive(weights_ready[j & 1]);
    }
    wait(output_full, tiles - 1);
    after_sync();
    const bool sees = limit_pos > 0, good = *(volatile int*)&gave_up == 0;
    const float inv = sees ? __fdiv_rn(1.0f, l) : 0.0f;
#pragma unroll 1
    for (int i = 0; i < HD; i += 16) {
      float o[16];
      __syncwarp();
      tmem_ld16(tlane + i, (uint32_t*)o);
      tmem_wait_ld();
      if (live_row && good) {
        if (TWO && tiles > kSumTiles) load_sums(i, o);
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = sees ? __fmul_rn(I4 ? __fmaf_rn(o[k], 1.0f / kUnit, zsum) : o[k], inv) : 0.0f;
        store_out(i, o);
      }
    }
    if (live_row && good && a.lse) a.lse[out_row * a.nh + h0 + head] = sees ? lse_of(mq, l) : -INFINITY;
    __syncwarp();
  }
  before_sync();
  __syncthreads();
  if (warp == 7) {
    after_sync();
    if (gave_up) {
      // what is in flight lands (or its wait runs out) before the CTA may go
      if (lane == 0) {
        mma_commit(smem_u32(&drained));
        mbar_wait(smem_u32(&drained), 0, nullptr);
        for (int i = 0; i < T::kStages; ++i) {  // one of the two is past
          mbar_wait(smem_u32(&pages_full[i]), 0, nullptr);
          mbar_wait(smem_u32(&pages_full[i]), 1, nullptr);
        }
      }
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <int HD, bool I4, bool TWO>
void launch_prompt(const KvqView& c, const KvqRows& r, const KvqAttend& a, int max_len, cudaStream_t st) {
  using T = PromptTile<HD, I4, TWO>;
  const Units us = units_of(a.nh, c.kv_heads);
  const int tokens = kPromptRows / us.heads;
  const unsigned ctas = (unsigned)(r.rows / tokens + r.runs) * us.per_row;
  auto* kernel = kvq_prompt_kernel<HD, I4, TWO>;
  static std::atomic<uint64_t> allowed{0};
  allow_shared((const void*)kernel, T::kSmem, allowed);
  const size_t run = a.bf16 ? 8 : 4;
  const int wide_q = (uintptr_t)a.q % 16 == 0 && a.ldq % run == 0;
  // 16 bytes of the output at a time, or 32 (f32)
  const int wide_out = (uintptr_t)a.out % 16 || a.ldo % run ? 0 : a.bf16 || (uintptr_t)a.out % 32 || a.ldo % 8 ? 1 : 2;
  kernel<<<ctas, kPromptThreads, T::kSmem, st>>>(c, r, a, max_len, wide_q, wide_out);
  count_launch();
}
template <int HD>
void launch_prompt_of(const KvqView& c, const KvqRows& r, const KvqAttend& a, int max_len, cudaStream_t st) {
  if (c.i4)
    a.bf16 ? launch_prompt<HD, true, false>(c, r, a, max_len, st) : launch_prompt<HD, true, true>(c, r, a, max_len, st);
  else
    a.bf16 ? launch_prompt<HD, false, false>(c, r, a, max_len, st) : launch_prompt<HD, false, true>(c, r, a, max_len, st);
}

}  // namespace

// Runs of rows are taken here where that is the faster way.  For 64 positions
// of every row's context a CTA of this kernel takes 1.6 us by itself and an SM
// with two of them 1.2 us a CTA (f32 rows 2.4 and 2.1 us); the single-token
// kernel takes 64 positions of one unit in 1.9 ns of the whole GPU.  These are
// heads of 128, up to four a unit; smaller heads take less of both, so that the
// two meet at about the same number of rows.  Measured (this kernel, the other;
// 8 units, us): behind 8000 positions 64 rows 281 and 109, 128 rows 285 and 188,
// 256 rows 293 and 352 (f32, I4, heads of 128), 64 rows 162 and 109, 128 rows 164
// and 190 (bf16); fresh prompts of 64 rows 25 and 23 (f32), 21 and 25 (bf16), 512
// rows 43 and 72 (f32).  128 rows behind 8000 positions with heads of 64 172 and
// 125 (f32), 129 and 125 (bf16), with heads of 32 147 and 102, 129 and 102.  The
// rule takes the faster of each but for bf16 rows: the fresh 64 (25) and the two
// of 129.
bool kvq_prompt_pays(const KvqView& c, const KvqRows& r, int nh, bool bf16) {
  if (!r.runs || (c.hd != 32 && c.hd != 64 && c.hd != 96 && c.hd != 128)) return false;
  const Units us = units_of(nh, c.kv_heads);
  const double ctas = ((double)r.rows / (kPromptRows / us.heads) + r.runs) * us.per_row;
  if (ctas > (double)INT_MAX) return false;
  return std::max(bf16 ? 1.6 : 2.4, (bf16 ? 1.2 : 2.1) * ctas / 148) < 1.9e-3 * r.rows * us.per_row;
}

void launch_kvq_prompt(const KvqView& c, const KvqRows& r, const KvqAttend& a, int max_len, cudaStream_t st) {
  if (r.rows <= 0 || r.runs <= 0) return;
  switch (c.hd) {
    case 32:
      return launch_prompt_of<32>(c, r, a, max_len, st);
    case 64:
      return launch_prompt_of<64>(c, r, a, max_len, st);
    case 96:
      return launch_prompt_of<96>(c, r, a, max_len, st);
    case 128:
      return launch_prompt_of<128>(c, r, a, max_len, st);
  }
}

}  // namespace bitnet
