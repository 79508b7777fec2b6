// kernels_kvq_attend.cu — GQA attention over the quantised paged cache, split
// over the context and joined.
#include "kvq_device.cuh"
#include "kvq_ring.h"

#include <algorithm>

namespace bitnet {

namespace {

// ---------------------------------------------------------------------------
// Attention.  A unit is the (up to kMaxHeads) query heads of one row that share
// a kv head; its work is the pages of the row's context.  The pages of all
// units form one line, row by row and unit by unit, that is cut into equal
// shares, one a CTA, so that a long context and a ragged batch load the GPU
// evenly without the host knowing the lengths.  A unit that lies inside one
// share is finished there.  One that is cut leaves a partial result (running
// maximum, sum, unnormalised output) in each share it touches; a second kernel
// joins them in the line's order, so a result depends on the lengths alone.
// A share holds at most two partial units: its first (slot 0) and its last
// (slot 1; a share inside one unit uses slot 0).
// ---------------------------------------------------------------------------
constexpr int kAttendCtas = 148 * 4;
struct ShareMeta {
  int row, unit;  // the unit that begins in this share and ends in a later one (row < 0: none)
  int ends;       // whether the unit of slot 0 ends in this share
  int pad;
};

// What row r sees: its sequence and how many positions (-1: the row belongs to no run).
__device__ __forceinline__ int row_context(const KvqView& c, const KvqRows& R, int r, int max_len, int* seq,
                                           int32_t* status) {
  long long len;
  if (R.runs) {
    if (r < R.cu[0] || r >= R.cu[R.runs]) return -1;
    int lo = 0, hi = R.runs;  // cu[lo] <= r < cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (R.cu[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    *seq = R.seq_ids[lo];
    len = (long long)R.starts[lo] + (r - R.cu[lo]) + 1;
  } else {
    *seq = R.row_seq[r];
    len = (long long)R.row_len[r] + R.len_bias;
  }
  if (len <= 0) return 0;
  if ((unsigned)*seq >= (unsigned)c.seqs) {
    atomicOr(status, kStatusBadContext);
    return 0;
  }
  if (len > max_len) {
    atomicOr(status, kStatusBadContext);
    len = max_len;
  }
  return (int)len;
}

__device__ __forceinline__ float* share_slot(void* space, int shares, int share, int slot, int hd, const Units& us) {
  return (float*)((ShareMeta*)space + shares) + ((size_t)share * 2 + slot) * (us.heads * (hd + 4));
}

// A partial result that a warp of the tensor-core kernel leaves for its CTA's
// join, behind the shares' slots; rows padded like the ring's.
__device__ __forceinline__ float* warp_slot(void* space, int shares, int warp, int hd, const Units& us) {
  const size_t slots = (size_t)shares * 2 * (us.heads * (hd + 4));
  return (float*)((ShareMeta*)space + shares) + slots + (size_t)warp * (us.heads * (hd + 4));
}

__device__ void write_empty_row(const KvqAttend& a, int hd, int r) {
  for (int i = threadIdx.x; i < a.nh * hd; i += blockDim.x) store_elem(a.out, (size_t)r * a.ldo + i, a.bf16, 0.0f);
  if (a.lse)
    for (int i = threadIdx.x; i < a.nh; i += blockDim.x) a.lse[(size_t)r * a.nh + i] = -INFINITY;
}

constexpr int kPlainWarps = 4;

// The simple form, for every head size: a warp takes whole pages; lanes share
// a score as 16 positions x 2 halves of the dimensions, then own dimensions of
// the output.
__global__ void __launch_bounds__(kPlainWarps * 32)
    kvq_attend_plain_kernel(KvqView c, KvqRows R, KvqAttend a, int max_len) {
  extern __shared__ float sm[];
  __shared__ int found[4];
  __shared__ long long total_sh, base_sh;
  const int hd = c.hd, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Units us = units_of(a.nh, c.kv_heads);
  float* qs = sm;                                   // [heads][hd], scaled
  float* part = qs + us.heads * hd;                 // [warps][heads][hd]
  float* ml = part + kPlainWarps * us.heads * hd;   // [warps][heads][2]
  const int shares = gridDim.x, share = blockIdx.x;
  ShareMeta* meta = (ShareMeta*)a.space;
  // the line's length, and rows that see nothing
  if (tid == 0) {
    total_sh = 0;
    found[0] = -1;
  }
  __syncthreads();
  long long mine = 0;
  for (int r = tid; r < R.rows; r += blockDim.x) {
    int seq;
    const int len = row_context(c, R, r, max_len, &seq, a.status);
    if (len > 0) mine += (len + kPage - 1) / kPage;
  }
  atomicAdd((unsigned long long*)&total_sh, (unsigned long long)mine);
  for (int r = share; r < R.rows; r += shares) {
    int seq;
    if (row_context(c, R, r, max_len, &seq, a.status) == 0) write_empty_row(a, hd, r);
  }
  __syncthreads();
  const long long total = total_sh * us.per_row;
  const long long cuts = min((long long)shares, (total + kPlainWarps - 1) / kPlainWarps);
  if (tid == 0) meta[share] = ShareMeta{-1, 0, 0, 0};
  if (share >= cuts) return;
  long long at = total * share / cuts;
  const long long end = total * (share + 1) / cuts;
  // the row in which the share begins
  if (tid == 0) {
    long long base = 0;
    for (int r = 0; r < R.rows; ++r) {
      int seq;
      const int len = row_context(c, R, r, max_len, &seq, a.status);
      const long long n = len > 0 ? (long long)((len + kPage - 1) / kPage) * us.per_row : 0;
      if (at < base + n) {
        found[0] = r;
        base_sh = base;
        break;
      }
      base += n;
    }
  }
  __syncthreads();
  int r = found[0];
  long long base = base_sh;
  const float qscale = __fdiv_rn(1.4426950408889634f, __fsqrt_rn((float)hd));
  while (at < end && r < R.rows) {
    int seq = 0;
    const int len = row_context(c, R, r, max_len, &seq, a.status);
    const int pages = len > 0 ? (len + kPage - 1) / kPage : 0;
    if (at >= base + (long long)pages * us.per_row) {
      base += (long long)pages * us.per_row;
      ++r;
      continue;
    }
    const int u = (int)((at - base) / pages), first_page = (int)((at - base) % pages);
    const int n_pages = (int)min((long long)(pages - first_page), end - at);
    int kvh, h0, heads;
    unit_heads(us, a.nh, c.kv_heads, u, &kvh, &h0, &heads);
    __syncthreads();
    for (int i = tid; i < heads * hd; i += blockDim.x)
      qs[i] = __fmul_rn(load_elem(a.q, (size_t)r * a.ldq + (size_t)h0 * hd + i, a.bf16), qscale);
    __syncthreads();
    float m[kMaxHeads], l[kMaxHeads], acc[kMaxHeads][kKvqMaxHd / 32];
#pragma unroll
    for (int h = 0; h < kMaxHeads; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.0f;
#pragma unroll
      for (int i = 0; i < kKvqMaxHd / 32; ++i) acc[h][i] = 0.0f;
    }
    for (int p = first_page + warp; p < first_page + n_pages; p += kPlainWarps) {
      uint8_t* block = block_of(c, seq, p * kPage, kvh);
      if (!block) {
        if (lane == 0) atomicOr(a.status, kStatusBadContext);
        continue;
      }
      const int slot = lane & 15, rowb = kvq_row_bytes(hd, c.i4);
      const bool live = p * kPage + slot < len;
      const float* kp = block_params(block, hd, c.i4, 0);
      const float* vp = block_params(block, hd, c.i4, 1);
      const float ks = kp[slot], kz = c.i4 ? kp[kPage + slot] : 0.0f;
      const float vs = live ? vp[slot] : 0.0f, vz = c.i4 && live ? vp[kPage + slot] : 0.0f;
      const uint8_t* kc = block + (size_t)slot * rowb;
#pragma unroll
      for (int h = 0; h < kMaxHeads; ++h) {
        if (h >= heads) continue;
        float dot = 0.0f;
        for (int d = lane >> 4; d < hd; d += 2) dot = __fmaf_rn(qs[h * hd + d], __fmaf_rn(code_at(kc, d, c.i4), ks, kz), dot);
        dot = __fadd_rn(dot, __shfl_xor_sync(0xffffffffu, dot, 16));
        if (!live) dot = -INFINITY;
        float top = dot;
#pragma unroll
        for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float mn = fmaxf(m[h], top), keep = exp2f(__fsub_rn(m[h], mn));
        const float w = live ? exp2f(__fsub_rn(dot, mn)) : 0.0f;
        m[h] = mn;
        float sum = w;
#pragma unroll
        for (int o = 8; o; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
        l[h] = __fmaf_rn(l[h], keep, sum);
#pragma unroll
        for (int i = 0; i < kKvqMaxHd / 32; ++i) acc[h][i] = __fmul_rn(acc[h][i], keep);
        for (int j = 0; j < kPage && p * kPage + j < len; ++j) {
          const float wj = __shfl_sync(0xffffffffu, w, j);
          const float s = __shfl_sync(0xffffffffu, vs, j), z = __shfl_sync(0xffffffffu, vz, j);
          const uint8_t* vc = block + (size_t)(kPage + j) * rowb;
#pragma unroll
          for (int i = 0; i < kKvqMaxHd / 32; ++i)
            if (lane + 32 * i < hd)
              acc[h][i] = __fmaf_rn(wj, __fmaf_rn(code_at(vc, lane + 32 * i, c.i4), s, z), acc[h][i]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kMaxHeads; ++h) {
      if (h >= heads) continue;
#pragma unroll
      for (int i = 0; i < kKvqMaxHd / 32; ++i)
        if (lane + 32 * i < hd) part[(warp * us.heads + h) * hd + lane + 32 * i] = acc[h][i];
      if (lane == 0) {
        ml[(warp * us.heads + h) * 2] = m[h];
        ml[(warp * us.heads + h) * 2 + 1] = l[h];
      }
    }
    __syncthreads();
    const bool begins = first_page == 0, ends = first_page + n_pages == pages;
    float* slot = share_slot(a.space, shares, share, begins && !ends ? 1 : 0, hd, us);
    for (int i = tid; i < heads * hd; i += blockDim.x) {
      const int h = i / hd, d = i % hd;
      float M = -INFINITY, L = 0.0f, o = 0.0f;
      for (int w = 0; w < kPlainWarps; ++w) M = fmaxf(M, ml[(w * us.heads + h) * 2]);
      for (int w = 0; w < kPlainWarps; ++w) {
        const float mw = ml[(w * us.heads + h) * 2], lw = ml[(w * us.heads + h) * 2 + 1];
        if (lw == 0.0f) continue;  // a warp without pages
        const float f = exp2f(__fsub_rn(mw, M));
        L = __fmaf_rn(lw, f, L);
        o = __fmaf_rn(part[(w * us.heads + h) * hd + d], f, o);
      }
      if (begins && ends) {
        store_elem(a.out, (size_t)r * a.ldo + (size_t)h0 * hd + i, a.bf16, __fdiv_rn(o, L));
        if (a.lse && d == 0) a.lse[(size_t)r * a.nh + h0 + h] = lse_of(M, L);
      } else {
        slot[h * (hd + 4) + d] = o;
        if (d == 0) {
          slot[h * (hd + 4) + hd] = M;
          slot[h * (hd + 4) + hd + 1] = L;
        }
      }
    }
    if (tid == 0) {
      if (begins && !ends) {
        meta[share].row = r;
        meta[share].unit = u;
      }
      if (!begins) meta[share].ends = ends;
    }
    at += n_pages;
  }
}

// ---------------------------------------------------------------------------
// The tensor-core form, for heads of 32, 64, 96 and 128.
//
// One warp multiplies a page (two of them in turn), its 16 positions (scores) or 16
// dimensions (output) being the M of a product, and four heads its N.
//   S[pos][head] = K codes . q        m16n8k32, 8-bit integers
//   O[dim][head] += V codes^T . w     m16n8k16, fp16 with f32 sums
// Scores: codes go into the product as they lie in memory (I4: as 16 (c - 8),
// with zero + 8 scale for the zero, so that neither part of a score outgrows
// it).  q is held as a
// 31-bit integer a dimension (relative to the head's largest element) in four
// balanced digits of base 256, one column each, so that the integer products
// are exact and a head's four columns, two in each of two products, are the
// score.  The scale of a K row multiplies it.
// Output: codes are exact in fp16.  A weight is not, so it is the sum of two
// fp16 terms (22 bits), in neighbouring columns; a lane's pair of sums belongs
// to one head.  The scale of a V row multiplies its weight before that is
// split.  An I4 zero enters scores (times the sum of q) and output as a sum of
// its own.
// The weights are multiplied by a power of two a head so that the largest
// product of a weight and a scale of V that the head has had is between 2^-2 and
// 2^9 (up to 2^15 with the slack; rescaled like the sums when a scale comes that
// might exceed it): two terms then hold 2^-23 of it.  The scales alone do not
// tell: a key with large values and no weight must not push the others below
// what fp16 holds.
//
// Each warp has a ring of pages of its own in shared memory.  One lane fetches
// a page with two copies of the asynchronous copy engine, the codes as a tile
// of 128-byte lines with their 16-byte pieces exchanged (128-byte swizzle), so
// that loads of 8 rows x 16 bytes meet no bank twice, and the parameters with
// them or by themselves.
// Measured on a batch of 256 contexts of 128 to 4096 (20 heads over 5, heads of
// 128, I8), with the same bytes asked for ahead: copies by each lane (cp.async)
// stop at 4.0 TB/s, since a load that goes through L1 needs an entry there
// until it lands; the ring takes 131 us, 5.1 TB/s, and 100003 positions of one
// sequence as I4 43 us, 2.7 TB/s, where instructions and the ends are the bound.
//
// Here the line of pages is cut into equal shares for the warps, not the
// CTAs, so that no warp waits for another before its share is done.  The warps
// of a CTA hold neighbouring shares: at the end the CTA joins the units that
// its warps cut, and leaves to the join kernel those that CTAs cut.
//
// The order of dimensions inside a product is free, so the words that ldmatrix
// leaves in a lane (V's transposed: two positions' bytes of a dimension) go into
// the products as they are; q, and the output as it is written, are in the order
// that this gives.
// ---------------------------------------------------------------------------
// The tensor cores cut their f32 sums, 2^-25 of the result a page on average, so
// every kSumPages pages they are added, rounded, to sums of a lane's own.
constexpr int kSumPages = 32;
constexpr int kMmaMaxWarps = 8;
constexpr int kMmaShares = 296;  // two CTAs an SM with up to four heads a unit, else one
template <int HD, bool I4, int NT>
struct MmaTile {
  static constexpr int kRow = I4 ? HD / 2 : HD;         // bytes of a row's codes
  static constexpr int kChunks = kRow / 16;             // 16-byte pieces of a row
  static constexpr int kCodes = 2 * kPage * kRow;         // bytes of a page's codes
  static constexpr int kParams = I4 ? 256 : 128;
  // The parameters come with the codes, as further lines of the tile, where
  // tiles rounded up to 1024 bytes leave room for them; else by themselves.
  static constexpr bool kWhole = kCodes + kParams <= 2 * 1024;
  static constexpr int kTile = (kCodes + (kWhole ? kParams : 0) + 1023) / 1024 * 1024;
  static constexpr int kApart = kWhole ? 0 : kParams;
  static constexpr int kLines = (kCodes + (kWhole ? kParams : 0)) / 128;
  // Warps a CTA and stages (of two pages) a warp: what shared memory holds
  // twice an SM (once with NT = 2).
  static constexpr int kWarps = NT == 1 && kTile > 3 * 1024 ? 6 : kMmaMaxWarps;
  static constexpr int kPair = kWarps * 2 * (kTile + kApart);
  static constexpr int kStages = NT == 2 ? 3 : 4 * kPair <= 104 * 1024 ? 4 : 104 * 1024 / kPair;
  static constexpr int kRing = kStages * 2 * kTile;  // a warp's tiles
  static constexpr int kSmem = kWarps * kStages * 2 * (kTile + kApart);
  static constexpr int kKSteps = HD / 32, kMTiles = HD / 16;
  static constexpr int kPartStride = HD + 4;  // floats a head of a warp's partial result
};

// Where byte x of a tile lies: 16-byte pieces of a 128-byte line are exchanged by the line's number.
__device__ __forceinline__ int swizzled(int x) { return x ^ ((x >> 3) & 0x70); }

// A tile of one block's codes, lines of 128 bytes, swizzled as above.
__device__ __forceinline__ void tma_codes(uint32_t dst, const CUtensorMap* map, int block, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %2, %3}], [%4];\n" ::"r"(dst),
      "l"((uint64_t)map), "r"(0), "r"(block), "r"(bar)
      : "memory");
}
// N (2 or 4) matrices of 8 rows x 16 bytes, whose row addresses the lanes
// 8 i .. 8 i + 7 hold for matrix i.  A lane gets bytes 4t .. 4t + 3 of row g;
// transposed (as 16-bit elements) bytes 2g, 2g + 1 of rows 2t and 2t + 1.
template <int N, bool TRANS>
__device__ __forceinline__ void load_matrices(uint32_t addr, uint32_t* w) {
  if constexpr (N == 4 && TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr));
  else if constexpr (N == 4)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr));
  else if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}
// All pieces of 16 rows: w[2 c + h] is piece c of rows 8 h .. 8 h + 7.
template <int CHUNKS, bool TRANS>
__device__ __forceinline__ void load_rows(uint32_t tile, const int* at, uint32_t* w) {
#pragma unroll
  for (int c = 0; c < CHUNKS; c += 2) {
    if (c + 1 < CHUNKS)
      load_matrices<4, TRANS>(tile + at[c / 2], w + 2 * c);
    else
      load_matrices<2, TRANS>(tile + at[c / 2], w + 2 * c);
  }
}
// c += product, fp16
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c = product (START) or c += product
template <bool START>
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if constexpr (START)
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};\n"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
  else
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
// x as balanced base-256 digits, the least in the lowest byte (|x| <= 2^30).
__device__ __forceinline__ uint32_t digits(int x) { return ((uint32_t)x + 0x80808080u) ^ 0x80808080u; }
// Byte `i` of four words.
__device__ __forceinline__ uint32_t gather_byte(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int i) {
  const uint32_t sel = (uint32_t)(i | ((i + 4) << 4));
  return __byte_perm(__byte_perm(a, b, sel), __byte_perm(c, d, sel), 0x5410);
}

// The line of work as every CTA sees it: thread t of the CTA sums a run of
// `each` rows, and before[t] is the line up to that run.
template <int THREADS>
struct Line {
  long long before[THREADS + 1];
  long long warp_sum[THREADS / 32];
  int len[THREADS], seq[THREADS];  // of the rows, where there is one a thread
};
// x / d, in 32 bits where that is enough (a 64-bit division takes some 100 instructions).
__device__ __forceinline__ long long div_fast(long long x, int d) {
  return (x >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)d) : x / d;
}
// A unit weighs its pages and kUnitCost more: what q, the first copies and the
// result of a unit cost a warp, in pages.
constexpr int kUnitCost = 2;
template <int THREADS>
__device__ void measure_line(Line<THREADS>& line, const KvqView& c, const KvqRows& R, int max_len, int per_row, int each,
                             int32_t* status) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = min(tid * each, R.rows), r1 = min(r0 + each, R.rows);
  long long mine = 0;
  for (int r = r0; r < r1; ++r) {
    int seq = 0;
    const int len = row_context(c, R, r, max_len, &seq, status);
    line.len[tid] = len;
    line.seq[tid] = seq;
    if (len > 0) mine += (long long)((len + kPage - 1) / kPage + kUnitCost) * per_row;
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) line.warp_sum[warp] = upto;
  __syncthreads();
  long long first = 0;
  for (int w = 0; w < warp; ++w) first += line.warp_sum[w];
  line.before[tid + 1] = first + upto;
  if (tid == 0) line.before[0] = 0;
  __syncthreads();
}

// What a warp leaves for the CTA's join: the unit that begins in its share and
// does not end there (in its ring), and the part of an earlier one (in its
// ring, or in the workspace when the warp went on after it).
struct WarpNote {
  int row, unit;        // row < 0: none begins here and ends later
  int has0, ends0, far0;
};

template <int HD, bool I4, int NT>
__global__ void __launch_bounds__(MmaTile<HD, I4, NT>::kWarps * 32, NT == 1 ? 2 : 1)
    kvq_attend_mma_kernel(KvqView c, KvqRows R, KvqAttend a, int max_len, int min_weight, int wide_q, int whole_units,
                          const __grid_constant__ CUtensorMap tmap) {
  using T = MmaTile<HD, I4, NT>;
  constexpr int kMmaWarps = T::kWarps, kThreads = kMmaWarps * 32;
  extern __shared__ __align__(1024) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[kMmaWarps][T::kStages];
  __shared__ int gave_up;
  __shared__ Line<kThreads> line;
  __shared__ float ml[kMmaWarps][2][kMaxHeads][2];  // of a warp's slots 0 and 1
  __shared__ WarpNote notes[kMmaWarps];
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const Units us = units_of(a.nh, c.kv_heads);
  const int shares = gridDim.x, share = blockIdx.x;
  if (lane == 0) {
    for (int i = 0; i < T::kStages; ++i) mbar_init(smem_u32(&full[warp][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (tid == 0) {
    gave_up = 0;
    asm volatile("prefetch.tensormap [%0];\n" ::"l"((uint64_t)&tmap) : "memory");
  }
  const int each = (R.rows + kThreads - 1) / kThreads;
  if (!whole_units) measure_line<kThreads>(line, c, R, max_len, us.per_row, each, a.status);
  // a row's sequence and length: with a row a thread they are here already
  auto context = [&](int r, int* seq) {
    if (each > 1 || whole_units) return row_context(c, R, r, max_len, seq, a.status);
    *seq = line.seq[r];
    return line.len[r];
  };
  long long at, end, base;
  int r;
  if (whole_units) {
    // a CTA to a unit, whose pages its warps share
    r = share / us.per_row;
    base = 0;
    int seq;
    const int len = row_context(c, R, r, max_len, &seq, a.status);
    if (len == 0 && share % us.per_row == 0) write_empty_row(a, HD, r);
    const int pages = len > 0 ? (len + kPage - 1) / kPage : 0;
    const long long first = (long long)(share % us.per_row) * (pages + kUnitCost) + kUnitCost;
    const int takers = max(min(pages, kMmaWarps), 1);  // neighbours, a page or more each
    at = first + (long long)pages * min(warp, takers) / takers;
    end = first + (long long)pages * min(warp + 1, takers) / takers;
    __syncthreads();  // the barriers are initialised
  } else {
    for (r = share; r < R.rows; r += shares) {
      int seq;
      if (context(r, &seq) == 0) write_empty_row(a, HD, r);
    }
    // shares of `quot` or one more
    const long long total = line.before[kThreads];
    const long long cuts = min((long long)shares * kMmaWarps, div_fast(total + min_weight - 1, min_weight));
    const long long quot = cuts ? div_fast(total, (int)cuts) : 0, over = total - quot * cuts;
    const long long nth = (long long)share * kMmaWarps + warp;
    at = nth < cuts ? quot * nth + min(nth, over) : 0;
    end = nth < cuts ? at + quot + (nth < over) : 0;
    int lo = 0, hi = kThreads;  // before[lo] <= at < before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (line.before[mid] <= at)
        lo = mid;
      else
        hi = mid;
    }
    r = lo * each;
    base = line.before[lo];
  }
  WarpNote note{-1, 0, 0, 0, 0};
  uint8_t* const mine = ring + warp * T::kRing;
  // where the parameters are: behind a tile's codes, or in a ring of their own
  uint8_t* const params = T::kWhole ? mine + T::kCodes : ring + kMmaWarps * T::kRing + warp * (T::kStages * 2 * T::kParams);
  constexpr int kParStride = T::kWhole ? T::kTile : T::kParams;
  const uint32_t mine_s = smem_u32(mine), params_s = smem_u32(params), bar_s = smem_u32(&full[warp][0]);
  const float qscale = __fdiv_rn(1.4426950408889634f, __fsqrt_rn((float)HD));
  // the rows that this lane names for the loads of K and V
  int at_k[(T::kChunks + 1) / 2], at_v[(T::kChunks + 1) / 2];
#pragma unroll
  for (int c = 0; c < T::kChunks; c += 2) {
    const int row = lane & 15, piece = min(c + (lane >> 4), T::kChunks - 1);
    at_k[c / 2] = swizzled(row * T::kRow + piece * 16);
    at_v[c / 2] = swizzled((kPage + row) * T::kRow + piece * 16);
  }
  StageRing<T::kStages> copies;
  bool failed = false;  // the same in all lanes

  while (at < end && r < R.rows) {
    int seq = 0;
    const int len = context(r, &seq);
    const int pages = len > 0 ? (len + kPage - 1) / kPage : 0;
    const int weight = pages ? pages + kUnitCost : 0;
    if (at >= base + (long long)weight * us.per_row) {
      base += (long long)weight * us.per_row;
      ++r;
      continue;
    }
    const int u = (int)div_fast(at - base, weight);
    const long long first = base + (long long)u * weight + kUnitCost;  // where the unit's pages begin
    const int p0 = (int)max(at - first, 0LL), p1 = (int)min(end - first, (long long)pages);
    at = first + pages;
    if (p1 <= p0) continue;
    int kvh, h0, heads;
    unit_heads(us, a.nh, c.kv_heads, u, &kvh, &h0, &heads);
    const int n_pages = p1 - p0;
    const int32_t* row_table = c.table + (size_t)seq * c.per_seq + p0;

    // the copies of pages i and i + 1; lane l of the ids holds page (block of 32) + l
    int ids = 0;
    auto fetch = [&](int i) {
      if (i >= n_pages) return;
      if ((i & 31) == 0) {
        ids = i + lane < n_pages ? row_table[i + lane] : 0;
        if ((unsigned)ids >= (unsigned)c.pages) {
          atomicOr(a.status, kStatusBadContext);
          ids = 0;
        }
      }
      const int first_block = __shfl_sync(0xffffffffu, ids, i & 31) * c.kv_heads + kvh;
      const int second_block = __shfl_sync(0xffffffffu, ids, (i + 1) & 31) * c.kv_heads + kvh;
      if (lane == 0) {
        const uint32_t bar = bar_s + copies.fill * 8, tile = mine_s + copies.fill * (2 * T::kTile);
        const uint32_t par = params_s + copies.fill * (2 * kParStride);
        const bool both = i + 1 < n_pages;
        mbar_expect_tx(bar, (T::kCodes + T::kParams) << both);
        tma_codes(tile, &tmap, first_block, bar);
        if (!T::kWhole)
          tma_bytes(par, c.pool + (size_t)first_block * (T::kCodes + T::kParams) + T::kCodes, T::kParams, bar);
        if (both) {
          tma_codes(tile + T::kTile, &tmap, second_block, bar);
          if (!T::kWhole)
            tma_bytes(par + T::kParams, c.pool + (size_t)second_block * (T::kCodes + T::kParams) + T::kCodes,
                      T::kParams, bar);
        }
      }
      copies.fetched();
    };
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < T::kStages; ++i) fetch(2 * i);

    // q: this lane's columns are head g / 2 of each tile of four, digits 3 - g % 2 and 1 - g % 2
    uint32_t qf[NT][T::kKSteps][2][2];
    float qs[NT], qsum[NT];  // of the heads whose sums this lane holds (t of each tile)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // of every 32 dimensions a lane's K codes are (I8) 4t .. 4t + 3 and 16 more, (I4) 8t .. 8t + 7
      float x[HD / 4];
      const int h = nt * 4 + (g >> 1);
      const size_t src = (size_t)r * a.ldq + (size_t)(h0 + min(h, heads - 1)) * HD + t * (I4 ? 8 : 4);
#pragma unroll
      for (int i = 0; i < HD / 4; i += 4) {
        const size_t at_q = src + i / 8 * 32 + i % 8 * (I4 ? 1 : 4);
        if (wide_q) {
          const float4 v = *(const float4*)((const float*)a.q + at_q);
          x[i] = v.x;
          x[i + 1] = v.y;
          x[i + 2] = v.z;
          x[i + 3] = v.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i + j] = load_elem(a.q, at_q + j, a.bf16);
        }
      }
      float top = 0.0f, sum = 0.0f, zero = 0.0f;
#pragma unroll
      for (int i = 0; i < HD / 4; ++i) {
        top = fmaxf(top, fabsf(x[i]));
        if constexpr (I4) sum = __fadd_rn(sum, x[i]);
        zero = __fmaf_rn(x[i], 0.0f, zero);  // NaN when an element is not finite
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if constexpr (I4) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
        zero = __fadd_rn(zero, __shfl_xor_sync(0xffffffffu, zero, o));
      }
      // 2^29 / 2^floor(log2 top), the exponents kept within what a float and its inverse can hold
      const int e = min(max((int)(__float_as_uint(top) >> 23), 36), 254);
      const float up = __uint_as_float((uint32_t)(283 - e) << 23), down = __uint_as_float((uint32_t)(e - 29) << 23);
      const int d3 = 3 - (g & 1), d1 = 1 - (g & 1);
#pragma unroll
      for (int s = 0; s < T::kKSteps; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          // the lane's elements of this half step, in the order in which the codes lie in a word
          const int d = I4 ? 8 * s + k : 8 * s + 4 * k, skip = I4 ? 2 : 1;
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = digits(__float2int_rn(__fmul_rn(x[d + j * skip], up)));
          qf[nt][s][0][k] = gather_byte(w[0], w[1], w[2], w[3], d3);
          qf[nt][s][1][k] = gather_byte(w[0], w[1], w[2], w[3], d1);
        }
      // a q that is not finite makes its head NaN
      const float f = __fadd_rn(__fmul_rn(I4 ? qscale / 16 : qscale, down), zero);
      qs[nt] = __shfl_sync(0xffffffffu, f, 8 * t);
      qsum[nt] = I4 ? __shfl_sync(0xffffffffu, __fmul_rn(sum, __fmul_rn(up, 16.0f)), 8 * t) : 0.0f;
    }

    // Scores stay in the units of the integer products times their scales;
    // qs (> 0) takes them to log2.  m is a maximum of theirs that lies at most
    // kSlack / qs below the true one, mq = m * qs.
    float m[NT], mq[NT], limit[NT], l[NT], zsum[NT], o[NT][T::kMTiles][4], sum[NT][T::kMTiles][2];
    float vf[NT], most[NT];  // the weights' power of two, and the largest weight (relative to m) times scale of V
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      vf[nt] = __uint_as_float(247u << 23);
      most[nt] = 0.0f;
      m[nt] = mq[nt] = limit[nt] = -INFINITY;
      l[nt] = zsum[nt] = 0.0f;
#pragma unroll
      for (int i = 0; i < T::kMTiles; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[nt][i][j] = sum[nt][i][j / 2] = 0.0f;
    }

    for (int i = 0; i < n_pages; i += 2) {
      // agreed on by the warp: what follows is done by all lanes together
      if (!__all_sync(0xffffffffu, mbar_wait(bar_s + copies.take * 8, copies.parity, &gave_up))) {
        give_up(&gave_up, a.status);
        failed = true;
        break;
      }
      if (i % kSumPages == 0 && i > 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < T::kMTiles; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              sum[nt][k][j] = __fadd_rn(sum[nt][k][j], __fadd_rn(o[nt][k][2 * j], o[nt][k][2 * j + 1]));
              o[nt][k][2 * j] = o[nt][k][2 * j + 1] = 0.0f;
            }
      }
      const uint32_t src = mine_s + copies.take * (2 * T::kTile);
      const uint8_t* par = params + copies.take * (2 * kParStride);
      // live positions from the first page on; with an odd number of pages the
      // second tile of the last pair holds what was there before
      const int left = min(len - (p0 + i) * kPage, (n_pages - i) * kPage);
      float raw[2][NT][2], vs[2][2], vz[2][2];  // [page][..][slot g or g + 8]
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        // scores
        int sc[NT][2][4];
        uint32_t kw[2 * T::kChunks];
        load_rows<T::kChunks, false>(src + pg * T::kTile, at_k, kw);
#pragma unroll
        for (int s = 0; s < T::kKSteps; ++s) {
          uint32_t x[2], y[2];  // rows g and g + 8
          if constexpr (I4) {
            // 16 (c - 8) as signed bytes
            x[0] = and_xor(kw[2 * s] << 4, 0xf0f0f0f0u, 0x80808080u);
            x[1] = and_xor(kw[2 * s], 0xf0f0f0f0u, 0x80808080u);
            y[0] = and_xor(kw[2 * s + 1] << 4, 0xf0f0f0f0u, 0x80808080u);
            y[1] = and_xor(kw[2 * s + 1], 0xf0f0f0f0u, 0x80808080u);
          } else {
            x[0] = kw[4 * s];
            y[0] = kw[4 * s + 1];
            x[1] = kw[4 * s + 2];
            y[1] = kw[4 * s + 3];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (s == 0)
                mma_s8<true>(sc[nt][j], x[0], y[0], x[1], y[1], qf[nt][s][j][0], qf[nt][s][j][1]);
              else
                mma_s8<false>(sc[nt][j], x[0], y[0], x[1], y[1], qf[nt][s][j][0], qf[nt][s][j][1]);
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          // parameter `kind` (K scale, [K zero,] V scale, [V zero]) of slot g + 8 k
          auto param = [&](int kind) {
            const int x = 64 * kind + 32 * k, line = (T::kCodes + x) / 128;
            const int turned = T::kWhole ? (line & 7) << 4 : 0;
            return *(const float*)(par + pg * kParStride + (x & ~127) + (((x & 127) ^ (turned & 96)) | ((4 * g) ^ (turned & 16))));
          };
          const float ks = param(0), kz = I4 ? __fmaf_rn(8.0f, ks, param(1)) : 0.0f;
          vs[pg][k] = param(I4 ? 2 : 1);
          vz[pg][k] = I4 ? __fmaf_rn(kNibbleMid, vs[pg][k], param(3)) : 0.0f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            // digits 3 and 2, 1 and 0: sums of at most 2^29
            const float x = __fmaf_rn((float)(sc[nt][0][2 * k] * 256 + sc[nt][0][2 * k + 1]), 65536.0f,
                                      (float)(sc[nt][1][2 * k] * 256 + sc[nt][1][2 * k + 1]));
            raw[pg][nt][k] = I4 ? __fmaf_rn(qsum[nt], kz, __fmul_rn(x, ks)) : __fmul_rn(x, ks);
          }
        }
      }
      if (left < 2 * kPage) {  // behind the context the bytes may be anything: no scale of theirs is used
#pragma unroll
        for (int pg = 0; pg < 2; ++pg)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (pg * kPage + 8 * k + g >= left) {
              vs[pg][k] = vz[pg][k] = 0.0f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) raw[pg][nt][k] = -INFINITY;
            }
      }
      const float vtop = fmaxf(fmaxf(vs[0][0], vs[0][1]), fmaxf(vs[1][0], vs[1][1]));
      bool again = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // a score above the slack, or a scale of V above what the weights' power of two allows
        again |= fmaxf(fmaxf(raw[0][nt][0], raw[0][nt][1]), fmaxf(raw[1][nt][0], raw[1][nt][1])) > limit[nt];
        again |= __fmul_rn(vtop, vf[nt]) > 512.0f;
      }
      if (__any_sync(0xffffffffu, again)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float top = fmaxf(fmaxf(raw[0][nt][0], raw[0][nt][1]), fmaxf(raw[1][nt][0], raw[1][nt][1]));
#pragma unroll
          for (int b = 4; b < 32; b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
          float keep = 1.0f;
          if (top > m[nt]) {
            m[nt] = top;
            const float nq = __fmul_rn(top, qs[nt]);
            keep = exp2_approx(__fsub_rn(mq[nt], nq));
            mq[nt] = nq;
            limit[nt] = __fadd_rn(top, __fdiv_rn(kSlack, qs[nt]));
          }
          float p = 0.0f;  // the largest product here (one that is not a number is passed over)
#pragma unroll
          for (int pg = 0; pg < 2; ++pg)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              p = fmaxf(p, __fmul_rn(exp2_approx(__fmaf_rn(raw[pg][nt][k], qs[nt], -mq[nt])), vs[pg][k]));
#pragma unroll
          for (int b = 4; b < 32; b <<= 1) p = fmaxf(p, __shfl_xor_sync(0xffffffffu, p, b));
          most[nt] = fmaxf(__fmul_rn(most[nt], keep), p);
          const float now = __fmul_rn(most[nt], vf[nt]);
          float f = 1.0f;
          if (most[nt] > 0.0f && !(now >= 0.25f && now <= 512.0f)) {
            const int e = min(max((int)(__float_as_uint(most[nt]) >> 23), 15), 252);
            const float nf = __uint_as_float((uint32_t)(256 - e) << 23);  // the product near 2^2
            f = __fdiv_rn(nf, vf[nt]);
            vf[nt] = nf;
          }
          l[nt] = __fmul_rn(l[nt], keep);
          zsum[nt] = __fmul_rn(zsum[nt], keep);
          keep = __fmul_rn(keep, f);
#pragma unroll
          for (int k = 0; k < T::kMTiles; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[nt][k][j] = __fmul_rn(o[nt][k][j], keep);
#pragma unroll
          for (int k = 0; k < T::kMTiles; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) sum[nt][k][j] = __fmul_rn(sum[nt][k][j], keep);
        }
      }
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        uint32_t wb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float w = exp2_approx(__fmaf_rn(raw[pg][nt][k], qs[nt], -mq[nt]));  // 0 behind the context
            l[nt] = __fadd_rn(l[nt], w);
            if constexpr (I4) zsum[nt] = __fmaf_rn(w, vz[pg][k], zsum[nt]);
            wb[nt][k] = transpose8x8(two_terms(__fmul_rn(__fmul_rn(w, vs[pg][k]), vf[nt])));
          }
        // output
        // a register of V holds two bytes each of two positions, so that a widened pair is one dimension at two
        // positions: of dimensions 2g, 2g + 1 of every 16 (I8), or 4g .. 4g + 3 of every 32 (I4)
        uint32_t vw[2 * T::kChunks];
        load_rows<T::kChunks, true>(src + pg * T::kTile, at_v, vw);
#pragma unroll
        for (int w = 0; w < T::kChunks; ++w) {
          if constexpr (I4) {
            uint32_t x[4], y[4];
            nibbles_f16(vw[2 * w], x);
            nibbles_f16(vw[2 * w + 1], y);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(o[nt][2 * w], x[0], x[1], y[0], y[1], wb[nt][0], wb[nt][1]);
              mma_f16(o[nt][2 * w + 1], x[2], x[3], y[2], y[3], wb[nt][0], wb[nt][1]);
            }
          } else {
            uint32_t x[2], y[2];
            bytes_f16(vw[2 * w], &x[0], &x[1]);
            bytes_f16(vw[2 * w + 1], &y[0], &y[1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][w], x[0], x[1], y[0], y[1], wb[nt][0], wb[nt][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      copies.used();
      fetch(i + 2 * T::kStages);
    }
    if (failed) {
      // copies still in flight land (or the wait for each runs out) before the CTA may go
      while (copies.flying) {
        mbar_wait(bar_s + copies.take * 8, copies.parity, nullptr);
        copies.used();
      }
      __syncwarp();
      break;
    }

    const bool begins = p0 == 0, ends = p1 == pages;
    const int slot = begins && !ends ? 1 : 0;
    if (!begins) {
      note.has0 = 1;
      note.ends0 = ends;
      note.far0 = at < end;  // the ring is needed again
    } else if (!ends) {
      note.row = r;
      note.unit = u;
    }
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 4 + t;
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) {
        l[nt] = __fadd_rn(l[nt], __shfl_xor_sync(0xffffffffu, l[nt], b));
        if constexpr (I4) zsum[nt] = __fadd_rn(zsum[nt], __shfl_xor_sync(0xffffffffu, zsum[nt], b));
      }
      if (h >= heads) continue;
      const float back = __fdiv_rn(I4 ? 1.0f / kNibbleUnit : 1.0f, vf[nt]);
      // the lane's dimensions: kRun from g * kRun of every 8 * kRun
      constexpr int kRun = I4 ? 4 : 2;
      float x[HD / 8];
#pragma unroll
      for (int k = 0; k < T::kMTiles; ++k) {
        x[2 * k] = __fmaf_rn(__fadd_rn(sum[nt][k][0], __fadd_rn(o[nt][k][0], o[nt][k][1])), back, zsum[nt]);
        x[2 * k + 1] = __fmaf_rn(__fadd_rn(sum[nt][k][1], __fadd_rn(o[nt][k][2], o[nt][k][3])), back, zsum[nt]);
      }
      if (begins && ends) {
        const float inv = __fdiv_rn(1.0f, l[nt]);
        const size_t dst = (size_t)r * a.ldo + (size_t)(h0 + h) * HD + g * kRun;
#pragma unroll
        for (int k = 0; k < HD / 8; ++k)
          store_elem(a.out, dst + k / kRun * (8 * kRun) + k % kRun, a.bf16, __fmul_rn(x[k], inv));
        if (a.lse && g == 0) a.lse[(size_t)r * a.nh + h0 + h] = lse_of(mq[nt], l[nt]);
      } else {
        float* part = !begins && at < end ? warp_slot(a.space, shares, share * kMmaWarps + warp, HD, us) : (float*)mine;
        part += h * T::kPartStride + g * kRun;
#pragma unroll
        for (int k = 0; k < HD / 8; k += kRun) {
          float* dst = part + k * 8;
          if constexpr (I4)
            *(float4*)dst = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
          else
            *(float2*)dst = make_float2(x[k], x[k + 1]);
        }
        if (g == 0) {
          ml[warp][slot][h][0] = mq[nt];
          ml[warp][slot][h][1] = l[nt];
        }
      }
    }
  }
  if (lane == 0) notes[warp] = note;
  __syncthreads();

  // Join what the CTA's warps left.  Chain w + 1 is the unit that begins in
  // warp w's share and ends later, chain 0 what came in from the share before;
  // its pieces are that warp's slot 1 and the slots 0 of the warps behind it.
  // A warp joins one head of one chain at a time, a lane first to a piece, then
  // to dimensions.  (The code runs once a CTA, so what it costs is its length:
  // instructions that no warp has met yet come from L2.)
  const WarpNote left = notes[min(lane, kMmaWarps - 1)];
  const unsigned begun = __ballot_sync(0xffffffffu, lane < kMmaWarps && left.row >= 0);
  const unsigned ended = __ballot_sync(0xffffffffu, lane < kMmaWarps && left.ends0);
  const unsigned far = __ballot_sync(0xffffffffu, lane < kMmaWarps && left.far0);
  const bool came_in = notes[0].has0;
  if (tid == 0) {
    const int last = 31 - __clz(begun);  // -1: none
    const bool open = begun && !(ended >> last >> 1);
    ((ShareMeta*)a.space)[share] =
        ShareMeta{open ? notes[last].row : -1, open ? notes[last].unit : 0, came_in && ended, 0};
  }
  for (int job = warp; job < (kMmaWarps + 1) * us.heads; job += kMmaWarps) {
    const int chain = job / us.heads, h = job - chain * us.heads;
    if (chain ? !(begun >> (chain - 1) & 1) : !came_in) continue;
    const unsigned ends_at = ended >> chain;
    const int to = ends_at ? chain + __ffs(ends_at) : kMmaWarps;  // slots 0 of the warps [chain, to)
    const int own = chain ? 1 : 0, pieces = own + to - chain;
    int kvh, h0 = 0, heads = us.heads;
    if (chain) unit_heads(us, a.nh, c.kv_heads, notes[chain - 1].unit, &kvh, &h0, &heads);
    if (h >= heads) continue;
    // lane i: piece i, which warp `of` left
    const int of = min(chain - own + lane, kMmaWarps - 1);
    const bool first = own && lane == 0, there = lane < pieces;
    const float mp = there ? ml[of][first][h][0] : -INFINITY, lp = there ? ml[of][first][h][1] : 0.0f;
    float M = mp;
#pragma unroll
    for (int b = 8; b; b >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, b));
    const float f = there ? exp2_approx(__fsub_rn(mp, M)) : 0.0f;
    float L = there ? __fmul_rn(lp, f) : 0.0f;
#pragma unroll
    for (int b = 8; b; b >>= 1) L = __fadd_rn(L, __shfl_xor_sync(0xffffffffu, L, b));
    M = __shfl_sync(0xffffffffu, M, 0);
    L = __shfl_sync(0xffffffffu, L, 0);
    constexpr int kRun = HD / 32;  // a lane's dimensions
    float sum[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k) sum[k] = 0.0f;
#pragma unroll 3
    for (int i = 0; i < pieces; ++i) {
      const int w = chain - own + i;
      const bool in_ring = (own && i == 0) || !(far >> w & 1);
      const float* part = in_ring ? (const float*)(ring + w * T::kRing)
                                  : warp_slot(a.space, shares, share * kMmaWarps + w, HD, us);
      part += h * T::kPartStride + lane * kRun;
      const float fi = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
      for (int k = 0; k < kRun; ++k) sum[k] = __fmaf_rn(part[k], fi, sum[k]);
    }
    if (own && ends_at) {
      const float inv = __fdiv_rn(1.0f, L);
      const size_t row = notes[chain - 1].row;
#pragma unroll
      for (int k = 0; k < kRun; ++k)
        store_elem(a.out, row * a.ldo + (size_t)(h0 + h) * HD + lane * kRun + k, a.bf16, __fmul_rn(sum[k], inv));
      if (a.lse && lane == 0) a.lse[row * a.nh + h0 + h] = lse_of(M, L);
    } else {
      float* dst = share_slot(a.space, shares, share, own, HD, us) + h * (HD + 4);
#pragma unroll
      for (int k = 0; k < kRun; ++k) dst[lane * kRun + k] = sum[k];
      if (lane == 0) {
        dst[HD] = M;
        dst[HD + 1] = L;
      }
    }
  }
}

// Joins the partial results of the unit that begins in this CTA's share and ends
// in a later one.  The CTA's warps are dealt to the unit's heads, several to a
// head, which take its pieces in turn and meet once in shared memory.  What
// the join costs is its three trips to L2, one after the other: the notes of
// the shares, the pieces' maxima, the pieces.
constexpr int kJoinWarps = 16;
__global__ void __launch_bounds__(kJoinWarps * 32) kvq_join_kernel(KvqView c, KvqAttend a, int shares) {
  __shared__ float sums[kJoinWarps][kKvqMaxHd];
  __shared__ float maxima[kJoinWarps], totals[kJoinWarps];
  pdl_wait();
  const ShareMeta* meta = (const ShareMeta*)after_wait((uint8_t*)a.space);
  const int share = blockIdx.x, hd = c.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const ShareMeta own = meta[share];
  int at = share + 1;
  unsigned ends = __ballot_sync(0xffffffffu, at + lane < shares && meta[min(at + lane, shares - 1)].ends);
  if (own.row < 0) return;
  while (!ends && at + 32 < shares) {
    at += 32;
    ends = __ballot_sync(0xffffffffu, at + lane < shares && meta[min(at + lane, shares - 1)].ends);
  }
  // pieces: slot 1 of this share, slot 0 of the later ones
  const int n = (ends ? at + __ffs(ends) - 1 : shares - 1) - share + 1;
  const Units us = units_of(a.nh, c.kv_heads);
  int kvh, h0, heads;
  unit_heads(us, a.nh, c.kv_heads, own.unit, &kvh, &h0, &heads);
  const int team = kJoinWarps / heads, h = warp / team, mine = warp % team;  // warps a head
  const bool on = h < heads;
  auto piece = [&](int i) { return share_slot(a.space, shares, share + i, i == 0, hd, us) + min(h, heads - 1) * (hd + 4); };
  // a lane's dimensions: four from 4 * lane, and four 128 further on
  float M = -INFINITY, L = 0.0f, o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.0f;
  const bool fours = hd % 4 == 0;
  // this warp's pieces: mine, mine + team, ... up to 32 of them at a time
  for (int i0 = mine; i0 < n && on; i0 += 32 * team) {
    const int i = i0 + lane * team;
    const float m = i < n ? piece(i)[hd] : -INFINITY, l = i < n ? piece(i)[hd + 1] : 0.0f;
    float top = m;
#pragma unroll
    for (int b = 16; b; b >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
    const float mn = fmaxf(M, top), keep = M == mn ? 1.0f : exp2_approx(__fsub_rn(M, mn));
    const float f = l == 0.0f ? 0.0f : exp2_approx(__fsub_rn(m, mn));
    M = mn;
    L = __fmaf_rn(L, keep, __fmul_rn(l, f));  // a lane's part
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = __fmul_rn(o[k], keep);
    const int here = min(32, (n - i0 + team - 1) / team);
#pragma unroll 8
    for (int j = 0; j < here; ++j) {
      const float* p = piece(i0 + j * team);
      const float fj = __shfl_sync(0xffffffffu, f, j);
      if (fours) {
        if (4 * lane < hd) {
          const float4 v = *(const float4*)(p + 4 * lane);
          o[0] = __fmaf_rn(v.x, fj, o[0]);
          o[1] = __fmaf_rn(v.y, fj, o[1]);
          o[2] = __fmaf_rn(v.z, fj, o[2]);
          o[3] = __fmaf_rn(v.w, fj, o[3]);
        }
        if (4 * lane + 128 < hd) {
          const float4 v = *(const float4*)(p + 4 * lane + 128);
          o[4] = __fmaf_rn(v.x, fj, o[4]);
          o[5] = __fmaf_rn(v.y, fj, o[5]);
          o[6] = __fmaf_rn(v.z, fj, o[6]);
          o[7] = __fmaf_rn(v.w, fj, o[7]);
        }
      } else {
        for (int k = 0; k < 8; ++k) {
          const int d = 4 * lane + k % 4 + k / 4 * 128;
          if (d < hd) o[k] = __fmaf_rn(p[d], fj, o[k]);
        }
      }
    }
  }
#pragma unroll
  for (int b = 16; b; b >>= 1) L = __fadd_rn(L, __shfl_xor_sync(0xffffffffu, L, b));
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int d = 4 * lane + k % 4 + k / 4 * 128;
    if (d < hd) sums[warp][d] = o[k];
  }
  if (lane == 0) {
    maxima[warp] = M;
    totals[warp] = L;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < heads * hd; d += kJoinWarps * 32) {
    const int head = d / hd, first = head * team;
    float top = -INFINITY, sum = 0.0f, total = 0.0f;
    for (int w = first; w < first + min(team, n); ++w) top = fmaxf(top, maxima[w]);
    for (int w = first; w < first + min(team, n); ++w) {
      const float f = totals[w] == 0.0f ? 0.0f : exp2_approx(__fsub_rn(maxima[w], top));
      sum = __fmaf_rn(sums[w][d - head * hd], f, sum);
      total = __fmaf_rn(totals[w], f, total);
    }
    store_elem(a.out, (size_t)own.row * a.ldo + (size_t)h0 * hd + d, a.bf16, __fdiv_rn(sum, total));
    if (a.lse && d == head * hd) a.lse[(size_t)own.row * a.nh + h0 + head] = lse_of(top, total);
  }
}

}  // namespace

size_t kvq_attend_space(int nh, int kv_heads, int hd) {
  const Units us = units_of(nh, kv_heads);
  const size_t plain = (size_t)kAttendCtas * (sizeof(ShareMeta) + 2 * us.heads * (hd + 4) * sizeof(float));
  const size_t mma = (size_t)kMmaShares * (sizeof(ShareMeta) + 2 * us.heads * (hd + 4) * sizeof(float) +
                                           kMmaMaxWarps * us.heads * (hd + 4) * sizeof(float)) + 16;
  return std::max(plain, mma);
}

namespace {
// Units of at most this many positions, and no more of them than CTAs, are taken
// by a CTA each: its warps' pages take less time than a second kernel, which
// joins what several CTAs leave.  Measured (whole, cut; us): heads of 128, I8, 5
// units of 1024 positions 16 and 18, of 2048 23 and 20; 40 units 14 and 23, 25 and
// 25; 165 units 23 and 29, 33 and 39.  So whole units are the faster way up to 1024
// positions always, and beyond where there are many of them, which this rule
// leaves to the cut.
constexpr int kWholeUnits = 1024;
constexpr int kMinWeight = kUnitCost + 1;  // the least share of a warp

// The codes of every block as a tensor of 128-byte lines: [blocks][lines][128].
template <class T>
bool codes_map(const KvqView& c, CUtensorMap* map) {
  const cuuint64_t dims[3] = {128, T::kLines, (cuuint64_t)c.pages * c.kv_heads};
  const cuuint64_t strides[2] = {128, T::kCodes + T::kParams};
  const cuuint32_t box[3] = {128, T::kLines, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, c.pool, dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool I4, int NT>
bool launch_mma(const KvqView& c, const KvqRows& r, const KvqAttend& a, int max_len, int wide_q, cudaStream_t st) {
  using T = MmaTile<HD, I4, NT>;
  static_assert(T::kRing >= NT * 4 * T::kPartStride * 4, "a warp's ring holds its partial result");
  CUtensorMap map;
  if (!codes_map<T>(c, &map)) return false;
  auto* kernel = kvq_attend_mma_kernel<HD, I4, NT>;
  static std::atomic<uint64_t> allowed{0};
  allow_shared((const void*)kernel, T::kSmem, allowed);
  int shares = NT == 1 ? kMmaShares : kMmaShares / 2;
  const size_t units = (size_t)r.rows * units_of(a.nh, c.kv_heads).per_row;
  const bool whole = max_len <= kWholeUnits && units <= (size_t)shares;
  if (whole) shares = (int)units;
  kernel<<<shares, T::kWarps * 32, T::kSmem, st>>>(c, r, a, max_len, kMinWeight, wide_q, whole, map);
  count_launch();
  if (whole) return true;
  launch_pdl(kvq_join_kernel, dim3(shares), dim3(kJoinWarps * 32), 0, st, c, a, shares);
  count_launch();
  return true;
}
using LaunchMma = bool (*)(const KvqView&, const KvqRows&, const KvqAttend&, int, int, cudaStream_t);
// The tensor-core kernel for a cache and number of heads a unit, or null.
template <int HD>
LaunchMma mma_of(bool i4, bool two) {
  return i4 ? (two ? launch_mma<HD, true, 2> : launch_mma<HD, true, 1>)
            : (two ? launch_mma<HD, false, 2> : launch_mma<HD, false, 1>);
}
LaunchMma mma_for(const KvqView& c, int heads) {
  if ((size_t)c.pages * c.kv_heads >= (1ull << 31) || !tensor_map_encoder()) return nullptr;
  switch (c.hd) {
    case 32:
      return mma_of<32>(c.i4, heads > 4);
    case 64:
      return mma_of<64>(c.i4, heads > 4);
    case 96:
      return mma_of<96>(c.i4, heads > 4);
    case 128:
      return mma_of<128>(c.i4, heads > 4);
  }
  return nullptr;
}
}  // namespace

const char* kvq_attend_kernel_name(const KvqView& c, const KvqRows& r, int nh, bool bf16) {
  if (kvq_prompt_pays(c, r, nh, bf16)) return "kvq_prompt_kernel";
  return mma_for(c, units_of(nh, c.kv_heads).heads) ? "kvq_attend_mma_kernel" : "kvq_attend_plain_kernel";
}

void launch_kvq_attend(const KvqView& c, const KvqRows& r, const KvqAttend& a, int max_len, cudaStream_t st) {
  if (r.rows <= 0) return;
  const Units us = units_of(a.nh, c.kv_heads);
  if (kvq_prompt_pays(c, r, a.nh, a.bf16)) {
    launch_kvq_prompt(c, r, a, max_len, st);
    return;
  }
  if (LaunchMma launch = mma_for(c, us.heads)) {
    const int wide_q = !a.bf16 && (uintptr_t)a.q % 16 == 0 && a.ldq % 4 == 0;
    if (launch(c, r, a, max_len, wide_q, st)) return;
  }
  const size_t smem = ((size_t)us.heads * c.hd + kPlainWarps * us.heads * (c.hd + 2)) * sizeof(float);
  kvq_attend_plain_kernel<<<kAttendCtas, kPlainWarps * 32, smem, st>>>(c, r, a, max_len);
  kvq_join_kernel<<<kAttendCtas, kJoinWarps * 32, 0, st>>>(c, a, kAttendCtas);
  count_launch(2);
}

}  // namespace bitnet
