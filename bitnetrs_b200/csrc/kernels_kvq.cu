// kernels_kvq.cu — the quantised paged key-value cache: rows quantised into
// their slots, rows read back, and GQA attention split over the context.
#include "kvq.cuh"

#include <algorithm>

namespace bitnet {

KvqView kvq_layer(const KvGeom& g, const int32_t* table, int seqs, int layer) {
  KvqView c;
  c.i4 = g.quant == BITNET_KV_I4;
  c.pool = (uint8_t*)g.pool + (size_t)layer * g.pages * g.kv_heads * kvq_block_bytes(g.hd, c.i4);
  c.table = table;
  c.pages = g.pages;
  c.seqs = seqs;
  c.per_seq = g.max_pages_per_seq;
  c.kv_heads = g.kv_heads;
  c.hd = g.hd;
  return c;
}

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
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// ---------------------------------------------------------------------------
// Store.  One warp quantises one row of one head: the largest magnitude (I8)
// or the extremes (I4) by a warp reduction, then the code nearest to each
// element.  The nearest code is exact, ties to even, whatever the scale: the
// product with the scale's reciprocal may land on the wrong side of a border,
// so the remainder of that code (one fma, exact at a border) puts it right.
// Elements are held in 64 bits, in which a rotated element is rounded once.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int nearest_code(double x, double scale, double inv, int least, int most) {
  double c = rint(x * inv);
  const double r = fma(-c, scale, x), h = 0.5 * scale;
  const bool odd = ((int)c & 1) != 0;
  if (r > h || (r == h && odd))
    c += 1.0;
  else if (r < -h || (r == -h && odd))
    c -= 1.0;
  return min(max((int)c, least), most);
}

constexpr int kStoreWarps = 8;
constexpr int kStorePairs = kKvqMaxHd / 64;  // pairs of dimensions a lane holds

__global__ void __launch_bounds__(kStoreWarps * 32) kvq_store_kernel(KvqView c, KvqStore s) {
  const int lane = threadIdx.x & 31;
  const int jobs = 2 * c.kv_heads + (s.q ? s.nh : 0);  // K heads, V heads, q heads of a row
  const size_t job = (size_t)blockIdx.x * kStoreWarps + (threadIdx.x >> 5);
  const int row = (int)(job / jobs), what = (int)(job % jobs);
  if (row >= s.rows) return;
  const int pos = s.row_pos ? s.row_pos[row] : row;
  if (pos < 0) return;
  const int seq = s.row_seq ? s.row_seq[row] : 0;
  const int kind = what < c.kv_heads ? 0 : 1;
  const int head = kind ? what - c.kv_heads : what;
  uint8_t* block = block_of(c, seq, pos, min(head, c.kv_heads - 1));
  if (!block || (s.rope_cos && pos >= s.rope_len)) {
    if (lane == 0) atomicOr(s.status, kStatusBadContext);
    return;
  }
  const int hd = c.hd, half = hd / 2;
  const float* cs = s.rope_cos ? s.rope_cos + (size_t)pos * half : nullptr;
  const float* sn = s.rope_cos ? s.rope_sin + (size_t)pos * half : nullptr;
  if (what >= 2 * c.kv_heads) {  // a q head, in the reference's f32 order (rope.rs:414-431)
    const int h = what - 2 * c.kv_heads;
    const float* x = s.q + (size_t)row * s.ldq + h * hd;
    float* o = s.q_out + ((size_t)row * s.nh + h) * hd;
    for (int p = lane; p < half; p += 32) {
      const float lo = x[p], hi = x[p + half];
      o[p] = __fsub_rn(__fmul_rn(lo, cs[p]), __fmul_rn(hi, sn[p]));
      o[p + half] = __fadd_rn(__fmul_rn(hi, cs[p]), __fmul_rn(lo, sn[p]));
    }
    return;
  }
  const void* src = kind ? s.v : s.k;
  const size_t at = (size_t)row * (kind ? s.ldv : s.ldk) + (size_t)head * hd;
  const bool turn = kind == 0 && cs;
  double x[kStorePairs][2];
  double top = 0.0, low = INFINITY;  // the largest x (I4) or |x| (I8), the least x
  if (c.i4) top = -INFINITY;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < kStorePairs; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int d = 2 * (lane + 32 * i) + j;
      x[i][j] = 0.0;
      if (d >= hd) continue;
      double v = load_elem(src, at + d, s.bf16);
      if (turn) {
        const int p = d < half ? d : d - half;
        const double w = load_elem(src, at + (d < half ? d + half : p), s.bf16);
        // each product is exact in 64 bits, the sum is rounded once
        v = d < half ? __dsub_rn(__dmul_rn(v, cs[p]), __dmul_rn(w, sn[p]))
                     : __dadd_rn(__dmul_rn(v, cs[p]), __dmul_rn(w, sn[p]));
      }
      finite &= isfinite(v) != 0;
      x[i][j] = v;
      top = fmax(top, c.i4 ? v : fabs(v));
      low = fmin(low, v);
    }
  finite = __all_sync(0xffffffffu, finite);
  top = warp_max(top);
  float zero = 0.0f, scale;
  if (c.i4) {
    low = -warp_max(-low);
    zero = __fadd_rn((float)low, 0.0f);  // never -0
    scale = __fadd_rn((float)((top - (double)zero) / 15.0), 0.0f);
  } else {
    scale = (float)(top / 127.0);
  }
  // a row that holds a value that is not finite reads back as NaN
  if (!finite || !isfinite(scale) || !isfinite(zero)) {
    scale = __int_as_float(0x7fc00000);
    if (lane == 0) atomicOr(s.status, kStatusNonFinite);
    finite = false;
  }
  const int slot = pos % kPage, rowb = kvq_row_bytes(hd, c.i4);
  uint8_t* codes = block + (size_t)(kind * kPage + slot) * rowb;
  const double inv = 1.0 / (double)scale;
#pragma unroll
  for (int i = 0; i < kStorePairs; ++i) {
    const int d = 2 * (lane + 32 * i);
    if (d >= hd) continue;
    int q[2] = {0, 0};
    if (finite && scale > 0.0f)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        q[j] = nearest_code(x[i][j] - (double)zero, scale, inv, c.i4 ? 0 : -127, c.i4 ? 15 : 127);
    if (c.i4)
      codes[d / 2] = (uint8_t)(q[0] | (q[1] << 4));
    else
      *(uint16_t*)(codes + d) = (uint16_t)((q[0] & 255) | (q[1] << 8));
  }
  if (lane == 0) {
    float* par = block_params(block, hd, c.i4, kind);
    par[slot] = scale;
    if (c.i4) par[kPage + slot] = zero;
  }
}

// ---------------------------------------------------------------------------
// Load.  One warp reads one row of one head.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float code_at(const uint8_t* codes, int d, int i4) {
  return i4 ? (float)((codes[d >> 1] >> ((d & 1) * 4)) & 15) : (float)(int8_t)codes[d];
}
__global__ void __launch_bounds__(kStoreWarps * 32)
    kvq_load_kernel(KvqView c, int rows, const int32_t* __restrict__ row_seq, const int32_t* __restrict__ row_pos,
                    void* __restrict__ k, size_t ldk, void* __restrict__ v, size_t ldv, int bf16, int32_t* status) {
  const int lane = threadIdx.x & 31;
  const size_t job = (size_t)blockIdx.x * kStoreWarps + (threadIdx.x >> 5);
  const int row = (int)(job / (2 * c.kv_heads)), what = (int)(job % (2 * c.kv_heads));
  if (row >= rows) return;
  const int pos = row_pos ? row_pos[row] : row;
  if (pos < 0) return;
  const int kind = what / c.kv_heads, head = what % c.kv_heads;
  uint8_t* block = block_of(c, row_seq ? row_seq[row] : 0, pos, head);
  if (!block) {
    if (lane == 0) atomicOr(status, kStatusBadContext);
    return;
  }
  const int slot = pos % kPage;
  const uint8_t* codes = block + (size_t)(kind * kPage + slot) * kvq_row_bytes(c.hd, c.i4);
  const float* par = block_params(block, c.hd, c.i4, kind);
  const float scale = par[slot], zero = c.i4 ? par[kPage + slot] : 0.0f;
  void* dst = kind ? v : k;
  const size_t at = (size_t)row * (kind ? ldv : ldk) + (size_t)head * c.hd;
  for (int d = lane; d < c.hd; d += 32)
    store_elem(dst, at + d, bf16, __fmaf_rn(code_at(codes, d, c.i4), scale, zero));
}

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
constexpr int kMaxHeads = 8;
constexpr int kAttendCtas = 148 * 4;
struct ShareMeta {
  int row, unit;  // the unit that begins in this share and ends in a later one (row < 0: none)
  int ends;       // whether the unit of slot 0 ends in this share
  int pad;
};

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

// What row r sees: its sequence and how many positions (-1: the row belongs to no run).
__device__ __forceinline__ int row_context(const KvqView& c, const KvqRows& R, int r, int max_len, int* seq,
                                           int32_t* status) {
  int len;
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
    len = R.starts[lo] + (r - R.cu[lo]) + 1;
  } else {
    *seq = R.row_seq[r];
    len = R.row_len[r] + R.len_bias;
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
  return len;
}

__device__ __forceinline__ float* share_slot(void* space, int shares, int share, int slot, int hd, const Units& us) {
  return (float*)((ShareMeta*)space + shares) + ((size_t)share * 2 + slot) * (us.heads * (hd + 2));
}

__device__ void write_empty_row(const KvqAttend& a, int hd, int r) {
  for (int i = threadIdx.x; i < a.nh * hd; i += blockDim.x) store_elem(a.out, (size_t)r * a.ldo + i, a.bf16, 0.0f);
  if (a.lse)
    for (int i = threadIdx.x; i < a.nh; i += blockDim.x) a.lse[(size_t)r * a.nh + i] = -INFINITY;
}

// One head's joined result (m in units of log2): output and log-sum-exp.
__device__ __forceinline__ float lse_of(float m, float l) {
  return l > 0.0f || isnan(l) ? __fmul_rn(__fadd_rn(m, log2f(l)), 0.69314718055994530942f) : -INFINITY;
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
  while (at < end) {
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
        slot[h * (hd + 2) + d] = o;
        if (d == 0) {
          slot[h * (hd + 2) + hd] = M;
          slot[h * (hd + 2) + hd + 1] = L;
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

// Joins the partial results of the unit that begins in this CTA's share and ends in a later one.
__global__ void __launch_bounds__(256) kvq_join_kernel(KvqView c, KvqAttend a, int shares) {
  const ShareMeta* meta = (const ShareMeta*)a.space;
  const int share = blockIdx.x, hd = c.hd;
  const ShareMeta own = meta[share];
  if (own.row < 0) return;
  const Units us = units_of(a.nh, c.kv_heads);
  int kvh, h0, heads;
  unit_heads(us, a.nh, c.kv_heads, own.unit, &kvh, &h0, &heads);
  int last = share + 1;
  while (last < shares - 1 && !meta[last].ends) ++last;
  for (int i = threadIdx.x; i < heads * hd; i += blockDim.x) {
    const int h = i / hd, d = i % hd;
    const float* p = share_slot(a.space, shares, share, 1, hd, us) + h * (hd + 2);
    float M = p[hd], L = p[hd + 1], o = p[d];
    for (int s = share + 1; s <= last; ++s) {
      p = share_slot(a.space, shares, s, 0, hd, us) + h * (hd + 2);
      const float m = p[hd], l = p[hd + 1];
      if (l == 0.0f) continue;
      const float mn = fmaxf(M, m), f = exp2f(__fsub_rn(M, mn)), g = exp2f(__fsub_rn(m, mn));
      L = __fmaf_rn(L, L == 0.0f ? 0.0f : f, __fmul_rn(l, g));
      o = __fmaf_rn(o, L == 0.0f ? 0.0f : f, __fmul_rn(p[d], g));
      M = mn;
    }
    store_elem(a.out, (size_t)own.row * a.ldo + (size_t)h0 * hd + i, a.bf16, __fdiv_rn(o, L));
    if (a.lse && d == 0) a.lse[(size_t)own.row * a.nh + h0 + h] = lse_of(M, L);
  }
}

}  // namespace

void launch_kvq_store(const KvqView& c, const KvqStore& s, cudaStream_t st) {
  if (s.rows <= 0) return;
  const size_t jobs = (size_t)s.rows * (2 * c.kv_heads + (s.q ? s.nh : 0));
  kvq_store_kernel<<<(unsigned)ceil_div(jobs, kStoreWarps), kStoreWarps * 32, 0, st>>>(c, s);
  count_launch();
}

void launch_kvq_load(const KvqView& c, int rows, const int32_t* row_seq, const int32_t* row_pos, void* k, size_t ldk,
                     void* v, size_t ldv, int bf16, int32_t* status, cudaStream_t st) {
  if (rows <= 0) return;
  const size_t jobs = (size_t)rows * 2 * c.kv_heads;
  kvq_load_kernel<<<(unsigned)ceil_div(jobs, kStoreWarps), kStoreWarps * 32, 0, st>>>(c, rows, row_seq, row_pos, k,
                                                                                      ldk, v, ldv, bf16, status);
  count_launch();
}

size_t kvq_attend_space(int nh, int kv_heads, int hd) {
  const Units us = units_of(nh, kv_heads);
  return (size_t)kAttendCtas * (sizeof(ShareMeta) + 2 * us.heads * (hd + 2) * sizeof(float));
}

const char* kvq_attend_kernel_name(const KvqView& c, int nh) {
  (void)c;
  (void)nh;
  return "kvq_attend_plain_kernel";
}

void launch_kvq_attend(const KvqView& c, const KvqRows& r, const KvqAttend& a, int max_len, cudaStream_t st) {
  if (r.rows <= 0) return;
  const Units us = units_of(a.nh, c.kv_heads);
  const size_t smem = ((size_t)us.heads * c.hd + kPlainWarps * us.heads * (c.hd + 2)) * sizeof(float);
  kvq_attend_plain_kernel<<<kAttendCtas, kPlainWarps * 32, smem, st>>>(c, r, a, max_len);
  kvq_join_kernel<<<kAttendCtas, 256, 0, st>>>(c, a, kAttendCtas);
  count_launch(2);
}

}  // namespace bitnet
