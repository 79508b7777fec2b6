// kernels_kvq.cu — the quantised paged key-value cache: rows quantised into
// their slots, and rows read back.
#include "kvq_device.cuh"

#include <algorithm>
#include <climits>

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

// ---------------------------------------------------------------------------
// Store.  A group of GROUP lanes (a power of two) quantises one row of one
// head, N neighbouring elements a lane: the largest magnitude (I8) or the
// extremes (I4) by a reduction over the group, then the code nearest to each
// element.
//
// The nearest code is exact, ties to even, whatever the scale.  In 32 bits
// t = x / scale is off by less than 127 * 3 * 2^-24 < 2^-15, so rint(t) is the
// code unless t lies that close to a border; there the quotient is taken in 64
// bits, and the remainder of the code it gives (one fma, exact at a border)
// decides.  Away from borders t is at least the least code and at most the
// largest, and a rounding, but for I4 rows of rotated K: an element is held in
// 64 bits there (its two products are exact and their sum is rounded once) and the
// row's zero in 32, so an element may lie below the zero by half of the zero's
// last place, which is many codes where a row is nearly constant.  A t outside
// the codes is sent to the same second look, which ends at the least or the
// largest code.
//
// Bound, for many rows, by the loads that a warp waits for and its instructions
// (some 500 for 16 elements a lane), for few by three dependent loads (position,
// page, and the row beside them).  Measured: 6605 rows of 8 kv heads of 128, bf16
// to I4, 20 us (1.7 TB/s); one row of 5 heads, rotated, 2.7 us with its launch.
// Neither more warps an SM (fewer registers), nor CTAs that stay and take row
// after row, nor reductions that do not wait for the row's page were faster.
// ---------------------------------------------------------------------------
__device__ __noinline__ int border_code(double x, double scale, int least, int most) {
  double c = rint(x / scale);
  const double r = fma(-c, scale, x), h = 0.5 * scale;
  const bool odd = ((int)c & 1) != 0;
  if (r > h || (r == h && odd))
    c += 1.0;
  else if (r < -h || (r == -h && odd))
    c -= 1.0;
  return min(max((int)c, least), most);
}
// x / scale as the sum with 1.5 * 2^23, whose rounding is that to the nearest
// integer, ties to even: the code is in its low bits.  *off is raised to the
// quotient's distance from it, or becomes NaN (a scale so small that its
// reciprocal is not finite): unless it stays below 0.4999 the codes are looked
// at again.
constexpr uint32_t kCodeBits = 0x4b400000u;
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// With BELOW it is raised, too, to how far the quotient lies outside [0, 15].
template <bool BELOW>
__device__ __forceinline__ uint32_t code_bits(float x, float inv, float* off) {
  const float t = __fmul_rn(x, inv), f = __fadd_rn(t, __uint_as_float(kCodeBits));
  *off = max_nan(*off, fabsf(__fsub_rn(t, __fsub_rn(f, __uint_as_float(kCodeBits)))));
  if (BELOW) *off = max_nan(*off, __fsub_rn(fabsf(__fsub_rn(t, 7.5f)), 7.5f));
  return __float_as_uint(f);
}

// x / 15 rounded to 32 bits.  The product with 1 / 15 is within 2^-51 of it, so
// the division is made only where that could matter.
__device__ __noinline__ float fifteenth_slow(double x) { return (float)(x / 15.0); }
__device__ __forceinline__ float fifteenth(double x) {
  const double y = x * (1.0 / 15.0), e = y * 0x1p-50;
  const float low = (float)(y - e), high = (float)(y + e);
  return low == high ? low : fifteenth_slow(x);
}

// N elements from x[i] on, in wide loads where `wide` says that they are aligned.
template <int N>
__device__ __forceinline__ void load_run(const void* x, size_t i, int bf16, bool wide, float* v) {
  if (N >= 8 && wide) {
    if (bf16) {
#pragma unroll
      for (int j = 0; j < N; j += 8) {
        const uint4 w = *(const uint4*)((const uint16_t*)x + i + j);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[(j + 2 * k) % N] = bf_lo(u[k]);
          v[(j + 2 * k + 1) % N] = bf_hi(u[k]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const float4 p = *(const float4*)((const float*)x + i + j);
        v[j] = p.x;
        v[(j + 1) % N] = p.y;
        v[(j + 2) % N] = p.z;
        v[(j + 3) % N] = p.w;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = load_elem(x, i + j, bf16);
  }
}

constexpr int kStoreWarps = 4;
constexpr int kLoadTeams = 148 * 320;  // warps, at most: eight times what the SMs hold

// Elements a lane, and lanes a row of one head.  A rotation pairs whole runs, so
// half a row is a multiple of a run of 8 or 16.  With many rows 16 elements a
// lane keep twice the bytes on the way (6605 rows of 8 kv heads, bf16 to I4: 25 us
// with 8, 20 us with 16); with few there are more lanes to share the work.
struct RowSplit {
  int group, run;
};
inline RowSplit split_row(int hd, bool many) {
  RowSplit s;
  s.run = many && hd % 32 == 0 ? 16 : hd % 16 == 0 ? 8 : 2;
  s.group = 1;
  while (s.group * s.run < hd && s.group < 32) s.group *= 2;
  return s;
}

// N elements a lane (8 or 16: once over the row; 2: as often as the row needs it).
template <int N, bool I4, bool ROPE>
__global__ void __launch_bounds__(kStoreWarps * 32) kvq_store_kernel(KvqView c, KvqStore s, int group, int wide) {
  constexpr int kRuns = N >= 8 ? 1 : kKvqMaxHd / 64;
  const int lane = threadIdx.x & 31, in = lane & (group - 1);
  const int jobs = 2 * c.kv_heads + (s.q ? s.nh : 0);  // K heads, V heads, q heads of a row
  const int hd = c.hd, half = hd / 2;
  const int lg = 31 - __clz(group);  // group is a power of two
  const uint32_t job = blockIdx.x * (uint32_t)(kStoreWarps * 32 >> lg) + (threadIdx.x >> lg);  // rows * jobs is below 2^31
  const uint32_t row32 = job / (uint32_t)jobs;
  const size_t row = row32;
  const int what = (int)(job - row32 * (uint32_t)jobs);
  // lanes without a row run on with the group's reductions
  const bool there = row < (size_t)s.rows;
  const int pos = there ? (s.row_pos ? s.row_pos[row] : (int)row) : -1, seq = there && s.row_seq ? s.row_seq[row] : 0;
  bool on = pos >= 0;
  if (on && ROPE && pos >= s.rope_len) {
    if (in == 0) atomicOr(s.status, kStatusBadContext);
    on = false;
  }
  const int kind = what < c.kv_heads ? 0 : 1, head = kind ? what - c.kv_heads : what;
  const bool is_q = what >= 2 * c.kv_heads;
  const void* src = is_q ? (const void*)s.q : kind ? s.v : s.k;
  const size_t at = row * (is_q ? s.ldq : kind ? s.ldv : s.ldk) + (size_t)(is_q ? what - 2 * c.kv_heads : head) * hd;
  const int bf16 = is_q ? 0 : s.bf16;
  float x[kRuns][N];
  float w[ROPE ? kRuns : 1][N], cs[ROPE ? kRuns : 1][N], sn[ROPE ? kRuns : 1][N];  // a rotation's other element, cos and sin
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    const int d = N * (in + 32 * i);
#pragma unroll
    for (int j = 0; j < N; ++j) x[i][j] = 0.0f;
    if (!there || d >= hd) continue;
    load_run<N>(src, at + d, bf16, wide, x[i]);  // before its place is known
    if (ROPE && on && (kind == 0 || is_q)) {
      const size_t angle = (size_t)pos * half;
      if (N >= 8) {
        const int p = d < half ? d : d - half;
        load_run<N>(src, at + (d < half ? d + half : p), bf16, wide, w[i]);
        load_run<N>(s.rope_cos, angle + p, 0, wide, cs[i]);
        load_run<N>(s.rope_sin, angle + p, 0, wide, sn[i]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int p = d + j < half ? d + j : d + j - half;
          w[i][j] = load_elem(src, at + (d + j < half ? d + j + half : p), bf16);
          cs[i][j] = s.rope_cos[angle + p];
          sn[i][j] = s.rope_sin[angle + p];
        }
      }
    }
  }
  uint8_t* block = on ? block_of(c, seq, pos, is_q ? 0 : head) : nullptr;
  if (on && !block) {
    if (in == 0) atomicOr(s.status, kStatusBadContext);
    on = false;
  }
  if (is_q) {  // in the reference's f32 order (rope.rs:414-431); a whole group, and no reduction below has others in it
    float* o = s.q_out + (row * s.nh + (what - 2 * c.kv_heads)) * hd;
    if (on)
#pragma unroll
      for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int d = N * (in + 32 * i) + j;
          if (!ROPE || d >= hd) continue;
          const float a = __fmul_rn(x[i][j], cs[i][j]), b = __fmul_rn(w[i][j], sn[i][j]);
          o[d] = d < half ? __fsub_rn(a, b) : __fadd_rn(a, b);
        }
    on = false;
  }
  double v[ROPE ? kRuns : 1][N];  // elements in 64 bits, where 32 do not hold them
  float top = I4 ? -INFINITY : 0.0f, low = INFINITY;  // the largest x (I4) or |x| (I8), the least x
  double top64 = top, low64 = low;
  int bad = 0;
#pragma unroll
  for (int i = 0; i < kRuns; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int run = N * (in + 32 * i), d = run + j;
      if (ROPE) v[i][j] = x[i][j];
      if (!on || run >= hd) continue;  // runs lie in a row whole
      if (ROPE) {
        if (kind == 0) {
          const double a = __dmul_rn(x[i][j], cs[i][j]), b = __dmul_rn(w[i][j], sn[i][j]);
          v[i][j] = d < half ? __dsub_rn(a, b) : __dadd_rn(a, b);
          x[i][j] = (float)v[i][j];
        }
        top64 = fmax(top64, I4 ? v[i][j] : fabs(v[i][j]));
        if (I4) low64 = fmin(low64, v[i][j]);
        bad |= !isfinite(x[i][j]);
      } else {
        top = max_nan(top, I4 ? x[i][j] : fabsf(x[i][j]));
        if (I4) low = min_nan(low, x[i][j]);
      }
    }
  float zero = 0.0f, scale;
  for (int o = group / 2; o; o >>= 1) {
    if (ROPE) {
      bad |= __shfl_xor_sync(0xffffffffu, bad, o);
      top64 = fmax(top64, __shfl_xor_sync(0xffffffffu, top64, o));
      if (I4) low64 = fmin(low64, __shfl_xor_sync(0xffffffffu, low64, o));
    } else {
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (I4) low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
  }
  if (!on) return;
  if (!ROPE) {
    bad = !isfinite(top) || (I4 && !isfinite(low));
    top64 = top;
    low64 = low;
  }
  if (I4) {
    zero = __fadd_rn((float)low64, 0.0f);  // never -0
    scale = __fadd_rn(fifteenth(top64 - (double)zero), 0.0f);
  } else {
    scale = ROPE ? (float)(top64 / 127.0) : __fdiv_rn(top, 127.0f);
  }
  // a row that holds a value that is not finite reads back as NaN
  if (bad || !isfinite(scale) || !isfinite(zero)) {
    scale = __int_as_float(0x7fc00000);
    if (in == 0) atomicOr(s.status, kStatusNonFinite);
    bad = 1;
  }
  const int slot = pos % kPage;
  uint8_t* codes = block + (size_t)(kind * kPage + slot) * kvq_row_bytes(hd, I4);
  const float inv = __fdiv_rn(1.0f, scale);
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    const int d = N * (in + 32 * i);
    if (d >= hd) continue;
    uint32_t word[4] = {0u, 0u, 0u, 0u};
    if (!bad && scale > 0.0f) {
      // what is divided: an element (I8), or an element less the zero (I4)
      auto part = [&](int j) { return I4 ? (ROPE ? (float)(v[i][j] - (double)zero) : __fsub_rn(x[i][j], zero)) : x[i][j]; };
      uint32_t bits[N];
      float off = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) bits[j] = code_bits<I4 && ROPE>(part(j), inv, &off);
      if (!(off < 0.4999f)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          float mine = 0.0f;
          code_bits<I4 && ROPE>(part(j), inv, &mine);
          if (!(mine < 0.4999f))
            bits[j] = kCodeBits + border_code((ROPE ? v[i][j] : (double)x[i][j]) - (double)zero, scale, I4 ? 0 : -127, I4 ? 15 : 127);
        }
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (I4)
          word[j / 8] += (bits[j] << (4 * (j % 8))) - (kCodeBits << (4 * (j % 8)));
        else if (j % 4 == 3)
          word[j / 4] = __byte_perm(__byte_perm(bits[j - 3], bits[j - 2], 0x0040), __byte_perm(bits[j - 1], bits[j], 0x0040), 0x5410);
        else if (N == 2 && j == 1)
          word[0] = __byte_perm(bits[0], bits[1], 0x0040);
      }
    }
    uint8_t* dst = codes + (I4 ? d / 2 : d);
    constexpr int kBytes = I4 ? N / 2 : N;
    if (kBytes == 16)
      *(uint4*)dst = make_uint4(word[0], word[1], word[2], word[3]);
    else if (kBytes == 8)
      *(uint2*)dst = make_uint2(word[0], word[1]);
    else if (kBytes == 4)
      *(uint32_t*)dst = word[0];
    else if (kBytes == 2)
      *(uint16_t*)dst = (uint16_t)word[0];
    else
      *dst = (uint8_t)word[0];
  }
  if (in == 0) {
    float* par = block_params(block, hd, I4, kind);
    par[slot] = scale;
    if (I4) par[kPage + slot] = zero;
  }
}

// ---------------------------------------------------------------------------
// Load.  Warps take rows in turn, all heads of K and V, the lanes over runs of
// N elements in the order in which they are written; several warps share a row
// when there are few.  Where the next row's blocks lie (three dependent loads)
// is asked for before this row is read, and kLoadAhead runs a lane before the
// first is written.  Codes become floats without conversions: a byte below the
// bits of 2^23 is 2^23 + c.  Bound by memory: 130870 rows of 8 kv heads of 128,
// I4 to bf16, 143 us (4.8 TB/s, most of it writes); 517 rows of 5, I8 to f32, 3 us.
// ---------------------------------------------------------------------------
constexpr int kLoadAhead = 4;
// Byte i of w (unsigned), less `bias`, as a float.
__device__ __forceinline__ float byte_f32(uint32_t w, int i, float bias) {
  return __fsub_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)), 8388608.0f + bias);
}
template <int N, bool I4>
__device__ __forceinline__ void codes_f32(const uint32_t* w, float* x) {
  if (I4) {
    const uint32_t even = w[0] & 0x0f0f0f0fu, odd = (w[0] >> 4) & 0x0f0f0f0fu;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = byte_f32(j % 2 ? odd : even, j / 2, 0.0f);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = byte_f32(w[j / 4] ^ 0x80808080u, j % 4, 128.0f);
  }
}
// HD: the head size, or 0 where it is not one of the common ones.
template <int HD, int N, bool I4>
__global__ void __launch_bounds__(kStoreWarps * 32)
    kvq_load_kernel(KvqView c, int rows, const int32_t* __restrict__ row_seq, const int32_t* __restrict__ row_pos,
                    void* __restrict__ k, size_t ldk, void* __restrict__ v, size_t ldv, int bf16, int wide,
                    int per_row, int32_t* status) {
  const int lane = threadIdx.x & 31, hd = HD ? HD : c.hd, runs = hd / N, all = 2 * c.kv_heads * runs;
  const int warp = blockIdx.x * kStoreWarps + (threadIdx.x >> 5), teams = gridDim.x * kStoreWarps / per_row;
  const int part = warp % per_row;
  const int rowb = kvq_row_bytes(hd, I4), block_bytes = kvq_block_bytes(hd, I4);
  int row = warp / per_row;
  if (row >= teams) return;  // warps that make no whole team
  int pos = -1, next_pos = -1;
  const uint8_t *first = nullptr, *next = nullptr;
  auto look_up = [&](int r, int* p) -> const uint8_t* {
    *p = r < rows ? (row_pos ? row_pos[r] : r) : -1;
    return *p >= 0 ? block_of(c, row_seq ? row_seq[r] : 0, *p, 0) : nullptr;
  };
  next = look_up(row, &next_pos);
  for (; row < rows; row += teams) {
    first = next;
    pos = next_pos;
    next = look_up(row > INT_MAX - teams ? INT_MAX : row + teams, &next_pos);
    if (!first) {
      if (lane == 0 && pos >= 0) atomicOr(status, kStatusBadContext);
      if (row > INT_MAX - teams) break;
      continue;
    }
    const uint8_t* from = first + pos % kPage * rowb;  // head 0's K codes, and its K parameters
    const float* par0 = block_params((uint8_t*)first, hd, I4, 0) + pos % kPage;
    const size_t row_k = (size_t)row * ldk, row_v = (size_t)row * ldv;
    for (int r0 = part * 32 + lane; r0 < all; r0 += per_row * 32 * kLoadAhead) {
      uint32_t w[kLoadAhead][2];
      float scale[kLoadAhead], zero[kLoadAhead];
#pragma unroll
      for (int i = 0; i < kLoadAhead; ++i) {
        const int r = r0 + i * per_row * 32;
        if (r >= all) continue;
        const int which = r / runs, d = r % runs * N, kind = which >= c.kv_heads;
        const uint32_t to_block = (which - kind * c.kv_heads) * block_bytes;
        const uint8_t* codes = from + (to_block + kind * (kPage * rowb));
        if (N == 8 && I4) {
          w[i][0] = *(const uint32_t*)(codes + d / 2);
        } else if (N == 8) {
          const uint2 u = *(const uint2*)(codes + d);
          w[i][0] = u.x;
          w[i][1] = u.y;
        } else {
          w[i][0] = I4 ? codes[d / 2] : *(const uint16_t*)(codes + d);
        }
        const float* par = (const float*)((const uint8_t*)par0 + (to_block + kind * (I4 ? 128 : 64)));
        scale[i] = par[0];
        zero[i] = I4 ? par[kPage] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kLoadAhead; ++i) {
        const int r = r0 + i * per_row * 32;
        if (r >= all) continue;
        const int kind = r >= all / 2;  // K and V rows are written in the order of r
        void* dst = kind ? v : k;
        const size_t at = (kind ? row_v : row_k) + (r - kind * (all / 2)) * N;
        float x[N];
        codes_f32<N, I4>(w[i], x);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = __fmaf_rn(x[j], scale[i], zero[i]);
        if (N == 8 && wide && bf16) {
          uint32_t u[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * j % N], x[(2 * j + 1) % N]);
            u[j] = *(const uint32_t*)&p;
          }
          *(uint4*)((uint16_t*)dst + at) = make_uint4(u[0], u[1], u[2], u[3]);
        } else if (N == 8 && wide) {
          *(float4*)((float*)dst + at) = make_float4(x[0], x[1], x[2 % N], x[3 % N]);
          *(float4*)((float*)dst + at + 4) = make_float4(x[4 % N], x[5 % N], x[6 % N], x[7 % N]);
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) store_elem(dst, at + j, bf16, x[j]);
        }
      }
    }
    if (row > INT_MAX - teams) break;
  }
}

}  // namespace

namespace {
// Whether runs of 8 elements of a matrix start on 16 bytes.
bool aligned_runs(const void* p, size_t ld, int bf16) { return (uintptr_t)p % 16 == 0 && ld % (bf16 ? 8 : 4) == 0; }

template <int N, bool I4, bool ROPE>
void launch_store(const KvqView& c, const KvqStore& s, int group, int wide, cudaStream_t st) {
  const size_t jobs = (size_t)s.rows * (2 * c.kv_heads + (s.q ? s.nh : 0));
  kvq_store_kernel<N, I4, ROPE>
      <<<(unsigned)ceil_div(jobs * group, kStoreWarps * 32), kStoreWarps * 32, 0, st>>>(c, s, group, wide);
}
template <int N>
void launch_store_of(const KvqView& c, const KvqStore& s, int group, int wide, cudaStream_t st) {
  if (c.i4)
    s.rope_cos ? launch_store<N, true, true>(c, s, group, wide, st) : launch_store<N, true, false>(c, s, group, wide, st);
  else
    s.rope_cos ? launch_store<N, false, true>(c, s, group, wide, st) : launch_store<N, false, false>(c, s, group, wide, st);
}
}  // namespace

void launch_kvq_store(const KvqView& c, const KvqStore& s, cudaStream_t st) {
  if (s.rows <= 0) return;
  const RowSplit split = split_row(c.hd, (size_t)s.rows * c.kv_heads >= 148 * 64);
  const int wide = aligned_runs(s.k, s.ldk, s.bf16) && aligned_runs(s.v, s.ldv, s.bf16) &&
                   (!s.q || aligned_runs(s.q, s.ldq, 0)) && (uintptr_t)s.rope_cos % 16 == 0 &&
                   (uintptr_t)s.rope_sin % 16 == 0;
  if (split.run == 16)
    launch_store_of<16>(c, s, split.group, wide, st);
  else if (split.run == 8)
    launch_store_of<8>(c, s, split.group, wide, st);
  else
    launch_store_of<2>(c, s, split.group, wide, st);
  count_launch();
}

void launch_kvq_load(const KvqView& c, int rows, const int32_t* row_seq, const int32_t* row_pos, void* k, size_t ldk,
                     void* v, size_t ldv, int bf16, int32_t* status, cudaStream_t st) {
  if (rows <= 0) return;
  const int run = split_row(c.hd, false).run, wide = aligned_runs(k, ldk, bf16) && aligned_runs(v, ldv, bf16);
  // few rows: more warps to each, so that all runs are asked for at once
  const int most = (int)ceil_div((size_t)2 * c.kv_heads * (c.hd / run), 32);
  const int per_row = rows >= 148 * 16 ? (int)ceil_div(most, 2 * kLoadAhead) : most;
  const unsigned blocks = (unsigned)ceil_div((size_t)std::min(rows, kLoadTeams) * per_row, kStoreWarps);
  auto* kernel = kvq_load_kernel<0, 2, false>;
  if (run == 2)
    kernel = c.i4 ? kvq_load_kernel<0, 2, true> : kvq_load_kernel<0, 2, false>;
  else if (c.hd == 128)
    kernel = c.i4 ? kvq_load_kernel<128, 8, true> : kvq_load_kernel<128, 8, false>;
  else if (c.hd == 64)
    kernel = c.i4 ? kvq_load_kernel<64, 8, true> : kvq_load_kernel<64, 8, false>;
  else
    kernel = c.i4 ? kvq_load_kernel<0, 8, true> : kvq_load_kernel<0, 8, false>;
  kernel<<<blocks, kStoreWarps * 32, 0, st>>>(c, rows, row_seq, row_pos, k, ldk, v, ldv, bf16, wide, per_row, status);
  count_launch();
}

}  // namespace bitnet
