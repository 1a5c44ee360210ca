// Many sequences over one paged key/value cache: rotary tables and rotation, rows written into pages (quantized) and read
// back, and the attention of one new token a sequence. The layout of the pools is in include/elmh.h.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "elm_dma.h"
#include "elm_dpp.h"
#include "elm_paged.h"
#include "elm_quant.h"
#include "elmh_internal.hpp"

namespace elmh {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
// loads of words that lie on less than their size
using u32_on1 = __attribute__((aligned(1))) uint32_t;
using u32_on2 = __attribute__((aligned(2))) uint32_t;
using u32x3_on4 = __attribute__((ext_vector_type(3), aligned(4))) uint32_t;
using u32x4_on8 = __attribute__((ext_vector_type(4), aligned(8))) uint32_t;

// ---------------------------------------------------------------- rotary tables and rotation

// m sin(a) and m cos(a) rounded to f32: a (in f64, |a| < 2^31) less its nearest multiple k of pi / 2, which adding 1.5 2^52 leaves
// in the low bits (pi / 2 in two parts, so that nothing is lost), then the Taylor sums to r^11 and r^12 on [-pi / 4, pi / 4]: the
// first terms left out are under 2^-36, a four-thousandth of a half step. Some 32 instructions; a library sine in f64 takes
// five times as many.
__device__ __forceinline__ void sincos_f64(double a, double m, float& sn, float& cs) {
  constexpr double kShift = 6755399441055744.0;
  const double t = fma(a, 0.63661977236758134308, kShift);
  const uint32_t q = (uint32_t)__double_as_longlong(t);
  const double k = t - kShift;
  double r = fma(k, -1.57079632679489655800, a);
  r = fma(k, -6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = fma(z, -1.0 / 39916800, 1.0 / 362880);
  s = fma(s, z, -1.0 / 5040);
  s = fma(s, z, 1.0 / 120);
  s = fma(s, z, -1.0 / 6);
  const double rm = r * m;
  s = fma(s * z, rm, rm);
  double c = fma(z, 1.0 / 479001600, -1.0 / 3628800);
  c = fma(c, z, 1.0 / 40320);
  c = fma(c, z, -1.0 / 720);
  c = fma(c, z, 1.0 / 24);
  c = fma(c, z, -0.5);
  c = fma(c, z * m, m);
  const float fs = (float)s, fc = (float)c;
  const bool swap = q & 1;
  sn = __uint_as_float(__float_as_uint(swap ? fc : fs) ^ ((q & 2) << 30));
  cs = __uint_as_float(__float_as_uint(swap ? fs : fc) ^ (((q + 1) & 2) << 30));
}

// Workgroups of whole rows (positions): each takes the pairs' frequencies into LDS once (a power in f64 costs as much as many
// angles), then its threads W neighbouring pairs at a time. Bound by the tables' writes (2^20 positions of 128: 95 us, 5.6 TB/s; a
// fill alone 6.9) and the f64 sums beside them (vector ALUs 64% busy).
template <int W>
__global__ __launch_bounds__(256) void rope_table_kernel(float* __restrict__ cs, float* __restrict__ sn, int64_t pos0,
                                                         int64_t n, int half, int rows, double theta, RopeBand band) {
  __shared__ double freq[512];
  for (int i = threadIdx.x; i < half; i += 256) freq[i] = rope_scaled(band, pow(theta, -2.0 * i / (2 * half)), i);
  __syncthreads();
  const int per = half / W;
  const int64_t first = (int64_t)blockIdx.x * rows;
  const int here = (int)(n - first < rows ? n - first : rows);
  const int drow = 256 / per, dcol = 256 % per;
  int row = threadIdx.x / per, col = threadIdx.x % per;
  while (row < here) {
    const double p = (double)(pos0 + first + row);
    float c[W], s[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      sincos_f64(p * freq[W * col + w], band.magnitude, s[w], c[w]);
    }
    const int64_t at = (first + row) * half + W * col;
    if constexpr (W == 4) {
      *reinterpret_cast<f32x4*>(cs + at) = f32x4{c[0], c[1], c[2], c[3]};
      *reinterpret_cast<f32x4*>(sn + at) = f32x4{s[0], s[1], s[2], s[3]};
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        cs[at + w] = c[w];
        sn[at + w] = s[w];
      }
    }
    row += drow;
    col += dcol;
    if (col >= per) {
      col -= per;
      ++row;
    }
  }
}

// What a thread does is the same for every row: it finds its head and values once and then takes rows blockIdx.y, + gridDim.y,
// ..., kRopeRows at a time. Both of a pair are one thread's, so that rows may be rotated in place. Bound by reading and writing
// the rows (7777 rows of 32 heads of 96: 41 us, 4.7 TB/s, of 5.1 to 5.4 that a copy reaches).
constexpr int kRopeRows = 4;

// Where everything is aligned: per head rot / 8 threads with two groups of four values, i .. and i + rot / 2 .. (half layout),
// and (hd - rot) / 4 with four that pass; interleaved: hd / 4 threads with four neighbours. A wave's accesses are contiguous.
__global__ __launch_bounds__(256) void rope_quads_kernel(const float* x, float* y, int T, int per_head, int n_heads, int hd,
                                                         int64_t x_row, int64_t y_row, const float* __restrict__ cs,
                                                         const float* __restrict__ sn, int max_pos, int rot, int inter,
                                                         const int32_t* __restrict__ pos, int64_t pos0) {
  const int u = blockIdx.x * 256 + threadIdx.x, head = u / per_head, i = u % per_head, half = rot / 2;
  if (head >= n_heads) return;
  const bool split = !inter && i < rot / 8, near = inter && i < rot / 4, turned = split || near;
  if (!turned && x == y) return;
  const int a = head * hd + 4 * i + (turned || inter ? 0 : half);  // half layout: the passing values follow both halves
  const int at = near ? 2 * i : 4 * i;
  for (int t0 = blockIdx.y * kRopeRows; t0 < T; t0 += gridDim.y * kRopeRows) {
    f32x4 va[kRopeRows], vb[kRopeRows], c[kRopeRows], s[kRopeRows];
    bool live[kRopeRows];
#pragma unroll
    for (int r = 0; r < kRopeRows; ++r) {
      const int t = min(t0 + r, T - 1);
      const int64_t p = pos ? pos[t] : pos0 + t;
      live[r] = t0 + r < T && p >= 0 && p < max_pos;
      const float* src = x + t * x_row + a;
      const int64_t row = (live[r] ? p : 0) * half;
      va[r] = *reinterpret_cast<const f32x4*>(src);
      if (split) {
        vb[r] = *reinterpret_cast<const f32x4*>(src + half);
        c[r] = *reinterpret_cast<const f32x4*>(cs + row + at);
        s[r] = *reinterpret_cast<const f32x4*>(sn + row + at);
      } else if (near) {
        const float2 c2 = *reinterpret_cast<const float2*>(cs + row + at), s2 = *reinterpret_cast<const float2*>(sn + row + at);
        c[r] = f32x4{c2.x, c2.x, c2.y, c2.y};
        s[r] = f32x4{-s2.x, s2.x, -s2.y, s2.y};  // u c - v s = u c + v (-s), to the bit
      }
    }
#pragma unroll
    for (int r = 0; r < kRopeRows; ++r) {
      if (!live[r]) continue;
      float* dst = y + (int64_t)(t0 + r) * y_row + a;
      f32x4 o = va[r];
      if (split) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = va[r][e] * c[r][e] - vb[r][e] * s[r][e];
        f32x4 q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = vb[r][e] * c[r][e] + va[r][e] * s[r][e];
        *reinterpret_cast<f32x4*>(dst + half) = q;
      } else if (near) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = va[r][e] * c[r][e] + va[r][e ^ 1] * s[r][e];
      }
      *reinterpret_cast<f32x4*>(dst) = o;
    }
  }
}

// Any alignment: hd / 2 threads a head, each a pair, or two neighbours that pass
__global__ __launch_bounds__(256) void rope_pairs_kernel(const float* x, float* y, int T, int per_head, int n_heads, int hd,
                                                         int64_t x_row, int64_t y_row, const float* __restrict__ cs,
                                                         const float* __restrict__ sn, int max_pos, int rot, int inter,
                                                         const int32_t* __restrict__ pos, int64_t pos0) {
  const int u = blockIdx.x * 256 + threadIdx.x, head = u / per_head, i = u % per_head, half = rot / 2;
  if (head >= n_heads) return;
  const bool turned = i < half, split = turned && !inter;
  if (!turned && x == y) return;
  const int a = head * hd + (split ? i : 2 * i), b = split ? a + half : a + 1;
  for (int t0 = blockIdx.y * kRopeRows; t0 < T; t0 += gridDim.y * kRopeRows) {
    float va[kRopeRows], vb[kRopeRows], c[kRopeRows], s[kRopeRows];
    bool live[kRopeRows];
#pragma unroll
    for (int r = 0; r < kRopeRows; ++r) {
      const int t = min(t0 + r, T - 1);
      const int64_t p = pos ? pos[t] : pos0 + t;
      live[r] = t0 + r < T && p >= 0 && p < max_pos;
      const int64_t at = (live[r] ? p : 0) * half + (turned ? i : 0);
      va[r] = x[t * x_row + a];
      vb[r] = x[t * x_row + b];
      c[r] = cs[at];
      s[r] = sn[at];
    }
#pragma unroll
    for (int r = 0; r < kRopeRows; ++r) {
      if (!live[r]) continue;
      float* dst = y + (int64_t)(t0 + r) * y_row;
      dst[a] = turned ? va[r] * c[r] - vb[r] * s[r] : va[r];
      dst[b] = turned ? vb[r] * c[r] + va[r] * s[r] : vb[r];
    }
  }
}

// ---------------------------------------------------------------- rows into pages and back

struct RowArgs {
  const float *k, *v;  // rows in (append)
  float *ko, *vo;      // rows out (read)
  int64_t row, head;
  int n;
  elmh_kv_pages pages;
  const int32_t* table;
  int n_seqs, max_pages;
  const int32_t *pos, *seq;
  const float *cs, *sn;
  int max_pos, rot, inter;
  uint32_t magic;   // page_magic(page_size)
  int head_shift;   // a workgroup's rows: of 2^head_shift heads
};

// Where a row of a call lies in the cache; page < 0: the row is skipped
struct RowPlace {
  int64_t page;
  int slot, pos;
};
__device__ __forceinline__ RowPlace row_place(const RowArgs& a, int pos, int seq) {
  if (seq < 0 || seq >= a.n_seqs || pos < 0 || (a.cs && pos >= a.max_pos)) return {-1, 0, 0};
  return {kv_page_of(a.table + (int64_t)seq * a.max_pages, a.max_pages, a.pages.n_pages, pos, a.magic),
          pos - page_index(pos, a.magic) * a.pages.page_size, pos};
}

// Value d of a head's row x, rotated
__device__ __forceinline__ float rotated(const float* x, int d, const float* cs, const float* sn, int half, int inter) {
  if (d >= 2 * half) return x[d];
  const int i = inter ? d >> 1 : d < half ? d : d - half;
  const bool second = inter ? d & 1 : d >= half;
  const float c = cs[i], s = sn[i], self = x[d];
  const float other = x[inter ? d ^ 1 : second ? d - half : d + half];
  return second ? self * c + other * s : self * c - other * s;
}

// Rows go by eight lanes each: lane c of them holds values 32 j + 4 c .. + 3 of every 32-value group j, so that eight lanes read
// or write 128 contiguous bytes of f32 a group, the group's q4 scale is a matter of eight lanes, and its eight 4-bit levels
// lie in neighbouring bytes. A workgroup: 32 rows in one pool (grid: tokens, heads, pools); of neighbouring heads of a token
// where those are neighbours outside the cache, in f32 most of what is moved, of one head elsewhere (36 thousand q8 tokens of 8
// heads read in 59 us, 5.2 TB/s, by token; 69 by head). Writing is half bound by the quantizer's vector work: 6800 q4 tokens 18 us, 3.5 TB/s.
constexpr int kRowLanes = 8;
constexpr int kRowsPerBlock = 256 / kRowLanes;

__device__ __forceinline__ int row_token(const RowArgs& a) {
  return (int)blockIdx.x * (kRowsPerBlock >> a.head_shift) + ((int)(threadIdx.x / kRowLanes) >> a.head_shift);
}
__device__ __forceinline__ int row_head(const RowArgs& a) {
  return ((int)blockIdx.y << a.head_shift) + ((int)(threadIdx.x / kRowLanes) & ((1 << a.head_shift) - 1));
}

// max over a row's eight lanes, in one instruction a step
__device__ __forceinline__ float row_max8(float v) {
  v = fmaxf(v, dpp_f<kDppQuadXor1>(v));
  v = fmaxf(v, dpp_f<kDppQuadXor2>(v));
  return fmaxf(v, dpp_f<kDppHalfMirror>(v));
}

// A row's values in lane c, and with the half layout those that the rotated ones pair with (read again from L1: they are another
// lane's, or this one's of another group). VEC: 16-byte loads (the host has checked that every one is aligned, and that a lane's
// four values are either all rotated or none, with their partners four values too).
template <int NB, bool VEC>
struct AppendRow {
  float x[NB][4];
  f32x4 o[VEC ? NB : 1];

  // what does not depend on the row's position, so that it is on its way while the table is looked up
  __device__ __forceinline__ void load(const float* src, int c, bool turn, int half, int inter) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int d = 32 * j + 4 * c;
        const f32x4 v = *reinterpret_cast<const f32x4*>(src + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] = v[e];
        if (turn && !inter && d < 2 * half) o[j] = *reinterpret_cast<const f32x4*>(src + (d >= half ? d - half : d + half));
      }
    }
  }
  // cs, sn: the position's row of the tables, or null
  __device__ __forceinline__ void rotate(const float* src, int c, const float* cs, const float* sn, int half, int inter) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int d = 32 * j + 4 * c;
      if constexpr (!VEC) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] = cs ? rotated(src, d + e, cs, sn, half, inter) : src[d + e];
      } else if (cs && d < 2 * half) {
        if (inter) {
          const float2 co = *reinterpret_cast<const float2*>(cs + d / 2), si = *reinterpret_cast<const float2*>(sn + d / 2);
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float cc = e ? co.y : co.x, ss = e ? si.y : si.x, u = x[j][e], v = x[j][e + 1];
            x[j][e] = u * cc - v * ss;
            x[j][e + 1] = v * cc + u * ss;
          }
        } else {
          const bool second = d >= half;
          const int i = second ? d - half : d;
          const f32x4 co = *reinterpret_cast<const f32x4*>(cs + i), si = *reinterpret_cast<const f32x4*>(sn + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float ss = second ? si[e] : -si[e];  // u c - v s = u c + v (-s), to the bit
            x[j][e] = x[j][e] * co[e] + o[j][e] * ss;
          }
        }
      }
    }
  }
};

// N bytes at a multiple of the largest power of two that divides N
template <int N>
__device__ __forceinline__ void store_bytes(uint8_t* p, const uint32_t* w) {
  constexpr int by = N % 16 == 0 ? 16 : N % 8 == 0 ? 8 : N % 4 == 0 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < N; i += by) {
    if constexpr (by == 16) *reinterpret_cast<u32x4*>(p + i) = u32x4{w[i / 4], w[i / 4 + 1], w[i / 4 + 2], w[i / 4 + 3]};
    else if constexpr (by == 8) *reinterpret_cast<u32x2*>(p + i) = u32x2{w[i / 4], w[i / 4 + 1]};
    else if constexpr (by == 4) *reinterpret_cast<uint32_t*>(p + i) = w[i / 4];
    else *reinterpret_cast<uint16_t*>(p + i) = (uint16_t)(w[i / 4] >> (8 * (i % 4)));
  }
}
template <int N>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* w) {
  constexpr int by = N % 16 == 0 ? 16 : N % 8 == 0 ? 8 : N % 4 == 0 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < N; i += by) {
    if constexpr (by == 16) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(p + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[i / 4 + k] = v[k];
    } else if constexpr (by == 8) {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p + i);
      w[i / 4] = v[0];
      w[i / 4 + 1] = v[1];
    } else if constexpr (by == 4) {
      w[i / 4] = *reinterpret_cast<const uint32_t*>(p + i);
    } else {
      const uint32_t v = *reinterpret_cast<const uint16_t*>(p + i);
      w[i / 4] = i % 4 ? w[i / 4] | v << 16 : v;
    }
  }
}

template <int DT, int NB, bool VEC>
__global__ __launch_bounds__(256) void paged_append_kernel(RowArgs a) {
  constexpr int HD = 32 * NB;
  const elmh_kv_pages& pg = a.pages;
  const int t = row_token(a), c = threadIdx.x % kRowLanes, h = row_head(a);
  const bool keys = blockIdx.z == 0;
  if (t >= a.n) return;  // whole rows: the lanes of a row stay together
  const bool turn = keys && a.cs;
  const int half = a.rot / 2;
  const float* src = (keys ? a.k : a.v) + t * a.row + h * a.head;
  const int pos = a.pos[t], seq = a.seq ? a.seq[t] : t;
  AppendRow<NB, VEC> r;
  r.load(src, c, turn, half, a.inter);
  const RowPlace w = row_place(a, pos, seq);
  if (w.page < 0) return;
  const int64_t at = (int64_t)w.pos * half;
  r.rotate(src, c, turn ? a.cs + at : nullptr, turn ? a.sn + at : nullptr, half, a.inter);
  const auto& x = r.x;
  const int64_t row = kv_row(w.page, h, w.slot, pg.n_kv, pg.page_size);
  uint8_t* dst = static_cast<uint8_t*>(keys ? pg.k : pg.v) + row * (DT == ELMH_F32 ? 4 * HD : DT == ELMH_Q8 ? HD : DT == ELMH_Q4 ? HD / 2 : 2 * HD);
  float* scales = keys ? pg.k_scale : pg.v_scale;
  if constexpr (DT == ELMH_F32) {
#pragma unroll
    for (int j = 0; j < NB; ++j) *reinterpret_cast<f32x4*>(dst + 128 * j + 16 * c) = f32x4{x[j][0], x[j][1], x[j][2], x[j][3]};
  } else if constexpr (DT == ELMH_F16 || DT == ELMH_BF16) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == ELMH_F16) u[e] = __builtin_bit_cast(uint16_t, (_Float16)x[j][e]);
        else u[e] = __builtin_bit_cast(uint16_t, (__bf16)x[j][e]);
      }
      *reinterpret_cast<u32x2*>(dst + 64 * j + 8 * c) = u32x2{u[0] | u[1] << 16, u[2] | u[3] << 16};
    }
  } else if constexpr (DT == ELMH_Q8) {
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(x[j][e]));
    amax = row_max8(amax);
    const float s = amax / 127.f, div = s == 0.f ? 1.f : s;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      float q[4];
      elm_level_group<4, -127, 127>(x[j], div, q);
      // bytes q + 128, two a conversion; then each less 128 again
      const uint32_t lo = (uint32_t)fmaf(q[1], 256.f, q[0] + 32896.f), hi = (uint32_t)fmaf(q[3], 256.f, q[2] + 32896.f);
      *reinterpret_cast<uint32_t*>(dst + 32 * j + 4 * c) = (lo | hi << 16) ^ 0x80808080u;
    }
    if (c == 0) scales[row] = s;
  } else {
    uint32_t b[NB];  // a group's two bytes of this lane
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      // the first value of largest magnitude: the largest or the smallest one, and where those are level, the first of them
      const float up = row_max8(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));
      const float down = row_max8(fmaxf(fmaxf(-x[j][0], -x[j][1]), fmaxf(-x[j][2], -x[j][3])));
      float peak = up >= down ? up : -down;
      if (__any(up == down && up != 0.f)) {
        float m = x[j][0];
#pragma unroll
        for (int e = 1; e < 4; ++e) m = fabsf(x[j][e]) > fabsf(m) ? x[j][e] : m;
        const uint32_t have = (uint32_t)(__ballot(fabsf(m) == fmaxf(up, down)) >> (threadIdx.x & 56)) & 0xFFu;
        peak = __shfl(m, (threadIdx.x & 56) + (have ? __builtin_ctz(have) : 0), 64);  // have: 0 only where a value is no number
      }
      const float s = peak / -8.f, div = s == 0.f ? 1.f : s;
      float q[4];
      elm_level_group<4, -8, 7>(x[j], div, q);
      // four nibbles q + 8 in one conversion: whole numbers under 2^16
      b[j] = (uint32_t)fmaf(q[3], 4096.f, fmaf(q[2], 256.f, fmaf(q[1], 16.f, q[0] + 34952.f)));
      if (c == 0) scales[kv_scale(w.page, h, w.slot, pg.n_kv, pg.page_size, NB) + (int64_t)j * pg.page_size] = s;
    }
    if (keys) {  // [c / 2][j]: words of which this lane has one half; the even lane stores them
      uint32_t o[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) o[j] = b[j] | (uint32_t)dpp_i<kDppQuadXor1>(b[j]) << 16;
      if (c % 2 == 0) store_bytes<4 * NB>(dst + c / 2 * 4 * NB, o);
    } else {  // [2 c][j], [2 c + 1][j]: all of this lane's bytes are neighbours
      uint32_t o[(2 * NB + 3) / 4] = {};
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        o[j / 4] |= (b[j] & 0xFF) << (8 * (j % 4));
        o[(NB + j) / 4] |= (b[j] >> 8) << (8 * ((NB + j) % 4));
      }
      store_bytes<2 * NB>(dst + 2 * c * NB, o);
    }
  }
}

template <int DT, int NB, bool VEC>
__global__ __launch_bounds__(256) void paged_read_kernel(RowArgs a) {
  constexpr int HD = 32 * NB;
  const elmh_kv_pages& pg = a.pages;
  const int t = row_token(a), c = threadIdx.x % kRowLanes, h = row_head(a);
  const bool keys = blockIdx.z == 0;
  if (t >= a.n) return;
  const RowPlace w = row_place(a, a.pos[t], a.seq ? a.seq[t] : t);
  if (w.page < 0) return;
  const int64_t row = kv_row(w.page, h, w.slot, pg.n_kv, pg.page_size);
  const uint8_t* src = static_cast<const uint8_t*>(keys ? pg.k : pg.v) +
                       row * (DT == ELMH_F32 ? 4 * HD : DT == ELMH_Q8 ? HD : DT == ELMH_Q4 ? HD / 2 : 2 * HD);
  const float* scales = keys ? pg.k_scale : pg.v_scale;
  float x[NB][4];
  if constexpr (DT == ELMH_F32) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(src + 128 * j + 16 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = v[e];
    }
  } else if constexpr (DT == ELMH_F16 || DT == ELMH_BF16) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const u32x2 u = *reinterpret_cast<const u32x2*>(src + 64 * j + 8 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint16_t b = (uint16_t)(u[e / 2] >> (16 * (e % 2)));
        if constexpr (DT == ELMH_F16) x[j][e] = (float)__builtin_bit_cast(_Float16, b);
        else x[j][e] = __uint_as_float((uint32_t)b << 16);
      }
    }
  } else if constexpr (DT == ELMH_Q8) {
    const float s = scales[row];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(src + 32 * j + 4 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = (float)(int8_t)(u >> (8 * e)) * s;
    }
  } else {
    const float* sc = scales + kv_scale(w.page, h, w.slot, pg.n_kv, pg.page_size, NB);
    uint32_t b[NB];  // keys: [c / 2][j], words of which this lane's are one half; values: [2 c][j], [2 c + 1][j]
    if (keys) {
      load_bytes<4 * NB>(src + c / 2 * 4 * NB, b);
#pragma unroll
      for (int j = 0; j < NB; ++j) b[j] >>= 16 * (c % 2);
    } else {
      uint32_t o[(2 * NB + 3) / 4];
      load_bytes<2 * NB>(src + 2 * c * NB, o);
#pragma unroll
      for (int j = 0; j < NB; ++j)
        b[j] = (o[j / 4] >> (8 * (j % 4)) & 0xFF) | (o[(NB + j) / 4] >> (8 * ((NB + j) % 4)) & 0xFF) << 8;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const uint32_t u = b[j];
      const float s = sc[(int64_t)j * pg.page_size];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = (float)((int)(u >> (4 * e) & 15) - 8) * s;
    }
  }
  float* dst = (keys ? a.ko : a.vo) + t * a.row + h * a.head;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int d = 32 * j + 4 * c;
    if constexpr (VEC) {
      *reinterpret_cast<f32x4*>(dst + d) = f32x4{x[j][0], x[j][1], x[j][2], x[j][3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[d + e] = x[j][e];
    }
  }
}

// ---------------------------------------------------------------- attention of one new token a sequence

// f(0), f(1), ..., f(N - 1) with compile-time indices
template <int N, int I = 0, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
}

constexpr int kPaWaves = 4;
constexpr int kPaHeads = 16;       // query heads a workgroup takes: the columns of a 16 x 16 tile
constexpr float kLog2e = 1.44269504088896340736f;

// The matrix instructions take 16-bit operands, 32 values deep, or f32 ones, 4 deep. Products are exact in both (f32
// accumulation); what is in 32 bits (queries, softmax weights) is split into 16-bit pieces whose sum has its 24 bits:
//   f16, q8, q4 caches: f16 operands (levels are exact in f16), two pieces of 11 bits, a power of two taken out first;
//   bf16 caches: bf16 operands, three pieces of 8 bits.
enum { kOpF32 = 0, kOpF16 = 1, kOpBF16 = 2 };
constexpr int op_of(int dt) { return dt == ELMH_F32 ? kOpF32 : dt == ELMH_BF16 ? kOpBF16 : kOpF16; }
constexpr int pieces_of(int dt) { return dt == ELMH_BF16 ? 3 : 2; }

template <int OP>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (OP == kOpBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// x[0..7] as the pieces of a 32-deep operand. f16: |x| < 2^15.
// minus_one: -1, opaque to the compiler, which then takes a residual in one mixed-precision instruction.
template <int OP>
__device__ __forceinline__ void split8(const float* x, u32x4* out, float minus_one) {
  if constexpr (OP == kOpF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto p = __builtin_amdgcn_cvt_pkrtz(x[2 * i], x[2 * i + 1]);
      const f16x2 r{(_Float16)fmaf((float)p[0], minus_one, x[2 * i]), (_Float16)fmaf((float)p[1], minus_one, x[2 * i + 1])};
      out[0][i] = __builtin_bit_cast(uint32_t, p);
      out[1][i] = __builtin_bit_cast(uint32_t, r);
    }
  } else {  // the top 16 bits, twice, and what is left: exact
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u[2][3];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = x[2 * i + e];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          u[e][k] = __float_as_uint(v);
          v -= __uint_as_float(u[e][k] & 0xFFFF0000u);
        }
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) out[k][i] = __builtin_amdgcn_perm(u[1][k], u[0][k], 0x07060302);
    }
  }
}

// Levels as f16, two an instruction. A small integer u in the low bits of a half is the subnormal u 2^-24, and the fused
// multiply-add takes it to (u - bias) 2^-9, exactly: levels are held times 2^-9 (kLevelExp), which the final factor undoes.
// (The subnormals themselves as operands, their bias taken off a score's sum, save the multiply-add but give errors of 2.7e-6
// in place of 2.8e-7: the matrix instruction aligns a subnormal's product by its exponent, not by its leading bit.)
constexpr int kLevelExp = 9;
__device__ __forceinline__ uint32_t f16_levels(uint32_t w, float mul, float add) {
  const f16x2 r = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)mul, (_Float16)mul},
                                            f16x2{(_Float16)add, (_Float16)add});
  return __builtin_bit_cast(uint32_t, r);
}
// bytes q + 128 in the halves' low bytes
__device__ __forceinline__ uint32_t f16_bytes(uint32_t w) { return f16_levels(w, 0x1p15f, -0x1p-2f); }
// nibbles q + 8 at bits 0-3, and at bits 4-7 (16 u 2^-24 times 2^11)
__device__ __forceinline__ uint32_t f16_low_nibbles(uint32_t w) { return f16_levels(w & 0x000F000Fu, 0x1p15f, -0x1p-6f); }
__device__ __forceinline__ uint32_t f16_high_nibbles(uint32_t w) { return f16_levels(w & 0x00F000F0u, 0x1p11f, -0x1p-6f); }
// a whole byte of two nibbles: 16 (q1 + 8) + (q0 + 8) - 136
__device__ __forceinline__ uint32_t f16_nibble_bytes(uint32_t w) { return f16_levels(w, 0x1p15f, -136 * 0x1p-9f); }

// ---- which values of a row a lane holds. Lane = 16 g + n.
// Keys (rows of the 16 x 32 operand are tokens, n): step j's eight values of lane group g.
template <int DT, int NB>
ELM_HD constexpr int key_dim(int j, int g, int e) {
  if (DT == ELMH_Q8 && !(NB % 2 == 1 && j == NB - 1)) return 64 * (j / 2) + 16 * g + 8 * (j % 2) + e;
  if (DT == ELMH_Q4) return 32 * j + 8 * g + (e / 2) + 4 * (e % 2);
  return 32 * j + 8 * g + e;
}
// Values (rows of the operand are the row's values, 16 of them an instruction): value x (0 .. 2 NB - 1) of lane n. A lane's
// values are neighbours in units of 32 values times 4, 2 or 1, so that sixteen lanes read a unit as one piece.
constexpr int unit_width(int NB, int x) {  // of the unit that value x is in
  int left = NB, at = 0;
  while (true) {
    const int w = left >= 4 ? 4 : left >= 2 ? 2 : 1;
    if (x < at + 2 * w) return w;
    at += 2 * w;
    left -= w;
  }
}
constexpr int unit_start(int NB, int x) {  // its first value index x
  int left = NB, at = 0;
  while (true) {
    const int w = left >= 4 ? 4 : left >= 2 ? 2 : 1;
    if (x < at + 2 * w) return at;
    at += 2 * w;
    left -= w;
  }
}
template <int DT, int NB>
__device__ __forceinline__ constexpr int value_dim(int x, int n) {
  if (DT == ELMH_Q4) return 32 * (x / 2) + 2 * n + x % 2;
  const int w = unit_width(NB, x), s = unit_start(NB, x);
  return 16 * s + 2 * w * n + (x - s);
}

// ---- a block of 16 tokens' rows in registers, as loaded
constexpr int key_words(int dt, int NB) { return dt == ELMH_F32 ? 8 * NB : dt == ELMH_Q8 ? 2 * NB : dt == ELMH_Q4 ? NB : 4 * NB; }
constexpr int value_words(int dt, int NB) {  // per token (four tokens a lane)
  return dt == ELMH_F32 ? 2 * NB : dt == ELMH_Q8 ? (NB + 1) / 2 : dt == ELMH_Q4 ? (NB + 3) / 4 : NB;
}

template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (WORDS >= 4) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[i];
    if constexpr (WORDS > 4) load_words<WORDS - 4>(p + 16, w + 4);
  } else if constexpr (WORDS >= 2) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    w[0] = v[0];
    w[1] = v[1];
    if constexpr (WORDS > 2) load_words<WORDS - 2>(p + 8, w + 2);
  } else if constexpr (WORDS == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// The loads take a uniform base (scalar registers) and a lane's 32-bit offset.
// base: the block's first key row; off: the lane's row and group, key_offset
template <int DT, int NB>
__device__ __forceinline__ uint32_t key_offset(int n, int g) {
  constexpr int HD = 32 * NB;
  if (DT == ELMH_F32) return n * 4 * HD + 16 * g;
  if (DT == ELMH_Q8) return n * HD;
  if (DT == ELMH_Q4) return n * (HD / 2) + 4 * NB * g;
  return n * 2 * HD + 16 * g;
}
template <int DT, int NB>
__device__ __forceinline__ void load_key(const uint8_t* base, uint32_t off, int g, uint32_t (&w)[key_words(DT, NB)]) {
  if constexpr (DT == ELMH_F32) {
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j) load_words<4>(base + off + 64 * j, w + 4 * j);
  } else if constexpr (DT == ELMH_Q8) {
#pragma unroll
    for (int j = 0; j + 1 < NB; j += 2) load_words<4>(base + (off + 16 * g) + 32 * j, w + 2 * j);
    if constexpr (NB % 2) load_words<2>(base + (off + 8 * g) + 32 * (NB - 1), w + 2 * (NB - 1));
  } else if constexpr (DT == ELMH_Q4) {
    if constexpr (NB == 3) {  // at 12 g
      const u32x3_on4 v = *reinterpret_cast<const u32x3_on4*>(base + off);
#pragma unroll
      for (int j = 0; j < 3; ++j) w[j] = v[j];
    } else if constexpr (NB == 6) {  // at 24 g
      const u32x4_on8 v = *reinterpret_cast<const u32x4_on8*>(base + off);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = v[j];
      load_words<2>(base + off + 16, w + 4);
    } else {
      load_words<NB>(base + off, w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NB; ++j) load_words<4>(base + off + 64 * j, w + 4 * j);
  }
}
// the operand of step j (16-bit forms)
template <int DT, int NB>
__device__ __forceinline__ u32x4 key_operand(const uint32_t (&w)[key_words(DT, NB)], int j) {
  if constexpr (DT == ELMH_Q8) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t u = w[2 * j + i] ^ 0x80808080u;
      o[2 * i] = f16_bytes(__builtin_amdgcn_perm(0, u, 0x0C010C00));
      o[2 * i + 1] = f16_bytes(__builtin_amdgcn_perm(0, u, 0x0C030C02));
    }
    return o;
  } else if constexpr (DT == ELMH_Q4) {
    const uint32_t u = w[j], v = u >> 8;
    return u32x4{f16_low_nibbles(u), f16_high_nibbles(u), f16_low_nibbles(v), f16_high_nibbles(v)};
  } else {
    return u32x4{w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]};
  }
}

// row: a token's value row less the lane's offset, off; n: the lane's part of it
// (As few loads as there can be: with a q4 row of 96 read by bytes, 24 sequences of 8 to 16 thousand took 73 us, so 47.)
template <int DT, int NB>
__device__ __forceinline__ void load_value(const uint8_t* row, uint32_t off, int n, uint32_t (&w)[value_words(DT, NB)]) {
  if constexpr (DT == ELMH_Q4) {  // NB bytes at n * NB
    if constexpr (NB == 1) {
      w[0] = row[off + n];
    } else if constexpr (NB == 2) {
      w[0] = *reinterpret_cast<const uint16_t*>(row + (off + 2 * n));
    } else if constexpr (NB == 3) {
      w[0] = *reinterpret_cast<const u32_on1*>(row + (off + 3 * n - (n == 15)));  // the last lane's from its second byte on
    } else if constexpr (NB == 6) {
      w[0] = *reinterpret_cast<const u32_on2*>(row + (off + 6 * n));
      w[1] = *reinterpret_cast<const uint16_t*>(row + (off + 6 * n + 4));
    } else {
      load_words<NB / 4>(row + (off + NB * n), w);
    }
  } else {
    constexpr int B = DT == ELMH_F32 ? 4 : DT == ELMH_Q8 ? 1 : 2;
    // units of 4, 2 and 1 times 32 values
    if constexpr (NB >= 4) load_words<2 * B>(row + (off + 8 * B * n), w);
    if constexpr (NB == 8) load_words<2 * B>(row + (off + 8 * B * n) + 128 * B, w + 2 * B);
    constexpr int done = NB / 4 * 4;
    if constexpr ((NB & 2) != 0) load_words<B>(row + (off + 4 * B * n) + 32 * done * B, w + done * B / 2);
    constexpr int last = NB & ~1;
    if constexpr ((NB & 1) != 0) {
      const uint8_t* p = row + (off + 2 * B * n) + 32 * last * B;
      if constexpr (B == 1) w[last / 2] = *reinterpret_cast<const uint16_t*>(p);
      else load_words<B / 2>(p, w + last * B / 2);
    }
  }
}
// The operand of value x over eight tokens: v[0..3] the first block's, v[4..7] the second's. q4: of an odd x the byte that holds it
// and its neighbour, 16 times the one plus the other: the neighbour's sum is taken off at the end (after the last tile).
template <int DT, int NB>
__device__ __forceinline__ u32x4 value_operand(const uint32_t (&v)[8][value_words(DT, NB)], int x, int n) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == ELMH_Q8) {
      const uint32_t a = v[2 * i][x / 4], b = v[2 * i + 1][x / 4];
      const uint32_t sel = 0x0C040C00u + (x % 4) * 0x00010001u;
      o[i] = f16_bytes(__builtin_amdgcn_perm(b, a, sel));  // the bytes were flipped to q + 128
    } else if constexpr (DT == ELMH_Q4) {
      const int j = x / 2;
      const uint32_t sel = 0x0C040C00u + (j % 4 + (NB == 3 && n == 15)) * 0x00010001u;
      const uint32_t w = __builtin_amdgcn_perm(v[2 * i + 1][j / 4], v[2 * i][j / 4], sel);
      o[i] = x % 2 ? f16_nibble_bytes(w) : f16_low_nibbles(w);
    } else {
      o[i] = __builtin_amdgcn_perm(v[2 * i + 1][x / 2], v[2 * i][x / 2], x % 2 ? 0x07060302u : 0x05040100u);
    }
  }
  return o;
}

struct PagedAttnArgs {
  const float* q;
  float* out;
  int64_t q_row;
  int n_heads, group, head_tiles;  // query heads; per kv head; workgroups a kv head's take
  elmh_kv_pages pages;
  const int32_t* table;
  int max_pages;
  uint32_t magic;  // page_magic(page_size)
  const int32_t* lens;
  int max_len;
  const float *cs, *sn;
  int rot, inter;
  int n_seqs;
  PartRule rule;      // the split: PagedShare
  float* part_o;      // [slot][head][head_dim], unnormalized
  float* part_s;      // [slot][head][2]: running maximum (base 2), sum
  int2* joins;        // [seq]: first slot, parts; null where no sequence is split
};

// One instruction for two or three operands (a NaN stays one), where fmaxf first quiets what may be signalling
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// max over the four lane groups: v_permlane16_swap of a value with itself leaves each lane its own and its neighbour row's
__device__ __forceinline__ float max_over_groups(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = max_of(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_of(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127

// The batch is split by its own lengths, which every workgroup reads: a part's size is the same for all sequences, and a
// sequence has as many parts of at most that size as it needs (one if it is empty), so that a long sequence among short ones
// is no longer on the way than the others. n_seqs + extra slots are always enough.
struct PagedShare {
  int seq, len, units;
  int part, parts, first;  // which of the sequence's, of how many, the first one's slot
};
// The share of a slot. Uniform (every lane of the wave calls); seq < 0: the slot is no sequence's. A workgroup's first hundreds of
// instructions come from memory (some 10 clocks each), so there is no division among them.
__device__ __forceinline__ PagedShare paged_share(const PagedAttnArgs& a, int slot) {
  const int lane = threadIdx.x & 63;
  const auto len_of = [&](int i) { return i < a.n_seqs ? min(max(a.lens[i], 0), a.max_len) : 0; };
  const auto units_of = [&](int len) { return (int)(((uint32_t)len + kSplitUnit - 1) / kSplitUnit); };
  const int len0 = len_of(lane);
  int total = wave_sum_i(units_of(len0));
  for (int i = 64; i < a.n_seqs; i += 64) total += wave_sum_i(units_of(len_of(i + lane)));
  const float inverse = part_inverse(part_size(total, a.rule));
  int before = 0, i = 0, len = len0;
  while (true) {
    const int units = units_of(len), parts = i + lane < a.n_seqs ? part_count(units, inverse) : 0;
    const int sum = wave_scan_i(parts);
    const uint64_t past = __ballot(before + sum > slot);
    if (past) {
      const int at = __builtin_ctzll(past);
      PagedShare s;
      s.seq = i + at;
      s.len = __builtin_amdgcn_readlane(len, at);
      s.units = __builtin_amdgcn_readlane(units, at);
      s.parts = __builtin_amdgcn_readlane(parts, at);
      s.first = before + __builtin_amdgcn_readlane(sum, at) - s.parts;
      s.part = slot - s.first;
      return s;
    }
    i += 64;
    if (i >= a.n_seqs) return {-1, 0, 0, 0, 0, 0};
    before += __builtin_amdgcn_readlane(sum, 63);
    len = len_of(i + lane);
  }
}

// Two blocks of 16 tokens (a wave's step): where they lie, and how many tokens of each count (0: behind the end, or no page)
struct PagedTile {
  int valid[2];
  int64_t row[2], scale[2];
};

// What a wave holds of a tile while it is on its way
template <int DT, int NB, bool COLS>
struct PagedRegs {
  uint32_t k[2][key_words(DT, NB)];
  uint32_t v[8][value_words(DT, NB)];
  // quantized: of tokens 4 g .. + 3 of a block. COLS: of the lane's group, for both blocks; else lane n has group n / 2 of block
  // n % 2 (q8: of block n % 2) in [0]
  f32x4 ks[COLS ? 2 : 1], vs[COLS ? 2 : 1];
};

// Registers for two workgroups a CU, or one
constexpr int attention_fits(int dt, int NB, bool cols) { return part_workgroups(dt, 32 * NB, cols) > 256 ? 2 : 1; }
// Query operands that stay in LDS (the same for all waves; [group][piece][lane] of 16 bytes): 64 registers less, so that two
// workgroups fit a CU (8 sequences of 17591 with 7 queries a kv head: 71 us, 108 with one; at 128 and 192 it gains nothing).
constexpr bool query_in_lds(int dt, int NB, bool cols) { return dt == ELMH_Q4 && NB == 8 && !cols; }

// One workgroup: one part of one sequence's cache for up to 16 query heads of one kv head, its waves taking 32 tokens at a time.
// Scores as K Q^T (tokens x heads) leave a lane with four tokens of one head, which is what the second product V^T P^T takes
// as its operand: no exchange between lanes but the maximum over the four lane groups. One pass: running maximum m and sum l.
// A wave's next keys are on their way while it takes the weights and the values, its next values while it takes the scores.
// Bound by reading the cache where it is long (100003 bf16 positions, 410 MB: 73 us, 5.6 TB/s, of 5.7 that a read alone reaches; 64 q4
// sequences of 8 to 16 thousand, 980 MB: 5.0 TB/s, vector ALUs 66% and matrix cores 23% busy), by the way to the first rows, four
// dependent loads, where it is short (137 f32 positions: 6.6 us a call). Four waves: with eight the same cases took 87 us for 79
// and 246 for 205. 32 tokens a step: the depth of a 16-bit matrix instruction in the second product.
// COLS (q4, where the heads times the NB groups of 32, made a power of two, fit in the 16 columns): column n = h + j HS, of the HS
// heads that fit, is head h and group j. Its
// query is zero outside the group, so a score's NB parts come out in NB lanes, each multiplied by its own group's scale and
// then added over them; and its weights take its own group's value scales, so that one split of 8 weights serves in place of
// NB.
template <int DT, int NB, bool COLS>
__global__ __launch_bounds__(64 * kPaWaves, attention_fits(DT, NB, COLS)) void paged_attention_kernel(PagedAttnArgs a) {
  constexpr int HD = 32 * NB, OP = op_of(DT), PC = pieces_of(DT);
  extern __shared__ float lds[];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x;
  const int h0 = kvh * a.group + blockIdx.z * kPaHeads;
  const int heads = min(kPaHeads, (kvh + 1) * a.group - h0);
  const elmh_kv_pages& pg = a.pages;
  const PagedShare share = paged_share(a, blockIdx.y);
  const int seq = share.seq, len = share.len;
  if (seq < 0) return;
  float* out = a.out + (int64_t)seq * a.n_heads * HD + (int64_t)h0 * HD;
  // for the join (written last: a store ahead of the table's loads would keep them off the scalar cache)
  const auto note = [&] {
    if (share.part == 0 && blockIdx.x + blockIdx.z == 0 && tid == 0 && a.joins) a.joins[seq] = make_int2(share.first, share.parts);
  };
  if (len == 0) {
    for (int i = tid; i < heads * HD; i += 64 * kPaWaves) out[i] = 0.f;
    note();
    return;
  }

  const int32_t* trow = a.table + (int64_t)seq * a.max_pages;
  const int ps = pg.page_size, last = (int)((uint32_t)(len - 1) / kPageStep);
  constexpr int RB = DT == ELMH_F32 ? 4 * HD : DT == ELMH_Q8 ? HD : DT == ELMH_Q4 ? HD / 2 : 2 * HD;
  constexpr int NG = DT == ELMH_Q8 ? 1 : DT == ELMH_Q4 ? NB : 0;
  const uint8_t* kpool = static_cast<const uint8_t*>(pg.k);
  const uint8_t* vpool = static_cast<const uint8_t*>(pg.v);
  const uint32_t koff = key_offset<DT, NB>(n, g), voff = 4 * g * RB;
  // the lane's scales: group j of block u, as PagedRegs says
  constexpr int HS = COLS ? cols_heads(HD) : 16;
  const int cj = n / HS;  // COLS: the column's group; past the last one its sums are 0 and not looked at
  const int sj = COLS ? min(cj, NG - 1) : NG > 1 ? min(n / 2, NG - 1) : 0, su = n & 1;
  const uint32_t soff = (uint32_t)(sj * ps + 4 * g) * 4;
  const int qn = COLS ? n % HS : n;  // the lane's head

  // the table's entries of a unit's two blocks (of the last block's, past the end)
  const auto ask = [&](int unit, int (&id)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) id[u] = trow[page_index(min(2 * unit + u, last) * kPageStep, a.magic)];
  };
  const int steps = (int)((uint32_t)ps / kPageStep);
  const auto place = [&](int unit, const int (&id)[2]) {
    PagedTile t;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int block = min(2 * unit + u, last);
      const int page = __builtin_amdgcn_readfirstlane(id[u]);
      const bool there = (uint32_t)page < (uint32_t)pg.n_pages;
      t.valid[u] = there && 2 * unit + u <= last ? min(kPageStep, len - block * kPageStep) : 0;
      const uint32_t head = (uint32_t)(there ? page : 0) * pg.n_kv + kvh;
      const uint32_t step = block - page_index(block * kPageStep, a.magic) * steps;
      t.row[u] = (int64_t)(head * steps + step) * kPageStep;  // the pool has fewer than 2^32 blocks
      t.scale[u] = NG == 1 ? t.row[u] : ((int64_t)(head * steps) * NG + step) * kPageStep;
    }
    return t;
  };
  PagedRegs<DT, NB, COLS> r;
  const auto load_scales = [&](f32x4* to, const float* pool, const PagedTile& t) {
    const auto at = [&](int64_t scale) { return *reinterpret_cast<const f32x4*>(reinterpret_cast<const uint8_t*>(pool + scale) + soff); };
    if constexpr (COLS) {
      to[0] = at(t.scale[0]);
      to[1] = at(t.scale[1]);
    } else if constexpr (NG > 0) {
      to[0] = at(su ? t.scale[1] : t.scale[0]);
    }
  };
  const auto load_keys = [&](const PagedTile& t) {
#pragma unroll
    for (int u = 0; u < 2; ++u) load_key<DT, NB>(kpool + t.row[u] * RB, koff, g, r.k[u]);
    load_scales(r.ks, pg.k_scale, t);
  };
  const auto load_values = [&](const PagedTile& t) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) load_value<DT, NB>(vpool + t.row[u] * RB + i * RB, voff, n, r.v[4 * u + i]);
    load_scales(r.vs, pg.v_scale, t);
  };

  const int end = __builtin_amdgcn_readfirstlane(part_begin(share.units, share.part + 1, share.parts));
  int unit = __builtin_amdgcn_readfirstlane(part_begin(share.units, share.part, share.parts)) + wave;
  const bool busy = unit < end;  // a wave without a unit joins with nothing
  int id[2];
  PagedTile tile;
  if (busy) {
    ask(unit, id);
    tile = place(unit, id);
    load_keys(tile);
    load_values(tile);
    ask(unit + kPaWaves, id);
  }

  // the queries, rotated at the last position
  const float* q = a.q + seq * a.q_row + (int64_t)h0 * HD;
  for (int i = tid; i < heads * HD; i += 64 * kPaWaves) {
    const int64_t at = (int64_t)(len - 1) * (a.rot / 2);
    lds[i] = a.cs ? rotated(q + i / HD * HD, i % HD, a.cs + at, a.sn + at, a.rot / 2, a.inter) : q[i];
  }
  lds_barrier();
  // as operands; `scale`: what a product is multiplied by to be a score in units of log2
  float minus_one = -1.f;
  asm("" : "+v"(minus_one));
  float scale = kLog2e / sqrtf((float)HD);
  u32x4 qo[OP == kOpF32 ? 1 : NB][OP == kOpF32 ? 1 : PC];
  float qf[OP == kOpF32 ? 8 * NB : 1];
  const float* qrow = lds + min(qn, heads - 1) * HD;
  if constexpr (OP == kOpF32) {
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[4 * j + i] = qrow[16 * j + 4 * g + i];
  } else {
    constexpr int QJ = COLS ? 1 : NB;  // groups that a lane reads: with COLS its own
    float x[QJ][8];
#pragma unroll
    for (int j = 0; j < QJ; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = qrow[32 * sj * COLS + key_dim<DT, NB>(j, g, e)];
    if constexpr (OP == kOpF16) {  // the head's largest value to 512 .. 1024: its 24 bits then lie in f16's range
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < QJ; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[j][e]));
      big = max_over_groups(big);
      if constexpr (COLS) {
        big = max_of(big, dpp_f<kDppRowRor8>(big));
        if constexpr (HS <= 4) big = max_of(big, dpp_f<kDppRowRor4>(big));
        if constexpr (HS <= 2) big = max_of(big, dpp_f<kDppRowRor2>(big));
      }
      const int ex = min(max((int)((__float_as_uint(big) >> 23) & 255) - 127, -100), 127);
      const float up = pow2(9 - ex);
      scale *= pow2(ex - 9 + (NG ? kLevelExp : 0));
#pragma unroll
      for (int j = 0; j < QJ; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] *= up;
    }
#pragma unroll
    for (int j = 0; j < QJ; ++j) split8<OP>(x[j], qo[j], minus_one);
    if constexpr (COLS) {
#pragma unroll
      for (int p = 0; p < PC; ++p) {
        const u32x4 o = qo[0][p];
#pragma unroll
        for (int j = 0; j < NB; ++j) qo[j][p] = cj == j ? o : u32x4{0, 0, 0, 0};
      }
    }
  }

  constexpr bool QLDS = query_in_lds(DT, NB, COLS);
  const u32x4* qlds = reinterpret_cast<const u32x4*>(lds) + lane;
  if constexpr (QLDS) {
    lds_barrier();  // the queries have been read
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (j % kPaWaves == wave) {
#pragma unroll
        for (int p = 0; p < PC; ++p) reinterpret_cast<u32x4*>(lds)[64 * (PC * j + p) + lane] = qo[j][p];
      }
    lds_barrier();
  }

  float m = -INFINITY, l = 0.f;
  int vexp = -100;  // q8, q4: the softmax weights take the value scales over 2^vexp, the largest seen
  f32x4 acc[2 * NB];
#pragma unroll
  for (int x = 0; x < 2 * NB; ++x) acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};

  const auto step = [&](auto more) {
    const bool whole = tile.valid[0] == kPageStep && tile.valid[1] == kPageStep;
    float s[8];
    int qat = 0;
    if constexpr (QLDS) asm("" : "+v"(qat));  // read in each step: the compiler would keep them in registers again
    static_for<2>([&](auto U) {
      constexpr int u = U;
      f32x4 sc{0.f, 0.f, 0.f, 0.f};
      if constexpr (OP == kOpF32) {
#pragma unroll
        for (int j = 0; j < 8 * NB; ++j) sc = mfma_f32(__uint_as_float(r.k[u][j]), qf[j], sc);
      } else {
        static_for<NB>([&](auto J) {
          constexpr int j = J;
          const u32x4 ko = key_operand<DT, NB>(r.k[u], j);
          constexpr bool apart = DT == ELMH_Q4 && !COLS;  // groups' sums, each with its scale
          f32x4 t = apart ? f32x4{0.f, 0.f, 0.f, 0.f} : sc;
#pragma unroll
          for (int p = PC - 1; p >= 0; --p) t = mfma<OP>(ko, QLDS ? qlds[qat + 64 * (PC * j + p)] : qo[j][p], t);
          if constexpr (apart) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[i] = fmaf(row_bcast<2 * j + u>(r.ks[0][i]), t[i], sc[i]);
          } else {
            sc = t;
          }
        });
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = sc[i];
        if constexpr (COLS) {  // the same sum in all of a head's lanes: halves, then quarters, ...
          v *= r.ks[u][i];
          v += dpp_f<kDppRowRor8>(v);
          if constexpr (HS <= 4) v += dpp_f<kDppRowRor4>(v);
          if constexpr (HS <= 2) v += dpp_f<kDppRowRor2>(v);
        } else if constexpr (DT == ELMH_Q8) {
          v *= row_bcast<u>(r.ks[0][i]);
        }
        s[4 * u + i] = v;
      }
    });
    const PagedTile now = tile;
    if constexpr (more) {
      unit += kPaWaves;
      tile = place(unit, id);
      load_keys(tile);
      ask(unit + kPaWaves, id);
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = 4 * g + i % 4 < now.valid[i / 4] ? s[i] : -INFINITY;
    }

    const float top = max_of(max_of(max_of(max_of(s[0], s[1]), s[2]), max_of(max_of(s[3], s[4]), s[5])), max_of(s[6], s[7]));
    const float mn = max_of(m, max_over_groups(top) * scale);
    const float ref = mn == -INFINITY ? 0.f : mn;  // no token so far: weights of 0, not of exp(-inf + inf)
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], scale, -ref));
    float fade = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    l = l * fade + (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));

    if (!whole) {
      if constexpr (NG == 0) {  // a slot behind the end may hold a NaN, which a weight of 0 does not remove
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int k = 0; k < value_words(DT, NB); ++k) r.v[i][k] = 4 * g + i % 4 < now.valid[i / 4] ? r.v[i][k] : 0u;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (COLS) {
            r.vs[0][i] = 4 * g + i < now.valid[0] ? r.vs[0][i] : 0.f;
            r.vs[1][i] = 4 * g + i < now.valid[1] ? r.vs[1][i] : 0.f;
          } else {
            r.vs[0][i] = 4 * g + i < (su ? now.valid[1] : now.valid[0]) ? r.vs[0][i] : 0.f;
          }
        }
      }
    }
    if constexpr (NG > 0) {
      float big = fmaxf(fmaxf(fabsf(r.vs[0][0]), fabsf(r.vs[0][1])), fmaxf(fabsf(r.vs[0][2]), fabsf(r.vs[0][3])));
      if constexpr (COLS)
        big = fmaxf(big, fmaxf(fmaxf(fabsf(r.vs[1][0]), fabsf(r.vs[1][1])), fmaxf(fabsf(r.vs[1][2]), fabsf(r.vs[1][3]))));
      if (__any(big > pow2(vexp))) {  // rare after the first tokens
        const int ex = min((int)(__float_as_uint(wave_max(big)) >> 23) - 126, 127);
        fade *= pow2(max(vexp - ex, -126));
        vexp = ex;
      }
    }
    if (__any(fade != 1.f)) {
#pragma unroll
      for (int x = 0; x < 2 * NB; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[x][i] *= fade;
    }

    if constexpr (OP == kOpF32) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int x = 0; x < 2 * NB; ++x) acc[x] = mfma_f32(__uint_as_float(r.v[i][x]), p[i], acc[x]);
    } else {
      // f16 pieces: weights up to 2^14, so that a weight 2^-28 of the largest is still a normal number
      if constexpr (OP == kOpF16) {
        const float up = pow2(14 - (NG ? vexp : 0));
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] *= up;
      }
      if constexpr (DT == ELMH_Q8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int k = 0; k < value_words(DT, NB); ++k) r.v[i][k] ^= 0x80808080u;
      }
      constexpr int runs = DT == ELMH_Q4 && !COLS ? NB : 1;  // of values that share their scale
      static_for<runs>([&](auto J) {
        constexpr int j = J;
        u32x4 po[PC];
        float t[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          t[i] = COLS ? r.vs[0][i] * p[i] : NG ? row_bcast<2 * j>(r.vs[0][i]) * p[i] : p[i];
          t[4 + i] = COLS ? r.vs[COLS][i] * p[4 + i] : NG ? row_bcast<2 * j + 1>(r.vs[0][i]) * p[4 + i] : p[4 + i];
        }
        split8<OP>(t, po, minus_one);
#pragma unroll
        for (int x = j * 2 * NB / runs; x < (j + 1) * 2 * NB / runs; ++x) {
          const u32x4 vo = value_operand<DT, NB>(r.v, x, n);
#pragma unroll
          for (int k = PC - 1; k >= 0; --k) acc[x] = mfma<OP>(vo, po[k], acc[x]);
        }
      });
    }
    if constexpr (more) load_values(tile);
  };
  if (busy) {
    while (unit + kPaWaves < end) step(std::true_type{});
    step(std::false_type{});
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  if constexpr (DT == ELMH_Q4) {  // value_operand
#pragma unroll
    for (int x = 1; x < 2 * NB; x += 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[x][i] = (acc[x][i] - acc[x - 1][i]) * 0x1p-4f;
  }
  // the waves' sums joined: o = sum_w 2^(m_w - M) o_w
  lds_barrier();  // the queries have been read
  float* stat = lds + kPaWaves * heads * HD;
  if (qn < heads) {
#pragma unroll
    for (int x = 0; x < 2 * NB; ++x)
      if (!COLS || x / 2 == cj) {
#pragma unroll
        for (int i = 0; i < 4; ++i) lds[(wave * heads + qn) * HD + value_dim<DT, NB>(x, 4 * g + i)] = acc[x][i];
      }
    if (g == 0 && qn == n) {
      stat[wave * kPaHeads + n] = m;
      stat[(kPaWaves + wave) * kPaHeads + n] = l;
      if (n == 0) stat[2 * kPaWaves * kPaHeads + wave] = OP == kOpF16 ? pow2((NG ? vexp + kLevelExp : 0) - 14) : 1.f;
    }
  }
  lds_barrier();
  for (int i = tid; i < heads * HD; i += 64 * kPaWaves) {
    const int h = i / HD, d = i % HD;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) M = fmaxf(M, stat[w * kPaHeads + h]);
    const float ref = M == -INFINITY ? 0.f : M;
    float o = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(stat[w * kPaHeads + h] - ref);
      o += f * stat[2 * kPaWaves * kPaHeads + w] * lds[(w * heads + h) * HD + d];
      L += f * stat[(kPaWaves + w) * kPaHeads + h];
    }
    if (share.parts == 1) {
      out[i] = L == 0.f ? 0.f : o / L;
    } else {
      const int64_t at = (int64_t)blockIdx.y * a.n_heads + h0 + h;
      a.part_o[at * HD + d] = o;
      if (d == 0) {
        a.part_s[at * 2] = M;
        a.part_s[at * 2 + 1] = L;
      }
    }
  }
  note();
}

// The parts of a (sequence, head) joined, always in the same order: the parts' weights 2^(m - M) first, then their rows, four
// values a thread, the threads' sums of every (256 / (head_dim / 4))-th part added in turn. Bound by latency, so a thread's
// first rows are asked for before the weights. A launch of its own: joined by the workgroup that ends last, the same parts have
// to cross from one XCD's L2 to another's, which with a fence takes the whole L2 each time (the 100k-position bf16 case 155 us,
// so 78), and with loads and stores past the L2 is slower too (88 us; 30k positions of q4 32 us, so 20).
constexpr int kJoinThreads = 256;
constexpr int kJoinAhead = 8;
template <int NB>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(PagedAttnArgs a) {
  constexpr int HD = 32 * NB, Q = HD / 4, G = kJoinThreads / Q;
  __shared__ float w[kPartMostExtra + 1], wave_m[kJoinThreads / 64], wave_l[kJoinThreads / 64];
  __shared__ f32x4 sum[G][Q];
  const int tid = threadIdx.x, head = blockIdx.x, seq = blockIdx.y;
  const int2 join = a.joins[seq];
  const int parts = join.y;
  if (parts < 2) return;
  const int64_t at = (int64_t)join.x * a.n_heads + head, step = a.n_heads;
  const int c = tid % Q, grp = tid / Q;
  const f32x4* rows = reinterpret_cast<const f32x4*>(a.part_o + at * HD) + c;
  f32x4 v[kJoinAhead];
#pragma unroll
  for (int i = 0; i < kJoinAhead; ++i) v[i] = rows[min(grp + i * G, parts - 1) * step * Q];
  const float2* stats = reinterpret_cast<const float2*>(a.part_s) + at;
  float M = -INFINITY;
  for (int s = tid; s < parts; s += kJoinThreads) M = fmaxf(M, stats[s * step].x);
  M = wave_max(M);
  if ((tid & 63) == 0) wave_m[tid >> 6] = M;
  lds_barrier();
  M = fmaxf(fmaxf(wave_m[0], wave_m[1]), fmaxf(wave_m[2], wave_m[3]));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  for (int s = tid; s < parts; s += kJoinThreads) {
    const float2 st = stats[s * step];
    const float f = __builtin_amdgcn_exp2f(st.x - ref);
    w[s] = f;
    L += f * st.y;
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) L += __shfl_xor(L, off, 64);
  if ((tid & 63) == 0) wave_l[tid >> 6] = L;
  lds_barrier();
  L = (wave_l[0] + wave_l[1]) + (wave_l[2] + wave_l[3]);
  if (grp < G) {
    f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      const int s = grp + i * G;
      const float f = s < parts ? w[s] : 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += s < parts ? f * v[i][k] : 0.f;
    }
#pragma unroll 4
    for (int s = grp + kJoinAhead * G; s < parts; s += G) {
      const f32x4 u = rows[s * step * Q];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += w[s] * u[k];
    }
    sum[grp][c] = o;
  }
  lds_barrier();
  if (tid < HD) {
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) o += sum[i][tid / 4][tid % 4];
    a.out[((int64_t)seq * a.n_heads + head) * HD + tid] = L == 0.f ? 0.f : o / L;
  }
}

template <int DT, int NB, bool COLS>
hipError_t launch_paged_attention_as(const PagedAttnArgs& a, int n_seqs, int extra, hipStream_t s) {
  const int heads = a.group < kPaHeads ? a.group : kPaHeads;
  size_t lds = (size_t)(kPaWaves * heads * 32 * NB + 2 * kPaWaves * kPaHeads + kPaWaves) * sizeof(float);
  if constexpr (query_in_lds(DT, NB, COLS)) lds = std::max<size_t>(lds, NB * pieces_of(DT) * 64 * sizeof(u32x4));
  if (lds > 64 * 1024) {
    static DeviceOnce once;
    if (!raise_dynamic_lds(once, (const void*)paged_attention_kernel<DT, NB, COLS>, 80 * 1024)) return hipErrorInvalidValue;
  }
  const dim3 grid(a.pages.n_kv, n_seqs + extra, a.head_tiles);  // slots of no sequence come last
  paged_attention_kernel<DT, NB, COLS><<<grid, 64 * kPaWaves, lds, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.part_o) return e;
  paged_join_kernel<NB><<<dim3(a.n_heads, n_seqs), kJoinThreads, 0, s>>>(a);
  return hipGetLastError();
}
template <int DT, int NB>
hipError_t launch_paged_attention_cols(const PagedAttnArgs& a, int n_seqs, int extra, hipStream_t s) {
  if constexpr (DT == ELMH_Q4 && NB > 1)
    if (part_cols(DT, 32 * NB, a.group)) return launch_paged_attention_as<DT, NB, true>(a, n_seqs, extra, s);
  return launch_paged_attention_as<DT, NB, false>(a, n_seqs, extra, s);
}
template <int DT>
hipError_t launch_paged_attention_of(const PagedAttnArgs& a, int n_seqs, int extra, hipStream_t s) {
  switch (a.pages.head_dim) {
    case 32: return launch_paged_attention_cols<DT, 1>(a, n_seqs, extra, s);
    case 64: return launch_paged_attention_cols<DT, 2>(a, n_seqs, extra, s);
    case 96: return launch_paged_attention_cols<DT, 3>(a, n_seqs, extra, s);
    case 128: return launch_paged_attention_cols<DT, 4>(a, n_seqs, extra, s);
    case 192: return launch_paged_attention_cols<DT, 6>(a, n_seqs, extra, s);
    case 256: return launch_paged_attention_cols<DT, 8>(a, n_seqs, extra, s);
  }
  return hipErrorInvalidValue;
}

RowArgs row_args(int n, int64_t row, int64_t head, const elmh_kv_pages& pages, const int32_t* table, int n_seqs,
                 int max_pages, const int32_t* pos, const int32_t* seq, const elmh_rope* rope) {
  const RowStrides st = row_strides(row, head, pages.n_kv, pages.head_dim);
  RowArgs a{};
  a.row = st.row;
  a.head = st.head;
  a.n = n;
  a.pages = pages;
  a.table = table;
  a.n_seqs = n_seqs;
  a.max_pages = max_pages;
  a.pos = pos;
  a.seq = seq;
  a.magic = page_magic(pages.page_size);
  if (a.head < a.row)
    while (a.head_shift < 5 && pages.n_kv % (2 << a.head_shift) == 0) ++a.head_shift;
  if (rope) {
    a.cs = rope->cos;
    a.sn = rope->sin;
    a.max_pos = rope->max_pos;
    a.rot = rope->rot_dim;
    a.inter = rope->interleaved;
  }
  return a;
}
template <int DT, int NB>
void launch_rows_as(const RowArgs& a, bool vec, hipStream_t s) {
  const int tokens = kRowsPerBlock >> a.head_shift;
  const dim3 grid((a.n + tokens - 1) / tokens, a.pages.n_kv >> a.head_shift, 2);
  if (a.ko) {
    if (vec) paged_read_kernel<DT, NB, true><<<grid, 256, 0, s>>>(a);
    else paged_read_kernel<DT, NB, false><<<grid, 256, 0, s>>>(a);
  } else {
    if (vec) paged_append_kernel<DT, NB, true><<<grid, 256, 0, s>>>(a);
    else paged_append_kernel<DT, NB, false><<<grid, 256, 0, s>>>(a);
  }
}
template <int DT>
void launch_rows_of(const RowArgs& a, bool vec, hipStream_t s) {
  switch (a.pages.head_dim) {
    case 32: return launch_rows_as<DT, 1>(a, vec, s);
    case 64: return launch_rows_as<DT, 2>(a, vec, s);
    case 96: return launch_rows_as<DT, 3>(a, vec, s);
    case 128: return launch_rows_as<DT, 4>(a, vec, s);
    case 192: return launch_rows_as<DT, 6>(a, vec, s);
    case 256: return launch_rows_as<DT, 8>(a, vec, s);
  }
}
hipError_t launch_rows(const RowArgs& a, bool vec, hipStream_t s) {
  switch (a.pages.dtype) {
    case ELMH_F32: launch_rows_of<ELMH_F32>(a, vec, s); break;
    case ELMH_F16: launch_rows_of<ELMH_F16>(a, vec, s); break;
    case ELMH_BF16: launch_rows_of<ELMH_BF16>(a, vec, s); break;
    case ELMH_Q8: launch_rows_of<ELMH_Q8>(a, vec, s); break;
    case ELMH_Q4: launch_rows_of<ELMH_Q4>(a, vec, s); break;
  }
  return hipGetLastError();
}
// Rows that can be read or written 16 bytes at a time
bool rows_aligned(const RowArgs& a, const float* k, const float* v) {
  return aligned16(k) && aligned16(v) && a.row % 4 == 0 && a.head % 4 == 0;
}

}  // namespace

hipError_t launch_rope_table(float* cs, float* sn, int64_t pos0, int64_t n, int rot_dim, double theta, const RopeBand& band,
                             hipStream_t s) {
  const int half = rot_dim / 2;
  const bool wide = half % 4 == 0 && aligned16(cs) && aligned16(sn);
  // rows a workgroup: up to 16 passes of its threads, as long as some 2048 workgroups are left
  const int64_t one = std::max<int64_t>(1, 256 / (wide ? half / 4 : half));
  const int64_t rows = one * std::min<int64_t>(16, std::max<int64_t>(1, n / (one * 2048)));
  const int64_t blocks = (n + rows - 1) / rows;
  if (blocks >= 1 << 24) return hipErrorInvalidValue;  // of 256 threads; more table than the card holds
  if (wide)
    rope_table_kernel<4><<<(unsigned)blocks, 256, 0, s>>>(cs, sn, pos0, n, half, (int)rows, theta, band);
  else
    rope_table_kernel<1><<<(unsigned)blocks, 256, 0, s>>>(cs, sn, pos0, n, half, (int)rows, theta, band);
  return hipGetLastError();
}

hipError_t launch_rope(const float* x, float* y, int T, int n_heads, int hd, int64_t x_row, int64_t y_row,
                       const elmh_rope& rope, const int32_t* pos, int64_t pos0, hipStream_t s) {
  const int64_t width = (int64_t)n_heads * hd;
  if (!x_row) x_row = width;
  if (!y_row) y_row = width;
  const bool inter = rope.interleaved != 0;
  const bool quads = hd % 4 == 0 && rope.rot_dim % (inter ? 4 : 8) == 0 && x_row % 4 == 0 && y_row % 4 == 0 && aligned16(x) &&
                     aligned16(y) && aligned16(rope.cos) && aligned16(rope.sin);
  const int per_head = !quads ? hd / 2 : inter ? hd / 4 : rope.rot_dim / 8 + (hd - rope.rot_dim) / 4;
  const int64_t blocks = ((int64_t)n_heads * per_head + 255) / 256;
  // some 8192 workgroups are enough to fill the card
  const int64_t rows = std::max<int64_t>(1, std::min<int64_t>((T + kRopeRows - 1) / kRopeRows, 8192 / blocks));
  const dim3 grid((unsigned)blocks, (unsigned)rows);
  if (quads)
    rope_quads_kernel<<<grid, 256, 0, s>>>(x, y, T, per_head, n_heads, hd, x_row, y_row, rope.cos, rope.sin, rope.max_pos,
                                           rope.rot_dim, rope.interleaved, pos, pos0);
  else
    rope_pairs_kernel<<<grid, 256, 0, s>>>(x, y, T, per_head, n_heads, hd, x_row, y_row, rope.cos, rope.sin, rope.max_pos,
                                           rope.rot_dim, rope.interleaved, pos, pos0);
  return hipGetLastError();
}

hipError_t launch_paged_append(const float* k, const float* v, int n, int64_t row, int64_t head, const elmh_kv_pages& pages,
                               const int32_t* table, int n_seqs, int max_pages, const int32_t* pos, const int32_t* seq,
                               const elmh_rope* rope, hipStream_t s) {
  RowArgs a = row_args(n, row, head, pages, table, n_seqs, max_pages, pos, seq, rope);
  a.k = k;
  a.v = v;
  const bool turns = !rope || (aligned16(rope->cos) && aligned16(rope->sin) &&
                               (rope->interleaved ? rope->rot_dim % 4 == 0 : rope->rot_dim % 8 == 0));
  return launch_rows(a, turns && rows_aligned(a, k, v), s);
}

hipError_t launch_paged_read(float* k, float* v, int n, int64_t row, int64_t head, const elmh_kv_pages& pages,
                             const int32_t* table, int n_seqs, int max_pages, const int32_t* pos, const int32_t* seq,
                             hipStream_t s) {
  RowArgs a = row_args(n, row, head, pages, table, n_seqs, max_pages, pos, seq, nullptr);
  a.ko = k;
  a.vo = v;
  return launch_rows(a, rows_aligned(a, k, v), s);
}

PagedSplit paged_attention_split(int dtype, int n_seqs, int n_heads, int n_kv, int head_dim, int max_len) {
  const int rows = n_kv * ((n_heads / n_kv + kPaHeads - 1) / kPaHeads);
  const int workgroups = part_workgroups(dtype, head_dim, part_cols(dtype, head_dim, n_heads / n_kv));
  PagedSplit p;
  p.extra = part_extra(workgroups, rows, n_seqs, max_len);
  p.rule = part_rule(workgroups, rows, n_seqs, max_len, p.extra, part_alone(dtype, head_dim, n_seqs * rows));
  if (max_len > p.rule.least * kSplitUnit)
    p.part_bytes = ((size_t)n_seqs + p.extra) * n_heads * (head_dim + 2) * sizeof(float) + n_seqs * sizeof(int2);
  return p;
}

hipError_t launch_paged_attention(const float* q, float* out, int64_t q_row, int n_heads, const elmh_kv_pages& pages,
                                  const int32_t* table, int n_seqs, int max_pages, const int32_t* lens, int max_len,
                                  const elmh_rope* rope, const PagedSplit& split, float* parts, hipStream_t s) {
  PagedAttnArgs a{};
  a.q = q;
  a.out = out;
  a.q_row = q_row ? q_row : (int64_t)n_heads * pages.head_dim;
  a.n_heads = n_heads;
  a.group = n_heads / pages.n_kv;
  a.head_tiles = (a.group + kPaHeads - 1) / kPaHeads;
  a.pages = pages;
  a.table = table;
  a.max_pages = max_pages;
  a.lens = lens;
  a.max_len = max_len;
  if (rope) {
    a.cs = rope->cos;
    a.sn = rope->sin;
    a.rot = rope->rot_dim;
    a.inter = rope->interleaved;
  }
  a.magic = page_magic(pages.page_size);
  a.n_seqs = n_seqs;
  a.rule = split.rule;
  if (split.part_bytes) {
    a.part_o = parts;
    a.part_s = parts + ((int64_t)n_seqs + split.extra) * n_heads * pages.head_dim;
    a.joins = reinterpret_cast<int2*>(a.part_s + ((int64_t)n_seqs + split.extra) * n_heads * 2);
  }
  switch (pages.dtype) {
    case ELMH_F32: return launch_paged_attention_of<ELMH_F32>(a, n_seqs, split.extra, s);
    case ELMH_F16: return launch_paged_attention_of<ELMH_F16>(a, n_seqs, split.extra, s);
    case ELMH_BF16: return launch_paged_attention_of<ELMH_BF16>(a, n_seqs, split.extra, s);
    case ELMH_Q8: return launch_paged_attention_of<ELMH_Q8>(a, n_seqs, split.extra, s);
    case ELMH_Q4: return launch_paged_attention_of<ELMH_Q4>(a, n_seqs, split.extra, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace elmh
