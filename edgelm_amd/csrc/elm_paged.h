// The paged key/value cache and rotary tables: what a call has to satisfy, where a row lies, and how a sequence is split over
// workgroups. Plain C++ (no HIP), so that all of it is checked without a GPU; the kernels use the same functions.
#pragma once
#include <cmath>
#include <cstddef>
#include <cstdint>

#include "elmh.h"

#ifdef __HIPCC__
#define ELM_HD __host__ __device__ inline
#else
#define ELM_HD inline
#endif

namespace elmh {

// ---------------------------------------------------------------- layout

constexpr int kPageStep = 16;   // pages hold a multiple of this many positions: one matrix-instruction tile of tokens
constexpr int kMaxPositions = 1 << 28;  // of a sequence
constexpr int kSplitUnit = 32;  // tokens a wave takes at a time; a sequence is split at multiples of it

ELM_HD bool kv_quantized(int dtype) { return dtype == ELMH_Q8 || dtype == ELMH_Q4; }
// f32 scales per row
ELM_HD int kv_groups(int dtype, int head_dim) { return dtype == ELMH_Q8 ? 1 : dtype == ELMH_Q4 ? head_dim / 32 : 0; }
// bytes of one row's values
ELM_HD int kv_row_bytes(int dtype, int head_dim) {
  return dtype == ELMH_F32 ? 4 * head_dim : dtype == ELMH_Q8 ? head_dim : dtype == ELMH_Q4 ? head_dim / 2 : 2 * head_dim;
}
// Rows [page][kv head][slot]: the index of a row, and of its first scale ([page][kv head][group][slot], groups page_size apart)
ELM_HD int64_t kv_row(int64_t page, int head, int slot, int n_kv, int page_size) {
  return (page * n_kv + head) * page_size + slot;
}
ELM_HD int64_t kv_scale(int64_t page, int head, int slot, int n_kv, int page_size, int groups) {
  return (page * n_kv + head) * groups * page_size + slot;
}
// The byte of a q4 row that holds value d (even d in the low nibble). Keys: [c][j][b], values 32 j + 8 c + 2 b, so that the
// eight values a lane multiplies of each group are one word and its words of all groups are contiguous. Value rows: [i][j],
// values 32 j + 2 i, so that sixteen lanes hold one group's values in the same byte.
ELM_HD int q4_key_byte(int d, int head_dim) { return (d % 32 / 8) * (head_dim / 8) + d / 32 * 4 + d % 8 / 2; }
ELM_HD int q4_value_byte(int d, int head_dim) { return d % 32 / 2 * (head_dim / 32) + d / 32; }

// 16-position steps over steps a page, without a division: step * page_magic(page_size) / 2^32, exact below 2^24 steps (the
// magic number is over 2^32 / steps by less than one part, so the product by less than 2^24 * 256 / 2^32 of a page)
ELM_HD uint32_t page_magic(int page_size) {
  const uint32_t per = (uint32_t)page_size / kPageStep;
  return per == 1 ? 0 : (uint32_t)(((uint64_t(1) << 32) + per - 1) / per);
}
ELM_HD int page_index(int pos, uint32_t magic) {
  const uint32_t step = (uint32_t)pos / kPageStep;
  return magic ? (int)(((uint64_t)step * magic) >> 32) : (int)step;
}

// The page of position pos in a sequence's row of the table, or -1: no such entry, or no such page
ELM_HD int64_t kv_page_of(const int32_t* table_row, int max_pages, int64_t n_pages, int pos, uint32_t magic) {
  if (pos < 0 || pos >= kMaxPositions) return -1;
  const int i = page_index(pos, magic);
  if (i >= max_pages) return -1;
  const int64_t p = table_row[i];
  return p >= 0 && p < n_pages ? p : -1;
}

// ---------------------------------------------------------------- the split of a sequence

constexpr int kPartLeastUnits = 4;   // of a part: one unit a wave
constexpr int kPartAloneUnits = 16;  // sequences up to this are not split: the second launch costs more (q8, 200 positions: 8.5 us
                                     // in one, 11.6 split; 500: 10.7 and 11.5; 1000: 14.4 and 11.5)
// Where the whole batch is a few workgroups and a unit takes long (large heads, f32), fewer: 2048 / head_dim, for f32 half of that
// (4 kv heads, 8 sequences of up to 500: f32 of 128 13.0 us, unsplit 18.4; f32 of 256 23.6 and 42; q4 of 256 13.6 and 17.8; of up
// to 300, split all the same, q8 of 192 14.0, unsplit 12.7. At 128 workgroups f32 of 128 takes 21.7 us split, 19.8 unsplit.)
constexpr int kPartFewWorkgroups = 64;
inline int part_alone(int dtype, int head_dim, int workgroups) {
  if (workgroups > kPartFewWorkgroups) return kPartAloneUnits;
  const int units = 2048 / (dtype == ELMH_F32 ? 2 * head_dim : head_dim);
  return units < kPartAloneUnits ? units : kPartAloneUnits;
}
inline int part_least(int max_len, int alone) { return max_len <= alone * kSplitUnit ? alone : kPartLeastUnits; }
constexpr int kPartFairUnits = 12;   // a part that is worth its start and end
constexpr int kPartLongUnits = 64;   // a part whose start and end no longer matter
constexpr int kPartMostExtra = 1024;
// Query heads a kv head whose groups of 32 values fit in the 16 columns of a tile together: the q4 attention's other form
ELM_HD constexpr int cols_heads(int head_dim) { return head_dim <= 64 ? 8 : head_dim <= 128 ? 4 : 2; }
constexpr bool part_cols(int dtype, int head_dim, int group) {
  return dtype == ELMH_Q4 && head_dim > 32 && group <= cols_heads(head_dim);
}
// Workgroups that are on the card together: as many a CU as the kernel's registers leave room for, one to four. Above a head size
// of 128 two fit where the cache has few bytes (a 16-bit type to 192, q8, q4), and are worth up to a sixth (8 sequences of 4 to 8
// thousand, 4 kv heads: q4 of 192 24.2 us, with one 28.8; q8 of 256 36 and 37). Counting three where two fit (q4 of 128, more heads
// than columns) costs up to a fifth: 54 sequences of up to 6000 53 us, so 48; 3 of up to 36 thousand 27 and 22. (bf16 of 96 fits
// three, and is better counted as two: 16 sequences of up to 3000 19 us, as three 20; two of some 70 thousand 96 and 92.)
constexpr int part_workgroups(int dtype, int head_dim, bool cols = false) {
  if (head_dim > 128) return 256 * (dtype == ELMH_Q8 || dtype == ELMH_Q4 || (dtype != ELMH_F32 && head_dim <= 192) ? 2 : 1);
  const bool two = dtype == ELMH_F32 || dtype == ELMH_BF16 || (dtype == ELMH_Q4 && head_dim > 96 && !cols);
  return 256 * (head_dim <= 64 ? 4 : two ? 2 : 3);
}
// Parts beside one a sequence: three times the workgroups on the card, over the `rows` (kv heads times their tiles) that take
// every part, but none that a batch of max_len cannot fill
inline int part_extra(int workgroups, int rows, int n_seqs, int max_len) {
  const int64_t units = (max_len + kSplitUnit - 1) / kSplitUnit;
  const int64_t most = (units + kPartLeastUnits - 1) / kPartLeastUnits * n_seqs;
  int64_t want = 3 * (int64_t)workgroups / rows;
  if (want < 1) want = 1;
  if (want > kPartMostExtra) want = kPartMostExtra;
  return (int)(want < most ? want : most);
}
// Parts that `total` is cut into where all of them are to be on the card together, their sequences' shorter last ones counted
inline int part_once(int workgroups, int rows, int n_seqs, int extra) {
  const int all = workgroups / rows, left = all - n_seqs > all / 2 ? all - n_seqs : all / 2;
  return left < 1 ? 1 : left < extra ? left : extra;
}
inline int part_few(int rows, int extra) {
  const int few = 256 / rows;
  return few < 1 ? 1 : few < extra ? few : extra;
}
// ceil(n / d) by a multiplication: at least that, and over it by one at most (exact while n stays under 2^32 / d)
struct CeilDiv {
  uint32_t below = 0;       // d - 1
  uint32_t lo = 1, hi = 1;  // floor(2^32 / d) + 1
};
inline CeilDiv ceil_div(int d) {
  const uint64_t m = (uint64_t(1) << 32) / (uint32_t)d + 1;
  return {(uint32_t)d - 1, (uint32_t)m, (uint32_t)(m >> 32)};
}
ELM_HD uint32_t mul_high(uint32_t a, uint32_t b) { return (uint32_t)(((uint64_t)a * b) >> 32); }
ELM_HD int ceil_of(int n, const CeilDiv& d) {
  const uint32_t x = (uint32_t)n + d.below;
  return (int)(mul_high(x, d.lo) + (d.hi ? x : 0));
}

// The rule that every workgroup applies to the batch's lengths
struct PartRule {
  CeilDiv few, once, extra;
  int least = 1;
};
inline PartRule part_rule(int workgroups, int rows, int n_seqs, int max_len, int extra, int alone = kPartAloneUnits) {
  return {ceil_div(part_few(rows, extra)), ceil_div(part_once(workgroups, rows, n_seqs, extra)), ceil_div(extra), part_least(max_len, alone)};
}
// Units a part: the batch's `total` over `once`, but of kPartFairUnits as long as `few` parts (one workgroup a CU) are left; where
// that gives parts of kPartLongUnits and more, over up to `extra`, so that uneven ends even out. (64 q4 sequences of 8 to 16
// thousand positions, 8 kv heads: 512 workgroups 212 us, 1536 201; one bf16 sequence of 100k: 512 78 us, 1536 85.)
ELM_HD int part_size(int total, const PartRule& r) {
  const int small = ceil_of(total, r.once), fair = ceil_of(total, r.few), least = ceil_of(total, r.extra);
  int per = fair < kPartFairUnits ? fair : kPartFairUnits;
  if (small > per) per = small;
  if (per > kPartLongUnits) per = kPartLongUnits;
  if (least > per) per = least;
  return per > r.least ? per : r.least;
}
// Parts of a sequence (one if it is empty), and where they begin: no divisions. The quotient is taken a 2^-20th low, so that a
// multiple of `per` units is not cut once more; a part of a very long sequence may then be longer than `per` by as much.
ELM_HD float part_inverse(int per) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_rcpf((float)per) * (1.f - 0x1p-20f);
#else
  return 1.f / (float)per * (1.f - 0x1p-20f);
#endif
}
ELM_HD int part_count(int units, float inverse) { return (int)((float)units * inverse) + 1; }
ELM_HD int part_begin(int units, int part, int parts) {  // of part `parts`: the end
  if (part == parts) return units;
#ifdef __HIP_DEVICE_COMPILE__
  const float each = (float)units * __builtin_amdgcn_rcpf((float)parts);
#else
  const float each = (float)units / (float)parts;
#endif
  const int at = (int)((float)part * each);
  return at < units ? at : units;
}

// ---------------------------------------------------------------- what a call has to satisfy

struct PagedFault {
  int code = ELMH_OK;
  const char* what = nullptr;
};

inline bool kv_head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 192 || hd == 256; }

inline PagedFault check_kv_shape(int dtype, int n_kv, int head_dim, int page_size) {
  if (dtype != ELMH_F32 && dtype != ELMH_F16 && dtype != ELMH_BF16 && !kv_quantized(dtype))
    return {ELMH_ERR_UNSUPPORTED, "cache type: f32, f16, bf16, q8 and q4 are held"};
  if (n_kv < 1 || n_kv > 1024) return {ELMH_ERR_ARG, "kv heads outside 1 .. 1024"};
  if (!kv_head_dim_ok(head_dim)) return {ELMH_ERR_UNSUPPORTED, "head_dim: 32, 64, 96, 128, 192 and 256 are held"};
  if (page_size < kPageStep || page_size % kPageStep || page_size > 4096)
    return {ELMH_ERR_ARG, "page_size: a multiple of 16 up to 4096"};
  return {};
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline PagedFault check_kv_pages(const elmh_kv_pages* p) {
  if (!p) return {ELMH_ERR_ARG, "null pages"};
  const PagedFault f = check_kv_shape(p->dtype, p->n_kv, p->head_dim, p->page_size);
  if (f.code) return f;
  if (p->n_pages < 1 || p->n_pages > INT32_MAX) return {ELMH_ERR_ARG, "n_pages outside 1 .. 2^31 - 1"};
  if (p->n_pages * p->n_kv > (int64_t(1) << 32) / (p->page_size / kPageStep) - 1)
    return {ELMH_ERR_ARG, "a pool of 2^36 rows or more"};
  if (!p->k || !p->v) return {ELMH_ERR_ARG, "null key or value pool"};
  if (!aligned16(p->k) || !aligned16(p->v)) return {ELMH_ERR_ARG, "pools start on 16 bytes"};
  if (kv_quantized(p->dtype)) {
    if (!p->k_scale || !p->v_scale) return {ELMH_ERR_ARG, "null scales of a quantized cache"};
    if (!aligned16(p->k_scale) || !aligned16(p->v_scale)) return {ELMH_ERR_ARG, "scales start on 16 bytes"};
  }
  return {};
}

inline PagedFault check_rope(const elmh_rope* r, int head_dim) {
  if (!r) return {};
  if (!r->cos || !r->sin) return {ELMH_ERR_ARG, "null rotary table"};
  if (r->max_pos < 1) return {ELMH_ERR_ARG, "rotary table without positions"};
  if (r->rot_dim < 2 || r->rot_dim % 2 || r->rot_dim > head_dim) return {ELMH_ERR_ARG, "rot_dim: even, 2 .. head_dim"};
  if (r->interleaved != 0 && r->interleaved != 1) return {ELMH_ERR_ARG, "interleaved: 0 or 1"};
  return {};
}

inline PagedFault check_table(const int32_t* table, int n_seqs, int max_pages, int page_size) {
  if (!table) return {ELMH_ERR_ARG, "null page table"};
  if (n_seqs < 1 || max_pages < 1) return {ELMH_ERR_ARG, "n_seqs and max_pages are at least 1"};
  if ((int64_t)max_pages * page_size > kMaxPositions) return {ELMH_ERR_ARG, "max_pages * page_size past 2^28 positions"};
  return {};
}

// n rows of n_kv heads: strides in values, 0 for the contiguous [n][n_kv][head_dim]
struct RowStrides {
  int64_t row = 0, head = 0;
};
inline RowStrides row_strides(int64_t row, int64_t head, int n_kv, int head_dim) {
  return {row ? row : (int64_t)n_kv * head_dim, head ? head : (int64_t)head_dim};
}
// written: the rows go to memory, so no two of them may share a value
inline PagedFault check_rows(int64_t n, int64_t row, int64_t head, int n_kv, int head_dim, bool written) {
  if (n < 1 || n > 1 << 23) return {ELMH_ERR_ARG, "rows outside 1 .. 2^23"};
  constexpr int64_t most = int64_t(1) << 40;
  if (row < 0 || head < 0 || row > most || head > most) return {ELMH_ERR_ARG, "row and head strides: 0 .. 2^40"};
  const RowStrides s = row_strides(row, head, n_kv, head_dim);
  const bool rows_apart = (n == 1 || s.row >= (n_kv - 1) * s.head + head_dim) && (n_kv == 1 || s.head >= head_dim);
  const bool heads_apart = (n_kv == 1 || s.head >= (n - 1) * s.row + head_dim) && (n == 1 || s.row >= head_dim);
  if (written && !rows_apart && !heads_apart) return {ELMH_ERR_ARG, "strides at which rows overlap"};
  return {};
}

inline PagedFault check_paged_rows(const float* k, const float* v, int64_t n, int64_t row, int64_t head,
                                   const elmh_kv_pages* pages, const int32_t* table, int n_seqs, int max_pages,
                                   const int32_t* pos, const int32_t* seq, const elmh_rope* rope, bool written) {
  if (!k || !v) return {ELMH_ERR_ARG, "null keys or values"};
  if (written && k == v) return {ELMH_ERR_ARG, "keys and values overlap"};
  PagedFault f = check_kv_pages(pages);
  if (!f.code) f = check_table(table, n_seqs, max_pages, pages->page_size);
  if (!f.code) f = check_rows(n, row, head, pages->n_kv, pages->head_dim, written);
  if (!f.code) f = check_rope(rope, pages->head_dim);
  if (f.code) return f;
  if (!pos) return {ELMH_ERR_ARG, "null positions"};
  if (!seq && n > n_seqs) return {ELMH_ERR_ARG, "without seq, row i is of sequence i: n <= n_seqs"};
  return {};
}

inline PagedFault check_paged_attention(const float* q, const float* out, int64_t q_row, int n_heads,
                                        const elmh_kv_pages* pages, const int32_t* table, int n_seqs, int max_pages,
                                        const int32_t* lens, int max_len, const elmh_rope* rope) {
  if (!q || !out || !lens) return {ELMH_ERR_ARG, "null q, out or lens"};
  PagedFault f = check_kv_pages(pages);
  if (!f.code) f = check_table(table, n_seqs, max_pages, pages->page_size);
  if (!f.code) f = check_rope(rope, pages->head_dim);
  if (f.code) return f;
  if (q == out) return {ELMH_ERR_ARG, "out may not overlap q"};
  if (n_heads < 1 || n_heads % pages->n_kv || n_heads / pages->n_kv > 256)
    return {ELMH_ERR_ARG, "n_heads: a multiple of the kv heads, at most 256 of each"};
  if (n_seqs > 4096) return {ELMH_ERR_ARG, "at most 4096 sequences a call"};
  if (q_row < 0 || q_row > (int64_t(1) << 40)) return {ELMH_ERR_ARG, "q_row: 0 .. 2^40"};
  if (max_len < 1 || max_len > (int64_t)max_pages * pages->page_size)
    return {ELMH_ERR_ARG, "max_len: 1 .. max_pages * page_size"};
  if ((int64_t)n_seqs * max_len > int64_t(1) << 35) return {ELMH_ERR_ARG, "n_seqs * max_len past 2^35 positions"};
  if (rope && max_len > rope->max_pos) return {ELMH_ERR_ARG, "max_len past the rotary table"};
  return {};
}

inline PagedFault check_rope_rows(const float* x, const float* y, int64_t T, int n_heads, int head_dim, int64_t x_row,
                                  int64_t y_row, const elmh_rope* rope, const int32_t* pos, int64_t pos0) {
  if (!x || !y || !rope) return {ELMH_ERR_ARG, "null x, y or rope"};
  if (T < 1 || T > (int64_t(1) << 24) || n_heads < 1 || n_heads > 4096) return {ELMH_ERR_ARG, "rows 1 .. 2^24, heads 1 .. 4096"};
  if (head_dim < 2 || head_dim > 1024 || head_dim % 2) return {ELMH_ERR_ARG, "head_dim: even, 2 .. 1024"};
  const PagedFault f = check_rope(rope, head_dim);
  if (f.code) return f;
  const int64_t width = (int64_t)n_heads * head_dim;
  if (x_row < 0 || y_row < 0 || x_row > (int64_t(1) << 40) || y_row > (int64_t(1) << 40))
    return {ELMH_ERR_ARG, "row strides: 0 .. 2^40"};
  if (T > 1 && y_row && y_row < width) return {ELMH_ERR_ARG, "y's rows overlap"};
  if (x == y && T > 1 && (x_row ? x_row : width) != (y_row ? y_row : width))
    return {ELMH_ERR_ARG, "in place: x and y have one stride"};
  if (!pos && (pos0 < 0 || pos0 + T > rope->max_pos)) return {ELMH_ERR_ARG, "positions past the rotary table"};
  return {};
}

inline PagedFault check_rope_table(const float* c, const float* s, int64_t pos0, int64_t n, int rot_dim, double theta,
                                   const elmh_rope_scaling* sc) {
  if (!c || !s) return {ELMH_ERR_ARG, "null cos or sin"};
  if (pos0 < 0 || n < 1 || pos0 > INT32_MAX || n > INT32_MAX || pos0 + n > INT32_MAX)
    return {ELMH_ERR_ARG, "positions 0 .. 2^31 - 2, at least one"};
  if (rot_dim < 2 || rot_dim % 2 || rot_dim > 1024) return {ELMH_ERR_ARG, "rot_dim: even, 2 .. 1024"};
  if (!(theta > 1.0) || !std::isfinite(theta)) return {ELMH_ERR_ARG, "theta: above 1 and finite"};
  if (!sc) return {};
  if (sc->kind != ELMH_ROPE_LINEAR && sc->kind != ELMH_ROPE_BANDS && sc->kind != ELMH_ROPE_YARN)
    return {ELMH_ERR_UNSUPPORTED, "scaling: linear, bands and yarn are known"};
  if (!(sc->factor >= 1.0) || !std::isfinite(sc->factor)) return {ELMH_ERR_ARG, "scaling factor: at least 1 and finite"};
  if (!(sc->magnitude > 0.0) || !std::isfinite(sc->magnitude)) return {ELMH_ERR_ARG, "magnitude: above 0 and finite"};
  if (sc->kind == ELMH_ROPE_LINEAR) return {};
  if (!(sc->orig_ctx >= 1.0) || !std::isfinite(sc->orig_ctx)) return {ELMH_ERR_ARG, "orig_ctx: at least 1 and finite"};
  if (!(sc->low > 0.0) || !(sc->high > sc->low) || !std::isfinite(sc->high)) return {ELMH_ERR_ARG, "low and high turns: 0 < low < high"};
  return {};
}

// ---------------------------------------------------------------- scaled rotary frequencies

// How the pair i's frequency f = theta^(-2 i / rot) is changed, as numbers that do not depend on i
struct RopeBand {
  int kind = 0;            // 0: none
  double factor = 1, magnitude = 1;
  double a = 0, b = 1;     // bands: keep = clamp(f * a - b); yarn: keep = 1 - clamp((i - a) * b)
};
inline RopeBand rope_band(int rot_dim, double theta, const elmh_rope_scaling* sc) {
  RopeBand r;
  if (!sc) return r;
  constexpr double kTwoPi = 6.283185307179586476925;
  r.kind = sc->kind;
  r.factor = sc->factor;
  r.magnitude = sc->magnitude;
  if (sc->kind == ELMH_ROPE_BANDS) {
    r.a = sc->orig_ctx / kTwoPi / (sc->high - sc->low);
    r.b = sc->low / (sc->high - sc->low);
  } else if (sc->kind == ELMH_ROPE_YARN) {
    // the (fractional) pair index that makes t turns over orig_ctx
    const auto pair = [&](double t) { return rot_dim * std::log(sc->orig_ctx / (kTwoPi * t)) / (2 * std::log(theta)); };
    const double lo = std::fmax(std::floor(pair(sc->high)), 0.0), hi = std::fmin(std::ceil(pair(sc->low)), rot_dim - 1.0);
    r.a = lo;
    r.b = 1.0 / std::fmax(hi - lo, 0.001);
  }
  return r;
}
ELM_HD double rope_scaled(const RopeBand& r, double f, int i) {
  if (r.kind == 0) return f;
  if (r.kind == ELMH_ROPE_LINEAR) return f / r.factor;
  double keep = r.kind == ELMH_ROPE_BANDS ? f * r.a - r.b : 1.0 - (i - r.a) * r.b;
  keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
  return f * (keep + (1.0 - keep) / r.factor);
}

}  // namespace elmh
