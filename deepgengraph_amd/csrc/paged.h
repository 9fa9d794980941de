// Attention over a paged key/value cache: launch parameters and the division of the work, shared by the attention kernels
// and the merge of paged_attention.hip.
//
// The batch is ragged: sequence b brings n_b query tokens (cu_q, or Sq each) and holds kv_b keys. The lengths are on the
// device and the grid on the host, so every workgroup divides the work itself, from the same numbers with the same
// arithmetic. All of it is per KV head; a sequence's n_b * G query rows that share the head are numbered token-major (row r
// is token r / G, query head r % G), its keys are counted in tiles of 128.
//
//   narrow  sequences of at most 32 rows. Their tiles, one sequence after the other, are cut into `narrow_wgs` equal
//           stretches, one for each workgroup: a workgroup streams as many keys as any other, whatever the lengths are. A
//           stretch's part of a sequence is a segment; segment (workgroup i, sequence b) leaves its partial in slot i + b.
//   wide    sequences of more rows, in row groups of R. The keys a row group sees are cut into ns_b slices, so that a unit
//           (row group, slice) is at most `slice` tiles long: the tiles of all units over the units wanted (wide_target).
//           sum nrg_b * ceil(tiles_b / slice) <= wide_target + sum nrg_b bounds the grid; the units of row groups with more
//           than one slice, which leave partials, are fewer than 2 * wide_target.
//   prefix  the first P keys, when the batch shares them: the rows of the whole batch over those keys, narrow (the first
//           stretch of tiles) or wide (the first units) by their number. Then every unit leaves a partial.
//
// Rows whose keys are one unit are written by it; the merge joins the partials of the others.
#pragma once

#include "common.h"

#include "attention_common.h"

namespace dgg_paged {

constexpr int kTile = 128;    // keys per tile of the division
constexpr int kGranule = 16;  // keys that are sure to lie in one page, one after another

struct PagedParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;              // [T, Hq], natural logarithm, or nullptr
  const int32_t* table;    // [B, W] page numbers, row stride table_sb
  const int32_t* kv_lens;  // [B]
  const int32_t* cu_q;     // [B + 1] or nullptr: Sq tokens each
  float* wide_o;           // [wide_slots, Hkv, wide_rows, D] unnormalised outputs
  float* wide_ml;          // [wide_slots, Hkv, wide_rows, 2] row maximum (exp2 domain) and row sum
  float* narrow_o;         // [narrow_slots, Hkv, narrow_rows, D], and so on
  float* narrow_ml;
  int64_t q_sb, q_ss, q_sh;
  int64_t o_sb, o_ss, o_sh;
  int64_t k_sp, k_ss, k_sh;  // page, row in the page, head
  int64_t v_sp, v_ss, v_sh;
  int64_t table_sb;
  int B, T, Sq, Hq, Hkv, G;
  int num_pages, gpp, cap;  // pages, granules per page, keys that a table row can name
  uint32_t gpp_mul, gpp_shift;  // page_index
  int P;                    // shared prefix (a multiple of the page size)
  int causal, window;
  int log2_r;               // row group of wide units
  int prefix_wide;          // the prefix's rows are more than 32
  int wide_units, wide_slots, wide_rows;  // units in the grid; partial slots, and rows of one
  int narrow_wgs, narrow_slots, narrow_rows;
  int rows_per_merge;
  float per_wide;           // (1 + 2^-11) / wide_target
  dgg_attn::AttnParams s;   // scale and soft-cap constants (score_value)
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }
__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// gi / gpp for gi < 2^26 (the quotient of a number of 32 bits by multiplication: gpp_mul = ceil(2^(32 + shift) / gpp) is
// off by less than gpp * 2^-(32 + shift) of it, and shift is at least log2(gpp) - 6).
__device__ __forceinline__ int page_index(const PagedParams& p, int gi) {
  return p.gpp == 1 ? gi : (int)(__umulhi((uint32_t)gi, p.gpp_mul) >> p.gpp_shift);
}

struct Seq {
  int t0, n, kv;  // first token, tokens, keys
};
__device__ __forceinline__ Seq load_seq(const PagedParams& p, int b) {
  Seq s;
  if (p.cu_q != nullptr) {
    s.t0 = clampi(p.cu_q[b], 0, p.T);
    s.n = max(0, clampi(p.cu_q[b + 1], 0, p.T) - s.t0);
  } else {
    s.t0 = b * p.Sq;
    s.n = p.Sq;
  }
  s.kv = clampi(p.kv_lens[b], 0, p.cap);
  return s;
}
constexpr int kNarrowRows = 32;
__device__ __forceinline__ bool is_wide(const PagedParams& p, const Seq& s) { return s.n * p.G > kNarrowRows; }
__device__ __forceinline__ int row_groups(const PagedParams& p, int rows) {
  return (rows + (1 << p.log2_r) - 1) >> p.log2_r;
}
// First key behind the prefix that any row of the sequence sees.
__device__ __forceinline__ int first_key(const PagedParams& p, const Seq& s) {
  return p.window > 0 ? max(p.P, s.kv - s.n - p.window + 1) : p.P;
}
__device__ __forceinline__ int key_tiles(int lo, int hi) { return hi > lo ? (hi + kTile - 1) / kTile - lo / kTile : 0; }

// Sums, extremes and inclusive prefix sums over a wave, on the DPP lane shifts (a sixth of the latency of ds_bpermute).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or(int old, int x) {
  return __builtin_amdgcn_update_dpp(old, x, CTRL, ROWS, 0xf, false);
}
// op over lanes 0 .. l in lane l; `none` leaves the other operand as it is.
template <typename F>
__device__ __forceinline__ int wave_scan(int x, int none, F op) {
  x = op(x, dpp_or<0x111, 0xf>(none, x));  // row_shr:1
  x = op(x, dpp_or<0x112, 0xf>(none, x));  // row_shr:2
  x = op(x, dpp_or<0x114, 0xf>(none, x));  // row_shr:4
  x = op(x, dpp_or<0x118, 0xf>(none, x));  // row_shr:8
  x = op(x, dpp_or<0x142, 0xa>(none, x));  // row_bcast:15 into rows 1 and 3
  x = op(x, dpp_or<0x143, 0xc>(none, x));  // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }
__device__ __forceinline__ int wave_scan_add(int x) {
  return wave_scan(x, 0, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_min_i(int x) {
  return last_lane(wave_scan(x, 0x7fffffff, [](int a, int b) { return min(a, b); }));
}
__device__ __forceinline__ int wave_max_i(int x) {
  return last_lane(wave_scan(x, (int)0x80000000, [](int a, int b) { return max(a, b); }));
}
__device__ __forceinline__ float wave_sum_f(float x) {
  return __int_as_float(last_lane(wave_scan(__float_as_int(x), 0, [](int a, int b) {
    return __float_as_int(__int_as_float(a) + __int_as_float(b));
  })));
}

// What every wave finds out from all the lengths.
struct Division {
  int slice;         // most key tiles of a wide unit
  int p_lo;          // first prefix key that any row sees
  int p_rg, p_ns;    // wide prefix: row groups and slices
  int p_tiles;       // narrow prefix: tiles
  int stretch;       // tiles of a narrow workgroup
  int tiles;         // all narrow tiles
};
__device__ __forceinline__ int seq_tiles(const PagedParams& p, const Seq& s) {
  return max(1, key_tiles(first_key(p, s), s.kv));  // (a sequence without keys has an output, too)
}
__device__ __forceinline__ Division divide(const PagedParams& p, int lane) {
  const int c = (p.B + 63) >> 6;
  float work = 0.f;  // (32 bits do: the quotient is rounded up, and every wave adds in the same order)
  int narrow = 0, lo = p.P;
  for (int j = 0; j < c; ++j) {
    const int b = lane * c + j;
    if (b >= p.B) break;
    const Seq s = load_seq(p, b);
    if (s.n == 0) continue;
    if (is_wide(p, s)) work += (float)row_groups(p, s.n * p.G) * (float)seq_tiles(p, s);
    else narrow += seq_tiles(p, s);
    lo = min(lo, p.window > 0 ? max(0, s.kv - s.n - p.window + 1) : 0);
  }
  Division d{};
  int p_tiles = 0;
  if (p.P > 0) {
    d.p_lo = wave_min_i(lo);
    p_tiles = key_tiles(d.p_lo, p.P);
  }
  if (p.narrow_wgs > 0) {
    d.tiles = last_lane(wave_scan_add(narrow));
    if (!p.prefix_wide) {
      d.p_tiles = p_tiles;
      d.tiles += p_tiles;
    }
    d.stretch = ceil_div(d.tiles, p.narrow_wgs);
  }
  if (p.wide_units > 0) {
    work = wave_sum_f(work);
    if (p.prefix_wide) {
      d.p_rg = row_groups(p, p.T * p.G);
      work += (float)d.p_rg * (float)p_tiles;
    }
    // At least work / wide_target: the sum of 4096 terms in fp32 is off by less than 2^-12 of it.
    d.slice = max(1, (int)ceilf(min(work * p.per_wide, 1e9f)));
    d.p_ns = ceil_div(d.p_rg > 0 ? p_tiles : 0, d.slice);
  }
  return d;
}

enum PlaceBy { kWideUnit, kNarrowTile, kToken };
// A sequence and what comes before it.
struct Place {
  int b;       // sequence, or -1: none has this number
  Seq s;
  int local;   // the number less that of the sequence's first
  int tile0;   // narrow tiles before it
  int slot0;   // wide partial slots before it (behind the prefix's)
};
__device__ __forceinline__ int wide_slices(const PagedParams& p, const Seq& s, const Division& d) {
  return ceil_div(seq_tiles(p, s), d.slice);
}

// Finds wide unit, narrow tile (those of sequences) or token number u.
template <int BY>
__device__ __forceinline__ Place find_place(const PagedParams& p, const Division& d, int u, int lane) {
  auto count = [&](const Seq& s, int& tiles, int& slots) {
    tiles = slots = 0;
    if (s.n == 0) return 0;
    int units = 0;
    if (is_wide(p, s)) {
      if (p.wide_units > 0) {
        const int ns = wide_slices(p, s, d);
        units = row_groups(p, s.n * p.G) * ns;
        slots = p.P > 0 || ns > 1 ? units : 0;
      }
    } else {
      tiles = seq_tiles(p, s);
    }
    return BY == kWideUnit ? units : BY == kNarrowTile ? tiles : s.n;
  };
  const int c = (p.B + 63) >> 6;
  int mine = 0, my_tiles = 0, my_slots = 0;
  Seq s0{};
  for (int j = 0; j < c; ++j) {
    const int b = lane * c + j;
    if (b >= p.B) break;
    s0 = load_seq(p, b);
    int tiles, slots;
    mine += count(s0, tiles, slots);
    my_tiles += tiles;
    my_slots += slots;
  }
  Place r{};
  r.b = -1;
  int incl = wave_scan_add(mine);
  unsigned long long hit = __ballot(u < incl);
  if (hit == 0) return r;
  int at = __ffsll(hit) - 1;
  int base = __builtin_amdgcn_readlane(incl - mine, at);
  r.tile0 = BY == kNarrowTile ? base : __builtin_amdgcn_readlane(wave_scan_add(my_tiles) - my_tiles, at);
  r.slot0 = __builtin_amdgcn_readlane(wave_scan_add(my_slots) - my_slots, at);
  r.b = at;
  if (c > 1) {  // lane j looks at the j-th of that lane's sequences (c <= 64: B <= 4096)
    const int b = at * c + lane;
    mine = my_tiles = my_slots = 0;
    if (lane < c && b < p.B) {
      s0 = load_seq(p, b);
      mine = count(s0, my_tiles, my_slots);
    }
    incl = wave_scan_add(mine);
    hit = __ballot(u - base < incl);
    if (hit == 0) {  // (cannot be: the lane's sum exceeds u - base)
      r.b = -1;
      return r;
    }
    const int first = at * c;
    at = __ffsll(hit) - 1;
    r.b = first + at;
    base += __builtin_amdgcn_readlane(incl - mine, at);
    r.tile0 += __builtin_amdgcn_readlane(wave_scan_add(my_tiles) - my_tiles, at);
    r.slot0 += __builtin_amdgcn_readlane(wave_scan_add(my_slots) - my_slots, at);
  }
  r.s.t0 = __builtin_amdgcn_readlane(s0.t0, at);
  r.s.n = __builtin_amdgcn_readlane(s0.n, at);
  r.s.kv = __builtin_amdgcn_readlane(s0.kv, at);
  r.local = u - base;
  return r;
}

// The sequence of token t (the number of sequences that end at or before it), or B for a token behind the last.
__device__ __forceinline__ int seq_of_token(const PagedParams& p, int t) {
  if (p.cu_q == nullptr) return t / p.Sq;
  int lo = 0, hi = p.B;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

}  // namespace dgg_paged
