// Attention over a paged key/value cache: launch parameters and the division of the work, shared by the attention
// kernels and the merge of paged_attention.hip.
//
// The batch is ragged: sequence b brings n_b query tokens (cu_q, or Sq each) and holds kv_b keys. The lengths are on
// the device and the grid on the host, so every workgroup divides the work itself, from the same numbers with the
// same arithmetic. All of it is per KV head; a sequence's n_b * G query rows that share the head are numbered
// token-major (row r is token r / G, query head r % G), its keys are counted in tiles of 128.
//
//   narrow  sequences of at most 32 rows. Their tiles, one sequence after the other, are cut into equal stretches,
//           one for each workgroup: a workgroup streams as many keys as any other, whatever the lengths are. A
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
  int narrow_wgs, narrow_most, narrow_slots, narrow_rows;  // workgroups among wide sequences, and at most
  int rows_per_merge;
  int places;               // workgroups that are resident at once
  int wide_target;          // wide units wanted, at most
  dgg_attn::AttnParams s;   // scale and soft-cap constants (score_value)
};

// Launch the kernels for p (paged_attention_d*.hip).
void launch_d64(const PagedParams& p, bool bf16, hipStream_t st);
void launch_d128(const PagedParams& p, bool bf16, hipStream_t st);
void launch_d256(const PagedParams& p, bool bf16, hipStream_t st);

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }
__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// gi / gpp for gi < 2^26 (the quotient of a number of 32 bits by multiplication: gpp_mul = ceil(2^(32 + shift) / gpp)
// is off by less than gpp * 2^-(32 + shift) of it, and shift is at least log2(gpp) - 6).
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

// Sums, extremes and inclusive prefix sums over a wave, on the DPP lane shifts (a sixth of the latency of
// ds_bpermute).
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

// What every wave finds out from all the lengths. Lane l looks at sequences l * c .. l * c + c - 1 (c = ceil(B /
// 64)); what it found is kept, so that looking up a sequence later takes a ballot and not a second look at the
// lengths.
struct Division {
  int slice;         // most key tiles of a wide unit
  int p_lo;          // first prefix key that any row sees
  int p_rg, p_ns;    // wide prefix: row groups and slices
  int p_tiles;       // narrow prefix: tiles
  int narrow;        // workgroups with narrow stretches
  int stretch;       // tiles of one
  int tiles;         // all narrow tiles
  bool invalid;      // the lengths make no sense
  // per lane: the last of its sequences, and its own and the running number of narrow tiles, wide units, partial slots
  Seq s;
  int my_tiles, my_units, my_slots, run_tiles, run_units, run_slots;
};
__device__ __forceinline__ int seq_tiles(const PagedParams& p, const Seq& s) {
  return max(1, key_tiles(first_key(p, s), s.kv));  // (a sequence without keys has an output, too)
}
__device__ __forceinline__ int wide_slices(const PagedParams& p, const Seq& s, int slice) {
  return ceil_div(seq_tiles(p, s), slice);
}
// Narrow tiles of a sequence, its wide units and their partial slots.
template <bool WIDE>
__device__ __forceinline__ void count_seq(const PagedParams& p, const Seq& s, int slice, int& tiles, int& units,
                                          int& slots) {
  tiles = units = slots = 0;
  if (s.n == 0) return;
  if (!is_wide(p, s)) {
    tiles = seq_tiles(p, s);
  } else if constexpr (WIDE) {
    const int ns = wide_slices(p, s, slice);
    units = row_groups(p, s.n * p.G) * ns;
    slots = p.P > 0 || ns > 1 ? units : 0;
  }
}
// WIDE false: nothing of the launch is wide.
template <bool WIDE>
__device__ __forceinline__ Division divide(const PagedParams& p, int lane) {
  const int c = (p.B + 63) >> 6;
  float work = 0.f, groups = 0.f;  // (32 bits do: the quotient is rounded up, and every wave adds in the same order)
  float tokens = 0.f;              // (fewer than 2^24: exact)
  int lo = p.P;
  Division d{};
  for (int j = 0; j < c; ++j) {
    const int b = lane * c + j;
    if (b >= p.B) break;
    d.s = load_seq(p, b);
    if (d.s.n == 0) continue;
    tokens += (float)d.s.n;
    if (!is_wide(p, d.s)) d.my_tiles += seq_tiles(p, d.s);
    else if (WIDE) {
      const float nrg = (float)row_groups(p, d.s.n * p.G);
      groups += nrg;
      work = fmaf(nrg, (float)seq_tiles(p, d.s), work);
    }
    lo = min(lo, p.window > 0 ? max(0, d.s.kv - d.s.n - p.window + 1) : 0);
  }
  // A cu_q that descends can name a token more than once, and more row groups than the grid and the workspace are
  // for: then nothing is computed.
  if (p.cu_q != nullptr && wave_sum_f(tokens) > (float)p.T) {
    d.s.n = d.my_tiles = 0;
    d.invalid = true;
    return d;
  }
  int p_tiles = 0;
  if (p.P > 0) {
    d.p_lo = wave_min_i(lo);
    p_tiles = key_tiles(d.p_lo, p.P);
  }
  d.run_tiles = wave_scan_add(d.my_tiles);
  d.tiles = last_lane(d.run_tiles);
  if (!WIDE || !p.prefix_wide) {
    d.p_tiles = p_tiles;
    d.tiles += p_tiles;
  }
  d.narrow = p.narrow_wgs;
  if constexpr (WIDE) {
    work = wave_sum_f(work);
    groups = wave_sum_f(groups);
    int units = p.wide_target;
    const bool only_prefix = groups == 0.f;  // no sequence is wide
    if (p.prefix_wide) {
      d.p_rg = row_groups(p, p.T * p.G);
      work = fmaf((float)d.p_rg, (float)p_tiles, work);
      groups += (float)d.p_rg;
    }
    // Then stretches and the prefix's units share the places by their tiles, so that everything is resident at once
    // and ends at about the same time. Measured on MI355X with the fixed numbers of host_plan / this, us: 64 decode
    // rows behind 8,192 keys, 32 / 8 heads of 128, 56 / 50, 16 heads of 64 62 / 48; 32 rows, 16 / 8 heads of 256, 57 /
    // 45; 64 x 1 or 2 tokens over up to 4,096 keys and no prefix, 16 heads of 64, 123 / 93. Among wide sequences,
    // whose last row groups and slices are uneven, the same rule gains and loses (a step of 28 decode rows and 4
    // chunks 132 / 135, 27 and 5 of head_dim 256 140 / 148, 8 chunks of up to 256 tokens 43 / 39).
    if (only_prefix && d.tiles > 0) {
      const float part = (float)d.tiles / ((float)d.tiles + work);
      d.narrow = clampi((int)rintf((float)p.places * part), 1, min(p.places - 1, p.narrow_most));
      units = min(p.places - d.narrow, p.wide_target);
    }
    const float per_unit = (1.0f + 1.0f / 2048) / (float)units;
    // At least work / wide_target: the sum of 4096 terms in fp32 is off by less than 2^-12 of it. Where the row
    // groups alone are three quarters of the units wanted, only those half as long again as the mean are cut (4 x
    // 1,024 tokens over 4,096 keys, 16 heads of 64: 512 row groups, 672 wanted; 109 us with each cut in two, 98
    // without).
    const float per = work * per_unit;
    d.slice = max(1, (int)ceilf(min(groups * per_unit >= 0.75f ? 1.5f * per : per, 1e9f)));
    if (d.p_rg > 0) d.p_ns = ceil_div(p_tiles, d.slice);
    if (c == 1) {
      if (lane < p.B) {
        int tiles;
        count_seq<WIDE>(p, d.s, d.slice, tiles, d.my_units, d.my_slots);
      }
    } else {
      for (int j = 0; j < c && lane * c + j < p.B; ++j) {
        int tiles, units, slots;
        count_seq<WIDE>(p, load_seq(p, lane * c + j), d.slice, tiles, units, slots);
        d.my_units += units;
        d.my_slots += slots;
      }
    }
    d.run_units = wave_scan_add(d.my_units);
    d.run_slots = wave_scan_add(d.my_slots);
  }
  d.stretch = d.narrow > 0 ? ceil_div(d.tiles, d.narrow) : 0;
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

// Finds wide unit, narrow tile (those of sequences) or token number u.
template <bool WIDE, int BY>
__device__ __forceinline__ Place find_place(const PagedParams& p, const Division& d, int u, int lane) {
  const int c = (p.B + 63) >> 6;
  Place r{};
  r.b = -1;
  if (d.invalid) return r;
  auto hits = [&](const Seq& s, int run_tiles, int run_units) {
    return __ballot(BY == kToken ? s.n > 0 && u < s.t0 + s.n : u < (BY == kWideUnit ? run_units : run_tiles));
  };
  unsigned long long hit = hits(d.s, d.run_tiles, d.run_units);
  if (hit == 0 && (BY != kToken || c == 1)) return r;
  Seq s = d.s;
  int at = hit != 0 ? __ffsll(hit) - 1 : 0;
  int tile0 = __builtin_amdgcn_readlane(d.run_tiles - d.my_tiles, at);
  int unit0 = WIDE ? __builtin_amdgcn_readlane(d.run_units - d.my_units, at) : 0;
  int slot0 = WIDE ? __builtin_amdgcn_readlane(d.run_slots - d.my_slots, at) : 0;
  r.b = at;
  if (c > 1) {
    if constexpr (BY == kToken) {  // (a lane's last sequence may be empty: its end is the largest of the lane's)
      int end = 0;
      for (int j = 0; j < c && lane * c + j < p.B; ++j) {
        const Seq x = load_seq(p, lane * c + j);
        if (x.n > 0) end = x.t0 + x.n;
      }
      hit = __ballot(u < end);
      r.b = -1;
      if (hit == 0) return r;
      at = __ffsll(hit) - 1;
      tile0 = __builtin_amdgcn_readlane(d.run_tiles - d.my_tiles, at);
      if (WIDE) slot0 = __builtin_amdgcn_readlane(d.run_slots - d.my_slots, at);
    }
    // Lane j looks at the j-th of that lane's sequences (c <= 64: B <= 4096).
    const int first = at * c;
    int tiles = 0, units = 0, slots = 0;
    s = Seq{0, 0, 0};
    if (lane < c && first + lane < p.B) {
      s = load_seq(p, first + lane);
      count_seq<WIDE>(p, s, d.slice, tiles, units, slots);
    }
    const int rt = wave_scan_add(tiles) + tile0, ru = WIDE ? wave_scan_add(units) + unit0 : 0;
    const int rs = WIDE ? wave_scan_add(slots) + slot0 : 0;
    hit = hits(s, rt, ru);
    r.b = -1;
    if (hit == 0) return r;
    at = __ffsll(hit) - 1;
    r.b = first + at;
    tile0 = __builtin_amdgcn_readlane(rt - tiles, at);
    if (WIDE) unit0 = __builtin_amdgcn_readlane(ru - units, at);
    if (WIDE) slot0 = __builtin_amdgcn_readlane(rs - slots, at);
  }
  r.s.t0 = __builtin_amdgcn_readlane(s.t0, at);
  r.s.n = __builtin_amdgcn_readlane(s.n, at);
  r.s.kv = __builtin_amdgcn_readlane(s.kv, at);
  r.tile0 = tile0;
  r.slot0 = slot0;
  r.local = u - (BY == kToken ? r.s.t0 : BY == kWideUnit ? unit0 : tile0);
  if (BY == kToken && r.local < 0) r.b = -1;  // (only where cu_q leaves tokens out)
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
