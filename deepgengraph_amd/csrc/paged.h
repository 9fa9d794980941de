// Attention over a paged key/value cache: launch parameters and the division of the work, shared by the attention kernels
// of paged_attention.hip and their merge.
//
// The batch is ragged: sequence b brings n_b query tokens (cu_q, or Sq each) and holds kv_b keys. The lengths are on the
// device and the grid on the host, so every workgroup divides the work itself, from the same numbers and with the same
// whole-number arithmetic:
//
//   rows    the n_b * G query rows that share a KV head (token-major: row r is token r / G, query head r % G), in row
//           groups of R; a row group is what one workgroup serves;
//   slices  the keys a row group sees, cut into ns_b slices, so that a unit (row group, slice) is at most `slice` key
//           tiles long; `slice` is the tiles of all units over the units wanted (target), so that long sequences get
//           many slices and short ones a single one;
//   prefix  the first P keys, when the batch shares them: row groups over the rows of the whole batch, slices alike.
//
// sum_b nrg_b * ceil(tiles_b / slice) <= target / Hkv + sum_b nrg_b, which bounds the grid; units of a sequence with one
// slice write the output itself, and the others' number is at most 2 * target / Hkv, which bounds the workspace.
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
  float* lse;             // [T, Hq], natural logarithm, or nullptr
  const int32_t* table;   // [B, W] page numbers, row stride table_sb
  const int32_t* kv_lens; // [B]
  const int32_t* cu_q;    // [B + 1] or nullptr: Sq tokens each
  float* part_o;          // [slots, Hkv, rows_stride, D] unnormalised outputs
  float* part_ml;         // [slots, Hkv, rows_stride, 2] row maximum (exp2 domain) and row sum
  int64_t q_sb, q_ss, q_sh;
  int64_t o_sb, o_ss, o_sh;
  int64_t k_sp, k_ss, k_sh;  // page, row in the page, head
  int64_t v_sp, v_ss, v_sh;
  int64_t table_sb;
  int B, T, Sq, Hq, Hkv, G;
  int num_pages, gpp, cap;  // pages, granules per page, keys that a table row can name
  int P;                    // shared prefix (a multiple of the page size)
  int causal, window;
  int R, rows_stride;       // rows per row group; rows of a partial (those that can be live)
  int min_slice;            // least tiles of a slice
  float per_target;         // (1 + 2^-11) Hkv / target: tiles of a unit, of all tiles of a KV head
  int grid_units, slots;
  dgg_attn::AttnParams s;   // scale and soft-cap constants (score_value)
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }
__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

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
__device__ __forceinline__ int row_groups(const PagedParams& p, const Seq& s) { return (s.n * p.G + p.R - 1) / p.R; }
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

// What the whole wave knows after a look at all lengths.
struct Division {
  int slice;     // most key tiles of a unit
  int p_lo;      // first prefix key that any row sees
  int p_rg, p_ns;  // row groups and slices of the prefix
};
// The place of a sequence's units: what=0 counts units, what=1 row groups.
struct Place {
  int b;          // sequence, or -1: none has this number
  Seq s;
  int ns;         // its slices
  int local;      // number within the sequence
  int slot;       // first partial slot of the sequence (it has nrg * ns of them), where it uses any
};

__device__ __forceinline__ int slices_of(const PagedParams& p, const Seq& s, int slice) {
  return max(1, ceil_div(key_tiles(first_key(p, s), s.kv), slice));
}

__device__ __forceinline__ Division divide(const PagedParams& p, int lane) {
  const int c = (p.B + 63) >> 6;
  float work = 0.f;  // (32 bits do: the quotient is rounded up, and every wave adds in the same order)
  int lo = p.P;
  for (int j = 0; j < c; ++j) {
    const int b = lane * c + j;
    if (b >= p.B) break;
    const Seq s = load_seq(p, b);
    work += (float)row_groups(p, s) * (float)key_tiles(first_key(p, s), s.kv);
    if (s.n > 0) lo = min(lo, p.window > 0 ? max(0, s.kv - s.n - p.window + 1) : 0);
  }
  work = wave_sum_f(work);
  Division d;
  d.p_lo = 0;
  d.p_rg = d.p_ns = 0;
  int p_tiles = 0;
  if (p.P > 0) {
    d.p_lo = wave_min_i(lo);
    d.p_rg = (p.T * p.G + p.R - 1) / p.R;
    p_tiles = key_tiles(d.p_lo, p.P);
    work += (float)d.p_rg * (float)p_tiles;
  }
  // At least work * Hkv / target: the sum of 4096 terms in fp32 is off by less than 2^-12 of it.
  const float per = work * p.per_target;
  d.slice = max(p.min_slice, (int)ceilf(min(per, 1e9f)));
  if (p.P > 0) d.p_ns = ceil_div(p_tiles, d.slice);
  return d;
}

// Finds unit number u (units: slices x row groups of a sequence) or row group number u (UNITS false) of the sequences.
template <bool UNITS>
__device__ __forceinline__ Place find_place(const PagedParams& p, const Division& d, int u, int lane) {
  const bool all_partial = p.P > 0;
  auto count = [&](const Seq& s, int& ns, int& slots) {
    const int nrg = row_groups(p, s);
    ns = slices_of(p, s, d.slice);
    slots = all_partial || ns > 1 ? nrg * ns : 0;
    return UNITS ? nrg * ns : nrg;
  };
  const int c = (p.B + 63) >> 6;
  int mine = 0, my_slots = 0;
  Seq s0{};
  int ns0 = 1;
  for (int j = 0; j < c; ++j) {
    const int b = lane * c + j;
    if (b >= p.B) break;
    const Seq s = load_seq(p, b);
    int ns, slots;
    mine += count(s, ns, slots);
    my_slots += slots;
    s0 = s;
    ns0 = ns;
  }
  Place r{};
  r.b = -1;
  int incl = wave_scan_add(mine), sincl = wave_scan_add(my_slots);
  unsigned long long hit = __ballot(u < incl);
  if (hit == 0) return r;
  int at = __ffsll(hit) - 1;
  int base = __builtin_amdgcn_readlane(incl - mine, at), sbase = __builtin_amdgcn_readlane(sincl - my_slots, at);
  r.b = at;
  if (c > 1) {  // lane j looks at the j-th of that lane's sequences (c <= 64: B <= 4096)
    const int b = at * c + lane;
    mine = my_slots = 0;
    if (lane < c && b < p.B) {
      s0 = load_seq(p, b);
      mine = count(s0, ns0, my_slots);
    }
    incl = wave_scan_add(mine);
    sincl = wave_scan_add(my_slots);
    hit = __ballot(u - base < incl);
    if (hit == 0) {  // (cannot be: the lane's sum exceeds u - base)
      r.b = -1;
      return r;
    }
    r.b = at * c;
    at = __ffsll(hit) - 1;
    r.b += at;
    base += __builtin_amdgcn_readlane(incl - mine, at);
    sbase += __builtin_amdgcn_readlane(sincl - my_slots, at);
  }
  r.s.t0 = __builtin_amdgcn_readlane(s0.t0, at);
  r.s.n = __builtin_amdgcn_readlane(s0.n, at);
  r.s.kv = __builtin_amdgcn_readlane(s0.kv, at);
  r.ns = __builtin_amdgcn_readlane(ns0, at);
  r.local = u - base;
  r.slot = sbase;
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
