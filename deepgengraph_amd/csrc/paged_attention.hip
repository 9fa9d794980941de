// Attention over a paged key/value cache (dgg_attn_paged): decode rows, drafted tokens and prompt chunks of a ragged batch
// in one launch, optionally behind a prefix that all sequences share. paged.h has the division of the work.
//
//   scores = cap(q . k^T * scale), masked; p = softmax(scores); o = p . v
//
// Each unit is a workgroup of NW waves with 32 rows each over one slice of the keys, in tiles of 32: K and V rows go
// global -> registers -> LDS one tile ahead of the compute, then
//   S^T (32 keys x 32 rows) = K . Q^T     v_mfma_f32_32x32x16, A = K from the LDS, B = Q in registers
//   O^T (D x 32 rows)      += V^T . P^T   A = V^T by transposing LDS reads, B = P from the S^T accumulator
// with one running maximum and sum per row, in fp32; P is rounded to the storage type, as the matrix instruction takes it
// (its error is that of the output's own rounding, spread over the keys). Partials of split rows are merged by a second
// kernel.
//
// Keys that no row of the sequence may see (behind kv_len, before the window, on a page number outside the pool) are never
// multiplied: their rows are replaced by a visible key's, so what memory holds there does not matter.
#include <climits>

#include "common.h"

#include "attention_common.h"
#include "paged.h"

namespace {

using namespace dgg_attn;
using namespace dgg_paged;

// Registers: two waves per SIMD at head_dim 64 and 128, one at 256 (Q 64 + O 128 registers).
template <typename T, int D, int NW, bool SOFTCAP>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(D >= 256 ? 1 : 2)))
paged_attn_kernel(PagedParams p) {
  typedef typename T::scalar S;
  typedef typename T::vec8 V8;
  typedef typename T::vec4 V4;
  constexpr int BN = kTile;
  constexpr int KP = D + 8;             // padded row (elements): 16-byte shift per row for both read patterns
  constexpr int NKK = D / 16;           // MFMA k-steps over the head dim
  constexpr int NDB = D / 32;           // 32-wide head-dim blocks of O^T
  constexpr int NPK = BN / 16;          // MFMA k-steps over the keys of a tile in P.V
  constexpr int NT = 64 * NW;
  constexpr int LPR = D / 8;            // threads per key row: consecutive lanes read consecutive 16-byte chunks
  constexpr int RPI = NT / LPR;         // key rows per load instruction of the workgroup
  constexpr int CPT = BN / RPI;         // 16-byte chunks per thread per tile (K and V each)
  static_assert(CPT * RPI == BN && RPI * LPR == NT, "tile mapping");

  __shared__ __attribute__((aligned(16))) S Ks[BN][KP];
  __shared__ __attribute__((aligned(16))) S Vs[BN][KP];

  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.y;

  // This workgroup's unit.
  const Division dv = divide(p, lane);
  const int p_units = dv.p_rg * dv.p_ns;
  const bool prefix = (int)blockIdx.x < p_units;
  Place pl{};
  int row0, rows, slot, lo, hi, kslice, nslices;  // first row, rows (of the row space), keys of the row group
  if (prefix) {
    kslice = (int)blockIdx.x / dv.p_rg;
    const int rg = (int)blockIdx.x - kslice * dv.p_rg;
    nslices = dv.p_ns;
    row0 = rg * p.R;
    rows = p.T * p.G;
    slot = rg * dv.p_ns + kslice;
    lo = dv.p_lo;
    hi = p.P;
  } else {
    pl = find_place<true>(p, dv, (int)blockIdx.x - p_units, lane);
    if (pl.b < 0) return;
    const int nrg = row_groups(p, pl.s);
    kslice = pl.local / nrg;
    const int rg = pl.local - kslice * nrg;
    nslices = pl.ns;
    row0 = rg * p.R;
    rows = pl.s.n * p.G;
    slot = p.P > 0 || pl.ns > 1 ? p_units + pl.slot + rg * pl.ns + kslice : -1;
    // keys that any of these rows sees
    const int off = pl.s.kv - pl.s.n;
    lo = first_key(p, pl.s);
    hi = pl.s.kv;
    if (p.causal) hi = min(hi, (min(row0 + p.R, rows) - 1) / p.G + off + 1);
    if (p.window > 0) lo = max(lo, row0 / p.G + off - p.window + 1);
  }
  const int b_table = prefix ? 0 : pl.b;
  const int tile0 = lo / BN, tiles = key_tiles(lo, hi), per = ceil_div(tiles, nslices);
  const int t_begin = tile0 + min(tiles, kslice * per), t_end = tile0 + min(tiles, kslice * per + per);

  // This lane's row (query column of S^T): lanes r and r + 32 share it.
  const int rl = w * 32 + r;  // row within the row group
  const int row = row0 + rl;
  bool row_ok = row < rows;
  int tok = 0, qi = 0, qg = 0, kv = 0, n = 0, b = 0;
  if (row_ok) {
    const int i = row / p.G;
    qg = row - i * p.G;
    if (prefix) {
      tok = i;
      b = seq_of_token(p, tok);
      row_ok = b < p.B;
      if (row_ok) {
        const Seq s = load_seq(p, b);
        qi = tok - s.t0;
        n = s.n;
        kv = s.kv;
        row_ok = qi >= 0 && qi < n;
      }
    } else {
      qi = i;
      b = pl.b;
      tok = pl.s.t0 + i;
      n = pl.s.n;
      kv = pl.s.kv;
    }
  }
  const int h = hk * p.G + qg;
  const int64_t q_off = p.cu_q != nullptr ? tok * p.q_ss : b * p.q_sb + qi * p.q_ss;

  // Q fragment (B operand of S^T = K.Q^T): the row's head-dim elements 16kk + 8g .. +8.
  const S* qp = static_cast<const S*>(p.q) + (row_ok ? q_off + h * p.q_sh : 0);
  V8 qf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) qf[kk] = ld16<V8>(qp + 16 * kk + 8 * g);
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    asm volatile("" : "+v"(qf[kk]));
    if (!row_ok) qf[kk] = V8{};
  }

  // Keys the row sees: k_lo <= key <= k_hi.
  int k_hi = min(hi, kv) - 1, k_lo = lo;
  if (p.causal) k_hi = min(k_hi, qi + kv - n);
  if (p.window > 0) k_lo = max(k_lo, qi + kv - n - p.window + 1);
  if (!row_ok) k_hi = k_lo - 1;
  // Wave-uniform tile classes: a tile inside [lo_max, hi_min] is seen whole by every row of the wave (a row with no key
  // in the unit makes every tile masked; lanes past the last row, whose results are dropped, do not count); a tile
  // outside [lo_min, hi_max] is seen by none.
  const bool empty = k_hi < k_lo;
  const int lo_max = wave_max_i(!row_ok ? INT_MIN : empty ? INT_MAX : k_lo);
  const int hi_min = wave_min_i(!row_ok ? INT_MAX : empty ? INT_MIN : k_hi);
  const int lo_min = wave_min_i(row_ok && !empty ? k_lo : INT_MAX);
  const int hi_max = wave_max_i(row_ok && !empty ? k_hi : INT_MIN);

  // Page numbers: lane l holds those of granule gbase + l (64 granules are 32 tiles), as element offsets of the granule's
  // first K and V row (negative: no such page); the next 64 are requested when these begin to be used.
  const int32_t* trow = p.table + b_table * p.table_sb;
  const int g_last = max(0, p.cap / kGranule - 1);
  auto page_of = [&](int gi) { return trow[min(gi, g_last) / p.gpp]; };
  auto offsets = [&](int gi, int page, int64_t& ko, int64_t& vo) {
    const int in = (min(gi, g_last) % p.gpp) * kGranule;
    const bool ok = page >= 0 && page < p.num_pages;
    ko = ok ? page * p.k_sp + in * p.k_ss : -1;
    vo = ok ? page * p.v_sp + in * p.v_ss : -1;
  };
  int gbase = 2 * t_begin;
  int64_t ko_l = -1, vo_l = -1;
  int page_next = 0;
  if (t_begin < t_end) {
    offsets(gbase + lane, page_of(gbase + lane), ko_l, vo_l);
    page_next = page_of(gbase + 64 + lane);
  }
  auto lane64 = [&](int64_t x, int at) {
    const unsigned lo32 = __builtin_amdgcn_readlane((int)(x & 0xffffffff), at);
    const int hi32 = __builtin_amdgcn_readlane((int)(x >> 32), at);
    return (int64_t)hi32 << 32 | lo32;
  };

  // Load i of a tile: thread tid reads 16-byte chunk tid % LPR of tile row i * RPI + tid / LPR, so one wave instruction
  // covers 64 / LPR whole rows. A K / V row is read once by a decode unit: the loads are non-temporal.
  const int krow = tid / LPR, c0 = tid % LPR;
  const S* kp = static_cast<const S*>(p.k) + hk * p.k_sh + c0 * 8;
  const S* vp = static_cast<const S*>(p.v) + hk * p.v_sh + c0 * 8;
  V8 kreg[CPT], vreg[CPT];
  int holes = 0;  // of the tile in the registers: bit 0 / 1, its first / second granule is no page; 3: nothing to see
  auto load = [&](int t) {
    if (2 * t - gbase >= 64) {
      gbase += 64;
      offsets(gbase + lane, page_next, ko_l, vo_l);
      page_next = page_of(gbase + 64 + lane);
    }
    const int at = 2 * t - gbase, kt = t * BN;
    const int64_t k0 = lane64(ko_l, at), k1 = lane64(ko_l, at + 1);
    const int64_t v0 = lane64(vo_l, at), v1 = lane64(vo_l, at + 1);
    holes = (k0 < 0 ? 1 : 0) | (k1 < 0 ? 2 : 0);
    const int a = max(kt, lo) - kt, z = min(kt + BN, hi) - 1 - kt;  // rows of the tile that are keys of the unit
    if (holes == 0 && a == 0 && z == BN - 1) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        const int rr = i * RPI + krow, in = rr & (kGranule - 1);
        const bool second = rr >= kGranule;
        kreg[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(kp + (second ? k1 : k0) + in * p.k_ss));
        vreg[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(vp + (second ? v1 : v0) + in * p.v_ss));
      }
      return;
    }
    // An edge tile, or one with a hole: rows that are no key read one that is.
    if (z < kGranule) holes |= 2;
    if (a >= kGranule) holes |= 1;
    if (holes == 3) return;
    const int spare = (holes & 1) ? max(a, kGranule) : a;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      int rr = i * RPI + krow;
      const bool ok = rr >= a && rr <= z && !(holes & (rr >= kGranule ? 2 : 1));
      rr = ok ? rr : spare;
      const int in = rr & (kGranule - 1);
      const bool second = rr >= kGranule;
      kreg[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(kp + (second ? k1 : k0) + in * p.k_ss));
      vreg[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(vp + (second ? v1 : v0) + in * p.v_ss));
    }
  };
  auto store = [&]() {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      *reinterpret_cast<V8*>(&Ks[i * RPI + krow][c0 * 8]) = kreg[i];
      *reinterpret_cast<V8*>(&Vs[i * RPI + krow][c0 * 8]) = vreg[i];
    }
  };

  f32x16 oacc[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) oacc[i] = f32x16{};
  float m_run = -INFINITY;  // reference maximum (value units)
  float l_part[4] = {0.f, 0.f, 0.f, 0.f};
  const float c = score_coeff<SOFTCAP, 0>(p.s);
  const int tr_krow = (lane & 15) >> 2;                         // key row within a group of 4
  const int tr_dcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);  // head-dim column within a 32-wide block

  auto tile = [&](const int kt, const int hole, auto masked) {
    f32x16 sacc = f32x16{};
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const V8 a = *reinterpret_cast<const V8*>(&Ks[r][16 * kk + 8 * g]);
      sacc = mfma32(a, qf[kk], sacc);
    }
    // element j holds key kt + 8*(j/4) + 4g + j%4
    const int rel_hi = k_hi - (kt + 4 * g), rel_lo = k_lo - (kt + 4 * g);
    float mloc = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float x = score_value<T, SOFTCAP, 0>(sacc[j], p.s);
      if constexpr (decltype(masked)::value) {
        const int o = 8 * (j >> 2) + (j & 3);
        x = (o <= rel_hi && o >= rel_lo && !(hole & (j < 8 ? 1 : 2))) ? x : -INFINITY;
      }
      sacc[j] = x;
      mloc = fmaxf(mloc, x);
    }
    mloc = half_swap_max(mloc);
    const float m_new = fmaxf(m_run, mloc);
    const bool need = m_new * c > m_run * c + kRescaleThreshold;
    if (__any(need)) {
      const float alpha = need ? fast_exp2((m_run - m_new) * c) : 1.0f;
      if (need) m_run = m_new;
#pragma unroll
      for (int i = 0; i < 4; ++i) l_part[i] *= alpha;
#pragma unroll
      for (int i = 0; i < NDB; ++i) oacc[i] *= alpha;
    }
    const float mc = m_run == -INFINITY ? 0.f : m_run * c;
#pragma unroll
    for (int kk = 0; kk < NPK; ++kk) {
      f32x8 pv;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float pe = fast_exp2(fmaf(sacc[8 * kk + e], c, -mc));
        l_part[e & 3] += pe;
        pv[e] = pe;
      }
      const V8 pb = from_f32x8<V8>(pv);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        // A = V^T rows db*32 + r, keys 16kk + 4g + {0..3} and 16kk + 8 + 4g + {0..3} (the P operand's key order)
        const S* vrow = &Vs[16 * kk + 4 * g + tr_krow][db * 32 + tr_dcol];
        const V4 lo4 = tr_read(vrow);
        const V4 hi4 = tr_read(vrow + 8 * KP);
        oacc[db] = mfma32(__builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7), pb, oacc[db]);
      }
    }
  };

  if (t_begin < t_end) load(t_begin);
  for (int t = t_begin; t < t_end; ++t) {
    const int hole = holes;
    if (hole != 3) store();
    __syncthreads();
    if (t + 1 < t_end) load(t + 1);  // in flight during this tile's compute
    const int kt = t * BN;
    if (hole != 3 && kt <= hi_max && kt + BN - 1 >= lo_min) {
      if (hole == 0 && kt >= lo_max && kt + BN - 1 <= hi_min) tile(kt, 0, std::false_type{});
      else tile(kt, hole, std::true_type{});
    }
    __syncthreads();
  }

  const float l_tot = half_swap_sum((l_part[0] + l_part[1]) + (l_part[2] + l_part[3]));
  if (!row_ok) return;
  if (slot < 0) {
    const float inv = l_tot == 0.f ? 0.f : 1.0f / l_tot;  // a row that sees no key: o = 0, lse = -inf
    S* op = static_cast<S*>(p.o) + (p.cu_q != nullptr ? tok * p.o_ss : b * p.o_sb + qi * p.o_ss) + h * p.o_sh;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        V4 ov;
#pragma unroll
        for (int e = 0; e < 4; ++e) ov[e] = to_s<S>(oacc[db][4 * jj + e] * inv);
        *reinterpret_cast<V4*>(op + db * 32 + 8 * jj + 4 * g) = ov;
      }
    if (p.lse != nullptr && g == 0)
      p.lse[(int64_t)tok * p.Hq + h] = l_tot == 0.f ? -INFINITY : (m_run * c + fast_log2(l_tot)) * kLn2;
    return;
  }
  if (slot >= p.slots) return;  // (only where cu_q descends)
  // Partial of this unit for the lane's row: unnormalised O, maximum (exp2 domain), sum.
  const int64_t pidx = ((int64_t)slot * p.Hkv + hk) * p.rows_stride + rl;
  float* po = p.part_o + pidx * D;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj)
      *reinterpret_cast<f32x4*>(po + db * 32 + 8 * jj + 4 * g) =
          f32x4{oacc[db][4 * jj], oacc[db][4 * jj + 1], oacc[db][4 * jj + 2], oacc[db][4 * jj + 3]};
  if (g == 0) {
    p.part_ml[pidx * 2 + 0] = m_run == -INFINITY ? -INFINITY : m_run * c;
    p.part_ml[pidx * 2 + 1] = l_tot;
  }
}

// Joins the partials of a row: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, lse = (M + log2 L) ln 2, with the
// prefix slices first and then the sequence's own. One wave per row at a time: its lanes hold the head dim.
constexpr int kMergeThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(PagedParams p, int rows_per_wg) {
  typedef typename T::scalar S;
  constexpr int E = D / 64;  // elements per lane
  typedef float fE __attribute__((ext_vector_type(E)));
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int hk = blockIdx.y;
  const Division dv = divide(p, lane);
  const Place pl = find_place<false>(p, dv, blockIdx.x, lane);
  if (pl.b < 0 || (p.P == 0 && pl.ns == 1)) return;
  const int rows = min(pl.s.n * p.G - pl.local * p.R, p.R);
  const int p_units = dv.p_rg * dv.p_ns;
  const int slot0 = p_units + pl.slot + pl.local * pl.ns;
  if (slot0 + pl.ns > p.slots) return;  // (only where cu_q descends)
  for (int rl = blockIdx.z * rows_per_wg + wv; rl < min(rows, (int)(blockIdx.z + 1) * rows_per_wg);
       rl += kMergeThreads / 64) {
    const int row = pl.local * p.R + rl;
    const int qi = row / p.G, tok = pl.s.t0 + qi, h = hk * p.G + (row - qi * p.G);
    const int prow = tok * p.G + (row - qi * p.G);
    const int prg = prow / p.R, prl = prow - prg * p.R;
    const int n_all = dv.p_ns + pl.ns;
    auto index = [&](int i) {
      const int64_t s = i < dv.p_ns ? prg * dv.p_ns + i : slot0 + (i - dv.p_ns);
      return (s * p.Hkv + hk) * p.rows_stride + (i < dv.p_ns ? prl : rl);
    };
    float M = -INFINITY;
    for (int i = lane; i < n_all; i += 64) M = fmaxf(M, p.part_ml[index(i) * 2]);
    M = wave_max(M);
    const float Mu = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    fE acc = {};
    for (int i = 0; i < n_all; ++i) {
      const int64_t x = index(i);
      const float wgt = fast_exp2(p.part_ml[x * 2] - Mu);
      L = fmaf(wgt, p.part_ml[x * 2 + 1], L);
      acc += wgt * *reinterpret_cast<const fE*>(p.part_o + x * D + lane * E);
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    S* op = static_cast<S*>(p.o) + (p.cu_q != nullptr ? tok * p.o_ss : pl.b * p.o_sb + qi * p.o_ss) + h * p.o_sh + lane * E;
    if constexpr (E == 1) {
      op[0] = to_s<S>(acc[0] * inv);
    } else {
      typedef S sE __attribute__((ext_vector_type(E)));
      sE ov;
#pragma unroll
      for (int e = 0; e < E; ++e) ov[e] = to_s<S>(acc[e] * inv);
      *reinterpret_cast<sE*>(op) = ov;
    }
    if (p.lse != nullptr && lane == 0)
      p.lse[(int64_t)tok * p.Hq + h] = L == 0.f ? -INFINITY : (M + fast_log2(L)) * kLn2;
  }
}

// The host's part of the division.
struct HostPlan {
  int nw, R, rows_stride, target, min_slice, grid_units, slots, merge_units;
};
HostPlan host_plan(int64_t B, int64_t T, bool ragged, int64_t Hq, int64_t Hkv, int64_t D, int64_t P) {
  HostPlan h{};
  const int64_t G = Hq / Hkv, Sq = B > 0 ? T / B : 0;
  const int64_t most = (ragged ? T : Sq) * G;             // most rows that a sequence can have
  const int64_t mean = B > 0 ? (T * G + B - 1) / B : 0;   // rows of the average one
  const int64_t typical = ragged ? std::max<int64_t>(mean, 1) : most;
  h.nw = std::max<int64_t>(typical, P > 0 ? std::min<int64_t>(T * G, 64) : 0) <= 32 ? 1 : typical <= 64 ? 2 : 4;
  if (P > 0 && T * G > 64) h.nw = 4;
  if (D == 256 && h.nw == 1) h.nw = 2;
  h.R = 32 * h.nw;
  h.rows_stride = (int)std::min<int64_t>(h.R, P > 0 ? T * G : most);
  h.target = (int)std::max<int64_t>(1024, Hkv);
  h.min_slice = 2;
  const int64_t nrg = ragged ? T * G / h.R + std::min(B, T) : B * ((Sq * G + h.R - 1) / h.R);
  const int64_t p_rg = P > 0 ? (T * G + h.R - 1) / h.R : 0;
  h.merge_units = (int)nrg;
  h.grid_units = (int)(h.target / Hkv + nrg + p_rg);
  h.slots = P > 0 ? h.grid_units : (int)(2 * h.target / Hkv);
  return h;
}

template <typename T, int D, int NW>
void launch_nw(const PagedParams& p, const HostPlan& h, hipStream_t st) {
  const dim3 grid(h.grid_units, p.Hkv);
  if (p.s.softcap > 0.f)
    hipLaunchKernelGGL((paged_attn_kernel<T, D, NW, true>), grid, dim3(64 * NW), 0, st, p);
  else
    hipLaunchKernelGGL((paged_attn_kernel<T, D, NW, false>), grid, dim3(64 * NW), 0, st, p);
  const int rpw = h.rows_stride <= 32 ? 4 : 32;
  hipLaunchKernelGGL((paged_merge_kernel<T, D>), dim3(h.merge_units, p.Hkv, (h.rows_stride + rpw - 1) / rpw),
                     dim3(kMergeThreads), 0, st, p, rpw);
}
template <typename T, int D>
void launch(const PagedParams& p, const HostPlan& h, hipStream_t st) {
  if (h.nw == 4) return launch_nw<T, D, 4>(p, h, st);
  if (h.nw == 2) return launch_nw<T, D, 2>(p, h, st);
  if constexpr (D < 256) launch_nw<T, D, 1>(p, h, st);
}

int check_sizes(const char* op, int64_t B, int64_t T, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix) {
  DGG_REQUIRE(B >= 0 && B <= 4096 && T >= 0 && T < (1 << 24), DGG_ERR_SHAPE,
              "%s: bad sizes (B=%lld of at most 4096, %lld tokens of fewer than 2^24)", op, (long long)B, (long long)T);
  DGG_REQUIRE(Sq >= 0 && (Sq == 0 || Sq * B == T), DGG_ERR_SHAPE, "%s: %lld tokens are not %lld sequences of %lld", op,
              (long long)T, (long long)B, (long long)Sq);
  DGG_REQUIRE(Hq > 0 && Hkv > 0 && Hq <= 1024 && Hq % Hkv == 0, DGG_ERR_SHAPE, "%s: bad head counts (Hq=%lld Hkv=%lld)",
              op, (long long)Hq, (long long)Hkv);
  DGG_REQUIRE(T * (Hq / Hkv) < (1 << 30), DGG_ERR_SHAPE, "%s: too many query rows", op);
  DGG_REQUIRE(D == 64 || D == 128 || D == 256, DGG_ERR_UNSUPPORTED, "%s: head_dim %lld not supported (64, 128, 256)",
              op, (long long)D);
  DGG_REQUIRE(prefix >= 0, DGG_ERR_SHAPE, "%s: prefix_len must be >= 0 (got %lld)", op, (long long)prefix);
  return DGG_OK;
}

}  // namespace

extern "C" int64_t dgg_attn_paged_workspace_bytes(int64_t B, int64_t T, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D,
                                                  int64_t prefix_len) {
  if (check_sizes("attn_paged_workspace_bytes", B, T, Sq, Hq, Hkv, D, prefix_len)) return -1;
  if (B == 0 || T == 0) return 0;
  const HostPlan h = host_plan(B, T, Sq == 0, Hq, Hkv, D, prefix_len);
  return (int64_t)h.slots * Hkv * h.rows_stride * (D + 2) * (int64_t)sizeof(float);
}

extern "C" int dgg_attn_paged(const void* q, const void* k_pages, const void* v_pages, void* o, float* lse,
                              const int32_t* block_table, const int32_t* kv_lens, const int32_t* cu_q, void* workspace,
                              int64_t workspace_bytes, int64_t B, int64_t T, int64_t Sq, int64_t Hq, int64_t Hkv,
                              int64_t D, int64_t num_pages, int64_t page_size, int64_t table_width, int64_t prefix_len,
                              const int64_t* strides, float scale, float softcap, int64_t window, uint32_t flags,
                              int dtype, void* stream) {
  const char* op = "attn_paged";
  DGG_REQUIRE(dtype == DGG_F16 || dtype == DGG_BF16, DGG_ERR_DTYPE, "%s: dtype code %d not supported (f16 or bf16)", op,
              dtype);
  if (int rc = check_sizes(op, B, T, Sq, Hq, Hkv, D, prefix_len)) return rc;
  DGG_REQUIRE((cu_q == nullptr) == (Sq > 0) || T == 0, DGG_ERR_SHAPE,
              "%s: give cu_q, or Sq tokens for every sequence, and not both", op);
  DGG_REQUIRE(num_pages >= 0 && num_pages < (1ll << 31), DGG_ERR_SHAPE, "%s: bad page count %lld", op,
              (long long)num_pages);
  DGG_REQUIRE(page_size > 0 && page_size % dgg_paged::kGranule == 0 && page_size <= (1 << 20), DGG_ERR_SHAPE,
              "%s: page_size %lld must be a multiple of %d of at most 2^20", op, (long long)page_size,
              dgg_paged::kGranule);
  DGG_REQUIRE(table_width >= 0 && table_width * page_size < (1ll << 30), DGG_ERR_SHAPE,
              "%s: a block table row of %lld pages of %lld is too long", op, (long long)table_width,
              (long long)page_size);
  DGG_REQUIRE(prefix_len % page_size == 0 && prefix_len <= table_width * page_size, DGG_ERR_SHAPE,
              "%s: prefix_len %lld must be whole pages of the block table", op, (long long)prefix_len);
  DGG_REQUIRE(std::isfinite(scale) && scale > 0.f, DGG_ERR_SHAPE, "%s: scale must be finite and > 0", op);
  DGG_REQUIRE(std::isfinite(softcap) && softcap >= 0.f, DGG_ERR_SHAPE, "%s: softcap must be finite and >= 0", op);
  DGG_REQUIRE(window >= 0, DGG_ERR_SHAPE, "%s: window must be >= 0 (got %lld)", op, (long long)window);
  DGG_REQUIRE((flags & ~DGG_ATTN_CAUSAL) == 0, DGG_ERR_UNSUPPORTED, "%s: flags 0x%x not supported", op, flags);
  DGG_REQUIRE(strides != nullptr, DGG_ERR_NULL, "%s: strides is NULL", op);
  for (int i = 0; i < 12; ++i)
    DGG_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, DGG_ERR_STRIDE,
                "%s: stride[%d] = %lld must be a non-negative multiple of 8 elements", op, i, (long long)strides[i]);
  DGG_REQUIRE(strides[12] >= 0, DGG_ERR_STRIDE, "%s: the block table's row stride is negative", op);
  if (B == 0 || T == 0) return DGG_OK;
  DGG_REQUIRE(q && o && kv_lens, DGG_ERR_NULL, "%s: null q/o/kv_lens pointer", op);
  const int64_t cap = num_pages > 0 ? table_width * page_size : 0;  // without pages nobody holds a key
  DGG_REQUIRE(cap == 0 || (k_pages && v_pages && block_table), DGG_ERR_NULL, "%s: null k/v/block_table pointer", op);
  DGG_REQUIRE(dgg::aligned16(q) && dgg::aligned16(o) && dgg::aligned16(k_pages) && dgg::aligned16(v_pages), DGG_ERR_ALIGN,
              "%s: q/k/v/o must be 16-byte aligned", op);
  const HostPlan h = host_plan(B, T, Sq == 0, Hq, Hkv, D, prefix_len);
  const int64_t need = dgg_attn_paged_workspace_bytes(B, T, Sq, Hq, Hkv, D, prefix_len);
  DGG_REQUIRE(workspace_bytes >= need, DGG_ERR_WORKSPACE, "%s: the partials need %lld bytes, workspace is %lld", op,
              (long long)need, (long long)workspace_bytes);
  DGG_REQUIRE(workspace != nullptr, DGG_ERR_NULL, "%s: null workspace", op);
  DGG_REQUIRE(dgg::aligned16(workspace), DGG_ERR_ALIGN, "%s: workspace must be 16-byte aligned", op);

  PagedParams p{};
  p.s = dgg_attn::make_params(q, k_pages, v_pages, o, B, 0, 0, Hq, Hkv, D, scale, softcap, 0, 0);
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.o = o;
  p.lse = lse;
  p.table = block_table;
  p.kv_lens = kv_lens;
  p.cu_q = Sq > 0 ? nullptr : cu_q;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + (int64_t)h.slots * Hkv * h.rows_stride * D;
  p.q_sb = strides[0]; p.q_ss = strides[1]; p.q_sh = strides[2];
  p.k_sp = strides[3]; p.k_ss = strides[4]; p.k_sh = strides[5];
  p.v_sp = strides[6]; p.v_ss = strides[7]; p.v_sh = strides[8];
  p.o_sb = strides[9]; p.o_ss = strides[10]; p.o_sh = strides[11];
  p.table_sb = strides[12];
  p.B = (int)B;
  p.T = (int)T;
  p.Sq = (int)Sq;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.G = (int)(Hq / Hkv);
  p.num_pages = (int)num_pages;
  p.gpp = (int)(page_size / dgg_paged::kGranule);
  p.cap = (int)cap;
  p.P = (int)std::min(prefix_len, cap);
  p.causal = (flags & DGG_ATTN_CAUSAL) != 0;
  p.window = (int)std::min<int64_t>(window, 1 << 30);
  p.R = h.R;
  p.rows_stride = h.rows_stride;
  p.target = h.target;
  p.min_slice = h.min_slice;
  p.grid_units = h.grid_units;
  p.slots = h.slots;
  hipStream_t st = dgg::as_stream(stream);
  if (dtype == DGG_BF16) {
    if (D == 64) launch<BF16, 64>(p, h, st);
    else if (D == 128) launch<BF16, 128>(p, h, st);
    else launch<BF16, 256>(p, h, st);
  } else {
    if (D == 64) launch<F16, 64>(p, h, st);
    else if (D == 128) launch<F16, 128>(p, h, st);
    else launch<F16, 256>(p, h, st);
  }
  return dgg::check_launch(op);
}
