// Attention over a paged key/value cache (dgg_attn_paged): decode rows, drafted tokens and prompt chunks of a ragged
// batch in one launch, optionally behind a prefix that all sequences share. paged.h has the division of the work.
//
//   scores = cap(q . k^T * scale), masked; p = softmax(scores); o = p . v
//
// in tiles of keys that go straight from the pages to the LDS (global_load_lds, DmaLayout of attention_common.h):
//   S^T (32 keys x 32 rows) = K . Q^T     v_mfma_f32_32x32x16, A = K from the LDS, B = Q in registers
//   O^T (D x 32 rows)      += V^T . P^T   A = V^T by transposing LDS reads, B = P from the S^T accumulator
// with one running maximum and sum per row, in fp32; P is rounded to the storage type, as the matrix instruction
// takes it (its error is that of the output's own rounding, spread over the keys). Two ways:
//   narrow  up to 32 rows of a KV head: bound by the stream of keys and values. The waves share the rows and take the
//           32-key tiles in turn, each with buffers of its own and no barrier, and add their states at the end;
//   wide    more rows: bound by the matrix products. The waves share the tiles and have rows of their own.
// Batches that may hold both run in one launch of workgroups that can do either. Partials are joined by the merge.
//
// A granule is 16 keys, which lie in one page one after another. Granules that hold no key of the unit (behind kv_len,
// before the window, on a page number outside the pool) are zeros in the LDS and masked; rows of a granule that are no
// keys are replaced by one that is. What memory holds there does not matter.
#pragma once

#include <climits>

#include "common.h"

#include "attention_common.h"
#include "paged.h"

namespace {

using namespace dgg_attn;
using namespace dgg_paged;

// The launch parameters, read from the kernel's arguments anew: a part of the kernel that begins with this does not
// keep scalar registers for what other parts use (without it 80 to 150 of them spill).
__device__ __forceinline__ const PagedParams& fresh_params() {
  auto at = (const PagedParams __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const PagedParams*)at;
}

// A unit of work: rows and keys.
struct Unit {
  bool prefix;
  int b;          // sequence (prefix: 0, whose table it reads)
  Seq s;
  int row0, rows; // first row; rows of the row space (the sequence's, or the whole batch's)
  int lo, hi;     // keys of it that any row of the row group sees
  int k0, k1;     // keys of the unit (k0 a multiple of kTile); those of [lo, hi) count
  int slot;       // partial slot, or -1: the unit writes the output
};
// Keys that the rows row0 .. of the sequence see.
__device__ __forceinline__ void set_range(const PagedParams& p, Unit& u, int most_rows) {
  const int off = u.s.kv - u.s.n;
  u.lo = first_key(p, u.s);
  u.hi = u.s.kv;
  if (p.causal) u.hi = min(u.hi, (min(u.row0 + most_rows, u.rows) - 1) / p.G + off + 1);
  if (p.window > 0) u.lo = max(u.lo, u.row0 / p.G + off - p.window + 1);
}

// A query row of the unit, as a lane holds it.
struct Row {
  bool ok;
  int lse;          // index of the row in lse
  int64_t q, o;     // element offsets of the row in q and o
  int k_lo, k_hi;   // keys it sees: k_lo <= key <= k_hi
};
__device__ __forceinline__ Row find_row(const PagedParams& p, const Unit& u, int rl, int hk) {
  Row x{};
  const int row = u.row0 + rl;
  x.ok = row < u.rows;
  int i = 0, b = u.b, tok = 0, h = 0;
  Seq s = u.s;
  if (x.ok) {
    i = row / p.G;
    h = hk * p.G + (row - i * p.G);
    if (u.prefix) {
      tok = i;
      b = seq_of_token(p, i);
      x.ok = b < p.B;
      if (x.ok) {
        s = load_seq(p, b);
        i -= s.t0;
        x.ok = i >= 0 && i < s.n;
      }
    } else {
      tok = s.t0 + i;
    }
  }
  if (!x.ok) return Row{false, 0, 0, 0, 0, -1};
  x.q = (p.cu_q != nullptr ? tok * p.q_ss : b * p.q_sb + i * p.q_ss) + h * p.q_sh;
  x.o = (p.cu_q != nullptr ? tok * p.o_ss : b * p.o_sb + i * p.o_ss) + h * p.o_sh;
  x.lse = tok * p.Hq + h;
  x.k_hi = min(u.hi, s.kv) - 1;
  x.k_lo = u.lo;
  if (p.causal) x.k_hi = min(x.k_hi, i + s.kv - s.n);
  if (p.window > 0) x.k_lo = max(x.k_lo, i + s.kv - s.n - p.window + 1);
  return x;
}

__device__ __forceinline__ int64_t shfl64(int64_t x, int lane) {
  return (int64_t)__shfl((int)(x >> 32), lane, 64) << 32 | (uint32_t)__shfl((int)x, lane, 64);
}

// What the rows of a wave see together: a block of keys inside [lo_max, hi_min] is seen whole by every row (a row that
// sees no key makes every block masked; lanes without a row do not count), one outside [lo_min, hi_max] by none.
struct Seen {
  int lo_max, hi_min, lo_min, hi_max;
};
// row: first row of the wave (32 of them).
__device__ __forceinline__ Seen seen_by_wave(const PagedParams& p, const Unit& u, const Row& x, int row) {
  Seen v;
  if (!u.prefix) {  // the rows' tokens are i0 .. i1
    const int off = u.s.kv - u.s.n, last = min(row + 32, u.rows) - 1;
    const int i0 = row / p.G, i1 = last / p.G;
    v.lo_min = p.window > 0 ? max(u.lo, i0 + off - p.window + 1) : u.lo;
    v.lo_max = p.window > 0 ? max(u.lo, i1 + off - p.window + 1) : u.lo;
    v.hi_min = p.causal ? min(u.hi - 1, i0 + off) : u.hi - 1;
    v.hi_max = p.causal ? min(u.hi - 1, i1 + off) : u.hi - 1;
    if (last < row) v = Seen{INT_MAX, INT_MIN, INT_MAX, INT_MIN};  // no row: nothing is full, nothing seen
    return v;
  }
  const bool empty = x.k_hi < x.k_lo;
  v.lo_max = __any(x.ok) ? wave_max_i(!x.ok ? INT_MIN : empty ? INT_MAX : x.k_lo) : INT_MAX;
  v.hi_min = wave_min_i(!x.ok ? INT_MAX : empty ? INT_MIN : x.k_hi);
  v.lo_min = wave_min_i(x.ok && !empty ? x.k_lo : INT_MAX);
  v.hi_max = wave_max_i(x.ok && !empty ? x.k_hi : INT_MIN);
  return v;
}

// The pages of 64 granules, one per lane, and which of the granules hold a key of the unit. The page numbers of the
// next 64 are requested when these are taken up, so that their latency is not waited for.
struct Granules {
  const int32_t* row;  // the sequence's row of the table
  int page, next;
  uint64_t live;       // bit l: the granule of lane l holds a key
  __device__ __forceinline__ int page_of(const PagedParams& p, int gi) {
    return row[page_index(p, min(gi, p.cap / kGranule - 1))];
  }
  // Takes up granule gi (per lane) with its page number in `next`, and requests that of gi_next.
  __device__ __forceinline__ void take(const PagedParams& p, const Unit& u, int gi, int gi_next) {
    page = next;
    next = page_of(p, gi_next);
    const int key = gi * kGranule;
    live = __ballot(page >= 0 && page < p.num_pages && key + kGranule > u.lo && key < min(u.hi, u.k1));
  }
  // Byte offset of the first row of granule gi, which lane `at` holds.
  __device__ __forceinline__ int64_t offset(const PagedParams& p, int gi, int at, int64_t sp, int64_t ss) const {
    const int pg = __builtin_amdgcn_readlane(page, at);
    const int in = (gi - page_index(p, gi) * p.gpp) * kGranule;
    return 2 * (pg * sp + in * ss);
  }
};

// dma16 (attention_common.h), with the non-temporal hint for NT: rows that one workgroup reads once.
template <bool NT>
__device__ __forceinline__ void copy16(uint32_t lds, const void* sbase, uint32_t voff) {
  if constexpr (NT)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(voff), "s"(sbase)
                 : "memory", "m0");
  else
    dma16(lds, sbase, voff);
}

// Copies one granule (16 rows of D) of K or V to `lds`, the place of its first 4- or 8-row group. kWhole: every row
// is a key. Otherwise rows outside [first, last] are replaced by the nearest that is inside.
template <int D, bool NT>
struct GranuleCopy {
  typedef DmaLayout<D> L;
  static constexpr int LOADS = kGranule / L::RPI;  // direct loads per granule
  uint32_t voff[L::NV];  // lane constants: row within the load's group, and the chunk that the layout puts there
  // D == 64: the swizzle depends on the 8-row group's number, whose parity is that of the load within the granule.
  static __device__ __forceinline__ int vi(int i) { return D == 64 ? i & 1 : i % L::IPG; }
  __device__ __forceinline__ void init(int lane, int64_t ss_b) {
    const int lrow = lane / L::LPR;
#pragma unroll
    for (int i = 0; i < L::NV; ++i) {
      voff[i] = (uint32_t)((D == 64 ? lrow : i * L::RPI + lrow) * ss_b) + chunk(lane, i);
      asm volatile("" : "+v"(voff[i]));
    }
  }
  // (the swizzle looks at the row within a granule only)
  static __device__ __forceinline__ uint32_t chunk(int lane, int i) {
    return (uint32_t)((lane % L::LPR) ^ L::swizzle(i * L::RPI + lane / L::LPR)) * 16u;
  }
  static __device__ __forceinline__ uint32_t place(int i) {
    return (uint32_t)((i / L::IPG) * L::GROUP_B + (i % L::IPG) * L::RPI * L::ROW_B);
  }
  __device__ __forceinline__ void one(uint32_t lds, const char* base, int64_t ss_b, int i) const {
    copy16<NT>(lds + place(i), base + (int64_t)(D == 64 ? i * L::RPI : (i / L::IPG) * L::GR) * ss_b, voff[vi(i)]);
  }
  __device__ __forceinline__ void whole(uint32_t lds, const char* base, int64_t ss_b) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) one(lds, base, ss_b, i);
  }
  static __device__ __forceinline__ void part(uint32_t lds, const char* base, int64_t ss_b, int first, int last, int lane) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = clampi(i * L::RPI + lane / L::LPR, first, last);
      dma16(lds + place(i), base + (row * ss_b + chunk(lane, vi(i))));
    }
  }
  static __device__ __forceinline__ void zero(uint32_t lds, int lane) {
    typedef float __attribute__((ext_vector_type(4))) f4;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      *reinterpret_cast<f4 __attribute__((address_space(3)))*>((lds_char*)(size_t)(lds + place(i) + 16 * lane)) = f4{};
  }
};

// LDS addresses of a tile's fragments, per lane. K fragment kk of the 32-key block at row 0: k[ki(kk)] + ko(kk). V
// transposing read of keys 16kk + 4g + .. (hi: + 8), head-dim block db: v[vb(db, hi)] + vo(kk, hi).
template <int D>
struct Fragments {
  typedef DmaLayout<D> L;
  static constexpr int NK = D == 64 ? D / 16 : D / 32, NV = D == 64 ? 2 * (D / 32) : D / 32;
  uint32_t k[NK], v[NV];
  static constexpr int ki(int kk) { return D == 64 ? kk : kk >> 1; }
  static constexpr int ko(int mb, int kk) { return mb * (32 / L::GR) * L::GROUP_B + (D == 64 ? 0 : 32 * (kk & 1)); }
  static constexpr int vb(int db, int hi) { return D == 64 ? 2 * db + hi : db; }
  static constexpr int vo(int kk, int hi) { return kk * (16 / L::GR) * L::GROUP_B + hi * (8 / L::GR) * L::GROUP_B; }
  // k_at, v_at: where the tile's K and V rows begin
  __device__ __forceinline__ void init(int lane, uint32_t k_at, uint32_t v_at) {
    const int r = lane & 31, g = lane >> 5, m4 = (lane & 15) >> 2, m3 = lane & 3;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int chunk = D == 64 ? 2 * i + g : 4 * i;  // (D >= 128: g and kk & 1 do not meet the swizzled bits)
      k[i] = k_at + (uint32_t)((r / L::GR) * L::GROUP_B + (r % L::GR) * L::ROW_B + 16 * (chunk ^ L::swizzle(r)) +
                               (D == 64 ? 0 : 16 * g));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int row = 4 * g + m4 + (D == 64 ? 8 * (i & 1) : 0);  // hi reads of D == 64 swizzle differently
      const int chunk = 4 * (D == 64 ? i >> 1 : i) + 2 * ((lane >> 4) & 1) + (m3 >> 1);
      v[i] = v_at + (uint32_t)(((row & 7) / L::GR) * L::GROUP_B + (row % L::GR) * L::ROW_B +
                               16 * (chunk ^ L::swizzle(row)) + 8 * (m3 & 1));
    }
  }
};

// Running softmax state of a wave's 32 rows (lanes r and r + 32 share row r).
template <int D>
struct State {
  f32x16 o[D / 32];
  float m;      // reference maximum (value units)
  float l[2];   // sums of this lane's probabilities
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = f32x16{};
    m = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  // Raises the maximum where mloc exceeds it by enough to matter.
  __device__ __forceinline__ void raise(float mloc, float c) {
    mloc = half_swap_max(mloc);
    const float m_new = fmaxf(m, mloc);
    const bool need = m_new * c > m * c + kRescaleThreshold;
    if (__any(need)) {
      const float alpha = need ? fast_exp2((m - m_new) * c) : 1.0f;
      if (need) m = m_new;
      l[0] *= alpha;
      l[1] *= alpha;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
    }
  }
};

constexpr int kOQ = 64 * 16 + 16;  // a quad of O registers of a wave in the LDS, and padding

// Leaves a wave's state in its slot: D / 8 quads of O, and (maximum in the exp2 domain, sum) of each row. ok: the
// lane has a row (lanes without one would take their turns at the LDS, too).
template <int D>
__device__ __forceinline__ void put_state(const State<D>& st, char* slot, f32x2* ml, float c, int lane, bool ok) {
  const float l = half_swap_sum(st.l[0] + st.l[1]);
  if (!ok) return;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj)
      *reinterpret_cast<f32x4*>(slot + (db * 4 + jj) * kOQ + lane * 16) =
          f32x4{st.o[db][4 * jj], st.o[db][4 * jj + 1], st.o[db][4 * jj + 2], st.o[db][4 * jj + 3]};
  if (lane < 32) ml[lane] = f32x2{st.m == -INFINITY ? -INFINITY : st.m * c, l};
}

// Joins KG states (slot i * step) of a row and writes 8 of its head-dim elements: the output, or a partial of the
// unit.
template <typename T, int D, int KG, bool WIDE>
__device__ __forceinline__ void write_row(const PagedParams& p, const Unit& u, const char* slots, const f32x2* ml, int step,
                                          int slot_b, int r, int quad, int64_t o_off, int lse_at, int rl, int hk) {
  typedef typename T::scalar S;
  typedef typename T::vec8 V8;
  float wt[KG], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < KG; ++i) m = fmaxf(m, ml[i * step * 32 + r][0]);
  const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < KG; ++i) {
    const f32x2 x = ml[i * step * 32 + r];
    wt[i] = fast_exp2(x[0] - mu);
    l = fmaf(wt[i], x[1], l);
  }
  f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
  for (int i = 0; i < KG; ++i) {
    const char* s = slots + (int64_t)i * step * slot_b + quad * kOQ + r * 16;
    lo += wt[i] * *reinterpret_cast<const f32x4*>(s);
    hi += wt[i] * *reinterpret_cast<const f32x4*>(s + 32 * 16);
  }
  if (u.slot < 0) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;  // a row that sees no key: o = 0, lse = -inf
    st16(static_cast<S*>(p.o) + o_off + 8 * quad,
         from_f32x8<V8>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7) * inv));
    if (p.lse != nullptr && quad == 0) p.lse[lse_at] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
    return;
  }
  const int64_t at = ((int64_t)u.slot * p.Hkv + hk) * (WIDE ? p.wide_rows : p.narrow_rows) + rl;
  float* po = (WIDE ? p.wide_o : p.narrow_o) + at * D + 8 * quad;
  *reinterpret_cast<f32x4*>(po) = lo;
  *reinterpret_cast<f32x4*>(po + 4) = hi;
  if (quad == 0) *reinterpret_cast<f32x2*>((WIDE ? p.wide_ml : p.narrow_ml) + 2 * at) = f32x2{m, l};
}

// Scores of one 32-key block in the exp2 domain's value units, masked where `masked`; returns their maximum.
template <typename T, bool SOFTCAP, bool MASKED>
__device__ __forceinline__ float block_scores(f32x16& s, const PagedParams& p, int rel_lo, int rel_hi, unsigned holes) {
  float mloc = -INFINITY;
#pragma unroll
  for (int j = 0; j < 16; ++j) {  // element j holds key 8*(j/4) + 4g + j%4 of the block (rel_*: less 4g)
    float x = score_value<T, SOFTCAP, 0>(s[j], p.s);
    if constexpr (MASKED) {
      const int o = 8 * (j >> 2) + (j & 3);
      x = (o <= rel_hi && o >= rel_lo && !(holes & (j < 8 ? 1u : 2u))) ? x : -INFINITY;
    }
    s[j] = x;
    mloc = fmaxf(mloc, x);
  }
  return mloc;
}

// LDS of the two ways: NW waves' K and V buffers (which their O takes afterwards) and row states; two stages of a
// tile of 16 keys per wave.
template <int D, int NW>
struct Lds {
  typedef DmaLayout<D> L;
  static constexpr int TILE_B = (32 / L::GR) * L::GROUP_B;  // K or V rows of 32 keys
  static constexpr int GRAN_B = (kGranule / L::GR) * L::GROUP_B;
  static constexpr int SLOT_B = (D / 8) * kOQ;
  static constexpr int WAVE_B = std::max(2 * TILE_B, SLOT_B);
  static constexpr int NARROW = NW * (WAVE_B + 32 * 8);
  static constexpr int WIDE = std::max(2 * 2 * NW * GRAN_B, NW * (SLOT_B + 32 * 8));
};

// A wave's tiles of a narrow unit: every NW-th of the 32-key tiles that hold a key.
template <int NW>
struct NarrowTiles {
  int lane, w, t_first, n;
  __device__ __forceinline__ explicit NarrowTiles(const Unit& u) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // the lane constants are made anew for each unit: kept over all of them, they spill
    lane = tid & 63;
    w = __builtin_amdgcn_readfirstlane(tid >> 6);
    t_first = max(u.k0, u.lo) / 32;
    n = u.k1 > u.k0 ? max(0, (ceil_div(min(u.k1, u.hi), 32) - t_first - w + NW - 1) / NW) : 0;
  }
  __device__ __forceinline__ int tile(int s) const { return t_first + w + NW * s; }
  // The lanes' granules of 32 tiles from the wave's tile s on.
  __device__ __forceinline__ int granule(int s) const { return 2 * tile(s + (lane >> 1)) + (lane & 1); }
  __device__ __forceinline__ int first_page(const PagedParams& p, const Unit& u) const {
    Granules gr;
    gr.row = p.table + u.b * p.table_sb;
    return n > 0 ? gr.page_of(p, granule(0)) : 0;
  }
};

// One narrow unit: its keys over NW waves. page: first_page(); ahead(): called when the first copies are on their way.
//
// Bound by the stream of keys and values: per 32-key tile a wave moves 16 KiB (head_dim 128) and runs 16 MFMAs, about
// a tenth of the time that its share of the memory takes. A wave has one K and one V buffer: K of the next tile is
// requested as soon as this one's products have read it, V likewise, so that nearly all of its 16 KiB is always in
// flight, with no barrier and no registers for it. The copies are non-temporal (each row is read once): 64 sequences
// of 7,000 keys, 32 / 8 heads, 317 us without the hint, 289 with. Measured on MI355X: 64 sequences of 512 to 32,768
// keys, fp16, 1.83 GB, 293 us (6.3 TB/s; the contiguous kernels reach 6.6 to 6.85 on caches of one length), 16
// sequences of 32 heads, 1.70 GB, 266 us (6.4).
template <typename T, int D, int NW, bool SOFTCAP, typename F>
__device__ __forceinline__ void narrow_unit(const Unit& u, char* smem, int hk, int page, F&& ahead) {
  typedef typename T::scalar S;
  typedef typename T::vec8 V8;
  typedef typename T::vec4 V4;
  constexpr int TILE_B = Lds<D, NW>::TILE_B, GRAN_B = Lds<D, NW>::GRAN_B, WAVE_B = Lds<D, NW>::WAVE_B;
  constexpr int LOADS = 2 * GranuleCopy<D, true>::LOADS;   // direct loads of a tile, K or V
  const PagedParams& p = fresh_params();
  const NarrowTiles<NW> mine(u);
  const int lane = mine.lane, w = mine.w, tid = 64 * w + lane, r = lane & 31, g = lane >> 5, n_own = mine.n;
  Granules gr;
  gr.row = p.table + u.b * p.table_sb;
  gr.next = page;

  const Row x = find_row(p, u, r, hk);
  const S* qp = static_cast<const S*>(p.q) + x.q;
  V8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) qf[kk] = ld16<V8>(qp + 16 * kk + 8 * g);

  const uint32_t wave_at = (uint32_t)(size_t)((lds_char*)smem) + w * WAVE_B;
  const int64_t k_ss_b = 2 * p.k_ss, v_ss_b = 2 * p.v_ss;
  GranuleCopy<D, true> kc, vc;
  kc.init(lane, k_ss_b);
  vc.init(lane, v_ss_b);
  const char* kp = static_cast<const char*>(p.k) + 2 * hk * p.k_sh;
  const char* vp = static_cast<const char*>(p.v) + 2 * hk * p.v_sh;

  // Copies the K (V) rows of own tile s to the wave's K (V) buffer.
  const int end = min(u.hi, u.k1);
  auto copy = [&](int s, bool values) {
    const int64_t ss_b = values ? v_ss_b : k_ss_b;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int at = 2 * (s & 31) + hh, key = mine.tile(s) * 32 + hh * kGranule;
      const uint32_t lds = wave_at + (values ? TILE_B : 0) + hh * GRAN_B;
      const char* base = values ? vp + gr.offset(p, key / kGranule, at, p.v_sp, p.v_ss)
                                : kp + gr.offset(p, key / kGranule, at, p.k_sp, p.k_ss);
      const GranuleCopy<D, true>& c = values ? vc : kc;
      if (!((gr.live >> at) & 1)) c.zero(lds, lane);
      else if (key >= u.lo && key + kGranule <= end) c.whole(lds, base, ss_b);
      else c.part(lds, base, ss_b, max(0, u.lo - key), min(kGranule, end - key) - 1, lane);
    }
  };
  auto holes_of = [&](int s) { return ~(unsigned)(gr.live >> (2 * (s & 31))) & 3u; };

  unsigned holes = 0;
  if (n_own > 0) {
    gr.take(p, u, mine.granule(0), mine.granule(32));
    copy(0, false);
    copy(0, true);
    holes = holes_of(0);
  }
  ahead();
  // (what the first tile needs besides, while it is on its way)
  Fragments<D> fr;
  fr.init(lane, wave_at, wave_at + TILE_B);
  const Seen see = seen_by_wave(p, u, x, u.row0);
  State<D> st;
  st.init();
  const float c = score_coeff<SOFTCAP, 0>(p.s);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    asm volatile("" : "+v"(qf[kk]));
    if (!x.ok) qf[kk] = V8{};
  }
  for (int s = 0; s < n_own; ++s) {
    const int kt = mine.tile(s) * 32;
    const bool more = s + 1 < n_own;
    const bool live = holes != 3 && kt <= see.hi_max && kt + 31 >= see.lo_min;
    const bool full = holes == 0 && kt >= see.lo_max && kt + 31 <= see.hi_min;
    // The K copies are the older half of what is outstanding (a hole's zeros are no copies: then wait for everything).
    if (holes == 0) wait_vmem<LOADS>();
    else wait_vmem<0>();
    f32x16 sacc = f32x16{};
    if (live) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        sacc = mfma32(lds_read<V8>(fr.k[fr.ki(kk)] + fr.ko(0, kk)), qf[kk], sacc);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the K buffer is read
    // The next K tile is requested before this one's softmax. (The values of a 32-tile window's last tile are copied
    // before its offsets are given up: V of tile s + 1 below uses the window that K took up.)
    unsigned next_holes = 0;
    if (more) {
      if (((s + 1) & 31) == 0) gr.take(p, u, mine.granule(s + 1), mine.granule(s + 33));
      next_holes = holes_of(s + 1);
      copy(s + 1, false);
    }
    if (live) {
      const int k4 = kt + 4 * g;
      const float mloc = full ? block_scores<T, SOFTCAP, false>(sacc, p, 0, 0, 0)
                              : block_scores<T, SOFTCAP, true>(sacc, p, x.k_lo - k4, x.k_hi - k4, holes);
      st.raise(mloc, c);
    }
    if (more && next_holes == 0) wait_vmem<LOADS>();
    else wait_vmem<0>();
    if (live) {
      const float mc = st.m == -INFINITY ? 0.f : st.m * c;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        f32x8 pv;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float pe = fast_exp2(fmaf(sacc[8 * kk + e], c, -mc));
          st.l[e & 1] += pe;
          pv[e] = pe;
        }
        const V8 pb = from_f32x8<V8>(pv);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
          const V4 a0 = tr_read_at(fr.v[fr.vb(db, 0)] + fr.vo(kk, 0), S{});
          const V4 a1 = tr_read_at(fr.v[fr.vb(db, 1)] + fr.vo(kk, 1), S{});
          st.o[db] = mfma32(__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), pb, st.o[db]);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the V buffer is read
    if (more) copy(s + 1, true);
    holes = next_holes;
  }

  // The waves' states over disjoint keys are joined: O = sum_i 2^(m_i - m) O_i, l alike.
  char* slots = smem;
  f32x2* ml = reinterpret_cast<f32x2*>(smem + NW * WAVE_B);
  wait_vmem<0>();
  put_state(st, slots + w * WAVE_B, ml + 32 * w, c, lane, x.ok);
  __syncthreads();
  const PagedParams& pe = fresh_params();
  const int items = min(32, u.rows - u.row0) * (D / 8);
  for (int it0 = 0; it0 < items; it0 += 64 * NW) {
    const int it = it0 + tid, row = min(it / (D / 8), 31), quad = it % (D / 8);
    const int64_t o_off = shfl64(x.o, row);  // (the lane that holds the row, in every wave)
    const int lse_at = __shfl(x.lse, row, 64);
    const bool ok = __shfl((int)x.ok, row, 64);
    if (it < items && ok) write_row<T, D, NW, false>(pe, u, slots, ml, 1, WAVE_B, row, quad, o_off, lse_at, row, hk);
  }
}

// Segment of the stretch that begins with tile f and ends before `to`; returns where it ends (0: there is none).
template <bool WIDE>
__device__ __forceinline__ int narrow_segment(const PagedParams& p, const Division& d, int f, int to, int wg, Unit& u) {
  u.row0 = 0;
  int first, tiles, index;  // the segment's sequence: its first tile and their number, and its place in the slots
  if (f < d.p_tiles) {
    u.prefix = true;
    u.b = 0;
    u.s = Seq{0, 0, 0};
    u.rows = p.T * p.G;
    u.lo = d.p_lo;
    u.hi = p.P;
    first = index = 0;
    tiles = d.p_tiles;
  } else {
    const Place pl = find_place<WIDE, kNarrowTile>(p, d, f - d.p_tiles, threadIdx.x & 63);
    if (pl.b < 0) return 0;
    u.prefix = false;
    u.b = pl.b;
    u.s = pl.s;
    u.rows = pl.s.n * p.G;
    u.lo = first_key(p, u.s);
    u.hi = pl.s.kv;
    first = d.p_tiles + pl.tile0;
    index = pl.b + (d.p_tiles > 0 ? 1 : 0);
    tiles = seq_tiles(p, u.s);
  }
  const int last = min(to, first + tiles), t0 = u.lo / kTile;
  u.k0 = (t0 + f - first) * kTile;
  u.k1 = (t0 + last - first) * kTile;
  u.slot = p.P == 0 && f == first && last == first + tiles ? -1 : wg + index;
  return last;
}

// The stretch of narrow workgroup `wg`, segment by segment. The first page numbers of the next segment are requested
// while the present one streams: behind its 32 MB in flight a load takes 5 us.
template <typename T, int D, int NW, bool WIDE, bool SOFTCAP>
__device__ __forceinline__ void narrow_stretch(const Division& d, char* smem, int hk, int wg) {
  const int from = wg * d.stretch, to = min(d.tiles, from + d.stretch);
  int page = 0;
  for (int f = from; f < to;) {
    Unit u;
    const int next = narrow_segment<WIDE>(fresh_params(), d, f, to, wg, u);
    if (next == 0) return;
    if (f == from) page = NarrowTiles<NW>(u).first_page(fresh_params(), u);
    narrow_unit<T, D, NW, SOFTCAP>(u, smem, hk, page, [&]() __attribute__((always_inline)) {
      if (next >= to) return;
      Unit v;
      if (narrow_segment<WIDE>(fresh_params(), d, next, to, wg, v) != 0)
        page = NarrowTiles<NW>(v).first_page(fresh_params(), v);
    });
    f = next;
    if (f < to) __syncthreads();  // the states in the LDS are read
  }
}

__device__ __forceinline__ bool wide_unit_of(const PagedParams& p, const Division& d, int n, Unit& u) {
  const int R = 1 << p.log2_r, p_units = d.p_rg * d.p_ns;
  int k, ns;
  u.prefix = n < p_units;
  if (u.prefix) {
    k = n / d.p_rg;
    const int rg = n - k * d.p_rg;
    ns = d.p_ns;
    u.b = 0;
    u.s = Seq{0, 0, 0};
    u.row0 = rg * R;
    u.rows = p.T * p.G;
    u.slot = rg * d.p_ns + k;
    u.lo = d.p_lo;
    u.hi = p.P;
  } else {
    const Place pl = find_place<true, kWideUnit>(p, d, n - p_units, threadIdx.x & 63);
    if (pl.b < 0) return false;
    const int nrg = row_groups(p, pl.s.n * p.G);
    ns = wide_slices(p, pl.s, d.slice);
    k = pl.local / nrg;
    // Under a causal mask the last row groups see the most keys: they go first (a prompt of 4,096 tokens 180 -> 150
    // us).
    const int rg = nrg - 1 - (pl.local - k * nrg);
    u.b = pl.b;
    u.s = pl.s;
    u.row0 = rg * R;
    u.rows = pl.s.n * p.G;
    u.slot = p.P == 0 && ns == 1 ? -1 : p_units + pl.slot0 + rg * ns + k;
    set_range(p, u, R);
  }
  const int tiles = key_tiles(u.lo, u.hi), per = ceil_div(tiles, ns), t0 = u.lo / kTile;
  u.k0 = (t0 + min(tiles, k * per)) * kTile;
  u.k1 = (t0 + min(tiles, (k + 1) * per)) * kTile;
  return true;
}

// One wide unit: NW waves over tiles of BN keys in a ring of two. KG: waves that share the same 32 rows, each taking
// BN / KG keys of every tile; a workgroup covers 32 * NW / KG rows. Each wave copies one granule of a tile (BN = 16
// NW).
//
// Bound by the matrix products and the LDS that feeds them, as the prefill forward, whose tiles, layout and order of
// copies these are. Measured on MI355X: 4 x 1,024 tokens over 8,192 keys, bf16, 32 / 8 heads 491 us, 1,050 TFLOP/s,
// beside 462 of that forward with an lse over a contiguous cache on the same box; where the 6% go was not found
// (looking up the next tile's pages among the MFMAs changed nothing). Full and masked tiles have loops of their own:
// one loop for both copied O from one's registers to the other's in every tile, 505 us against 476.
template <typename T, int D, int NW, int KG, int OCC, bool SOFTCAP>
__device__ __forceinline__ void wide_unit(const Unit& u, char* smem, int hk) {
  typedef DmaLayout<D> L;
  typedef typename T::scalar S;
  typedef typename T::vec8 V8;
  typedef typename T::vec4 V4;
  constexpr int BN = kGranule * NW, SBN = BN / KG, NMB = SBN / 32, NWR = NW / KG;
  constexpr int TILE_B = (BN / L::GR) * L::GROUP_B, STAGE_B = 2 * TILE_B;
  constexpr int GRAN_B = Lds<D, NW>::GRAN_B, SLOT_B = Lds<D, NW>::SLOT_B;
  constexpr int WINDOW = 64 / NW;                    // tiles whose granules the lanes hold
  constexpr int LOADS = GranuleCopy<D, false>::LOADS;
  static_assert(SBN % 32 == 0, "key groups");
  const PagedParams& p = fresh_params();
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = KG == 1 ? w : w % NWR, kg = KG == 1 ? 0 : w / NWR;
  const int koff = SBN * kg;

  const int end = min(u.hi, u.k1);
  const int t_first = max(u.k0, u.lo) / BN, t_end = u.k1 > u.k0 ? ceil_div(end, BN) : t_first;
  auto gran_of = [&](int t0) { return NW * (t0 + lane / NW) + lane % NW; };
  Granules gr;
  gr.row = p.table + u.b * p.table_sb;
  if (t_first < t_end) gr.next = gr.page_of(p, gran_of(t_first));

  const int rl = 32 * wr + r;
  const Row x = find_row(p, u, rl, hk);
  const S* qp = static_cast<const S*>(p.q) + x.q;
  V8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) qf[kk] = ld16<V8>(qp + 16 * kk + 8 * g);

  const uint32_t smem_at = (uint32_t)(size_t)((lds_char*)smem);
  const int64_t k_ss_b = 2 * p.k_ss, v_ss_b = 2 * p.v_ss;
  GranuleCopy<D, false> kc, vc;
  kc.init(lane, k_ss_b);
  vc.init(lane, v_ss_b);
  const char* kp = static_cast<const char*>(p.k) + 2 * hk * p.k_sh;
  const char* vp = static_cast<const char*>(p.v) + 2 * hk * p.v_sh;

  // The wave's granule of the tile that is copied next, and the holes of that tile.
  int w_tile = t_first;  // first tile of the lanes' window
  const char *kb = nullptr, *vb = nullptr;
  int g_key = 0;
  unsigned next_holes = 0;
  bool g_live = false, g_whole = false;
  auto aim = [&](int t) {
    if (t - w_tile == WINDOW) {
      w_tile = t;
      gr.take(p, u, gran_of(t), gran_of(t + WINDOW));
    }
    const int at = (t - w_tile) * NW + w;
    kb = kp + gr.offset(p, t * NW + w, at, p.k_sp, p.k_ss);
    vb = vp + gr.offset(p, t * NW + w, at, p.v_sp, p.v_ss);
    g_key = t * BN + w * kGranule;
    g_live = (gr.live >> at) & 1;
    g_whole = g_live && g_key >= u.lo && g_key + kGranule <= end;
    next_holes = ~(unsigned)(gr.live >> ((t - w_tile) * NW)) & ((1u << NW) - 1);
  };
  auto issue = [&](int t) {
    const uint32_t dst = smem_at + (uint32_t)((t & 1) * STAGE_B + w * GRAN_B);
    if (!g_live) {
      kc.zero(dst, lane);
      vc.zero(dst + TILE_B, lane);
    } else if (g_whole) {
      kc.whole(dst, kb, k_ss_b);
      vc.whole(dst + TILE_B, vb, v_ss_b);
    } else {
      const int first = max(0, u.lo - g_key), last = min(kGranule, end - g_key) - 1;
      kc.part(dst, kb, k_ss_b, first, last, lane);
      vc.part(dst + TILE_B, vb, v_ss_b, first, last, lane);
    }
  };

  if (t_first < t_end) {
    gr.take(p, u, gran_of(t_first), gran_of(t_first + WINDOW));
    aim(t_first);
    issue(t_first);
  }
  // (what the first tile needs besides, while it is on its way)
  Fragments<D> fr;
  fr.init(lane, smem_at + (koff / L::GR) * L::GROUP_B, smem_at + TILE_B + (koff / L::GR) * L::GROUP_B);
  const Seen see = seen_by_wave(p, u, x, u.row0 + 32 * wr);
  State<D> st;
  st.init();
  const float c = score_coeff<SOFTCAP, 0>(p.s);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    if (!x.ok) qf[kk] = V8{};
    if constexpr (OCC == 1) asm volatile("" : "+a"(qf[kk]));
    else asm volatile("" : "+v"(qf[kk]));
  }

  // One tile. Full tiles issue the next tile's copies one by one among their QK^T steps, so that the issue overlaps
  // the MFMAs instead of following the barrier as one burst.
  constexpr int CPS = (2 * LOADS + D / 16 - 1) / (D / 16);  // copies per QK^T step
  auto tile = [&](const int t, const unsigned holes, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    const uint32_t sto = (uint32_t)((t & 1) * STAGE_B);
    uint32_t kbase[Fragments<D>::NK], vbase[Fragments<D>::NV];
#pragma unroll
    for (int i = 0; i < Fragments<D>::NK; ++i) {
      kbase[i] = sto + fr.k[i];
      asm volatile("" : "+v"(kbase[i]));
    }
#pragma unroll
    for (int i = 0; i < Fragments<D>::NV; ++i) {
      vbase[i] = sto + fr.v[i];
      asm volatile("" : "+v"(vbase[i]));
    }
    bool blk_live[NMB], blk_full[NMB];
    unsigned blk_holes[NMB];
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb) {
      const int kb0 = t * BN + koff + mb * 32;
      blk_holes[mb] = MASKED ? (holes >> ((koff + mb * 32) / kGranule)) & 3u : 0u;
      blk_live[mb] = !MASKED || (kb0 <= see.hi_max && kb0 + 31 >= see.lo_min && blk_holes[mb] != 3);
      blk_full[mb] = !MASKED || (kb0 >= see.lo_max && kb0 + 31 <= see.hi_min && blk_holes[mb] == 0);
    }
    f32x16 sacc[NMB];
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb) sacc[mb] = f32x16{};
    if constexpr (MASKED) {
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb) {
        if (!blk_live[mb]) continue;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          sacc[mb] = mfma32(lds_read<V8>(kbase[fr.ki(kk)] + fr.ko(mb, kk)), qf[kk], sacc[mb]);
      }
    } else {
      const uint32_t dst = smem_at + (uint32_t)(((t + 1) & 1) * STAGE_B + w * GRAN_B);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
        for (int i = kk * CPS; i < std::min((kk + 1) * CPS, 2 * LOADS); ++i) {
          if (i < LOADS) kc.one(dst, kb, k_ss_b, i);
          else vc.one(dst + TILE_B, vb, v_ss_b, i - LOADS);
        }
#pragma unroll
        for (int mb = 0; mb < NMB; ++mb)
          sacc[mb] = mfma32(lds_read<V8>(kbase[fr.ki(kk)] + fr.ko(mb, kk)), qf[kk], sacc[mb]);
      }
    }
    float mloc = -INFINITY;
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb) {
      const int k4 = t * BN + koff + mb * 32 + 4 * g;
      if (MASKED && !blk_live[mb]) {
#pragma unroll
        for (int j = 0; j < 16; ++j) sacc[mb][j] = -INFINITY;
      } else if (MASKED && !blk_full[mb]) {
        mloc = fmaxf(mloc, block_scores<T, SOFTCAP, true>(sacc[mb], p, x.k_lo - k4, x.k_hi - k4, blk_holes[mb]));
      } else {
        mloc = fmaxf(mloc, block_scores<T, SOFTCAP, false>(sacc[mb], p, 0, 0, 0));
      }
    }
    st.raise(mloc, c);
    const float mc = st.m == -INFINITY ? 0.f : st.m * c;
#pragma unroll
    for (int kk = 0; kk < SBN / 16; ++kk) {
      if (MASKED && !blk_live[kk >> 1]) continue;  // P = 0 there
      f32x8 pv;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float pe = fast_exp2(fmaf(sacc[kk >> 1][8 * (kk & 1) + e], c, -mc));
        st.l[e & 1] += pe;
        pv[e] = pe;
      }
      const V8 pb = from_f32x8<V8>(pv);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        const V4 a0 = tr_read_at(vbase[fr.vb(db, 0)] + fr.vo(kk, 0), S{});
        const V4 a1 = tr_read_at(vbase[fr.vb(db, 1)] + fr.vo(kk, 1), S{});
        st.o[db] = mfma32(__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), pb, st.o[db]);
      }
      asm volatile("" : "+v"(st.l[0]), "+v"(st.l[1]));  // (the sums stay among the MFMAs)
    }
  };

  // Runs of full tiles and of others, in loops of their own (one loop with both would copy O from one's registers to
  // the other's in every tile). look: the kind of tile t, and the granule copied during it.
  unsigned holes = 0;
  bool more = false, full = false;
  auto look = [&](int t) __attribute__((always_inline)) {
    holes = next_holes;
    more = t + 1 < t_end;
    if (more) aim(t + 1);
    const int kb0 = t * BN + koff;
    full = more && g_whole && holes == 0 && kb0 >= see.lo_max && kb0 + SBN - 1 <= see.hi_min;
  };
  int t = t_first;
  if (t < t_end) look(t);
  while (t < t_end) {
    while (t < t_end && full) {
      wait_vmem<0>();
      __syncthreads();
      tile(t, 0, std::false_type{});
      if (++t < t_end) look(t);
    }
    while (t < t_end && !full) {
      wait_vmem<0>();
      __syncthreads();
      if (more) issue(t + 1);
      const int kb0 = t * BN + koff;
      if (kb0 <= see.hi_max && kb0 + SBN - 1 >= see.lo_min) tile(t, holes, std::true_type{});
      if (++t < t_end) look(t);
    }
  }

  // States go through the LDS, so that the stores cover whole rows; KG states of a row are joined.
  f32x2* ml = reinterpret_cast<f32x2*>(smem + NW * SLOT_B);
  __syncthreads();  // every wave is done with the tiles
  put_state(st, smem + w * SLOT_B, ml + 32 * w, c, lane, x.ok);
  __syncthreads();
  const PagedParams& pe = fresh_params();
  // Each wave writes a KG-th of the rows that it holds.
  constexpr int RW = 32 / KG;
#pragma unroll 2
  for (int it = lane; it < RW * (D / 8); it += 64) {
    const int row = kg * RW + it / (D / 8), quad = it % (D / 8);
    const int64_t o_off = shfl64(x.o, row);
    const int lse_at = __shfl(x.lse, row, 64);
    const bool ok = __shfl((int)x.ok, row, 64);
    if (ok)
      write_row<T, D, KG, true>(pe, u, smem + wr * SLOT_B, ml + 32 * wr, NWR, SLOT_B, row, quad, o_off, lse_at,
                                32 * wr + row, hk);
  }
}

constexpr int kNarrowWaves = 4;

// Everything narrow. Waves per SIMD: as many workgroups per CU as the LDS holds (67 KiB at head_dim 128, 133 at 256);
// three at 64.
template <typename T, int D, bool SOFTCAP>
__global__ void __launch_bounds__(64 * kNarrowWaves)
__attribute__((amdgpu_waves_per_eu(D >= 256 ? 1 : D >= 128 ? 2 : 3))) paged_narrow_kernel(PagedParams p) {
  __shared__ __attribute__((aligned(1024))) char smem[Lds<D, kNarrowWaves>::NARROW];
  const int hk = blockIdx.x % p.Hkv, n = blockIdx.x / p.Hkv;
  const Division d = divide<false>(p, threadIdx.x & 63);
  narrow_stretch<T, D, kNarrowWaves, false, SOFTCAP>(d, smem, hk, n);
}

// Narrow stretches, then wide units.
template <typename T, int D, int NW, int KG, int OCC, bool SOFTCAP>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC, OCC)))
paged_mixed_kernel(PagedParams p) {
  __shared__ __attribute__((aligned(1024))) char smem[std::max(Lds<D, NW>::NARROW, Lds<D, NW>::WIDE)];
  const int hk = blockIdx.x % p.Hkv, n = blockIdx.x / p.Hkv;
  const Division d = divide<true>(p, threadIdx.x & 63);
  if (n < d.narrow) {
    narrow_stretch<T, D, NW, true, SOFTCAP>(d, smem, hk, n);
    return;
  }
  Unit u;
  if (wide_unit_of(p, d, n - d.narrow, u)) wide_unit<T, D, NW, KG, OCC, SOFTCAP>(u, smem, hk);
}

// Joins the partials of rows: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, lse = (M + log2 L) ln 2, with those
// of the prefix first and then the sequence's own. A wave takes rows_per_merge rows of the batch (token-major, as the
// prefix numbers them) of a KV head, by itself: its time is the chain lengths -> partials -> output, once for each
// sequence that its rows touch. Its groups of D / 4 lanes (four head-dim elements each) take rows in turn, or share
// one of many partials. TEAM: the four waves of a workgroup share one row, where there are few.
constexpr int kMergeWaves = 4;
template <typename T, int D, bool WIDE, bool TEAM>
__global__ void __launch_bounds__(64 * kMergeWaves) paged_merge_kernel(PagedParams p) {
  typedef typename T::scalar S;
  typedef typename T::vec4 V4;
  constexpr int COLS = D / 4, NG = 64 / COLS;
  const int lane = threadIdx.x & 63, col = lane % COLS, grp = lane / COLS;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = TEAM ? blockIdx.x : blockIdx.x * kMergeWaves + w;
  __shared__ f32x4 team_o[TEAM ? kMergeWaves : 1][COLS];
  __shared__ f32x2 team_ml[TEAM ? kMergeWaves : 1];
  const int hk = wave % p.Hkv;
  const int from = wave / p.Hkv * p.rows_per_merge, to = min(p.T * p.G, from + p.rows_per_merge);
  const Division d = divide<WIDE>(p, lane);
  for (int f = from; f < to;) {
    const Place pl = find_place<WIDE, kToken>(p, d, f / p.G, lane);
    if (pl.b < 0) return;  // behind the last sequence
    const int r_from = pl.local * p.G + (f - f / p.G * p.G);  // rows of the sequence
    const int r_to = min(pl.s.n * p.G, r_from + (to - f));
    f += r_to - r_from;
    // Its own partials: slots own0 + (wide: row group * ns) + 0 .. n_own - 1; the prefix's likewise.
    const bool wide = WIDE && is_wide(p, pl.s);
    int n_own, own0;
    if (wide) {
      n_own = wide_slices(p, pl.s, d.slice);
      own0 = d.p_rg * d.p_ns + pl.slot0;
    } else {
      const int t0 = d.p_tiles + pl.tile0, t1 = t0 + seq_tiles(p, pl.s) - 1;
      own0 = t0 / d.stretch;
      n_own = t1 / d.stretch - own0 + 1;
      own0 += pl.b + (d.p_tiles > 0 ? 1 : 0);
    }
    const int n_pre = d.p_ns > 0 ? d.p_ns : d.p_tiles > 0 ? (d.p_tiles - 1) / d.stretch + 1 : 0;
    const int n_all = n_pre + n_own;
    if (p.P == 0 && n_own == 1) continue;  // written by its unit
    const bool share = NG > 1 && (TEAM || n_all > 8 || r_to - r_from < NG);  // all groups on one row
    const int sub = (share ? grp : 0) + (TEAM ? w * NG : 0), step = (share ? NG : 1) * (TEAM ? kMergeWaves : 1);
    const int at_once = share ? 1 : NG;
    for (int r0 = r_from; r0 < r_to; r0 += at_once) {
      const int row = r0 + (share ? 0 : grp);
      const int rc = min(row, r_to - 1);
      const int qi = rc / p.G, qg = rc - qi * p.G, tok = pl.s.t0 + qi, h = hk * p.G + qg;
      const int prow = tok * p.G + qg;
      const float *pre_o, *pre_ml, *own_o, *own_ml;
      int64_t pre_step, own_step;  // rows from one partial to the next
      auto locate = [&](bool w, int slot, int rl, const float*& po, const float*& pm, int64_t& st) {
        const int rows = w ? p.wide_rows : p.narrow_rows;
        const int64_t at = ((int64_t)slot * p.Hkv + hk) * rows + rl;
        st = (int64_t)p.Hkv * rows;
        po = (w ? p.wide_o : p.narrow_o) + at * D + 4 * col;
        pm = (w ? p.wide_ml : p.narrow_ml) + at * 2;
      };
      const int rg = rc >> p.log2_r, prg = prow >> p.log2_r, rmask = (1 << p.log2_r) - 1;
      const bool pw = WIDE && p.prefix_wide;
      locate(wide, own0 + (wide ? rg * n_own : 0), wide ? rc & rmask : rc, own_o, own_ml, own_step);
      locate(pw, pw ? prg * d.p_ns : 0, pw ? prow & rmask : prow, pre_o, pre_ml, pre_step);
      float M = -INFINITY, Ls = 0.f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      auto sweep = [&](auto in_flight) __attribute__((always_inline)) {
        constexpr int U = decltype(in_flight)::value;
        for (int i0 = sub; i0 < n_all; i0 += step * U) {
          f32x4 o[U];
          f32x2 x[U];
#pragma unroll
          for (int k = 0; k < U; ++k) {
            const int i = min(i0 + step * k, n_all - 1);
            const bool pre = i < n_pre;
            const int64_t at = pre ? i * pre_step : (i - n_pre) * own_step;
            x[k] = *reinterpret_cast<const f32x2*>((pre ? pre_ml : own_ml) + 2 * at);
            o[k] = *reinterpret_cast<const f32x4*>((pre ? pre_o : own_o) + at * D);
          }
          float m = M;
#pragma unroll
          for (int k = 0; k < U; ++k) {
            if (i0 + step * k >= n_all) x[k] = f32x2{-INFINITY, 0.f};
            m = fmaxf(m, x[k][0]);
          }
          const float mu = m == -INFINITY ? 0.f : m, a = fast_exp2(M - mu);
          acc *= a;
          Ls *= a;
#pragma unroll
          for (int k = 0; k < U; ++k) {
            const float wgt = fast_exp2(x[k][0] - mu);
            acc += wgt * o[k];
            Ls = fmaf(wgt, x[k][1], Ls);
          }
          M = m;
        }
      };
      // Loads on their way at once, no more than there are partials (past the last they are repeated: 16 where 8 do, 64
      // decode rows behind 8,192 keys 49.8 / 48.7 us, 128 behind 16,384 92.7 / 91.0).
      if (n_all > 8 * step) sweep(std::integral_constant<int, 16>{});
      else if (n_all > 4 * step) sweep(std::integral_constant<int, 8>{});
      else sweep(std::integral_constant<int, 4>{});
      if (share) {  // (the groups' states, exchanged among lanes of the same elements)
#pragma unroll
        for (int off = COLS; off < 64; off <<= 1) {
          const float m2 = __shfl_xor(M, off, 64), l2 = __shfl_xor(Ls, off, 64);
          f32x4 o2;
#pragma unroll
          for (int e = 0; e < 4; ++e) o2[e] = __shfl_xor(acc[e], off, 64);
          const float m = fmaxf(M, m2), mu = m == -INFINITY ? 0.f : m;
          const float wa = fast_exp2(M - mu), wb = fast_exp2(m2 - mu);
          acc = acc * wa + o2 * wb;
          Ls = Ls * wa + l2 * wb;
          M = m;
        }
      }
      if constexpr (TEAM) {  // (rows_per_merge is 1: once)
        if (grp == 0) team_o[w][col] = acc;
        if (lane == 0) team_ml[w] = f32x2{M, Ls};
        __syncthreads();
        M = -INFINITY;
#pragma unroll
        for (int i = 0; i < kMergeWaves; ++i) M = fmaxf(M, team_ml[i][0]);
        const float mu = M == -INFINITY ? 0.f : M;
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
        Ls = 0.f;
#pragma unroll
        for (int i = 0; i < kMergeWaves; ++i) {
          const float wgt = fast_exp2(team_ml[i][0] - mu);
          acc += wgt * team_o[i][col];
          Ls = fmaf(wgt, team_ml[i][1], Ls);
        }
      }
      if (row >= r_to || sub != 0) continue;
      const float inv = Ls == 0.f ? 0.f : 1.0f / Ls;
      S* op = static_cast<S*>(p.o) + (p.cu_q != nullptr ? tok * p.o_ss : pl.b * p.o_sb + qi * p.o_ss) + h * p.o_sh;
      V4 ov;
#pragma unroll
      for (int e = 0; e < 4; ++e) ov[e] = to_s<S>(acc[e] * inv);
      *reinterpret_cast<V4*>(op + 4 * col) = ov;
      if (p.lse != nullptr && col == 0)
        p.lse[(int64_t)tok * p.Hq + h] = Ls == 0.f ? -INFINITY : (M + fast_log2(Ls)) * kLn2;
    }
  }
}

template <typename T, int D, bool SOFTCAP>
void launch_cap(const PagedParams& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.wide_units + p.narrow_wgs) * p.Hkv);
  if (p.wide_units == 0)
    hipLaunchKernelGGL((paged_narrow_kernel<T, D, SOFTCAP>), grid, dim3(64 * kNarrowWaves), 0, st, p);
  else {
    constexpr int OCC = D == 64 ? 3 : D == 128 ? 2 : 1;
    if constexpr (D == 128) {
      if (p.log2_r == 8) {
        hipLaunchKernelGGL((paged_mixed_kernel<T, D, 8, 1, OCC, SOFTCAP>), grid, dim3(512), 0, st, p);
        return;
      }
    }
    if (p.log2_r == 6) hipLaunchKernelGGL((paged_mixed_kernel<T, D, 4, 2, OCC, SOFTCAP>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_mixed_kernel<T, D, 4, 1, OCC, SOFTCAP>), grid, dim3(256), 0, st, p);
  }
}
template <typename T, int D>
void launch_paged(const PagedParams& p, hipStream_t st) {
  if (p.s.softcap > 0.f) launch_cap<T, D, true>(p, st);
  else launch_cap<T, D, false>(p, st);
  const int64_t rows = (int64_t)p.T * p.G;
  const int64_t waves = (rows + p.rows_per_merge - 1) / p.rows_per_merge * p.Hkv;
  // A workgroup per row up to 512 rows: two per CU (8 sequences of one token behind a prefix of 8,192, 256 rows of up
  // to 66 partials: 22.5 us against 25.4 with a wave for each; 64 sequences, 2,048 rows: 297 against 293).
  const bool team = rows * p.Hkv <= 512;
  const dim3 grid((unsigned)(team ? waves : (waves + kMergeWaves - 1) / kMergeWaves)), block(64 * kMergeWaves);
  if (p.wide_units > 0) {
    if (team) hipLaunchKernelGGL((paged_merge_kernel<T, D, true, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((paged_merge_kernel<T, D, true, false>), grid, block, 0, st, p);
  } else {
    if (team) hipLaunchKernelGGL((paged_merge_kernel<T, D, false, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((paged_merge_kernel<T, D, false, false>), grid, block, 0, st, p);
  }
}

}  // namespace
