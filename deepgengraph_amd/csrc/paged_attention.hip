// dgg_attn_paged: the host's side of the attention over a paged cache. paged.h has the division of the work,
// paged_attention.h the kernels, which paged_attention_d*.hip instantiate.
#include "common.h"

#include "paged.h"

namespace {

using dgg_paged::PagedParams;

// The host's part of the division.
struct HostPlan {
  int log2_r, places, wide_target, wide_units, wide_slots, wide_rows, narrow_wgs, narrow_most, narrow_slots, narrow_rows,
      prefix_wide;
  int64_t floats(int64_t Hkv, int64_t D) const {
    return ((int64_t)wide_slots * wide_rows + (int64_t)narrow_slots * narrow_rows) * Hkv * (D + 2);
  }
};
// Row groups. 64 rows (waves in pairs over the same rows) where there are no more; otherwise 128 rows, two workgroups
// of four waves per CU, so that one streams or computes while the other begins or ends; but at head_dim 128 256 rows,
// one workgroup of eight waves, for chunks that fill the chip with them: half the keys and values through the LDS.
// Measured on MI355X, bf16, 32 / 8 heads, 128 / 256 rows, us: 2 x 1,024 tokens, 8,192 keys 272 / 245; 16 x 128, 2,048
// 92 / 83; 8 x 512, 512 55 / 52; 4 x 128, 4,096 57.5 / 57.7; 262 tokens of 16 sequences behind a prefix of 16,384 104
// / 122; a step of 28 decode rows and 4 chunks 137 / 146. Units wanted: as many as are resident at once or a little
// fewer, for the row groups' last slices are short (the same step at 256, 384, 448, 512 units 138, 136, 135, 131; 8
// chunks of up to 1,024 tokens 148, 147, 147, 158; the prefix of 16,384 133, 106, 101, 100). Narrow stretches: one
// for each resident workgroup, of at most two per CU (32 x 16 heads of 64, up to 4,000 keys: 512 stretches 53, 768
// 56). Beside wide units one per CU: that many saturate the memory, and more only lengthen the latency that the wide
// units see (the step of 28 decode rows and 4 chunks at 128, 256, 384 stretches 129, 127, 132). Where no sequence is
// wide, which the lengths tell, the device divides the places anew (divide() in paged.h); the grid has room for them:
// places <= wide_target + narrow_wgs for every number of heads.
HostPlan host_plan(int64_t B, int64_t T, bool ragged, int64_t Hq, int64_t Hkv, int64_t D, int64_t P) {
  HostPlan h{};
  const int64_t G = Hq / Hkv, Sq = T / B, CUs = 256;
  const int64_t most = (ragged ? T : Sq) * G;  // most rows that a sequence can have
  h.prefix_wide = P > 0 && T * G > dgg_paged::kNarrowRows;
  const bool wide = most > dgg_paged::kNarrowRows || h.prefix_wide;
  const bool narrow = ragged || most <= dgg_paged::kNarrowRows;
  const int64_t per_cu = D == 64 ? 3 : D == 128 ? 2 : 1;  // workgroups of four waves on a CU
  if (wide) {
    const int64_t typical = h.prefix_wide ? T * G : ragged ? 2 * T * G / B : most;
    const bool large = D == 128 && !ragged && T * G / 256 * Hkv >= CUs;
    h.log2_r = typical <= 64 ? 6 : large ? 8 : 7;
    h.wide_target = (int)std::max<int64_t>(1, (large ? CUs : CUs * per_cu * 7 / 8) / Hkv);
    h.places = (int)std::max<int64_t>(2, CUs * (large ? 1 : per_cu) / Hkv);
    const int64_t R = 1ll << h.log2_r;
    // ragged: a sequence's rows fill row groups but for its last; only sequences of more than 32 rows count
    const int64_t nrg = ragged ? T * G / R + std::min(B, T * G / (dgg_paged::kNarrowRows + 1))
                               : most > dgg_paged::kNarrowRows ? B * ((most + R - 1) / R) : 0;
    const int64_t p_rg = h.prefix_wide ? (T * G + R - 1) / R : 0;
    h.wide_units = (int)(h.wide_target + nrg + p_rg);
    h.wide_slots = P > 0 ? h.wide_units : 2 * h.wide_target;
    h.wide_rows = (int)std::min<int64_t>(R, h.prefix_wide ? T * G : most);
  }
  if (narrow) {
    h.narrow_most = (int)std::max<int64_t>(1, CUs * std::min<int64_t>(per_cu, 2) / Hkv);
    h.narrow_wgs = wide ? (int)std::max<int64_t>(1, std::min(CUs, CUs * per_cu * 3 / 4) / Hkv) : h.narrow_most;
    h.narrow_slots = (int)(h.narrow_most + B + 1);
    h.narrow_rows = (int)std::min<int64_t>(dgg_paged::kNarrowRows, P > 0 && !h.prefix_wide ? T * G : most);
  }
  return h;
}

int check_sizes(const char* op, int64_t B, int64_t T, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix) {
  DGG_REQUIRE(B >= 0 && B <= 4096 && T >= 0 && T < (1 << 24), DGG_ERR_SHAPE,
              "%s: bad sizes (B=%lld of at most 4096, %lld tokens of fewer than 2^24)", op, (long long)B, (long long)T);
  DGG_REQUIRE(Sq >= 0 && Sq < (1 << 24) && (Sq == 0 || Sq * B == T), DGG_ERR_SHAPE,
              "%s: %lld tokens are not %lld sequences of %lld", op, (long long)T, (long long)B, (long long)Sq);
  DGG_REQUIRE(Hq > 0 && Hkv > 0 && Hq <= 1024 && Hq % Hkv == 0, DGG_ERR_SHAPE, "%s: bad head counts (Hq=%lld Hkv=%lld)",
              op, (long long)Hq, (long long)Hkv);
  DGG_REQUIRE(T * Hq < (1 << 28), DGG_ERR_SHAPE, "%s: too many query rows (%lld tokens of %lld heads)", op, (long long)T,
              (long long)Hq);
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
  return host_plan(B, T, Sq == 0, Hq, Hkv, D, prefix_len).floats(Hkv, D) * (int64_t)sizeof(float);
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
  DGG_REQUIRE(table_width >= 0 && table_width < (1ll << 30) && table_width * page_size < (1ll << 30), DGG_ERR_SHAPE,
              "%s: a block table row of %lld pages of %lld is too long", op, (long long)table_width,
              (long long)page_size);
  DGG_REQUIRE(B * table_width * page_size < (1ll << 37), DGG_ERR_SHAPE, "%s: a block table of more than 2^37 keys", op);
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
  DGG_REQUIRE(strides[4] < (1 << 24) && strides[7] < (1 << 24), DGG_ERR_STRIDE,
              "%s: a page's rows are too far apart (strides %lld, %lld; fewer than 2^24 elements)", op,
              (long long)strides[4], (long long)strides[7]);
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
  float* ws = static_cast<float*>(workspace);
  auto carve = [&](int64_t n) {
    float* at = ws;
    ws += n;
    return at;
  };
  const int64_t wide_all = (int64_t)h.wide_slots * h.wide_rows * Hkv;
  const int64_t narrow_all = (int64_t)h.narrow_slots * h.narrow_rows * Hkv;
  p.wide_o = carve(wide_all * D);
  p.narrow_o = carve(narrow_all * D);
  p.wide_ml = carve(wide_all * 2);
  p.narrow_ml = carve(narrow_all * 2);
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
  int log2_up = 0;
  while ((1 << log2_up) < p.gpp) ++log2_up;
  p.gpp_shift = (uint32_t)std::max(0, log2_up - 6);
  p.gpp_mul = p.gpp == 1 ? 0 : (uint32_t)(((1ull << (32 + p.gpp_shift)) + p.gpp - 1) / p.gpp);
  p.P = (int)std::min(prefix_len, cap);
  p.causal = (flags & DGG_ATTN_CAUSAL) != 0;
  p.window = (int)std::min<int64_t>(window, 1 << 30);
  p.log2_r = h.log2_r;
  p.prefix_wide = h.prefix_wide;
  p.wide_units = h.wide_units;
  p.wide_slots = h.wide_slots;
  p.wide_rows = h.wide_rows;
  p.narrow_wgs = h.narrow_wgs;
  p.narrow_most = h.narrow_most;
  p.narrow_slots = h.narrow_slots;
  p.narrow_rows = h.narrow_rows;
  p.wide_target = h.wide_target;
  p.places = h.places;
  p.rows_per_merge = (int)std::max<int64_t>(1, T * p.G * Hkv / 4096);
  hipStream_t st = dgg::as_stream(stream);
  if (D == 64) dgg_paged::launch_d64(p, dtype == DGG_BF16, st);
  else if (D == 128) dgg_paged::launch_d128(p, dtype == DGG_BF16, st);
  else dgg_paged::launch_d256(p, dtype == DGG_BF16, st);
  return dgg::check_launch(op);
}
