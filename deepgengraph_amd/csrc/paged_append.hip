// Appending keys and values to a paged cache, with the rotary embedding of the keys (and of the step's queries) on the
// way: one pass over the projection's result instead of a rotary kernel, two scatters and their index arithmetic.
//
//   token i of sequence b sits at pos = kv_len[b] - n_b + i; angle_j = pos * theta^(-2j/D), pairs (j, j + D/2):
//   k_page[pos % page] = (x cos - y sin, y cos + x sin), v_page[pos % page] = v, query likewise to its own output.
//
// Bound by the bytes of a large call (6,072 tokens of 32 + 32 + 32 heads, fp16, 299 MB read and written: 57 us in the
// kernel trace, 5.3 TB/s, where a large copy reaches 4.8) and by the chain lengths -> page number -> store of a small
// one (64 tokens: 4 us). A workgroup takes a part of one token's heads: its data are requested before the token's
// position and page are known, and the D/2 (cos, sin) pairs are computed once, in the LDS, for all heads. The angle
// is taken in 64 bits, as turns (pos * theta^(-2j/D) / 2 pi, less its nearest whole number): in 32 bits a position of
// 100,000 would leave an error of a hundredth of a radian. From there on 32 bits do: one rounding to the storage type
// at the end.
#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxD = 512;

struct AppendParams {
  const void* q;   // may be null
  const void* k;
  const void* v;
  void* q_out;
  void* k_pages;
  void* v_pages;
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu_q;  // or nullptr: Sq tokens each
  int64_t q_sb, q_ss, q_sh;
  int64_t qo_sb, qo_ss, qo_sh;
  int64_t k_sb, k_ss, k_sh;
  int64_t v_sb, v_ss, v_sh;
  int64_t kp_sp, kp_ss, kp_sh;
  int64_t vp_sp, vp_ss, vp_sh;
  int64_t table_sb;
  int B, T, Sq, Hq, Hkv, D;  // Hq 0: no query
  int num_pages, page, width;
  double log2_step;  // log2(theta) * 2 / D
};

template <typename T>
__device__ __forceinline__ f32x8 load8(const typename T::scalar* p) {
  if constexpr (sizeof(typename T::scalar) == 4) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    return to_f32x8(ld16<typename T::vec8>(p));
  }
}
template <typename T>
__device__ __forceinline__ void store8(typename T::scalar* p, f32x8 v) {
  if constexpr (sizeof(typename T::scalar) == 4) {
    *reinterpret_cast<f32x4*>(p) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    *reinterpret_cast<f32x4*>(p + 4) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
  } else {
    st16(p, from_f32x8<typename T::vec8>(v));
  }
}

// An item is 8 elements of each half of a head: the query heads' first, then the keys', then the values'. One for
// each thread: more workgroups per token, which repeat the look-up and the angles, but shorter ones (64 tokens of 32
// + 8 + 8 heads 4.0 us against 4.6 with four, 4,096 of them 23.8 against 25.9).
template <typename T, bool ROPE>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(AppendParams p) {
  typedef typename T::scalar S;
  __shared__ __attribute__((aligned(16))) float cs[2][kMaxD / 2];
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int half = p.D / 2, per_head = p.D / 16;
  const int n_q = p.Hq * per_head, n_k = p.Hkv * per_head, n_items = n_q + 2 * n_k;

  // The token's sequence: the number of sequences that end at or before it.
  int b, i, n;
  if (p.cu_q == nullptr) {
    b = t / p.Sq;
    i = t - b * p.Sq;
    n = p.Sq;
  } else {
    b = 0;
    for (int j0 = 0; j0 < p.B; j0 += 64) {
      const int j = j0 + lane;
      b += __popcll(__ballot(j < p.B && p.cu_q[min(j, p.B - 1) + 1] <= t));
    }
    if (b >= p.B) return;  // a row behind the last sequence
    const int first = p.cu_q[b];
    i = t - first;
    n = p.cu_q[b + 1] - first;
    if (i < 0) return;  // (only where cu_q does not begin at 0 or descends)
  }

  // Requests first: nothing below depends on them until the rotation.
  const int item = blockIdx.y * kThreads + tid;
  const bool busy = item < n_items;
  const int head = item / per_head, e = (item - head * per_head) * 8;
  f32x8 x = {}, y = {};
  if (busy) {
    const int64_t tq = p.cu_q ? t * p.q_ss : b * p.q_sb + i * p.q_ss;
    const int64_t tk = p.cu_q ? t * p.k_ss : b * p.k_sb + i * p.k_ss;
    const int64_t tv = p.cu_q ? t * p.v_ss : b * p.v_sb + i * p.v_ss;
    const S* src = head < p.Hq ? static_cast<const S*>(p.q) + tq + head * p.q_sh
                   : head < p.Hq + p.Hkv ? static_cast<const S*>(p.k) + tk + (head - p.Hq) * p.k_sh
                                         : static_cast<const S*>(p.v) + tv + (head - p.Hq - p.Hkv) * p.v_sh;
    x = load8<T>(src + e);
    y = load8<T>(src + half + e);
  }

  const int64_t pos = (int64_t)p.kv_lens[b] - n + i;
  int64_t page = -1;
  if (pos >= 0 && pos < (int64_t)p.width * p.page) page = p.table[b * p.table_sb + pos / p.page];
  const int row = (int)(pos % p.page);

  if constexpr (ROPE) {
    for (int j = tid; j < half; j += kThreads) {
      const double turns = (double)pos * (exp2(-p.log2_step * j) * 0.15915494309189533577);  // 1 / (2 pi)
      const float f = (float)(turns - rint(turns));
      float s, c;
      sincospif(2.0f * f, &s, &c);
      cs[0][j] = c;
      cs[1][j] = s;
    }
    __syncthreads();
  }

  if (!busy) return;
  if (ROPE && head < p.Hq + p.Hkv) {
    const f32x8 c = *reinterpret_cast<const f32x8*>(&cs[0][e]), s = *reinterpret_cast<const f32x8*>(&cs[1][e]);
    const f32x8 a = x * c - y * s;
    y = y * c + x * s;
    x = a;
  }
  S* dst;
  if (head < p.Hq) {
    dst = static_cast<S*>(p.q_out) + (p.cu_q ? t * p.qo_ss : b * p.qo_sb + i * p.qo_ss) + head * p.qo_sh;
  } else {
    if (page < 0 || page >= p.num_pages) return;
    dst = head < p.Hq + p.Hkv
              ? static_cast<S*>(p.k_pages) + page * p.kp_sp + row * p.kp_ss + (head - p.Hq) * p.kp_sh
              : static_cast<S*>(p.v_pages) + page * p.vp_sp + row * p.vp_ss + (head - p.Hq - p.Hkv) * p.vp_sh;
  }
  store8<T>(dst + e, x);
  store8<T>(dst + half + e, y);
}

template <typename T>
void launch(const AppendParams& p, bool rope, hipStream_t st) {
  const int items = (p.Hq + 2 * p.Hkv) * (p.D / 16);
  const dim3 grid(p.T, (items + kThreads - 1) / kThreads);
  if (rope) hipLaunchKernelGGL((paged_append_kernel<T, true>), grid, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL((paged_append_kernel<T, false>), grid, dim3(kThreads), 0, st, p);
}

}  // namespace

extern "C" int dgg_paged_append(const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages,
                                const int32_t* block_table, const int32_t* kv_lens, const int32_t* cu_q, int64_t B,
                                int64_t T, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D, int64_t num_pages,
                                int64_t page_size, int64_t table_width, const int64_t* strides, float rope_theta,
                                int dtype, void* stream) {
  const char* op = "paged_append";
  DGG_REQUIRE(dgg::valid_dtype(dtype), DGG_ERR_DTYPE, "%s: unsupported dtype code %d", op, dtype);
  DGG_REQUIRE(B >= 0 && B <= (1 << 20) && T >= 0 && T < (1 << 24), DGG_ERR_SHAPE,
              "%s: bad sizes (B=%lld of at most 2^20, %lld tokens of fewer than 2^24)", op, (long long)B, (long long)T);
  DGG_REQUIRE(Sq >= 0 && Sq < (1 << 24) && (Sq == 0 || Sq * B == T), DGG_ERR_SHAPE,
              "%s: %lld tokens are not %lld sequences of %lld", op, (long long)T, (long long)B, (long long)Sq);
  DGG_REQUIRE((cu_q == nullptr) == (Sq > 0) || T == 0, DGG_ERR_SHAPE,
              "%s: give cu_q, or Sq tokens for every sequence, and not both", op);
  DGG_REQUIRE(Hq >= 0 && Hq <= 1024 && Hkv > 0 && Hkv <= 1024, DGG_ERR_SHAPE, "%s: bad head counts %lld / %lld", op,
              (long long)Hq, (long long)Hkv);
  DGG_REQUIRE(D > 0 && D % 16 == 0 && D <= kMaxD, DGG_ERR_UNSUPPORTED,
              "%s: head_dim must be a positive multiple of 16 up to %d (got %lld)", op, kMaxD, (long long)D);
  DGG_REQUIRE(num_pages >= 0 && num_pages < (1ll << 31), DGG_ERR_SHAPE, "%s: bad page count %lld", op,
              (long long)num_pages);
  DGG_REQUIRE(page_size > 0 && page_size <= (1 << 20), DGG_ERR_SHAPE, "%s: page_size %lld must be in [1, 2^20]", op,
              (long long)page_size);
  DGG_REQUIRE(table_width >= 0 && table_width < (1ll << 31) && table_width * page_size < (1ll << 31), DGG_ERR_SHAPE,
              "%s: a block table row of %lld pages of %lld is too long", op, (long long)table_width,
              (long long)page_size);
  DGG_REQUIRE(rope_theta == 0.f || (std::isfinite(rope_theta) && rope_theta > 0.f), DGG_ERR_SHAPE,
              "%s: rope_theta must be finite and > 0, or 0 for no rotation", op);
  DGG_REQUIRE(Hq == 0 || rope_theta > 0.f, DGG_ERR_SHAPE, "%s: a query needs a rope_theta", op);
  DGG_REQUIRE(strides != nullptr, DGG_ERR_NULL, "%s: strides is NULL", op);
  const int vec = 16 / dgg::dtype_size(dtype);
  for (int i = 0; i < 18; ++i)
    DGG_REQUIRE(strides[i] >= 0 && strides[i] % vec == 0, DGG_ERR_STRIDE,
                "%s: stride[%d] = %lld must be a non-negative multiple of %d elements", op, i, (long long)strides[i], vec);
  DGG_REQUIRE(strides[18] >= 0, DGG_ERR_STRIDE, "%s: the block table's row stride is negative", op);
  if (B == 0 || T == 0) return DGG_OK;
  DGG_REQUIRE(k && v && kv_lens && (Hq == 0 || (q && q_out)), DGG_ERR_NULL, "%s: null pointer", op);
  DGG_REQUIRE(num_pages == 0 || table_width == 0 || (k_pages && v_pages && block_table), DGG_ERR_NULL,
              "%s: null k_pages/v_pages/block_table pointer", op);
  DGG_REQUIRE(dgg::aligned16(q) && dgg::aligned16(k) && dgg::aligned16(v) && dgg::aligned16(q_out) &&
                  dgg::aligned16(k_pages) && dgg::aligned16(v_pages),
              DGG_ERR_ALIGN, "%s: pointers must be 16-byte aligned", op);
  AppendParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.table = block_table;
  p.kv_lens = kv_lens;
  p.cu_q = Sq > 0 ? nullptr : cu_q;
  p.q_sb = strides[0]; p.q_ss = strides[1]; p.q_sh = strides[2];
  p.k_sb = strides[3]; p.k_ss = strides[4]; p.k_sh = strides[5];
  p.v_sb = strides[6]; p.v_ss = strides[7]; p.v_sh = strides[8];
  p.qo_sb = strides[9]; p.qo_ss = strides[10]; p.qo_sh = strides[11];
  p.kp_sp = strides[12]; p.kp_ss = strides[13]; p.kp_sh = strides[14];
  p.vp_sp = strides[15]; p.vp_ss = strides[16]; p.vp_sh = strides[17];
  p.table_sb = strides[18];
  p.B = (int)B;
  p.T = (int)T;
  p.Sq = (int)Sq;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.D = (int)D;
  p.num_pages = (int)num_pages;
  p.page = (int)page_size;
  p.width = num_pages > 0 ? (int)table_width : 0;
  const bool rope = rope_theta > 0.f;
  if (rope) p.log2_step = std::log2((double)rope_theta) * 2.0 / (double)D;
  hipStream_t st = dgg::as_stream(stream);
  if (dtype == DGG_F32) launch<F32>(p, rope, st);
  else if (dtype == DGG_F16) launch<F16>(p, rope, st);
  else launch<BF16>(p, rope, st);
  return dgg::check_launch(op);
}
