// 4-bit pools (kv_int4.h): the append of rows, alone or as the tail of the QKV projection's epilogue, and the
// read-back of pages as fp16.
//
// A row is held by D / 8 lanes, 8 elements each. The epilogue (per-head RMSNorm, rotary embedding; see qk_rope_append.hip) stays
// in fp32 from the fp16 inputs to the one rounding of q and to the quantiser: a K row is not rounded to fp16 on the way,
// which would move one element in some hundred over a code's border. The sum of squares is taken in fp64, where the order
// of its additions does not show, and each product and sum behind it is rounded by itself (no contraction): codes next
// to a border are then the same however a row's lanes are laid out.
//
// Bound by memory: 10366 tokens of 64 + 16 heads of 128 in 78 to 83 us, 5 TB/s of q read and written, k, v and the codes, which is
// what a large copy reaches; a few tokens in 3.5 us, which is a launch.
#include <type_traits>

#include "common.h"
#include "kv_int4.h"

namespace litekv {

// Rows [0, num_q_heads) of a token are q's, the next num_kv_heads K's, then V's. num_q_heads 0: the append alone. A lane has 16 bytes of
// one token (of two or four, with their loads ahead of the work: 1 to 3% longer for many rows, up to 70% for few).
template <int L>
__global__ __launch_bounds__(256) void int4_append_kernel(
    half_t *__restrict__ q, int64_t q_stride, const half_t *__restrict__ k, int64_t k_stride,
    const half_t *__restrict__ v, int64_t v_stride, const half_t *__restrict__ q_weight,
    const half_t *__restrict__ k_weight, const half_t *__restrict__ cos_rows,
    const half_t *__restrict__ sin_rows, int64_t cs_stride, const int32_t *__restrict__ slot_mapping,
    uint8_t *__restrict__ pool, int32_t num_q_heads, int32_t num_kv_heads, int64_t num_slots, float eps) {
#pragma clang fp contract(off)
  constexpr int kDim = 8 * L;
  const int l = threadIdx.x & (L - 1);
  const int r = (int)blockIdx.y * (256 / L) + (int)(threadIdx.x / L);
  if (r >= num_q_heads + 2 * num_kv_heads) return;  // whole L-lane groups leave together
  const bool is_v = r >= num_q_heads + num_kv_heads;
  const bool is_q = r < num_q_heads;
  const int head = is_q ? r : (is_v ? r - num_q_heads - num_kv_heads : r - num_q_heads);
  const int64_t token = blockIdx.x;
  const half_t *src = is_q   ? q + token * q_stride + (int64_t)head * kDim
                      : is_v ? v + token * v_stride + (int64_t)head * kDim
                             : k + token * k_stride + (int64_t)head * kDim;
  const half8_t x = *(const half8_t *)(src + 8 * l);
  const int64_t slot = slot_mapping[token];
  half8_t c = half8_t{0, 0, 0, 0, 0, 0, 0, 0}, sn = c, w = c;
  if (cos_rows != nullptr && !is_v) {
    const int j = 8 * (l & (L / 2 - 1));  // the first D / 2 entries of a cos / sin row
    c = *(const half8_t *)(cos_rows + token * cs_stride + j);
    sn = *(const half8_t *)(sin_rows + token * cs_stride + j);
  }
  const half_t *weight = is_q ? q_weight : k_weight;
  if (weight != nullptr && !is_v) w = *(const half8_t *)(weight + 8 * l);

  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (float)x[i];
  if (weight != nullptr && !is_v) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fma((double)y[i], (double)y[i], ss);
    ss = over_row<L>(ss, [](double a, double b) { return a + b; });
    const double ms = ss * (1.0 / kDim) + (double)eps;
    // 1 / sqrt(ms): the hardware's approximation, twice improved (one step leaves about 2^-50 of it)
    double rs = __builtin_amdgcn_rsq(ms);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      const double e = __builtin_fma(-ms * rs, rs, 1.0);
      rs = __builtin_fma(0.5 * rs, e, rs);
    }
    const float rrms = ms == (double)INFINITY ? 0.f : (float)rs;   // (where a step has made NaN of it)
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * rrms * (float)w[i];
  }
  if (cos_rows != nullptr && !is_v) {
    // partner: element i + D / 2 for the first half of the row, i - D / 2 for the second
    const float sign = l < L / 2 ? -1.0f : 1.0f;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = half_a_row_away<L>(y[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float own = y[i] * (float)c[i], other = p[i] * (float)sn[i];
      y[i] = own + sign * other;
    }
  }
  if (is_q) {
    half8_t o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (half_t)y[i];
    *(half8_t *)(q + token * q_stride + (int64_t)head * kDim + 8 * l) = o;
  } else {
    const Int4Row row = int4_row<L>(y);
    if (slot >= 0 && slot < num_slots) {
      int4_store<kDim>(pool, slot, num_kv_heads, is_v ? num_kv_heads + head : head, l, row);
    }
  }
}

// Tokens as fp16 [slots][2 * Hkv][D]. A lane makes 8 elements of four consecutive tokens' rows of a head, neighbouring lanes
// neighbouring elements and heads, so that stores are whole lines; the four rows' codes are four dwords of K and one load of
// V, whose column holds them together. `no_values`: NaN for V. This is workgroup `tile` of those that take `tokens` slots from `block` on (the first of a block).
template <int D>
__device__ __forceinline__ void int4_to_half(const uint8_t *block, half_t *dst, int32_t kv_heads, int32_t tokens, int32_t tile,
                                             bool no_values = false) {
  constexpr int kPieces = D / 8;   // of a row
  const int32_t item = tile * 256 + (int32_t)threadIdx.x;
  const int w = item % kPieces, row = item / kPieces;
  const int quad = row / (2 * kv_heads), head = row - quad * (2 * kv_heads);
  if (quad >= tokens / 4) return;
  const int g = quad & 3;
  const uint8_t *at = block + (int64_t)(quad >> 2) * int4_block_bytes(kv_heads, D);
  const uint8_t *codes = at + int4_codes_at(head, D);
  const uint2_t words = *(const uint2_t *)(at + int4_words_at(head, kv_heads, D) + 8 * g);
  half8_t y[4];
  auto twice = [&](int i) { return __builtin_amdgcn_perm(0u, words[i >> 1], i & 1 ? 0x03020302u : 0x01000100u); };
  if (head < kv_heads) {
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *(const uint32_t *)(codes + (4 * g + i) * (D / 2) + 4 * w);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = int4x8_to_half(x[i], twice(i));
  } else {
    const uint4_t x = *(const uint4_t *)(codes + g * (2 * D) + 16 * w);
    if constexpr (D == 128) {   // column w: two units of rows 4g, 4g + 1, then of 4g + 2, 4g + 3
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t c = __builtin_amdgcn_perm(x[2 * (i >> 1) + 1], x[2 * (i >> 1)], i & 1 ? 0x07060302u : 0x05040100u);
        y[i] = int4x8_to_half(c, twice(i));
      }
    } else {                    // columns 2w, 2w + 1: four elements of two rows at once, each row's under its own scale
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const half8_t left = int4x8_to_half(x[p], words[p]), right = int4x8_to_half(x[2 + p], words[p]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          y[2 * p + i] = half8_t{left[i], left[2 + i], left[4 + i], left[6 + i], right[i], right[2 + i], right[4 + i], right[6 + i]};
        }
      }
    }
  }
  if (no_values && head >= kv_heads) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __builtin_bit_cast(half8_t, uint4_t{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u});
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) *(half8_t *)(dst + ((int64_t)(4 * quad + i) * (2 * kv_heads) + head) * D + 8 * w) = y[i];
}

template <int D>
__global__ __launch_bounds__(256) void page_dequant_int4_kernel(
    const uint8_t *__restrict__ src_pool, half_t *__restrict__ dst_pool, const int32_t *__restrict__ src_ids,
    const int32_t *__restrict__ dst_ids, int32_t kv_heads, int32_t page_size, int64_t num_src_pages,
    int64_t num_dst_pages, int32_t tiles) {
  const int64_t i = blockIdx.x / (uint32_t)tiles;
  const int64_t sp = src_ids[i];
  const int64_t dp = dst_ids ? (int64_t)dst_ids[i] : i;
  if (sp < 0 || sp >= num_src_pages || dp < 0 || dp >= num_dst_pages) return;
  int4_to_half<D>(src_pool + (sp * (page_size / kInt4Block)) * int4_block_bytes(kv_heads, D),
                  dst_pool + dp * page_size * (int64_t)(2 * kv_heads) * D, kv_heads, page_size, (int32_t)(blockIdx.x - i * tiles));
}

// The keys of a prefill launch as fp16 pages of kInt4StagePage tokens, `capacity` tokens a sequence (a multiple of that), and
// their block table. A workgroup has part `x % tiles` of block x / tiles of sequence y. (8113 tokens of 8 heads of 128, 42 MB read and
// written, in 13 us.)
template <int D>
__global__ __launch_bounds__(256) void int4_stage_kernel(
    const uint8_t *__restrict__ pool, half_t *__restrict__ staged, int32_t *__restrict__ staged_table,
    const int32_t *__restrict__ block_table, int32_t bt_stride, const int32_t *__restrict__ cu_q_lens,
    const int32_t *__restrict__ context_lens, int32_t kv_heads, int32_t page_shift, int32_t num_pages, int32_t capacity,
    int32_t tiles) {
  const int b = (int)blockIdx.y, p = (int)blockIdx.x / tiles, tile = (int)blockIdx.x - p * tiles;
  constexpr int kBlocks = kInt4StagePage / kInt4Block;
  const int64_t page = ((int64_t)b * capacity) / kInt4StagePage + p / kBlocks;
  if (tile == 0 && p % kBlocks == 0 && threadIdx.x == 0) staged_table[page] = (int32_t)page;
  const int rows = as_uniform(cu_q_lens)[b + 1] - as_uniform(cu_q_lens)[b];
  const int64_t keys = (int64_t)rows + (context_lens != nullptr ? as_uniform(context_lens)[b] : 0);
  const int at = rows > 0 ? int4_stage_entry(p, keys, page_shift, bt_stride) : -1;
  if (at < 0) return;
  const int entry = as_uniform(block_table)[(int64_t)b * bt_stride + at];
  int4_to_half<D>(pool + (int64_t)sub_page_id(entry, p, page_shift, num_pages) * int4_block_bytes(kv_heads, D),
                  staged + ((int64_t)b * capacity + (int64_t)p * kInt4Block) * (2 * kv_heads) * D, kv_heads, kInt4Block, tile,
                  p == 0 && keys > capacity);   // the launch was told of fewer: rows of NaN, not rows that lack their last keys
}

int launch_int4_stage(const char *what, const void *pool, void *staged, int32_t *staged_table, const int32_t *block_table,
                      int32_t block_table_stride, const int32_t *cu_q_lens, const int32_t *context_lens, int32_t batch,
                      int32_t num_kv_heads, int32_t head_dim, int32_t page_shift, int64_t num_pages, int64_t capacity,
                      void *stream) {
  const int64_t tiles = ((int64_t)(kInt4Block / 4) * 2 * num_kv_heads * (head_dim / 8) + 255) / 256;
  const int64_t blocks = capacity / kInt4Block * tiles;
  LITEKV_REQUIRE(batch <= 65535 && blocks <= 0x7fffffffLL, "%s: too many keys to stage", what);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)batch), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const uint8_t *>(pool), static_cast<half_t *>(staged), staged_table, block_table,
                       block_table_stride, cu_q_lens, context_lens, num_kv_heads, page_shift, (int32_t)num_pages,
                       (int32_t)capacity, (int32_t)tiles);
  };
  if (head_dim == 64) {
    launch(int4_stage_kernel<64>);
  } else {
    launch(int4_stage_kernel<128>);
  }
  return check_launch(what);
}

static int launch_int4_append(const char *what, void *q, int64_t q_token_stride, const void *k,
                              int64_t k_token_stride, const void *v, int64_t v_token_stride,
                              const void *q_norm_weight, const void *k_norm_weight, const void *cos_rows,
                              const void *sin_rows, int64_t cos_sin_token_stride, const int32_t *slot_mapping,
                              void *kv_pool, int32_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads,
                              int32_t head_dim, int64_t num_slots, float rms_eps, void *stream) {
  LITEKV_REQUIRE(num_tokens >= 0, "%s: num_tokens %d < 0", what, num_tokens);
  LITEKV_REQUIRE(int4_head_dim(head_dim), "%s: head_dim %d unsupported (64 or 128)", what, head_dim);
  LITEKV_REQUIRE(num_q_heads >= 0 && num_kv_heads > 0 && num_q_heads <= 65535 && num_kv_heads <= 65535,
                 "%s: num_q_heads %d / num_kv_heads %d invalid", what, num_q_heads, num_kv_heads);
  if (num_tokens == 0) {
    clear_error();
    return LITEKV_OK;
  }
  LITEKV_REQUIRE((q || num_q_heads == 0) && k && v && slot_mapping && kv_pool, "%s: null pointer", what);
  LITEKV_REQUIRE((q_norm_weight == nullptr) == (k_norm_weight == nullptr),
                 "%s: q_norm_weight and k_norm_weight go together", what);
  LITEKV_REQUIRE((cos_rows == nullptr) == (sin_rows == nullptr), "%s: cos and sin go together", what);
  LITEKV_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(kv_pool) &&
                     aligned16(q_norm_weight) && aligned16(k_norm_weight) && aligned16(cos_rows) &&
                     aligned16(sin_rows),
                 "%s: all tensors must be 16-byte aligned", what);
  LITEKV_REQUIRE((num_q_heads == 0 || (q_token_stride >= (int64_t)num_q_heads * head_dim && q_token_stride % 8 == 0)) &&
                     k_token_stride >= (int64_t)num_kv_heads * head_dim && k_token_stride % 8 == 0 &&
                     v_token_stride >= (int64_t)num_kv_heads * head_dim && v_token_stride % 8 == 0,
                 "%s: token strides (%lld, %lld, %lld) invalid", what, (long long)q_token_stride,
                 (long long)k_token_stride, (long long)v_token_stride);
  LITEKV_REQUIRE(cos_rows == nullptr || (cos_sin_token_stride >= head_dim / 2 && cos_sin_token_stride % 8 == 0),
                 "%s: cos/sin token stride %lld invalid (>= %d, multiple of 8)", what,
                 (long long)cos_sin_token_stride, head_dim / 2);
  LITEKV_REQUIRE(num_slots > 0 && num_slots % kInt4Block == 0, "%s: num_slots %lld is not a positive multiple of 16",
                 what, (long long)num_slots);
  LITEKV_REQUIRE(rms_eps >= 0.f, "%s: rms_eps %g < 0", what, (double)rms_eps);
  const int rows_per_wg = 256 / (head_dim / 8);
  const int row_blocks = (num_q_heads + 2 * num_kv_heads + rows_per_wg - 1) / rows_per_wg;
  LITEKV_REQUIRE(row_blocks <= 65535, "%s: too many heads", what);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)num_tokens, (unsigned)row_blocks), dim3(256), 0,
                       static_cast<hipStream_t>(stream), static_cast<half_t *>(q), q_token_stride,
                       static_cast<const half_t *>(k), k_token_stride, static_cast<const half_t *>(v), v_token_stride,
                       static_cast<const half_t *>(q_norm_weight), static_cast<const half_t *>(k_norm_weight),
                       static_cast<const half_t *>(cos_rows), static_cast<const half_t *>(sin_rows),
                       cos_sin_token_stride, slot_mapping, static_cast<uint8_t *>(kv_pool), num_q_heads, num_kv_heads,
                       num_slots, rms_eps);
  };
  if (head_dim == 64) {
    launch(int4_append_kernel<8>);
  } else {
    launch(int4_append_kernel<16>);
  }
  return check_launch(what);
}

}  // namespace litekv

extern "C" int litekv_kv_append_int4(const void *k, const void *v, int64_t k_token_stride, int64_t v_token_stride,
                                     const int32_t *slot_mapping, void *kv_pool_int4, int32_t num_tokens,
                                     int32_t num_kv_heads, int32_t head_dim, int64_t num_slots, void *stream) {
  return litekv::launch_int4_append("kv_append_int4", nullptr, 0, k, k_token_stride, v, v_token_stride, nullptr,
                                    nullptr, nullptr, nullptr, 0, slot_mapping, kv_pool_int4, num_tokens, 0,
                                    num_kv_heads, head_dim, num_slots, 0.f, stream);
}

extern "C" int litekv_qk_norm_rope_append_int4(void *q, int64_t q_token_stride, const void *k, int64_t k_token_stride,
                                               const void *v, int64_t v_token_stride, const void *q_norm_weight,
                                               const void *k_norm_weight, const void *cos_rows, const void *sin_rows,
                                               int64_t cos_sin_token_stride, const int32_t *slot_mapping,
                                               void *kv_pool_int4, int32_t num_tokens, int32_t num_q_heads,
                                               int32_t num_kv_heads, int32_t head_dim, int64_t num_slots,
                                               float rms_eps, void *stream) {
  if (num_q_heads <= 0) {
    return litekv::fail(LITEKV_ERR_INVALID_ARGUMENT, "qk_norm_rope_append_int4: num_q_heads %d invalid", num_q_heads);
  }
  return litekv::launch_int4_append("qk_norm_rope_append_int4", q, q_token_stride, k, k_token_stride, v,
                                    v_token_stride, q_norm_weight, k_norm_weight, cos_rows, sin_rows,
                                    cos_sin_token_stride, slot_mapping, kv_pool_int4, num_tokens, num_q_heads,
                                    num_kv_heads, head_dim, num_slots, rms_eps, stream);
}

extern "C" int litekv_page_dequant_int4(const void *kv_pool_int4, void *dst_pool, const int32_t *src_ids,
                                        const int32_t *dst_ids, int32_t n, int32_t num_kv_heads, int32_t head_dim,
                                        int32_t page_size, int64_t num_src_pages, int64_t num_dst_pages,
                                        void *stream) {
  using namespace litekv;
  LITEKV_REQUIRE(n >= 0, "page_dequant_int4: n %d < 0", n);
  if (n == 0) {
    clear_error();
    return LITEKV_OK;
  }
  LITEKV_REQUIRE(kv_pool_int4 && dst_pool && src_ids, "page_dequant_int4: null pointer");
  LITEKV_REQUIRE(int4_head_dim(head_dim), "page_dequant_int4: head_dim %d unsupported (64 or 128)", head_dim);
  LITEKV_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65535, "page_dequant_int4: num_kv_heads %d invalid", num_kv_heads);
  LITEKV_REQUIRE(page_shift_of(page_size) >= 0, "page_dequant_int4: page_size %d unsupported (16, 32, 64, 128 or 256)",
                 page_size);
  LITEKV_REQUIRE(aligned16(kv_pool_int4) && aligned16(dst_pool), "page_dequant_int4: pools must be 16-byte aligned");
  LITEKV_REQUIRE(num_src_pages > 0 && num_dst_pages > 0, "page_dequant_int4: empty pool");
  LITEKV_REQUIRE(dst_ids != nullptr || n <= num_dst_pages,
                 "page_dequant_int4: %d pages do not fit a destination of %lld", n, (long long)num_dst_pages);
  const int64_t items = (int64_t)(page_size / 4) * 2 * num_kv_heads * (head_dim / 8);
  const int64_t tiles = (items + 255) / 256;
  LITEKV_REQUIRE(items <= 0x7fffffffLL && tiles * n <= 0x7fffffffLL,
                 "page_dequant_int4: %d pages are too many for one launch", n);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * n)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const uint8_t *>(kv_pool_int4), static_cast<half_t *>(dst_pool), src_ids, dst_ids,
                       num_kv_heads, page_size, num_src_pages, num_dst_pages, (int32_t)tiles);
  };
  if (head_dim == 64) {
    launch(page_dequant_int4_kernel<64>);
  } else {
    launch(page_dequant_int4_kernel<128>);
  }
  return check_launch("page_dequant_int4");
}
