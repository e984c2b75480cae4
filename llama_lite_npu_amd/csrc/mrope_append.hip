// The QKV projection's epilogue for tokens whose position has several axes (time, height, width): per-head RMSNorm of q and k, the
// rotation of their halves by angles that each take one axis' position, and the append of K and V, in one launch.
//
// Pair i of a row (elements i and i + D / 2) turns by entry i of the cos / sin row of position positions[axis(i)][token]. The
// axis of a pair comes with the launch's arguments, two bits each: any split of the pairs, runs or interleaved. A lane holds 8
// elements of a row and gathers the 8 entries of its pairs once for all the rows that it works on.
//
// From the fp16 inputs to the one rounding of q and to the pool's format everything is fp32, each product and sum rounded by
// itself (no contraction), and the sum of squares fp64, where the order of its additions does not show: codes next to a
// border are then the same however a row's lanes are laid out.
//
// Bound by memory: 10366 tokens of 64 + 16 heads of 128 over an fp16 pool in 82 to 84 us, 5.1 TB/s of what is read and written once,
// which is what a large copy reaches; one token in 2.4 us, which is a launch.
#include <type_traits>

#include "common.h"
#include "kv_int4.h"

namespace litekv {

constexpr int kMaxAxes = 4;

struct MropeArgs {
  half_t *q;
  const half_t *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const half_t *q_weight, *k_weight, *cos_table, *sin_table;
  int64_t table_stride;
  int64_t table_rows;
  const void *positions;
  int64_t axis_stride, token_stride;
  const int32_t *slot_mapping;
  void *pool;
  const float *scales;
  int64_t num_slots;
  int32_t num_q_heads, num_kv_heads, num_axes;
  int32_t wide_positions;     // int64
  int32_t mixed;              // some run of 8 pairs has several axes
  int32_t each;               // rows of a lane
  float eps;
  uint64_t axes0, axes1, axes2, axes3;   // two bits a pair (by name: of an array indexed by the lane a copy is kept in memory)
};

// Sums and neighbours over the L lanes of a row (kv_int4.h has 8 and 16).
template <int L>
__device__ __forceinline__ double row_total(double x) {
  if constexpr (L == 4) {
    x += dpp<kDppXor1>(x);
    return x + dpp<kDppXor2>(x);
  } else if constexpr (L == 32) {
    x = over_row<16>(x, [](double a, double b) { return a + b; });
    return x + __shfl_xor(x, 16, 32);
  } else {
    return over_row<L>(x, [](double a, double b) { return a + b; });
  }
}
template <int L>
__device__ __forceinline__ float across_halves(float x) {
  if constexpr (L == 4) return dpp<kDppXor2>(x);
  if constexpr (L == 32) return __shfl_xor(x, 16, 32);
  if constexpr (L == 8 || L == 16) return half_a_row_away<L>(x);
}

// Eight fp32 numbers as codes of a pool with scale `scale`. The quotient is the correctly rounded one. What is not finite goes as in
// the other quantising appends: NaN to the most negative code, infinities to the outermost.
template <int KV>
__device__ __forceinline__ uint2_t floats_to_codes(const float (&x)[8], float scale) {
  constexpr float kMost = KV == kKvFp8 ? kFp8Max : 127.0f;
  const float inv = 1.0f / scale, limit = 2.0f * kMost * scale;
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float n = quotient(__builtin_fminf(__builtin_fmaxf(x[i], -limit), limit), scale, inv);
    c[i] = __builtin_fminf(__builtin_fmaxf(KV == kKvInt8 ? __builtin_rintf(n) : n, -kMost), kMost);
  }
  if constexpr (KV == kKvFp8) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
    return uint2_t{(uint32_t)lo, (uint32_t)hi};
  } else {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)(int)c[i] & 0xffu) << (8 * (i & 3));
    return uint2_t{w[0], w[1]};
  }
}

// A lane's 8 elements of row r of a token (see below); the three pointers each count from row 0.
template <int D>
__device__ __forceinline__ half8_t head_row(int r, int kv0, int v0, const half_t *q, const half_t *k, const half_t *v) {
  uint64_t at = (uint64_t)v;       // (numbers: of a choice among pointers the compiler keeps a table in memory)
  at = r < v0 ? (uint64_t)k : at;
  at = r < kv0 ? (uint64_t)q : at;
  at += (uint64_t)((int64_t)r * D * 2);
  return *(const __attribute__((address_space(1))) half8_t *)at;
}

// Rows [0, num_q_heads) of a token are q's, the next num_kv_heads K's, then V's. Grid: x = token, y = run of each * 256 / L rows; a
// lane has `each` of them, 256 / L apart, the next one's load ahead of a row's work.
template <int KV, int L>
__global__ __launch_bounds__(256) void qk_norm_mrope_append_kernel(const MropeArgs a) {
#pragma clang fp contract(off)
  constexpr int kDim = 8 * L, kApart = 256 / L;
  const int l = threadIdx.x & (L - 1);
  const int64_t token = blockIdx.x;
  const int kv0 = a.num_q_heads, v0 = kv0 + a.num_kv_heads, rows = v0 + a.num_kv_heads;
  int r = (int)blockIdx.y * (a.each * kApart) + (int)(threadIdx.x / L);
  if (r >= rows) return;                                     // whole rows of lanes leave together
  const int end = r + a.each * kApart < rows ? r + a.each * kApart : rows;
  const half_t *q_row = a.q + token * a.q_stride + 8 * l, *k_row = a.k + token * a.k_stride + 8 * l - (int64_t)kv0 * kDim,
               *v_row = a.v + token * a.v_stride + 8 * l - (int64_t)v0 * kDim;
  half8_t next = head_row<kDim>(r, kv0, v0, q_row, k_row, v_row);
  const int64_t slot = a.slot_mapping[token];
  // (what else a row needs is here, or comes with it: a load between a row and the next would be waited for with both)
  half8_t q_weight = half8_t{0, 0, 0, 0, 0, 0, 0, 0}, k_weight = q_weight;
  const bool norm = a.q_weight != nullptr;
  if (norm) {
    q_weight = *(const half8_t *)(a.q_weight + 8 * l);
    k_weight = *(const half8_t *)(a.k_weight + 8 * l);
  }
  constexpr bool kScaled = KV == kKvFp8 || KV == kKvInt8;
  float next_scale = 1.0f;
  if constexpr (kScaled) next_scale = a.scales[r < kv0 ? 0 : r - kv0];

  // the entries of this lane's pairs
  const int run = l & (L / 2 - 1);
  uint64_t near = run & 4 ? a.axes1 : a.axes0;
  if constexpr (L == 32) near = run & 8 ? (run & 4 ? a.axes3 : a.axes2) : near;
  const uint32_t mine = (uint32_t)(near >> (16 * (run & 3))) & 0xffffu;       // the axes of its eight pairs
  // Where an axis' rows begin in the tables. (Both halves of a position are asked for at once, whatever its type.)
  auto row_of = [&](int axis) -> int64_t {
    const int32_t *at = reinterpret_cast<const int32_t *>(static_cast<const char *>(a.positions) +
                                                          (axis * a.axis_stride + token * a.token_stride) * (a.wide_positions ? 8 : 4));
    const int32_t low = at[0], high = at[a.wide_positions];
    const int64_t p = a.wide_positions ? (int64_t)high << 32 | (uint32_t)low : low;
    return (p < 0 ? 0 : p < a.table_rows ? p : a.table_rows - 1) * a.table_stride + 8 * run;
  };
  float c[8], s[8];
  if (!a.mixed) {
    const int64_t at = row_of((int)(mine & 3u));
    const half8_t cc = *(const half8_t *)(a.cos_table + at), ss = *(const half8_t *)(a.sin_table + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = (float)cc[i];
      s[i] = (float)ss[i];
    }
  } else {
    // (axes that there are not repeat the last)
    half8_t cc[kMaxAxes], ss[kMaxAxes];
#pragma unroll
    for (int axis = 0; axis < kMaxAxes; ++axis) {
      const int64_t at = row_of(axis < a.num_axes ? axis : a.num_axes - 1);
      cc[axis] = *(const half8_t *)(a.cos_table + at);
      ss[axis] = *(const half8_t *)(a.sin_table + at);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t axis = mine >> (2 * i) & 3u;
      half_t hc = cc[0][i], hs = ss[0][i];
#pragma unroll
      for (int n = 1; n < kMaxAxes; ++n) {
        hc = axis == (uint32_t)n ? cc[n][i] : hc;
        hs = axis == (uint32_t)n ? ss[n][i] : hs;
      }
      c[i] = (float)hc;
      s[i] = (float)hs;
    }
  }
  // element i of the first half becomes a c - b s, of the second b c + a s
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = l < L / 2 ? -s[i] : s[i];

  const bool there = slot >= 0 && slot < a.num_slots;
#pragma unroll 1
  for (; r < end; r += kApart) {
    const half8_t x = next;
    const float scale = next_scale;
    if constexpr (kScaled) next_scale = a.scales[r + kApart < kv0 || r + kApart >= rows ? 0 : r + kApart - kv0];
    if (r + kApart < end) next = head_row<kDim>(r + kApart, kv0, v0, q_row, k_row, v_row);
    const bool is_q = r < kv0, is_v = r >= v0;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (float)x[i];
    if (norm && !is_v) {
      const half8_t w = is_q ? q_weight : k_weight;
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __builtin_fma((double)y[i], (double)y[i], sum);
      const double ms = row_total<L>(sum) * (1.0 / kDim) + (double)a.eps;
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
    if (!is_v) {
      float other[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) other[i] = across_halves<L>(y[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float own = y[i] * c[i], turned = other[i] * s[i];
        y[i] = own + turned;
      }
    }
    if (is_q) {
      half8_t o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = (half_t)y[i];
      *(half8_t *)(a.q + token * a.q_stride + (int64_t)r * kDim + 8 * l) = o;
      continue;
    }
    const int head = r - kv0;                                // as in the pool: K heads, then V heads
    if constexpr (KV == kKvInt4) {
      const Int4Row row = int4_row<L>(y);
      if (there) int4_store<kDim>(static_cast<uint8_t *>(a.pool), slot, a.num_kv_heads, head, l, row);
    } else {
      if (!there) continue;
      const int64_t at = (slot * (int64_t)(2 * a.num_kv_heads) + head) * kDim + 8 * l;
      if constexpr (KV == kKvF16) {
        half8_t o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (half_t)y[i];
        *(half8_t *)(static_cast<half_t *>(a.pool) + at) = o;
      } else {
        *(uint2_t *)(static_cast<uint8_t *>(a.pool) + at) = floats_to_codes<KV>(y, scale);
      }
    }
  }
}

}  // namespace litekv

extern "C" int litekv_qk_norm_mrope_append(void *q, int64_t q_token_stride, const void *k, int64_t k_token_stride, const void *v,
                                           int64_t v_token_stride, const void *q_norm_weight, const void *k_norm_weight,
                                           const void *cos_table, const void *sin_table, int64_t table_stride,
                                           int64_t table_rows, const void *positions, int32_t positions_int64,
                                           int64_t axis_stride, int64_t token_stride, int32_t num_axes,
                                           const uint8_t *axis_of_pair, const int32_t *slot_mapping, void *kv_pool,
                                           const float *kv_scales, int32_t pool_format, int32_t num_tokens,
                                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int64_t num_slots,
                                           float rms_eps, void *stream) {
  using namespace litekv;
  const char *what = "qk_norm_mrope_append";
  LITEKV_REQUIRE(pool_format >= kKvF16 && pool_format <= kKvInt4, "%s: pool_format %d is not 0 (fp16), 1 (fp8), 2 (int8) or 3 (4-bit)",
                 what, pool_format);
  LITEKV_REQUIRE(num_tokens >= 0, "%s: num_tokens %d < 0", what, num_tokens);
  LITEKV_REQUIRE(pool_format == kKvInt4 ? int4_head_dim(head_dim) : head_dim == kHeadDim || generic_head_dim(head_dim),
                 "%s: head_dim %d unsupported (32, 64, 128 or 256; over 4-bit codes 64 or 128)", what, head_dim);
  LITEKV_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads <= 65535 && num_kv_heads <= 65535,
                 "%s: num_q_heads %d / num_kv_heads %d invalid", what, num_q_heads, num_kv_heads);
  LITEKV_REQUIRE(num_axes >= 1 && num_axes <= kMaxAxes, "%s: num_axes %d out of [1, %d]", what, num_axes, kMaxAxes);
  LITEKV_REQUIRE(axis_of_pair != nullptr, "%s: axis_of_pair is null", what);
  MropeArgs a{};
  for (int i = 0; i < head_dim / 2; ++i) {
    LITEKV_REQUIRE(axis_of_pair[i] < num_axes, "%s: pair %d has axis %d of %d", what, i, axis_of_pair[i], num_axes);
    (i < 32 ? a.axes0 : i < 64 ? a.axes1 : i < 96 ? a.axes2 : a.axes3) |= (uint64_t)axis_of_pair[i] << (2 * (i & 31));
    a.mixed |= axis_of_pair[i] != axis_of_pair[i & ~7];
  }
  if (num_tokens == 0) {
    clear_error();
    return LITEKV_OK;
  }
  const bool scaled = pool_format == kKvFp8 || pool_format == kKvInt8;
  LITEKV_REQUIRE(q && k && v && slot_mapping && kv_pool && cos_table && sin_table && positions, "%s: null pointer", what);
  LITEKV_REQUIRE(scaled == (kv_scales != nullptr), "%s: pools of 8-bit codes have scales, others none", what);
  LITEKV_REQUIRE((q_norm_weight == nullptr) == (k_norm_weight == nullptr),
                 "%s: q_norm_weight and k_norm_weight go together", what);
  LITEKV_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(kv_pool) && aligned16(q_norm_weight) &&
                     aligned16(k_norm_weight) && aligned16(cos_table) && aligned16(sin_table),
                 "%s: all tensors must be 16-byte aligned", what);
  LITEKV_REQUIRE(q_token_stride >= (int64_t)num_q_heads * head_dim && q_token_stride % 8 == 0 &&
                     k_token_stride >= (int64_t)num_kv_heads * head_dim && k_token_stride % 8 == 0 &&
                     v_token_stride >= (int64_t)num_kv_heads * head_dim && v_token_stride % 8 == 0,
                 "%s: token strides (%lld, %lld, %lld) invalid", what, (long long)q_token_stride,
                 (long long)k_token_stride, (long long)v_token_stride);
  LITEKV_REQUIRE(table_rows > 0 && table_stride >= head_dim / 2 && table_stride % 8 == 0,
                 "%s: tables of %lld rows with stride %lld invalid (>= %d, multiple of 8)", what, (long long)table_rows,
                 (long long)table_stride, head_dim / 2);
  LITEKV_REQUIRE(num_slots > 0 && (pool_format != kKvInt4 || num_slots % kInt4Block == 0), "%s: num_slots %lld invalid", what,
                 (long long)num_slots);
  LITEKV_REQUIRE(rms_eps >= 0.f, "%s: rms_eps %g < 0", what, (double)rms_eps);
  a.q = static_cast<half_t *>(q);
  a.k = static_cast<const half_t *>(k);
  a.v = static_cast<const half_t *>(v);
  a.q_stride = q_token_stride;
  a.k_stride = k_token_stride;
  a.v_stride = v_token_stride;
  a.q_weight = static_cast<const half_t *>(q_norm_weight);
  a.k_weight = static_cast<const half_t *>(k_norm_weight);
  a.cos_table = static_cast<const half_t *>(cos_table);
  a.sin_table = static_cast<const half_t *>(sin_table);
  a.table_stride = table_stride;
  a.table_rows = table_rows;
  a.positions = positions;
  a.axis_stride = axis_stride;
  a.token_stride = token_stride;
  a.slot_mapping = slot_mapping;
  a.pool = kv_pool;
  a.scales = kv_scales;
  a.num_slots = num_slots;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.num_axes = num_axes;
  a.wide_positions = positions_int64 != 0;
  a.eps = rms_eps;
  const int rows = num_q_heads + 2 * num_kv_heads, apart = 256 / (head_dim / 8);
  // All rows of a token to a workgroup, the entries of its pairs gathered once for all, where that leaves every compute unit one; a
  // pass of rows to one where there are fewer tokens. us, all rows / a pass, 64 / 8 heads of 128: 64 tokens 5.6 / 4.1, 256 6.2 / 6.1,
  // 512 8.5 / 10.1, 2048 18.1 / 28.3, 8192 67 / 114; 32 / 8 heads of 64: 64 tokens 4.0 / 3.6, 256 4.2 / 4.1, 2048 11.0 / 13.2.
  const int passes = (rows + apart - 1) / apart;
  a.each = num_tokens >= 256 ? passes : 1;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)num_tokens, (unsigned)((passes + a.each - 1) / a.each)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), a);
  };
  LITEKV_REQUIRE((rows + apart - 1) / apart <= 65535, "%s: too many heads", what);
  auto by_format = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    if constexpr (L == 8 || L == 16) {
      if (pool_format == kKvInt4) return launch(qk_norm_mrope_append_kernel<kKvInt4, L>);
    }
    if (pool_format == kKvFp8) return launch(qk_norm_mrope_append_kernel<kKvFp8, L>);
    if (pool_format == kKvInt8) return launch(qk_norm_mrope_append_kernel<kKvInt8, L>);
    launch(qk_norm_mrope_append_kernel<kKvF16, L>);
  };
  switch (head_dim) {
    case 32: by_format(std::integral_constant<int, 4>{}); break;
    case 64: by_format(std::integral_constant<int, 8>{}); break;
    case 256: by_format(std::integral_constant<int, 32>{}); break;
    default: by_format(std::integral_constant<int, 16>{}); break;
  }
  return check_launch(what);
}
