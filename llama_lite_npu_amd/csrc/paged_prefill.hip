// Host side of the varlen causal prefill and of the shared-prefix pass of a decode step: argument
// checks, launch shapes and the C ABI. The kernel is in prefill_tile.h.
#include <algorithm>
#include <cmath>

#include "prefill_tile.h"

namespace litekv {
inline namespace LITEKV_HD_NS {
using namespace prefill_tile;

// What is added to the modes of this build's launches (see kCross in prefill_tile.h).
constexpr int kCrossBit = LITEKV_CROSS ? kCross : 0;

static int validate_prefill(const char *what, const void *q, int64_t q_stride, const void *out,
                            int64_t out_stride, int32_t batch, int32_t hq, int32_t hkv,
                            int32_t head_dim, int32_t max_q_len) {
  LITEKV_REQUIRE(batch >= 0 && batch <= 65535, "%s: batch %d out of [0, 65535]", what, batch);
  LITEKV_REQUIRE(head_dim == kHD, "%s: head_dim %d unsupported (32, 64, 128 or 256)", what,
                 head_dim);
  LITEKV_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0 && hq <= 65535,
                 "%s: num_q_heads %d / num_kv_heads %d invalid", what, hq, hkv);
  LITEKV_REQUIRE(hq / hkv <= kMaxGroup, "%s: %d query heads per kv head unsupported (max %d)", what,
                 hq / hkv, kMaxGroup);
  LITEKV_REQUIRE(max_q_len >= 0, "%s: max_q_len %d < 0", what, max_q_len);
  if (batch == 0 || max_q_len == 0) return LITEKV_OK;
  LITEKV_REQUIRE(q && out, "%s: null pointer", what);
  LITEKV_REQUIRE(aligned16(q) && aligned16(out), "%s: q and out must be 16-byte aligned", what);
  const int64_t row = (int64_t)hq * head_dim;
  LITEKV_REQUIRE(q_stride >= row && q_stride % 8 == 0 && out_stride >= row && out_stride % 8 == 0,
                 "%s: token strides (%lld, %lld) invalid", what, (long long)q_stride,
                 (long long)out_stride);
  // q rows are staged with 32-bit byte offsets from the block's first row
  LITEKV_REQUIRE(q_stride < (1 << 25), "%s: q token stride %lld too large", what, (long long)q_stride);
  return LITEKV_OK;
}

// Whether a 256-wide prefill goes to the tiled kernel: all of them but rows it cannot address
// (16-byte stores of the output, 32-bit offsets into q) and scales its arithmetic is not made for
// (tile_scale: 0, below 0, not a number), which stay with the general kernel. Four prompts of 300
// to 2048 tokens, 16 / 4 heads: 9198 us there, without matrix instructions and with every K row
// read by one lane at a time, 76 us here.
[[maybe_unused]] static bool tiled_256(int64_t q_stride, int64_t out_stride, int32_t num_kv_heads,
                                       float softmax_scale) {
  return q_stride < (1 << 25) && out_stride % 8 == 0 && num_kv_heads <= 1024 &&
         tile_scale(softmax_scale * kLog2eP);
}

// How a GQA group of `group` heads is cut into workgroups.
struct PrefillShape {
  int head_splits, heads_per_wg, row_tiles;
  unsigned row_blocks;
};
static PrefillShape prefill_shape(int group, int max_q_len, int wg_col_tiles = kWgColTiles) {
  PrefillShape s;
  s.head_splits = (group + wg_col_tiles - 1) / wg_col_tiles;
  s.heads_per_wg = (group + s.head_splits - 1) / s.head_splits;
  s.row_tiles = wg_col_tiles / s.heads_per_wg;
  s.row_blocks = (unsigned)((max_q_len + 16 * s.row_tiles - 1) / (16 * s.row_tiles));
  return s;
}

// Folds the key slices of a split prefill: the lanes of a (query row, head), four elements each, read the row's
// `slices` log-sum-exps and partial rows (fp32, normalised per slice) and write the fp16 row. A slice without keys has
// log-sum-exp -inf and weight 0; a causal row's last slice always has keys, a row that sees another sequence's keys may have none. Rows behind the last sequence, which no slice wrote, are left as they
// are in `out` (their cells are read, and only the store waits for the number of rows). Bound by memory trips, then by memory: no lane needs another's
// numbers, and all loads are ahead of the arithmetic (64 rows of 16 heads of 128 in 8 slices 3.8 us, 1224 rows of 32 heads
// of 64 in 2 7.7; with a wavefront a row that gathers them by shuffles 5.5 and 15).
constexpr int kMergeLanes = kHD / 4, kMergeRows = 4 * kWave / kMergeLanes;   // of a row; rows of a workgroup
__global__ __launch_bounds__(4 * kWave) void prefill_split_merge_kernel(
    const float *__restrict__ part_o, const float *__restrict__ part_lse, half_t *__restrict__ out,
    int64_t out_stride, int64_t num_tokens, int32_t num_q_heads, int32_t slices, const int32_t *__restrict__ live_rows) {
  const int live = *as_uniform(live_rows);
  const int at = 4 * (threadIdx.x % kMergeLanes);
  const int64_t id = (int64_t)blockIdx.x * kMergeRows + threadIdx.x / kMergeLanes;
  if (id >= num_tokens * num_q_heads) return;
  const int64_t token = id / num_q_heads;
  const int head = (int)(id - token * num_q_heads);
  const int64_t piece_stride = num_tokens * num_q_heads;  // cells between the slices of a row
  float w[kMaxPrefillKeySlices];
  float4_t row[kMaxPrefillKeySlices];
#pragma unroll
  for (int i = 0; i < kMaxPrefillKeySlices; ++i) {
    w[i] = i < slices ? part_lse[i * piece_stride + id] : -INFINITY;
    row[i] = i < slices ? *(const float4_t *)(part_o + (i * piece_stride + id) * kHD + at) : float4_t{0.f, 0.f, 0.f, 0.f};
  }
  float mx = w[0];
#pragma unroll
  for (int i = 1; i < kMaxPrefillKeySlices; ++i) mx = fmaxf(mx, w[i]);
  if (kCrossBit != 0 && mx == -INFINITY) mx = 0.f;   // a sequence without keys: no slice has any
#pragma unroll
  for (int i = 0; i < kMaxPrefillKeySlices; ++i) w[i] = i < slices ? fast_exp2((w[i] - mx) * 1.4426950408889634f) : 0.f;
  static_assert(kMaxPrefillKeySlices == 8, "the order of the sum");
  const float den = ((w[0] + w[4]) + (w[2] + w[6])) + ((w[1] + w[5]) + (w[3] + w[7]));
  float4_t o = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kMaxPrefillKeySlices; ++i) {  // in slice order: the sum does not depend on timing
    if (i < slices) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += w[i] * row[i][j];
    }
  }
  const float inv = kCrossBit == 0 || den > 0.f ? 1.0f / den : 0.f;
  if (token >= live) return;
  *(half4_t *)(out + token * out_stride + (int64_t)head * kHD + at) =
      half4_t{(half_t)(o[0] * inv), (half_t)(o[1] * inv), (half_t)(o[2] * inv), (half_t)(o[3] * inv)};
}

static size_t prefill_split_workspace_bytes(int64_t num_tokens, int32_t num_q_heads, int32_t key_slices) {
  if (num_tokens <= 0 || num_q_heads <= 0 || key_slices <= 1) return 0;
  return (size_t)key_slices * (size_t)num_tokens * (size_t)num_q_heads * (kHD + 1) * sizeof(float);
}

// Compute units of the current device.
static int device_cus() {
  static thread_local int cached_device = -1, cached_cus = 0;  // compute units of the current device
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = -2;
  if (dev != cached_device) {
    int cus = 0;
    if (dev < 0 || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        cus <= 0) {
      cus = 256;
    }
    cached_device = dev;
    cached_cus = cus;
  }
  return cached_cus;
}

// Whether the blocks of a launch of `wgs` workgroups (counted as if every sequence had max_q_len rows, in
// `row_blocks` blocks) whose rows see up to `max_keys` keys are attended by two groups of wavefronts each
// (varlen_prefill_two_group_kernel): where a workgroup would have its compute unit to itself, the narrow
// form does not take it, and half of the key tiles saves more than the larger workgroup and the meeting of
// the groups cost. That is from 10 tiles on; over codes, whose conversion the groups share, from 4; where
// a sequence has one or two blocks of 128-wide fp16 rows and the launch streams its K and V, from 24. Time with
// two groups / one, 136 to 256 workgroups, 1 to 32 sequences, 64 / 8, 16 / 8 and 32 / 4 heads: 4 tiles 0.97 to 1.04
// (fp8 0.94 to 0.99), 9 1.01 to 1.04 (0.95 to 0.97), 10 0.96 to 1.02, 16 0.92 to 0.98, 32 0.88 to 0.95, 128 0.85 to
// 0.94; one or two blocks a sequence: 9 1.03 to 1.09, 16 0.96 to 1.03, 24 0.94 to 1.00; 32 / 8 heads of 64: 9 1.00 to 1.03,
// 10 0.94 to 0.98, 128 0.79 to 0.91. (The width of a block table says little about the keys: 8 chunks of 64 rows,
// nothing cached, in a table of 2048 pages took 8.2 us in two groups, 6.6 in one.)
static bool two_key_groups(int64_t wgs, unsigned row_blocks, int64_t max_keys, bool codes) {
  const int from = codes ? 4 : kHD == 128 && row_blocks <= 2 ? 24 : 10;
  return kHD != 256 && max_keys > (from - 1) * kKvTile && wgs <= device_cus();
}

// Whether a launch of `wgs` workgroups of 128 columns runs with 64 columns a workgroup, one column tile
// per wavefront, instead: where that still leaves at most one workgroup per compute unit. Twice as many
// wavefronts with half of a key tile's products and exponentials each, and less to load, normalise and store around
// them: 0.68 to 0.95 of the time with 128 columns (32 to 128 workgroups, 1 to 128 key tiles, the layouts above). One
// request, us with 128 columns and with 64: 203 rows of a fresh prompt, 16 / 8 heads, 9.2, 7.6; 64 rows, 64 / 8 heads,
// 5.3, 4.4; 128 rows over 2048 tokens 40.1, 30.5; 32 / 8 heads of 64, 256 rows 7.3, 5.8. With more
// workgroups the K and V tiles staged twice cost as much as that saves (400 rows, 64 / 8 heads: 200 workgroups).
static bool narrow_fits(int64_t wgs) {
  return kHD != 256 && 2 * wgs <= device_cus();
}

// Whether narrow workgroups would bring K and V in from memory twice at a cost: those of more than 4 heads per kv
// head share the heads of a block, not its rows, and land on different XCDs, so where every sequence has one block
// (of 128-wide fp16 rows) nothing else keeps its K and V near. From 7/16 of the compute units and 13 key tiles a
// workgroup on (or where nobody says how many, 0) that costs more than the rest saves: 16 rows a sequence, 64 / 8
// heads, time with 64 columns / with 128: 112 workgroups 16 tiles 0.97, 64 tiles 1.05, 128 workgroups 12 tiles 1.00, 16
// 1.05, 32 1.12 (41 us with 128); 96 workgroups 0.82 to 0.96; 16 / 8 heads 0.84 to 0.96, codes and rows of 64 0.73 to
// 0.87. In 8 key slices, two sequences of 30 000 tokens: 77.3 us with 128 columns, 84.1 with 64.
static bool narrow_reads_twice(int64_t wgs, int group, unsigned row_blocks, int64_t max_keys, bool codes) {
  return kHD == 128 && !codes && group > kTiledWaves && row_blocks == 1 && 16 * wgs >= 7 * device_cus() &&
         (max_keys <= 0 || max_keys > 12 * kKvTile);
}

// Key slices for a paged prefill whose row blocks alone would not fill the device, if the longest
// row sees `max_kv_len` keys: the count (at most kMaxPrefillKeySlices) with the smallest estimated
// time, 1 (do not split) unless that is at least 5 % less than unsplit. The estimate, in
// microseconds, head dim 128 (fits to one request's chunk of 64 to 512 rows over 0 to 32k cached
// tokens, 64 query / 8 kv heads): a workgroup walks max_kv_len / 64 / n key tiles at 1.0 us each
// while it has its compute unit to itself (0.75 us with 64 columns, narrow_fits; 0.95 uncut in two groups of
// wavefronts, two_key_groups) and at 1.7 us once the launch has more workgroups than compute units (two share
// one), times the rounds the launch needs on the device's resident slots; a cut costs the merge launch, 6 us, and
// a partial row (fp32) written and read back per query row, head and slice at 6 MB/us. Rows of 64: 0.6 us a
// tile with 64 columns as with 128 (priced at 0.45, chunks of 8 to 64 rows over 1000 tokens were left uncut: 12.1 us, 8.6
// in eight slices; over int8 15.7, 8.9). Over 1121 shapes (8 to 512 rows, 200 to 30 000 tokens, 1 to 4 chunks, the
// layouts above and 32 / 8 heads of 64, codes among them) the choice takes 1.019 times as long as the best count, rows of
// 64 1.020 (1.042 before). (One chunk over 30 000
// tokens, plain against sliced:
// 128 rows 364 -> 148 us, 256 rows 388 -> 269 us, 512 rows 480 -> 485 us; 128 rows over 2048 tokens
// 30.5 -> 25.5 us in four slices; 512 rows over 2048 tokens in two slices 48 -> 62 us and 128 rows of a
// fresh prompt in eight 14 -> 29 us, which the estimate rules out.)
static int32_t prefill_key_slices(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                  int32_t max_q_len, int64_t max_kv_len) {
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      max_q_len <= 0 || max_kv_len <= 0 || num_q_heads / num_kv_heads > kMaxGroup) {
    return 1;
  }
  const PrefillShape s = prefill_shape(num_q_heads / num_kv_heads, max_q_len);
  const int64_t wgs = (int64_t)num_kv_heads * s.head_splits * s.row_blocks * batch;
  const int64_t cus = device_cus();
  const int64_t slots = cus * kWgPerCu;
  if (2 * wgs > slots) return 1;
  const double tile_us = kHD == 64 ? 0.6 : 1.0;
  const double tiles = (double)((max_kv_len + kKvTile - 1) / kKvTile);
  const double partial_us = (double)batch * max_q_len * num_q_heads * (kHD + 1) * 2.0 * sizeof(float) / 6.0e6;
  auto estimate = [&](int64_t n) {
    const int64_t resident = wgs * n;
    const double per_tile = narrow_fits(resident) ? (kHD == 64 ? 1.0 : 0.75) * tile_us
                            : n == 1 && two_key_groups(resident, s.row_blocks, max_kv_len, false) ? 0.95 * tile_us
                            : resident <= cus ? tile_us
                                              : 1.7 * tile_us * (double)((resident + slots - 1) / slots);
    return tiles / (double)n * per_tile + (n > 1 ? 6.0 + partial_us * (double)n : 0.0);
  };
  const double unsplit = estimate(1);
  int64_t best = 1;
  double best_us = 0.95 * unsplit;
  for (int64_t n = 2; n <= kMaxPrefillKeySlices; ++n) {
    const double t = estimate(n);
    if (t < best_us) {
      best = n;
      best_us = t;
    }
  }
  return (int32_t)best;
}

// Causal chunk attention over paged KV; `kv_scales` selects the fp8 pool.
static int launch_paged_prefill(const char *what, const void *q, int64_t q_token_stride,
                                const void *kv_pool, const float *kv_scales,
                                const int32_t *block_table, int32_t block_table_stride,
                                const int32_t *cu_q_lens, const int32_t *context_lens, void *out,
                                int64_t out_token_stride, int32_t batch, int32_t num_q_heads,
                                int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                int64_t num_pages, int32_t max_q_len, float softmax_scale,
                                void *stream, int format, const PrefillKeySplit &split) {
  const bool fp8 = format != kKvF16;  // a pool of codes
  const bool scaled = fp8 && format != kKvInt4;  // by head (4-bit rows carry their own scales)
  LITEKV_REQUIRE(split.key_slices >= 1 && split.key_slices <= kMaxPrefillKeySlices,
                 "%s: key_slices %d out of [1, %d]", what, split.key_slices, kMaxPrefillKeySlices);
  LITEKV_REQUIRE(split.key_slices == 1 || head_dim == 128 || head_dim == 64,
                 "%s: key slices take head_dim 64 or 128", what);
#if LITEKV_CROSS
  LITEKV_REQUIRE(head_dim == 128 || head_dim == 64, "%s: head_dim %d unsupported (64 or 128)", what, head_dim);
  LITEKV_REQUIRE(batch == 0 || max_q_len == 0 || context_lens != nullptr, "%s: null pointer (kv_lens)", what);
#endif
#if LITEKV_CROSS && LITEKV_HD == 128
  if (head_dim == 64) {  // another head dim's build of this file
    return hd64_cross(what, q, q_token_stride, kv_pool, kv_scales, block_table, block_table_stride, cu_q_lens,
                      context_lens, out, out_token_stride, batch, num_q_heads, num_kv_heads, head_dim, page_size,
                      num_pages, max_q_len, softmax_scale, stream, format, split);
  }
#elif LITEKV_HD == 128
  const PrefillBuild *build = head_dim == 64 ? &hd64_prefill()
                              : head_dim == 256 && tiled_256(q_token_stride, out_token_stride, num_kv_heads,
                                                                 softmax_scale)
                                  ? &hd256_prefill()
                                  : nullptr;
  if (build != nullptr) {  // another head dim's build of this file
    return build->paged(what, q, q_token_stride, kv_pool, kv_scales, block_table, block_table_stride, cu_q_lens,
                        context_lens, out, out_token_stride, batch, num_q_heads, num_kv_heads, head_dim,
                        page_size, num_pages, max_q_len, softmax_scale, stream, format, split);
  }
#endif
  if (head_dim != kHD && generic_head_dim(head_dim)) {  // see generic_attention.hip
    LITEKV_REQUIRE(max_q_len >= 0, "%s: max_q_len %d < 0", what, max_q_len);
    LITEKV_REQUIRE(batch == 0 || max_q_len == 0 || (kv_pool && block_table && cu_q_lens),
                   "%s: null pointer", what);
    LITEKV_REQUIRE(!scaled || kv_scales, "%s: null pointer (kv_scales)", what);
    GenericLaunch g;
    g.q = q;
    g.q_row_stride = q_token_stride;
    g.out = out;
    g.out_row_stride = out_token_stride;
    g.kv_pool = const_cast<void *>(kv_pool);
    g.scales = kv_scales;
    g.format = format;
    g.block_table = block_table;
    g.bt_stride = block_table_stride;
    g.page_size = page_size;
    g.num_pages = num_pages;
    g.cu_q_lens = cu_q_lens;
    g.context_lens = context_lens;
    g.batch = batch;
    g.rows_per_seq = max_q_len;
    g.num_q_heads = num_q_heads;
    g.num_kv_heads = num_kv_heads;
    g.head_dim = head_dim;
    g.softmax_scale = softmax_scale;
    g.stream = stream;
    return launch_generic_attention(what, g);
  }
  int rc = validate_prefill(what, q, q_token_stride, out, out_token_stride, batch, num_q_heads,
                            num_kv_heads, head_dim, max_q_len);
  if (rc != LITEKV_OK) return rc;
  const int page_shift = page_shift_of(page_size);
  LITEKV_REQUIRE(page_shift >= 0, "%s: page_size %d unsupported (16, 32, 64, 128 or 256)", what, page_size);
  if (batch == 0 || max_q_len == 0) {
    clear_error();
    return LITEKV_OK;
  }
  LITEKV_REQUIRE(kv_pool && block_table && cu_q_lens, "%s: null pointer", what);
  LITEKV_REQUIRE(!scaled || kv_scales, "%s: null pointer (kv_scales)", what);
  LITEKV_REQUIRE(aligned16(kv_pool), "%s: kv_pool must be 16-byte aligned", what);
  LITEKV_REQUIRE(block_table_stride >= 1, "%s: block_table_stride %d < 1", what, block_table_stride);
  LITEKV_REQUIRE(num_pages >= 1 && num_pages <= 0x7fffffffLL / page_size,
                 "%s: num_pages %lld out of range", what, (long long)num_pages);
  LITEKV_REQUIRE(num_kv_heads <= 1024, "%s: num_kv_heads %d > 1024", what, num_kv_heads);
  PagedSource paged{static_cast<const half_t *>(kv_pool), block_table, block_table_stride,
                    num_kv_heads, (int32_t)num_pages, kv_scales, page_shift};
  PackedSource packed{nullptr, nullptr, 0, 0, nullptr};
  const int group = num_q_heads / num_kv_heads;
#if LITEKV_HD != 256
  if (split.key_slices > 1) {
    // every block's keys in key_slices runs of tiles, one workgroup each, then the merge
    const int slices = split.key_slices;
    const int64_t rows = split.num_tokens;
    LITEKV_REQUIRE(rows >= 1 && rows * num_q_heads * slices <= 0x7fffffffLL,
                   "%s: num_tokens %lld out of range for %d key slices", what, (long long)rows, slices);
    const size_t need = prefill_split_workspace_bytes(rows, num_q_heads, slices);
    LITEKV_REQUIRE(split.workspace != nullptr && aligned16(split.workspace) && split.workspace_bytes >= need,
                   "%s: workspace of %zu bytes needed for %d key slices, got %zu", what, need, slices,
                   split.workspace_bytes);
    PrefillShape s = prefill_shape(group, max_q_len);
    // 64 columns a workgroup (narrow_fits); short slices (at most 16 tiles, as far as the block table can
    // say) up to twice as many: 128 rows, 64 / 8 heads, in 4 slices over 2048 tokens 29.6, 25.5 us, over 8192
    // 54.7, 56.2, over 30 000 169.7, 181.0.
    const int64_t wgs = (int64_t)num_kv_heads * s.head_splits * s.row_blocks * slices * batch;
    const int64_t slice_keys = (int64_t)block_table_stride * page_size / slices;  // at most, by the table
    const bool narrow = (narrow_fits(wgs) || (wgs <= device_cus() && slice_keys <= 16 * kKvTile)) &&
                        !narrow_reads_twice(wgs, group, s.row_blocks, slice_keys, fp8);
    if (narrow) s = prefill_shape(group, max_q_len, kTiledWaves);
    LITEKV_REQUIRE((uint64_t)s.row_blocks * slices <= 65535u, "%s: max_q_len %d too large for %d key slices",
                   what, max_q_len, slices);
    float *part_o = static_cast<float *>(split.workspace);
    float *part_lse = part_o + (size_t)slices * rows * num_q_heads * kHD;
    const PrefixTask task{part_o, part_lse, 0, (int32_t)rows, num_q_heads, 0, 0};
    const dim3 grid((unsigned)(num_kv_heads * s.head_splits), s.row_blocks * (unsigned)slices, (unsigned)batch);
    auto launch_slices = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(kTiledWaves * kWave), 0, static_cast<hipStream_t>(stream),
                         static_cast<const half_t *>(q), q_token_stride, static_cast<half_t *>(out),
                         out_token_stride, paged, packed, task, cu_q_lens, (const int32_t *)nullptr,
                         context_lens, group, s.head_splits, s.heads_per_wg, s.row_tiles,
                         softmax_scale * kLog2eP, slices);
    };
    auto by_width = [&](auto mode_tag) {
      constexpr int MODE = decltype(mode_tag)::value;
      if (narrow) {
        launch_slices(varlen_prefill_tiled_kernel<MODE, 1>);
      } else {
        launch_slices(varlen_prefill_tiled_kernel<MODE>);
      }
    };
    if (format == kKvInt4) {
      by_width(std::integral_constant<int, kPagedPrefillSplitInt4 | kCrossBit>{});
    } else if (format == kKvInt8) {
      by_width(std::integral_constant<int, kPagedPrefillSplitInt8 | kCrossBit>{});
    } else if (format == kKvFp8) {
      by_width(std::integral_constant<int, kPagedPrefillSplitFp8 | kCrossBit>{});
    } else {
      by_width(std::integral_constant<int, kPagedPrefillSplit | kCrossBit>{});
    }
    int rc2 = check_launch(what);
    if (rc2 != LITEKV_OK) return rc2;
    const int64_t merge_rows = rows * num_q_heads;
    hipLaunchKernelGGL(prefill_split_merge_kernel, dim3((unsigned)((merge_rows + kMergeRows - 1) / kMergeRows)), dim3(4 * kWave), 0,
                       static_cast<hipStream_t>(stream), part_o, part_lse, static_cast<half_t *>(out),
                       out_token_stride, rows, num_q_heads, slices, cu_q_lens + batch);
    return check_launch(what);
  }
#endif  // LITEKV_HD != 256
  PrefillShape s = prefill_shape(group, max_q_len);
  LITEKV_REQUIRE(s.row_blocks <= 65535u, "%s: max_q_len %d too large", what, max_q_len);
  dim3 grid((unsigned)(num_kv_heads * s.head_splits), s.row_blocks, (unsigned)batch);
  auto launch = [&](auto mode_tag) {
    constexpr int MODE = decltype(mode_tag)::value;
    auto with = [&](auto kernel, int waves) {
      hipLaunchKernelGGL(kernel, grid, dim3(waves * kWave), 0, static_cast<hipStream_t>(stream),
                         static_cast<const half_t *>(q), q_token_stride, static_cast<half_t *>(out),
                         out_token_stride, paged, packed, PrefixTask{}, cu_q_lens,
                         (const int32_t *)nullptr, context_lens, group, s.head_splits, s.heads_per_wg,
                         s.row_tiles, softmax_scale * kLog2eP, 1);
    };
#if LITEKV_HD != 256
    const int64_t max_keys = context_lens != nullptr ? split.max_kv_len : max_q_len;
    const int64_t wgs = (int64_t)grid.x * grid.y * grid.z;
    if (narrow_fits(wgs) && !narrow_reads_twice(wgs, group, s.row_blocks, max_keys, fp8)) {
      s = prefill_shape(group, max_q_len, kTiledWaves);
      grid = dim3((unsigned)(num_kv_heads * s.head_splits), s.row_blocks, (unsigned)batch);
      with(varlen_prefill_tiled_kernel<MODE, 1>, kTiledWaves);
      return;
    }
    if (two_key_groups(wgs, s.row_blocks, max_keys, fp8)) {
      with(varlen_prefill_two_group_kernel<MODE>, 2 * kTiledWaves);
      return;
    }
#endif
    with(varlen_prefill_tiled_kernel<MODE>, prefill_waves(MODE));
  };
#if LITEKV_HD != 256
  if (format == kKvInt4) {
    launch(std::integral_constant<int, kPagedPrefillInt4 | kCrossBit>{});
    return check_launch(what);
  }
#endif
  if (format == kKvInt8) {
    launch(std::integral_constant<int, kPagedPrefillInt8 | kCrossBit>{});
  } else if (format == kKvFp8) {
    launch(std::integral_constant<int, kPagedPrefillFp8 | kCrossBit>{});
  } else {
    launch(std::integral_constant<int, kPagedPrefill | kCrossBit>{});
  }
  return check_launch(what);
}

#if !LITEKV_CROSS
// Causal attention over packed, contiguous K/V.
static int launch_varlen_prefill(const void *q, int64_t q_token_stride, const void *k,
                                 int64_t k_token_stride, const void *v, int64_t v_token_stride,
                                 const int32_t *seq_starts, const int32_t *seq_lens, void *out,
                                 int64_t out_token_stride, int32_t batch, int32_t num_q_heads,
                                 int32_t num_kv_heads, int32_t head_dim, int32_t max_seq_len,
                                 int64_t num_tokens, float softmax_scale, void *stream) {
#if LITEKV_HD == 128
  const PrefillBuild *build =
      head_dim == 64 ? &hd64_prefill()
      : head_dim == 256 && tiled_256(q_token_stride, out_token_stride, num_kv_heads, softmax_scale) &&
              k_token_stride < (1 << 25) && v_token_stride < (1 << 25)
          ? &hd256_prefill()
          : nullptr;
  if (build != nullptr) {  // another head dim's build of this file
    return build->varlen(q, q_token_stride, k, k_token_stride, v, v_token_stride, seq_starts, seq_lens, out,
                         out_token_stride, batch, num_q_heads, num_kv_heads, head_dim, max_seq_len,
                         num_tokens, softmax_scale, stream);
  }
#endif
  if (head_dim != kHD && generic_head_dim(head_dim)) {  // see generic_attention.hip
    LITEKV_REQUIRE(max_seq_len >= 0, "varlen_prefill: max_seq_len %d < 0", max_seq_len);
    GenericLaunch g;
    g.q = q;
    g.q_row_stride = q_token_stride;
    g.out = out;
    g.out_row_stride = out_token_stride;
    g.k = k;
    g.v = v;
    g.k_stride = k_token_stride;
    g.v_stride = v_token_stride;
    g.seq_starts = seq_starts;
    g.q_lens = seq_lens;
    g.batch = num_tokens == 0 ? 0 : batch;
    g.rows_per_seq = max_seq_len;
    g.num_q_heads = num_q_heads;
    g.num_kv_heads = num_kv_heads;
    g.head_dim = head_dim;
    g.softmax_scale = softmax_scale;
    g.stream = stream;
    return launch_generic_attention("varlen_prefill", g);
  }
  int rc = validate_prefill("varlen_prefill", q, q_token_stride, out, out_token_stride, batch,
                            num_q_heads, num_kv_heads, head_dim, max_seq_len);
  if (rc != LITEKV_OK) return rc;
  if (batch == 0 || max_seq_len == 0 || num_tokens == 0) {
    clear_error();
    return LITEKV_OK;
  }
  LITEKV_REQUIRE(k && v && seq_starts && seq_lens, "varlen_prefill: null pointer");
  LITEKV_REQUIRE(aligned16(k) && aligned16(v), "varlen_prefill: k and v must be 16-byte aligned");
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  LITEKV_REQUIRE(k_token_stride >= row && k_token_stride % 8 == 0 && v_token_stride >= row &&
                     v_token_stride % 8 == 0,
                 "varlen_prefill: k/v token strides (%lld, %lld) invalid",
                 (long long)k_token_stride, (long long)v_token_stride);
  LITEKV_REQUIRE(k_token_stride < (1 << 25) && v_token_stride < (1 << 25),
                 "varlen_prefill: k/v token strides (%lld, %lld) too large",
                 (long long)k_token_stride, (long long)v_token_stride);
  PagedSource paged{nullptr, nullptr, 0, num_kv_heads, 1, nullptr};
  PackedSource packed{static_cast<const half_t *>(k), static_cast<const half_t *>(v),
                      k_token_stride, v_token_stride, seq_starts};
  const int group = num_q_heads / num_kv_heads;
  PrefillShape s = prefill_shape(group, max_seq_len);
  LITEKV_REQUIRE(s.row_blocks <= 65535u, "varlen_prefill: max_seq_len %d too large", max_seq_len);
  dim3 grid((unsigned)(num_kv_heads * s.head_splits), s.row_blocks, (unsigned)batch);
  auto launch = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, grid, dim3(waves * kWave), 0, static_cast<hipStream_t>(stream),
                       static_cast<const half_t *>(q), q_token_stride, static_cast<half_t *>(out),
                       out_token_stride, paged, packed, PrefixTask{}, seq_starts, seq_lens,
                       (const int32_t *)nullptr, group, s.head_splits, s.heads_per_wg, s.row_tiles,
                       softmax_scale * kLog2eP, 1);
  };
#if LITEKV_HD != 256
  const int64_t wgs = (int64_t)grid.x * grid.y * grid.z;
  if (narrow_fits(wgs) && !narrow_reads_twice(wgs, group, s.row_blocks, max_seq_len, false)) {
    s = prefill_shape(group, max_seq_len, kTiledWaves);
    grid = dim3((unsigned)(num_kv_heads * s.head_splits), s.row_blocks, (unsigned)batch);
    launch(varlen_prefill_tiled_kernel<kPackedPrefill, 1>, kTiledWaves);
    return check_launch("varlen_prefill");
  }
  if (two_key_groups(wgs, s.row_blocks, max_seq_len, false)) {
    launch(varlen_prefill_two_group_kernel<kPackedPrefill>, 2 * kTiledWaves);
    return check_launch("varlen_prefill");
  }
#endif
  launch(varlen_prefill_tiled_kernel<kPackedPrefill>, prefill_waves(kPackedPrefill));
  return check_launch("varlen_prefill");
}
#endif  // !LITEKV_CROSS
}  // namespace LITEKV_HD_NS

#if LITEKV_CROSS && LITEKV_HD == 64
int hd64_cross(const char *what, const void *q, int64_t q_token_stride, const void *kv_pool, const float *kv_scales,
               const int32_t *block_table, int32_t block_table_stride, const int32_t *cu_q_lens,
               const int32_t *kv_lens, void *out, int64_t out_token_stride, int32_t batch, int32_t num_q_heads,
               int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int64_t num_pages, int32_t max_q_len,
               float softmax_scale, void *stream, int format, const PrefillKeySplit &split) {
  return launch_paged_prefill(what, q, q_token_stride, kv_pool, kv_scales, block_table, block_table_stride, cu_q_lens,
                              kv_lens, out, out_token_stride, batch, num_q_heads, num_kv_heads, head_dim, page_size,
                              num_pages, max_q_len, softmax_scale, stream, format, split);
}
#elif LITEKV_CROSS
#elif LITEKV_HD == 64
const PrefillBuild &hd64_prefill() {
  static const PrefillBuild build{launch_paged_prefill, launch_varlen_prefill, prefill_key_slices};
  return build;
}
#elif LITEKV_HD == 256
const PrefillBuild &hd256_prefill() {
  static const PrefillBuild build{launch_paged_prefill, launch_varlen_prefill, nullptr};
  return build;
}
#endif
}  // namespace litekv

#if LITEKV_CROSS && LITEKV_HD == 128
// Slices of the keys for a launch of few rows over an encoder's states: as many as balance the chain of tiles that a workgroup walks
// (0.8 us a tile, 0.4 of 64-wide heads) against the partial rows written and read back (6 MB/us), up to four workgroups a compute unit, since lengths
// are seldom even; none where that comes to fewer than four, or a launch that has a workgroup on every other compute unit
// walks fewer than 48 tiles. us, uncut / by this rule / in the best of 1, 2, 3, 4, 6 and 8: 32 sequences of 5 rows over up to 6400 states,
// 64 / 8 heads 124 / 112 / 112 (int8 111 / 83 / 83), 16 / 8 125 / 101 / 101 (112 / 81 / 79); 12 of up to 9 over up to 3000 41 / 25 / 24,
// 32 / 8 heads of 64, int8, 38 / 18 / 18; 4 of 40 over 1000, 16 / 8, 15.8 / 12.9 / 12.3; 2 of 300 over 6400, 32 / 4, 82 / 58 / 58; 8 of 64 over
// 1600, 64 / 8, 28 / 28 / 28 (in four slices 37). Over 88 shapes (1 to 64 sequences of 2 to 300 rows over 500 to 6400 states, the
// layouts 64 / 8, 16 / 8, 32 / 4 and 32 / 8 of 64, fp16 and int8) it takes 1.04 times as long as the best count, uncut launches 1.49.
extern "C" int32_t litekv_paged_cross_key_slices(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                 int32_t max_q_len, int64_t max_kv_len, int64_t num_tokens) {
  using namespace litekv;
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || max_q_len <= 0 ||
      max_kv_len <= 0 || num_tokens <= 0 || num_q_heads / num_kv_heads > kMaxGroup || (head_dim != 64 && head_dim != 128)) {
    return 1;
  }
  const PrefillShape s = prefill_shape(num_q_heads / num_kv_heads, max_q_len);
  const int64_t wgs = (int64_t)num_kv_heads * s.head_splits * s.row_blocks * batch, cus = device_cus();
  const int64_t tiles = (max_kv_len + kKvTile - 1) / kKvTile;
  if (wgs > cus || (2 * wgs >= cus && tiles < 48)) return 1;
  const double chain_us = (head_dim == 64 ? 0.4 : 0.8) * (double)tiles;
  const double partial_us = (double)num_tokens * num_q_heads * (head_dim + 1) * 2.0 * sizeof(float) / 6.0e6;
  const int64_t n = std::min<int64_t>(std::min<int64_t>(kMaxPrefillKeySlices, 4 * cus / wgs), (int64_t)(std::sqrt(chain_us / partial_us) + 0.5));
  return n < 4 ? 1 : (int32_t)n;
}

extern "C" int litekv_paged_cross_attention(const void *q, int64_t q_token_stride, const void *kv_pool,
                                            const float *kv_scales, int32_t pool_format,
                                            const int32_t *block_table, int32_t block_table_stride,
                                            const int32_t *cu_q_lens, const int32_t *kv_lens, void *out,
                                            int64_t out_token_stride, int32_t batch, int32_t num_q_heads,
                                            int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                            int64_t num_pages, int32_t max_q_len, int64_t max_kv_len,
                                            int64_t num_tokens, int32_t key_slices, void *workspace,
                                            size_t workspace_bytes, float softmax_scale, void *stream) {
  using namespace litekv;
  const char *what = "paged_cross_attention";
  LITEKV_REQUIRE(pool_format >= kKvF16 && pool_format <= kKvInt4, "%s: pool_format %d is not 0 (fp16), 1 (fp8), 2 (int8) or 3 (4-bit)",
                 what, pool_format);
  LITEKV_REQUIRE((pool_format == kKvFp8 || pool_format == kKvInt8) == (kv_scales != nullptr),
                 "%s: pools of 8-bit codes have scales, others none", what);
  PrefillKeySplit split;
  split.key_slices = key_slices;
  split.workspace = workspace;
  split.workspace_bytes = workspace_bytes;
  split.num_tokens = num_tokens;
  split.max_kv_len = max_kv_len;
  return launch_paged_prefill(what, q, q_token_stride, kv_pool, kv_scales, block_table, block_table_stride, cu_q_lens,
                              kv_lens, out, out_token_stride, batch, num_q_heads, num_kv_heads, head_dim, page_size,
                              num_pages, max_q_len, softmax_scale, stream, pool_format, split);
}
#elif LITEKV_HD == 128 && !LITEKV_CROSS  // the C ABI lives in the head dim 128 build of this file

extern "C" int litekv_paged_prefill(const void *q, int64_t q_token_stride, const void *kv_pool,
                                    const int32_t *block_table, int32_t block_table_stride,
                                    const int32_t *cu_q_lens, const int32_t *context_lens,
                                    void *out, int64_t out_token_stride, int32_t batch,
                                    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t page_size, int64_t num_pages, int32_t max_q_len,
                                    float softmax_scale, void *stream) {
  return litekv::launch_paged_prefill("paged_prefill", q, q_token_stride, kv_pool, nullptr, block_table,
                                      block_table_stride, cu_q_lens, context_lens, out,
                                      out_token_stride, batch, num_q_heads, num_kv_heads, head_dim,
                                      page_size, num_pages, max_q_len, softmax_scale, stream,
                                      litekv::kKvF16, litekv::PrefillKeySplit{});
}

extern "C" int litekv_paged_prefill_bounded(const void *q, int64_t q_token_stride, const void *kv_pool,
                                            const float *kv_scales, int32_t pool_is_int8,
                                            const int32_t *block_table, int32_t block_table_stride,
                                            const int32_t *cu_q_lens, const int32_t *context_lens,
                                            void *out, int64_t out_token_stride, int32_t batch,
                                            int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                            int32_t page_size, int64_t num_pages, int32_t max_q_len,
                                            int64_t max_kv_len, float softmax_scale, void *stream) {
  const int format = kv_scales == nullptr ? litekv::kKvF16 : pool_is_int8 ? litekv::kKvInt8 : litekv::kKvFp8;
  const char *what = format == litekv::kKvF16    ? "paged_prefill"
                     : format == litekv::kKvInt8 ? "paged_prefill_int8"
                                                 : "paged_prefill_fp8";
  litekv::PrefillKeySplit split;
  split.max_kv_len = max_kv_len;
  return litekv::launch_paged_prefill(what, q, q_token_stride, kv_pool, kv_scales, block_table,
                                      block_table_stride, cu_q_lens, context_lens, out,
                                      out_token_stride, batch, num_q_heads, num_kv_heads, head_dim,
                                      page_size, num_pages, max_q_len, softmax_scale, stream, format, split);
}

extern "C" size_t litekv_paged_prefill_split_workspace_bytes(int64_t num_tokens, int32_t num_q_heads,
                                                             int32_t head_dim, int32_t key_slices) {
  if (head_dim != 128 && head_dim != 64) return 0;
  if (num_tokens <= 0 || num_q_heads <= 0 || key_slices <= 1) return 0;
  return (size_t)key_slices * (size_t)num_tokens * (size_t)num_q_heads * (size_t)(head_dim + 1) * sizeof(float);
}

extern "C" int32_t litekv_paged_prefill_key_slices(int32_t batch, int32_t num_q_heads,
                                                   int32_t num_kv_heads, int32_t head_dim,
                                                   int32_t max_q_len, int64_t max_kv_len) {
  if (head_dim == 64) {
    return litekv::hd64_prefill().key_slices(batch, num_q_heads, num_kv_heads, max_q_len, max_kv_len);
  }
  if (head_dim != 128) return 1;
  return litekv::prefill_key_slices(batch, num_q_heads, num_kv_heads, max_q_len, max_kv_len);
}

extern "C" int litekv_paged_prefill_split(const void *q, int64_t q_token_stride, const void *kv_pool,
                                          const int32_t *block_table, int32_t block_table_stride,
                                          const int32_t *cu_q_lens, const int32_t *context_lens,
                                          void *out, int64_t out_token_stride, int32_t batch,
                                          int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                          int32_t page_size, int64_t num_pages, int32_t max_q_len,
                                          int64_t num_tokens, int32_t key_slices, void *workspace,
                                          size_t workspace_bytes, float softmax_scale, void *stream) {
  litekv::PrefillKeySplit split;
  split.key_slices = key_slices;
  split.workspace = workspace;
  split.workspace_bytes = workspace_bytes;
  split.num_tokens = num_tokens;
  return litekv::launch_paged_prefill("paged_prefill_split", q, q_token_stride, kv_pool, nullptr,
                                      block_table, block_table_stride, cu_q_lens, context_lens, out,
                                      out_token_stride, batch, num_q_heads, num_kv_heads, head_dim,
                                      page_size, num_pages, max_q_len, softmax_scale, stream,
                                      litekv::kKvF16, split);
}

extern "C" int litekv_paged_prefill_split_q8(const void *q, int64_t q_token_stride, const void *kv_pool,
                                             const float *kv_scales, int32_t pool_is_int8,
                                             const int32_t *block_table, int32_t block_table_stride,
                                             const int32_t *cu_q_lens, const int32_t *context_lens,
                                             void *out, int64_t out_token_stride, int32_t batch,
                                             int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                             int32_t page_size, int64_t num_pages, int32_t max_q_len,
                                             int64_t num_tokens, int32_t key_slices, void *workspace,
                                             size_t workspace_bytes, float softmax_scale, void *stream) {
  litekv::PrefillKeySplit split;
  split.key_slices = key_slices;
  split.workspace = workspace;
  split.workspace_bytes = workspace_bytes;
  split.num_tokens = num_tokens;
  return litekv::launch_paged_prefill(pool_is_int8 ? "paged_prefill_split_int8" : "paged_prefill_split_fp8", q,
                                      q_token_stride, kv_pool, kv_scales, block_table, block_table_stride,
                                      cu_q_lens, context_lens, out, out_token_stride, batch, num_q_heads,
                                      num_kv_heads, head_dim, page_size, num_pages, max_q_len,
                                      softmax_scale, stream, pool_is_int8 ? litekv::kKvInt8 : litekv::kKvFp8,
                                      split);
}

extern "C" int litekv_paged_prefill_fp8(const void *q, int64_t q_token_stride, const void *kv_pool,
                                        const float *kv_scales, const int32_t *block_table,
                                        int32_t block_table_stride, const int32_t *cu_q_lens,
                                        const int32_t *context_lens, void *out,
                                        int64_t out_token_stride, int32_t batch,
                                        int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                        int32_t page_size, int64_t num_pages, int32_t max_q_len,
                                        float softmax_scale, void *stream) {
  return litekv::launch_paged_prefill("paged_prefill_fp8", q, q_token_stride, kv_pool, kv_scales,
                                      block_table, block_table_stride, cu_q_lens, context_lens, out,
                                      out_token_stride, batch, num_q_heads, num_kv_heads, head_dim,
                                      page_size, num_pages, max_q_len, softmax_scale, stream,
                                      litekv::kKvFp8, litekv::PrefillKeySplit{});
}

extern "C" int litekv_paged_prefill_int8(const void *q, int64_t q_token_stride, const void *kv_pool,
                                         const float *kv_scales, const int32_t *block_table,
                                         int32_t block_table_stride, const int32_t *cu_q_lens,
                                         const int32_t *context_lens, void *out,
                                         int64_t out_token_stride, int32_t batch,
                                         int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                         int32_t page_size, int64_t num_pages, int32_t max_q_len,
                                         float softmax_scale, void *stream) {
  return litekv::launch_paged_prefill("paged_prefill_int8", q, q_token_stride, kv_pool, kv_scales,
                                      block_table, block_table_stride, cu_q_lens, context_lens, out,
                                      out_token_stride, batch, num_q_heads, num_kv_heads, head_dim,
                                      page_size, num_pages, max_q_len, softmax_scale, stream,
                                      litekv::kKvInt8, litekv::PrefillKeySplit{});
}

// Where the keys of a launch over 4-bit codes lie as fp16, in its workspace behind the partial rows of its key slices. Decoded once
// they cost a launch and their bytes, some 14 us for 33 MB; decoded by every block of rows, a third of its tile loop. 512
// rows over 7601 tokens, 64 / 8 heads: 178 -> 153 us (fp16 pool: 129 to 135); 8 prompts of 128 to 2048 tokens 261 -> 236 (225 to
// 235); four chunks of up to 512 over up to 8000, 32 / 8 heads of 64, uncut, 163 -> 128 (107); 16 prompts of 1024 118 -> 107; 200 rows over
// 8000, 64 / 8 heads (13 blocks), 91 -> 83. With fewer blocks: 128 rows over 4000, 64 / 8 heads (8 blocks), 44 in both forms; 32 / 8 heads
// (4 blocks), 26.6 -> 33.8; 8 prompts of 512, 32 / 8 heads (16 blocks, a key attended by 8 on the average), 44.3 -> 45.3. Up to 1 GiB: a cache in 4 bits is there to save memory. (The room is the longest
// sequence's for each, whatever the others' lengths, which the host does not know: one of 8000 tokens and 15 short ones, 8 kv heads of
// 128, 537 MB for some 34 MB of keys; workgroups of tokens that a sequence has not leave at once.)
struct Int4Staging {
  int64_t capacity = 0;   // tokens of a sequence, 0: they are decoded where they are attended
  size_t table_at = 0, pool_at = 0, bytes = 0;
};
static Int4Staging int4_staging(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t max_q_len,
                                int64_t max_kv_len, int64_t num_tokens, int32_t key_slices) {
  Int4Staging s;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  s.table_at = up(litekv_paged_prefill_split_workspace_bytes(num_tokens, num_q_heads, head_dim, key_slices));
  s.bytes = s.table_at;
  if (batch < 1 || batch > 65535 || num_kv_heads < 1 || num_kv_heads > 1024 || num_q_heads < num_kv_heads || max_q_len < 1 ||
      max_kv_len < 1 || max_kv_len > 0x3fffffff) {
    return s;
  }
  // Blocks of rows that attend a key, on the average (a chunk's own keys by half of its blocks)
  const double blocks = (double)(((int64_t)(num_q_heads / num_kv_heads) * max_q_len + 127) / 128);
  const double visits = blocks * (1.0 - 0.5 * std::min<double>(1.0, (double)max_q_len / (double)max_kv_len));
  if (visits < 12.0) return s;
  const int64_t capacity = (max_kv_len + litekv::kInt4StagePage - 1) / litekv::kInt4StagePage * litekv::kInt4StagePage;
  const double bytes = (double)batch * (double)capacity * 4.0 * num_kv_heads * head_dim;
  if (bytes > 1073741824.0) return s;
  s.capacity = capacity;
  s.pool_at = s.table_at + up((size_t)batch * (size_t)(capacity / litekv::kInt4StagePage) * sizeof(int32_t));
  s.bytes = s.pool_at + (size_t)bytes;
  return s;
}

// As litekv_paged_prefill_key_slices, but two for three chunks and more over long histories that it leaves uncut: the launch then
// takes as long as its longest chain of keys, which chunks of one batch seldom share evenly. 4 chunks of up to 512 rows over 2000 to
// 8000 tokens, 32 / 8 heads of 64: 126 -> 97 us, of 128 175 -> 131; 3 of up to 400 over up to 30000 609 -> 467; 4 equal ones of 512
// over 8000 239 -> 234; 16 of up to 128 over up to 4000, heads of 64, 98 -> 84, but over up to 2000, heads of 128, 73 -> 75, 6 of up to
// 300 over up to 1000 48 -> 53, and two of up to 1000 over 4000 88 -> 104. (Other pools would gain as much.) One chunk of 64 rows, 16 / 8
// heads, in 8 slices takes 11 to 12 us with one key tile a slice over any pool (of them the merge 3.2, the rest one memory trip after another:
// lengths, page ids, keys, partial rows), and a tile more 0.7 us over fp16, 0.9 over int8 and 1.1 over 4-bit codes, whose conversion nothing
// covers in so short a chain.
extern "C" int32_t litekv_paged_prefill_int4_key_slices(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                        int32_t max_q_len, int64_t max_kv_len) {
  const int32_t slices = litekv_paged_prefill_key_slices(batch, num_q_heads, num_kv_heads, head_dim, max_q_len, max_kv_len);
  return slices == 1 && batch >= 3 && max_kv_len >= 3000 && max_kv_len >= 2 * (int64_t)max_q_len ? 2 : slices;
}

extern "C" size_t litekv_paged_prefill_int4_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                                            int32_t head_dim, int32_t max_q_len, int64_t max_kv_len,
                                                            int64_t num_tokens, int32_t key_slices) {
  if (!litekv::int4_head_dim(head_dim)) return 0;
  return int4_staging(batch, num_q_heads, num_kv_heads, head_dim, max_q_len, max_kv_len, num_tokens, key_slices).bytes;
}

extern "C" int litekv_paged_prefill_int4(const void *q, int64_t q_token_stride, const void *kv_pool_int4,
                                         const int32_t *block_table, int32_t block_table_stride,
                                         const int32_t *cu_q_lens, const int32_t *context_lens,
                                         void *out, int64_t out_token_stride, int32_t batch,
                                         int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                         int32_t page_size, int64_t num_pages, int32_t max_q_len,
                                         int64_t max_kv_len, int64_t num_tokens, int32_t key_slices,
                                         void *workspace, size_t workspace_bytes, float softmax_scale,
                                         void *stream) {
  using namespace litekv;
  const char *what = "paged_prefill_int4";
  LITEKV_REQUIRE(int4_head_dim(head_dim), "%s: head_dim %d unsupported (64 or 128)", what, head_dim);
  PrefillKeySplit split;
  split.key_slices = key_slices;
  split.workspace = workspace;
  split.workspace_bytes = workspace_bytes;
  split.num_tokens = num_tokens;
  split.max_kv_len = max_kv_len;
  int format = kKvInt4;
  const Int4Staging s = int4_staging(batch, num_q_heads, num_kv_heads, head_dim, max_q_len, max_kv_len, num_tokens, key_slices);
  if (s.capacity > 0 && workspace != nullptr && workspace_bytes >= s.bytes) {
    const int page_shift = page_shift_of(page_size);
    LITEKV_REQUIRE(page_shift >= 0, "%s: page_size %d unsupported (16, 32, 64, 128 or 256)", what, page_size);
    LITEKV_REQUIRE(kv_pool_int4 && block_table && cu_q_lens, "%s: null pointer", what);
    LITEKV_REQUIRE(aligned16(kv_pool_int4) && aligned16(workspace), "%s: kv_pool and workspace must be 16-byte aligned", what);
    LITEKV_REQUIRE(block_table_stride >= 1, "%s: block_table_stride %d < 1", what, block_table_stride);
    LITEKV_REQUIRE(num_pages >= 1 && num_pages <= 0x7fffffffLL / page_size, "%s: num_pages %lld out of range", what,
                   (long long)num_pages);
    char *base = static_cast<char *>(workspace);
    int32_t *table = reinterpret_cast<int32_t *>(base + s.table_at);
    const int rc = launch_int4_stage(what, kv_pool_int4, base + s.pool_at, table, block_table, block_table_stride, cu_q_lens,
                                     context_lens, batch, num_kv_heads, head_dim, page_shift, num_pages, s.capacity, stream);
    if (rc != LITEKV_OK) return rc;
    kv_pool_int4 = base + s.pool_at;
    block_table = table;
    block_table_stride = (int32_t)(s.capacity / kInt4StagePage);
    page_size = kInt4StagePage;
    num_pages = batch * (s.capacity / kInt4StagePage);
    format = kKvF16;
  }
  return launch_paged_prefill(what, q, q_token_stride, kv_pool_int4, nullptr, block_table, block_table_stride, cu_q_lens,
                              context_lens, out, out_token_stride, batch, num_q_heads, num_kv_heads, head_dim, page_size,
                              num_pages, max_q_len, softmax_scale, stream, format, split);
}

extern "C" int litekv_varlen_prefill(const void *q, int64_t q_token_stride, const void *k,
                                     int64_t k_token_stride, const void *v, int64_t v_token_stride,
                                     const int32_t *seq_starts, const int32_t *seq_lens, void *out,
                                     int64_t out_token_stride, int32_t batch, int32_t num_q_heads,
                                     int32_t num_kv_heads, int32_t head_dim, int32_t max_seq_len,
                                     int64_t num_tokens, float softmax_scale, void *stream) {
  return litekv::launch_varlen_prefill(q, q_token_stride, k, k_token_stride, v, v_token_stride,
                                       seq_starts, seq_lens, out, out_token_stride, batch,
                                       num_q_heads, num_kv_heads, head_dim, max_seq_len, num_tokens,
                                       softmax_scale, stream);
}
#endif  // LITEKV_HD == 128
