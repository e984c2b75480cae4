// Paged flash-decoding over a 4-bit pool (kv_int4.h): a workgroup per (sequence, kv head, split), whose wavefronts attend a
// part of the split's keys each; partial rows of several splits are merged by litekv_paged_decode_merge.
//
// The kernel works on the codes. With q the rows of up to 16 query heads of the kv head as columns, key i's score is
//     S[i] = s_i * (sum_d c_id q_d - z_i * sum_d q_d)
// and an output row
//     O[d] = sum_i (p_i s'_i) (c'_id - z'_i)       p = softmax of S, s', z', c' those of V
// so a scale and a zero point cost a few instructions per key instead of one per element. Codes reach the matrix cores with
// nothing but shifts and masks:
//  * K as int8: a nibble in the low half of a byte. q is a fixed-point number in four int8 digits to the base 256, with the row's
//    largest element between 2^29 and 2^30 units: elements are exact down to 2^-19 of the largest, off by half a unit below that.
//    Products of integers are exact, whatever they stand beside. (Three 8-bit floating-point numbers hold q as well, for 28 vector
//    instructions of a step fewer, but their matrix products add neighbours in a window of some 14 bits: beside one element of
//    300, scores were up to 6e-3 off.) S^T is four products of 16x16x64 per 16 keys, two with heads of 64, and twice as many
//    with more than 8 heads: up to 8, the columns that they leave empty take the lower two digits.
//  * V as fp16. c in bits 4 .. 7 is the subnormal c * 2^-20. The matrix cores take it as it is, but do not normalise it: the eight
//    products of a lane are lined up by the exponents of their factors and cut off some 24 bits below the largest. From bits 4 .. 7
//    that leaves 21 bits of a code's own size; in bits 0 .. 3, which need two instructions fewer for eight codes, 17 (333 keys with
//    one that carries nearly all of the weight: outputs 1e-5 of sum p |v| off, all to one side). For the same reason the z' are
//    summed by an MFMA of their own and taken off every kFold blocks, and not at the end from accumulators that would have
//    grown to some twenty times the result.
//
// A wavefront takes two blocks of 16 keys a step. S^T[key][col] is the accumulator of the first product and in the same lanes
// the right operand of the second, O^T[d][col] += V^T[d][key] P^T[key][col] (16x16x32): no LDS. p s' as fp16 would
// cost the result as much again as its own rounding, so it is kept as two fp16 numbers, the second what the first leaves. Up to
// 8 query heads leave half of the columns empty: there columns 0 .. 7 do the softmax of the first block and columns 8 .. 15 that of
// the second, and one exchange of 8 lanes makes the second product's operand, the first numbers in columns 0 .. 7, the others in
// 8 .. 15. With more heads a second MFMA takes the others.
//
// The reference of the exponentials is the largest p s' so far, not the largest p: in fp16 it is p s' that has to fit. It is put
// at 2^7 and may grow to 2^15 before the accumulators are rescaled.
//
// Bound: by what one compute unit takes in, some 40 GB/s at one sequence per head (32768 tokens on 8 compute units: 110 us), and by memory once
// there are as many workgroups as compute units: 64 sequences of 8192 tokens, 32 / 4 heads of 128, take 47 us, 5.9 TB/s of cache read (a
// large copy reads and writes 5.0). A step is 177 vector and 17 matrix instructions for 32 keys and 8 heads (D = 128), 219 and 34
// with more: 64 / 4 heads take 51 us over the same bytes, 8 sequences of 4096 tokens 24.0 with 16 heads per kv head and 19.4 with
// 8. 164 registers leave room for three wavefronts per SIMD with two steps' loads in flight each. Of its twelve wavefronts a
// compute unit holds one workgroup of eight or three of four. Eight are faster while there are no more workgroups than compute
// units (20 sequences of 4096, 8 kv heads: 20.8 us against 23.6; 4096 to 16384 tokens in 64: 71.6 against 80.4), four where there
// are more (38 of 4096: 37.1 against 41.8; 100 of 2048: 42.6 against 51.4). Streaming loads, whose lines are the first to leave the
// caches, suit a cache larger than those (the case above with ordinary ones: 52 us), as that of a model's layers one after the
// other is; inside them ordinary ones are faster (20 of 4096: 20.1 against 20.7).
//
// Around its keys a workgroup spends some 5 us, most of it one memory trip after another and the first run through its code: the
// sequence's length, block-table entries, keys, the fold. So q, the first 64 entries of the table row and the new rows are
// requested ahead of the length, q is converted once for the workgroup and not by every wavefront for itself (9.8 -> 8.2 us a launch
// for one sequence of 778 tokens, 22.0 -> 20.4 for 32 of 256 to 4096), and the last, masked steps are one piece of code
// (8.2 -> 7.6, with the fold's loads ahead of its arithmetic).
#include <type_traits>

#include "common.h"
#include "kv_int4.h"

namespace litekv {

typedef uint32_t uint2v_t __attribute__((ext_vector_type(2)));
typedef float float2v_t __attribute__((ext_vector_type(2)));

constexpr int kInt4Waves = 8;            // of a workgroup, at most
constexpr float kInt4Top = 7.0f;         // log2 of where the largest p s' is put
constexpr float kInt4Grown = 32768.0f;   // and what it may grow to
constexpr int kDepth = 2;                // steps whose loads are in flight
constexpr int kStreaming = 2;            // of a buffer load: not read again soon
constexpr int kFold = 32;                // blocks between two subtractions of the zero points
constexpr float kLog2eI4 = 1.4426950408889634f, kLn2I4 = 0.6931471805599453f;

// A block of 16 tokens as a lane (n = lane % 16, g = lane / 16) holds it: of K row n the g-th quarter, of V rows 4g .. 4g + 3
// column n, and the words of rows 4g .. 4g + 3 of both.
template <int D>
struct Int4Regs {
  uint32_t k[D / 32], v[D / 32];
  uint32_t kw[2], vw[2];
};

// Codes of K as the matrix cores take them in the first product: each nibble on its own in a byte.
typedef int int4v_t __attribute__((ext_vector_type(4)));
template <int D>
__device__ __forceinline__ void int4_k_bytes(const uint32_t (&k)[D / 32], int4v_t (&a)[D / 64]) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    a[i / 2][2 * (i & 1)] = (int)(k[i] & 0x0f0f0f0fu);
    a[i / 2][2 * (i & 1) + 1] = (int)((k[i] >> 4) & 0x0f0f0f0fu);
  }
}
// D(16x16) += A(16x64) * B(64x16), int8: lane l supplies 16 bytes of row (column) l % 16, at 16 * (l / 16).
__device__ __forceinline__ int4v_t mfma_16x16x64_i8(int4v_t a, int4v_t b, int4v_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// Eight codes of V in a dword as fp16 pairs, times 2^-20.
__device__ __forceinline__ void int4_pairs(uint32_t x, uint32_t (&out)[4]) {
  out[0] = (x << 4) & 0x00f000f0u;
  out[1] = x & 0x00f000f0u;
  out[2] = (x >> 4) & 0x00f000f0u;
  out[3] = (x >> 8) & 0x00f000f0u;
}
__device__ __forceinline__ half8_t as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(half8_t, uint4_t{a, b, c, d});
}

// TWO: more than 8 query heads, whose second part of p s' has MFMAs of its own.
template <int D, bool TWO>
__global__ __launch_bounds__(kInt4Waves *kWave) __attribute__((amdgpu_waves_per_eu(3, 3))) void paged_decode_int4_kernel(
    const half_t *__restrict__ q, int64_t q_batch_stride, uint8_t *pool, const int32_t *__restrict__ block_table,
    int32_t bt_stride, const int32_t *__restrict__ seq_lens, const half_t *__restrict__ k_new,
    const half_t *__restrict__ v_new, int64_t k_new_stride, int64_t v_new_stride, half_t *__restrict__ out,
    float *__restrict__ part_o, float *__restrict__ part_lse, int32_t num_q_heads, int32_t num_kv_heads,
    int32_t batch, int32_t group_all, int32_t slices, int32_t max_splits, int32_t min_pages_per_split,
    int32_t num_pages, int32_t page_shift, float scale_log2) {
  constexpr int kSteps = D / 32;   // MFMAs of a block's scores; dwords a lane holds of K and of V
  constexpr int kTiles = D / 16;   // 16-row tiles of O^T
  constexpr int kUnits = D / 64;   // see int4_v_unit
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  // Workgroups with the same pages -- the heads of a sequence's split, whose words share cache lines -- land on one XCD: they
  // are dealt out round robin, so eight (sequence, split) pairs' take turns. Splits are the slowest index: a launch of more
  // workgroups than the device holds ends with splits of one size.
  const int pairs = batch * max_splits, heads_x = gridDim.x / pairs;
  const int deal = (int)blockIdx.x / (8 * heads_x), at = (int)blockIdx.x - deal * 8 * heads_x;
  const int turns = pairs - 8 * deal < 8 ? pairs - 8 * deal : 8;
  const int pair = 8 * deal + at % turns;
  const int split = pair / batch, b = pair - split * batch;
  const HeadSlice hs = head_slice(at / turns, slices, group_all);
  const int share = (int)(blockDim.x >> 6), part = wave;   // the wavefronts attend a part of the split's keys each
  const int h = hs.kv_head, group = hs.q_heads, hq0 = hs.q_head0;
  constexpr int L = D / 8;                 // lanes of a row, 8 elements each
  constexpr int kHeads = TWO ? 16 : 8;     // rows of q (the last one again past the group)
  // What does not depend on the sequence's length is requested ahead of it: rows of q, the first entries of the block-table row (one
  // a lane), the step's new rows (K's in the first L lanes, V's in the next).
  const int32_t *row_of_table = block_table + (int64_t)b * bt_stride;
  const int first_entries = row_of_table[lane < bt_stride ? lane : bt_stride - 1];
  half8_t q_in = half8_t{0, 0, 0, 0, 0, 0, 0, 0}, new_row = q_in;
  if (wave < kHeads * L / kWave) {
    const int head = (int)threadIdx.x / L;
    q_in = *(const half8_t *)(q + (int64_t)b * q_batch_stride + (int64_t)(hq0 + (head < group ? head : group - 1)) * D +
                              8 * (threadIdx.x % L));
  }
  if (k_new != nullptr) {
    const half_t *src = lane & L ? v_new + (int64_t)b * v_new_stride : k_new + (int64_t)b * k_new_stride;
    new_row = *(const half8_t *)(src + (int64_t)h * D + 8 * (lane & (L - 1)));
  }
  const int len = as_uniform(seq_lens)[b];
  half_t *out_row = out + ((int64_t)b * num_q_heads + hq0) * D;
  if (len <= 0) {
    if (split == 0 && part == 0) {
      for (int i = lane; i < group * (D / 8); i += kWave) *(half8_t *)(out_row + 8 * i) = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
    }
    return;
  }
  const int pages = pages_of(len);
  const int n_splits = splits_for_pages(pages, max_splits, min_pages_per_split);
  if (split >= n_splits) return;
  const int first = (int)(((int64_t)split * pages) / n_splits);
  const int last = (int)(((int64_t)(split + 1) * pages) / n_splits);
  const int steps = (last - first + 1) / 2;   // of two blocks
  // (the last wavefront, which has the new token and the keys to be masked, has no more of them than the others)
  const int p0 = first + 2 * ((steps * part + share - 1) / share);
  const int p1_even = first + 2 * ((steps * (part + 1) + share - 1) / share);
  const int p1 = p1_even < last ? p1_even : last;
  const bool any = p0 < p1;   // (a wavefront without a part has nothing to add)

  const int64_t block_bytes = int4_block_bytes(num_kv_heads, D);
  // The block-table entry of a page, and the block it means. A length beyond what a row can name re-reads the row's last entry;
  // pages past the wavefront's last re-read that.
  auto place = [&](int p) {
    const int pp = p < p1 ? p : p1 - 1;
    return pp > 0 ? pp : 0;
  };
  auto entry_at = [&](int p) {
    const int at = place(p) >> page_shift;
    return at < bt_stride ? at : bt_stride - 1;
  };
  auto entry_of = [&](int p) { return as_uniform(row_of_table)[entry_at(p)]; };
  auto first_entry_of = [&](int p) {   // from the registers where it is there
    const int at = entry_at(p);
    return at < kWave ? __builtin_amdgcn_readlane(first_entries, at) : entry_of(p);
  };
  auto block_of = [&](int p, int entry) { return sub_page_id(entry, place(p), page_shift, num_pages); };

  // The step's new token goes into the last block before anything of it is read (by this wavefront, the only one that reads it
  // in this launch; the slices of a wide group all write the same bytes).
  if (k_new != nullptr && any && p1 == pages && pages <= (bt_stride << page_shift)) {
    const int entry = first_entry_of(pages - 1);
    if (lane < 2 * L && names_page(entry, num_pages)) {
      const bool is_v = lane >= L;
      const int l = lane & (L - 1);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)new_row[i];
      const int64_t slot = (int64_t)block_of(pages - 1, entry) * kInt4Block + ((len - 1) & (kInt4Block - 1));
      int4_store<D>(pool, slot, num_kv_heads, is_v ? num_kv_heads + h : h, l, int4_row<L>(x));
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the stores are done
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  }

  const uint32_t k_off = (uint32_t)(int4_codes_at(h, D) + n * (D / 2) + g * (D / 8));
  const uint32_t v_off = (uint32_t)(int4_codes_at(num_kv_heads + h, D) + g * (2 * D) + n * (D / 8));
  const uint32_t kw_off = (uint32_t)(int4_words_at(h, num_kv_heads, D) + 8 * g);
  const uint32_t vw_off = (uint32_t)(int4_words_at(num_kv_heads + h, num_kv_heads, D) + 8 * g);
  // Loads of pages past the split's last name a buffer of no bytes: they return zeros and touch no memory, and the loop has the
  // same number of them in flight at every step, so that each wait covers the page it needs and no younger one.
  auto request = [&](int p, int entry, Int4Regs<D> &r) {
    const auto block = __builtin_amdgcn_make_buffer_rsrc(pool + (int64_t)block_of(p, entry) * block_bytes, 0, p < p1 ? (int)block_bytes : 0,
                                                         0x00020000);
    if constexpr (D == 128) {
      const uint4_t kk = __builtin_amdgcn_raw_buffer_load_b128(block, k_off, 0, kStreaming);
      const uint4_t vv = __builtin_amdgcn_raw_buffer_load_b128(block, v_off, 0, kStreaming);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        r.k[i] = kk[i];
        r.v[i] = vv[i];
      }
    } else {
      const uint2v_t kk = __builtin_amdgcn_raw_buffer_load_b64(block, k_off, 0, kStreaming);
      const uint2v_t vv = __builtin_amdgcn_raw_buffer_load_b64(block, v_off, 0, kStreaming);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        r.k[i] = kk[i];
        r.v[i] = vv[i];
      }
    }
    const uint2v_t kw = __builtin_amdgcn_raw_buffer_load_b64(block, kw_off, 0, 0);
    const uint2v_t vw = __builtin_amdgcn_raw_buffer_load_b64(block, vw_off, 0, 0);
    r.kw[0] = kw[0];
    r.kw[1] = kw[1];
    r.vw[0] = vw[0];
    r.vw[1] = vw[1];
  };
  // Two blocks a step, kDepth steps' in flight. Block-table entries are read a step before the requests that they are for, and not
  // looked at before: a scalar load that is waited for on the spot cost every step its whole trip.
  Int4Regs<D> buf[kDepth][2];
  int entry0 = first_entry_of(p0), entry1 = first_entry_of(p0 + 1);
  auto request_pair = [&](int p, Int4Regs<D> (&r)[2]) {
    request(p, entry0, r[0]);
    request(p + 1, entry1, r[1]);
    entry0 = entry_of(p + 2);
    entry1 = entry_of(p + 3);
  };
#pragma unroll
  for (int i = 0; i < kDepth; ++i) request_pair(p0 + 2 * i, buf[i]);

  // q as the right operand of the first product: column n, the elements of the bytes that the lane of the same g holds of K,
  // in four digits. Up to 8 heads: the upper two in columns 0 .. 7, the lower two in 8 .. 15. More: the lower two in a sum of their own.
  // Made once for the workgroup and handed out through LDS.
  constexpr int kDigits = 4, kSets = TWO ? 4 : 2;   // of a row; of a lane's column
  constexpr float kUpper = 0x1p16f;                 // what a sum over the upper two counts for
  extern __shared__ __attribute__((aligned(16))) float int4_lds[];
  constexpr int kRowBytes = kDigits * D + 16;                 // of a row of q: the digits, the sum and the factor of its scores
  char *const q_rows = (char *)int4_lds;
  float *const int4_rows = int4_lds + kHeads * kRowBytes / 4;
  if (wave < kHeads * L / kWave) {
    const int l = threadIdx.x % L;
    char *row = q_rows + (threadIdx.x / L) * kRowBytes;
    float x[8], most = 0.f, sum = 0.f, odd = 0.f;   // odd: an element that is not finite
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = (float)q_in[i];
      most = __builtin_fmaxf(most, __builtin_fabsf(x[i]));
      odd = __builtin_fabsf(x[i]) < INFINITY ? odd : 1.f;
    }
    most = over_row<L>(most, [](float a, float b) { return __builtin_fmaxf(a, b); });
    odd = over_row<L>(odd, [](float a, float b) { return a + b; });
    const int up = most > 0.f ? 30 - __builtin_amdgcn_frexp_expf(most) : 0;
    uint32_t digits[8];   // an element's, lowest first: signed, since each borrows 128 from the next
    constexpr uint32_t kBorrow = 0x00808080u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float units = __builtin_rintf(__builtin_amdgcn_ldexpf(x[i], up));
      sum += units;
      digits[i] = ((uint32_t)(odd > 0.f ? 0 : (int)units) + kBorrow) ^ kBorrow;
    }
#pragma unroll
    for (int of = 0; of < kDigits; ++of) {   // highest digit first
      const uint32_t sel = (uint32_t)(kDigits - 1 - of);
      uint2v_t bytes;   // elements of the lower and of the upper nibbles
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        constexpr int kOrder[2][4] = {{0, 4, 1, 5}, {2, 6, 3, 7}};
        const uint32_t low = __builtin_amdgcn_perm(digits[kOrder[u][1]], digits[kOrder[u][0]], 0x0c0c0000u | ((sel + 4) << 8) | sel);
        const uint32_t high = __builtin_amdgcn_perm(digits[kOrder[u][3]], digits[kOrder[u][2]], 0x00000c0cu | ((sel + 4) << 24) | (sel << 16));
        bytes[u] = low | high;
      }
      *(uint2v_t *)(row + of * D + 8 * l) = bytes;
    }
    sum = over_row<L>(sum, [](float a, float b) { return a + b; });
    if (l == 0) {
      const float mul = odd > 0.f ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(scale_log2, -up);
      *(float2v_t *)(row + kDigits * D) = float2v_t{sum * 0x1p24f * mul, mul};   // (the zero points come as z * 2^-24)
    }
  }
  __syncthreads();
  int4v_t qf[kSets][D / 64];
  float q_sum, mul_own, mul_other;   // of the lane's own sums, and of those that it gets (TWO: of the upper digits' sums, of the lower ones')
  {
    const char *row = q_rows + (TWO ? n : (n & 7)) * kRowBytes;
    const float2v_t both = *(const float2v_t *)(row + kDigits * D);
    q_sum = both[0];
    mul_own = TWO || n < 8 ? both[1] * kUpper : both[1];
    mul_other = TWO || n < 8 ? both[1] : both[1] * kUpper;
    if constexpr (!TWO) row += n < 8 ? 0 : 2 * D;
#pragma unroll
    for (int of = 0; of < kSets; ++of) {
#pragma unroll
      for (int j = 0; j < D / 64; ++j) qf[of][j] = *(const int4v_t *)(row + of * D + (D / 4) * g + 16 * j);   // of two dwords of K
    }
  }
  const bool second = n >= 8;   // !TWO: the lane's scores are those of the second block's keys

  // O^T, and what is to be subtracted from every element of it (see kFold)
  float4_t acc[kTiles], acc_z = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < kTiles; ++j) acc[j] = float4_t{0.f, 0.f, 0.f, 0.f};
  auto fold_zeros = [&]() {
#pragma unroll
    for (int j = 0; j < kTiles; ++j) acc[j] -= acc_z;
    acc_z = float4_t{0.f, 0.f, 0.f, 0.f};
  };
  float ref = -1e30f, total = 0.f;   // reference of the exponentials; sum of p
  const int end = len < p1 * kInt4Block ? len : p1 * kInt4Block;

  auto attend = [&](Int4Regs<D> (&r)[2], int p, auto masked_tag) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    constexpr int kKeys = TWO ? 8 : 4;   // keys a lane has the scores of: of its column all of 4g .. 4g + 3, or one block's
    int4v_t st[2], st_low[2];   // sums over two digits; TWO: over the upper and the lower two
    int4v_t a[2][D / 64];
#pragma unroll
    for (int u = 0; u < 2; ++u) int4_k_bytes<D>(r[u].k, a[u]);
    auto add_digit = [&](const int4v_t (&digit)[D / 64], int4v_t (&sums)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int j = 0; j < D / 64; ++j) sums[u] = mfma_16x16x64_i8(a[u][j], digit[j], sums[u]);
      }
    };
    auto two_digits = [&](const int4v_t (&high)[D / 64], const int4v_t (&low)[D / 64], int4v_t (&sums)[2]) {
      sums[0] = sums[1] = int4v_t{0, 0, 0, 0};
      add_digit(high, sums);
      sums[0] <<= 8;
      sums[1] <<= 8;
      add_digit(low, sums);
    };
    two_digits(qf[0], qf[1], st);
    if constexpr (TWO) two_digits(qf[2], qf[3], st_low);
    uint32_t kw[kKeys / 2], vw[kKeys / 2];   // words of the lane's keys 2i, 2i + 1
    uint32_t vz[4];                          // z' of the eight keys of its g, times 2^-20
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (MASKED) {
        // rows past the end: finite values for zero probabilities to multiply
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int left = end - (p + u) * kInt4Block - 4 * g - 2 * i;
          const uint32_t keep = left >= 2 ? ~0u : left == 1 ? 0xffffu : 0u;
          r[u].kw[i] &= keep;
          r[u].vw[i] &= keep;
        }
      }
      vz[i] = (r[0].vw[i] << 4) & 0x00f000f0u;
      vz[2 + i] = (r[1].vw[i] << 4) & 0x00f000f0u;
      if constexpr (TWO) {
        kw[i] = r[0].kw[i];
        kw[2 + i] = r[1].kw[i];
        vw[i] = r[0].vw[i];
        vw[2 + i] = r[1].vw[i];
      } else {
        kw[i] = second ? r[1].kw[i] : r[0].kw[i];
        vw[i] = second ? r[1].vw[i] : r[0].vw[i];
      }
    }
    float x[kKeys], vs[kKeys];   // scores in log2 units, scales of V
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const half2_t ks = int4_scales(kw[i >> 1]), kz = __builtin_bit_cast(half2_t, kw[i >> 1] & 0x000f000fu);
      vs[i] = (float)int4_scales(vw[i >> 1])[i & 1];
      // (the other digits of the block that the lane's scores are of are in the other half of the columns)
      const float own = (float)(TWO ? st[i >> 2][i & 3] : second ? st[1][i] : st[0][i]);
      const float other = TWO ? (float)st_low[i >> 2][i & 3] : dpp<kDppRotate8>((float)(second ? st[0][i] : st[1][i]));
      const float dot = __builtin_fmaf(-(float)kz[i & 1], q_sum, own * mul_own);
      x[i] = __builtin_fmaf(other, mul_other, dot) * (float)ks[i & 1];
      if constexpr (MASKED) {
        const int u = TWO ? i >> 2 : second ? 1 : 0;
        if ((p + u) * kInt4Block + 4 * g + (i & 3) >= end) x[i] = -INFINITY;
      }
    }
    float w[kKeys], sum;   // p s'; sum of p
    auto exponentials = [&]() {
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        const float pr = fast_exp2(x[i] - ref);
        sum += pr;
        w[i] = __builtin_fmaf(pr, vs[i], 0.0f);
      }
    };
    exponentials();
    float most = sum * 0x1p-40f;   // (p alone may outgrow fp32 where s' is tiny or 0)
#pragma unroll
    for (int i = 0; i < kKeys; ++i) most = __builtin_fmaxf(most, w[i]);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(most > kInt4Grown) != 0, false)) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        top = __builtin_fmaxf(top, x[i] + fast_log2(__builtin_fmaxf(vs[i], 0x1p-24f)));
      }
      if constexpr (!TWO) top = __builtin_fmaxf(top, dpp<kDppRotate8>(top));
      top = __builtin_fmaxf(top, xor_lane(top, 16));
      top = __builtin_fmaxf(top, xor_lane(top, 32)) - kInt4Top;
      const float next = __builtin_fmaxf(ref, top);
      const float alpha = fast_exp2(ref - next);
      ref = next;
      total *= alpha;
      acc_z *= alpha;
#pragma unroll
      for (int j = 0; j < kTiles; ++j) acc[j] *= alpha;
      exponentials();
    }
    total += sum;
    // p s' as two fp16 numbers, the second what the first leaves, of keys 2i, 2i + 1
    auto toward_zero = [&](float a, float b) {
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    };
    uint32_t hi[kKeys / 2], lo[kKeys / 2];
#pragma unroll
    for (int i = 0; i < kKeys / 2; ++i) {
      hi[i] = toward_zero(w[2 * i], w[2 * i + 1]);
      const half2_t off = __builtin_bit_cast(half2_t, hi[i]);
      lo[i] = toward_zero(w[2 * i] - (float)off[0], w[2 * i + 1] - (float)off[1]);
    }
    half8_t ph, pl;
    if constexpr (TWO) {
      ph = as_half8(hi[0], hi[1], hi[2], hi[3]);
      pl = as_half8(lo[0], lo[1], lo[2], lo[3]);
      acc_z = mfma_16x16x32(as_half8(vz[0], vz[1], vz[2], vz[3]), ph, acc_z);
      acc_z = mfma_16x16x32(as_half8(vz[0], vz[1], vz[2], vz[3]), pl, acc_z);
    } else {
      // columns 0 .. 7 carry the first numbers of both blocks' keys, columns 8 .. 15 the second: each half has one block's
      uint32_t x0[2], x1[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x0[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)hi[i], (int)lo[i], kDppRotate8, 0xf, 0xc, false);
        x1[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)lo[i], (int)hi[i], kDppRotate8, 0xf, 0x3, false);
      }
      ph = pl = as_half8(x0[0], x0[1], x1[0], x1[1]);
      acc_z = mfma_16x16x32(as_half8(vz[0], vz[1], vz[2], vz[3]), ph, acc_z);
    }
#pragma unroll
    for (int e = 0; e < kUnits; ++e) {
      uint32_t x0[4], x1[4], x2[4], x3[4];   // rows 4g, 4g + 1 of the first block, 4g + 2, 4g + 3, the same of the second
      int4_pairs(r[0].v[e], x0);
      int4_pairs(r[0].v[kUnits + e], x1);
      int4_pairs(r[1].v[e], x2);
      int4_pairs(r[1].v[kUnits + e], x3);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const half8_t a = as_half8(x0[j], x1[j], x2[j], x3[j]);
        acc[4 * e + j] = mfma_16x16x32(a, ph, acc[4 * e + j]);
        if constexpr (TWO) acc[4 * e + j] = mfma_16x16x32(a, pl, acc[4 * e + j]);
      }
    }
  };

  int p = p0;
  int fold_at = p + kFold;
  while ((p + 2 * kDepth) * kInt4Block <= end) {
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      attend(buf[i], p + 2 * i, std::false_type{});
      request_pair(p + 2 * i + 2 * kDepth, buf[i]);
    }
    p += 2 * kDepth;
    if (p >= fold_at) {
      fold_zeros();
      fold_at = p + kFold;
    }
  }
  static_assert(kDepth == 2, "the last steps, one after the other");
#pragma unroll 1
  for (; p < p1; p += 2) {
    attend(buf[0], p, std::true_type{});
#pragma unroll
    for (int u = 0; u < 2; ++u) buf[0][u] = buf[1][u];
  }

  fold_zeros();
  if constexpr (!TWO) total += dpp<kDppRotate8>(total);
  total += xor_lane(total, 16);
  total += xor_lane(total, 32);
  const int head = TWO ? n : (n & 7);
  const bool whole = n_splits == 1;
  const int64_t cell0 = ((int64_t)b * num_q_heads + hq0) * max_splits + split;
  // O^T tile (e, j): row m is element m * D / 16 + kUnits * j + e of the output row; a lane has rows 4g .. 4g + 3: row i of them
  // as kTiles neighbours of the output row, from (4g + i) * kTiles on
  auto elements = [&](int i, float scale, float (&y)[kTiles]) {
#pragma unroll
    for (int e = 0; e < kUnits; ++e) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a = acc[4 * e + j][i];
        if constexpr (!TWO) a += dpp<kDppRotate8>(a);
        y[kUnits * j + e] = a * scale;
      }
    }
  };
  // (!TWO: both halves of the columns have the rows, each stores two of the four)
  auto mine = [&](int i) { return head < group && (TWO || (i >> 1) == (n >> 3)); };
  // The wavefronts that share a split leave their rows, references and sums in LDS, and fold them in order.
  constexpr int kArea = kHeads * D + 32;   // of a wavefront: rows, references, sums
  float *area = int4_rows + part * kArea;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[kTiles];
    elements(i, 0x1p20f, y);
    if (!mine(i)) continue;
#pragma unroll
    for (int j = 0; j < kTiles; j += 4) {
      *(float4_t *)(area + head * D + (4 * g + i) * kTiles + j) = float4_t{y[j], y[j + 1], y[j + 2], y[j + 3]};
    }
  }
  if (g == 0 && n < kHeads) {
    area[kHeads * D + n] = ref;
    area[kHeads * D + 16 + n] = total;
  }
  __syncthreads();
  for (int i = part * kWave + lane; i < group * (D / 4); i += share * kWave) {
    const int of = i / (D / 4), at_row = 4 * (i % (D / 4));
    const float *stats = int4_rows + kHeads * D + of;
    float refs[kInt4Waves], sums[kInt4Waves];
    float4_t parts[kInt4Waves];
#pragma unroll
    for (int s = 0; s < kInt4Waves; ++s) {
      const int at = s < share ? s : share - 1;
      refs[s] = stats[at * kArea];
      sums[s] = stats[at * kArea + 16];
      parts[s] = *(const float4_t *)(int4_rows + at * kArea + of * D + at_row);
    }
    float top = refs[0];
#pragma unroll
    for (int s = 1; s < kInt4Waves; ++s) top = __builtin_fmaxf(top, refs[s]);
    float sum = 0.f;
    float4_t y = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kInt4Waves; ++s) {
      const float weight = s < share ? fast_exp2(refs[s] - top) : 0.f;
      sum += weight * sums[s];
      y += weight * parts[s];
    }
    y *= 1.0f / sum;
    if (whole) {
      *(half4_t *)(out_row + (int64_t)of * D + at_row) = half4_t{(half_t)y[0], (half_t)y[1], (half_t)y[2], (half_t)y[3]};
    } else {
      const int64_t cell = cell0 + (int64_t)of * max_splits;
      __builtin_nontemporal_store(y, (float4_t *)(part_o + cell * D + at_row));
      if (at_row == 0) __builtin_nontemporal_store((top + fast_log2(sum)) * kLn2I4, part_lse + cell);
    }
  }
}

}  // namespace litekv

// Up to 256 (sequence, kv head) pairs, a compute unit has at most one, and splits fill the device: of 512 tokens and more where
// the longest sequence has over 1024 (8 kv heads: one sequence of 2000 tokens in splits of 512 / 1024 tokens, or unsplit, 9.6 / 11.0 /
// 11.8 us, six of 2048 10.2 / 11.7 / 12.2, eight of 4096 in splits of 1024 / 2048 12.9 / 15.3, unsplit 19.1; one of 778 in two 9.4 us, unsplit
// 7.7). With more, splits only even out the lengths and the last turn of the workgroups, from 4096 tokens a split (in splits of 1024 /
// 2048 / 4096 tokens, 8 kv heads: 40 sequences of 16384 131 / 117 / 110 us, 131 unsplit; 64 of them, which are even as they are, 199 / 182 /
// 177, 171 unsplit: the rule does not look at that, and costs them 3%).
// No more than 16 where that makes them shorter than 4096 tokens: their merge takes longer the more there are (one sequence of 32768
// tokens, 8 kv heads: 8 / 16 / 32 splits 22.7 / 17.4 / 19.5 us). Powers of two: a captured step holds their number, and growing
// sequences should not ask for a new one every thousand tokens.
extern "C" int32_t litekv_paged_decode_int4_splits(int32_t batch, int32_t num_kv_heads, int64_t max_pages, int64_t total_pages,
                                                   int32_t page_size, int32_t *min_pages_per_split) {
  using namespace litekv;
  if (batch < 0 || num_kv_heads < 1 || max_pages < 0 || max_pages > 0x7fffffff || total_pages > (int64_t)batch * max_pages ||
      page_shift_of(page_size) < 0 || min_pages_per_split == nullptr) {
    return 0;
  }
  const int64_t pairs = (int64_t)batch * num_kv_heads;
  const bool few = pairs <= 256;
  const int64_t least = (few ? 512 : 4096) / page_size;
  *min_pages_per_split = (int32_t)least;
  if (max_pages * page_size <= 1024) return 1;
  int64_t most = max_pages * page_size / 4096 > 16 ? max_pages * page_size / 4096 : 16;
  if (few) {
    const int64_t rows = total_pages < 0 ? pairs * max_pages : total_pages * num_kv_heads;   // of pages, a head's share each
    const int64_t fill = 256 * max_pages / (rows > 0 ? rows : 1);
    if (most > fill) most = fill;
  }
  int64_t splits = 1;
  while (2 * splits <= most && splits * least < max_pages && splits < 32768) splits *= 2;
  return (int32_t)splits;
}

extern "C" int litekv_paged_decode_int4(const void *q, int64_t q_batch_stride, void *kv_pool_int4,
                                        const int32_t *block_table, int32_t block_table_stride,
                                        const int32_t *seq_lens, const void *k_new, const void *v_new,
                                        int64_t k_new_stride, int64_t v_new_stride, void *out, void *workspace,
                                        size_t workspace_bytes, int32_t batch, int32_t num_q_heads,
                                        int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int64_t num_pages,
                                        int32_t max_splits, int32_t min_pages_per_split, float softmax_scale,
                                        void *stream) {
  using namespace litekv;
  const char *what = "paged_decode_int4";
  LITEKV_REQUIRE(max_splits >= 1 && max_splits <= 65535, "%s: max_splits %d out of [1, 65535]", what, max_splits);
  LITEKV_REQUIRE(min_pages_per_split >= 1, "%s: min_pages_per_split %d < 1", what, min_pages_per_split);
  LITEKV_REQUIRE(batch >= 0 && batch <= 65535, "%s: batch %d out of [0, 65535]", what, batch);
  LITEKV_REQUIRE(int4_head_dim(head_dim), "%s: head_dim %d unsupported (64 or 128)", what, head_dim);
  const int page_shift = page_shift_of(page_size);
  LITEKV_REQUIRE(page_shift >= 0, "%s: page_size %d unsupported (16, 32, 64, 128 or 256)", what, page_size);
  LITEKV_REQUIRE(num_q_heads > 0 && num_q_heads <= 65535 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
                 "%s: num_q_heads %d / num_kv_heads %d invalid", what, num_q_heads, num_kv_heads);
  const int group = num_q_heads / num_kv_heads;
  LITEKV_REQUIRE(group <= kMaxGroup, "%s: %d query heads per kv head unsupported (max %d)", what, group, kMaxGroup);
  LITEKV_REQUIRE(num_kv_heads <= 1024, "%s: num_kv_heads %d > 1024", what, num_kv_heads);
  if (batch == 0) {
    clear_error();
    return LITEKV_OK;
  }
  LITEKV_REQUIRE(q && kv_pool_int4 && block_table && seq_lens && out, "%s: null pointer", what);
  LITEKV_REQUIRE((k_new == nullptr) == (v_new == nullptr), "%s: k_new and v_new go together", what);
  LITEKV_REQUIRE(aligned16(q) && aligned16(kv_pool_int4) && aligned16(out) && aligned16(k_new) && aligned16(v_new),
                 "%s: q, kv_pool, out, k_new and v_new must be 16-byte aligned", what);
  LITEKV_REQUIRE(q_batch_stride >= (int64_t)num_q_heads * head_dim && q_batch_stride % 8 == 0,
                 "%s: q_batch_stride %lld invalid", what, (long long)q_batch_stride);
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  LITEKV_REQUIRE(k_new == nullptr || (k_new_stride >= row && v_new_stride >= row && k_new_stride % 8 == 0 &&
                                      v_new_stride % 8 == 0),
                 "%s: k_new/v_new strides (%lld, %lld) invalid", what, (long long)k_new_stride, (long long)v_new_stride);
  LITEKV_REQUIRE(block_table_stride >= 1 &&
                     (int64_t)block_table_stride * (page_size / kPageSize) <= 0x7fffffffLL / 4,
                 "%s: block_table_stride %d out of range", what, block_table_stride);
  LITEKV_REQUIRE(num_pages >= 1 && num_pages <= 0x7fffffffLL / page_size, "%s: num_pages %lld out of range", what,
                 (long long)num_pages);
  const size_t need = litekv_paged_decode_workspace_bytes(batch, num_q_heads, head_dim, max_splits);
  LITEKV_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && aligned16(workspace)),
                 "%s: 16-byte aligned workspace of %zu bytes needed, got %zu", what, need,
                 workspace ? workspace_bytes : (size_t)0);
  // (the kernels count in 16-token pages; saturating)
  const int64_t min16 = (int64_t)min_pages_per_split * (page_size / kPageSize);
  const int slices = head_slices(group);
  const int slice_heads = num_kv_heads * slices;
  LITEKV_REQUIRE(slice_heads <= 65535, "%s: num_q_heads %d too large", what, num_q_heads);
  float *part_o = max_splits > 1 ? static_cast<float *>(workspace) : nullptr;
  float *part_lse = max_splits > 1 ? part_o + (size_t)batch * num_q_heads * max_splits * head_dim : nullptr;
  const int64_t units = (int64_t)batch * slice_heads * max_splits;
  // (256 compute units: see the top of the file)
  const int share = units > 256 ? kInt4Waves / 2 : kInt4Waves;
  LITEKV_REQUIRE(units <= 0x7fffffffLL / 8, "%s: too many workgroups", what);
  const bool two = (group + slices - 1) / slices > 8;
  const int heads = two ? 16 : 8;
  const size_t lds = (size_t)share * (heads * head_dim + 32) * sizeof(float) + (size_t)heads * (4 * head_dim + 16);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)units), dim3((unsigned)(share * kWave)), lds,
                       static_cast<hipStream_t>(stream), static_cast<const half_t *>(q), q_batch_stride,
                       static_cast<uint8_t *>(kv_pool_int4), block_table, block_table_stride, seq_lens,
                       static_cast<const half_t *>(k_new), static_cast<const half_t *>(v_new), k_new_stride,
                       v_new_stride, static_cast<half_t *>(out), part_o, part_lse, num_q_heads, num_kv_heads, batch, group,
                       slices, max_splits, (int32_t)(min16 < 0x7fffffffLL ? min16 : 0x7fffffffLL),
                       (int32_t)num_pages, page_shift, softmax_scale * kLog2eI4);
  };
  if (head_dim == 64) {
    two ? launch(paged_decode_int4_kernel<64, true>) : launch(paged_decode_int4_kernel<64, false>);
  } else {
    two ? launch(paged_decode_int4_kernel<128, true>) : launch(paged_decode_int4_kernel<128, false>);
  }
  const int rc = check_launch(what);
  if (rc != LITEKV_OK || max_splits == 1) return rc;
  return litekv_paged_decode_merge(seq_lens, out, workspace, workspace_bytes, batch, num_q_heads, head_dim, page_size,
                                   max_splits, min_pages_per_split, stream);
}
