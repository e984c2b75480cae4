// 4-bit storage of K/V rows. Every row (token, kv head) is quantised over its own range, 0 included:
//     lo = min(0, min x)   hi = max(0, max x)
//     s  = (hi - lo) / 15, rounded up to 7 significant bits (below 2^-14: to a multiple of 2^-20)
//     z  = rint(-lo / s)   c = clamp(rint(x / s) + z, 0, 15)          halves go to the even integer
//     value = s * (c - z)
// c - z has 4 bits and a sign and s has 7, so every value is an fp16 number: attention over a 4-bit pool is fp16
// attention over the values, whether a kernel forms them or works on the codes and applies s and z afterwards. (Rounded up,
// s loses at most 2^-6 of its size, and no element of the row is further than s / 2 from its value.) Elements
// saturate at +-57344, where s * (c - z) is still finite, and NaN counts as 0. With s == 0 (a row of zeros) every code is 0.
//
// Layout: 16 consecutive slots are a block of 2 * Hkv * (8 * D + 32) bytes, in a pool
// uint8 [slots][2 * Hkv][D / 2 + 2], so that a page is one contiguous run whatever its size. The block holds
//     codes [2 * Hkv][8 * D bytes]     heads [0, Hkv) are K, [Hkv, 2 * Hkv) V
//     words [2 * Hkv][16] uint16       fp16 bits of s (its low 4 mantissa bits are 0) | z
// A K head's codes are its 16 rows of D / 2 bytes: dword w of a row holds elements 8w .. 8w + 7, element 8w + 2i in
// nibble i and 8w + 2i + 1 in nibble 4 + i, so that a dword masked with 0x000f000f, shifted or not, is a pair of
// neighbours. A V head's codes are laid out as a wavefront feeds them to the second product: for rows 4g .. 4g + 3 and
// column c of 16 (D / 16 elements each) the D / 8 bytes are dwords (p, e), whose low half is row 4g + 2p and
// high half row 4g + 2p + 1: nibble j is element c * D / 16 + (D / 64) * j + e of the row. One dwordx4 (D = 64: x2) per
// lane then is a matrix operand's worth of V, 1 KiB per wavefront, with no trip through LDS. A row never shares a byte with
// another, so rows are appended with plain stores.
#pragma once

#include "kv_fp8.h"

namespace litekv {

constexpr int kKvInt4 = 3;                 // beside kKvF16, kKvFp8 and kKvInt8
constexpr int kInt4Block = 16;             // slots of a block
constexpr float kInt4Most = 57344.0f;      // where elements saturate

__host__ __device__ constexpr bool int4_head_dim(int d) { return d == 64 || d == 128; }
__host__ __device__ constexpr int64_t int4_block_bytes(int kv_heads, int d) {
  return (int64_t)2 * kv_heads * (8 * d + 2 * kInt4Block);
}
// Inside a block: where the codes of head `head` (V heads counted behind the K heads) and its words begin.
__host__ __device__ constexpr int int4_codes_at(int head, int d) { return head * 8 * d; }
__host__ __device__ constexpr int int4_words_at(int head, int kv_heads, int d) {
  return 2 * kv_heads * 8 * d + head * 2 * kInt4Block;
}
// The keys of a prefill launch decoded once (see kv_int4.hip): fp16 pages of kInt4StagePage tokens and their block table.
constexpr int kInt4StagePage = 256;
// The block-table entry of 16-token page p of a sequence with that many keys, -1 for a page that it has not: the row may end behind
// its last one. (A sequence with more keys than the row can name re-reads the row's last entry.)
__host__ __device__ constexpr int int4_stage_entry(int p, int64_t keys, int page_shift, int bt_stride) {
  if (p < 0 || (int64_t)p * kInt4Block >= keys) return -1;
  return (p >> page_shift) < bt_stride ? p >> page_shift : bt_stride - 1;
}
int launch_int4_stage(const char *what, const void *pool, void *staged, int32_t *staged_table, const int32_t *block_table,
                      int32_t block_table_stride, const int32_t *cu_q_lens, const int32_t *context_lens, int32_t batch,
                      int32_t num_kv_heads, int32_t head_dim, int32_t page_shift, int64_t num_pages, int64_t capacity,
                      void *stream);

// Inside a V head's codes: unit e of column c of row t (two bytes).
template <int D>
__device__ __forceinline__ int int4_v_unit(int t, int c, int e) {
  return (t >> 2) * (2 * D) + c * (D / 8) + ((t >> 1) & 1) * (D / 16) + 4 * e + 2 * (t & 1);
}

// The value of the lane that `CTRL` (a DPP control: all lanes of a row of 16 read one) names.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  typedef int int2_t __attribute__((ext_vector_type(2)));
  int2_t v = __builtin_bit_cast(int2_t, x);
  v[0] = __builtin_amdgcn_update_dpp(0, v[0], CTRL, 0xf, 0xf, true);
  v[1] = __builtin_amdgcn_update_dpp(0, v[1], CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, v);
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppMirror4 = 0x1B, kDppMirror8 = 0x141, kDppMirror16 = 0x140,
              kDppRotate8 = 0x128;

// `op` over the L lanes (8 or 16, aligned) that hold a row; every lane gets the result. In the vector ALU: a shuffle
// through the LDS crossbar takes some hundred cycles a step.
template <int L, typename T, typename Op>
__device__ __forceinline__ T over_row(T x, Op op) {
  static_assert(L == 8 || L == 16, "lanes of a row");
  x = op(x, dpp<kDppXor1>(x));
  x = op(x, dpp<kDppXor2>(x));
  x = op(x, dpp<kDppMirror8>(x));
  if constexpr (L == 16) x = op(x, dpp<kDppMirror16>(x));
  return x;
}
// What the lane half a row away holds.
template <int L>
__device__ __forceinline__ float half_a_row_away(float x) {
  static_assert(L == 8 || L == 16, "lanes of a row");
  if constexpr (L == 16) return dpp<kDppRotate8>(x);
  return dpp<kDppMirror8>(dpp<kDppMirror4>(x));     // (l ^ 3) ^ 7
}

// The quotient x / y correctly rounded (short of a subnormal one), given inv = 1 / y: the division's error is an fp32 number,
// and folded back in leaves the quotient within 2^-46 of itself before its one rounding. In particular a quotient that
// lies exactly between two integers comes out so, and goes to the even one.
__device__ __forceinline__ float quotient(float x, float y, float inv) {
  const float n = x * inv;
  return __builtin_fmaf(__builtin_fmaf(-n, y, x), inv, n);
}

// A row in 4 bits, as the L = D / 8 lanes that hold it see it: lane l has elements 8l .. 8l + 7.
struct Int4Row {
  uint32_t code[8];
  uint32_t word;      // the same in every lane
};
template <int L>
__device__ __forceinline__ Int4Row int4_row(const float (&in)[8]) {
  float x[8], lo = 0.f, hi = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = in[i] == in[i] ? __builtin_fminf(__builtin_fmaxf(in[i], -kInt4Most), kInt4Most) : 0.f;
    lo = __builtin_fminf(lo, x[i]);
    hi = __builtin_fmaxf(hi, x[i]);
  }
  lo = over_row<L>(lo, [](float a, float b) { return __builtin_fminf(a, b); });
  hi = over_row<L>(hi, [](float a, float b) { return __builtin_fmaxf(a, b); });
  const float step = quotient(hi - lo, 15.0f, 1.0f / 15.0f);
  const float up = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, step) + 0x1ffffu) & ~0x1ffffu);
  const float s = step < 0x1p-14f ? __builtin_ceilf(step * 0x1p20f) * 0x1p-20f : up;
  const float inv = s > 0.f ? 1.0f / s : 0.f;
  const float z = __builtin_rintf(quotient(-lo, s, inv));
  Int4Row r;
  r.word = (uint32_t)__builtin_bit_cast(uint16_t, (half_t)s) | (uint32_t)z;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = __builtin_rintf(quotient(x[i], s, inv)) + z;
    r.code[i] = (uint32_t)__builtin_fminf(__builtin_fmaxf(c, 0.f), 15.f);
  }
  return r;
}
// Eight codes in a dword, even elements in the low nibbles.
__device__ __forceinline__ uint32_t int4_pack(const uint32_t (&c)[8]) {
  return c[0] | (c[2] << 4) | (c[4] << 8) | (c[6] << 12) | (c[1] << 16) | (c[3] << 20) | (c[5] << 24) | (c[7] << 28);
}

// Stores lane l's eight elements of a row into slot `slot` (of the block-wise layout above), K or V head `head`, counted as in
// the pool. The row's first lane also stores its word.
template <int D>
__device__ __forceinline__ void int4_store(uint8_t *pool, int64_t slot, int kv_heads, int head, int l,
                                           const Int4Row &r) {
  uint8_t *block = pool + (slot >> 4) * int4_block_bytes(kv_heads, D);
  const int t = (int)(slot & 15);
  uint8_t *codes = block + int4_codes_at(head, D);
  if (head < kv_heads) {
    *(uint32_t *)(codes + t * (D / 2) + 4 * l) = int4_pack(r.code);
  } else if constexpr (D == 128) {
    const uint32_t x = int4_pack(r.code);       // column l: even elements are unit 0, odd ones unit 1
    *(uint16_t *)(codes + int4_v_unit<D>(t, l, 0)) = (uint16_t)x;
    *(uint16_t *)(codes + int4_v_unit<D>(t, l, 1)) = (uint16_t)(x >> 16);
  } else {
    const uint32_t (&c)[8] = r.code;            // columns 2l, 2l + 1
    *(uint16_t *)(codes + int4_v_unit<D>(t, 2 * l, 0)) = (uint16_t)(c[0] | (c[1] << 4) | (c[2] << 8) | (c[3] << 12));
    *(uint16_t *)(codes + int4_v_unit<D>(t, 2 * l + 1, 0)) = (uint16_t)(c[4] | (c[5] << 4) | (c[6] << 8) | (c[7] << 12));
  }
  if (l == 0) *(uint16_t *)(block + int4_words_at(head, kv_heads, D) + 2 * t) = (uint16_t)r.word;
}

// ---- reading --------------------------------------------------------------------------------------------------------
// The scale and the zero point of two rows' words.
__device__ __forceinline__ half2_t int4_scales(uint32_t words) { return __builtin_bit_cast(half2_t, words & 0xfff0fff0u); }

// Eight codes of one row (see int4_pack) and its word, twice in a dword, as eight fp16 values, exact: nibbles under the exponent of
// 1024 (64 for the upper ones of a byte) are 1024 + c (64 + c), from which 1024 + z (64 + z) is subtracted.
__device__ __forceinline__ half8_t int4x8_to_half(uint32_t x, uint32_t words) {
  const half2_t s = int4_scales(words);
  const half2_t z0 = __builtin_bit_cast(half2_t, (words & 0x000f000fu) | 0x64006400u);
  const half2_t z1 = __builtin_bit_cast(half2_t, ((words & 0x000f000fu) << 4) | 0x54005400u);
  const uint32_t y = x >> 8;
  const half2_t a = (__builtin_bit_cast(half2_t, (x & 0x000f000fu) | 0x64006400u) - z0) * s;
  const half2_t b = (__builtin_bit_cast(half2_t, (x & 0x00f000f0u) | 0x54005400u) - z1) * s;
  const half2_t c = (__builtin_bit_cast(half2_t, (y & 0x000f000fu) | 0x64006400u) - z0) * s;
  const half2_t d = (__builtin_bit_cast(half2_t, (y & 0x00f000f0u) | 0x54005400u) - z1) * s;
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace litekv
