// One token per row of logits, drawn with a given uniform number under temperature, top-k, top-p and min-p.
//
// With y = x / T and p = exp(y - max y), the three filters each keep a prefix of the tokens ordered by p (ties: the lowest index
// first), so what is kept is the shortest of three prefixes: everything above one logit, and the first few of those that equal
// it. The token is the first, by index, at which the kept mass exceeds u times all of it.
//
// Nothing is sorted. A first launch cuts the rows into slices, a workgroup each, and leaves per slice a histogram over y (bins of
// 1/8 on a grid that all slices share, each with the number and the mass of its tokens) and a list of its likeliest tokens. A
// second one, a workgroup per row, adds the histograms up and walks the bins to the one in which a filter's prefix ends. Its
// tokens come from the lists or, where these do not reach so far, from a pass over the row; the end among them, and
// in the kept ones the token drawn, are found by the digits of their keys and, once they are few, by ranking them.
//
// Sums of mass are sums of whole numbers: the mass of a token is rounded to 2^-40 of its bin's top (y enters in fp64, and exp by a
// polynomial over the width of a bin), so no order of additions shows in a token, and a bin's top is a factor applied once. A
// cumulative mass is then within 2^-40 of itself wherever it is compared, which in a row of 150 000 tokens moves one draw in some
// millions to a neighbour of the token that exact arithmetic gives. (Beside that y has 2^-53 of itself from its one rounding, as the
// grid is that of all slices and not of the row's largest: more than 2^-40 from some 2^12 temperatures away from zero on.)
//
// Measured, us of the slices' and of the rows' kernel: 1 x 32000 fp16 with top-k and top-p 6 and 10, 32 x 151936 fp16 with all
// filters 10 and 12, 33 x 49999 fp32 9 and 12, 256 x 128000 bf16 with top-p 34 and 43 (65 MB: a copy takes 13). The first is bound
// by its instructions, 17 a token for the histogram, 12 of them fp64, and 11 for the rest (conversion, maximum, list), and by its atomics
// in LDS (vector instructions issue in 90 % of the cycles there, the LDS is busy in 45 %, three fifths of that with bank conflicts). The second by latency, some twelve to twenty steps of about 0.7 us (a memory trip, a scan, a barrier), and
// where a bin has to be listed from the row (half the rows of the last case) by the pass over it: 12 us, 5.4 TB/s over the device. A
// row whose end lies in a bin of more tokens than a list takes (151936 logits of standard deviation 1: 7500) takes 110 us, and one of
// nothing but equal logits up to 600, whichever their number: one compute unit goes over it several times.
#include <cmath>

#include "common.h"
#include "kv_int4.h"

// Products are rounded before they are subtracted from: z - floor(z) with a product z in one operation would leave z's own rounding
// error beside the place in the bin, and of a large z nothing else.
#pragma clang fp contract(off)

namespace litekv {

constexpr int kSampleBins = 322;              // of 1/8: what is further than 40 below a row's largest y is never drawn
constexpr int kSampleSlots = 512;             // a slice's bins lie at their place on the grid modulo this
constexpr int kSampleThreads = 256;           // of a slice's workgroup
constexpr int kSampleSlice = 8192;            // tokens of a slice at most: their number has 14 bits of a bin's word
// Tokens of a slice's list. (us of the whole call with 32 / 64 / 128: 32 x 151936 19.9 / 20.8 / 22.4; 33 x 49999, few slices, 26.5 / 18.6
// / 19.5; 64 x 32000 33.5 / 17.3 / 17.7)
constexpr int kSliceList = 64;
constexpr int kRowThreads = 512;              // of a row's workgroup
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int kMostFew = 2048;                // tokens that are taken from the slices' lists
// And of these, which are ranked against each other all at once, 256 where two filters end among them, 128 for one. (us of the whole call so /
// filter by filter: 32 x 151936 20.7 / 25.9, 1 x 32000 17.3 / 21.4, top-k and top-p up to 200; 16 x 151936 with top-k alone up to 200 23.1 / 21.0.)
constexpr int kOneGo = 256;
constexpr int kMostListed = 6144;             // tokens of a bin that are listed: 12 a thread on the average
constexpr int kOwnPlaces = 30;                // places that a thread has for them at first
constexpr int kSampleMaxVocab = 1 << 20;
constexpr int kMaxSlices = 512;
constexpr int kRanked = 64;                   // tokens that are ranked against each other; more go by their digits (with 128 no faster)
constexpr int kCountShift = 50;
constexpr uint64_t kUnitsMask = (1ull << kCountShift) - 1;
constexpr uint64_t kFloorUnits = 7ull << 37;  // 7/8, below exp(-1/8): a bin's word has the sum of what is above it
constexpr double kUnit = 0x1p-40 / (1.0 - 0x1p-20);   // of a bin's top (see MassPolynomial)
constexpr double kCut = -40.0;
constexpr double kReached = 1.0 - 0x1p-40;    // a border that rounding alone keeps from being reached is
constexpr float kMostFloat = 3.4028234663852886e38f;

struct SampleSlice {      // of the workspace, in front of the histograms and the lists
  double top;             // the bin of its largest y, counted from 0
  float most;             // its largest logit, -inf: nothing can be drawn
  int32_t at;             // greedy rows: the first token that has it
  int32_t listed;         // tokens of its list: all of the `listed_bins` bins from its top on
  int32_t listed_bins;
};

// The vectors of 16 bytes that a row's slices are counted in: of V elements, the first of them anywhere in its vector.
__host__ __device__ constexpr int64_t sample_vectors(int64_t vocab, int size) { return (vocab * size + 30) / 16; }
// Slices of 8192 tokens, or of half and a quarter of that where there are fewer than compute units: us of the whole call: 33 x 49999
// 25.4 in 231 slices of 8192, 18.6 in 429; 8 x 128000 42 in 128, 44 in 256; 1 x 32000 17.3 in slices of 2048, 20.9 in slices of 1024.
static int sample_slice_vectors(int32_t batch, int32_t vocab, int size) {
  int tokens = kSampleSlice;
  while (tokens > 2048 && (int64_t)batch * ((vocab + tokens - 1) / tokens) < 256) tokens /= 2;
  return tokens * size / 16;
}

enum { kLogitsF16 = 0, kLogitsBf16 = 1, kLogitsF32 = 2 };
constexpr int logit_size(int type) { return type == kLogitsF32 ? 4 : 2; }

// The largest finite logit of a type.
template <int TYPE>
constexpr float kMostLogit = TYPE == kLogitsF16 ? 65504.0f : TYPE == kLogitsBf16 ? 0x1.fep+127f : kMostFloat;
// Element i of a vector as a float, as it is.
template <int TYPE>
__device__ __forceinline__ float raw_logit(uint4_t raw, int i) {
  if constexpr (TYPE == kLogitsF32) {
    const uint32_t word = raw[i];        // (a bit cast of the element itself is one of the first)
    return __builtin_bit_cast(float, word);
  } else if constexpr (TYPE == kLogitsBf16) {
    const uint32_t word = i & 1 ? raw[i >> 1] & 0xffff0000u : raw[i >> 1] << 16;
    return __builtin_bit_cast(float, word);
  } else {
    return (float)__builtin_bit_cast(half_t, (uint16_t)(raw[i >> 1] >> (16 * (i & 1))));
  }
}
// NaN cannot be drawn and becomes -inf, infinity the largest finite float, which among 16-bit logits is above all others.
__device__ __forceinline__ float clean_logit(float x) { return __builtin_fminf(__builtin_fmaxf(x, -INFINITY), kMostFloat); }
// Whether a vector has an element that is not finite: two at a time by their bits without the signs.
template <int TYPE>
__device__ __forceinline__ bool has_special(uint4_t raw) {
  static_assert(TYPE != kLogitsF32, "16-bit logits");
  typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
  ushort2_t top = __builtin_bit_cast(ushort2_t, raw[0] & 0x7fff7fffu);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const uint32_t word = raw[i] & 0x7fff7fffu;
    top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2_t, word));
  }
  constexpr uint16_t kInfinity = TYPE == kLogitsF16 ? 0x7c00 : 0x7f80;
  return top[0] >= kInfinity || top[1] >= kInfinity;
}

// Where the vector `at` of a row is; only those with an element of the row are read.
struct LogitsRow {
  const char *base;        // the row's first vector
  int lead;                // elements in front of the row in it
  int64_t vectors;
  // Its vector v, the last for those behind it.
  __device__ __forceinline__ uint4_t vector(int64_t v) const {
    return *(const __attribute__((address_space(1))) uint4_t *)(uint64_t)(base + (v < vectors ? v : vectors - 1) * 16);
  }
};
template <int TYPE>
__device__ __forceinline__ LogitsRow logits_row(const void *logits, int64_t row_stride, int row, int32_t vocab) {
  constexpr int kSize = logit_size(TYPE);
  const uintptr_t at = (uintptr_t)logits + (uintptr_t)((int64_t)row * row_stride * kSize);
  LogitsRow r;
  r.base = (const char *)(at & ~(uintptr_t)15);
  r.lead = (int)(at & 15) / kSize;
  r.vectors = ((int64_t)(r.lead + vocab) * kSize + 15) / 16;
  return r;
}
// The elements of vector `at`, -inf in the places that are not the row's.
template <int TYPE>
__device__ __forceinline__ void logits_of(const LogitsRow &in, uint4_t raw, int64_t at, int32_t vocab,
                                          float (&x)[16 / logit_size(TYPE)]) {
  constexpr int kPer = 16 / logit_size(TYPE);
  const int64_t first = at * kPer - in.lead;
  const bool inside = first >= 0 && first + kPer <= vocab;
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = clean_logit(raw_logit<TYPE>(raw, i));
  if (!inside) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (first + i < 0 || first + i >= vocab) x[i] = -INFINITY;
    }
  }
}

// z = 8 y; its bin is floor(z). 8 / T: the hardware's approximation, twice improved (exact for powers of two).
__device__ __forceinline__ double z_factor(float t) {
  const double d = (double)t;
  double r = __builtin_amdgcn_rcp(d);
#pragma unroll
  for (int step = 0; step < 2; ++step) r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  return 8.0 * r;
}
__device__ __forceinline__ double z_of(float x, double z_per_x) { return (double)x * z_per_x; }
// (1 - 2^-20) exp((f - 1) / 8) - 7/8 in units of 2^-40, f in [0, 1) the place in a bin: below 2^37, and above 0. By the polynomial of
// degree 6 that agrees with it in seven Chebyshev points, within 0.02 of a unit but for c0, which with the 2^52 that is added to have the result in a double's low bits is a whole number, 0.01 from its own.
// (The coefficients in scalar registers, where they stay: as literals each is moved in front of its step, two instructions a
// coefficient and token.)
struct MassPolynomial {
  double c0 = 0x1.00001eb4308b7p+52, c1 = 0x1.c3d686115b6e3p+36, c2 = 0x1.c3d68623f9176p+32, c3 = 0x1.2d39a7c5007cap+28,
         c4 = 0x1.2d3c27a6b0e5fp+23, c5 = 0x1.e10f01fb822cdp+17, c6 = 0x1.56123fcc468c2p+12;
  __device__ __forceinline__ void keep() { asm("" : "+s"(c0), "+s"(c1), "+s"(c2), "+s"(c3), "+s"(c4), "+s"(c5)); }
  __device__ __forceinline__ uint64_t bits(double f) const { return __builtin_bit_cast(uint64_t, raised(f)); }
  __device__ __forceinline__ double raised(double f) const {       // ... and 2^52
    double e = __builtin_fma(c6, f, c5);
    e = __builtin_fma(e, f, c4);
    e = __builtin_fma(e, f, c3);
    e = __builtin_fma(e, f, c2);
    e = __builtin_fma(e, f, c1);
    return __builtin_fma(e, f, c0);
  }
};
constexpr uint64_t kMassOne = 0x4330000000000000ull;      // 2^52's bits
__device__ __forceinline__ uint64_t units_of(const MassPolynomial &mass, double z) {
  return mass.bits(z - __builtin_floor(z)) - kMassOne;
}
// In whole numbers; out of their range the nearest, as the conversion does it, which C++ leaves open.
__device__ __forceinline__ uint32_t whole_of(double x) {
  uint32_t n;
  asm("v_cvt_u32_f64 %0, %1" : "=v"(n) : "v"(x));
  return n;
}

__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);         // (the two zeros are one)
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of_order(uint32_t k) {
  return __builtin_bit_cast(float, k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

// Tokens are told apart, and ordered like p and the index, by a key: the order of the logit without the bits that its type leaves
// alike, then the index from the last down, in as many bits as the vocabulary takes (with more, the keys' digits would be few).
// Infinity, which has become the largest float, has the order of infinity there: what is left of its own is bf16's largest finite one.
template <int TYPE>
constexpr int kAlike = TYPE == kLogitsF16 ? 13 : TYPE == kLogitsBf16 ? 16 : 0;
template <int TYPE>
struct Keys {
  int bits;
  uint32_t most;
  __device__ __forceinline__ explicit Keys(int32_t vocab) : bits(32 - __builtin_clz((uint32_t)vocab | 1u)), most((1u << bits) - 1u) {}
  __device__ __forceinline__ uint64_t of(uint32_t order, int32_t at) const {
    return (uint64_t)(upwards(order) >> kAlike<TYPE>) << bits | (uint64_t)(most - (uint32_t)at);
  }
  __device__ __forceinline__ int32_t index(uint64_t key) const { return (int32_t)(most - ((uint32_t)key & most)); }
  __device__ __forceinline__ float logit(uint64_t key) const {
    const uint32_t o = (uint32_t)(key >> bits) << kAlike<TYPE>;
    const float x = logit_of_order(o & 0x80000000u ? o : o | ((1u << kAlike<TYPE>) - 1u));
    return TYPE == kLogitsF32 ? x : __builtin_fminf(x, kMostFloat);
  }
  // The lowest key of a token whose order is at least `order`.
  __device__ __forceinline__ uint64_t lowest(uint32_t order) const { return (uint64_t)(upwards(order) >> kAlike<TYPE>) << bits; }
  // The order itself, or the next that a logit of the type has, in the bits that are not alike. (Orders end with infinity's, 0xff800000.)
  static __device__ __forceinline__ uint32_t upwards(uint32_t order) {
    return order + ((uint32_t)((int32_t)order >> 31) & ((1u << kAlike<TYPE>) - 1u));      // (a negative token's alike bits are ones)
  }
};

__device__ __forceinline__ float row_temperature(const float *temperature, int row) {
  const float t = temperature != nullptr ? temperature[row] : 1.0f;
  return t > kMostFloat ? kMostFloat : t;      // (NaN stays)
}
__device__ __forceinline__ bool greedy_temperature(float t) { return !(t > 0.f); }
__device__ __forceinline__ int slot_of(double bin) { return (int)(bin - 512.0 * __builtin_floor(bin * 0x1p-9)); }

__device__ __forceinline__ float wave_max(float x) {
  x = __builtin_fmaxf(x, dpp<kDppXor1>(x));
  x = __builtin_fmaxf(x, dpp<kDppXor2>(x));
  x = __builtin_fmaxf(x, dpp<kDppMirror8>(x));
  x = __builtin_fmaxf(x, dpp<kDppMirror16>(x));
  return max_over_lane_groups(x);
}
// What the lane `CTRL` names holds, 0 where there is none or the row of 16 is not in ROWS.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T lane_at(T x) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, true));
  } else {
    typedef int int2_t __attribute__((ext_vector_type(2)));
    int2_t v = __builtin_bit_cast(int2_t, x);
    v[0] = __builtin_amdgcn_update_dpp(0, v[0], CTRL, ROWS, 0xf, true);
    v[1] = __builtin_amdgcn_update_dpp(0, v[1], CTRL, ROWS, 0xf, true);
    return __builtin_bit_cast(T, v);
  }
}
// Inclusive sums over a wavefront's lanes, in one order: rows of 16 by shifts, then their ends.
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
  x += lane_at<0x111, 0xf>(x);
  x += lane_at<0x112, 0xf>(x);
  x += lane_at<0x114, 0xf>(x);
  x += lane_at<0x118, 0xf>(x);
  x += lane_at<0x142, 0xa>(x);
  x += lane_at<0x143, 0xc>(x);
  return x;
}
// The lowest logit, by order, that `above` holds for, which grows with the logit: within a few floats of a guess. (Each wavefront
// finds it for itself.)
template <typename Above>
__device__ __forceinline__ uint32_t border(double guess, Above above) {
  const float near = (float)__builtin_fmin(__builtin_fmax(guess, -(double)kMostFloat), (double)kMostFloat);
  const int64_t lowest = order_of(-kMostFloat), highest = order_of(kMostFloat);
  const int64_t o = (int64_t)order_of(near) + (int)(threadIdx.x % kWave) - 32;
  const uint64_t all = __builtin_amdgcn_ballot_w64(o > highest || (o >= lowest && above(logit_of_order((uint32_t)o))));
  const int64_t first = (int64_t)order_of(near) + (all != 0 ? __builtin_ctzll(all) : 63) - 32;
  return (uint32_t)(first < lowest ? lowest : first);
}
// The lowest logit whose bin, counted from 0, is at least `limit`.
__device__ __forceinline__ uint32_t lowest_of_bin(double limit, float t, double z_per_x) {
  return border(limit * 0.125 * (double)t, [&](float x) { return __builtin_floor(z_of(x, z_per_x)) >= limit; });
}

// A slice: its largest logit, then its histogram, in two copies for two wavefronts each. A token adds its mass's bits as they are to
// its bin: the words' top 12 bits then hold 0x433 times the number of tokens, modulo 4096.
template <int TYPE>
__global__ __launch_bounds__(kSampleThreads) void sample_slices_kernel(
    const void *__restrict__ logits, int64_t row_stride, const float *__restrict__ temperature, int32_t vocab,
    int32_t slice_vectors, int32_t slices, SampleSlice *__restrict__ heads, uint64_t *__restrict__ bins,
    uint64_t *__restrict__ lists) {
  constexpr int kPer = 16 / logit_size(TYPE);
  constexpr int kMostVectors = kSampleSlice / kPer / kSampleThreads;
  constexpr int kWaves = kSampleThreads / kWave, kCopies = 2;
  static_assert(kSampleSlice / kCopies <= 4096, "a copy counts modulo 4096");
  static_assert(2 * kSampleThreads >= kSampleBins, "two bins a thread");
  __shared__ uint64_t hist[kCopies][2 * kSampleThreads];
  __shared__ float wave_most[kWaves];
  __shared__ int wave_at[kWaves];
  __shared__ int found_bins, found_n;
  const int tid = threadIdx.x, row = blockIdx.y, slice = blockIdx.x, wave = tid / kWave;
  const LogitsRow in = logits_row<TYPE>(logits, row_stride, row, vocab);
  const int64_t v0 = (int64_t)slice * slice_vectors;
  uint4_t raw[kMostVectors];
#pragma unroll
  for (int i = 0; i < kMostVectors; ++i) {
    const int v = i * kSampleThreads + tid;
    raw[i] = in.vector(v0 + v);                                // (what is not the slice's is masked; a condition would have each load waited for)
  }
  const float t = row_temperature(temperature, row);
  const double z_per_x = z_factor(t);
#pragma unroll
  for (int i = 0; i < kCopies * 2; ++i) hist[i / 2][i % 2 * kSampleThreads + tid] = 0;
  if (tid == 0) {
    found_bins = 0;
    found_n = 0;
  }
  const int first = (int)((v0 + tid) * kPer) - in.lead;        // this thread's first element, of the row's
  float x[kMostVectors][kPer];
  bool special = TYPE == kLogitsF32;
#pragma unroll
  for (int i = 0; i < kMostVectors; ++i) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) x[i][k] = raw_logit<TYPE>(raw[i], k);
    if constexpr (TYPE != kLogitsF32) special |= has_special<TYPE>(raw[i]);
  }
  if (__builtin_amdgcn_ballot_w64(special) != 0) {
#pragma unroll
    for (int i = 0; i < kMostVectors * kPer; ++i) x[i / kPer][i % kPer] = clean_logit(x[i / kPer][i % kPer]);
  }
  if (slice == 0 || v0 + kMostVectors * kSampleThreads >= in.vectors || slice_vectors < kMostVectors * kSampleThreads) {
    // -inf in the places that are not the row's, or not the slice's
#pragma unroll
    for (int i = 0; i < kMostVectors; ++i) {
      const bool there = i * kSampleThreads + tid < slice_vectors;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        if (!there || (uint32_t)(first + i * kSampleThreads * kPer + k) >= (uint32_t)vocab) x[i][k] = -INFINITY;
      }
    }
  }
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMostVectors * kPer; ++i) most = __builtin_fmaxf(most, x[i / kPer][i % kPer]);
  most = wave_max(most);
  if (tid % kWave == 0) wave_most[wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) most = __builtin_fmaxf(most, wave_most[w]);
  SampleSlice *head = heads + (int64_t)row * slices + slice;
  if (most == -INFINITY) {
    if (tid == 0) *head = SampleSlice{0.0, -INFINITY, 0, 0, kSampleBins};
    return;
  }
  if (greedy_temperature(t)) {
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kMostVectors; ++i) {
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int e = first + i * kSampleThreads * kPer + k;
        if (x[i][k] == most) at = e < at ? e : at;
      }
    }
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int other = __shfl_xor(at, off, kWave);
      at = other < at ? other : at;
    }
    if (tid % kWave == 0) wave_at[wave] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) at = wave_at[w] < at ? wave_at[w] : at;
    if (tid == 0) *head = SampleSlice{0.0, most, at, 0, 0};
    return;
  }
  const double top = __builtin_floor(z_of(most, z_per_x));
  uint64_t *mine = hist[wave / (kWaves / kCopies)];
  MassPolynomial mass;
  mass.keep();
  const uint32_t aside = kSampleBins + tid % kWave;        // (what is too far below goes to a place of the lane's, without a branch)
  static_assert(kSampleBins + kWave <= 2 * kSampleThreads, "which is behind the bins");
#pragma unroll
  for (int i = 0; i < kMostVectors; ++i) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const double z = z_of(x[i][k], z_per_x), b = __builtin_floor(z);
      uint32_t d = whole_of(top - b);                            // (-inf: far below)
      d = d < aside ? d : aside;
      atomicAdd((unsigned long long *)&mine[d], (unsigned long long)mass.bits(z - b));
    }
    __builtin_amdgcn_sched_barrier(0);                           // (more tokens at a time take more registers than there are)
  }
  __syncthreads();
  // Two bins a thread, to their places; and how many from the top on have no more tokens than a list takes.
  const int64_t place = (int64_t)row * slices + slice;
  const int top_slot = slot_of(top);
  int count = 0, count_first = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = 2 * tid + i;
    uint64_t n_all = 0, units = 0;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      const uint64_t w = hist[c][b];
      uint64_t n = ((w >> 52) * 1787u) & 4095u;            // 1787 * 0x433 = 1 modulo 4096
      const uint64_t u = w & ((1ull << 52) - 1);
      n = n == 0 && u != 0 ? 4096 : n;
      n_all += n;
      units += u;
    }
    if (b < kSampleBins) {
      bins[place * kSampleSlots + ((top_slot - b) & (kSampleSlots - 1))] = units | n_all << kCountShift;
      count += (int)n_all;
    }
    if (i == 0) count_first = count;
  }
  int upto = wave_scan(count);
  if (tid % kWave == kWave - 1) wave_at[wave] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w) upto += w < wave ? wave_at[w] : 0;
  const int first_upto = upto - count + count_first;
  // (both grow with the bin: as many as hold are the bins from the top on)
  const int fit = __builtin_popcountll(__builtin_amdgcn_ballot_w64(first_upto <= kSliceList)) +
                  __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= kSliceList));
  if (tid % kWave == 0 && fit > 0) atomicAdd(&found_bins, fit);
  __syncthreads();
  const int listed_bins = found_bins < kSampleBins ? found_bins : kSampleBins;
  if (listed_bins > 0) {
    const float least = logit_of_order(lowest_of_bin(top - (listed_bins - 1), t, z_per_x));
    uint64_t those[kMostVectors * kPer];
    int n = 0;
#pragma unroll
    for (int i = 0; i < kMostVectors * kPer; ++i) {
      those[i] = __builtin_amdgcn_ballot_w64(x[i / kPer][i % kPer] >= least);
      n += __builtin_popcountll(those[i]);
    }
    int at = 0;
    if (tid % kWave == 0 && n > 0) at = atomicAdd(&found_n, n);
    at = __builtin_amdgcn_readfirstlane(at);
    uint64_t *to = lists + place * kSliceList;
#pragma unroll
    for (int i0 = 0; i0 < kMostVectors * kPer; i0 += kPer) {
      uint64_t any = 0;
#pragma unroll
      for (int i = i0; i < i0 + kPer; ++i) any |= those[i];
      if (any == 0) continue;
#pragma unroll
      for (int i = i0; i < i0 + kPer; ++i) {
        if (those[i] == 0) continue;
        const float e = x[i / kPer][i % kPer];
        const int slot = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(those[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)those[i], 0));
        if (e >= least && slot < kSliceList) {
          to[slot] = (uint64_t)__builtin_bit_cast(uint32_t, e) << 32 | (uint32_t)(first + i / kPer * kSampleThreads * kPer + i % kPer);
        }
        at += __builtin_popcountll(those[i]);
      }
    }
    __syncthreads();
  }
  if (tid == 0) *head = SampleSlice{top, most, 0, found_n < kSliceList ? found_n : kSliceList, listed_bins};
}

// ---- a row ---------------------------------------------------------------------------------------------------------------------
struct RowRoom {           // of a scan; two are used in turn, so that one barrier is enough
  double mass[kRowWaves];
  unsigned long long units[kRowWaves];
  int32_t count[kRowWaves];
};
// Inclusive sums over the workgroup's threads, in one order, and all of them.
template <typename T>
__device__ __forceinline__ T row_scan(T x, T *room, T *all) {
  const int wave = threadIdx.x / kWave;
  x = wave_scan(x);
  if (threadIdx.x % kWave == kWave - 1) room[wave] = x;
  __syncthreads();
  T before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    const T part = room[w];
    before += w < wave ? part : T(0);
    sum += part;
  }
  *all = sum;
  return before + x;
}
template <typename T, typename U>
__device__ __forceinline__ void row_scan2(T &x, T *room_x, U &y, U *room_y) {
  const int wave = threadIdx.x / kWave;
  x = wave_scan(x);
  y = wave_scan(y);
  if (threadIdx.x % kWave == kWave - 1) {
    room_x[wave] = x;
    room_y[wave] = y;
  }
  __syncthreads();
  T bx = 0;
  U by = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves - 1; ++w) {
    bx += w < wave ? room_x[w] : T(0);
    by += w < wave ? room_y[w] : U(0);
  }
  x += bx;
  y += by;
}

// Whether a word of a vector may have a logit of [least, most]: 16-bit ones two at a time, by their bits in the order of whole numbers.
template <int TYPE>
struct RangeTest {
  typedef int16_t short2_t __attribute__((ext_vector_type(2)));
  typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
  float least, most;
  uint32_t low, beyond;      // twice: the lowest, and how far behind it the range has ended
  __device__ __forceinline__ RangeTest(float least_x, float most_x) : least(least_x), most(most_x), low(0), beyond(0) {
    if constexpr (TYPE != kLogitsF32) {
      // (the zeros and, in fp16, those next to an end are looked at again)
      const int from = least_x == 0.f ? -1 : in_order(bits_of(least_x));
      const int to = most_x == 0.f ? 0 : in_order(bits_of(most_x));
      low = (uint16_t)from * 0x10001u;
      beyond = (uint16_t)(to - from + 1) * 0x10001u;
    } else if (most_x == kMostFloat) {
      most = INFINITY;
    }
  }
  static __device__ __forceinline__ int in_order(uint16_t bits) { return (int16_t)(bits ^ ((int16_t)bits >> 15 & 0x7fff)); }
  static __device__ __forceinline__ uint16_t bits_of(float x) {
    if (x > kMostLogit<TYPE>) return TYPE == kLogitsF16 ? 0x7c00 : 0x7f80;          // infinity's
    if constexpr (TYPE == kLogitsF16) return __builtin_bit_cast(uint16_t, (half_t)x);
    return (uint16_t)(__builtin_bit_cast(uint32_t, x) >> 16);
  }
  // How far the two logits of a word are from the lowest.
  __device__ __forceinline__ uint32_t from_low(uint32_t word) const {
    const short2_t x = __builtin_bit_cast(short2_t, word);
    const short2_t o = x ^ ((x >> 15) & (short2_t)0x7fff);
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(ushort2_t, o) - __builtin_bit_cast(ushort2_t, low));
  }
  static __device__ __forceinline__ bool any_nearer(uint32_t from_low, uint32_t end) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(ushort2_t, from_low), __builtin_bit_cast(ushort2_t, end))) != end;
  }
  __device__ __forceinline__ bool any(uint32_t word) const {
    if constexpr (TYPE == kLogitsF32) {
      const float x = __builtin_bit_cast(float, word);
      return x >= least && x <= most;
    } else {
      return any_nearer(from_low(word), beyond);
    }
  }
};

// Bound by latency: one memory trip or one pass over the row after another, with barriers between them. So loads are made whatever
// their place (clamped, and masked where they are used), loops over a list have no branches, and what few threads can find, each
// wavefront finds for itself.
template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_rows_kernel(
    const void *__restrict__ logits, int64_t row_stride, const float *__restrict__ uniforms,
    const float *__restrict__ temperature, const int32_t *__restrict__ top_k, const float *__restrict__ top_p,
    const float *__restrict__ min_p, int64_t *__restrict__ tokens, float *__restrict__ logprobs, int32_t vocab,
    int32_t slice_vectors, int32_t slices, const SampleSlice *__restrict__ heads, const uint64_t *__restrict__ bins,
    const uint64_t *__restrict__ lists) {
  constexpr int kPer = 16 / logit_size(TYPE);
  static_assert(kRowThreads == kSampleSlots, "a thread has a slot");
  constexpr int kRun = (kSampleMaxVocab + kRowThreads - 1) / kRowThreads;    // indexes of a run, at most
  __shared__ double bin_top[kSampleSlots];            // exp(the bin's top - the row's largest y), in units
  __shared__ double mass_to[kSampleSlots];            // inclusive
  __shared__ int32_t count_to[kSampleSlots];
  __shared__ int32_t shift[kMaxSlices];               // of a slice's bins against the row's, kSampleBins: it has none
  __shared__ int32_t slice_listed[kMaxSlices];
  __shared__ double slice_mass[kMaxSlices];
  __shared__ unsigned long long slice_units[kMaxSlices];
  __shared__ uint64_t list[kMostListed];              // keys, in any order
  __shared__ unsigned long long radix_units[kRowThreads];
  __shared__ int32_t radix_count[kRowThreads];
  __shared__ union {
    struct {
      unsigned long long key[kRun], units[kRun];
    } rank;
    uint32_t own[kOwnPlaces + 2][kRowThreads];        // (two places more are written to and never read)
  } room;
  auto &rank_key = room.rank.key, &rank_units = room.rank.units;
  __shared__ RowRoom rooms[2];
  __shared__ float room_f[kRowWaves];
  __shared__ int32_t found_k, found_p, found_last, found_at, found_slice, found_n, complete;
  __shared__ unsigned long long found_key, found_units;
  const int tid = threadIdx.x, row = blockIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const LogitsRow in = logits_row<TYPE>(logits, row_stride, row, vocab);
  const Keys<TYPE> keys(vocab);
  const SampleSlice *head = heads + (int64_t)row * slices;
  const uint64_t *row_bins = bins + (int64_t)row * slices * kSampleSlots;
  const uint64_t *row_lists = lists + (int64_t)row * slices * kSliceList;
  int turn = 0;                                        // which room the next scan has

  // The words of the first slices are asked for before it is known what they mean.
  constexpr int kAhead = 20;
  uint64_t words[kAhead];
  auto load_words = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      words[i] = row_bins[(int64_t)(s0 + i < slices ? s0 + i : slices - 1) * kSampleSlots + tid];
    }
  };
  const SampleSlice own_head = head[tid < slices ? tid : slices - 1];
  const float t = row_temperature(temperature, row);
  const int32_t k = top_k != nullptr ? top_k[row] : 0;
  const float p = top_p != nullptr ? top_p[row] : 1.0f;
  const float m = min_p != nullptr ? min_p[row] : 0.0f;
  double u = (double)uniforms[row];
  load_words(0);
  u = u > 0.0 ? (u < 1.0 - 0x1p-24 ? u : 1.0 - 0x1p-24) : 0.0;

  // the row's largest logit
  static_assert(kMaxSlices <= kRowThreads, "a thread has a slice");
  float most = wave_max(own_head.most);
  if (lane == 0) room_f[wave] = most;
  if (tid == 0) {
    found_k = complete = kSampleBins;
    found_last = found_n = 0;
    found_at = 0x7fffffff;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) most = __builtin_fmaxf(most, room_f[w]);
  if (most == -INFINITY) {                            // nothing can be drawn
    if (tid == 0) {
      tokens[row] = -1;
      if (logprobs != nullptr) logprobs[row] = -INFINITY;
    }
    return;
  }
  if (greedy_temperature(t)) {
    if (tid < slices && own_head.most == most) atomicMin(&found_at, own_head.at);
    __syncthreads();
    if (tid == 0) {
      tokens[row] = found_at;
      if (logprobs != nullptr) logprobs[row] = 0.f;
    }
    return;
  }
  const double z_per_x = z_factor(t);
  const double z_most = z_of(most, z_per_x), top = __builtin_floor(z_most);
  const int top_slot = slot_of(top);
  if (tid < slices) {
    const uint32_t d = own_head.most == -INFINITY ? kSampleBins : whole_of(top - own_head.top);
    shift[tid] = d < (uint32_t)kSampleBins ? (int)d : kSampleBins;
    slice_listed[tid] = own_head.listed;
    if (d < (uint32_t)kSampleBins && own_head.listed_bins < kSampleBins) atomicMin(&complete, (int)d + own_head.listed_bins);
  }
  bin_top[tid] = kUnit * exp(((top - z_most) + (double)(1 - tid)) * 0.125);     // (of z of any size: the first difference is exact)
  __syncthreads();
  // Bin b of the row in slice s, from what lies in its place, which need not be the slice's.
  auto word = [&](uint64_t w, int s, int b) __attribute__((always_inline)) -> uint64_t {
    return b < kSampleBins && (uint32_t)(b - shift[s]) < (uint32_t)kSampleBins ? w : 0;
  };
  // its bins: a thread adds up a slot of the slices' and hands it over
  {
    const int b = (top_slot - tid) & (kSampleSlots - 1);
    uint32_t count = 0;
    uint64_t units = 0;
    for (int s0 = 0; s0 < slices; s0 += kAhead) {
      if (s0 != 0) load_words(s0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int s = s0 + i;
        const uint64_t x = s < slices ? word(words[i], s, b) : 0;
        count += (uint32_t)(x >> kCountShift);
        units += x & kUnitsMask;
      }
    }
    radix_units[b] = units + kFloorUnits * (uint64_t)count;
    radix_count[b] = (int32_t)count;
  }
  __syncthreads();
  const int32_t count_here = radix_count[tid];
  double mass = (double)radix_units[tid] * bin_top[tid];
  int32_t count = count_here;
  row_scan2(count, rooms[0].count, mass, rooms[0].mass);
  turn = 1;
  count_to[tid] = count;
  mass_to[tid] = mass;
  {
    const uint64_t any = __builtin_amdgcn_ballot_w64(count_here > 0);
    if (lane == 0 && any != 0) atomicMax(&found_last, wave * kWave + 63 - __builtin_clzll(any));       // the last bin with a token
  }
  if (k > 0 && count - count_here < k && count >= k) found_k = tid;      // (one thread's)
  __syncthreads();
  const int last_bin = found_last;
  const int32_t live = count_to[last_bin];
  const double mass_live = mass_to[last_bin];
  bool by_k = k > 0 && k < live, by_p = p < 1.0f;
  const bool by_m = m > 0.0f;
  double log_m = 0.0;

  // The first bin with a token by whose end the mass is `target`; the last with a token if none is.
  auto bin_reaching = [&](double target) __attribute__((always_inline)) -> int {
    __syncthreads();
    if (tid == 0) found_p = last_bin;
    __syncthreads();
    const uint64_t past = __builtin_amdgcn_ballot_w64(count_here > 0 && mass >= target);
    if (lane == 0 && past != 0) atomicMin(&found_p, wave * kWave + __builtin_ctzll(past));
    __syncthreads();
    return found_p;
  };
  MassPolynomial polynomial;
  polynomial.keep();
  auto units_of_key = [&](uint64_t key) __attribute__((always_inline)) -> uint64_t {
    return units_of(polynomial, z_of(keys.logit(key), z_per_x)) + kFloorUnits;
  };

  // Of y's that are not cut off. In the few tokens' case as whole numbers of 2^-51, so that 2^11 of them are within 2^-40 of what they
  // sum up to and their sums within 63 bits; a token that is kept has one at least, as the smallest numbers take the first that is.
  const double x_cut = kCut * (double)t;
  auto mass_of = [&](uint64_t key) __attribute__((always_inline)) -> double {
    const float x = keys.logit(key);
    const double z = z_of(x, z_per_x), b = __builtin_floor(z);
    const uint32_t d = whole_of(top - b);
    const double units = polynomial.raised(z - b) - (0x1p52 - (double)kFloorUnits);
    const bool kept_x = (double)x - (double)most >= x_cut && d < (uint32_t)kSampleBins;
    return kept_x ? units * bin_top[d < (uint32_t)kSampleBins ? d : 0u] : 0.0;
  };
  auto units_kept = [&](uint64_t key) __attribute__((always_inline)) -> uint64_t {
    const double mass_here = mass_of(key);
    const double units = __builtin_fmax(mass_here * 0x1p51, mass_here > 0.0 ? 1.0 : 0.0);
    return __builtin_bit_cast(uint64_t, units + 0x1p52) - kMassOne;
  };
  const uint64_t most_key = keys.of(order_of(most), 0);
  auto answer = [&](uint64_t token, double all) __attribute__((always_inline)) {
    tokens[row] = keys.index(token);
    if (logprobs != nullptr) {
      logprobs[row] = (float)(((double)keys.logit(token) - (double)most) * z_per_x * 0.125 - log(all));
    }
  };
  // min_p's lowest key.
  auto least_kept = [&]() __attribute__((always_inline)) -> uint32_t {
    return border((double)most + log_m, [&](float x) { return x >= most || (double)x - (double)most >= log_m; });
  };

  // Where the prefixes end; one that ends behind min_p's end (bin_m, or a bin more) says nothing, but top_k says what top_p is a
  // share of.
  const int bin_k = by_k ? found_k : last_bin;
  int bin_p = last_bin, bin_m = last_bin;
  if (by_m) {
    log_m = log((double)(m < 1.0f ? m : 1.0f)) * (double)t;          // kept: x - most >= log_m
    const double b = top - __builtin_floor(z_most + log_m * z_per_x) + 1.0;
    if (b < (double)bin_m) bin_m = (int)b;
  }
  if (by_p && !by_k) {
    bin_p = bin_reaching((double)p * mass_live * kReached);
    by_p = bin_p <= bin_m;
  } else if (!by_p) {
    by_k = by_k && bin_k <= bin_m;
  }
  // Where the slices' lists have all tokens that come into question, those are the row's list, and the draw's; else it has a
  // bin's tokens at a time, if they fit.
  const int most_bin = by_k ? bin_k : by_p ? bin_p : bin_m;
  const bool few = most_bin < complete && count_to[most_bin] <= kMostFew;
  auto enlist = [&](uint64_t key) __attribute__((always_inline)) {
    const int to = atomicAdd(&found_n, 1);
    if (to < kMostListed) list[to] = key;
  };
  int listed = 0;
  if (few) {
    const uint64_t least = keys.lowest(lowest_of_bin(top - most_bin, t, z_per_x));
#pragma unroll 4
    for (int i = tid; i < slices * kSliceList; i += kRowThreads) {
      const uint64_t entry = row_lists[i];               // a logit's bits and its index
      const uint32_t bits = (uint32_t)(entry >> 32);
      const uint64_t key = keys.of(order_of(__builtin_bit_cast(float, bits)), (int32_t)(uint32_t)entry);
      if (i % kSliceList < slice_listed[i / kSliceList] && key >= least) enlist(key);
    }
    __syncthreads();
    listed = found_n < kMostListed ? found_n : kMostListed;
  }
  if (few && listed <= (by_k && by_p ? kOneGo : kOneGo / 2)) {
    // All at once: ranked against each other, the sums of their masses in that order, the first that is not kept, and of the kept ones
    // the sums in the order of the index. Against each other by several threads a token, each a share of the others.
    const int n = listed;
    const int threads = n <= kWave ? kWave : n <= 2 * kWave ? 2 * kWave : kOneGo;     // of a share
    const int one = tid & (threads - 1), each = (n + kRowThreads / threads - 1) / (kRowThreads / threads);
    const int from = __builtin_amdgcn_readfirstlane(tid / threads) * each, to = from + each < n ? from + each : n;
    radix_count[tid] = 0;
    slice_units[tid] = 0;
    __syncthreads();
    uint64_t mine = one < n ? list[one] : 0;
    int before = 0;
#pragma unroll 8
    for (int i = from; i < to; ++i) before += list[i] > mine;
    atomicAdd(&radix_count[one], before);
    const uint64_t units = units_kept(mine);
    __syncthreads();
    if (tid < n) {
      rank_key[radix_count[tid]] = mine;
      rank_units[radix_count[tid]] = units;
    }
    __syncthreads();
    mine = tid < n ? rank_key[tid] : 0;
    const unsigned long long here = tid < n ? rank_units[tid] : 0;
    unsigned long long all_units;
    const unsigned long long upto = row_scan(here, rooms[turn].units, &all_units);
    radix_units[tid] = upto;
    const uint64_t least = by_m ? keys.lowest(least_kept()) : 0;
    __syncthreads();
    const double p_target = (double)p * (by_k ? (double)radix_units[k - 1] : mass_live * 0x1p51) * kReached;
    const bool out = tid > 0 && (tid >= n || (by_k && tid >= k) || mine < least || (by_p && (double)(upto - here) >= p_target));
    const uint64_t those = __builtin_amdgcn_ballot_w64(out);
    if (lane == 0 && those != 0) atomicMin(&found_at, wave * kWave + __builtin_ctzll(those));
    __syncthreads();
    const int kept_n = found_at < n ? found_at : n;
    const unsigned long long sum = radix_units[kept_n - 1];
    const double target = u * (double)sum * (2.0 - kReached);
    const uint64_t at = rank_key[one < n ? one : 0] & keys.most;
    const int kept_each = (kept_n + kRowThreads / threads - 1) / (kRowThreads / threads);
    const int kept_from = __builtin_amdgcn_readfirstlane(tid / threads) * kept_each;
    const int kept_to = kept_from + kept_each < kept_n ? kept_from + kept_each : kept_n;
    unsigned long long part = 0;
#pragma unroll 8
    for (int i = kept_from; i < kept_to; ++i) part += (rank_key[i] & keys.most) > at ? rank_units[i] : 0;
    atomicAdd(&slice_units[one], part);
    __syncthreads();
    if (tid >= kept_n) return;
    const unsigned long long units_before = slice_units[tid];
    if ((double)(units_before + here) > target && !((double)units_before > target)) {
      answer(mine, (double)sum / (double)units_kept(most_key));
    }
    return;
  }
  int last = last_bin;                                  // the bin that the kept prefix ends in
  bool whole = true;                                    // all of it; or its tokens from the key `cut` on
  uint64_t cut = 0;
  double kept = mass_live;
  uint64_t list_from = few ? 0 : 1, list_to = few ? ~0ull : 0;        // the keys whose tokens are listed; others are read from the row
  // All tokens with the logits of [from, to], which are whole ones. First each thread's, its elements by their numbers (16-bit logits
  // with how far they are from the lowest): every element is written to the next place, which is moved on behind one of the range,
  // without a branch. Then as keys, side by side.
  static_assert(kSampleMaxVocab / kRowThreads + 8 * kPer <= 1 << 16, "an element's number has 16 bits");
  auto list_logits = [&](uint64_t from, uint64_t to) __attribute__((always_inline)) {
    const RangeTest<TYPE> test(keys.logit(from), keys.logit(to));
    uint32_t *const places = &room.own[0][tid];
    uint32_t *const last_place = places + kOwnPlaces * kRowThreads;
    uint32_t *place = places;
    constexpr int kVectors = 4;
    uint4_t raw[kVectors], next[kVectors];                   // (the next ones on their way while these are looked at)
    auto load = [&](int64_t v0, uint4_t (&into)[kVectors]) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const int64_t v = v0 + j * kRowThreads;
        into[j] = in.vector(v);
      }
    };
    load(tid, next);
    uint32_t number = 0;
#pragma unroll 1
    for (int64_t v0 = tid; v0 < in.vectors; v0 += kVectors * kRowThreads) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j) raw[j] = next[j];
      load(v0 + kVectors * kRowThreads, next);
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const bool there = v0 + j * kRowThreads < in.vectors;
        if constexpr (TYPE == kLogitsF32) {
          bool hit[4], any = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            hit[i] = there && test.any(raw[j][i]);
            any |= hit[i];
          }
          if (__builtin_amdgcn_ballot_w64(any) == 0) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            *place = number + (uint32_t)(kPer * j + i);
            place += hit[i] ? kRowThreads : 0;
            if (i & 1) place = place < last_place ? place : last_place;
          }
        } else {
          const uint32_t end = there ? test.beyond : 0;
          uint32_t far[4];
          bool any = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            far[i] = test.from_low(raw[j][i]);
            any |= RangeTest<TYPE>::any_nearer(far[i], end);
          }
          if (__builtin_amdgcn_ballot_w64(any) == 0) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t at = number + (uint32_t)(kPer * j + 2 * i);
            *place = far[i] << 16 | at;
            place += (uint16_t)far[i] < (uint16_t)end ? kRowThreads : 0;
            *place = (far[i] & 0xffff0000u) | (at + 1);
            place += far[i] < (end & 0xffff0000u) ? kRowThreads : 0;
            place = place < last_place ? place : last_place;
          }
        }
      }
      number += kPer * kVectors;
    }
    const int own = (int)(place - places) / kRowThreads;
    int all;
    const int before = row_scan(own < kOwnPlaces ? own : kMostListed + 1, rooms[turn].count, &all) - own;
    turn ^= 1;
    listed = all;
    if (all > kMostListed) return;                           // (too many of them are some thread's)
#pragma unroll 4
    for (int i = 0; i < own; ++i) {
      const uint32_t word = places[i * kRowThreads], n = word & 0xffffu;
      const int32_t at = (int32_t)((n / kPer * kRowThreads + tid) * kPer + n % kPer) - in.lead;
      uint32_t bits;
      if constexpr (TYPE == kLogitsF32) {
        bits = *(const __attribute__((address_space(1))) uint32_t *)(uint64_t)(in.base + (int64_t)(at + in.lead) * 4);
      } else {
        const int32_t o = (int16_t)(uint16_t)((word >> 16) + test.low);
        bits = (uint16_t)(o ^ ((o >> 31) & 0x7fff));
      }
      const float e = clean_logit(raw_logit<TYPE>(uint4_t{bits, bits, bits, bits}, 0));
      list[before + i] = (uint32_t)at < (uint32_t)vocab ? keys.of(order_of(e), at) : 0;      // (no token's key)
    }
    __syncthreads();
  };
  // Every token of the row whose key is in [from, to].
  auto over_the_row = [&](uint64_t from, uint64_t to, auto &&what) __attribute__((always_inline)) {
    const RangeTest<TYPE> test(keys.logit(from), keys.logit(to));
    constexpr int kVectors = 4, kPerWord = kPer / 4;
    uint4_t raw[kVectors], next[kVectors];                   // (the next ones on their way while these are looked at)
    auto load = [&](int64_t v0, uint4_t (&into)[kVectors]) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const int64_t v = v0 + j * kRowThreads;
        into[j] = in.vector(v);
      }
    };
    load(tid, next);
#pragma unroll 1
    for (int64_t v0 = tid; v0 < in.vectors; v0 += kVectors * kRowThreads) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j) raw[j] = next[j];
      load(v0 + kVectors * kRowThreads, next);
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const int64_t v = v0 + j * kRowThreads;
        uint32_t those = 0;                                  // words with an element in the range
#pragma unroll
        for (int i = 0; i < 4; ++i) those |= (test.any(raw[j][i]) ? 1u : 0u) << i;
        while (those != 0) {
          const int i = __builtin_ctz(those);
          those &= those - 1;
          uint32_t one = raw[j][0];
#pragma unroll
          for (int n = 1; n < 4; ++n) one = i == n ? raw[j][n] : one;
#pragma unroll
          for (int h = 0; h < kPerWord; ++h) {
            const float e = clean_logit(raw_logit<TYPE>(uint4_t{one, one, one, one}, h));
            const int32_t at = (int32_t)(v * kPer - in.lead) + i * kPerWord + h;
            const uint64_t key = keys.of(order_of(e), at);
            if (key >= from && key <= to && (uint32_t)at < (uint32_t)vocab) what(key, true);
          }
        }
      }
    }
  };
  auto each_listed = [&](uint64_t from, uint64_t to, auto &&what) __attribute__((always_inline)) {
#pragma unroll 4
    for (int i = tid; i < listed; i += kRowThreads) {
      const uint64_t key = list[i];
      what(key, key >= from && key <= to);
    }
  };
  auto each_token = [&](uint64_t from, uint64_t to, auto &&what) __attribute__((always_inline)) {
    if (from >= list_from && to <= list_to) {
      each_listed(from, to, what);
    } else {
      over_the_row(from, to, what);
    }
  };

  // Filter 0 is top_k, 1 top_p, 2 min_p and what the draw needs.
  uint64_t low = 0, high = 0;                           // the keys of the bin's tokens
#pragma unroll 1
  for (int filter = 0; filter < 3; ++filter) {
    int bin;
    int32_t end_count = 0;         // the end is the first token with which the bin's are so many, if above 0,
    double end_units = 0.0;        // or have so many units
    if (filter == 0) {
      if (!by_k) continue;
      bin = last = bin_k;
      kept = mass_to[last];
      if (count_to[last] == k) continue;
      end_count = k - (last > 0 ? count_to[last - 1] : 0);
    } else if (filter == 1) {
      if (!by_p) continue;
      const double target = (double)p * kept * kReached;
      if (by_k) {
        bin_p = bin_reaching(target);
        if (bin_p > last) bin_p = last;
      }
      bin = bin_p;
      end_units = __builtin_fmax((target - (bin > 0 ? mass_to[bin - 1] : 0.0)) / bin_top[bin], 1.0);
    } else {
      if (by_m) {
        const uint32_t order = least_kept();
        const double d = top - __builtin_floor(z_of(logit_of_order(order), z_per_x));
        const int b = d < (double)kSampleBins ? (int)d : kSampleBins;
        const uint64_t least = keys.lowest(order);
        if (b < kSampleBins && (b < last || (b == last && (whole || least > cut)))) {
          last = b;
          whole = false;
          cut = least;
        }
      }
      if (few || whole) break;
      bin = last;
    }
    const uint32_t low_order = lowest_of_bin(top - bin, t, z_per_x);
    low = keys.lowest(low_order);
    high = bin > 0 ? keys.lowest(lowest_of_bin(top - bin + 1.0, t, z_per_x)) - 1 : most_key;
    if (filter == 2) break;

    // Where the prefix ends in the bin: while its tokens are many, by the next ten bits of their keys; then by ranking them.
    int32_t n_above = 0, n_left = count_to[bin] - (bin > 0 ? count_to[bin - 1] : 0);
    uint64_t u_above = 0, from = low, to = high;
    while (true) {
      const bool whole_logits = from == low && to == high;
      if (n_left <= (whole_logits ? kMostListed : kMostFew) && !(from >= list_from && to <= list_to)) {
        __syncthreads();
        if (whole_logits) {
          list_logits(from, to);
        } else {
          if (tid == 0) found_n = 0;
          __syncthreads();
          over_the_row(from, to, [&](uint64_t key, bool) __attribute__((always_inline)) { enlist(key); });
          __syncthreads();
          listed = found_n;
        }
        list_from = listed <= kMostListed ? from : 1;
        list_to = listed <= kMostListed ? to : 0;
      }
      __syncthreads();
      if (tid == 0) {
        found_n = 0;
        found_at = -1;
        found_key = from;
        found_units = 0;
      }
      if (n_left > kRanked) {
        int down = 0;
        while (((to - from) >> down) >= (uint64_t)kRowThreads) ++down;
        radix_units[tid] = 0;
        radix_count[tid] = 0;
        __syncthreads();
        // (one outside adds nothing somewhere: without branches several are on their way at once)
        each_token(from, to, [&](uint64_t key, bool inside) __attribute__((always_inline)) {
          const uint32_t r = inside ? (uint32_t)((to - key) >> down) : (uint32_t)tid;          // from the largest
          const uint64_t units = units_of_key(key);
          atomicAdd(&radix_count[r], inside ? 1 : 0);
          atomicAdd(&radix_units[r], (unsigned long long)(inside ? units : 0));
        });
        __syncthreads();
        const int32_t n = radix_count[tid];
        const unsigned long long units = radix_units[tid];
        int32_t n_to = n;
        unsigned long long u_to = units;
        row_scan2(n_to, rooms[turn].count, u_to, rooms[turn].units);
        turn ^= 1;
        // the digit in which the end lies: not reached in front of it, and reached with it, or the last that there is
        const bool open = end_count > 0 ? n_above + n_to - n < end_count : (double)(u_above + u_to - units) < end_units;
        const uint64_t those = __builtin_amdgcn_ballot_w64(n > 0 && open);
        if (lane == 0 && those != 0) atomicMax(&found_at, wave * kWave + 63 - __builtin_clzll(those));
        __syncthreads();
        const int digit = found_at;
        if (digit < 0) break;                                // (no token: a bin that is asked for has one)
        if (tid == digit) {
          found_n = n;
          found_key = (uint64_t)(uint32_t)(n_above + n_to - n);
          found_units = u_above + (u_to - units);
        }
        __syncthreads();
        n_left = found_n;                                    // tokens of the digit; tokens, units in front of it
        n_above = (int32_t)found_key;
        u_above = found_units;
        to -= (uint64_t)digit << down;
        const uint64_t width = (1ull << down) - 1;
        from = to - from > width ? to - width : from;
        continue;
      }
      __syncthreads();
      each_token(from, to, [&](uint64_t key, bool inside) __attribute__((always_inline)) {
        if (!inside) return;
        const int i = atomicAdd(&found_n, 1);
        if (i < kRanked) {
          rank_key[i] = key;
          rank_units[i] = units_of_key(key);
        }
      });
      __syncthreads();
      const int n = found_n < kRanked ? found_n : kRanked;
      if (tid < n) {
        const uint64_t mine = rank_key[tid];
        int32_t before = n_above, ahead_of = 0;
        uint64_t units_before = u_above;
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
          const bool ahead = rank_key[i] > mine;
          ahead_of += ahead;
          units_before += ahead ? rank_units[i] : 0;
        }
        before += ahead_of;
        const uint64_t with = units_before + rank_units[tid];
        const bool is_last = ahead_of + 1 == n;             // (where a rounding keeps the end from being reached)
        const bool ends = end_count > 0 ? before + 1 == end_count || (is_last && before + 1 < end_count)
                                        : (double)units_before < end_units && ((double)with >= end_units || is_last);
        if (ends) {
          found_key = mine;
          found_units = with;
        }
      }
      __syncthreads();
      break;
    }
    const uint64_t end = found_key;
    if (filter == 0) {
      whole = false;
      cut = end;
      kept = (last > 0 ? mass_to[last - 1] : 0.0) + (double)found_units * bin_top[last];
    } else if (bin < last || whole || end > cut) {
      last = bin;
      whole = false;
      cut = end;
    }
  }

  // Kept are the tokens from the key `cut` on, and above the cut of y.
  uint64_t token = 0;
  double all = 1.0;                                      // of the largest's mass: exactly 1 where it is all that is kept
  if (few) {
    // By the index: the run of indexes in which the target lies, then the token in it.
    const int width = (vocab + kRowThreads - 1) / kRowThreads;
    __syncthreads();
    radix_units[tid] = 0;
    if (tid == 0) found_n = 0;
    __syncthreads();
    each_listed(cut, ~0ull, [&](uint64_t key, bool inside) __attribute__((always_inline)) {
      if (inside) atomicAdd(&radix_units[keys.index(key) / width], (unsigned long long)units_kept(key));
    });
    __syncthreads();
    const unsigned long long here = radix_units[tid];
    unsigned long long sum;
    const unsigned long long upto = row_scan(here, rooms[turn].units, &sum);
    turn ^= 1;
    const double target = u * (double)sum * (2.0 - kReached);
    if ((double)upto > target && !((double)(upto - here) > target)) {
      found_at = tid;
      found_units = upto - here;
    }
    __syncthreads();
    const int run = found_at;
    const uint64_t before_run = found_units;
    each_listed(cut, ~0ull, [&](uint64_t key, bool inside) __attribute__((always_inline)) {
      if (!inside || keys.index(key) / width != run) return;
      const int to = atomicAdd(&found_n, 1);
      rank_key[to] = key;                                  // (of `width` indexes, at most kRun)
      rank_units[to] = units_kept(key);
    });
    __syncthreads();
    const int n = found_n;
    for (int i = tid; i < n; i += kRowThreads) {
      const uint64_t mine = rank_key[i];
      const int32_t at = keys.index(mine);
      uint64_t units_before = before_run;
#pragma unroll 8
      for (int j = 0; j < n; ++j) units_before += keys.index(rank_key[j]) < at ? rank_units[j] : 0;
      if ((double)(units_before + rank_units[i]) > target && !((double)units_before > target)) token = mine;
    }
    if (token == 0) return;
    all = (double)sum / (double)units_kept(most_key);
  } else {
    // The kept mass of each slice: its bins in front of the last, and what it has of that one.
    if (whole) cut = keys.lowest(lowest_of_bin(top - last, t, z_per_x));      // (top_k may end with a bin)
    for (int s = tid; s < slices; s += kRowThreads) slice_units[s] = 0;
    __syncthreads();
    if (!whole) {
      each_token(cut > low ? cut : low, high, [&](uint64_t key, bool inside) __attribute__((always_inline)) {
        const int s = inside ? (keys.index(key) + in.lead) / kPer / slice_vectors : 0;
        const uint64_t units = units_of_key(key);
        atomicAdd(&slice_units[s], (unsigned long long)(inside ? units : 0));
      });
    }
    // (16 lanes a slice)
    const int bins_kept = last + (whole ? 1 : 0);
    for (int s0 = 0; s0 < slices; s0 += kRowThreads / 16) {
      const int s = s0 + tid / 16 < slices ? s0 + tid / 16 : slices - 1;
      double sum = 0.0;
      constexpr int kBinsAhead = 8;
      for (int b0 = tid % 16; b0 < bins_kept; b0 += 16 * kBinsAhead) {
        uint64_t w[kBinsAhead];
#pragma unroll
        for (int i = 0; i < kBinsAhead; ++i) {
          w[i] = row_bins[(int64_t)s * kSampleSlots + ((top_slot - (b0 + 16 * i)) & (kSampleSlots - 1))];
        }
#pragma unroll
        for (int i = 0; i < kBinsAhead; ++i) {
          const int b = b0 + 16 * i;
          const uint64_t x = b < bins_kept ? word(w[i], s, b) : 0;
          sum += (double)((x & kUnitsMask) + kFloorUnits * (x >> kCountShift)) * bin_top[b & (kSampleSlots - 1)];
        }
      }
      sum = over_row<16>(sum, [](double a, double b) { return a + b; });
      if (s0 + tid / 16 < slices && tid % 16 == 0) slice_mass[s] = sum;
    }
    __syncthreads();
    if (wave == 0) {
      // 64 slices at a time: the sums of mass, then the first slice by whose end the target is passed; the last if none
      const double above = whole ? 0.0 : bin_top[last];
      double sum = 0.0;
      for (int s0 = 0; s0 < slices; s0 += kWave) {
        const int s = s0 + lane;
        const double to = wave_scan(s < slices ? slice_mass[s] + (double)slice_units[s] * above : 0.0) + sum;
        if (s < slices) slice_mass[s] = to;
        sum = __shfl(to, kWave - 1, kWave);
      }
      const double target = u * sum * (2.0 - kReached);
      int slice = slices - 1;
      for (int s0 = 0; s0 < slices; s0 += kWave) {
        const int s = s0 + lane;
        const uint64_t past = __builtin_amdgcn_ballot_w64(s < slices && slice_mass[s] > target);
        if (past != 0) {
          slice = s0 + __builtin_ctzll(past);
          break;
        }
      }
      if (lane == 0) {
        found_slice = slice;
        rooms[turn].mass[0] = sum;
        rooms[turn].mass[1] = target - (slice > 0 ? slice_mass[slice - 1] : 0.0);
      }
    }
    __syncthreads();
    all = rooms[turn].mass[0];
    double target = rooms[turn].mass[1];
    turn ^= 1;
#pragma unroll 1
    for (int s = found_slice; s < slices; ++s) {
      // a thread has neighbouring elements
      constexpr int kVectors = kSampleSlice / kPer / kRowThreads;
      float x[kVectors][kPer];
      const int each = (slice_vectors + kRowThreads - 1) / kRowThreads;
      const int64_t v0 = (int64_t)s * slice_vectors + (int64_t)tid * each;
      uint4_t raw[kVectors];
#pragma unroll
      for (int i = 0; i < kVectors; ++i) raw[i] = in.vector(v0 + i);
      double share[kVectors * kPer], sum = 0.0;
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        logits_of<TYPE>(in, raw[i], i < each && tid * each + i < slice_vectors ? v0 + i : in.vectors, vocab, x[i]);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const uint64_t key = keys.of(order_of(x[i][j]), (int32_t)((v0 + i) * kPer - in.lead + j));
          const double of_it = mass_of(key);                 // (of any: without branches several are on their way at once)
          share[i * kPer + j] = x[i][j] > -INFINITY && key >= cut ? of_it : 0.0;
          sum += share[i * kPer + j];
        }
      }
      if (tid == 0) found_at = 0x7fffffff;
      double slice_all;
      double upto = row_scan(sum, rooms[turn].mass, &slice_all) - sum;
      turn ^= 1;
      int here = 0x7fffffff;
      uint64_t here_key = 0;
#pragma unroll
      for (int i = 0; i < kVectors * kPer; ++i) {
        upto += share[i];
        if (here == 0x7fffffff && share[i] > 0.0 && upto > target) {
          here = (int)(v0 * kPer + i - in.lead);
          here_key = keys.of(order_of(x[i / kPer][i % kPer]), here);
        }
      }
      if (here != 0x7fffffff) atomicMin(&found_at, here);
      __syncthreads();
      if (found_at != 0x7fffffff) {
        if (here != found_at) return;
        token = here_key;
        break;
      }
      target = 0.0;                                        // (a rounding: the next that is kept)
      __syncthreads();
    }
    all /= mass_of(most_key);
    if (token == 0) {                                      // (never: u is below 1, so some slice passes the target)
      if (tid == 0) tokens[row] = -1;
      return;
    }
  }
  answer(token, all);
}

}  // namespace litekv

extern "C" size_t litekv_sample_tokens_workspace_bytes(int32_t logits_type, int32_t batch, int32_t vocab) {
  using namespace litekv;
  if (logits_type < kLogitsF16 || logits_type > kLogitsF32 || batch < 1 || batch > 65535 || vocab < 1 || vocab > kSampleMaxVocab) return 0;
  const int size = logit_size(logits_type), per = sample_slice_vectors(batch, vocab, size);
  const int64_t slices = (sample_vectors(vocab, size) + per - 1) / per;
  return (size_t)batch * (size_t)slices * (sizeof(SampleSlice) + (kSampleSlots + kSliceList) * sizeof(uint64_t));
}

extern "C" int litekv_sample_tokens(const void *logits, int32_t logits_type, int64_t row_stride, const float *uniforms,
                                    const float *temperature, const int32_t *top_k, const float *top_p,
                                    const float *min_p, int64_t *tokens, float *logprobs, int32_t batch, int32_t vocab,
                                    void *workspace, size_t workspace_bytes, void *stream) {
  using namespace litekv;
  const char *what = "sample_tokens";
  LITEKV_REQUIRE(logits_type >= kLogitsF16 && logits_type <= kLogitsF32, "%s: logits_type %d is not 0 (fp16), 1 (bf16) or 2 (fp32)",
                 what, logits_type);
  LITEKV_REQUIRE(batch >= 0 && batch <= 65535, "%s: batch %d out of [0, 65535]", what, batch);
  LITEKV_REQUIRE(vocab >= 1 && vocab <= kSampleMaxVocab, "%s: vocab %d out of [1, %d]", what, vocab, kSampleMaxVocab);
  if (batch == 0) {
    clear_error();
    return LITEKV_OK;
  }
  const int size = logit_size(logits_type);
  LITEKV_REQUIRE(logits && uniforms && tokens, "%s: null pointer", what);
  LITEKV_REQUIRE((uintptr_t)logits % size == 0, "%s: logits must be aligned to an element", what);
  LITEKV_REQUIRE(batch == 1 || row_stride >= 0, "%s: row stride %lld < 0", what, (long long)row_stride);
  const size_t need = litekv_sample_tokens_workspace_bytes(logits_type, batch, vocab);
  LITEKV_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, "%s: workspace of %zu bytes needed, got %zu", what,
                 need, workspace_bytes);
  const int per = sample_slice_vectors(batch, vocab, size);
  const int slices = (int)((sample_vectors(vocab, size) + per - 1) / per);
  SampleSlice *heads = static_cast<SampleSlice *>(workspace);
  uint64_t *bins = reinterpret_cast<uint64_t *>(heads + (int64_t)batch * slices);
  uint64_t *lists = bins + (int64_t)batch * slices * kSampleSlots;
  auto launch = [&](auto slices_kernel, auto rows_kernel) {
    hipLaunchKernelGGL(slices_kernel, dim3((unsigned)slices, (unsigned)batch), dim3(kSampleThreads), 0,
                       static_cast<hipStream_t>(stream), logits, row_stride, temperature, vocab, per, slices, heads, bins, lists);
    const int rc = check_launch(what);
    if (rc != LITEKV_OK) return rc;
    hipLaunchKernelGGL(rows_kernel, dim3((unsigned)batch), dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), logits,
                       row_stride, uniforms, temperature, top_k, top_p, min_p, tokens, logprobs, vocab, per, slices, heads, bins, lists);
    return check_launch(what);
  };
  switch (logits_type) {
    case kLogitsF16: return launch(sample_slices_kernel<kLogitsF16>, sample_rows_kernel<kLogitsF16>);
    case kLogitsBf16: return launch(sample_slices_kernel<kLogitsBf16>, sample_rows_kernel<kLogitsBf16>);
    default: return launch(sample_slices_kernel<kLogitsF32>, sample_rows_kernel<kLogitsF32>);
  }
}
