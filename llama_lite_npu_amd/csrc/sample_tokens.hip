// One token per row of logits, drawn with a given uniform number under temperature, top-k, top-p and min-p.
//
// With y = x / T and p = exp(y - max y), the three filters each keep a prefix of the tokens ordered by p (ties: the lowest index
// first), so what is kept is the shortest of three prefixes: everything above one logit, and the first few of those that equal
// it. The token is the first, by index, at which the kept mass exceeds u times all of it.
//
// Nothing is sorted. A first launch cuts the rows into slices, a workgroup each, and leaves per slice a histogram over y: bins of
// 1/8 on a grid that all slices share, each with the number and the mass of its tokens. A second one, a workgroup per row, adds
// them up, walks the bins to the one in which a filter's prefix ends, reads the row's tokens of that bin again and finds the
// logit by their bits, ten at a time. Sums of mass are sums of whole numbers: the mass of a token is rounded to 2^-40
// of its bin's top (y enters in fp64, and exp by a polynomial over the width of a bin), so no order of additions shows in a
// token, and a bin's top is a factor applied once. A cumulative mass is then within 2^-41 of itself wherever it is compared, which
// in a row of 150 000 tokens moves one draw in some millions to a neighbour of the token that exact arithmetic gives.
#include <cmath>

#include "common.h"

namespace litekv {

constexpr int kSampleBins = 322;              // of 1/8: what is further than 40 below a row's largest y is never drawn
constexpr int kSampleThreads = 256;           // of a slice's workgroup
constexpr int kSampleSlice = 8192;            // tokens of a slice at most: their number has 14 bits of a bin's word
constexpr int kRowThreads = 1024;             // of a row's workgroup
constexpr int kSampleList = 8192;             // tokens that a row's workgroup holds
constexpr int kSampleMaxVocab = 1 << 20;
constexpr int kRadix = 1024;
constexpr double kUnit = 0x1p-40;             // of a bin's top
constexpr double kFloor = 0.875;              // below exp(-1/8): a bin's word has the sum of what is above it
constexpr uint64_t kFloorUnits = 7ull << 37;
constexpr uint64_t kMostUnits = (1ull << 37) - 1;
constexpr int kCountShift = 50;
constexpr uint64_t kUnitsMask = (1ull << kCountShift) - 1;
constexpr double kCut = -40.0;
constexpr double kReached = 1.0 - 0x1p-40;    // a border that rounding alone keeps from being reached is

struct SampleSlice {      // of the workspace, in front of the histograms
  double top;             // the bin of its largest y, counted from 0
  float most;             // its largest logit, -inf: nothing can be drawn
  int32_t at;             // the first token that has it
};

// The vectors of 16 bytes that a row's slices are counted in: of V elements, the first of them anywhere in its vector.
__host__ __device__ constexpr int64_t sample_vectors(int64_t vocab, int size) { return (vocab * size + 30) / 16; }
static int sample_slice_vectors(int32_t batch, int32_t vocab, int size) {
  int tokens = kSampleSlice;
  while (tokens > 2048 && (int64_t)batch * ((vocab + tokens - 1) / tokens) < 256) tokens /= 2;
  return tokens * size / 16;
}

enum { kLogitsF16 = 0, kLogitsBf16 = 1, kLogitsF32 = 2 };
constexpr int logit_size(int type) { return type == kLogitsF32 ? 4 : 2; }

// The elements of one vector as floats; what cannot be drawn is -inf. NaN is such a one; infinity is the largest finite number.
template <int TYPE>
__device__ __forceinline__ void logits_of(uint4_t raw, int64_t first, int32_t vocab, float (&x)[16 / logit_size(TYPE)]) {
  constexpr int kPer = 16 / logit_size(TYPE);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    float f;
    if constexpr (TYPE == kLogitsF32) {
      const uint32_t word = raw[i];        // (a bit cast of the element itself is one of the first)
      f = __builtin_bit_cast(float, word);
    } else if constexpr (TYPE == kLogitsBf16) {
      f = __builtin_bit_cast(float, i & 1 ? raw[i >> 1] & 0xffff0000u : raw[i >> 1] << 16);
    } else {
      f = (float)__builtin_bit_cast(half_t, (uint16_t)(raw[i >> 1] >> (16 * (i & 1))));
    }
    const int64_t at = first + i;
    const bool there = at >= 0 && at < vocab && f == f;
    x[i] = there ? __builtin_fminf(f, 3.4028234663852886e38f) + 0.0f : -INFINITY;   // (+ 0: the two zeros are one)
  }
}

// Where the vector `at` of a row is; only those with an element of the row are read.
struct LogitsRow {
  const char *base;        // the row's first vector
  int lead;                // elements in front of the row in it
  int64_t vectors;
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

// The bin of y = x / T counted from 0, and the token's mass in units of the bin's top, less the floor's.
struct Binned {
  double bin;
  uint64_t units;
};
__device__ __forceinline__ double bin_of(float x, double inv_t) { return __builtin_floor((double)x * inv_t * 8.0); }
__device__ __forceinline__ Binned binned(float x, double inv_t) {
  const double y = (double)x * inv_t;
  const double b = __builtin_floor(y * 8.0);
  // exp(y - top), top = (b + 1) / 8: exp(-1/16) exp(r), |r| <= 1/16, to 2^-43 of itself
  const double r = (y - b * 0.125) - 0.0625;
  double e = 1.0 / 5040.0;
  e = __builtin_fma(e, r, 1.0 / 720.0);
  e = __builtin_fma(e, r, 1.0 / 120.0);
  e = __builtin_fma(e, r, 1.0 / 24.0);
  e = __builtin_fma(e, r, 1.0 / 6.0);
  e = __builtin_fma(e, r, 0.5);
  e = __builtin_fma(e, r, 1.0);
  e = __builtin_fma(e, r, 1.0);
  constexpr double kMiddle = 0.93941306281347578611;      // exp(-1/16)
  // in whole units, as the low bits of a sum with 2^52
  const double u = __builtin_fma(e, kMiddle / kUnit, -kFloor / kUnit);
  const uint64_t bits = __builtin_bit_cast(uint64_t, __builtin_fmin(__builtin_fmax(u, 0.0), (double)kMostUnits) + 0x1p52);
  return Binned{b, bits & ((1ull << 52) - 1)};
}

__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of_order(uint32_t k) {
  return __builtin_bit_cast(float, k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ float row_temperature(const float *temperature, int row) {
  const float t = temperature != nullptr ? temperature[row] : 1.0f;
  return t > 3.4028234663852886e38f ? 3.4028234663852886e38f : t;      // (NaN stays)
}
__device__ __forceinline__ bool greedy_temperature(float t) { return !(t > 0.f); }

// A slice: its largest logit, then its histogram. Bound by memory, and behind it by the LDS additions.
template <int TYPE>
__global__ __launch_bounds__(kSampleThreads) void sample_slices_kernel(
    const void *__restrict__ logits, int64_t row_stride, const float *__restrict__ temperature, int32_t vocab,
    int32_t slice_vectors, int32_t slices, SampleSlice *__restrict__ heads, uint64_t *__restrict__ bins) {
  constexpr int kPer = 16 / logit_size(TYPE);
  constexpr int kMostVectors = kSampleSlice / kPer / kSampleThreads;
  __shared__ uint64_t hist[kSampleBins];
  __shared__ float wave_most[kSampleThreads / kWave];
  __shared__ int wave_at[kSampleThreads / kWave];
  const int tid = threadIdx.x, row = blockIdx.y, slice = blockIdx.x;
  const LogitsRow in = logits_row<TYPE>(logits, row_stride, row, vocab);
  const float t = row_temperature(temperature, row);
  for (int i = tid; i < kSampleBins; i += kSampleThreads) hist[i] = 0;
  const int64_t v0 = (int64_t)slice * slice_vectors;
  float x[kMostVectors][kPer];
  uint4_t raw[kMostVectors];
#pragma unroll
  for (int i = 0; i < kMostVectors; ++i) {
    const int v = i * kSampleThreads + tid;
    raw[i] = uint4_t{0, 0, 0, 0};
    if (v < slice_vectors && v0 + v < in.vectors) raw[i] = *(const uint4_t *)(in.base + (v0 + v) * 16);
  }
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMostVectors; ++i) {
    const int v = i * kSampleThreads + tid;
    const bool there = v < slice_vectors && v0 + v < in.vectors;
    logits_of<TYPE>(raw[i], there ? (v0 + v) * kPer - in.lead : -kPer, vocab, x[i]);
#pragma unroll
    for (int k = 0; k < kPer; ++k) most = fmaxf(most, x[i][k]);
  }
  const int wave = tid / kWave;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) most = fmaxf(most, __shfl_xor(most, off, kWave));
  if (tid % kWave == 0) wave_most[wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSampleThreads / kWave; ++w) most = fmaxf(most, wave_most[w]);
  SampleSlice *head = heads + (int64_t)row * slices + slice;
  if (most == -INFINITY) {
    if (tid == 0) *head = SampleSlice{0.0, -INFINITY, 0};
    return;
  }
  if (greedy_temperature(t)) {
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kMostVectors; ++i) {
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int e = (int)((v0 + i * kSampleThreads + tid) * kPer - in.lead + k);
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
    for (int w = 0; w < kSampleThreads / kWave; ++w) at = wave_at[w] < at ? wave_at[w] : at;
    if (tid == 0) *head = SampleSlice{0.0, most, at};
    return;
  }
  const double inv_t = 1.0 / (double)t;
  const double top = bin_of(most, inv_t);
#pragma unroll
  for (int i = 0; i < kMostVectors; ++i) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (x[i][k] > -INFINITY) {
        const Binned b = binned(x[i][k], inv_t);
        const double d = top - b.bin;
        if (d < (double)kSampleBins) {
          atomicAdd((unsigned long long *)&hist[(int)d], (unsigned long long)(b.units | (1ull << kCountShift)));
        }
      }
    }
  }
  __syncthreads();
  uint64_t *to = bins + ((int64_t)row * slices + slice) * kSampleBins;
  for (int i = tid; i < kSampleBins; i += kSampleThreads) to[i] = hist[i];
  if (tid == 0) *head = SampleSlice{top, most, 0};
}

// ---- a row ---------------------------------------------------------------------------------------------------------------------
// Inclusive sums over the workgroup's threads, in one order.
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const T up = __shfl_up(x, off, kWave);
    if (lane >= off) x += up;
  }
  return x;
}
template <typename T>
__device__ __forceinline__ T row_scan(T x, T *room, T *total) {      // room: kRowThreads / kWave
  const int wave = threadIdx.x / kWave;
  x = wave_scan(x);
  __syncthreads();
  if (threadIdx.x % kWave == kWave - 1) room[wave] = x;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / kWave; ++w) {
    before += w < wave ? room[w] : T(0);
    all += room[w];
  }
  *total = all;
  return before + x;
}

// What a filter's end in a bin comes to: of the bin's tokens those above `order`, and the first `ties` of those that equal it.
struct Ending {
  uint32_t order;
  int32_t ties;
  uint64_t units;       // of the bin's tokens that are kept
};

template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_rows_kernel(
    const void *__restrict__ logits, int64_t row_stride, const float *__restrict__ uniforms,
    const float *__restrict__ temperature, const int32_t *__restrict__ top_k, const float *__restrict__ top_p,
    const float *__restrict__ min_p, int64_t *__restrict__ tokens, float *__restrict__ logprobs, int32_t vocab,
    int32_t slice_vectors, int32_t slices, const SampleSlice *__restrict__ heads, const uint64_t *__restrict__ bins) {
  constexpr int kPer = 16 / logit_size(TYPE);
  constexpr int kMaxSlices = 520;
  __shared__ double bin_top[kSampleBins];            // exp(the bin's top - the row's largest y), in units
  __shared__ double mass_to[kSampleBins];            // inclusive
  __shared__ int32_t count_to[kSampleBins];
  __shared__ int32_t shift[kMaxSlices];              // of a slice's bins against the row's, kSampleBins: it has none
  __shared__ int32_t slice_from[kMaxSlices + 1];     // where its tokens begin in the list
  __shared__ double slice_mass[kMaxSlices];
  __shared__ unsigned long long slice_units[kMaxSlices];
  __shared__ int32_t slice_ties[kMaxSlices];
  __shared__ uint32_t list_order[kSampleList];
  __shared__ int32_t list_at[kSampleList];
  __shared__ unsigned long long radix_units[kRadix];
  __shared__ int32_t radix_count[kRadix];
  __shared__ double room_d[kRowThreads / kWave];
  __shared__ unsigned long long room_u[kRowThreads / kWave];
  __shared__ int32_t room_i[kRowThreads / kWave];
  __shared__ float room_f[kRowThreads / kWave];
  __shared__ int32_t found_bin, found_k, found_at, found_slice;
  __shared__ uint32_t bound_low, bound_high;
  __shared__ Ending ending;
  const int tid = threadIdx.x, row = blockIdx.x, wave = tid / kWave, lane = tid % kWave;
  const LogitsRow in = logits_row<TYPE>(logits, row_stride, row, vocab);
  const SampleSlice *head = heads + (int64_t)row * slices;
  const uint64_t *row_bins = bins + (int64_t)row * slices * kSampleBins;
  const float t = row_temperature(temperature, row);

  // the row's largest logit
  float most = -INFINITY;
  for (int s = tid; s < slices; s += kRowThreads) most = fmaxf(most, head[s].most);
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) most = fmaxf(most, __shfl_xor(most, off, kWave));
  if (lane == 0) room_f[wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowThreads / kWave; ++w) most = fmaxf(most, room_f[w]);
  if (most == -INFINITY) {                            // nothing can be drawn
    if (tid == 0) {
      tokens[row] = -1;
      if (logprobs != nullptr) logprobs[row] = -INFINITY;
    }
    return;
  }
  if (greedy_temperature(t)) {
    if (tid == 0) {
      int at = 0x7fffffff;
      for (int s = 0; s < slices; ++s) {
        if (head[s].most == most) {                   // (slices are in the tokens' order)
          at = head[s].at;
          break;
        }
      }
      tokens[row] = at;
      if (logprobs != nullptr) logprobs[row] = 0.f;
    }
    return;
  }
  const double inv_t = 1.0 / (double)t;
  const double y_most = (double)most * inv_t;
  const double top = __builtin_floor(y_most * 8.0);
  for (int s = tid; s < slices; s += kRowThreads) {
    const double d = head[s].most == -INFINITY ? (double)kSampleBins : top - head[s].top;
    shift[s] = d < (double)kSampleBins ? (int)d : kSampleBins;
  }
  __syncthreads();
  auto word_of = [&](int s, int b) -> uint64_t {      // bin b of the row in slice s
    const int at = b - shift[s];
    return at >= 0 && shift[s] < kSampleBins ? row_bins[(int64_t)s * kSampleBins + at] : 0;
  };
  // its bins
  {
    int32_t count = 0;
    double mass = 0.0;
    if (tid < kSampleBins) {
      uint64_t units = 0;
      for (int s = 0; s < slices; ++s) {
        const uint64_t w = word_of(s, tid);
        count += (int32_t)(w >> kCountShift);
        units += w & kUnitsMask;
      }
      const double scale = kUnit * exp((top * 0.125 - y_most) + (1 - tid) * 0.125);   // (of any size: the first difference is exact)
      bin_top[tid] = scale;
      mass = (double)(units + kFloorUnits * (uint64_t)count) * scale;
    }
    int32_t count_all;
    double mass_all;
    count = row_scan(count, room_i, &count_all);
    mass = row_scan(mass, room_d, &mass_all);
    if (tid < kSampleBins) {
      count_to[tid] = count;
      mass_to[tid] = mass;
    }
  }
  __syncthreads();
  const int32_t live = count_to[kSampleBins - 1];
  const double mass_live = mass_to[kSampleBins - 1];

  const int32_t k = top_k != nullptr ? top_k[row] : 0;
  const float p = top_p != nullptr ? top_p[row] : 1.0f;
  const float m = min_p != nullptr ? min_p[row] : 0.0f;
  bool by_k = k > 0 && k < live, by_p = p < 1.0f;
  const bool by_m = m > 0.0f;

  // The interval of logits, by order, that bins `from` to `to` have: the border of a bin is within a few floats of its place.
  auto bounds = [&](int from, int to) {
    __syncthreads();
    if (wave < 2) {
      // wave 0: the lowest logit whose bin is at most `to`; wave 1: the lowest whose bin is below `from`
      const double limit = top - (wave == 0 ? to : from - 1);        // its bin, counted from 0
      const float guess = (float)__builtin_fmin(__builtin_fmax(limit * 0.125 * (double)t, -3.4028234663852886e38), 3.4028234663852886e38);
      const int64_t o = (int64_t)order_of(guess + 0.0f) + lane - 32;
      const uint32_t lowest = order_of(-3.4028234663852886e38f), highest = order_of(3.4028234663852886e38f);
      const bool above = o > (int64_t)highest || (o >= (int64_t)lowest && bin_of(logit_of_order((uint32_t)o), inv_t) >= limit);
      const uint64_t all = __builtin_amdgcn_ballot_w64(above);
      const int first = all != 0 ? __builtin_ctzll(all) : 63;
      if (lane == first) {
        const uint32_t border = o < (int64_t)lowest ? lowest : (uint32_t)o;
        if (wave == 0) {
          bound_low = border;
        } else {
          bound_high = border - 1;
        }
      }
    }
    __syncthreads();
    if (from <= 0 && tid == 0) bound_high = order_of(most);
    __syncthreads();
  };

  // The tokens of bins [list_bins_from, list_bins_to], in their order; a wavefront takes a slice at a time.
  int list_from = 0, list_to = -1, listed = 0;
  auto gather = [&](int from, int to) {
    if (list_from <= from && to <= list_to) return;
    bounds(from, to);
    const uint32_t low = bound_low, high = bound_high;
    for (int s = wave; s < slices; s += kRowThreads / kWave) {
      int32_t n = 0;
      for (int b = from + lane; b <= to; b += kWave) n += (int32_t)(word_of(s, b) >> kCountShift);
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) n += __shfl_xor(n, off, kWave);
      if (lane == 0) slice_ties[s] = n;
    }
    __syncthreads();
    if (tid == 0) {
      int32_t at = 0;
      for (int s = 0; s < slices; ++s) {
        slice_from[s] = at;
        at += slice_ties[s];
      }
      slice_from[slices] = at;
    }
    __syncthreads();
    for (int s = wave; s < slices; s += kRowThreads / kWave) {
      int32_t at = slice_from[s];
      if (slice_from[s + 1] == at) continue;
      for (int v = 0; v < slice_vectors; v += kWave) {
        const int64_t vec = (int64_t)s * slice_vectors + v + lane;
        const bool there = v + lane < slice_vectors && vec < in.vectors;
        const uint4_t raw = there ? *(const uint4_t *)(in.base + vec * 16) : uint4_t{0, 0, 0, 0};
        float x[kPer];
        const int64_t first = there ? vec * kPer - in.lead : -kPer;
        logits_of<TYPE>(raw, first, vocab, x);
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const uint32_t o = order_of(x[i]);
          mine |= (o >= low && o <= high ? 1u : 0u) << i;
        }
        if (__builtin_amdgcn_ballot_w64(mine != 0) == 0) continue;
        const int32_t n = __builtin_popcount(mine);
        const int32_t upto = wave_scan(n);
        int32_t to_at = at + upto - n;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if ((mine >> i & 1) && to_at < kSampleList) {
            list_order[to_at] = order_of(x[i]);
            list_at[to_at++] = (int32_t)(first + i);
          }
        }
        at += __shfl(upto, kWave - 1, kWave);
      }
    }
    __syncthreads();
    list_from = from;
    list_to = to;
    listed = slice_from[slices] < kSampleList ? slice_from[slices] : kSampleList;
  };
  // Whether a bin's tokens fit the list; else they are read from the row each time.
  auto fits = [&](int from, int to) { return count_to[to] - (from > 0 ? count_to[from - 1] : 0) <= kSampleList; };

  // Every token of a bin: from the list, or from the row.
  auto each_of_bin = [&](int bin, bool in_list, uint32_t low, uint32_t high, auto &&what) {
    if (in_list) {
      for (int i = tid; i < listed; i += kRowThreads) {
        const uint32_t o = list_order[i];
        if (o >= low && o <= high) what(o, list_at[i]);
      }
    } else {
      for (int64_t v = tid; v < in.vectors; v += kRowThreads) {
        float x[kPer];
        const int64_t first = v * kPer - in.lead;
        logits_of<TYPE>(*(const uint4_t *)(in.base + v * 16), first, vocab, x);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const uint32_t o = order_of(x[i]);
          if (o >= low && o <= high) what(o, (int32_t)(first + i));
        }
      }
    }
  };
  // Where a prefix ends in a bin: at the first token with which the bin's tokens are `count` (count > 0), or have `units` (a
  // number above 0 of units). The bits of their orders are looked at ten at a time.
  auto end_in_bin = [&](int bin, int32_t count, double units) -> Ending {
    const bool in_list = fits(bin, bin);
    if (in_list) gather(bin, bin);
    bounds(bin, bin);
    uint32_t low = bound_low, high = bound_high;
    int32_t n_above = 0;
    uint64_t u_above = 0;
    while (true) {
      int down = 0;
      while (((high - low) >> down) >= (uint32_t)kRadix) ++down;
      for (int i = tid; i < kRadix; i += kRowThreads) {
        radix_units[i] = 0;
        radix_count[i] = 0;
      }
      __syncthreads();
      each_of_bin(bin, in_list, low, high, [&](uint32_t o, int32_t) {
        const uint32_t r = (high - o) >> down;          // from the largest
        atomicAdd(&radix_count[r], 1);
        atomicAdd(&radix_units[r], (unsigned long long)(binned(logit_of_order(o), inv_t).units + kFloorUnits));
      });
      __syncthreads();
      static_assert(kRadix == kRowThreads, "a thread has a digit");
      int32_t n_all;
      unsigned long long u_all;
      const int32_t n = radix_count[tid];
      const unsigned long long u = radix_units[tid];
      const int32_t n_to = row_scan(n, room_i, &n_all);
      const unsigned long long u_to = row_scan(u, room_u, &u_all);
      if (tid == 0) found_at = kRadix;
      __syncthreads();
      const bool reached = count > 0 ? n_above + n_to >= count : (double)(u_above + u_to) >= units;
      if (n > 0 && reached) atomicMin(&found_at, tid);
      // (nowhere, by a rounding: the last that there is)
      if (tid == 0) found_k = -1;
      __syncthreads();
      if (n > 0) atomicMax(&found_k, tid);
      __syncthreads();
      const int digit = found_at < kRadix ? found_at : found_k;
      if (digit < 0) return Ending{low, 0x7fffffff, u_above};      // (no token: a bin that is asked for has one)
      if (tid == digit) {
        ending.ties = n_above + n_to - n;                 // tokens, units in front of the digit
        ending.units = u_above + (u_to - u);
        ending.order = (uint32_t)n;
      }
      __syncthreads();
      n_above = ending.ties;
      u_above = ending.units;
      const int32_t here = (int32_t)ending.order;
      const uint32_t new_high = high - ((uint32_t)digit << down);
      const uint32_t width = (1u << down) - 1;
      const uint32_t new_low = new_high - low > width ? new_high - width : low;
      __syncthreads();
      low = new_low;
      high = new_high;
      if (down == 0) {
        const uint64_t each = binned(logit_of_order(high), inv_t).units + kFloorUnits;
        int32_t ties = here;
        if (count > 0) {
          ties = count - n_above < here ? count - n_above : here;
        } else {
          const double more = __builtin_ceil((units - (double)u_above) / (double)each);
          if (more < (double)here) ties = more < 1.0 ? 1 : (int32_t)more;
        }
        return Ending{high, ties, u_above + each * (uint64_t)ties};
      }
    }
  };

  // The filters, one after the other. `last`: the bin that the kept prefix ends in; `cut`: what of it is kept.
  int last = kSampleBins - 1;
  bool whole = true;                                    // all of bin `last`
  Ending cut{0u, 0, 0};
  double kept = mass_live;
  // The first bin of those with a token that is reached; the last with a token if none is.
  auto first_bin = [&](auto &&reached) -> int {
    __syncthreads();
    if (tid == 0) found_bin = kSampleBins;
    if (tid == 1) found_k = 0;
    __syncthreads();
    if (tid < kSampleBins && count_to[tid] > (tid > 0 ? count_to[tid - 1] : 0)) {
      if (reached(tid)) atomicMin(&found_bin, tid);
      atomicMax(&found_k, tid);
    }
    __syncthreads();
    return found_bin < kSampleBins ? found_bin : found_k;
  };
  // Where the prefixes end; one that ends behind min_p's (bin_m, or a bin more) says nothing, but top_k says what top_p is of.
  int bin_k = kSampleBins - 1, bin_p = kSampleBins - 1, bin_m = kSampleBins - 1;
  double log_m = 0.0;
  if (by_m) {
    log_m = log((double)(m < 1.0f ? m : 1.0f)) * (double)t;          // kept: x - most >= log_m
    const double b = top - __builtin_floor((y_most + log_m * inv_t) * 8.0) + 1.0;
    if (b < (double)bin_m) bin_m = (int)b;
  }
  if (by_k) bin_k = first_bin([&](int b) { return count_to[b] >= k; });
  if (by_p && !by_k) {
    const double target = (double)p * mass_live * kReached;
    bin_p = first_bin([&](int b) { return mass_to[b] >= target; });
    by_p = bin_p <= bin_m;
  } else if (!by_p) {
    by_k = by_k && bin_k <= bin_m;
  }
  // Where few tokens come into question they are listed at once, the draw's among them.
  const int most_bin = by_k ? bin_k : by_p ? bin_p : bin_m;
  const bool few = fits(0, most_bin);
  if (few) gather(0, most_bin);
  if (by_k) {
    last = bin_k;
    const int32_t before = last > 0 ? count_to[last - 1] : 0;
    if (count_to[last] > k) {
      whole = false;
      cut = end_in_bin(last, k - before, 0.0);
      kept = (last > 0 ? mass_to[last - 1] : 0.0) + (double)cut.units * bin_top[last];
    } else {
      kept = mass_to[last];
    }
  }
  if (by_p) {
    const double target = (double)p * kept * kReached;
    int bin = first_bin([&](int b) { return mass_to[b] >= target; });
    if (bin > last) bin = last;
    const double before = bin > 0 ? mass_to[bin - 1] : 0.0;
    Ending e = end_in_bin(bin, 0, __builtin_fmax((target - before) / bin_top[bin], 1.0));
    if (bin < last || whole || e.order > cut.order || (e.order == cut.order && e.ties < cut.ties)) {
      last = bin;
      whole = false;
      cut = e;
    }
  }
  if (by_m) {
    // the lowest order that is kept: within a few floats of most + log_m
    __syncthreads();
    if (wave == 0) {
      const float guess = (float)__builtin_fmax((double)most + log_m, -3.4028234663852886e38);
      const int64_t o = (int64_t)order_of(guess + 0.0f) + lane - 32;
      const int64_t lowest = order_of(-3.4028234663852886e38f);
      const bool above = o >= (int64_t)order_of(most) ||
                         (o >= lowest && (double)logit_of_order((uint32_t)o) - (double)most >= log_m);
      const uint64_t all = __builtin_amdgcn_ballot_w64(above);
      const int first = all != 0 ? __builtin_ctzll(all) : 63;
      if (lane == first) bound_low = (uint32_t)(o < lowest ? lowest : o);
    }
    __syncthreads();
    const uint32_t order = bound_low;
    const double d = top - bin_of(logit_of_order(order), inv_t);
    const int bin = d < (double)kSampleBins ? (int)d : kSampleBins;
    if (bin < kSampleBins && (bin < last || (bin == last && (whole || order > cut.order)))) {
      last = bin;
      whole = false;
      cut = Ending{order, 0x7fffffff, 0};
    }
  }
  __syncthreads();

  // Kept tokens: order above cut.order, or equal and among the first cut.ties; whole: all of them above the cut of y.
  const uint32_t least = whole ? 0u : cut.order;
  const int32_t most_ties = whole ? 0x7fffffff : cut.ties;
  double u = (double)uniforms[row];
  u = u > 0.0 ? (u < 1.0 - 0x1p-24 ? u : 1.0 - 0x1p-24) : 0.0;
  const double x_cut = kCut * (double)t;
  auto mass_of = [&](uint32_t o) -> double {
    const float x = logit_of_order(o);
    if ((double)x - (double)most < x_cut) return 0.0;
    const Binned b = binned(x, inv_t);
    const double d = top - b.bin;
    return d < (double)kSampleBins ? (double)(b.units + kFloorUnits) * bin_top[(int)d] : 0.0;
  };
  auto finish = [&](int32_t token, uint32_t order, double all) {
    tokens[row] = token;
    if (logprobs != nullptr) {
      logprobs[row] = (float)(((double)logit_of_order(order) - (double)most) * inv_t - log(all));
    }
  };
  if (few) {
    // the list has them all, in their order: a thread has a run of it
    constexpr int kRun = kSampleList / kRowThreads;
    const int each = (listed + kRowThreads - 1) / kRowThreads;
    double mass[kRun];
    int32_t ties = 0, ties_all;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int at = tid * each + i;
      if (i < each && at < listed && list_order[at] == least) ++ties;
    }
    int32_t tie = row_scan(ties, room_i, &ties_all) - ties;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int at = tid * each + i;
      mass[i] = 0.0;
      if (i < each && at < listed) {
        const uint32_t o = list_order[at];
        if (o > least || (o == least && tie++ < most_ties)) mass[i] = mass_of(o);
      }
      sum += mass[i];
    }
    double all;
    double upto = row_scan(sum, room_d, &all) - sum;
    const double target = u * all * (2.0 - kReached);
    if (tid == 0) found_at = kSampleList;
    __syncthreads();
    int here = kSampleList;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      upto += mass[i];
      if (here == kSampleList && mass[i] > 0.0 && upto > target) here = tid * each + i;
    }
    if (here < kSampleList) atomicMin(&found_at, here);
    __syncthreads();
    if (tid == 0) {
      const int at = found_at < kSampleList ? found_at : listed - 1;
      finish(list_at[at], list_order[at], all);
    }
    return;
  }

  // The kept mass of each slice: its bins in front of the last, and what it has of that one.
  for (int s = tid; s < slices; s += kRowThreads) {
    slice_units[s] = 0;
    slice_ties[s] = 0;
  }
  __syncthreads();
  if (!whole) {
    const bool in_list = fits(last, last);
    if (in_list) gather(last, last);
    for (int s = tid; s < slices; s += kRowThreads) slice_ties[s] = 0;        // (the gather's)
    bounds(last, last);
    const uint32_t low = bound_low > least ? bound_low : least, high = bound_high;
    each_of_bin(last, in_list, low, high, [&](uint32_t o, int32_t at) {
      const int s = (int)((at + in.lead) / kPer / slice_vectors);
      if (o == least) {
        atomicAdd(&slice_ties[s], 1);
      } else {
        atomicAdd(&slice_units[s], (unsigned long long)(binned(logit_of_order(o), inv_t).units + kFloorUnits));
      }
    });
    __syncthreads();
  }
  for (int s = wave; s < slices; s += kRowThreads / kWave) {
    double sum = 0.0;
    for (int b = lane; b < last + (whole ? 1 : 0); b += kWave) {
      const uint64_t w = word_of(s, b);
      sum += (double)((w & kUnitsMask) + kFloorUnits * (w >> kCountShift)) * bin_top[b];
    }
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) sum += __shfl_xor(sum, off, kWave);
    if (lane == 0) slice_mass[s] = sum;
  }
  __syncthreads();
  if (tid == 0) {
    const double each = whole ? 0.0 : mass_of(least);
    int32_t left = most_ties;
    double all = 0.0;
    for (int s = 0; s < slices; ++s) {
      const int32_t n = slice_ties[s] < left ? slice_ties[s] : left;
      slice_from[s] = left;                              // ties that a slice may keep
      left -= n;
      slice_mass[s] += (double)slice_units[s] * (whole ? 0.0 : bin_top[last]) + (double)n * each;
      all += slice_mass[s];
    }
    const double target = u * all * (2.0 - kReached);
    double upto = 0.0;
    int s = 0;
    while (s + 1 < slices && !(upto + slice_mass[s] > target)) upto += slice_mass[s++];
    found_slice = s;
    room_d[0] = all;
    room_d[1] = target - upto;
  }
  __syncthreads();
  const double all = room_d[0];
  double target = room_d[1];
  for (int s = found_slice; s < slices; ++s) {
    // a thread has neighbouring elements
    constexpr int kVectors = kSampleSlice / kPer / kRowThreads;
    uint32_t order[kVectors * kPer];
    int32_t ties = 0, ties_all;
    const int each = (slice_vectors + kRowThreads - 1) / kRowThreads;
    const int64_t v0 = (int64_t)s * slice_vectors + (int64_t)tid * each;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const bool there = i < each && tid * each + i < slice_vectors && v0 + i < in.vectors;
      float x[kPer];
      logits_of<TYPE>(there ? *(const uint4_t *)(in.base + (v0 + i) * 16) : uint4_t{0, 0, 0, 0},
                      there ? (v0 + i) * kPer - in.lead : -kPer, vocab, x);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        order[i * kPer + j] = x[j] > -INFINITY ? order_of(x[j]) : 0u;
        if (order[i * kPer + j] == least && !whole) ++ties;
      }
    }
    int32_t tie = row_scan(ties, room_i, &ties_all) - ties;
    const int32_t may = slice_from[s];
    double sum = 0.0;
    double mass[kVectors * kPer];
#pragma unroll
    for (int i = 0; i < kVectors * kPer; ++i) {
      const bool is = order[i] > least || (order[i] == least && !whole && tie++ < may);
      mass[i] = is && order[i] != 0u ? mass_of(order[i]) : 0.0;
      sum += mass[i];
    }
    double slice_all;
    double upto = row_scan(sum, room_d, &slice_all) - sum;
    if (tid == 0) found_at = 0x7fffffff;
    __syncthreads();
    int here = 0x7fffffff;
    uint32_t here_order = 0;
#pragma unroll
    for (int i = 0; i < kVectors * kPer; ++i) {
      upto += mass[i];
      if (here == 0x7fffffff && mass[i] > 0.0 && upto > target) {
        here = (int)(v0 * kPer + i - in.lead);
        here_order = order[i];
      }
    }
    if (here != 0x7fffffff) atomicMin(&found_at, here);
    __syncthreads();
    if (found_at != 0x7fffffff) {
      if (here == found_at) finish(here, here_order, all);
      return;
    }
    target = 0.0;                                        // (a rounding: the next that is kept)
    __syncthreads();
  }
}

}  // namespace litekv

extern "C" size_t litekv_sample_tokens_workspace_bytes(int32_t logits_type, int32_t batch, int32_t vocab) {
  using namespace litekv;
  if (logits_type < kLogitsF16 || logits_type > kLogitsF32 || batch < 1 || batch > 65535 || vocab < 1 || vocab > kSampleMaxVocab) return 0;
  const int size = logit_size(logits_type), per = sample_slice_vectors(batch, vocab, size);
  const int64_t slices = (sample_vectors(vocab, size) + per - 1) / per;
  return (size_t)batch * (size_t)slices * (sizeof(SampleSlice) + kSampleBins * sizeof(uint64_t));
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
  auto launch = [&](auto slices_kernel, auto rows_kernel) {
    hipLaunchKernelGGL(slices_kernel, dim3((unsigned)slices, (unsigned)batch), dim3(kSampleThreads), 0,
                       static_cast<hipStream_t>(stream), logits, row_stride, temperature, vocab, per, slices, heads, bins);
    const int rc = check_launch(what);
    if (rc != LITEKV_OK) return rc;
    hipLaunchKernelGGL(rows_kernel, dim3((unsigned)batch), dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), logits,
                       row_stride, uniforms, temperature, top_k, top_p, min_p, tokens, logprobs, vocab, per, slices, heads, bins);
    return check_launch(what);
  };
  switch (logits_type) {
    case kLogitsF16: return launch(sample_slices_kernel<kLogitsF16>, sample_rows_kernel<kLogitsF16>);
    case kLogitsBf16: return launch(sample_slices_kernel<kLogitsBf16>, sample_rows_kernel<kLogitsBf16>);
    default: return launch(sample_slices_kernel<kLogitsF32>, sample_rows_kernel<kLogitsF32>);
  }
}
