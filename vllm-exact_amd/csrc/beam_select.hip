// Beam search's selection over beams and vocabulary (gfx950).
//
//   score(b, v) = scores[b] + x_bv - log sum_u exp(x_bu)
// for the beams b of a request; the `count` largest, in order. An fp64 score of a beam's log-sum, whose terms are fp32 and whose sums
// are fp64, orders beams against each other, equal ones by b; within a beam the logits themselves do, equal ones by v. (A score in which
// the logits drown, as of a beam held at -1e30, is the same for all tokens of the beam. As a score rises with its logit, this
// is one order of all continuations, by which slices and requests choose alike.)
//
// A row of logits is cut into slices, a workgroup each. A thread holds its values in registers, so the logits are read
// once: maximum, sum of exponentials, and the slice's `count` largest. Those are among the values that are at least the
// count-th largest of a wave's 64 lane maxima, a handful more than `count`. A second kernel, a workgroup for each request,
// joins the slices' sums and picks from their candidates in the same way.
// A slice's place goes by the vocabulary alone, so a row's sums are the same bits in any batch and at any alignment.
//
// What bounds it: 256 rows of 248320 bf16 logits are 127 MB, 26 us at the rate of a large copy (19 at that of plain reads); the slices take
// 41.0 us and the join 8.5. Vector instructions are in flight for 76 % of the slices' cycles: 19 a logit, of which 10 take a logit apart
// twice and add its exponential (one of them at a quarter of the rate), the others find the bar, look through the runs near it and
// rank the candidates, work that a slice has whatever its size (half as many logits a thread: 48.9 us, the join 13.5). Loads alone are 30:
// a workgroup has one slice, and while it computes only the others' loads are in flight. (Workgroups that stay and ask for their
// next slice first need its registers as well, which costs as many waves: 58 us.) 4 rows of 151936: 7.0 + 5.5, two launches' latency.

#include "attention_common.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kWords = 32;                 // of a thread's values, as they are in memory: 62 to 80 registers, 6 to 8 waves a SIMD
template <int DTYPE>
constexpr int kEach = DTYPE == VXA_F32 ? kWords : 2 * kWords;  // values of a thread, in runs of 8
template <int DTYPE>
constexpr int kSlice = kThreads * kEach<DTYPE>;                // values of a workgroup
constexpr int kMost = 64;                  // of `count`: a wave has so many lane maxima
constexpr int kWaveList = 128;             // candidates that a wave may list; where more values are near (many equal ones) it looks closer
constexpr int kMostSlices = 4096;          // of a request

typedef unsigned long long u64;

struct BeamParams {
  const void* logits;
  int64_t stride;
  const float* scores;
  int32_t n, beams, vocab, count, slices;
  double* sums;   // [n * beams][slices][waves]: of exp(x - top)
  float* tops;    // [n * beams][slices][waves]: the largest value, -inf: none
  u64* keys;      // [n * beams][slices][count], the largest first, 0: none
  float* out_scores;
  int32_t* out_parents;
  int64_t* out_tokens;
};

// Order of floats as whole numbers; -inf is 0, which is no candidate. Keys order by value, then the lower place first.
__device__ inline uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 is 0
  return x == -__builtin_huge_valf() ? 0u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ inline float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ inline u64 key_of(uint32_t order, uint32_t place) { return order ? (u64)order << 32 | (uint32_t)~place : 0; }

__device__ inline u64 shfl_u64(u64 x, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_ds_bpermute(lane << 2, (int)(x >> 32)) << 32 |
         (uint32_t)__builtin_amdgcn_ds_bpermute(lane << 2, (int)(uint32_t)x);
}
__device__ inline u64 wave_max(u64 x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const u64 y = shfl_u64(x, lane ^ m);
    x = y > x ? y : x;
  }
  return x;
}
__device__ inline double wave_sum(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) x += __builtin_bit_cast(double, shfl_u64(__builtin_bit_cast(u64, x), lane ^ m));
  return x;
}

// exp(d) for -80 <= d <= 0, off by a few 2^-25 where |d| is not much above 10, as it is for what carries a sum of 2^17 terms: the power
// of 2 of the rounded product with log2(e), and what the rounding left, d less the product times log(2), as a factor of 1 more than it.
__device__ inline float exp_of(float d) {
  const float p = d * 1.44269504f, e = exp2_hw(p);
  return fmaf(e, fmaf(p, -0.693147182f, d), e);
}

// Element of a row of logits, which may start at any element.
template <int DTYPE>
using Element = std::conditional_t<DTYPE == VXA_F32, float, uint16_t>;
template <int DTYPE>
__device__ inline float value(Element<DTYPE> e) {
  if constexpr (DTYPE == VXA_F32)
    return e;
  else if constexpr (DTYPE == VXA_BF16)
    return bf16_to_f32(e);
  else
    return (float)__builtin_bit_cast(_Float16, e);
}
template <int DTYPE>
__device__ inline uint32_t word(Element<DTYPE> e) {  // in the lower half, or the whole
  if constexpr (DTYPE == VXA_F32)
    return __float_as_uint(e);
  else
    return e;
}

template <int DTYPE>
__global__ __launch_bounds__(kThreads, 6) void beam_slice_kernel(BeamParams p) {
  constexpr int kEach = ::kEach<DTYPE>, kSlice = ::kSlice<DTYPE>, kRun = 8 * kWords / kEach;  // words of a run
  __shared__ u64 s_list[kWaves * kWaveList];
  __shared__ int s_count;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slice = blockIdx.x % p.slices, row = blockIdx.x / p.slices;
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();

  // Run r of a thread: places slice * kSlice + r * 8 * kThreads + 8 * thread + 0..7. Its values stay as they came; each pass takes
  // them apart again, which costs less than the waves that twice as many registers would.
  const Element<DTYPE>* logits = reinterpret_cast<const Element<DTYPE>*>(p.logits) + (int64_t)row * p.stride;
  auto place_of = [&](int i) { return slice * kSlice + (i / 8 * kThreads + (int)threadIdx.x) * 8 + i % 8; };
  uint32_t w[kWords];
  auto x = [&](int i) {
    if constexpr (DTYPE == VXA_F32)
      return __uint_as_float(w[i]);
    else if constexpr (DTYPE == VXA_BF16)
      return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    else
      return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i / 2] >> (16 * (i % 2))));
  };
  auto again = [&] {
    if constexpr (DTYPE != VXA_F32)
#pragma unroll
      for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
  };
  constexpr uint32_t kNothing = DTYPE == VXA_F32 ? 0xFF800000u : DTYPE == VXA_BF16 ? 0xFF80FF80u : 0xFC00FC00u;  // -inf
  const bool whole = (slice + 1) * kSlice <= p.vocab;
  if (whole || p.vocab >= 8) {
#pragma unroll
    for (int r = 0; r < kEach / 8; ++r) __builtin_memcpy(w + r * kRun, logits + (whole ? place_of(8 * r) : min(place_of(8 * r), p.vocab - 8)), 4 * kRun);
  }
  if (!whole) {
#pragma unroll
    for (int r = 0; r < kEach / 8; ++r) {
      const int place = place_of(8 * r);
      if (place + 8 > p.vocab) {
#pragma unroll
        for (int j = 0; j < kRun; ++j) w[r * kRun + j] = kNothing;
        if (place < p.vocab) {  // the run that the row ends in
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t e = word<DTYPE>(logits[min(place + j, p.vocab - 1)]);
            uint32_t& to = w[r * kRun + j * kRun / 8];
            if (place + j < p.vocab) to = DTYPE == VXA_F32 ? e : j % 2 ? (to & 0xFFFFu) | e << 16 : (to & 0xFFFF0000u) | e;
          }
        }
      }
    }
  }

  float runs[kEach / 8], top = kNegInf;  // the largest values; a NaN where there is one
#pragma unroll
  for (int r = 0; r < kEach / 8; ++r) {
    runs[r] = x(8 * r);
#pragma unroll
    for (int j = 1; j < 8; ++j) runs[r] = __builtin_elementwise_maximum(runs[r], x(8 * r + j));
    top = __builtin_elementwise_maximum(top, runs[r]);
  }
  if (top != top) top = __builtin_nanf("");
  const uint32_t mine = order_of(top);
  const uint32_t highest = (uint32_t)(wave_max((u64)mine << 32) >> 32);
  const float most = value_of(highest);  // a NaN's order is above all others
  double sum = 0.0;
  again();
  if (highest != 0 && !(most < __builtin_huge_valf())) {
    sum = __builtin_nan("");
  } else if (highest != 0) {  // what is more than 80 below counts as nothing in fp64 sums of 2^31 terms
#pragma unroll
    for (int i = 0; i < kEach; i += 8) {
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) part += exp_of(__builtin_amdgcn_fmed3f(x(i + j) - most, -80.0f, 0.0f));
      sum += (double)part;
    }
    sum = wave_sum(sum);
  }
  if (lane == 0) p.tops[(int64_t)blockIdx.x * kWaves + wave] = highest ? most : kNegInf, p.sums[(int64_t)blockIdx.x * kWaves + wave] = sum;

  // The count-th largest order among the lanes' maxima, bit by bit; at least 1. (Orders of 16-bit types differ in the upper bits.)
  uint32_t bar = 0;
#pragma unroll
  for (int b = 31; b >= (DTYPE == VXA_F32 ? 0 : DTYPE == VXA_BF16 ? 16 : 13); --b)
    if (__popcll(__ballot(mine >= (bar | 1u << b))) >= p.count) bar |= 1u << b;
  const float least = bar == 0 ? -3.402823466e38f : value_of(bar);
  // This lane's values that are not below the bar, one bit each. Few runs have one: those are read again.
  u64 mask = 0;
  uint32_t near = 0;
#pragma unroll
  for (int r = 0; r < kEach / 8; ++r) near |= runs[r] >= least ? 1u << r : 0u;
  for (; near != 0; near &= near - 1) {
    const int r = __builtin_ctz(near), place = place_of(8 * r);
    Element<DTYPE> e[8];
    int skip = 0;
    if (whole || p.vocab >= 8) {
      skip = max(place - (p.vocab - 8), 0);
      __builtin_memcpy(e, logits + (place - skip), sizeof(e));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = logits[min(j, p.vocab - 1)];
    }
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) bits |= value<DTYPE>(e[j]) >= least ? 1u << j : 0u;
    if (p.vocab < 8) bits &= (1u << p.vocab) - 1;
    mask |= (u64)(bits >> skip) << (8 * r);
  }
  const int many = __popcll(mask);
  const int before = wave_scan(many, [](int a, int b) { return a + b; });
  const int all = __builtin_amdgcn_readlane(before, 63);
  if (all <= kWaveList) {
    int at = 0;
    if (lane == 0 && all) at = atomicAdd(&s_count, all);
    at = __builtin_amdgcn_readfirstlane(at) + before - many;
    for (; mask != 0; mask &= mask - 1) {  // a lane's only one is its maximum
      const int place = place_of(__builtin_ctzll(mask));
      s_list[at++] = key_of(order_of(many > 1 ? value<DTYPE>(logits[place]) : top), (uint32_t)place);
    }
  } else {  // many values are near the bar: the wave's count-th largest value, then all above it and the first that equal it
    uint32_t order = 0;
#pragma unroll 1
    for (uint32_t bit = 1u << 31; bit != 0; bit >>= 1) {
      const float v = value_of(order | bit);
      again();
      int n = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) n += x(i) >= v;
      if (wave_reduce(n, [](int a, int b) { return a + b; }) >= p.count) order |= bit;
    }
    const float kth = value_of(order);
    int at = 0;
    if (lane == 0) at = atomicAdd(&s_count, p.count);
    at = __builtin_amdgcn_readfirstlane(at);
    const int end = at + p.count;
#pragma unroll
    for (int equal = 0; equal < 2; ++equal) {
      again();
#pragma unroll
      for (int r = 0; r < kEach; r += 8) {  // places rise with the run, then the lane, then within the run
        int n = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) n += equal ? x(r + j) == kth : x(r + j) > kth;
        const int upto = wave_scan(n, [](int a, int b) { return a + b; });
        int mine_at = at + upto - n;
        if (n)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((equal ? x(r + j) == kth : x(r + j) > kth) && mine_at < end) s_list[mine_at++] = key_of(order_of(x(r + j)), (uint32_t)place_of(r + j));
        at += __builtin_amdgcn_readlane(upto, 63);
      }
    }
  }
  __syncthreads();

  // A candidate's rank is how many are larger; 2^share threads compare one.
  const int listed = s_count;
  u64* keys = p.keys + (int64_t)blockIdx.x * p.count;
  int share = 0, valid = 0;
  while (share < 3 && listed << (share + 1) <= kThreads) ++share;
  for (int i0 = 0; i0 < listed; i0 += kThreads >> share) {
    const int i = i0 + ((int)threadIdx.x >> share), part = threadIdx.x & ((1 << share) - 1);
    const u64 key = i < listed ? s_list[i] : 0;
    int rank = 0;
    if (key != 0)
      for (int j = part; j < listed; j += 1 << share) rank += s_list[j] > key;
    for (int m = 1; m < 1 << share; m *= 2) rank += __builtin_amdgcn_ds_bpermute((lane ^ m) << 2, rank);
    if (key != 0 && rank < p.count && part == 0) keys[rank] = key;
    valid += __syncthreads_count(key != 0 && part == 0);
  }
  for (int i = valid + (int)threadIdx.x; i < p.count; i += kThreads) keys[i] = 0;
}

// Order of fp64 scores as whole numbers; -inf is 0.
__device__ inline u64 order_of(double x) {
  const u64 u = __builtin_bit_cast(u64, x + 0.0);
  return x == -__builtin_huge_val() ? 0 : u ^ ((u64)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ inline double score_of(u64 o) { return __builtin_bit_cast(double, o >> 63 ? o ^ 0x8000000000000000ull : ~o); }

constexpr int kJoin = 1024;

// A request has at most 4096 slices, each with its `count` largest in order. Of the slices' first ones the count-th largest is a bar
// that no candidate below passes, so at most count slices, count^2 candidates, are ranked in LDS.
__global__ __launch_bounds__(kJoin) void beam_join_kernel(BeamParams p) {
  // Of beam b: its largest logit, the log of its sum of exp(x - largest), its score (-inf: no continuations).
  __shared__ float s_top[kMost * 16];
  __shared__ double s_log[kMost * 16], s_score[kMost * 16];
  __shared__ u64 s_order[kMostSlices];        // of the slices' best, then of the candidates
  __shared__ u64 s_tail[kMostSlices];         // order of the logit, then ~place, a place being beam * vocab + token
  __shared__ int s_count, s_bar, s_nan;
  const int request = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row0 = (int64_t)request * p.beams;
  if (threadIdx.x == 0) s_count = 0, s_bar = -1, s_nan = 0;
  __syncthreads();
  for (int b = wave; b < p.beams; b += kJoin / 64) {
    const int parts = p.slices * kWaves;
    const float* tops = p.tops + (row0 + b) * parts;
    const double* sums = p.sums + (row0 + b) * parts;
    float m = kNegInf;
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, tops[i]);
#pragma unroll
    for (int k = 1; k < 64; k *= 2) m = fmaxf(m, shfl_xor_f32(m, k));
    double s = 0.0;
    for (int i = lane; i < parts; i += 64) s += tops[i] == kNegInf ? sums[i] : sums[i] * exp((double)tops[i] - (double)m);
    s = wave_sum(s);
    const float given = p.scores[row0 + b];
    const double score = s == 0.0 ? -__builtin_huge_val() : (double)given;  // no token, or a beam that has ended
    const double l = log(s);
    if (lane == 0) {
      s_top[b] = m, s_log[b] = l, s_score[b] = score;
      if (!(given < __builtin_huge_valf()) || (score != -__builtin_huge_val() && !(score - l - (double)m < __builtin_huge_val() && l == l))) s_nan = 1;
    }
  }
  __syncthreads();
  const int64_t out = (int64_t)request * p.count;
  if (s_nan) {
    for (int i = threadIdx.x; i < p.count; i += kJoin) p.out_scores[out + i] = __builtin_nanf(""), p.out_parents[out + i] = -1, p.out_tokens[out + i] = -1;
    return;
  }
  const int groups = p.beams * p.slices;
  const u64* keys = p.keys + row0 * p.slices * p.count;
  auto score = [&](int group, int rank, u64& order, u64& tail) {
    const u64 key = keys[(int64_t)group * p.count + rank];
    const int b = group / p.slices;
    // the differences first: they are exact, or nearly, where logits are large
    order = key && s_score[b] != -__builtin_huge_val() ? order_of(s_score[b] + (((double)value_of((uint32_t)(key >> 32)) - (double)s_top[b]) - s_log[b])) : 0;
    tail = key - (uint32_t)b * (uint32_t)p.vocab;  // ~(x + y) = ~x - y, and no borrow: places are less than 2^31
  };
  auto beam_of = [&](u64 tail) { return ~(uint32_t)tail / (uint32_t)p.vocab; };
  // Scores, then beams, then logits, then tokens. With equal scores tails alone say it, but where two beams' logits differ.
  auto above = [&](u64 o, u64 t, u64 order, u64 tail) {
    return o != order ? o > order : beam_of(t) == beam_of(tail) ? t > tail : (uint32_t)t > (uint32_t)tail;
  };
  // f(i, how many are above number i), of the n in LDS, for one of the 2^share threads that compare number i together.
  auto rank_all = [&](int n, auto&& f) {
    int share = 0;  // at most 4
    while (n >> share > 4 && n << (share + 1) <= kJoin) ++share;
    const int part = threadIdx.x & ((1 << share) - 1);
    for (int i0 = 0; i0 < n; i0 += kJoin >> share) {
      const int i = i0 + ((int)threadIdx.x >> share);
      const u64 order = i < n ? s_order[i] : 0, tail = i < n ? s_tail[i] : 0;
      int rank = 0;
      if (order) {
        uint32_t differ = 0;
        for (int j = part; j < n; j += 1 << share) {
          const u64 o = s_order[j], t = s_tail[j];
          rank += o > order || (o == order && t > tail);
          differ |= o == order ? (uint32_t)((t ^ tail) >> 32) : 0u;
        }
        if (differ) {  // rare: scores in which logits drown
          rank = 0;
          for (int j = part; j < n; j += 1 << share) rank += above(s_order[j], s_tail[j], order, tail);
        }
      }
      for (int m = 1; m < 1 << share; m *= 2) rank += __builtin_amdgcn_ds_bpermute((lane ^ m) << 2, rank);
      if (order && part == 0) f(i, rank);
    }
  };
  for (int g = threadIdx.x; g < groups; g += kJoin) score(g, 0, s_order[g], s_tail[g]);
  __syncthreads();
  // The slice whose best is the count-th: no candidate below it is among the best.
  rank_all(groups, [&](int g, int rank) {
    if (rank == p.count - 1) s_bar = g;
  });
  __syncthreads();
  const int bar = s_bar;
  const u64 least = bar >= 0 ? s_order[bar] : 1, least_tail = bar >= 0 ? s_tail[bar] : 0;
  __syncthreads();
  // At most count slices have candidates from there on, of count each: a slice's first one is its best in this order too.
  for (int i = threadIdx.x; i < groups * p.count; i += kJoin) {
    u64 order, tail;
    score(i / p.count, i % p.count, order, tail);
    if (order && !above(least, least_tail, order, tail)) {
      const int at = atomicAdd(&s_count, 1);
      s_order[at] = order, s_tail[at] = tail;
    }
  }
  __syncthreads();
  const int listed = s_count;
  rank_all(listed, [&](int i, int rank) {
    if (rank < p.count) {
      const uint32_t place = ~(uint32_t)s_tail[i];
      p.out_scores[out + rank] = (float)score_of(s_order[i]);
      p.out_parents[out + rank] = (int32_t)(row0 + place / (uint32_t)p.vocab);
      p.out_tokens[out + rank] = place % (uint32_t)p.vocab;
    }
  });
  for (int i = listed + (int)threadIdx.x; i < p.count; i += kJoin)
    p.out_scores[out + i] = kNegInf, p.out_parents[out + i] = -1, p.out_tokens[out + i] = -1;
}

int64_t slices_of(int64_t vocab) { return cdiv<int64_t>(vocab, kSlice<VXA_F32>); }  // the most, of any type

int check_sizes(int64_t n, int64_t beams, int64_t vocab, int64_t count) {
  if (n < 0 || beams <= 0 || vocab <= 0 || count <= 0) return VXA_ERR_ARG;
  if (count > kMost || beams > kMost * 16 || vocab > (1LL << 31) - kSlice<VXA_BF16> || beams * vocab >= 1LL << 31 || beams * slices_of(vocab) > kMostSlices ||
      n > (1 << 30) || n * beams > (1LL << 31) - 1)
    return VXA_ERR_UNSUPPORTED;
  return VXA_OK;
}

}  // namespace

extern "C" int vxa_beam_select_workspace(int64_t n, int64_t beams, int64_t vocab, int64_t count, size_t* ws_bytes) {
  const int rc = check_sizes(n, beams, vocab, count);
  if (rc != VXA_OK || !ws_bytes) return rc != VXA_OK ? rc : VXA_ERR_ARG;
  const int64_t slices = product({n, beams, slices_of(vocab)});
  *ws_bytes = (size_t)product({slices, 8 * count + 12 * kWaves});
  return VXA_OK;
}

extern "C" int vxa_beam_select(const void* logits, int64_t stride_row, int dtype, const float* scores, int64_t n, int64_t beams,
                               int64_t vocab, int64_t count, float* out_scores, int32_t* out_parents, int64_t* out_tokens, void* ws,
                               size_t ws_bytes, vxa_stream_t stream) {
  size_t bytes = 0;
  const int rc = vxa_beam_select_workspace(n, beams, vocab, count, &bytes);
  if (rc != VXA_OK) return rc;
  if (dtype != VXA_F32 && dtype != VXA_BF16 && dtype != VXA_F16) return VXA_ERR_ARG;
  if (n == 0) return VXA_OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens) return VXA_ERR_ARG;
  if (!ws || (uintptr_t)ws % 16 || ws_bytes < bytes) return VXA_ERR_WORKSPACE;
  BeamParams p;
  p.logits = logits, p.stride = stride_row, p.scores = scores;
  p.n = (int32_t)n, p.beams = (int32_t)beams, p.vocab = (int32_t)vocab, p.count = (int32_t)count, p.slices = (int32_t)cdiv<int64_t>(vocab, dtype == VXA_F32 ? kSlice<VXA_F32> : kSlice<VXA_BF16>);
  const int64_t blocks = n * beams * p.slices;
  if (!launchable(blocks, kThreads) || !launchable(n, kJoin)) return VXA_ERR_UNSUPPORTED;
  p.sums = reinterpret_cast<double*>(ws);
  p.keys = reinterpret_cast<u64*>(p.sums + blocks * kWaves);
  p.tops = reinterpret_cast<float*>(p.keys + blocks * count);
  p.out_scores = out_scores, p.out_parents = out_parents, p.out_tokens = out_tokens;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), threads(kThreads);
  if (dtype == VXA_F32)
    hipLaunchKernelGGL(beam_slice_kernel<VXA_F32>, grid, threads, 0, st, p);
  else if (dtype == VXA_BF16)
    hipLaunchKernelGGL(beam_slice_kernel<VXA_BF16>, grid, threads, 0, st, p);
  else
    hipLaunchKernelGGL(beam_slice_kernel<VXA_F16>, grid, threads, 0, st, p);
  VXA_CHECK_LAUNCH();
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)n), dim3(kJoin), 0, st, p);
  VXA_CHECK_LAUNCH();
  return VXA_OK;
}
