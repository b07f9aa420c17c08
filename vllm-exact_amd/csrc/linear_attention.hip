// Linear attention with a decay for each head (gfx950): whole prompts, and one new token of every sequence.
//
//   S_t = exp(g) S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
// for every row t of a sequence, S a D x D matrix of each head in fp32, g the head's log_decay. A sequence starts from a slot of
// a pool of states (or zeros) and ends in one.

#include <algorithm>

#include "attention_common.h"

namespace {

struct LinearParams {
  const uint16_t* q;
  int64_t sqt, sqh;
  const uint16_t* k;
  int64_t skt, skh;
  const uint16_t* v;
  int64_t svt, svh;
  const int32_t* cu;  // of prompts
  int32_t n, total, H, G;
  int32_t part;  // rows of a part of a long sequence
  const float* log_decay;
  float scale;
  void* out;
  int64_t sot, soh;
  int32_t out_dtype;
  bool out_wide;  // the output has the input's type and its rows start on 16 bytes
  float* state;
  int64_t sss, ssh;
  int32_t slots;
  const int32_t *read, *write;  // null: zeros, and not kept
};

// A sequence's slots, -1: none. bad: a slot that the pool does not have, or that another sequence writes, or reads where this
// one writes it: such a sequence's rows are NaN and its state is not written.
struct Slots {
  int read, write;
  bool bad;
};
__device__ inline Slots find_slots(const LinearParams& p, int seq) {
  Slots s{p.read ? p.read[seq] : -1, p.write ? p.write[seq] : -1, false};
  bool bad = s.read >= p.slots || s.write >= p.slots;
  if (p.n == 1 || !p.write) {  // no other sequence writes
    s.bad = bad;
    return s;
  }
  for (int j = threadIdx.x; j < p.n; j += blockDim.x) {
    const int w = p.write[j];
    if (j != seq) bad |= (w >= 0 && (w == s.write || w == s.read)) || (p.read && s.write >= 0 && p.read[j] == s.write);
  }
  s.bad = __syncthreads_or(bad);
  return s;
}

// exp(g rows), what a state decays by, as an fp32 number and its rest: rounded to fp32 alone, its error would grow with every step and
// every call, as the states' own roundings do not.
struct Decay {
  float whole, rest;
};
__device__ inline Decay decay_of(float g, int rows) {
  const double exact = exp((double)g * rows);
  return {(float)exact, (float)(exact - (double)(float)exact)};
}
// exp(g) s + add of a state's value. The rest counts for finite values alone: an infinity times it would be NaN, or one of the other sign.
// (Infinities are clamped. A NaN is what the first product is in any case.) Subtracted in place of added, through a register that
// the compiler does not see into: an addition's result would take the place of its summand, and a state that is updated in place registers for two.
__device__ inline float decayed(float s, Decay decay, float add) {
  float less = fmaf(__builtin_amdgcn_fmed3f(s, kLowest, -kLowest), -decay.rest, -add);
  asm("" : "+v"(less));
  return fmaf(s, decay.whole, -less);
}
// A value that all lanes have, in a scalar register.
__device__ inline float uniform(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }
__device__ inline Decay uniform(Decay x) { return {uniform(x.whole), uniform(x.rest)}; }

// ---------------------------------------------------------------------------------- single tokens
constexpr int kCols = 32;  // columns of a state that a workgroup takes

// A workgroup takes 32 columns of one head's state of one sequence: 128 bytes of each row, D / 8 rows a thread, so that a thread has
// all its loads in flight at once and 64 sequences make 8192 workgroups. It reads and writes every value of the state once, and that is what
// bounds it: 64 sequences, 32 heads of 128, that read 40 different slots, 219 MB: 41 us where a part of the states is in the last cache (62 MB
// fetched, 132 written), 50 us, 4.4 TB/s, where none is. One sequence of 8 heads: 3.7 us, a launch and two dependent loads.
template <typename T, int D>
__global__ __launch_bounds__(256) void linear_step_kernel(LinearParams p) {
  constexpr int kRows = D / 8;  // of the state, of a thread
  __shared__ float s_q[D], s_k[D], s_o[8][kCols];
  constexpr int kSlabs = D / kCols;
  const int slab = blockIdx.x % kSlabs, head = (int)(blockIdx.x / kSlabs) % p.H, seq = (int)(blockIdx.x / kSlabs) / p.H;
  const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
  const Slots slots = find_slots(p, seq);
  const int64_t at = seq * p.sot + head * p.soh + slab * kCols + col;
  if (slots.bad) {
    if (part == 0) store_f32_as(p.out, p.out_dtype, at, __builtin_nanf(""));
    return;
  }
  const int64_t place = head * p.ssh + part * kRows * D + slab * kCols + col;
  float s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) s[i] = slots.read >= 0 ? p.state[slots.read * p.sss + place + (int64_t)i * D] : 0.0f;
  for (int x = threadIdx.x; x < D; x += 256) {
    s_q[x] = T::to_f32(p.q[seq * p.sqt + head * p.sqh + x]);
    s_k[x] = T::to_f32(p.k[seq * p.skt + head / p.G * p.skh + x]);
  }
  const float v = T::to_f32(p.v[seq * p.svt + head / p.G * p.svh + slab * kCols + col]);
  const Decay decay = decay_of(p.log_decay[head], 1);
  __syncthreads();
  float o = 0.0f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    s[i] = decayed(s[i], decay, s_k[part * kRows + i] * v);
    o = fmaf(s_q[part * kRows + i], s[i], o);
  }
  s_o[part][col] = o;
  if (slots.write >= 0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) p.state[slots.write * p.sss + place + (int64_t)i * D] = s[i];
  }
  __syncthreads();
  if (part == 0) {
    o = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o += s_o[i][col];
    store_f32_as(p.out, p.out_dtype, at, o * p.scale);
  }
}

template <typename T>
hipError_t launch_step(int64_t D, const LinearParams& p, hipStream_t st) {
  const int64_t blocks = (int64_t)p.n * p.H * (D / kCols);
  if (!launchable(blocks, 256)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks);
  if (D == 64)
    hipLaunchKernelGGL((linear_step_kernel<T, 64>), grid, dim3(256), 0, st, p);
  else if (D == 128)
    hipLaunchKernelGGL((linear_step_kernel<T, 128>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((linear_step_kernel<T, 256>), grid, dim3(256), 0, st, p);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------- prompts
// Rows go in chunks: with S the state before a chunk of n rows and i, j the rows in it,
//   o_i = scale (exp(g (i + 1)) q_i S + sum_{j <= i} exp(g (i - j)) (q_i . k_j) v_j)
//   S'  = exp(g n) S + sum_j k_j (exp(g (n - 1 - j)) v_j)^T
// All of it runs on the matrix cores, with sums in fp32. What is not 16 bits wide already goes there as several bf16 numbers:
//   S in q S, and the weighted scores: two where outputs have 16 bits, off by at most 2^-17 of each term; such an output is rounded to
//   2^-8 or 2^-11 afterwards. Three where outputs have 32 bits, exactly. (A call of 8192 rows with such outputs, bf16 and 128 dims: 143 us,
//   160 with two parts and chunks of 64 rows; three parts of the scores take chunks of 32. fp16 and 256 dims: 221 and 200. With outputs of 16
//   bits three parts would take 118 us in place of 104, and 195 in place of 174, for last bits of 2 values in 1000.)
//   The weighted values, whose products add up to the state that later tokens start from: three, whose sum is the fp32 number itself.
//   fp16 queries, keys and values beside them: two, exactly. The product of the last parts of both is left out (of two parts 2^-16 of a
//   term, of three 2^-24, in S 2^-22).
// The weights are powers of a whole number of rows, at most 1, never quotients of two powers, which would overflow.
//
// A sequence is walked in order, so 32 heads of one prompt of 8192 rows would be 32 workgroups. It is cut into parts of 320 to 512 rows:
// one launch computes what each part adds to the state (half the work of outputs, 34 us for 8192 rows of 32 heads of 128), one adds
// these up (11 us, and only where a sequence may have three parts), one computes the outputs (69 us). A token at
// a time, one after the other, the same call takes 4128 us. Where the cuts are goes by the sequence
// and the heads alone, and so do a row's bits.
//
// What bounds it: 17.2 GF are 15 us at the rate of a large product, 170 MB 35 us at that of a copy. Behind a 32 x 32 x 16
// product go four vector instructions, and more add up (a loop of products with 0, 4, 8 and 12 fmas to each, two waves a SIMD: 37, 37,
// 47 and 57 clocks a product). Per chunk of 64 rows a wave has 98 products and some 1000 vector instructions that split, weight and
// stage; registers allow two waves a SIMD. Of the outputs' cycles matrix pipes are busy for 31 %, vector instructions in flight for 44 %.
//
// Few heads of a few prompts leave CUs idle with long parts; with many there are enough workgroups, and what counts is each part's state,
// which is written and read. us of a call, bf16, the geometric mean over prompts of 1024, 2048, 4096 and 8192 rows and batches of
// 4 x 1024, 16 x 700 and 3 x 3000, with parts of 320, 384 and 512 rows:
//   64 dims:   8 heads 38, 42, 51;    16: 42, 45, 53;     20: 45, 47, 57;    24: 47, 48, 56;     32: 53, 53, 58;     64: 72, 71, 77
//   128 dims:  8 heads 51, 55, 68;    16: 62, 64, 73;     20: 73, 72, 81;    24: 77, 76, 82;     32: 90, 88, 92;     64: 143, 139, 135
//   256 dims:                         16: 166, 172, 189;                     24: 237, 222, 231;  32: 278, 265, 260
// (32 heads of 128, one of 8192 rows: 136, 129, 115; 16 of 700: 169, 135, 141. 256 dims and 16 heads take 384, as 320 keep a fifth more
// states. Parts of 256 rows: as those of 320, within 9 %.)
constexpr int kMostRows = 512;  // of a part
inline int part_rows(int64_t heads, int64_t dims) { return heads <= 16 && dims <= 128 ? 320 : heads < 32 || dims <= 64 ? 384 : kMostRows; }

__device__ inline float power(float g, int e) { return e == 0 ? 1.0f : expf(g * (float)e); }  // exp(-inf * 0) is 1 here

// Fp32 values as two bf16 operands, off by at most 2^-17 of a value; 16 significant bits are exact. N dwords of two values.
template <int N, typename W>
__device__ inline void split(const float (&x)[N], W (&part)[2]) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    part[0][j / 2] = BF16::pack(x[j], x[j + 1]);
    const v2f f = BF16::unpack(part[0][j / 2]);
    part[1][j / 2] = BF16::pack(x[j] - f.x, x[j + 1] - f.y);
  }
}
// The same as three bf16 operands whose sum they are exactly: cut off after 8 bits, and again. (Cutting takes one instruction
// for two values where rounding takes two or three; with two operands its error would be four times as large.)
template <int N, typename W>
__device__ inline void split(const float (&x)[N], W (&part)[3]) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    float a = x[j], b = x[j + 1];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
      part[n][j / 2] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
      if (n < 2) a -= __uint_as_float(ua & 0xFFFF0000u), b -= __uint_as_float(ub & 0xFFFF0000u);
    }
  }
}
template <typename T>
__device__ inline void floats(v4u32 w, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const v2f f = T::unpack(w[j]);
    x[2 * j] = f.x, x[2 * j + 1] = f.y;
  }
}
// A lane's id, whose uses the compiler does not move across this: places that go by it alone are found again for every
// chunk. Kept, they would take more registers than there are.
__device__ inline int again(int id) {
  asm volatile("" : "+v"(id));
  return id;
}

// Part `part` of sequence seq. The grid has floor(tokens / rows of a part) + n places: the whole parts come first, then what is left of the
// sequences (and empty ones), 64 sequences at a time the longest first, so that the last workgroups are short ones.
struct Part {
  int seq, lo, len, part, parts;  // parts: of the sequence, at least 1
};
__device__ inline Part find_part(const LinearParams& p, int index) {
  const int lane = threadIdx.x & 63;
  auto add = [](int a, int b) { return a + b; };
  auto lengths = [&](int j, int& lo, int& len) {
    lo = len = 0;
    if (j < p.n) {
      lo = min(max(p.cu[j], 0), p.total);
      len = max(min(p.cu[j + 1], p.total) - lo, 0);
    }
  };
  auto found = [&](int j, int lo, int len, int at, bool whole, int part) {  // of lane `at`
    lo = __builtin_amdgcn_readlane(lo, at), len = __builtin_amdgcn_readlane(len, at);
    const int all = len / p.part;
    return Part{j + at, lo, len, whole ? part : all, max(1, all + (len > all * p.part))};
  };
  for (int j0 = 0; j0 < p.n; j0 += 64) {
    int lo, len;
    lengths(j0 + lane, lo, len);
    const int mine = len / p.part, upto = wave_scan(mine, add), all = __builtin_amdgcn_readlane(upto, 63);
    if (index < all) {
      const int at = __builtin_ctzll(__ballot(upto > index));
      return found(j0, lo, len, at, true, index - __builtin_amdgcn_readlane(upto - mine, at));
    }
    index -= all;
  }
  for (int j0 = 0; j0 < p.n; j0 += 64) {
    int lo, len;
    lengths(j0 + lane, lo, len);
    const int rest = len % p.part;
    const bool has = j0 + lane < p.n && (rest != 0 || len == 0);
    const int all = __popcll(__ballot(has)), key = has ? rest * 64 + lane : -1;
    if (index < all) {
      int rank = 0;
      for (int m = 0; m < min(64, p.n - j0); ++m) rank += __builtin_amdgcn_readlane(key, m) > key;
      return found(j0, lo, len, __builtin_ctzll(__ballot(has && rank == index)), false, 0);
    }
    index -= all;
  }
  return Part{0, 0, 0, 0, 0};
}
// Where the state before part `part` of a sequence of several parts is kept: 2 floor(lo / rows of a part) + part. (The parts of a
// sequence longer than one are at most twice its whole ones. Half of the places stay empty: the first state of a sequence needs one where
// it is kept apart alone, and where the sequences before end only their lengths say.)
__device__ inline int64_t kept_at(const LinearParams& p, int lo, int part, int head, int size) {
  return ((int64_t)(2 * (lo / p.part) + part) * p.H + head) * size;
}

// A tile's 16-byte chunks lie at chunk ^ swizzle(row): 16 rows that are read at one chunk meet 16 different ones.
template <typename T, int D, bool OUT, bool WIDE>
struct Shared {
  static constexpr bool F16 = std::is_same_v<T, FP16>;
  // Rows of a chunk: 64 (the state is split and decayed half as often as with 32: 120 us in place of 132 for 8192 rows), where two workgroups'
  // tiles fit a CU's LDS; 32 in fp16, whose queries and keys lie there twice, at 256 dims, and with scores of three parts at 128.
  static constexpr int C = !F16 && D <= (WIDE ? 64 : 128) ? 64 : 32;
  static constexpr int kParts = WIDE ? 3 : 2;  // of the state and the scores as operands
  static constexpr int kTile = C * 2 * D;
  char q[OUT ? kTile : 16], k[OUT ? kTile : 16];                       // for the scores
  char qs[OUT && F16 ? 2 : 1][OUT && F16 ? kTile : 16];                // fp16: queries as two bf16 parts
  char kt[F16 ? 2 : 1][kTile], v[kTile];                               // for transposed reads; fp16: keys as two bf16 parts
  char scores[OUT ? (C == 64 ? 6 : 2) : 1][kParts][OUT ? 1024 : 16];   // operands of 16 keys and 32 queries
  float power[C];                                                      // scale exp(g (C - 1 - x))
  float left[C];                                                       // exp(g (n - 1 - j)) of row j of the chunk, 0 past its end
  int met;                                                             // whether something was not finite
};

// The heads of one KV head on one XCD.
__device__ inline int head_of(const LinearParams& p, int x) { return p.H % 8 == 0 ? (x % 8) * (p.H / 8) + x / 8 : x; }
// A sequence of several parts that writes the slot that it reads keeps its first state apart: its last part may end before the first
// begins.
__device__ inline bool kept_apart(const Part& part, const Slots& slots) { return part.part == 0 && part.parts > 1 && slots.read >= 0 && slots.read == slots.write; }
// Where the state before a part is (null: zeros), for its rows or for what it adds to a state, and where the one after it goes (null: nowhere).
template <bool OUT>
__device__ inline const float* state_before(const LinearParams& p, float* kept, const Part& part, const Slots& slots, int head, int size) {
  if (OUT && (part.part > 0 || kept_apart(part, slots))) return kept + kept_at(p, part.lo, part.part, head, size);
  return part.part == 0 && slots.read >= 0 ? p.state + slots.read * p.sss + head * p.ssh : nullptr;
}
template <bool OUT>
__device__ inline float* state_after(const LinearParams& p, float* kept, const Part& part, const Slots& slots, int head, int size) {
  if (!OUT) return kept + kept_at(p, part.lo, part.part + 1, head, size);
  return part.part == part.parts - 1 && slots.write >= 0 ? p.state + slots.write * p.sss + head * p.ssh : nullptr;
}

// A part's rows through the recurrence, one after the other in fp32, where something was not finite: one of the rows, or the state that
// they start from. Which sums are infinite, of which sign, and which are NaN the chunks' products do not tell (an infinity's second
// part is NaN, and its products meet in another order). What is not finite here takes the place of what was stored, what is finite
// keeps its bits. 32 rows of the state at a time: whether an output is infinite or NaN is the sum of what they say, bits of +inf (or
// NaN) and of -inf (or NaN) for each row and lane, which lie in the tiles' place. s: the state after the rows from the chunks.
// All arguments are read and found again, as they would keep scalar registers through all that comes before (8192 tokens: 104 us in
// place of 107). Such a call of 8192 tokens takes 2 ms, one of 17 tokens 26 us.
template <typename T, int D, bool OUT>
__device__ inline void recurrence(const v16f (&s)[D / 32], uint64_t* signs) {
  struct Args {
    LinearParams p;
    float* kept;
  };
  typedef const __attribute__((address_space(4))) Args ConstantArgs;
  ConstantArgs* args = (ConstantArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const LinearParams p = *(const LinearParams*)&args->p;
  float* const kept = args->kept;
  int block = blockIdx.x, thread = threadIdx.x;
  asm volatile("" : "+s"(block), "+v"(thread));
  const int lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), half = lane >> 5, col = 32 * wave + (lane & 31);
  const int head = head_of(p, block % p.H);
  const Part part = find_part(p, block / p.H);
  const Slots slots = find_slots(p, part.seq);
  const float* const from = state_before<OUT>(p, kept, part, slots, head, D * D);
  float* const to = state_after<OUT>(p, kept, part, slots, head, D * D);
  const int rows = min(p.part, part.len - part.part * p.part);
  const int64_t base = part.lo + part.part * p.part;
  const uint16_t* const q = p.q + base * p.sqt + head * p.sqh;
  const uint16_t* const k = p.k + base * p.skt + head / p.G * p.skh;
  const uint16_t* const v = p.v + base * p.svt + head / p.G * p.svh + col;
  const Decay one = uniform(decay_of(p.log_decay[head], 1));
  signs += wave * 2 * p.part;
  for (int i = lane; OUT && i < 2 * rows; i += 64) signs[i] = 0;
  __threadfence_block();
  static_for<D / 32>([&](auto t) {
    v16f x;
    auto each = [&](auto f) {  // value r: row 32 t + 8 (r / 4) + 4 half + r % 4 of column col
#pragma unroll
      for (int r = 0; r < 16; ++r) f(r, (int64_t)(32 * t + 8 * (r / 4) + 4 * half + r % 4) * D + col);
    };
    each([&](int r, int64_t) { x[r] = 0.0f; });
    if (from) each([&](int r, int64_t at) { x[r] = from[at]; });
#pragma unroll 1
    for (int row = 0; row < rows; ++row) {
      const float value = T::to_f32(v[row * p.svt]);
      auto four = [&](const uint16_t* at, float (&f)[4]) {
        const v2u32 w = *reinterpret_cast<const v2u32*>(at);
        const v2f low = T::unpack(w.x), high = T::unpack(w.y);
        f[0] = low.x, f[1] = low.y, f[2] = high.x, f[3] = high.y;
      };
      float o = 0.0f;
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        float f[4];
        four(k + row * p.skt + 32 * t + 8 * a + 4 * half, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * a + e] = decayed(x[4 * a + e], one, f[e] * value);
        if constexpr (OUT) {
          four(q + row * p.sqt + 32 * t + 8 * a + 4 * half, f);
#pragma unroll
          for (int e = 0; e < 4; ++e) o = fmaf(f[e], x[4 * a + e], o);
        }
      }
      if constexpr (OUT) {
        const uint64_t plus = __ballot(!(o < __builtin_huge_valf())), minus = __ballot(!(o > kNegInf));
        if (lane == 0) signs[2 * row] |= plus, signs[2 * row + 1] |= minus;
      }
    }
    if (to) each([&](int r, int64_t at) { to[at] = __builtin_isfinite(x[r]) && __builtin_isfinite(s[t][r]) ? s[t][r] : x[r]; });
  });
  if constexpr (OUT) {
    __threadfence_block();  // the bits; and other lanes of the wave have stored these rows
#pragma unroll 1
    for (int row = 0; row < rows; ++row) {
      const uint64_t plus = signs[2 * row], minus = signs[2 * row + 1];
      const bool high = (plus | plus >> 32) >> (lane & 31) & 1, low = (minus | minus >> 32) >> (lane & 31) & 1;
      if (half == 0 && (high || low))
        store_f32_as(p.out, p.out_dtype, (base + row) * p.sot + head * p.soh + col, p.scale * (high && low ? __builtin_nanf("") : high ? __builtin_huge_valf() : kNegInf));
    }
  }
}

// A workgroup of D / 32 waves takes one head of a part. A wave keeps 32 columns of the state in the accumulators of 32 x 32 x 16
// MFMAs, where they are the operand of the next product as they lie. (Twice as many waves of 16 columns, four a SIMD: 80 us in place of 77
// for the outputs of 8192 rows, since each of them splits, weights and waits as often.)
// OUT: the rows' outputs from the state that the part starts from, and the sequence's end state (WIDE: outputs of 32 bits). Else: the state that a
// part leaves, for all parts but a sequence's last; the first starts from the sequence's state, the others from zeros.
template <typename T, int D, bool OUT, bool WIDE>
__global__ __launch_bounds__(2 * D, 2) void linear_chunk_kernel(LinearParams p, float* kept) {
  using S = Shared<T, D, OUT, WIDE>;
  static_assert(!OUT || sizeof(S) >= D / 32 * 2 * kMostRows * sizeof(uint64_t), "recurrence() keeps bits there");
  constexpr bool F16 = S::F16;
  constexpr int C = S::C, kRow = 2 * D, kParts = S::kParts;
  constexpr int DT = D / 32, IT = C / 32, CT = C / 16;  // blocks of the state's rows, of queries, of keys
  constexpr int kPieces = C / 16;                       // of a row tile, 16 bytes each, of a thread
  constexpr bool kLate = OUT;                           // the next rows are asked for when little but the state is held in registers
  constexpr bool kFull = WIDE && F16 && D == 256;       // no registers to keep the values in for the state
  __shared__ __attribute__((aligned(1024))) S sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int head = head_of(p, (int)(blockIdx.x % p.H));
  const float g = p.log_decay[head];
  const Part part = find_part(p, (int)(blockIdx.x / p.H));
  if (part.part >= part.parts - (OUT ? 0 : 1)) return;
  const int row0 = part.part * p.part, rows = min(p.part, part.len - row0);
  const int64_t base = part.lo + row0;
  const Decay full = uniform(decay_of(g, C)), last = uniform(decay_of(g, (rows - 1) % C + 1));
  char* const out = reinterpret_cast<char*>(p.out);
  const uint16_t* const qh = p.q + head * p.sqh;
  const uint16_t* const kh = p.k + head / p.G * p.skh;
  const uint16_t* const vh = p.v + head / p.G * p.svh;

  // Staging: this thread's 16-byte pieces are chunk `piece` of rows srow + 16 r.
  v4u32 gq[kPieces], gk[kPieces], gv[kPieces];
  auto fetch = [&](int t0) {  // rows past the end repeat the last one
    const int id = again((int)threadIdx.x), srow = id / (D / 8), piece = id % (D / 8);
    auto piece_of = [&](const uint16_t* head_rows, int64_t stride, int r) {
      const char* chunk = reinterpret_cast<const char*>(head_rows + (base + t0) * stride);
      return *reinterpret_cast<const v4u32*>(chunk + 2u * (__umul24(min(srow + 16 * r, rows - 1 - t0), (uint32_t)stride) + 8u * piece));
    };
#pragma unroll
    for (int r = 0; r < kPieces; ++r) {
      if (OUT) gq[r] = piece_of(qh, p.sqt, r);
      gk[r] = piece_of(kh, p.skt, r);
      gv[r] = piece_of(vh, p.svt, r);
    }
  };
  // For the scores, queries and keys lie with the dims of each 16 in the order 0-3, 8-11, 4-7, 12-15: the order in which a lane holds
  // the state's rows, 16 bytes of it for one half of the lanes.
  auto stage_row = [&](char* tile, int row, int piece, v4u32 w) {
    char* at = tile + row * kRow + 8 * (piece & 1);
    const int c = piece & ~1;
    *reinterpret_cast<v2u32*>(at + 16 * (c ^ key_swizzle<D>(row))) = v2u32{w.x, w.y};
    *reinterpret_cast<v2u32*>(at + 16 * ((c + 1) ^ key_swizzle<D>(row))) = v2u32{w.z, w.w};
  };
  auto stage = [&](int count) {
    const int id = again((int)threadIdx.x), srow = id / (D / 8), piece = id % (D / 8);
    if (count < C) {
#pragma unroll
      for (int r = 0; r < kPieces; ++r)
        if (srow + 16 * r >= count) gq[r] = gk[r] = gv[r] = v4u32{0, 0, 0, 0};
    }
#pragma unroll
    for (int r = 0; r < kPieces; ++r) {
      const int row = srow + 16 * r;
      const int wide = row * kRow + 16 * (piece ^ value_swizzle<D>(row));
      if constexpr (OUT) {
        stage_row(sh.q, row, piece, gq[r]);
        stage_row(sh.k, row, piece, gk[r]);
      }
      *reinterpret_cast<v4u32*>(sh.v + wide) = gv[r];
      if constexpr (F16) {
        float f[8];
        v4u32 two[2];
        if constexpr (OUT) {
          floats<T>(gq[r], f);
          split(f, two);
          stage_row(sh.qs[0], row, piece, two[0]);
          stage_row(sh.qs[1], row, piece, two[1]);
        }
        floats<T>(gk[r], f);
        split(f, two);
        *reinterpret_cast<v4u32*>(sh.kt[0] + wide) = two[0];
        *reinterpret_cast<v4u32*>(sh.kt[1] + wide) = two[1];
      } else {
        *reinterpret_cast<v4u32*>(sh.kt[0] + wide) = gk[r];
      }
    }
    if (count < C && (int)threadIdx.x < C) sh.left[threadIdx.x] = (int)threadIdx.x < count ? power(g, count - 1 - (int)threadIdx.x) : 0.0f;
  };

  // The state: rows 32 t + 8 (r / 4) + 4 half + r % 4 of column 32 wave + col.
  v16f s[DT];
  const int64_t corner = (int64_t)4 * half * D + 32 * wave + col;
  auto state_rows = [&](auto f) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) f(t, r, (int64_t)(32 * t + 8 * (r / 4) + r % 4) * D + corner);
  };
  if (rows > 0) fetch(0);
  const Slots slots = find_slots(p, part.seq);
  if (slots.bad) {
    if (OUT)
      for (int i = threadIdx.x; i < rows * D; i += 2 * D) store_f32_as(out, p.out_dtype, (base + i / D) * p.sot + head * p.soh + i % D, __builtin_nanf(""));
    return;
  }
  if (threadIdx.x == 0) sh.met = 0;
  if (rows == 0) __syncthreads();
  if ((int)threadIdx.x < C) {
    const float w = power(g, C - 1 - (int)threadIdx.x);
    sh.power[threadIdx.x] = w * p.scale, sh.left[threadIdx.x] = w;
  }
  const float* const from = state_before<OUT>(p, kept, part, slots, head, D * D);
  if (from)
    state_rows([&](int t, int r, int64_t at) { s[t][r] = from[at]; });
  else
    state_rows([&](int t, int r, int64_t) { s[t][r] = 0.0f; });
  if (!OUT && kept_apart(part, slots)) {
    float* to = kept + kept_at(p, part.lo, 0, head, D * D);
    state_rows([&](int t, int r, int64_t at) { to[at] = s[t][r]; });
  }

  // Transposed reads of a tile: block b of 32 columns, step c of 16 rows; the rows 16 c + 4 half + 0..3 and 8 further.
  auto transposed = [&](int now, const char* tile, int c, int b) {
    const int trow = 4 * (now >> 5) + (now & 15) / 4, tchunk = 2 * ((now >> 4) & 1) + (now & 3) / 2;
    const char* at = tile + (16 * c + trow) * kRow + 8 * (now & 1) + 16 * ((4 * b + tchunk) ^ value_swizzle<D>(trow));
    const v2u32 lo = read_transposed(at), hi = read_transposed(at + 8 * kRow);
    return v4u32{lo.x, lo.y, hi.x, hi.y};
  };
  float* const to = state_after<OUT>(p, kept, part, slots, head, D * D);
  float grow[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) grow[i] = OUT ? p.scale * power(g, 32 * i + col + 1) : 0.0f;
  bool met = false;  // sums that are not finite
  for (int t0 = 0; t0 < rows; t0 += C) {
    const int count = min(C, rows - t0);
    __syncthreads();  // the last chunk's tiles have been read
    stage(count);
    if (!kLate && t0 + C < rows) fetch(t0 + C);
    __syncthreads();
    const int now = again(lane);
    v16f o[IT];
    // Scores in blocks of 16 keys 16 jt + 4 (lane / 16) + r and 16 queries 16 it + lane % 16, those that some query sees and the
    // ones beside them that complete an operand: block b of 4 (or 12) of the waves in turn. Their products come first, what is made
    // of them after those with the state, which hide that they wait.
    constexpr int kBlocks = C == 64 ? 12 : 4, kEach = (kBlocks + DT - 1) / DT;  // kEach of a wave
    const bool scoring = OUT && (kBlocks % DT == 0 || wave < kBlocks);
    auto query_of = [](int b) { return 16 * (b < 4 ? b >> 1 : 2 + ((b - 4) >> 2)); };
    auto key_of = [](int b) { return 16 * (b < 4 ? b & 1 : (b - 4) & 3); };
    v4f sc[kEach];
    if (scoring) {
#pragma unroll
      for (int n = 0; n < kEach; ++n) {
        const int b = wave + n * DT, l16 = now & 15, l4 = now >> 4;
        sc[n] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < D / 32; ++u) {
          const int at = l16 * kRow + 16 * ((4 * u + l4) ^ key_swizzle<D>(l16));
          sc[n] = T::mfma16(*reinterpret_cast<const v4u32*>(sh.k + key_of(b) * kRow + at), *reinterpret_cast<const v4u32*>(sh.q + query_of(b) * kRow + at), sc[n]);
        }
      }
    }
    // q S, transposed: columns of the state as rows, queries as columns.
    auto from_state = [&] {
#pragma unroll
      for (int i = 0; i < IT; ++i) o[i] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < D / 16; ++u) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = s[u / 2][8 * (u % 2) + j];
        v4u32 part[kParts];
        split(f, part);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int row = 32 * i + (now & 31), at = row * kRow + 16 * ((2 * u + (now >> 5)) ^ key_swizzle<D>(row));
          if constexpr (F16) {
            const v4u32 qhi = *reinterpret_cast<const v4u32*>(sh.qs[0] + at), qlo = *reinterpret_cast<const v4u32*>(sh.qs[1] + at);
#pragma unroll
            for (int n = 0; n < kParts; ++n) o[i] = BF16::mfma32(part[n], qhi, o[i]);
#pragma unroll
            for (int n = 0; n < kParts - 1; ++n) o[i] = BF16::mfma32(part[n], qlo, o[i]);
          } else {
            const v4u32 q = *reinterpret_cast<const v4u32*>(sh.q + at);
#pragma unroll
            for (int n = 0; n < kParts; ++n) o[i] = BF16::mfma32(part[n], q, o[i]);
          }
        }
        if (D == 256 && u % 2) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= grow[i];
    };
    // Waves in products go before those that stage or wait: 75 to 72 us for 8192 rows, and 34 to 33 without outputs.
    __builtin_amdgcn_s_setprio(3);
    if constexpr (OUT) from_state();
    __builtin_amdgcn_s_setprio(0);
    if (scoring) {
#pragma unroll
      for (int n = 0; n < kEach; ++n) {
        const int b = wave + n * DT, l16 = now & 15, l4 = now >> 4, query = query_of(b) + l16, key = key_of(b) + 4 * l4;
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = sh.power[min(C - 1 - query + key + r, C - 1)];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = query >= key + r ? sc[n][r] * x[r] : 0.0f;  // a later key's score may be an infinity
        v2u32 part[kParts];
        split(x, part);
        const int at = (32 * (l4 & 1) + (query & 31)) * 16 + 8 * (l4 >> 1), operand = (b < 4 ? 0 : 2) + key_of(b) / 16;
#pragma unroll
        for (int n = 0; n < kParts; ++n) *reinterpret_cast<v2u32*>(sh.scores[operand][n] + at) = part[n];
      }
    }
    v4u32 v[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) v[c] = transposed(now, sh.v, c, wave);
    if constexpr (OUT) {
      __syncthreads();  // the scores
      auto add_rows = [&](const v4u32 (&vs)[CT]) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          v4u32 two[2] = {vs[c], vs[c]};
          if constexpr (F16) {
            float f[8];
            floats<T>(vs[c], f);
            split(f, two);
          }
#pragma unroll
          for (int i = c / 2; i < IT; ++i) {
            v4u32 part[kParts];
#pragma unroll
            for (int n = 0; n < kParts; ++n) part[n] = *reinterpret_cast<const v4u32*>(sh.scores[(i ? 2 : 0) + c][n] + 16 * lane);
#pragma unroll
            for (int n = 0; n < kParts; ++n) o[i] = BF16::mfma32(two[0], part[n], o[i]);
#pragma unroll
            for (int n = 0; F16 && n < kParts - 1; ++n) o[i] = BF16::mfma32(two[1], part[n], o[i]);
          }
        }
      };
      add_rows(v);
      // 0 times an infinity or NaN of a later row is NaN. Where sums end up not finite, the rows are added again without such values:
      // right for the rows before theirs. Those from theirs on are put right at the end.
      float odd = 0.0f;
#pragma unroll
      for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd = fmaf(o[i][r], 0.0f, odd);
      if (__builtin_expect(__any(odd != 0.0f), 0)) {
#pragma unroll
        for (int t = 0; t < DT; ++t) asm volatile("" : "+v"(s[t]));  // computed again, not kept from above
        from_state();
        v4u32 fine[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) fine[c][j] = only_finite<T>(v[c][j]);
        add_rows(fine);
        met = true;
      }
      // Row 32 i + col, dims 32 wave + 8 a + 4 half + 0..3 for a = 0..3: with 16-bit outputs the halves exchange what the other stores.
      const int there = again(lane);
      char* const chunk = out + (p.out_dtype == VXA_F32 ? 4 : 2) * ((base + t0) * p.sot + head * p.soh + 32 * wave);
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int row = 32 * i + (there & 31);
        const uint32_t at = __umul24(row, (uint32_t)p.sot);
        if (p.out_wide) {
#pragma unroll
          for (int a = 0; a < 4; a += 2) {
            uint32_t w[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              w[0][j] = T::pack(o[i][4 * a + 2 * j], o[i][4 * a + 2 * j + 1]), w[1][j] = T::pack(o[i][4 * a + 4 + 2 * j], o[i][4 * a + 5 + 2 * j]);
              const auto x = __builtin_amdgcn_permlane32_swap(w[0][j], w[1][j], false, false);
              w[0][j] = x[0], w[1][j] = x[1];
            }
            if (row < count) *reinterpret_cast<v4u32*>(chunk + 2u * (at + 8 * a + 8 * (there >> 5))) = v4u32{w[0][0], w[0][1], w[1][0], w[1][1]};
          }
        } else if (row < count) {
#pragma unroll
          for (int r = 0; r < 16; ++r) store_f32_as(chunk, p.out_dtype, at + 8 * (r / 4) + 4 * (there >> 5) + r % 4, o[i][r]);
        }
      }
    }
    if (OUT && t0 + C >= rows && !to) break;  // nobody takes the state behind these rows (3 prompts of 2111, fp16, 256 dims, parts of 512: 142 to 139 us)
    if (kLate && t0 + C < rows) fetch(t0 + C);
    __builtin_amdgcn_s_setprio(3);
    // The state. Values are weighted and split into three parts, which keep the 24 bits of the products; the keys are exact.
    const Decay decay = t0 + C < rows ? full : last;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float less = s[t][r] * -decay.rest;
        asm("" : "+v"(less));  // as in decayed(): with 256 dims there would not be registers enough
        s[t][r] = fmaf(s[t][r], decay.whole, -less);
      }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float f[8];
      floats<T>(kFull ? transposed(now, sh.v, c, wave) : v[c], f);
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const v4f w = *reinterpret_cast<const v4f*>(sh.left + 16 * c + 4 * (now >> 5) + 2 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[j + e] *= w[e];
      }
      v4u32 three[3];
      split(f, three);
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const v4u32 k = transposed(now, sh.kt[0], c, t);
#pragma unroll
        for (int n = 0; n < 3; ++n) s[t] = BF16::mfma32(k, three[n], s[t]);
        if constexpr (F16) {
          const v4u32 low = transposed(now, sh.kt[1], c, t);
          s[t] = BF16::mfma32(low, three[0], s[t]);
          s[t] = BF16::mfma32(low, three[1], s[t]);
        }
        if (D == 256 && t % 2) __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  }
  float odd = 0.0f, odd2 = 0.0f;
  if (to) state_rows([&](int t, int r, int64_t) { (r % 2 ? odd2 : odd) = fmaf(s[t][r], 0.0f, r % 2 ? odd2 : odd); });
  if (met || odd != 0.0f || odd2 != 0.0f) sh.met = 1;
  __syncthreads();
  if (__builtin_expect(sh.met == 0, 1)) {
    if (to) state_rows([&](int t, int r, int64_t at) { to[at] = s[t][r]; });
    return;
  }
  recurrence<T, D, OUT>(s, reinterpret_cast<uint64_t*>(&sh));
}

// The states before a long sequence's third part and later, from what each part adds: 4 values of one head a thread.
__global__ __launch_bounds__(256) void linear_parts_kernel(LinearParams p, float* kept, int size) {
  const int pieces = size / 1024, head = (int)(blockIdx.x / pieces) % p.H, seq = (int)(blockIdx.x / pieces) / p.H;
  const int lo = min(max(p.cu[seq], 0), p.total), len = min(max(p.cu[seq + 1], lo), p.total) - lo;
  const int parts = (len + p.part - 1) / p.part;
  if (parts < 3) return;
  v4f* x = reinterpret_cast<v4f*>(kept + kept_at(p, lo, 1, head, size)) + (int)(blockIdx.x % pieces) * 256 + (int)threadIdx.x;
  const int64_t step = (int64_t)p.H * size / 4;
  const Decay decay = decay_of(p.log_decay[head], p.part);
  const float one = power(p.log_decay[head], 1);  // an infinity is one still where exp(g rows) is 0 and exp(g) is not
  v4f s = *x;
#pragma unroll 4
  for (int i = 2; i < parts; ++i) {
    const v4f add = x[(i - 1) * step];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = __builtin_isfinite(s[e]) ? fmaf(s[e], decay.whole, fmaf(s[e], decay.rest, add[e])) : fmaf(s[e], one, add[e]);
    x[(i - 1) * step] = s;
  }
}

int64_t kept_states(int64_t tokens, int64_t heads, int64_t dims) {
  const int64_t part = part_rows(heads, dims);
  return tokens > part ? 2 * (tokens / part) + 2 : 0;
}

template <typename T, int D>
hipError_t launch_prompt(const LinearParams& p, float* kept, hipStream_t st) {
  const int64_t blocks = (int64_t)p.H * (p.total / p.part + p.n);
  const int64_t pieces = (int64_t)p.n * p.H * (D * D / 1024);
  if (!launchable(blocks, 2 * D) || !launchable(pieces, 256)) return hipErrorInvalidConfiguration;
  if (p.total > p.part) {  // some sequence may have several parts
    hipLaunchKernelGGL((linear_chunk_kernel<T, D, false, false>), dim3((unsigned)blocks), dim3(2 * D), 0, st, p, kept);
    if (p.total > 2 * p.part) hipLaunchKernelGGL(linear_parts_kernel, dim3((unsigned)pieces), dim3(256), 0, st, p, kept, D * D);
  }
  if (p.out_dtype == VXA_F32)
    hipLaunchKernelGGL((linear_chunk_kernel<T, D, true, true>), dim3((unsigned)blocks), dim3(2 * D), 0, st, p, kept);
  else
    hipLaunchKernelGGL((linear_chunk_kernel<T, D, true, false>), dim3((unsigned)blocks), dim3(2 * D), 0, st, p, kept);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_prompt(int64_t D, const LinearParams& p, float* kept, hipStream_t st) {
  if (D == 64) return launch_prompt<T, 64>(p, kept, st);
  if (D == 128) return launch_prompt<T, 128>(p, kept, st);
  return launch_prompt<T, 256>(p, kept, st);
}

// What both entry points check, and their parameters.
int linear_params(LinearParams& p, const void* q, int64_t sqt, int64_t sqh, const void* k, int64_t skt, int64_t skh, const void* v,
                  int64_t svt, int64_t svh, int dtype, int64_t n, int64_t tokens, const float* log_decay, float scale, void* out,
                  int out_dtype, int64_t sot, int64_t soh, float* state, int64_t slots, int64_t sss, int64_t ssh,
                  const int32_t* read_slots, const int32_t* write_slots, int64_t H, int64_t KV, int64_t D) {
  if (n < 0 || tokens < 0 || H <= 0 || KV <= 0 || D <= 0 || slots < 0 || H % KV != 0) return VXA_ERR_ARG;
  if (dtype != VXA_BF16 && dtype != VXA_F16) return VXA_ERR_ARG;
  if (out_dtype != VXA_F32 && out_dtype != VXA_BF16 && out_dtype != VXA_F16) return VXA_ERR_ARG;
  if ((read_slots || write_slots) && !state) return VXA_ERR_ARG;
  if (D != 64 && D != 128 && D != 256) return VXA_ERR_UNSUPPORTED;
  if (H > (1 << 16) || tokens > (1 << 30) || n > (1 << 30) || slots > (1 << 30)) return VXA_ERR_UNSUPPORTED;
  if (n == 0) return VXA_OK;
  if (!log_decay || (tokens && (!q || !k || !v || !out))) return VXA_ERR_ARG;
  if (std::max({sqt, skt, svt, sot}) >= 1 << 23 || std::min({sqt, skt, svt, sot}) < 0) return VXA_ERR_UNSUPPORTED;  // 64 rows' bytes are a 32-bit number
  // Rows are read in 16-byte pieces.
  if ((uintptr_t)q % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || sqt % 8 || sqh % 8 || skt % 8 || skh % 8 || svt % 8 || svh % 8 ||
      (uintptr_t)state % 16 || sss % 4 || ssh % 4)
    return VXA_ERR_UNSUPPORTED;
  p.q = reinterpret_cast<const uint16_t*>(q), p.sqt = sqt, p.sqh = sqh;
  p.k = reinterpret_cast<const uint16_t*>(k), p.skt = skt, p.skh = skh;
  p.v = reinterpret_cast<const uint16_t*>(v), p.svt = svt, p.svh = svh;
  p.cu = nullptr, p.part = part_rows(H, D);
  p.n = (int32_t)n, p.total = (int32_t)tokens, p.H = (int32_t)H, p.G = (int32_t)(H / KV);
  p.log_decay = log_decay, p.scale = scale;
  p.out = out, p.sot = sot, p.soh = soh, p.out_dtype = out_dtype;
  p.out_wide = out_dtype == dtype && (uintptr_t)out % 16 == 0 && sot % 8 == 0 && soh % 8 == 0;
  p.state = state, p.sss = sss, p.ssh = ssh, p.slots = (int32_t)slots, p.read = read_slots, p.write = write_slots;
  return VXA_OK;
}

int status_of(hipError_t err) {
  if (err == hipErrorInvalidConfiguration) return VXA_ERR_UNSUPPORTED;
  return err == hipSuccess ? VXA_OK : VXA_ERR_LAUNCH;
}

}  // namespace

extern "C" int vxa_linear_prompt_workspace(int64_t tokens, int64_t num_heads, int64_t head_dim, size_t* ws_bytes) {
  if (tokens < 0 || num_heads <= 0 || head_dim <= 0 || !ws_bytes) return VXA_ERR_ARG;
  *ws_bytes = (size_t)product({kept_states(tokens, num_heads, head_dim), num_heads, head_dim, head_dim, 4});
  return VXA_OK;
}

extern "C" int vxa_linear_prompt(const void* q, int64_t sqt, int64_t sqh, const void* k, int64_t skt, int64_t skh, const void* v,
                                 int64_t svt, int64_t svh, int dtype, const int32_t* starts, int64_t n, int64_t tokens,
                                 const float* log_decay, float scale, void* out, int out_dtype, int64_t sot, int64_t soh, float* state,
                                 int64_t slots, int64_t sss, int64_t ssh, const int32_t* read_slots, const int32_t* write_slots,
                                 int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, void* ws, size_t ws_bytes,
                                 vxa_stream_t stream) {
  LinearParams p;
  const int rc = linear_params(p, q, sqt, sqh, k, skt, skh, v, svt, svh, dtype, n, tokens, log_decay, scale, out, out_dtype, sot, soh,
                               state, slots, sss, ssh, read_slots, write_slots, num_heads, num_kv_heads, head_dim);
  if (rc != VXA_OK || n == 0) return rc;
  if (!starts) return VXA_ERR_ARG;
  size_t bytes = 0;
  vxa_linear_prompt_workspace(tokens, num_heads, head_dim, &bytes);
  if (bytes && (!ws || (uintptr_t)ws % 16 || ws_bytes < bytes)) return VXA_ERR_WORKSPACE;
  p.cu = starts;
  float* kept = reinterpret_cast<float*>(ws);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return status_of(dtype == VXA_BF16 ? launch_prompt<BF16>(head_dim, p, kept, st) : launch_prompt<FP16>(head_dim, p, kept, st));
}

extern "C" int vxa_linear_step(const void* q, int64_t sqt, int64_t sqh, const void* k, int64_t skt, int64_t skh, const void* v,
                               int64_t svt, int64_t svh, int dtype, int64_t n, const float* log_decay, float scale, void* out,
                               int out_dtype, int64_t sot, int64_t soh, float* state, int64_t slots, int64_t sss, int64_t ssh,
                               const int32_t* read_slots, const int32_t* write_slots, int64_t num_heads, int64_t num_kv_heads,
                               int64_t head_dim, vxa_stream_t stream) {
  LinearParams p;
  const int rc = linear_params(p, q, sqt, sqh, k, skt, skh, v, svt, svh, dtype, n, n, log_decay, scale, out, out_dtype, sot, soh, state,
                               slots, sss, ssh, read_slots, write_slots, num_heads, num_kv_heads, head_dim);
  if (rc != VXA_OK || n == 0) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return status_of(dtype == VXA_BF16 ? launch_step<BF16>(head_dim, p, st) : launch_step<FP16>(head_dim, p, st));
}
