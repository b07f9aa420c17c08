// Attention of drafted tokens over a paged cache (gfx950), with a fixed reduction order.
//
// A request has T >= 1 drafted tokens (the nodes of a tree), whose keys and values are the last T of its L
// cached ones. Node i attends to every key of the context (the first L - T) and to the drafted key j where bit
// j of its mask is set; without masks, to the drafted keys up to its own (a chain; T = 1 is plain decoding):
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i.k_j - max_j scale q_i.k_j).
// A row that attends to nothing is 0. The cache holds 16-bit elements of the query's type, or 8 bits with one
// scale per token and head for K and for V: q.k = kscale (q . k8), p v = (p vscale) v8, so the 8-bit values
// enter the matrix instructions as they are.
//
// Work split. The T * G rows of a (request, KV head) share its keys, so they are the columns of one matrix
// product: S^T = K Q^T with 16 x 16 x 32 MFMAs (keys are the rows), then O^T = V^T P^T. A lane holds one
// column of S^T and of O^T, so the softmax and its rescaling stay in the lane, and the order of the keys in the
// second product is chosen so that the lane's own scores are its operand: P is never exchanged between lanes.
// V is loaded by rows, each lane 8 keys of the same D / 16 dims, and transposed in registers, one byte permute
// for every two elements. K and V go from HBM to registers; LDS holds the places and scales of a segment's keys and the
// sums that are folded. Requests of more than wide_rows(D) rows take a kernel that shares tiles of K and V through LDS (below).
//
// Order. Keys are cut into segments of kSeg and groups of kGroup segments. Strand w of a segment, its 32-key tiles w,
// w + 4, ..., is summed with one running maximum; the segments of a strand are folded in order, the four strands of a
// group joined, the groups folded in order. It depends on a request's own length and number of rows, and the running maxima
// on a row's own scores: a row's bits do not change with the batch, nor with the queries of the request's other nodes. A
// workgroup's waves take the four strands of a group, one each, and need each other only at its end; where that
// leaves too few workgroups, a workgroup takes one strand and its waves one segment each: the same sums.
//
// Rounding. Scores, maxima, sums and accumulators are fp32. P is split into two 16-bit parts, hi + lo, with one
// MFMA each: P keeps 16 bits (in fp16 22, or what counts to 2^-32 of the row's largest weight), as the 16-bit output is rounded
// once from an fp32 sum; the 8-bit cache always takes bf16 parts there, because P vscale can leave the fp16 range.
//
// What bounds it (32 heads on 8, 128 dims). 64 requests of 8192 keys with one token, 16-bit cache: 330 us, 6.5 TB/s, the rate
// at which pages are read. With 8 tokens and the 8-bit cache: 262 us, 4.3 TB/s of half the bytes, two thirds of that rate
// (4096 to 8192 keys: 197 us, the same). There a tile of 32 keys costs a wave some 430 vector instructions, 192 of them to
// make 16-bit operands of its bytes, and 48 MFMAs; 245 registers leave two waves a SIMD. The vector instructions alone are
// half of the cycles, and the waves wait for 36 % of theirs. One request of 16384 keys and one token: 14.5 us, a chain of dependent loads and four tiles (10) and a
// second launch for the merge (4).

#include <algorithm>

#include "attention_common.h"

namespace {

constexpr int kSeg = 512;    // keys of a segment
constexpr int kGroup = 4;    // segments that are folded one after the other
constexpr int kTile = 32;    // keys of a wave's step
constexpr int kWaves = 4;
constexpr int kWaveKeys = kSeg / kWaves;
constexpr int kMaxNodes = 64;
// Requests with more rows (nodes times heads of a group) take the wide kernel. 128 dims: 96 and 64 are alike from 97 rows on,
// 80 rows of 16 requests took 50 us in the narrow kernel and 61 in the wide one. 256 dims, where the narrow kernel has one
// wave a SIMD for 32 rows: 107 requests of 72 to 144 rows 152 us wide from 33 rows on, 198 from 97 on; 8 of 24 rows
// 70 us narrow, 105 wide.
constexpr int wide_rows(int d) { return d == 256 ? 32 : 96; }
constexpr int kWaves256 = 8;    // of its workgroups at 256 dims
constexpr int kFill = 256;      // keys whose places the wide kernel looks up at a time
constexpr int kManyWorkgroups = 256;  // of whole groups: one a CU
constexpr int kSearched = 256;  // requests

struct TreeParams {
  const uint16_t* q;
  int64_t sqt, sqh;
  const char* kc;
  int64_t skb, skp, skh;  // strides of the caches in bytes, of the scales in elements
  const char* vc;
  int64_t svb, svp, svh;
  const float* ks;
  int64_t sksb, sksp, sksh;
  const float* vs;
  int64_t svsb, svsp, svsh;
  const int32_t* bt;
  int64_t sbt;
  int32_t cols, page;     // block-table entries of a request, tokens of a page
  Divisor by_page;
  int64_t blocks;
  const int32_t* sl;
  const int32_t* qsl;
  const int64_t* mask;
  float scale_log2;
  int32_t n, total, KV, G, ns, row_blocks, max_nodes, max_len, wide_rows;
  bool by_size;  // workgroups of whole groups go by their work, the largest first
  bool strands;  // a workgroup for each strand of a group of segments, not for each group
  int64_t parts;  // partial sums that a row has place for
  bool out_wide;  // the output has the query's type and its rows start on 8 bytes
  float* mp;  // [total][H][parts]
  float* lp;
  float* ap;  // [total][H][parts][D]
  void* out;
  int64_t sot, soh;
  int32_t out_dtype;
};

__device__ inline int page_of(const TreeParams& p, int key) { return divide(key, p.by_page); }

// The request's keys, nodes and first query row; `bad` where they do not fit the call (a length below its
// nodes, more nodes or keys than the call's bounds): its rows become NaN.
struct Request {
  int32_t L, T, q0;
  bool bad;
};
__device__ inline Request request_of(const TreeParams& p, int b) {
  Request r;
  r.L = p.sl[b];
  r.q0 = max(p.qsl[b], 0);
  r.T = min(p.qsl[b + 1], p.total) - r.q0;
  r.bad = r.T > p.max_nodes || r.L < r.T || r.L > p.max_len || (int64_t)r.L > (int64_t)p.cols * p.page;
  return r;
}

// Two 8-bit values (byte e of a and of b) as bf16 elements, exact.
template <int E>
__device__ inline uint32_t bytes_as_bf16(uint32_t a, uint32_t b) {
  const float fa = (float)(int8_t)(a >> (8 * E)), fb = (float)(int8_t)(b >> (8 * E));
  return __builtin_amdgcn_perm(__float_as_uint(fb), __float_as_uint(fa), 0x07060302u);
}
// Four 8-bit values as two dwords of bf16 or fp16 elements, exact. fp16: the byte plus 128 in the low bits of
// 1024, less 1152.
template <typename T>
__device__ inline void bytes_as(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (std::is_same_v<T, BF16>) {
    const float f0 = (float)(int8_t)w, f1 = (float)(int8_t)(w >> 8), f2 = (float)(int8_t)(w >> 16), f3 = (float)(int8_t)(w >> 24);
    lo = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u);
    hi = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u);
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const v2h bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias);
  }
}

template <int W>
struct Words {
  uint32_t w[W];
};
template <int W>
__device__ inline Words<W> load_words(const char* p) {
  Words<W> r;
  if constexpr (W == 1) {
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  } else if constexpr (W == 2) {
    const v2u32 u = __builtin_nontemporal_load(reinterpret_cast<const v2u32*>(p));
    r.w[0] = u.x, r.w[1] = u.y;
  } else {
#pragma unroll
    for (int c = 0; c < W / 4; ++c) {
      const v4u32 u = __builtin_nontemporal_load(reinterpret_cast<const v4u32*>(p) + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[4 * c + i] = u[i];
    }
  }
  return r;
}

// What the wave's lanes have written to LDS is there for all of them: a wave's LDS operations end in order.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The state (ma, la, sums a) of some segments followed by (mb, lb, sums b): a = a x + b y for every sum.
template <typename F>
__device__ inline void fold(float& ma, float& la, float mb, float lb, F&& sums) {
  const float mn = fmaxf(ma, mb);
  const float x = exp2_hw(ma - mn), y = exp2_hw(mb - mn);
  la = fmaf(la, x, lb * y);
  ma = mn;
  sums(x, y);
}

// Maximum, sum and four dims' weighted values of a row over some keys; add: over those of b, which come after.
struct State {
  float m, l;
  v4f a;
  __device__ inline void add(const State& b) {
    fold(m, l, b.m, b.l, [&](float x, float y) {
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = fmaf(a[e], x, b.a[e] * y);
    });
  }
};
// The first `count` strands of a group, into s[0].
__device__ inline void join(State (&s)[kWaves], int count) {
  float m = s[0].m, l = 0.0f;
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
    if (w < count) m = fmaxf(m, s[w].m);
  v4f a = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w >= count) break;
    const float x = exp2_hw(s[w].m - m);
    l = fmaf(s[w].l, x, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = fmaf(s[w].a[e], x, a[e]);
  }
  s[0] = State{m, l, a};
}

// What row (node, head) attends to is nothing: its sum is 0 by definition, not by underflow.
__device__ inline bool attends_to_nothing(const TreeParams& p, const Request& rq, int node) {
  if (rq.L > rq.T || p.mask == nullptr) return false;
  const uint64_t all = rq.T >= 64 ? ~0ull : (1ull << rq.T) - 1;
  return ((uint64_t)p.mask[rq.q0 + node] & all) == 0;
}

// Gives whether there are sums that are not finite, though the scores are.
template <typename T>
__device__ inline bool store_row(const TreeParams& p, const Request& rq, int node, int head, int dim, v4f a, float l) {
  const float inv = 1.0f / l;
  const bool nothing = l == 0.0f && attends_to_nothing(p, rq, node);
  float odd = 0.0f;  // 0 where all four are finite, else NaN
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    odd = fmaf(a[e], 0.0f, odd);
    a[e] = nothing ? 0.0f : a[e] * inv;
  }
  const int64_t to = (int64_t)(rq.q0 + node) * p.sot + (int64_t)head * p.soh + dim;
  if (p.out_wide) {
    *reinterpret_cast<v2u32*>(reinterpret_cast<uint16_t*>(p.out) + to) = v2u32{T::pack(a[0], a[1]), T::pack(a[2], a[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) store_f32_as(p.out, p.out_dtype, to + e, a[e]);
  }
  return odd != 0.0f && l > 0.0f;  // l is NaN where a score is +inf or NaN, or a page is missing
}
// The arguments, read again: for code at the end or seldom reached, which would keep registers through all that comes before.
__device__ inline TreeParams arguments_again() {
  typedef const __attribute__((address_space(4))) TreeParams Args;
  Args* args = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  return *(const TreeParams*)args;
}
// For those: values that are infinities or NaN, of keys that the row attends to, take the place of what was stored.
template <typename T, bool INT8>
__device__ inline void find_specials(const TreeParams& p, const Request& rq, int b, int node, int head, int dim) {
  const int g = head / p.G, ctx = rq.L - rq.T;
  const uint64_t seen = p.mask != nullptr ? (uint64_t)p.mask[rq.q0 + node] : (2ull << node) - 1;
  v4f special = {0, 0, 0, 0};
  constexpr int kAhead = 8;  // keys on their way together
#pragma unroll 1
  for (int first = 0, page = 0; first < rq.L; first += p.page, ++page) {
    const int64_t block = p.bt[(int64_t)b * p.sbt + page];
    if (block < 0 || block >= p.blocks) continue;
    const char* values = p.vc + block * p.svb + (int64_t)g * p.svh + (INT8 ? 1 : 2) * dim;
    const float* scales = INT8 ? p.vs + block * p.svsb + (int64_t)g * p.svsh : nullptr;
    const int count = min(p.page, rq.L - first);
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += kAhead) {
      v2u32 w[kAhead];  // 16-bit values, or a scale
      bool any = false;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int at = min(i0 + i, count - 1);
        if constexpr (INT8)
          w[i] = v2u32{__float_as_uint(scales[at * p.svsp]), 0};
        else
          w[i] = *reinterpret_cast<const v2u32*>(values + at * p.svp);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        any |= INT8 ? !__builtin_isfinite(__uint_as_float(w[i].x)) : (only_special<T>(w[i].x) | only_special<T>(w[i].y)) != 0;
      if (!any) continue;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int draft = first + i0 + i - ctx;
        if (i0 + i >= count || (draft >= 0 && !((seen >> draft) & 1))) continue;
        if constexpr (INT8) {
          const uint32_t q = *reinterpret_cast<const uint32_t*>(values + (i0 + i) * p.svp);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = (float)(int8_t)(q >> (8 * e)) * __uint_as_float(w[i].x);
            if (!__builtin_isfinite(f)) special[e] += f;
          }
        } else {
          add_specials<T>(special, w[i]);
        }
      }
    }
  }
  store_specials(p.out, p.out_dtype, (int64_t)(rq.q0 + node) * p.sot + (int64_t)head * p.soh + dim, special);
}

// The row block of a workgroup, and what it shares with the other row blocks in `id`. Workgroups go to the 8 XCDs in turn:
// the row blocks of the same keys are 8 apart, next to each other on one XCD and its L2.
__device__ inline int row_block_of(const TreeParams& p, uint32_t& id) {
  const uint32_t y = blockIdx.x / 8, rb = y % (uint32_t)p.row_blocks;
  id = y / (uint32_t)p.row_blocks * 8 + blockIdx.x % 8;
  return (int)rb;
}

// Unit `unit` of the requests' groups, those of four segments first, then those of three, two and one. A request that does
// not fit the call is one small unit: its rows become NaN.
struct GroupOf {
  int request, group;  // request < 0: no such unit
};
__device__ inline GroupOf find_group(const TreeParams& p, int unit) {
  const int lane = threadIdx.x & 63;
  for (int left = kGroup; left > 0; --left) {
    for (int j0 = 0; j0 < p.n; j0 += 64) {
      int count = 0, rest = 0;
      if (j0 + lane < p.n) {
        const Request rq = request_of(p, j0 + lane);
        const int segs = (rq.L + kSeg - 1) / kSeg;
        rest = rq.bad ? 0 : segs / kGroup;
        if (rq.T > 0 && rq.bad)
          count = left == 1;
        else if (rq.T > 0 && rq.T * p.G <= p.wide_rows)
          count = left == kGroup ? segs / kGroup : segs % kGroup == left;
      }
      const int sum = wave_scan(count, [](int a, int b) { return a + b; });
      const int total = __builtin_amdgcn_readlane(sum, 63);
      if (unit < total) {
        const int at = __builtin_ctzll(__ballot(sum > unit));
        // A whole group is counted from its request's first; a part comes after them; a misfit has group 0.
        const int before = __builtin_amdgcn_readlane(sum - count, at);
        return GroupOf{j0 + at, left == kGroup ? unit - before : __builtin_amdgcn_readlane(rest, at)};
      }
      unit -= total;
    }
  }
  return GroupOf{-1, 0};
}

// Registers of a lane that live through a tile: sums and queries, and one tile's keys and values. Two workgroups share a
// CU where those leave room; the next tile is loaded ahead where its registers do not cost that.
constexpr int lane_regs(int d, int nq, bool int8, int tiles) { return 3 * d * nq / 8 + tiles * d / (int8 ? 4 : 2); }
constexpr bool shares_cu(int d, int nq, bool int8) { return lane_regs(d, nq, int8, 1) <= 180; }
constexpr bool loads_ahead(int d, int nq, bool int8) {
  return lane_regs(d, nq, int8, 2) <= (shares_cu(d, nq, int8) ? 180 : 300);
}

// T: the query's element type; INT8: the cache's; NQ: 16-row blocks of a workgroup.
template <typename T, bool INT8, int D, int NQ>
__global__ __launch_bounds__(64 * kWaves, shares_cu(D, NQ, INT8) ? 2 : 1) void tree_partial_kernel(TreeParams p) {
  using PT = std::conditional_t<INT8, BF16, T>;  // the type of P and V
  constexpr bool AHEAD = loads_ahead(D, NQ, INT8);
  constexpr int QS = D / 32;                     // MFMA steps over the head's dims
  constexpr int DPL = D / 16;                    // dims of a lane in V, and 16-dim blocks of O^T
  constexpr int KW = INT8 ? D / 16 : D / 8;      // dwords of a lane's share of a key
  constexpr int VW = INT8 ? DPL / 4 : DPL / 2;   // dwords of a lane's dims of one key's value
  __shared__ int64_t s_koff[kWaves][kWaveKeys], s_voff[kWaves][kWaveKeys];
  __shared__ __attribute__((aligned(16))) float s_ks[kWaves][INT8 ? kWaveKeys : 4], s_vs[kWaves][INT8 ? kWaveKeys : 4];
  __shared__ float s_m[kWaves][16 * NQ], s_l[kWaves][16 * NQ];
  __shared__ v4f s_acc[kWaves][16 * NQ][D / 4];  // [wave][row][4 dims ^ row]

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15;
  const int grp = lane >> 4;

  uint32_t id;
  const int rb = row_block_of(p, id);
  const int g = (int)(id % (uint32_t)p.KV);
  id /= (uint32_t)p.KV;
  int b, group, strand = 0;
  if (p.by_size) {
    const GroupOf at = find_group(p, (int)id);
    if (at.request < 0) return;
    b = __builtin_amdgcn_readfirstlane(at.request), group = __builtin_amdgcn_readfirstlane(at.group);
  } else {
    b = (int)(id % (uint32_t)p.n);
    id /= (uint32_t)p.n;
    group = p.strands ? (int)id / kWaves : (int)id, strand = (int)id % kWaves;  // past the groups: nothing to do
  }

  // The pages of the wave's own keys of a segment, tile after tile. They are asked for before the request's length is
  // known: past it, table entries are read and not used.
  constexpr int kOwn = kWaveKeys / 64;
  auto key_of = [&](int seg, int first, int i) { return seg * kSeg + ((64 * i + lane) / kTile * kWaves + first) * kTile + lane % kTile; };
  auto find = [&](int seg, int first, int32_t (&pages)[kOwn]) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      pages[i] = p.cols == 0 ? -1 : p.bt[(int64_t)b * p.sbt + min(page_of(p, key_of(seg, first, i)), p.cols - 1)];
  };
  // This wave's segments of the group and its tiles of them: strand `wave` of all four, or a strand of segment `wave`.
  // The first tile of a short request may be its strand 0 all the same: that choice waits for its length.
  int32_t pages[kOwn];
  find(group * kGroup + (p.strands ? wave : 0), p.strands ? strand : wave, pages);
  const Request rq = request_of(p, b);
#pragma unroll
  for (int i = 0; i < kOwn; ++i) asm volatile("" : "+v"(pages[i]));
  const int rows = rq.T * p.G;
  const int row0 = rb * 16 * NQ;
  if (row0 >= rows || (rows > p.wide_rows && !rq.bad)) return;
  const int H = p.KV * p.G;
  if (rq.bad) {
    if (group == 0 && rb == 0 && (!p.strands || strand == 0))
      for (int64_t i = threadIdx.x; i < (int64_t)rows * D; i += 64 * kWaves) {
        const int row = (int)(i / D);
        store_f32_as(p.out, p.out_dtype,
                     (int64_t)(rq.q0 + row / p.G) * p.sot + (int64_t)(g * p.G + row % p.G) * p.soh + i % D, __builtin_nanf(""));
      }
    return;
  }
  const int segs = (rq.L + kSeg - 1) / kSeg;
  const bool alone = segs <= kGroup;             // one group: its workgroup takes all strands and writes the output
  const bool whole = alone || !p.strands;
  if (group * kGroup >= segs || (alone && p.strands && strand != 0)) return;
  const int first = whole ? wave : strand;       // the wave's first tile of a segment
  const int seg0 = group * kGroup + (whole ? 0 : wave);
  const int seg_end = min(group * kGroup + kGroup, whole ? segs : min(seg0 + 1, segs));
  if (alone && p.strands) find(seg0, first, pages);
  const int ctx = rq.L - rq.T;
  const float reach = PT::reach(rq.L);

  // Row offsets and scales of the wave's own keys. Keys past the last one repeat the wave's first, masked. A page that the
  // cache does not have makes the request's rows NaN.
  bool bad_page = false;
  float scales[kOwn][2];
  struct Strides {
    int64_t kb, kp, vb, vp, ksb, ksp, ksh, vsb, vsp, vsh;
  };
  auto place = [&](int seg, const int32_t (&pages)[kOwn]) {
    Strides a;
    if constexpr (NQ == 2 && D < 256) {
      // Read again from the arguments: kept through the tiles of 32 rows, they cost more registers than there are.
      typedef const __attribute__((address_space(4))) TreeParams Args;
      Args* args = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
      asm volatile("" : "+s"(args));
      a = Strides{args->skb, args->skp, args->svb, args->svp, args->sksb, args->sksp, args->sksh, args->svsb, args->svsp, args->svsh};
    } else {
      a = Strides{p.skb, p.skp, p.svb, p.svp, p.sksb, p.sksp, p.sksh, p.svsb, p.svsp, p.svsh};
    }
    const int key0 = seg * kSeg + first * kTile;
    const int32_t page0 = __builtin_amdgcn_readfirstlane(pages[0]);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      int key = key_of(seg, first, i);
      int64_t block = key < rq.L ? pages[i] : page0;
      if (key >= rq.L) key = key0;
      const int off = key - page_of(p, key) * p.page;
      if (block < 0 || block >= p.blocks) {
        bad_page |= key0 < rq.L;
        block = 0;
      }
      s_koff[wave][64 * i + lane] = block * a.kb + (int64_t)off * a.kp;
      s_voff[wave][64 * i + lane] = block * a.vb + (int64_t)off * a.vp;
      if constexpr (INT8) {
        scales[i][0] = p.ks[block * a.ksb + (int64_t)off * a.ksp + (int64_t)g * a.ksh];
        scales[i][1] = p.vs[block * a.vsb + (int64_t)off * a.vsp + (int64_t)g * a.vsh];
      }
    }
    wave_sync();
  };

  // This lane's rows: their masks over the drafted keys, and q as the second operand.
  v4u32 qf[NQ][QS];
  uint64_t seen[NQ];
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    const int row = min(row0 + 16 * t + col, rows - 1);
    const int node = row / p.G;
    const uint16_t* q = p.q + (int64_t)(rq.q0 + node) * p.sqt + (int64_t)(g * p.G + row - node * p.G) * p.sqh;
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      const int dim = INT8 ? 64 * (i / 2) + 16 * grp + 8 * (i % 2) : 32 * i + 8 * grp;
      qf[t][i] = *reinterpret_cast<const v4u32*>(q + dim);
    }
    const uint64_t all = rq.T >= 64 ? ~0ull : (1ull << rq.T) - 1;
    seen[t] = all & (p.mask != nullptr ? (uint64_t)p.mask[rq.q0 + node] : (2ull << node) - 1);
  }
  const char* kbase = p.kc + (int64_t)g * p.skh + 16 * grp;
  const char* vbase = p.vc + (int64_t)g * p.svh + VW * 4 * col;
  struct Loads {
    Words<KW> k[2];
    Words<VW> v[8];
  };
  auto load = [&](int j, Loads& r) {  // the wave's tile j; key slots of a lane: 4 grp + i of each half tile
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* k = kbase + s_koff[wave][j * kTile + 16 * h + col];
#pragma unroll
      for (int c = 0; c < KW / 4; ++c) {
        const Words<4> w = load_words<4>(k + 64 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.k[h].w[4 * c + i] = w.w[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) r.v[4 * h + i] = load_words<VW>(vbase + s_voff[wave][j * kTile + 16 * h + 4 * grp + i]);
    }
  };

  float m[NQ], l[NQ];
  v4f acc[NQ][DPL];
  auto clear = [&] {
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      m[t] = kLowest;
      l[t] = 0.0f;
#pragma unroll
      for (int e = 0; e < DPL; ++e) acc[t][e] = v4f{0, 0, 0, 0};
    }
  };

  // DRAFTED: the tile holds drafted keys, or ends past the last key. CAREFUL: values of keys that some rows do not attend
  // to may be infinities or NaN, and 0 times those is NaN; here they enter the product as 0 and are added to the rows that
  // attend to them. (8-bit values are finite.)
  auto compute = [&](int start, int tile, const Loads& r, auto drafted_c, auto careful_c) {
    constexpr bool drafted = decltype(drafted_c)::value, CAREFUL = decltype(careful_c)::value;
    const Words<KW>(&kr)[2] = r.k;
    const Words<VW>(&vr)[8] = r.v;
    const int own = tile / kWaves * kTile;  // the tile's first key among the wave's
    v4f s[NQ][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < NQ; ++t) s[t][h] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < QS; ++i) {
        v4u32 a;
        if constexpr (INT8) {
          uint32_t x0, x1, x2, x3;
          bytes_as<T>(kr[h].w[2 * i], x0, x1);
          bytes_as<T>(kr[h].w[2 * i + 1], x2, x3);
          a = v4u32{x0, x1, x2, x3};
        } else {
          a = v4u32{kr[h].w[4 * i], kr[h].w[4 * i + 1], kr[h].w[4 * i + 2], kr[h].w[4 * i + 3]};
        }
#pragma unroll
        for (int t = 0; t < NQ; ++t) s[t][h] = T::mfma16(a, qf[t][i], s[t][h]);
      }
    }

    const int key0 = start + tile * kTile;
    uint32_t phi[NQ][4], plo[NQ][4], flag[NQ][4];
    const v4f one = {p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2};
    v4f ks[2] = {one, one}, vs[2];
    if constexpr (INT8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[h] = *reinterpret_cast<const v4f*>(&s_ks[wave][own + 16 * h + 4 * grp]);
        vs[h] = *reinterpret_cast<const v4f*>(&s_vs[wave][own + 16 * h + 4 * grp]);
      }
    }
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      uint32_t live = 0xFF;  // bit 4 h + j: this row attends to the key
      if constexpr (drafted) {
        live = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = key0 + 16 * h + 4 * grp - ctx;  // the first of the lane's four keys among the drafted ones
          const uint64_t on = d >= 0 ? seen[t] >> min(d, 63) : seen[t] << min(-d, 63) | ((1ull << min(-d, 63)) - 1);
          live |= d >= 64 ? 0u : ((uint32_t)on & 15u) << (4 * h);
        }
      }
      float top = kLowest;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = s[t][h][j] * ks[h][j];
          s[t][h][j] = drafted && !((live >> (4 * h + j)) & 1) ? kNegInf : x;
          top = fmaxf(top, s[t][h][j]);
        }
      top = rows_max(top);
      if (__any(top > m[t] + reach)) {
        const float mn = top > m[t] + reach ? (top - reach) + kSlack : m[t];
        const float c = exp2_hw(m[t] - mn);
        l[t] *= c;
#pragma unroll
        for (int e = 0; e < DPL; ++e) acc[t][e] = acc[t][e] * c;
        m[t] = mn;
      }
      float pv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = exp2_hw(s[t][i / 4][i % 4] - m[t]);
        l[t] += x;
        pv[i] = x;
        if constexpr (INT8) {
          pv[i] = x * vs[i / 4][i % 4];
          if (drafted && !((live >> i) & 1)) pv[i] = 0.0f;  // a masked key's scale may be NaN
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        phi[t][i] = PT::pack(pv[2 * i], pv[2 * i + 1]);
        const v2f back = PT::unpack(phi[t][i]);
        plo[t][i] = PT::pack(pv[2 * i] - back[0], pv[2 * i + 1] - back[1]);
        if constexpr (CAREFUL)
          flag[t][i] = ((live >> (2 * i)) & 1 ? (uint32_t)PT::kOne : 0u) | ((live >> (2 * i + 1)) & 1 ? (uint32_t)PT::kOne << 16 : 0u);
      }
    }

    static_for<DPL>([&](auto ec) {
      constexpr int e = decltype(ec)::value;
      v4u32 a;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (INT8)
          a[i] = bytes_as_bf16<e % 4>(vr[2 * i].w[e / 4], vr[2 * i + 1].w[e / 4]);
        else
          a[i] = __builtin_amdgcn_perm(vr[2 * i + 1].w[e / 2], vr[2 * i].w[e / 2], e % 2 ? 0x07060302u : 0x05040100u);
      }
      if constexpr (CAREFUL) {
        v4u32 plus, minus;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          plus[i] = special_flags<PT, 0>(a[i]);
          minus[i] = special_flags<PT, 1>(a[i]);
          a[i] = only_finite<PT>(a[i]);
        }
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          const v4u32 f = {flag[t][0], flag[t][1], flag[t][2], flag[t][3]};
          const v4f up = PT::mfma16(plus, f, v4f{0, 0, 0, 0}), down = PT::mfma16(minus, f, v4f{0, 0, 0, 0});
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (up[r] > 0.0f) acc[t][e][r] += __builtin_huge_valf();
            if (down[r] > 0.0f) acc[t][e][r] += kNegInf;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        acc[t][e] = PT::mfma16(a, v4u32{phi[t][0], phi[t][1], phi[t][2], phi[t][3]}, acc[t][e]);
        acc[t][e] = PT::mfma16(a, v4u32{plo[t][0], plo[t][1], plo[t][2], plo[t][3]}, acc[t][e]);
      }
    });
  };
  // The wave's sums over its segments lie in LDS, folded as a segment ends; every lane reads what it wrote itself.
  float jm[NQ], jl[NQ];
  auto at_acc = [&](int t, int r, int e) -> v4f& { return s_acc[wave][16 * t + col][(((4 * grp + r) * DPL + e) / 4) ^ col]; };

  Loads cur, next;
  if (seg0 < seg_end) {
    place(seg0, pages);
    if constexpr (AHEAD) load(0, cur);
  }
  for (int seg = seg0; seg < seg_end; ++seg) {
    if constexpr (INT8) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        s_ks[wave][64 * i + lane] = scales[i][0] * p.scale_log2;
        s_vs[wave][64 * i + lane] = scales[i][1];
      }
      wave_sync();
    }
    const bool more = seg + 1 < seg_end;
    if (more) find(seg + 1, first, pages);
    // The next tile's loads are in flight while a tile is computed. Segments with drafted keys take the step that looks
    // at the masks for all their tiles: one loop's instructions to fetch.
    const int start = seg * kSeg, end = min(start + kSeg, rq.L);
    const int tiles = (end - start + kTile - 1) / kTile;
    const int plain = end > ctx ? 0 : tiles;
    clear();
    int tile = first;
    if constexpr (AHEAD && NQ == 1) {
      // Two tiles a turn, so that no registers are moved (15.5 us -> 14.6 for one row over 16384 keys; with 32 rows the
      // second copy of the step costs more registers than there are: 216 us -> 233).
      static_assert(kWaveKeys / kTile % 2 == 0);  // a segment of the context alone is whole: an even number of tiles
#pragma unroll 1
      for (; tile < plain; tile += 2 * kWaves) {
        load(tile / kWaves + 1, next);
        compute(start, tile, cur, std::false_type{}, std::false_type{});
        if (tile + 2 * kWaves < plain) load(tile / kWaves + 2, cur);
        compute(start, tile + kWaves, next, std::false_type{}, std::false_type{});
      }
    } else {
#pragma unroll 1
      for (; tile < plain; tile += kWaves) {
        if constexpr (AHEAD) {
          if (tile + kWaves < tiles) load(tile / kWaves + 1, next);
        } else {
          load(tile / kWaves, cur);
        }
        compute(start, tile, cur, std::false_type{}, std::false_type{});
        if constexpr (AHEAD) cur = next;
      }
    }
#pragma unroll 1
    for (; tile < tiles; tile += kWaves) {
      if constexpr (AHEAD) {
        if (tile + kWaves < tiles) load(tile / kWaves + 1, next);
      } else {
        load(tile / kWaves, cur);
      }
      compute(start, tile, cur, std::true_type{}, std::false_type{});
      if constexpr (AHEAD) cur = next;
    }
    if constexpr (!INT8) {
      float odd = 0.0f;  // 0 where all sums are finite, else NaN
#pragma unroll
      for (int t = 0; t < NQ; ++t)
#pragma unroll
        for (int e = 0; e < DPL; ++e)
#pragma unroll
          for (int r = 0; r < 4; ++r) odd = fmaf(acc[t][e][r], 0.0f, odd);
      if (plain == 0 && __any(odd != 0.0f)) {
        clear();
#pragma unroll 1
        for (tile = first; tile < tiles; tile += kWaves) {
          load(tile / kWaves, cur);
          compute(start, tile, cur, std::true_type{}, std::true_type{});
        }
      }
    }
    if (more) {
      place(seg + 1, pages);
      if constexpr (AHEAD) load(0, cur);
    }
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      const float sum = rows_sum(l[t]);
      if (seg == seg0) {
        jm[t] = m[t], jl[t] = sum;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < DPL; e += 4) at_acc(t, r, e) = v4f{acc[t][e][r], acc[t][e + 1][r], acc[t][e + 2][r], acc[t][e + 3][r]};
      } else {
        fold(jm[t], jl[t], m[t], sum, [&](float x, float y) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < DPL; e += 4) {
              v4f a = at_acc(t, r, e);
#pragma unroll
              for (int i = 0; i < 4; ++i) a[i] = fmaf(a[i], x, acc[t][e + i][r] * y);
              at_acc(t, r, e) = a;
            }
        });
      }
    }
  }
  if (grp == 0 && seg0 < seg_end) {
#pragma unroll
    for (int t = 0; t < NQ; ++t) s_m[wave][16 * t + col] = jm[t], s_l[wave][16 * t + col] = jl[t];
  }
  const bool bad = __syncthreads_or(bad_page);

  // The workgroup's waves: strands of a group are joined, segments of a strand folded in order.
  const int waves = whole ? kWaves : min(kWaves, segs - group * kGroup);
#pragma unroll 1
  for (int at = threadIdx.x; at < 16 * NQ * (D / 4); at += 64 * kWaves) {
    const int in_block = at / (D / 4), c = at % (D / 4);
    const int row = row0 + in_block;
    if (row >= rows) break;
    State s[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (w < waves) s[w] = State{s_m[w][in_block], s_l[w][in_block], s_acc[w][in_block][c ^ (in_block & 15)]};
    if (whole) {
      join(s, kWaves);
    } else {
#pragma unroll
      for (int w = 1; w < kWaves; ++w)
        if (w < waves) s[0].add(s[w]);
    }
    if (bad) s[0].l = __builtin_nanf("");
    const int node = row / p.G, head = g * p.G + row % p.G;
    if (alone) {
      const bool spoiled = store_row<T>(p, rq, node, head, 4 * c, s[0].a, s[0].l);
      if (__builtin_expect(spoiled, 0)) find_specials<T, INT8>(arguments_again(), rq, b, node, head, 4 * c);
    } else {
      const int64_t part = ((int64_t)(rq.q0 + node) * H + head) * p.parts + (whole ? group : group * kWaves + strand);
      if (c == 0) p.mp[part] = s[0].m, p.lp[part] = s[0].l;
      reinterpret_cast<v4f*>(p.ap)[part * (D / 4) + c] = s[0].a;
    }
  }
}

// Keys of a workgroup of the wide kernel, by the request's own length: more of them halve the partial sums.
__device__ __host__ inline int wide_chunk(int keys) { return keys <= 4096 ? kSeg : 2 * kSeg; }

// Requests of more than wide_rows(D) rows. A workgroup takes 128 rows of a (request, KV head), 32 a wave, and a chunk of
// keys in tiles that its waves share through LDS, as 16-bit elements: a key is converted once for 128 rows. 32 x 32 x 16
// MFMAs, otherwise as above: S^T = K Q^T, then O^T = V^T P^T with V transposed by the LDS read. Tiles of a 16-bit cache are
// copied straight into LDS, those of an 8-bit one through registers, the next tile while one is computed.
template <typename T, bool INT8, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void tree_decode_kernel_wide(TreeParams p) {
  using PT = std::conditional_t<INT8, BF16, T>;
  constexpr int kKeys = 64, KU = kKeys / 32;
  constexpr int QS = D / 16, DB = D / 32;
  constexpr int kRow = 2 * D, kTileBytes = kKeys * kRow;
  constexpr int kPer = 1024 / kRow, kRound = kPer * kWaves, kCopies = kKeys / kRound;  // as copied: keys of a copy, of a round
  constexpr int KL = kKeys * D / 16 / (64 * kWaves);                                   // as converted: 16-byte pieces a thread
  __shared__ __attribute__((aligned(1024))) char s_kv[2][2][kTileBytes];
  __shared__ int64_t s_koff[kFill], s_voff[kFill];
  __shared__ __attribute__((aligned(16))) float s_ks[2][INT8 ? kFill : 4], s_vs[2][INT8 ? kFill : 4];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  uint32_t id;
  const int rb = row_block_of(p, id);
  const int g = (int)(id % (uint32_t)p.KV);
  id /= (uint32_t)p.KV;
  const int b = (int)(id % (uint32_t)p.n);
  const int chunk = (int)(id / (uint32_t)p.n);
  const Request rq = request_of(p, b);
  const int rows = rq.T * p.G, row0 = rb * 32 * kWaves;
  if (rq.bad || rows <= p.wide_rows || row0 >= rows) return;
  const int keys = wide_chunk(rq.L);
  const int start = chunk * keys, end = min(start + keys, rq.L);
  if (start >= end) return;
  const int ctx = rq.L - rq.T;
  const float reach = PT::reach(rq.L);
  const int H = p.KV * p.G;

  // Places of kFill keys; those past the last one repeat it.
  bool bad_page = false;
  auto page_at = [&](int fill) {
    const int key = min(start + fill * kFill + (int)threadIdx.x, end - 1);
    return p.bt[(int64_t)b * p.sbt + page_of(p, key)];
  };
  auto place = [&](int fill, int32_t page) {
    const int key = min(start + fill * kFill + (int)threadIdx.x, end - 1);
    const int off = key - page_of(p, key) * p.page;
    int64_t block = page;
    if (block < 0 || block >= p.blocks) {
      bad_page = true;
      block = 0;
    }
    s_koff[threadIdx.x] = block * p.skb + (int64_t)off * p.skp;
    s_voff[threadIdx.x] = block * p.svb + (int64_t)off * p.svp;
    if constexpr (INT8) {
      s_ks[fill & 1][threadIdx.x] = p.ks[block * p.sksb + (int64_t)off * p.sksp + (int64_t)g * p.sksh] * p.scale_log2;
      s_vs[fill & 1][threadIdx.x] = p.vs[block * p.svsb + (int64_t)off * p.svsp + (int64_t)g * p.svsh];
    }
    __syncthreads();
  };
  int32_t page = page_at(0);

  const int row = min(row0 + 32 * wave + col, rows - 1), node = row / p.G, head = g * p.G + row - node * p.G;
  v4u32 qf[QS];
  {
    const uint16_t* q = p.q + (int64_t)(rq.q0 + node) * p.sqt + (int64_t)head * p.sqh + 8 * half;
#pragma unroll
    for (int i = 0; i < QS; ++i) qf[i] = *reinterpret_cast<const v4u32*>(q + 16 * i);
  }
  const uint64_t all = rq.T >= 64 ? ~0ull : (1ull << rq.T) - 1;
  const uint64_t seen = all & (p.mask != nullptr ? (uint64_t)p.mask[rq.q0 + node] : (2ull << node) - 1);

  const int tiles = (end - start + kKeys - 1) / kKeys;
  const int plain = min(max(ctx - start, 0) / kKeys, tiles);  // tiles of the context alone
  const char* kh = p.kc + (int64_t)g * p.skh;
  const char* vh = p.vc + (int64_t)g * p.svh;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t*)&s_kv[0][0][0]) + wave * 1024;
  v4u32 kr[INT8 ? KL : 1], vr[INT8 ? KL : 1];
  auto load = [&](int t) {
    const int at = t * kKeys % kFill;
    if constexpr (INT8) {
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const int u = threadIdx.x + i * 64 * kWaves, key = u / (D / 16), c = u % (D / 16);
        kr[i] = *reinterpret_cast<const v4u32*>(kh + s_koff[at + key] + 16 * c);
        vr[i] = *reinterpret_cast<const v4u32*>(vh + s_voff[at + key] + 16 * c);
      }
    } else {
      const uint32_t dst = lds0 + (t & 1) * 2 * kTileBytes;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int key = i * kRound + wave * kPer + lane / (kRow / 16), c = lane % (kRow / 16);
        copy_to_lds(kh + s_koff[at + key] + 16 * (c ^ key_swizzle<D>(key)), dst + i * kWaves * 1024);
        copy_to_lds(vh + s_voff[at + key] + 16 * (c ^ value_swizzle<D>(key)), dst + kTileBytes + i * kWaves * 1024);
      }
    }
  };
  auto store = [&](int t) {
    if constexpr (INT8) {
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const int u = threadIdx.x + i * 64 * kWaves, key = u / (D / 16), c = u % (D / 16);
        char* kd = s_kv[t & 1][0] + key * kRow;
        char* vd = s_kv[t & 1][1] + key * kRow;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t x[4], y[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            bytes_as<T>(kr[i][2 * j + e], x[2 * e], x[2 * e + 1]);
            bytes_as<PT>(vr[i][2 * j + e], y[2 * e], y[2 * e + 1]);
          }
          *reinterpret_cast<v4u32*>(kd + 16 * ((2 * c + j) ^ key_swizzle<D>(key))) = v4u32{x[0], x[1], x[2], x[3]};
          *reinterpret_cast<v4u32*>(vd + 16 * ((2 * c + j) ^ value_swizzle<D>(key))) = v4u32{y[0], y[1], y[2], y[3]};
        }
      }
    }
  };

  const int vkey = 4 * half + (lane & 15) / 4;
  const int vdim = 2 * ((lane >> 4) & 1) + (lane & 3) / 2;  // chunk in a 32-dim block
  const int vbyte = vkey * kRow + 8 * (lane & 1);
  float m, l[4];
  v16f acc[DB];
  auto step = [&](int t, auto drafted_c, auto careful_c) {
    constexpr bool DRAFTED = decltype(drafted_c)::value, CAREFUL = decltype(careful_c)::value;
    // Tile t is there for every wave, and every wave has read tile t - 1: its buffer takes tile t + 1.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < tiles) {
      if ((t + 1) * kKeys % kFill == 0) {
        place((t + 1) * kKeys / kFill, page);
        if ((t + 1) * kKeys + kFill < keys) page = page_at((t + 1) * kKeys / kFill + 1);
      }
      load(t + 1);
    }
    const int key0 = start + t * kKeys, at = t * kKeys % kFill, fill = t * kKeys / kFill & 1;
    const char* kt = s_kv[t & 1][0] + col * kRow;
    const char* vt = s_kv[t & 1][1] + vbyte;
    v16f s[KU];
#pragma unroll
    for (int u = 0; u < KU; ++u) s[u] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < QS; ++i)
#pragma unroll
      for (int u = 0; u < KU; ++u)
        s[u] = T::mfma32(*reinterpret_cast<const v4u32*>(kt + 32 * u * kRow + 16 * ((2 * i + half) ^ key_swizzle<D>(col))), qf[i], s[u]);
    uint32_t live[KU][4];  // bit j of [u][i]: this row attends to key 32 u + 8 i + 4 half + j of the tile
    float top = kLowest;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DRAFTED) {
          const int d = key0 + 32 * u + 8 * i + 4 * half - ctx;
          const uint64_t on = d >= 0 ? seen >> min(d, 63) : seen << min(-d, 63) | ((1ull << min(-d, 63)) - 1);
          live[u][i] = d >= 64 ? 0u : (uint32_t)on & 15u;
        }
        v4f ks = {p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2};
        if constexpr (INT8) ks = *reinterpret_cast<const v4f*>(&s_ks[fill][at + 32 * u + 8 * i + 4 * half]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = s[u][4 * i + j] * ks[j];
          if (DRAFTED && !((live[u][i] >> j) & 1)) x = kNegInf;
          s[u][4 * i + j] = x;
          top = fmaxf(top, x);
        }
      }
    float ta = top, tb = top;
    swap32(ta, tb);
    top = fmaxf(ta, tb);
    if (__any(top > m + reach)) {
      const float mn = top > m + reach ? (top - reach) + kSlack : m;
      const float c = exp2_hw(m - mn);
#pragma unroll
      for (int i = 0; i < 4; ++i) l[i] *= c;
#pragma unroll
      for (int i = 0; i < DB; ++i) acc[i] = acc[i] * c;
      m = mn;
    }
    v4u32 phi[2 * KU], plo[2 * KU];
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float pv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pv[j] = exp2_hw(s[u][4 * i + j] - m);
          l[j] += pv[j];
        }
        if constexpr (INT8) {
          const v4f vs = *reinterpret_cast<const v4f*>(&s_vs[fill][at + 32 * u + 8 * i + 4 * half]);
#pragma unroll
          for (int j = 0; j < 4; ++j) pv[j] = DRAFTED && !((live[u][i] >> j) & 1) ? 0.0f : pv[j] * vs[j];  // a masked key's scale may be NaN
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t hi = PT::pack(pv[2 * j], pv[2 * j + 1]);
          const v2f back = PT::unpack(hi);
          phi[2 * u + i / 2][2 * (i % 2) + j] = hi;
          plo[2 * u + i / 2][2 * (i % 2) + j] = PT::pack(pv[2 * j] - back[0], pv[2 * j + 1] - back[1]);
        }
      }
    if constexpr (INT8) __builtin_amdgcn_sched_barrier(0);  // no registers for values read ahead of the weights
#pragma unroll
    for (int c = 0; c < 2 * KU; ++c)
#pragma unroll
      for (int i = 0; i < DB; i += 2) {  // two sums in turn: neither waits for the other
        v4u32 a[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const char* from = vt + 16 * c * kRow + 16 * ((4 * (i + k) + vdim) ^ value_swizzle<D>(vkey));
          const v2u32 lo = read_transposed(from), hi = read_transposed(from + 8 * kRow);
          a[k] = v4u32{lo.x, lo.y, hi.x, hi.y};
          if constexpr (CAREFUL) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a[k][j] = only_finite<PT>(a[k][j]);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i + k % 2] = PT::mfma32(a[k % 2], k < 2 ? phi[c] : plo[c], acc[i + k % 2]);
      }
    if (t + 1 < tiles) store(t + 1);
  };
  auto begin = [&] {
    place(0, page);
    if (kFill < keys) page = page_at(1);
    m = kLowest;
#pragma unroll
    for (int i = 0; i < 4; ++i) l[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    load(0);
    store(0);
  };
  begin();
  int t = 0;
#pragma unroll 1
  for (; t < plain; ++t) step(t, std::false_type{}, std::false_type{});
#pragma unroll 1
  for (; t < tiles; ++t) step(t, std::true_type{}, std::false_type{});
  // As in the narrow kernel: values of masked keys that are infinities or NaN have spoiled the sums; the tiles with
  // drafted keys are computed without such values, which are added at the end to the rows that attend to them.
  bool careful = false;
  if constexpr (!INT8) {
    if (plain < tiles) {
      float odd = 0.0f;  // 0 where all sums are finite, else NaN
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd = fmaf(acc[i][r], 0.0f, odd);
      careful = __syncthreads_or(odd != 0.0f);
      if (careful) {
        page = page_at(0);
        begin();
#pragma unroll 1
        for (t = 0; t < plain; ++t) step(t, std::false_type{}, std::false_type{});
#pragma unroll 1
        for (; t < tiles; ++t) step(t, std::true_type{}, std::true_type{});
      }
    }
  }
  const bool bad = __syncthreads_or(bad_page);
  float la = (l[0] + l[1]) + (l[2] + l[3]), lb = la;
  swap32(la, lb);
  const float sum = bad ? __builtin_nanf("") : la + lb;
  const TreeParams q = arguments_again();
  int own = col;  // the row's node and head are found again, too
  asm volatile("" : "+v"(own));
  own += row0 + 32 * wave;
  if (own >= rows) return;
  const int out_node = own / q.G, out_head = g * q.G + own - out_node * q.G;
  const bool alone = rq.L <= keys;
  bool spoiled = false;
  const int64_t part = ((int64_t)(rq.q0 + out_node) * H + out_head) * q.parts + chunk;
  if (!alone && half == 0) q.mp[part] = m, q.lp[part] = sum;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int dim = 32 * i + 2 * r + 4 * half;
      v4f o = {acc[i][r], acc[i][r + 1], acc[i][r + 2], acc[i][r + 3]};
      if (careful) {
#pragma unroll 1
        for (int key = start + plain * kKeys; key < end; ++key) {
          const int32_t block = p.bt[(int64_t)b * p.sbt + page_of(p, key)];
          const bool on = (key < ctx || (seen >> (key - ctx)) & 1) && block >= 0 && block < p.blocks;
          if (!on) continue;
          const v2u32 w = *reinterpret_cast<const v2u32*>(vh + block * p.svb + (int64_t)(key - page_of(p, key) * p.page) * p.svp + 2 * dim);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float f = T::to_f32((uint16_t)(w[j / 2] >> (16 * (j % 2))));
            if (!__builtin_isfinite(f)) o[j] += f;
          }
        }
      }
      if (alone)
        spoiled |= store_row<T>(q, rq, out_node, out_head, dim, o, sum);
      else
        *reinterpret_cast<v4f*>(q.ap + part * D + dim) = o;
    }
  if (__builtin_expect(spoiled, 0))
#pragma unroll 1
    for (int dim = 4 * half; dim < D; dim += 8) find_specials<T, INT8>(q, rq, b, out_node, out_head, dim);
}

// The same for 256 dims, with 8 waves of 16 rows and 16 x 16 x 32 MFMAs: two waves a SIMD, where 32 rows leave one. Six
// trees of 61 nodes, 488 rows: 45 us where that took 52. (8-bit keys of 128 dims: 199 us this way, 133 with 32 rows.)
template <typename T, bool INT8>
__global__ __launch_bounds__(64 * kWaves256, 2) void tree_decode_kernel_wide_256(TreeParams p) {
  constexpr int D = 256, kThreads = 64 * kWaves256;
  using PT = std::conditional_t<INT8, BF16, T>;
  constexpr int kKeys = 32, KT = kKeys / 16;  // keys of a tile, in blocks of 16
  constexpr int QS = D / 32, DB = D / 16;
  constexpr int kRow = 2 * D, kTileBytes = kKeys * kRow;
  constexpr int kPer = 1024 / kRow, kRound = kPer * kWaves256, kCopies = kKeys / kRound;  // as copied: keys of a copy, of a round
  static_assert(kKeys * D / 16 == kThreads && kFill <= kThreads);  // as converted: a 16-byte piece a thread
  __shared__ __attribute__((aligned(1024))) char s_kv[2][2][kTileBytes];
  __shared__ int64_t s_koff[kFill], s_voff[kFill];
  __shared__ __attribute__((aligned(16))) float s_ks[2][INT8 ? kFill : 4], s_vs[2][INT8 ? kFill : 4];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  uint32_t id;
  const int rb = row_block_of(p, id);
  const int g = (int)(id % (uint32_t)p.KV);
  id /= (uint32_t)p.KV;
  const int b = (int)(id % (uint32_t)p.n);
  const int chunk = (int)(id / (uint32_t)p.n);
  const Request rq = request_of(p, b);
  const int rows = rq.T * p.G, row0 = rb * 16 * kWaves256;
  if (rq.bad || rows <= p.wide_rows || row0 >= rows) return;
  const int keys = wide_chunk(rq.L);
  const int start = chunk * keys, end = min(start + keys, rq.L);
  if (start >= end) return;
  const int ctx = rq.L - rq.T;
  const float reach = PT::reach(rq.L);
  const int H = p.KV * p.G;

  // Places of kFill keys; those past the last one repeat it.
  bool bad_page = false;
  auto page_at = [&](int fill) {
    const int key = min(start + fill * kFill + (int)threadIdx.x % kFill, end - 1);
    return p.bt[(int64_t)b * p.sbt + page_of(p, key)];
  };
  auto place = [&](int fill, int32_t page) {
    const int key = min(start + fill * kFill + (int)threadIdx.x % kFill, end - 1);
    const int off = key - page_of(p, key) * p.page;
    int64_t block = page;
    if (block < 0 || block >= p.blocks) {
      bad_page = true;
      block = 0;
    }
    if (threadIdx.x < kFill) {
      s_koff[threadIdx.x] = block * p.skb + (int64_t)off * p.skp;
      s_voff[threadIdx.x] = block * p.svb + (int64_t)off * p.svp;
      if constexpr (INT8) {
        s_ks[fill & 1][threadIdx.x] = p.ks[block * p.sksb + (int64_t)off * p.sksp + (int64_t)g * p.sksh] * p.scale_log2;
        s_vs[fill & 1][threadIdx.x] = p.vs[block * p.svsb + (int64_t)off * p.svsp + (int64_t)g * p.svsh];
      }
    }
    __syncthreads();
  };
  int32_t page = page_at(0);

  const int row = min(row0 + 16 * wave + col, rows - 1), node = row / p.G, head = g * p.G + row - node * p.G;
  v4u32 qf[QS];
  {
    const uint16_t* q = p.q + (int64_t)(rq.q0 + node) * p.sqt + (int64_t)head * p.sqh + 8 * grp;
#pragma unroll
    for (int i = 0; i < QS; ++i) qf[i] = *reinterpret_cast<const v4u32*>(q + 32 * i);
  }
  const uint64_t all = rq.T >= 64 ? ~0ull : (1ull << rq.T) - 1;
  const uint64_t seen = all & (p.mask != nullptr ? (uint64_t)p.mask[rq.q0 + node] : (2ull << node) - 1);

  const int tiles = (end - start + kKeys - 1) / kKeys;
  const int plain = min(max(ctx - start, 0) / kKeys, tiles);  // tiles of the context alone
  const char* kh = p.kc + (int64_t)g * p.skh;
  const char* vh = p.vc + (int64_t)g * p.svh;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t*)&s_kv[0][0][0]) + wave * 1024;
  v4u32 kr, vr;
  const int piece_key = threadIdx.x / (D / 16), piece = threadIdx.x % (D / 16);
  // 16 lanes read two chunks of four keys of V, 64 lanes of 16: eight keys meet the 256 bytes of the banks.
  auto swv = [](int key) { return 2 * (key & 7); };
  auto load = [&](int t) {
    const int at = t * kKeys % kFill;
    if constexpr (INT8) {
      kr = *reinterpret_cast<const v4u32*>(kh + s_koff[at + piece_key] + 16 * piece);
      vr = *reinterpret_cast<const v4u32*>(vh + s_voff[at + piece_key] + 16 * piece);
    } else {
      const uint32_t dst = lds0 + (t & 1) * 2 * kTileBytes;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int key = i * kRound + wave * kPer + lane / (kRow / 16), c = lane % (kRow / 16);
        copy_to_lds(kh + s_koff[at + key] + 16 * (c ^ key_swizzle<D>(key)), dst + i * kThreads * 16);
        copy_to_lds(vh + s_voff[at + key] + 16 * (c ^ swv(key)), dst + kTileBytes + i * kThreads * 16);
      }
    }
  };
  auto store = [&](int t) {
    if constexpr (INT8) {
      char* kd = s_kv[t & 1][0] + piece_key * kRow;
      char* vd = s_kv[t & 1][1] + piece_key * kRow;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t x[4], y[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          bytes_as<T>(kr[2 * j + e], x[2 * e], x[2 * e + 1]);
          bytes_as<PT>(vr[2 * j + e], y[2 * e], y[2 * e + 1]);
        }
        *reinterpret_cast<v4u32*>(kd + 16 * ((2 * piece + j) ^ key_swizzle<D>(piece_key))) = v4u32{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<v4u32*>(vd + 16 * ((2 * piece + j) ^ swv(piece_key))) = v4u32{y[0], y[1], y[2], y[3]};
      }
    }
  };

  const int vkey = 4 * grp + col / 4;
  const int vbyte = vkey * kRow + 8 * (lane & 1);
  float m, l;
  v4f acc[DB];
  auto step = [&](int t, auto drafted_c, auto careful_c) {
    constexpr bool DRAFTED = decltype(drafted_c)::value, CAREFUL = decltype(careful_c)::value;
    // Tile t is there for every wave, and every wave has read tile t - 1: its buffer takes tile t + 1.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < tiles) {
      if ((t + 1) * kKeys % kFill == 0) {
        place((t + 1) * kKeys / kFill, page);
        if ((t + 1) * kKeys + kFill < keys) page = page_at((t + 1) * kKeys / kFill + 1);
      }
      load(t + 1);
    }
    const int key0 = start + t * kKeys, at = t * kKeys % kFill, fill = t * kKeys / kFill & 1;
    const char* kt = s_kv[t & 1][0] + col * kRow;
    const char* vt = s_kv[t & 1][1] + vbyte;
    v4f s[KT];
#pragma unroll
    for (int u = 0; u < KT; ++u) s[u] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < QS; ++i)
#pragma unroll
      for (int u = 0; u < KT; ++u)
        s[u] = T::mfma16(*reinterpret_cast<const v4u32*>(kt + 16 * u * kRow + 16 * ((4 * i + grp) ^ key_swizzle<D>(col))), qf[i], s[u]);
    uint32_t live[KT];  // bit j of [u]: this row attends to key 16 u + 4 grp + j of the tile
    float top = kLowest;
#pragma unroll
    for (int u = 0; u < KT; ++u) {
      if constexpr (DRAFTED) {
        const int d = key0 + 16 * u + 4 * grp - ctx;
        const uint64_t on = d >= 0 ? seen >> min(d, 63) : seen << min(-d, 63) | ((1ull << min(-d, 63)) - 1);
        live[u] = d >= 64 ? 0u : (uint32_t)on & 15u;
      }
      v4f ks = {p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2};
      if constexpr (INT8) ks = *reinterpret_cast<const v4f*>(&s_ks[fill][at + 16 * u + 4 * grp]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = s[u][j] * ks[j];
        if (DRAFTED && !((live[u] >> j) & 1)) x = kNegInf;
        s[u][j] = x;
        top = fmaxf(top, x);
      }
    }
    top = rows_max(top);
    if (__any(top > m + reach)) {
      const float mn = top > m + reach ? (top - reach) + kSlack : m;
      const float c = exp2_hw(m - mn);
      l *= c;
#pragma unroll
      for (int e = 0; e < DB; ++e) acc[e] = acc[e] * c;
      m = mn;
    }
    v4u32 phi, plo;
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < KT; ++u) {
      float pv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pv[j] = exp2_hw(s[u][j] - m);
        sum[j % 2] += pv[j];
      }
      if constexpr (INT8) {
        const v4f vs = *reinterpret_cast<const v4f*>(&s_vs[fill][at + 16 * u + 4 * grp]);
#pragma unroll
        for (int j = 0; j < 4; ++j) pv[j] = DRAFTED && !((live[u] >> j) & 1) ? 0.0f : pv[j] * vs[j];  // a masked key's scale may be NaN
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t hi = PT::pack(pv[2 * j], pv[2 * j + 1]);
        const v2f back = PT::unpack(hi);
        phi[2 * u + j] = hi;
        plo[2 * u + j] = PT::pack(pv[2 * j] - back[0], pv[2 * j + 1] - back[1]);
      }
    }
    l += sum[0] + sum[1];
#pragma unroll
    for (int e = 0; e < DB; e += 2) {  // two sums in turn: neither waits for the other
      v4u32 a[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const char* from = vt + 16 * ((2 * (e + k) + (lane & 3) / 2) ^ swv(vkey));
        const v2u32 lo = read_transposed(from), hi = read_transposed(from + 16 * kRow);
        a[k] = v4u32{lo.x, lo.y, hi.x, hi.y};
        if constexpr (CAREFUL) {
#pragma unroll
          for (int j = 0; j < 4; ++j) a[k][j] = only_finite<PT>(a[k][j]);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[e + k % 2] = PT::mfma16(a[k % 2], k < 2 ? phi : plo, acc[e + k % 2]);
    }
    if (t + 1 < tiles) store(t + 1);
  };
  auto begin = [&] {
    place(0, page);
    if (kFill < keys) page = page_at(1);
    m = kLowest, l = 0.0f;
#pragma unroll
    for (int e = 0; e < DB; ++e) acc[e] = v4f{0, 0, 0, 0};
    load(0);
    store(0);
  };
  begin();
  int t = 0;
#pragma unroll 1
  for (; t < plain; ++t) step(t, std::false_type{}, std::false_type{});
#pragma unroll 1
  for (; t < tiles; ++t) step(t, std::true_type{}, std::false_type{});
  // As in the narrow kernel: values of masked keys that are infinities or NaN have spoiled the sums; the tiles with
  // drafted keys are computed without such values, which are added at the end to the rows that attend to them.
  bool careful = false;
  if constexpr (!INT8) {
    if (plain < tiles) {
      float odd = 0.0f;  // 0 where all sums are finite, else NaN
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) odd = fmaf(acc[i][r], 0.0f, odd);
      careful = __syncthreads_or(odd != 0.0f);
      if (careful) {
        page = page_at(0);
        begin();
#pragma unroll 1
        for (t = 0; t < plain; ++t) step(t, std::false_type{}, std::false_type{});
#pragma unroll 1
        for (; t < tiles; ++t) step(t, std::true_type{}, std::true_type{});
      }
    }
  }
  const bool bad = __syncthreads_or(bad_page);
  l = rows_sum(l);
  if (bad) l = __builtin_nanf("");
  const TreeParams q = arguments_again();
  int own = col;  // the row's node and head are found again, too
  asm volatile("" : "+v"(own));
  own += row0 + 16 * wave;
  if (own >= rows) return;
  const int out_node = own / q.G, out_head = g * q.G + own - out_node * q.G;
  const bool alone = rq.L <= keys;
  bool spoiled = false;
  const int64_t part = ((int64_t)(rq.q0 + out_node) * H + out_head) * q.parts + chunk;
  if (!alone && grp == 0) q.mp[part] = m, q.lp[part] = l;
#pragma unroll
  for (int e = 0; e < DB; ++e) {
    const int dim = 16 * e + 4 * grp;
    v4f o = acc[e];
    if (careful) {
#pragma unroll 1
      for (int key = start + plain * kKeys; key < end; ++key) {
        const int32_t block = p.bt[(int64_t)b * p.sbt + page_of(p, key)];
        const bool on = (key < ctx || (seen >> (key - ctx)) & 1) && block >= 0 && block < p.blocks;
        if (!on) continue;
        const v2u32 w = *reinterpret_cast<const v2u32*>(vh + block * p.svb + (int64_t)(key - page_of(p, key) * p.page) * p.svp + 2 * dim);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = T::to_f32((uint16_t)(w[j / 2] >> (16 * (j % 2))));
          if (!__builtin_isfinite(f)) o[j] += f;
        }
      }
    }
    if (alone)
      spoiled |= store_row<T>(q, rq, out_node, out_head, dim, o, l);
    else
      *reinterpret_cast<v4f*>(q.ap + part * D + dim) = o;
  }
  if (__builtin_expect(spoiled, 0))
#pragma unroll 1
    for (int dim = 4 * grp; dim < D; dim += 16) find_specials<T, INT8>(q, rq, b, out_node, out_head, dim);
}

// Joins a row's groups: the strands of a group where workgroups have left them apart, then the groups in order; of the wide
// kernel four chunks are a group. A workgroup joins one row, GROUPS groups at a time, 4 dims a lane: their partials are on
// their way together. A row of several groups attends to its context, so its sum is not empty.
template <typename T, bool INT8, int D, int GROUPS>
__global__ __launch_bounds__(D * GROUPS / 4) void tree_merge_kernel(TreeParams p) {
  constexpr int kLanes = D / 4;
  __shared__ float s_ml[GROUPS][2];
  __shared__ v4f s_a[GROUPS][kLanes];
  const int H = p.KV * p.G;
  const int mine = threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  const int head = (int)(blockIdx.x % (uint32_t)H);
  const uint32_t bn = blockIdx.x / (uint32_t)H;
  const int b = (int)(bn / (uint32_t)p.max_nodes), node = (int)(bn % (uint32_t)p.max_nodes);
  const Request rq = request_of(p, b);
  const bool wide = rq.T * p.G > p.wide_rows, apart = wide || p.strands;
  const int keys = wide ? wide_chunk(rq.L) : kSeg;
  const int chunks = (rq.L + keys - 1) / keys, groups = (chunks + kGroup - 1) / kGroup;
  if (rq.bad || node >= rq.T || chunks <= (wide ? 1 : kGroup)) return;
  const int64_t part = ((int64_t)(rq.q0 + node) * H + head) * p.parts;
  State sum;
  for (int g0 = 0; g0 < groups; g0 += GROUPS) {
    if (g0 + mine < groups) {
      State s[kWaves];
      const int64_t at = part + (g0 + mine) * (apart ? kWaves : 1);
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        if (w == 0 || (apart && (!wide || (g0 + mine) * kGroup + w < chunks))) s[w] = State{p.mp[at + w], p.lp[at + w], reinterpret_cast<const v4f*>(p.ap)[(at + w) * kLanes + c]};
      if (apart) join(s, wide ? chunks - (g0 + mine) * kGroup : kWaves);
      if (c == 0) s_ml[mine][0] = s[0].m, s_ml[mine][1] = s[0].l;
      s_a[mine][c] = s[0].a;
    }
    __syncthreads();
    if (mine == 0) {
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        if (g0 + i >= groups) break;
        const State s{s_ml[i][0], s_ml[i][1], s_a[i][c]};
        if (g0 + i == 0) sum = s; else sum.add(s);
      }
    }
    __syncthreads();
  }
  if (mine != 0) return;
  const bool spoiled = store_row<T>(p, rq, node, head, 4 * c, sum.a, sum.l);
  if (__builtin_expect(spoiled, 0)) find_specials<T, INT8>(arguments_again(), rq, b, node, head, 4 * c);
}

// The most chunks of any request of at most `keys` keys.
int64_t most_chunks(int64_t keys) {
  const int64_t few = std::min<int64_t>(keys, 4096);
  return std::max(cdiv<int64_t>(few, wide_chunk((int)few)), cdiv<int64_t>(keys, wide_chunk((int)keys)));
}

int64_t num_segments(int64_t keys) { return std::max<int64_t>(1, cdiv<int64_t>(keys, kSeg)); }

// How a call's rows and keys are split, and the partial sums that a row has place for.
struct Plan {
  int64_t narrow, row_blocks, groups, parts;  // narrow: rows that the narrow kernel covers, of requests that do not take the wide one
  int nq;
  bool strands, by_size, wide;
};
Plan plan_of(int64_t n, int64_t KV, int64_t G, int64_t D, int64_t max_nodes, int64_t max_len) {
  Plan p;
  const int64_t rows = max_nodes * G, most = wide_rows((int)D), ns = num_segments(max_len);
  p.narrow = std::min<int64_t>(rows, most / G * G);
  p.nq = p.narrow <= 16 ? 1 : 2;
  p.row_blocks = std::max<int64_t>(1, cdiv<int64_t>(p.narrow, 16 * p.nq));
  p.wide = rows > most;
  // A workgroup for each group of segments, or for each of its strands where the former would leave CUs without one. The
  // order of the sums, and so every bit, is the same. (10 requests of up to 8000 keys, 8 tokens, 320 groups: 54 us in
  // strands, 45 in groups; 20 of up to 16384, 2 tokens, 1440 groups: 118 and 98; with 256 the same.)
  p.groups = cdiv<int64_t>(ns, kGroup);
  p.strands = p.groups > 1 && product({n, KV, p.row_blocks, p.groups}) < kManyWorkgroups;
  // The last rounds of workgroups end together where the large ones have gone first. The search takes a turn for every 64
  // requests, and there are many rounds where they are many.
  p.by_size = !p.strands && p.groups > 1 && n <= kSearched;
  // A single group of segments has no partial sums, but they are few and counted for its chunks in the wide kernel.
  p.parts = ns <= kGroup ? ns : p.strands ? p.groups * kWaves : std::max(p.groups, p.wide ? most_chunks(max_len) : 0);
  return p;
}

template <typename T, bool INT8, int D>
hipError_t launch_tree(TreeParams p, const Plan& plan, hipStream_t st) {
  p.wide_rows = wide_rows(D);
  p.row_blocks = (int32_t)plan.row_blocks;
  p.strands = plan.strands, p.by_size = plan.by_size;
  TreeParams w = p;
  w.row_blocks = (int32_t)cdiv<int64_t>((int64_t)p.max_nodes * p.G, 128);
  // Every launch is looked at before the first.
  const int64_t blocks = product({cdiv<int64_t>(product({p.KV, p.n, plan.groups, plan.strands ? kWaves : 1}), 8), 8, p.row_blocks});
  const int64_t wide = product({cdiv<int64_t>(product({p.KV, p.n, most_chunks(p.max_len)}), 8), 8, w.row_blocks});
  const int64_t merges = product({p.n, p.max_nodes, p.KV, p.G});
  const int threads = 64 * kWaves, wide_threads = D == 256 ? 64 * kWaves256 : threads;
  const bool merged = p.ns > (plan.wide ? 1 : kGroup), few = merges <= 2048;
  if (!launchable(blocks, threads) || (plan.wide && !launchable(wide, wide_threads)) || (merged && !launchable(merges, D * (few ? 16 : 2) / 4)))
    return hipErrorInvalidConfiguration;
  if (plan.nq == 1)
    hipLaunchKernelGGL((tree_partial_kernel<T, INT8, D, 1>), dim3((unsigned)blocks), dim3(threads), 0, st, p);
  else
    hipLaunchKernelGGL((tree_partial_kernel<T, INT8, D, 2>), dim3((unsigned)blocks), dim3(threads), 0, st, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  if (plan.wide) {
    if constexpr (D == 256)
      hipLaunchKernelGGL((tree_decode_kernel_wide_256<T, INT8>), dim3((unsigned)wide), dim3(wide_threads), 0, st, w);
    else
      hipLaunchKernelGGL((tree_decode_kernel_wide<T, INT8, D>), dim3((unsigned)wide), dim3(wide_threads), 0, st, w);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  if (!merged) return hipSuccess;
  // Few rows: latency counts, and all their groups are read at once (one row over 16384 keys: 16.7 us -> 14.6). Many rows: the
  // fewer threads that wait for others, the better (16384 rows of 2 to 5 groups: 218 us with 16 groups at a time, 198 with 2).
  if (few)
    hipLaunchKernelGGL((tree_merge_kernel<T, INT8, D, 16>), dim3((unsigned)merges), dim3(D * 16 / 4), 0, st, p);
  else
    hipLaunchKernelGGL((tree_merge_kernel<T, INT8, D, 2>), dim3((unsigned)merges), dim3(D * 2 / 4), 0, st, p);
  return hipGetLastError();
}

template <typename T, bool INT8>
hipError_t dispatch_dim(int64_t D, const TreeParams& p, const Plan& plan, hipStream_t st) {
  if (D == 64) return launch_tree<T, INT8, 64>(p, plan, st);
  if (D == 128) return launch_tree<T, INT8, 128>(p, plan, st);
  return launch_tree<T, INT8, 256>(p, plan, st);
}

// Bytes of `parts` partial sums for each row, 0 for one; less than 0 where that is no size of anything.
int64_t workspace_bytes(int64_t tokens, int64_t H, int64_t D, int64_t parts) {
  if (parts <= 1) return 0;
  int64_t bytes;
  const bool over = __builtin_mul_overflow(tokens, H, &bytes) || __builtin_mul_overflow(bytes, parts, &bytes) ||
                    __builtin_mul_overflow(bytes, (D + 2) * (int64_t)sizeof(float), &bytes);
  return over ? -1 : bytes;
}

}  // namespace

extern "C" int vxa_tree_decode_workspace(int64_t tokens, int64_t num_heads, int64_t head_dim, int64_t max_seq_len,
                                         size_t* ws_bytes) {
  if (tokens < 0 || num_heads <= 0 || head_dim <= 0 || max_seq_len < 0 || !ws_bytes) return VXA_ERR_ARG;
  // The most of any plan: a partial sum for each strand of each group of segments.
  const int64_t ns = num_segments(max_seq_len);
  const int64_t bytes = workspace_bytes(tokens, num_heads, head_dim, ns <= kGroup ? ns : cdiv<int64_t>(ns, kGroup) * kWaves);
  if (bytes < 0) return VXA_ERR_UNSUPPORTED;
  *ws_bytes = (size_t)bytes;
  return VXA_OK;
}

extern "C" int vxa_tree_decode_call_workspace(int64_t n, int64_t tokens, int64_t num_heads, int64_t num_kv_heads,
                                              int64_t head_dim, int64_t max_nodes, int64_t max_seq_len, size_t* ws_bytes) {
  if (n < 0 || tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || max_nodes < 0 || max_seq_len < 0 || !ws_bytes ||
      num_heads % num_kv_heads != 0)
    return VXA_ERR_ARG;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return VXA_ERR_UNSUPPORTED;
  if (n > 0x7FFFFFFFLL || tokens > 0x7FFFFFFFLL || num_heads > (1 << 16) || max_nodes > kMaxNodes || max_seq_len > (1 << 30))
    return VXA_ERR_UNSUPPORTED;
  const int64_t bytes = workspace_bytes(tokens, num_heads, head_dim,
                                        plan_of(n, num_kv_heads, num_heads / num_kv_heads, head_dim, max_nodes, max_seq_len).parts);
  if (bytes < 0) return VXA_ERR_UNSUPPORTED;
  *ws_bytes = (size_t)bytes;
  return VXA_OK;
}

extern "C" int vxa_tree_decode(const void* q, int64_t sqt, int64_t sqh, int q_dtype, const void* k_cache, int64_t skb,
                               int64_t skp, int64_t skh, const void* v_cache, int64_t svb, int64_t svp, int64_t svh,
                               const float* k_scale, int64_t sksb, int64_t sksp, int64_t sksh, const float* v_scale,
                               int64_t svsb, int64_t svsp, int64_t svsh, int64_t num_blocks, int64_t block_size,
                               const int32_t* block_table, int64_t sbt, int64_t bt_cols, const int32_t* seq_lens,
                               const int32_t* query_starts, const int64_t* tree_mask, float scale, void* out,
                               int out_dtype, int64_t sot, int64_t soh, int64_t n, int64_t tokens, int64_t num_heads,
                               int64_t num_kv_heads, int64_t head_dim, int64_t max_nodes, int64_t max_seq_len, void* ws,
                               size_t ws_bytes, vxa_stream_t stream) {
  if (n < 0 || tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_blocks < 0 || block_size <= 0 ||
      bt_cols < 0 || max_nodes < 0 || max_seq_len < 0)
    return VXA_ERR_ARG;
  if (q_dtype != VXA_BF16 && q_dtype != VXA_F16) return VXA_ERR_ARG;
  if (out_dtype != VXA_F32 && out_dtype != VXA_BF16 && out_dtype != VXA_F16) return VXA_ERR_ARG;
  if (num_heads % num_kv_heads != 0 || (k_scale == nullptr) != (v_scale == nullptr)) return VXA_ERR_ARG;
  if (n == 0 || tokens == 0 || max_nodes == 0) return VXA_OK;
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !query_starts || !out || num_blocks == 0) return VXA_ERR_ARG;
  const bool int8 = k_scale != nullptr;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return VXA_ERR_UNSUPPORTED;
  if (max_nodes > kMaxNodes || num_heads > (1 << 16) || block_size > (1 << 30)) return VXA_ERR_UNSUPPORTED;
  if (n > 0x7FFFFFFFLL || tokens > 0x7FFFFFFFLL || max_seq_len > (1 << 30) || bt_cols > 0x7FFFFFFFLL ||
      num_blocks > 0x7FFFFFFFLL)
    return VXA_ERR_UNSUPPORTED;
  // Rows are read in 16-byte pieces.
  const int64_t piece = int8 ? 16 : 8, size = int8 ? 1 : 2;
  if ((uintptr_t)q % 16 || (uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || sqt % 8 || sqh % 8 || skb % piece ||
      skp % piece || skh % piece || svb % piece || svp % piece || svh % piece)
    return VXA_ERR_UNSUPPORTED;
  size_t need = 0;
  const int rc = vxa_tree_decode_call_workspace(n, tokens, num_heads, num_kv_heads, head_dim, max_nodes, max_seq_len, &need);
  if (rc != VXA_OK) return rc;
  if (need > 0 && (!ws || ws_bytes < need)) return VXA_ERR_WORKSPACE;
  if (need > 0 && (uintptr_t)ws % 16) return VXA_ERR_UNSUPPORTED;

  TreeParams p;
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.sqt = sqt, p.sqh = sqh;
  p.kc = reinterpret_cast<const char*>(k_cache);
  p.skb = skb * size, p.skp = skp * size, p.skh = skh * size;
  p.vc = reinterpret_cast<const char*>(v_cache);
  p.svb = svb * size, p.svp = svp * size, p.svh = svh * size;
  p.ks = k_scale, p.sksb = sksb, p.sksp = sksp, p.sksh = sksh;
  p.vs = v_scale, p.svsb = svsb, p.svsp = svsp, p.svsh = svsh;
  p.bt = block_table, p.sbt = sbt, p.cols = (int32_t)bt_cols, p.page = (int32_t)block_size, p.blocks = num_blocks;
  p.sl = seq_lens, p.qsl = query_starts, p.mask = tree_mask;
  p.scale_log2 = (float)((double)scale * 1.4426950408889634);
  p.n = (int32_t)n, p.total = (int32_t)tokens, p.KV = (int32_t)num_kv_heads, p.G = (int32_t)(num_heads / num_kv_heads);
  const Plan plan = plan_of(n, p.KV, p.G, head_dim, max_nodes, max_seq_len);
  p.ns = (int32_t)num_segments(max_seq_len), p.row_blocks = 1, p.max_nodes = (int32_t)max_nodes, p.max_len = (int32_t)max_seq_len;
  p.strands = false, p.by_size = false, p.parts = plan.parts;
  // The weighted values first, on 16 bytes as the workspace is.
  const int64_t parts = tokens * num_heads * p.parts;
  float* w = reinterpret_cast<float*>(ws);
  p.ap = w, p.mp = need > 0 ? w + parts * head_dim : nullptr, p.lp = need > 0 ? p.mp + parts : nullptr;
  p.out = out, p.sot = sot, p.soh = soh, p.out_dtype = out_dtype;
  p.out_wide = out_dtype == q_dtype && (uintptr_t)out % 8 == 0 && sot % 4 == 0 && soh % 4 == 0;
  p.by_page = make_divisor(block_size);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipError_t err;
  if (q_dtype == VXA_BF16)
    err = int8 ? dispatch_dim<BF16, true>(head_dim, p, plan, st) : dispatch_dim<BF16, false>(head_dim, p, plan, st);
  else
    err = int8 ? dispatch_dim<FP16, true>(head_dim, p, plan, st) : dispatch_dim<FP16, false>(head_dim, p, plan, st);
  if (err == hipErrorInvalidConfiguration) return VXA_ERR_UNSUPPORTED;
  return err == hipSuccess ? VXA_OK : VXA_ERR_LAUNCH;
}
