// Causal attention over whole prompts, packed one after the other (gfx950).
//
//   o_i = sum_{j <= i} p_ij v_j / sum_{j <= i} p_ij,   p_ij = exp(scale q_i.k_j - max_j scale q_i.k_j)
// for every row i of every sequence, with groups of G = H / KV query heads on one key/value head.
//
// Work split. A workgroup of 4 waves computes 32 rows of four heads of one KV head (64 rows of two, 128 of one where
// the group has no more), 32 rows of one head a wave, and walks the keys up to its last row in tiles of 64 with one running
// maximum and sum: every score is computed once and kept in registers. A wave's rows are the columns of S^T = K Q^T
// (32 x 32 x 16 MFMAs) and of O^T = V^T P^T, so a lane holds scores of one row only, and with the keys of the second
// product taken in the order in which the first one leaves them in the lane, P goes from one product to the other
// without leaving the lane. The tiles of K and V are copied straight into LDS, two in turn; V is transposed as it is read
// from there. Two workgroups share a CU. At 256 dims a wave takes 16 rows (below). The workgroups furthest from their
// sequence's start, which take longest, go first.
// A row's order of operations depends on its place in its sequence and its own scores, so its bits depend on its query and on
// the keys and values up to its own, not on other rows or the batch.
//
// Rounding. Scores, maxima, sums and accumulators are fp32; P is rounded to the 16-bit element type for the second
// product, an error of the size of the output's own rounding (in fp16, weights below 2^-21 of a row's largest are off by up to
// 2^-32 of it), while its sum takes the fp32 values.
//
// What bounds it. One prompt of 8192 tokens (32 heads on 8, 128 dims, bf16) takes 521 to 555 us on different cards, 990 to
// 1055 TFLOP/s of the scores that count; a large library matrix product reaches 1189, and this kernel runs at 1.9 GHz: power.
// The matrix pipes are busy 52 % of the cycles; the next tile's scores among this one's softmax instructions, in one wave, gave
// no time back (519 to 540 us). 16 prompts of up to 1024 tokens take 93 us, 570 TFLOP/s: 7 us of every workgroup's 20 go
// to finding its rows, the first loads and the output.

#include <algorithm>
#include <cmath>

#include "attention_common.h"

namespace {

constexpr int kWaves = 4;     // of a workgroup
constexpr int kWaves256 = 8;  // ... of the kernel for 256 dims

struct PromptParams {
  const uint16_t* q;
  int64_t sqt, sqh;
  const uint16_t* k;
  int64_t skt, skh;
  const uint16_t* v;
  int64_t svt, svh;
  const int32_t* cu;
  float scale_log2;  // > 0: the sign and a zero of the scale are in q's elements,
  uint32_t q_and, q_xor;  // (q & q_and) ^ q_xor, so that scaled scores keep the order of the products
  int32_t n, total, H, G, tiles;
  int32_t heads, rows;  // of a workgroup: heads of one KV head, and rows of each: a wave's rows are of one head
  void* out;
  int64_t sot, soh;
  int32_t out_dtype;
  bool out_wide;  // the output has the input's type and its rows start on 16 bytes
};

// The sequence and rows of tile `tile`. Tiles of p.rows rows are counted from those furthest from their sequence's start,
// which take longest, over all sequences (256 sequences at a time).
struct Tile {
  int base, len, row0;  // first packed row of the sequence, its length (0: no such tile), the tile's first row in it
};
__device__ inline Tile find_tile(const PromptParams& p, int tile) {
  if (p.n == 1) {
    const int lo = max(p.cu[0], 0), len = max(min(p.cu[1], p.total) - lo, 0), count = (len + p.rows - 1) / p.rows;
    return tile < count ? Tile{lo, len, (count - 1 - tile) * p.rows} : Tile{0, 0, 0};
  }
  const int lane = threadIdx.x & 63;
  for (int j0 = 0; j0 < p.n; j0 += 256) {
    int lo[4], len[4], count[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int j = j0 + 64 * c + lane;
      lo[c] = 0, len[c] = 0;
      if (j < p.n) {
        lo[c] = max(p.cu[j], 0);
        len[c] = max(min(p.cu[j + 1], p.total) - lo[c], 0);
      }
      count[c] = (len[c] + p.rows - 1) / p.rows;
    }
    // below(k) tiles are among their sequences' first k.
    auto below = [&](int k) { return wave_reduce(min(count[0], k) + min(count[1], k) + min(count[2], k) + min(count[3], k), [](int a, int b) { return a + b; }); };
    const int total = below(0x7FFFFFFF);
    if (tile >= total) {
      tile -= total;
      continue;
    }
    int left = total - 1 - tile, level = 0, under = 0;
    const int most = wave_reduce(max(max(count[0], count[1]), max(count[2], count[3])), [](int a, int b) { return max(a, b); });
    for (int step = 1 << (31 - __builtin_clz(most)); step > 0; step /= 2) {
      const int s = below(level + step);
      if (s <= left) level += step, under = s;
    }
    left -= under;  // the sequence is number `left` of those with more than `level` tiles
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint64_t more = __ballot(count[c] > level);
      const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(more >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)more, 0));
      const uint64_t hit = __ballot(count[c] > level && before == left);
      if (hit != 0) {
        const int at = __builtin_ctzll(hit);
        return Tile{__builtin_amdgcn_readlane(lo[c], at), __builtin_amdgcn_readlane(len[c], at), level * p.rows};
      }
      left -= __popcll(more);
    }
  }
  return Tile{0, 0, 0};
}

// Four dims of a row after a careful pass: the infinities and NaN among the values of its keys from `masked` on, 8 bytes a key.
template <typename T>
__device__ inline void add_masked_specials(float (&o)[4], const char* values, int64_t stride, int masked, int row) {
  v4f special = {0, 0, 0, 0};
#pragma unroll 1
  for (int key = masked; key <= row; ++key) add_specials<T>(special, *reinterpret_cast<const v2u32*>(values + key * stride));
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] += special[j];
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void prompt_attention_kernel(PromptParams p) {
  constexpr int kKeys = 64, KU = kKeys / 32;  // keys of a tile, in blocks of 32
  constexpr int QS = D / 16;       // MFMA steps over the head's dims
  constexpr int DB = D / 32;       // 32-dim blocks of O^T
  constexpr int kRow = 2 * D;      // bytes of a key in LDS
  constexpr int kTileBytes = kKeys * kRow;
  constexpr int kPer = 1024 / kRow;                   // keys that one wave's copy moves
  constexpr int kRound = kPer * kWaves;               // ... that all waves' copies move
  constexpr int kCopies = kKeys / kRound;             // copies of a wave for a tile of K, and of V
  static_assert(kRound % 16 == 0);                    // K's swizzle is the same for every copy of a wave
  __shared__ __attribute__((aligned(1024))) char s_kv[2][2][kTileBytes];  // [buffer][K, V][key][16-byte chunk, swizzled]
  auto swk = [](int key) { return key_swizzle<D>(key); };
  auto swv = [](int key) { return value_swizzle<D>(key); };

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;

  // Workgroups of one KV head run on one XCD, longest rows first.
  const int groups = p.H / p.heads;
  const int x = (int)(blockIdx.x % groups);
  const int head = (groups % 8 == 0 ? (x % 8) * (groups / 8) + x / 8 : x) * p.heads + wave % p.heads;
  const Tile tile = find_tile(p, (int)(blockIdx.x / groups));
  if (tile.len == 0) return;
  const int base = __builtin_amdgcn_readfirstlane(tile.base);
  const int len = __builtin_amdgcn_readfirstlane(tile.len);
  const int row0 = __builtin_amdgcn_readfirstlane(tile.row0);
  const char* kh = reinterpret_cast<const char*>(p.k + (int64_t)base * p.skt + (int64_t)(head / p.G) * p.skh);
  const char* vh = reinterpret_cast<const char*>(p.v + (int64_t)base * p.svt + (int64_t)(head / p.G) * p.svh);
  const int64_t skt = 2 * p.skt, svt = 2 * p.svt;

  const int wrow = row0 + wave / p.heads * 32;  // the wave's first row
  const int row = wrow + col;
  const float reach = T::reach(row + 1);
  const int last = min(row0 + p.rows, len);  // keys of the workgroup
  const int tiles = (last + kKeys - 1) / kKeys;

  // Tiles go straight from memory into LDS. Copy i of a wave moves keys i * kRound + wave * kPer + [0, kPer).
  const int key_l = wave * kPer + lane / (kRow / 16), chunk = lane % (kRow / 16);
  const char* ksrc = kh + key_l * skt + 16 * (chunk ^ swk(key_l));
  const char* vsrc = vh + key_l * svt + 16 * (chunk ^ swv(key_l));
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t*)&s_kv[0][0][0]) + wave * 1024;
  auto load = [&](int t, int buf) {
    const uint32_t dst = lds0 + buf * 2 * kTileBytes;
    if ((t + 1) * kKeys <= len) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        copy_to_lds(ksrc + (int64_t)(t * kKeys + i * kRound) * skt, dst + i * kWaves * 1024);
        copy_to_lds(vsrc + (int64_t)(t * kKeys + i * kRound) * svt, dst + kTileBytes + i * kWaves * 1024);
      }
    } else {  // keys past the sequence's end repeat its last one
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int in_tile = i * kRound + key_l, key = min(t * kKeys + in_tile, len - 1);
        copy_to_lds(kh + key * skt + 16 * (chunk ^ swk(in_tile)), dst + i * kWaves * 1024);
        copy_to_lds(vh + key * svt + 16 * (chunk ^ swv(in_tile)), dst + kTileBytes + i * kWaves * 1024);
      }
    }
  };

  // Where this lane reads: K's row `col` of a 32-key block, V's rows 4 half + (lane % 16) / 4 and 8 further.
  const int vkey = 4 * half + (lane & 15) / 4;
  const int vdim = 2 * ((lane >> 4) & 1) + (lane & 3) / 2;  // chunk in a 32-dim block
  const int vbyte = vkey * kRow + 8 * (lane & 1);

  float m, l[4];
  v16f acc[DB];

  const int full = min((wrow + 1) / kKeys, tiles);  // tiles without masked keys
  auto start = [&] {
    m = kLowest;
#pragma unroll
    for (int i = 0; i < 4; ++i) l[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    load(0, 0);
  };
  start();
  v4u32 qf[QS];  // after the first tile has been asked for: changing their signs waits for them
  {
    const uint16_t* q = p.q + (int64_t)(base + min(row, len - 1)) * p.sqt + (int64_t)head * p.sqh + 8 * half;
#pragma unroll
    for (int i = 0; i < QS; ++i) qf[i] = (*reinterpret_cast<const v4u32*>(q + 16 * i) & p.q_and) ^ p.q_xor;
  }
  // One tile. MASKED: some of its keys may come after some of the wave's rows.
  // CAREFUL: values may be infinities or NaN, and 0 times those is NaN, for a key that a row does not attend to as for a weight
  // that is too small for its type. Here they enter the product as 0. Rows that attend to all of the tile add them with
  // weights of 1, the others add those that they attend to at the end. The pass that does not look ends with sums that are
  // not finite wherever that mattered.
  auto step = [&](int t, auto masked_c, auto careful_c) {
    constexpr bool MASKED = decltype(masked_c)::value, CAREFUL = decltype(careful_c)::value;
    constexpr uint32_t kOnes = T::kOne | T::kOne << 16;
    // Tile t has landed, for every wave, and every wave has read tile t - 1: its buffer takes tile t + 1.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int buf = t & 1;
    if (t + 1 < tiles) load(t + 1, buf ^ 1);
    const int key0 = t * kKeys;
    if (MASKED && key0 > wrow + 31) return;  // no row of the wave attends to the tile
    const char* kt = s_kv[buf][0] + col * kRow;
    const char* vt = s_kv[buf][1] + vbyte;
    v16f s[KU];
#pragma unroll
    for (int u = 0; u < KU; ++u) s[u] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < QS; ++i)
#pragma unroll
      for (int u = 0; u < KU; ++u)
        s[u] = T::mfma32(*reinterpret_cast<const v4u32*>(kt + 32 * u * kRow + 16 * ((2 * i + half) ^ swk(col))), qf[i], s[u]);
    if constexpr (MASKED) {
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + 32 * u + (r & 3) + 8 * (r >> 2) + 4 * half > row) s[u][r] = kNegInf;
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
    float ta = top, tb = top;
    swap32(ta, tb);
    top = fmaxf(ta, tb) * p.scale_log2;
    if (__any(top > m + reach)) {
      const float mn = top > m + reach ? (top - reach) + kSlack : m;
      const float c = exp2_hw(m - mn);
#pragma unroll
      for (int i = 0; i < 4; ++i) l[i] *= c;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = CAREFUL ? scaled(acc[i][r], c) : acc[i][r] * c;
      m = mn;
    }
    v4u32 pf[2 * KU];
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float a = exp2_hw(fmaf(s[u][r], p.scale_log2, -m)), b = exp2_hw(fmaf(s[u][r + 1], p.scale_log2, -m));
        l[r % 4] += a;
        l[r % 4 + 1] += b;
        pf[2 * u + r / 8][r % 8 / 2] = T::pack(a, b);
      }
    // Chunk c of P holds, for j = 0..7, the keys 16 c + 4 half + j % 4 + 8 (j / 4): the order of the lane's scores.
    auto values = [&](int c, int i) {
      const char* at = vt + 16 * c * kRow + 16 * ((4 * i + vdim) ^ swv(vkey));
      const v2u32 lo = read_transposed(at), hi = read_transposed(at + 8 * kRow);
      return v4u32{lo.x, lo.y, hi.x, hi.y};
    };
#pragma unroll
    for (int c = 0; c < 2 * KU; ++c)
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        v4u32 a = values(c, i);
        if constexpr (CAREFUL) {
          v4u32 special;
#pragma unroll
          for (int j = 0; j < 4; ++j) special[j] = only_special<T>(a[j]), a[j] ^= special[j];
          if constexpr (!MASKED) acc[i] = T::mfma32(special, v4u32{kOnes, kOnes, kOnes, kOnes}, acc[i]);
        }
        acc[i] = T::mfma32(a, pf[c], acc[i]);
      }
  };
  int t = 0;
  for (; t < full; ++t) step(t, std::false_type{}, std::false_type{});
  for (; t < tiles; ++t) step(t, std::true_type{}, std::false_type{});
  float odd = 0.0f;  // 0 where all sums are finite, else NaN
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd = fmaf(acc[i][r], 0.0f, odd);
  const bool careful = __syncthreads_or(odd != 0.0f);
  if (careful) {
    start();
    for (t = 0; t < full; ++t) step(t, std::false_type{}, std::true_type{});
    for (; t < tiles; ++t) step(t, std::true_type{}, std::true_type{});
  }
  float la = (l[0] + l[1]) + (l[2] + l[3]), lb = la;
  swap32(la, lb);
  const float sum = la + lb, inv = sum > 0.0f ? 1.0f / sum : __builtin_nanf("");  // 0: every score is -inf
  if (row >= len) return;
  const int64_t at = (int64_t)(base + row) * p.sot + (int64_t)head * p.soh;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += 8) {
      uint32_t w[2][2];  // dims 32 i + 2 r0 + 8 k + 4 half + 0..3
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = acc[i][r0 + 4 * k + j] * inv;
        const int dim = 32 * i + 2 * r0 + 8 * k + 4 * half;
        if (careful) add_masked_specials<T>(o, vh + 2 * dim, svt, full * kKeys, row);
        w[k][0] = T::pack(o[0], o[1]), w[k][1] = T::pack(o[2], o[3]);
        if (!p.out_wide) {
#pragma unroll
          for (int j = 0; j < 4; ++j) store_f32_as(p.out, p.out_dtype, at + dim + j, o[j]);
        }
      }
      if (p.out_wide) {  // 8 dims a lane: the halves exchange what the other stores
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const auto x = __builtin_amdgcn_permlane32_swap(w[0][j], w[1][j], false, false);
          w[0][j] = x[0], w[1][j] = x[1];
        }
        *reinterpret_cast<v4u32*>(reinterpret_cast<uint16_t*>(p.out) + at + 32 * i + 2 * r0 + 8 * half) =
            v4u32{w[0][0], w[0][1], w[1][0], w[1][1]};
      }
    }
}

// The same for 256 dims, with 8 waves of 16 rows and 16 x 16 x 32 MFMAs: 32 rows of a wave take 430 registers and leave one
// wave a SIMD, whose softmax and products follow each other; 16 rows take 201 and leave two, though each reads K and V from
// LDS for half as many rows. Three prompts of up to 2111 tokens: 119 us -> 90; one of 5000: 650 -> 470 (870 TFLOP/s). With
// 64 or 128 dims, where two waves of 32 rows fit, they are faster (8192 tokens, 128 dims: 525 us against 575).
template <typename T>
__global__ __launch_bounds__(64 * kWaves256, 2) void prompt_attention_kernel_256(PromptParams p) {
  constexpr int D = 256, NW = kWaves256;
  constexpr int kKeys = 32;
  constexpr int KT = kKeys / 16;   // 16-key blocks of S^T
  constexpr int QS = D / 32;       // MFMA steps over the head's dims
  constexpr int DB = D / 16;       // 16-dim blocks of O^T
  constexpr int kRow = 2 * D, kTileBytes = kKeys * kRow;
  constexpr int kPer = 1024 / kRow, kRound = kPer * NW, kCopies = kKeys / kRound;
  static_assert(kRound == 16);     // K's swizzle is the same for every copy of a wave
  __shared__ __attribute__((aligned(1024))) char s_kv[2][2][kTileBytes];
  auto swk = [](int key) { return key_swizzle<D>(key); };
  // Here 16 lanes read two chunks of four keys, and 64 lanes of 16: eight keys meet the 256 bytes of the banks.
  auto swv = [](int key) { return 2 * (key & 7); };

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int groups = p.H / p.heads;
  const int x = (int)(blockIdx.x % groups);
  const int head = (groups % 8 == 0 ? (x % 8) * (groups / 8) + x / 8 : x) * p.heads + wave % p.heads;
  const Tile tile = find_tile(p, (int)(blockIdx.x / groups));
  if (tile.len == 0) return;
  const int base = __builtin_amdgcn_readfirstlane(tile.base);
  const int len = __builtin_amdgcn_readfirstlane(tile.len);
  const int row0 = __builtin_amdgcn_readfirstlane(tile.row0);
  const char* kh = reinterpret_cast<const char*>(p.k + (int64_t)base * p.skt + (int64_t)(head / p.G) * p.skh);
  const char* vh = reinterpret_cast<const char*>(p.v + (int64_t)base * p.svt + (int64_t)(head / p.G) * p.svh);
  const int64_t skt = 2 * p.skt, svt = 2 * p.svt;
  const int wrow = row0 + wave / p.heads * 16;  // the wave's first row
  const int row = wrow + col;
  const float reach = T::reach(row + 1);
  const int last = min(row0 + p.rows, len);  // keys of the workgroup
  const int tiles = (last + kKeys - 1) / kKeys;

  const int key_l = wave * kPer + lane / (kRow / 16), chunk = lane % (kRow / 16);
  const char* ksrc = kh + key_l * skt + 16 * (chunk ^ swk(key_l));
  const char* vsrc = vh + key_l * svt + 16 * (chunk ^ swv(key_l));
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t*)&s_kv[0][0][0]) + wave * 1024;
  auto load = [&](int t, int buf) {
    const uint32_t dst = lds0 + buf * 2 * kTileBytes;
    if ((t + 1) * kKeys <= len) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        copy_to_lds(ksrc + (int64_t)(t * kKeys + i * kRound) * skt, dst + i * NW * 1024);
        copy_to_lds(vsrc + (int64_t)(t * kKeys + i * kRound) * svt, dst + kTileBytes + i * NW * 1024);
      }
    } else {  // keys past the sequence's end repeat its last one
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int in_tile = i * kRound + key_l, key = min(t * kKeys + in_tile, len - 1);
        copy_to_lds(kh + key * skt + 16 * (chunk ^ swk(in_tile)), dst + i * NW * 1024);
        copy_to_lds(vh + key * svt + 16 * (chunk ^ swv(in_tile)), dst + kTileBytes + i * NW * 1024);
      }
    }
  };

  // Where this lane reads: K's row `col` of a 16-key block, V's rows 4 grp + col / 4 and 16 further.
  const int vkey = 4 * grp + col / 4;
  const int vbyte = vkey * kRow + 8 * (lane & 1);
  const int full = min((wrow + 1) / kKeys, tiles);  // tiles without masked keys
  float m, l;
  v4f acc[DB];
  auto start = [&] {
    m = kLowest, l = 0.0f;
#pragma unroll
    for (int e = 0; e < DB; ++e) acc[e] = v4f{0, 0, 0, 0};
    load(0, 0);
  };
  start();
  v4u32 qf[QS];
  {
    const uint16_t* q = p.q + (int64_t)(base + min(row, len - 1)) * p.sqt + (int64_t)head * p.sqh + 8 * grp;
#pragma unroll
    for (int i = 0; i < QS; ++i) qf[i] = (*reinterpret_cast<const v4u32*>(q + 32 * i) & p.q_and) ^ p.q_xor;
  }
  auto step = [&](int t, auto masked_c, auto careful_c) {
    constexpr bool MASKED = decltype(masked_c)::value, CAREFUL = decltype(careful_c)::value;
    constexpr uint32_t kOnes = T::kOne | T::kOne << 16;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int buf = t & 1;
    if (t + 1 < tiles) load(t + 1, buf ^ 1);
    const int key0 = t * kKeys;
    if (MASKED && key0 > wrow + 15) return;
    const char* kt = s_kv[buf][0] + col * kRow;
    const char* vt = s_kv[buf][1] + vbyte;
    v4f s[KT];
#pragma unroll
    for (int u = 0; u < KT; ++u) s[u] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < QS; ++i)
#pragma unroll
      for (int u = 0; u < KT; ++u)
        s[u] = T::mfma16(*reinterpret_cast<const v4u32*>(kt + 16 * u * kRow + 16 * ((4 * i + grp) ^ swk(col))), qf[i], s[u]);
    if constexpr (MASKED) {
#pragma unroll
      for (int u = 0; u < KT; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 16 * u + 4 * grp + r > row) s[u][r] = kNegInf;
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < KT; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[u][r]);
    top = rows_max(top) * p.scale_log2;
    if (__any(top > m + reach)) {
      const float mn = top > m + reach ? (top - reach) + kSlack : m;
      const float c = exp2_hw(m - mn);
      l *= c;
#pragma unroll
      for (int e = 0; e < DB; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[e][r] = CAREFUL ? scaled(acc[e][r], c) : acc[e][r] * c;
      m = mn;
    }
    v4u32 pf[KT / 2];
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < KT; ++u)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float a = exp2_hw(fmaf(s[u][r], p.scale_log2, -m)), b = exp2_hw(fmaf(s[u][r + 1], p.scale_log2, -m));
        sum[0] += a;
        sum[1] += b;
        pf[u / 2][2 * (u % 2) + r / 2] = T::pack(a, b);
      }
    l += sum[0] + sum[1];
#pragma unroll
    for (int c = 0; c < KT / 2; ++c)
#pragma unroll
      for (int e = 0; e < DB; ++e) {
        const char* at = vt + 32 * c * kRow + 16 * ((2 * e + (lane & 3) / 2) ^ swv(vkey));
        const v2u32 lo = read_transposed(at), hi = read_transposed(at + 16 * kRow);
        v4u32 a = {lo.x, lo.y, hi.x, hi.y};
        if constexpr (CAREFUL) {
          v4u32 special;
#pragma unroll
          for (int j = 0; j < 4; ++j) special[j] = only_special<T>(a[j]), a[j] ^= special[j];
          if constexpr (!MASKED) acc[e] = T::mfma16(special, v4u32{kOnes, kOnes, kOnes, kOnes}, acc[e]);
        }
        acc[e] = T::mfma16(a, pf[c], acc[e]);
      }
  };
  int t = 0;
  for (; t < full; ++t) step(t, std::false_type{}, std::false_type{});
  for (; t < tiles; ++t) step(t, std::true_type{}, std::false_type{});
  float odd = 0.0f;  // 0 where all sums are finite, else NaN
#pragma unroll
  for (int e = 0; e < DB; ++e)
#pragma unroll
    for (int r = 0; r < 4; ++r) odd = fmaf(acc[e][r], 0.0f, odd);
  const bool careful = __syncthreads_or(odd != 0.0f);
  if (careful) {
    start();
    for (t = 0; t < full; ++t) step(t, std::false_type{}, std::true_type{});
    for (; t < tiles; ++t) step(t, std::true_type{}, std::true_type{});
  }
  const float sum = rows_sum(l), inv = sum > 0.0f ? 1.0f / sum : __builtin_nanf("");
  if (row >= len) return;
  const int64_t at = (int64_t)(base + row) * p.sot + (int64_t)head * p.soh;
#pragma unroll
  for (int e0 = 0; e0 < DB; e0 += 2) {
    uint32_t w[2][2];  // dims 16 (e0 + k) + 4 grp + 0..3
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = acc[e0 + k][j] * inv;
      const int dim = 16 * (e0 + k) + 4 * grp;
      if (careful) add_masked_specials<T>(o, vh + 2 * dim, svt, full * kKeys, row);
      w[k][0] = T::pack(o[0], o[1]), w[k][1] = T::pack(o[2], o[3]);
      if (!p.out_wide) {
#pragma unroll
        for (int j = 0; j < 4; ++j) store_f32_as(p.out, p.out_dtype, at + dim + j, o[j]);
      }
    }
    if (p.out_wide) {  // 8 dims a lane: neighbouring groups exchange what the other stores
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const auto y = __builtin_amdgcn_permlane16_swap(w[0][j], w[1][j], false, false);
        w[0][j] = y[0], w[1][j] = y[1];
      }
      *reinterpret_cast<v4u32*>(reinterpret_cast<uint16_t*>(p.out) + at + 16 * (e0 + (grp & 1)) + 4 * (grp & 2)) =
          v4u32{w[0][0], w[0][1], w[1][0], w[1][1]};
    }
  }
}

template <typename T>
hipError_t launch_prompt(int64_t D, PromptParams p, hipStream_t st) {
  auto launch = [&](auto kernel, int waves, int rows) {
    p.rows = rows * waves / p.heads;
    // At most this many tiles: each sequence's last one may be part filled.
    p.tiles = (int32_t)std::min<int64_t>(cdiv<int64_t>(p.total, p.rows) + p.n, p.total);
    const int64_t blocks = (int64_t)p.tiles * (p.H / p.heads);
    if (!launchable(blocks, 64 * waves)) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * waves), 0, st, p);
    return hipGetLastError();
  };
  if (D == 64) return launch(prompt_attention_kernel<T, 64>, kWaves, 32);
  if (D == 128) return launch(prompt_attention_kernel<T, 128>, kWaves, 32);
  return launch(prompt_attention_kernel_256<T>, kWaves256, 16);
}

}  // namespace

extern "C" int vxa_prompt_attention(const void* q, int64_t sqt, int64_t sqh, const void* k, int64_t skt, int64_t skh,
                                    const void* v, int64_t svt, int64_t svh, int dtype, const int32_t* starts, int64_t n,
                                    int64_t tokens, float scale, void* out, int out_dtype, int64_t sot, int64_t soh,
                                    int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, vxa_stream_t stream) {
  if (n < 0 || tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return VXA_ERR_ARG;
  if (dtype != VXA_BF16 && dtype != VXA_F16) return VXA_ERR_ARG;
  if (out_dtype != VXA_F32 && out_dtype != VXA_BF16 && out_dtype != VXA_F16) return VXA_ERR_ARG;
  if (num_heads % num_kv_heads != 0) return VXA_ERR_ARG;
  if (n == 0 || tokens == 0) return VXA_OK;
  if (!q || !k || !v || !starts || !out) return VXA_ERR_ARG;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return VXA_ERR_UNSUPPORTED;
  if (num_heads > (1 << 16) || tokens > (1 << 30) || n > (1 << 30)) return VXA_ERR_UNSUPPORTED;
  // Rows are read in 16-byte pieces.
  if ((uintptr_t)q % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || sqt % 8 || sqh % 8 || skt % 8 || skh % 8 || svt % 8 ||
      svh % 8)
    return VXA_ERR_UNSUPPORTED;
  PromptParams p;
  p.q = reinterpret_cast<const uint16_t*>(q), p.sqt = sqt, p.sqh = sqh;
  p.k = reinterpret_cast<const uint16_t*>(k), p.skt = skt, p.skh = skh;
  p.v = reinterpret_cast<const uint16_t*>(v), p.svt = svt, p.svh = svh;
  p.cu = starts;
  p.scale_log2 = scale == 0.0f ? 1.0f : (float)(std::fabs((double)scale) * 1.4426950408889634);
  p.q_and = scale == 0.0f ? 0u : 0xFFFFFFFFu;
  p.q_xor = scale < 0.0f ? 0x80008000u : 0u;
  p.n = (int32_t)n, p.total = (int32_t)tokens, p.H = (int32_t)num_heads, p.G = (int32_t)(num_heads / num_kv_heads);
  p.heads = p.G % 4 == 0 ? 4 : p.G % 2 == 0 ? 2 : 1;
  p.out = out, p.sot = sot, p.soh = soh, p.out_dtype = out_dtype;
  p.out_wide = out_dtype == dtype && (uintptr_t)out % 16 == 0 && sot % 8 == 0 && soh % 8 == 0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const hipError_t err = dtype == VXA_BF16 ? launch_prompt<BF16>(head_dim, p, st) : launch_prompt<FP16>(head_dim, p, st);
  if (err == hipErrorInvalidConfiguration) return VXA_ERR_UNSUPPORTED;
  return err == hipSuccess ? VXA_OK : VXA_ERR_LAUNCH;
}
