// Causal attention over whole prompts, packed one after the other (gfx950).
//
//   o_i = sum_{j <= i} p_ij v_j / sum_{j <= i} p_ij,   p_ij = exp(scale q_i.k_j - max_j scale q_i.k_j)
// for every row i of every sequence, with groups of G = H / KV query heads on one key/value head.
//
// Work split. A workgroup of 4 waves computes 128 rows of one (sequence, head), 32 rows a wave, and walks the
// keys up to its last row in tiles of 64 (32 at 256 dims) with one running maximum and sum: every score is computed once and kept
// in registers. A wave's rows are the columns of S^T = K Q^T (32 x 32 x 16 MFMAs) and of O^T = V^T P^T, so a lane
// holds scores of one row only, and with the keys of the second product taken in the order in which the first one
// leaves them in the lane, P goes from one product to the other without leaving the lane. The tiles of K and V go
// through registers into LDS, V transposed on the way (a byte permute for two elements), two tiles in turn.
// A row's order of operations depends on its place in its sequence alone, not on the batch.
//
// Rounding. Scores, maxima, sums and accumulators are fp32; P is rounded to the 16-bit element type for the second
// product, an error of the size of the output's own rounding, while its sum takes the fp32 values.

#include <algorithm>
#include <cmath>

#include "attention_common.h"

namespace {

constexpr int kRows = 128;  // query rows of a workgroup
constexpr int kThreads = 256;

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
  void* out;
  int64_t sot, soh;
  int32_t out_dtype;
};

// The sequence and rows of tile `tile`, counted over the sequences' tiles of kRows rows in order.
struct Tile {
  int base, len, row0;  // first packed row of the sequence, its length (0: no such tile), the tile's first row in it
};
__device__ inline Tile find_tile(const PromptParams& p, int tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int j0 = 0; j0 < p.n; j0 += 64) {
    const int j = j0 + lane;
    int lo = 0, len = 0;
    if (j < p.n) {
      lo = max(p.cu[j], 0);
      len = max(min(p.cu[j + 1], p.total) - lo, 0);
    }
    const int mine = (len + kRows - 1) / kRows;
    int sum = mine;  // inclusive over the lanes
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const int up = __shfl_up(sum, x);
      if (lane >= x) sum += up;
    }
    const uint64_t hit = __ballot(before + sum > tile);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      const int first = before + __shfl(sum - mine, at);
      return Tile{__shfl(lo, at), __shfl(len, at), (tile - first) * kRows};
    }
    before += __shfl(sum, 63);
  }
  return Tile{0, 0, 0};
}

// Values of keys that some rows do not attend to may be infinities or NaN, and 0 times those is NaN. In a tile with
// masked keys they enter the product as 0, and what they add is added to the rows that attend to them. a: 8 keys
// (key0 + j % 4 + 8 (j / 4)) of one dim.
template <typename T>
__device__ inline void add_special(v4u32& a, int key0, int row, v16f& acc) {
  if (!__any(any_special<T>(a[0]) || any_special<T>(a[1]) || any_special<T>(a[2]) || any_special<T>(a[3]))) return;
  v4u32 plus, minus, seen;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    plus[i] = special_flags<T, 0>(a[i]);
    minus[i] = special_flags<T, 1>(a[i]);
    a[i] = only_finite<T>(a[i]);
    const int key = key0 + 2 * (i % 2) + 8 * (i / 2);
    seen[i] = (key <= row ? (uint32_t)T::kOne : 0u) | (key + 1 <= row ? (uint32_t)T::kOne << 16 : 0u);
  }
  const v16f zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  const v16f up = T::mfma32(plus, seen, zero);
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (up[r] > 0.0f) acc[r] += __builtin_huge_valf();
  const v16f down = T::mfma32(minus, seen, zero);
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (down[r] > 0.0f) acc[r] += kNegInf;
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void prompt_kernel(PromptParams p) {
  constexpr int kKeys = D == 256 ? 32 : 64;  // keys of a tile: at 256 dims 64 keys leave no registers for the loads ahead
  constexpr int KU = kKeys / 32, KCH = kKeys / 8;
  constexpr int QS = D / 16;   // MFMA steps over the head's dims
  constexpr int DB = D / 32;   // 32-dim blocks of O^T
  constexpr int KC = D / 8;    // 16-byte chunks of a key
  constexpr int KL = kKeys * KC / kThreads;             // chunks of K a thread stages
  constexpr int VD = D == 64 ? 2 : 4;                   // dims of a unit of V, 8 keys
  constexpr int VU = kKeys / 8 * (D / VD) / kThreads;   // units of V a thread stages
  __shared__ v4u32 s_k[2][kKeys * KC];   // [key][chunk ^ key]
  __shared__ v4u32 s_v[2][D * KCH];        // [dim][chunk of 8 keys, swizzled]

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;

  // Workgroups of one KV head run on one XCD, longest rows first.
  const int x = (int)(blockIdx.x % p.H);
  const int head = p.H % 8 == 0 ? (x % 8) * (p.H / 8) + x / 8 : x;
  const Tile tile = find_tile(p, p.tiles - 1 - (int)(blockIdx.x / p.H));
  if (tile.len == 0) return;
  const int base = __builtin_amdgcn_readfirstlane(tile.base);
  const int len = __builtin_amdgcn_readfirstlane(tile.len);
  const int row0 = __builtin_amdgcn_readfirstlane(tile.row0);
  const uint16_t* kh = p.k + (int64_t)base * p.skt + (int64_t)(head / p.G) * p.skh;
  const uint16_t* vh = p.v + (int64_t)base * p.svt + (int64_t)(head / p.G) * p.svh;

  const int wrow = row0 + 32 * wave;  // the wave's first row
  const int row = wrow + col;
  v4u32 qf[QS];
  {
    const uint16_t* q = p.q + (int64_t)(base + min(row, len - 1)) * p.sqt + (int64_t)head * p.sqh + 8 * half;
#pragma unroll
    for (int i = 0; i < QS; ++i) qf[i] = (*reinterpret_cast<const v4u32*>(q + 16 * i) & p.q_and) ^ p.q_xor;
  }

  const int last = min(row0 + kRows, len);              // keys of the workgroup
  const int tiles = (last + kKeys - 1) / kKeys;
  v4u32 kr[KL];
  uint32_t vr[VU][8][VD / 2];
  // V's slots: chunk c of a tile holds, for j = 0..7, the key 32 (c / 4) + 16 (c / 2 % 2) + 4 (c % 2) + (j % 4) + 8 (j / 4),
  // which is the order in which an S^T tile's registers hold a lane's keys.
  auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int u = threadIdx.x + i * kThreads;
      kr[i] = *reinterpret_cast<const v4u32*>(kh + (int64_t)min(t * kKeys + u / KC, len - 1) * p.skt + 8 * (u % KC));
    }
#pragma unroll
    for (int i = 0; i < VU; ++i) {
      const int u = threadIdx.x + i * kThreads;
      const int c = u / (D / VD), d = VD * (u % (D / VD));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = t * kKeys + 32 * (c / 4) + 16 * (c / 2 % 2) + 4 * (c % 2) + j % 4 + 8 * (j / 4);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(vh + (int64_t)min(key, len - 1) * p.svt + d);
        if constexpr (VD == 2) {
          vr[i][j][0] = *src;
        } else {
          const v2u32 w = *reinterpret_cast<const v2u32*>(src);
          vr[i][j][0] = w.x, vr[i][j][1] = w.y;
        }
      }
    }
  };
  auto vslot = [](int d, int c) { return d * KCH + (c ^ ((d ^ (d >> 3)) & (KCH - 1))); };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int u = threadIdx.x + i * kThreads;
      const int key = u / KC, c = u % KC;
      s_k[buf][key * KC + (c ^ (key & (KC < 16 ? 7 : 15)))] = kr[i];
    }
#pragma unroll
    for (int i = 0; i < VU; ++i) {
      const int u = threadIdx.x + i * kThreads;
      const int c = u / (D / VD), d = VD * (u % (D / VD));
#pragma unroll
      for (int e = 0; e < VD; ++e) {
        v4u32 w;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = __builtin_amdgcn_perm(vr[i][2 * j + 1][e / 2], vr[i][2 * j][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
        s_v[buf][vslot(d + e, c)] = w;
      }
    }
  };

  float m = kLowest, l = 0.0f;
  v16f acc[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) acc[i] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

  load(0);
  store(0);
  for (int t = 0; t < tiles; ++t) {
    const int buf = t & 1;
    __syncthreads();
    if (t + 1 < tiles) load(t + 1);
    const int key0 = t * kKeys;
    if (key0 <= wrow + 31) {  // some row of the wave attends to the tile
      v16f s[KU];
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        s[u] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        const int key = 32 * u + col;
#pragma unroll
        for (int i = 0; i < QS; ++i)
          s[u] = T::mfma32(s_k[buf][key * KC + ((2 * i + half) ^ (key & (KC < 16 ? 7 : 15)))], qf[i], s[u]);
      }
      const bool masked = key0 + kKeys - 1 > wrow;
      if (masked) {
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
      if (__any(top > m)) {
        const float mn = fmaxf(m, top);
        const float c = exp2_hw(m - mn);
        l *= c;
#pragma unroll
        for (int i = 0; i < DB; ++i) acc[i] = acc[i] * c;
        m = mn;
      }
      v4u32 pf[2 * KU];
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float a = exp2_hw(fmaf(s[u][r], p.scale_log2, -m)), b = exp2_hw(fmaf(s[u][r + 1], p.scale_log2, -m));
          l += a;
          l += b;
          pf[2 * u + r / 8][r % 8 / 2] = T::pack(a, b);
        }
#pragma unroll
      for (int c = 0; c < 2 * KU; ++c)
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          v4u32 a = s_v[buf][vslot(32 * i + col, 2 * c + half)];
          if (masked) add_special<T>(a, key0 + 32 * (c / 2) + 16 * (c % 2) + 4 * half, row, acc[i]);
          acc[i] = T::mfma32(a, pf[c], acc[i]);
        }
    }
    if (t + 1 < tiles) store(buf ^ 1);
  }
  float la = l, lb = l;
  swap32(la, lb);
  l = la + lb;
  if (row >= len) return;
  const int64_t at = (int64_t)(base + row) * p.sot + (int64_t)head * p.soh;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      store_f32_as(p.out, p.out_dtype, at + 32 * i + (r & 3) + 8 * (r >> 2) + 4 * half, acc[i][r] / l);
}

template <typename T>
hipError_t launch_prompt(int64_t D, const PromptParams& p, hipStream_t st) {
  const int64_t blocks = (int64_t)p.tiles * p.H;
  if (blocks > 0x7FFFFFFFLL) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks), threads(kThreads);
  if (D == 64)
    hipLaunchKernelGGL((prompt_kernel<T, 64>), grid, threads, 0, st, p);
  else if (D == 128)
    hipLaunchKernelGGL((prompt_kernel<T, 128>), grid, threads, 0, st, p);
  else
    hipLaunchKernelGGL((prompt_kernel<T, 256>), grid, threads, 0, st, p);
  return hipGetLastError();
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
  // At most this many tiles: each sequence's last one may be part filled.
  p.tiles = (int32_t)std::min<int64_t>(cdiv<int64_t>(tokens, kRows) + n, tokens);
  p.out = out, p.sot = sot, p.soh = soh, p.out_dtype = out_dtype;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const hipError_t err = dtype == VXA_BF16 ? launch_prompt<BF16>(head_dim, p, st) : launch_prompt<FP16>(head_dim, p, st);
  if (err == hipErrorInvalidConfiguration) return VXA_ERR_UNSUPPORTED;
  return err == hipSuccess ? VXA_OK : VXA_ERR_LAUNCH;
}
