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
// for every two elements. K and V go from HBM to registers; LDS holds only the segment's row offsets and scales.
//
// Order. Keys are cut into segments of kSeg. A wave of a workgroup takes the segment's 32-key tiles w, w + 4,
// ... with one running maximum, the 4 waves are merged as ((0 + 2) + (1 + 3)), segments in order. It depends on
// a request's own length only, so its bits do not change with the batch.
//
// Rounding. Scores, maxima, sums and accumulators are fp32. P is split into two 16-bit parts, hi + lo, with one
// MFMA each: P keeps 16 bits (22 in fp16), as the 16-bit output is rounded once from an fp32 sum; the 8-bit
// cache always takes bf16 parts there, because P vscale can leave the fp16 range.

#include <algorithm>

#include "attention_common.h"

namespace {

constexpr int kSeg = 512;    // keys of a segment
constexpr int kTile = 32;    // keys of a wave's step
constexpr int kWaves = 4;
constexpr int kMaxNodes = 64;

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
  int64_t blocks;
  const int32_t* sl;
  const int32_t* qsl;
  const int64_t* mask;
  float scale_log2;
  int32_t n, total, KV, G, ns, row_blocks, max_nodes, max_len;
  float* mp;  // [total][H][ns]
  float* lp;
  float* ap;  // [total][H][ns][D]
  void* out;
  int64_t sot, soh;
  int32_t out_dtype;
};

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

// T: the query's element type; INT8: the cache's; NQ: 16-row blocks of a workgroup.
template <typename T, bool INT8, int D, int NQ>
__global__ __launch_bounds__(64 * kWaves) void tree_partial_kernel(TreeParams p) {
  using PT = std::conditional_t<INT8, BF16, T>;  // the type of P and V
  constexpr int QS = D / 32;                     // MFMA steps over the head's dims
  constexpr int DPL = D / 16;                    // dims of a lane in V, and 16-dim blocks of O^T
  constexpr int KW = INT8 ? D / 16 : D / 8;      // dwords of a lane's share of a key
  constexpr int VW = INT8 ? DPL / 4 : DPL / 2;   // dwords of a lane's dims of one key's value
  __shared__ int64_t s_koff[kSeg], s_voff[kSeg];
  __shared__ float s_ks[INT8 ? kSeg : 1], s_vs[INT8 ? kSeg : 1];
  __shared__ float s_m[2][16 * NQ], s_l[2][16 * NQ];
  __shared__ float s_acc[2][DPL * NQ][4][64];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15;
  const int grp = lane >> 4;

  int64_t id = blockIdx.x;
  const int rb = (int)(id % p.row_blocks);
  id /= p.row_blocks;
  const int g = (int)(id % p.KV);
  id /= p.KV;
  const int b = (int)(id % p.n);
  const int seg = (int)(id / p.n);
  const Request rq = request_of(p, b);
  const int rows = rq.T * p.G;
  const int row0 = rb * 16 * NQ;
  if (row0 >= rows) return;
  const int H = p.KV * p.G;
  if (rq.bad) {
    if (seg == 0 && rb == 0)
      for (int64_t i = threadIdx.x; i < (int64_t)rows * D; i += 64 * kWaves) {
        const int row = (int)(i / D);
        store_f32_as(p.out, p.out_dtype,
                     (int64_t)(rq.q0 + row / p.G) * p.sot + (int64_t)(g * p.G + row % p.G) * p.soh + i % D, __builtin_nanf(""));
      }
    return;
  }
  const int start = seg * kSeg;
  const int end = min(start + kSeg, rq.L);
  if (start >= end) return;
  const int ctx = rq.L - rq.T;

  // Row offsets (and scales) of the segment's keys; keys past its end repeat the last one. A page that the cache
  // does not have makes the request's rows NaN.
  bool bad_page = false;
  for (int i = threadIdx.x; i < kSeg; i += 64 * kWaves) {
    const int key = min(start + i, end - 1);
    const int pg = (int)((uint32_t)key / (uint32_t)p.page);
    const int off = key - pg * p.page;
    int64_t block = p.bt[(int64_t)b * p.sbt + pg];
    if (block < 0 || block >= p.blocks) {
      bad_page = true;
      block = 0;
    }
    s_koff[i] = block * p.skb + (int64_t)off * p.skp;
    s_voff[i] = block * p.svb + (int64_t)off * p.svp;
    if constexpr (INT8) {
      s_ks[i] = p.ks[block * p.sksb + (int64_t)off * p.sksp + (int64_t)g * p.sksh] * p.scale_log2;
      s_vs[i] = p.vs[block * p.svsb + (int64_t)off * p.svsp + (int64_t)g * p.svsh];
    }
  }

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
  bad_page = __syncthreads_or(bad_page);

  const char* kbase = p.kc + (int64_t)g * p.skh + 16 * grp;
  const char* vbase = p.vc + (int64_t)g * p.svh + VW * 4 * col;
  Words<KW> kr[2];
  Words<VW> vr[8];
  auto load = [&](int tile) {  // key slots of a lane: 4 grp + j of each half tile
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* k = kbase + s_koff[tile * kTile + 16 * h + col];
#pragma unroll
      for (int c = 0; c < KW / 4; ++c) {
        const Words<4> w = load_words<4>(k + 64 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) kr[h].w[4 * c + i] = w.w[i];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) vr[4 * h + j] = load_words<VW>(vbase + s_voff[tile * kTile + 16 * h + 4 * grp + j]);
    }
  };

  float m[NQ], l[NQ];
  v4f acc[NQ][DPL];
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    m[t] = kLowest;
    l[t] = 0.0f;
#pragma unroll
    for (int e = 0; e < DPL; ++e) acc[t][e] = v4f{0, 0, 0, 0};
  }

  const int tiles = (end - start + kTile - 1) / kTile;
  for (int tile = wave; tile < tiles; tile += kWaves) {
    load(tile);
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
    const bool drafted = key0 + kTile > ctx;  // the tile holds drafted keys, or ends past the last key
    uint32_t phi[NQ][4], plo[NQ][4], flag[NQ][4];
    const v4f one = {p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2};
    v4f ks[2] = {one, one}, vs[2];
    if constexpr (INT8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[h] = *reinterpret_cast<const v4f*>(&s_ks[tile * kTile + 16 * h + 4 * grp]);
        vs[h] = *reinterpret_cast<const v4f*>(&s_vs[tile * kTile + 16 * h + 4 * grp]);
      }
    }
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      uint32_t live = 0xFF;  // bit 4 h + j: this row attends to the key
      if (drafted) {
        live = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int d = key0 + 16 * h + 4 * grp + j - ctx;
            const bool on = d < 0 || (d < 64 && ((seen[t] >> (d & 63)) & 1));
            live |= on ? 1u << (4 * h + j) : 0u;
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
      if (__any(top > m[t])) {
        const float mn = fmaxf(m[t], top);
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
        if constexpr (!INT8)
          flag[t][i] = ((live >> (2 * i)) & 1 ? (uint32_t)PT::kOne : 0u) | ((live >> (2 * i + 1)) & 1 ? (uint32_t)PT::kOne << 16 : 0u);
      }
    }

    // Values of keys that some rows do not attend to may be infinities or NaN, and 0 times those is NaN: where a
    // tile with masked keys holds any, they enter the product as 0 and are added to the rows that attend to them.
    bool special = false;
    if constexpr (!INT8) {
      if (drafted) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < VW; ++i) special |= any_special<PT>(vr[k].w[i]);
        special = __any(special);
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
      if constexpr (!INT8) {
        if (special) {
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
      }
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        acc[t][e] = PT::mfma16(a, v4u32{phi[t][0], phi[t][1], phi[t][2], phi[t][3]}, acc[t][e]);
        acc[t][e] = PT::mfma16(a, v4u32{plo[t][0], plo[t][1], plo[t][2], plo[t][3]}, acc[t][e]);
      }
    });
  }
#pragma unroll
  for (int t = 0; t < NQ; ++t) l[t] = rows_sum(l[t]);

  // Merge the waves: 2 and 3 into 0 and 1, then 1 into 0.
  auto give = [&](int slot) {
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      if (grp == 0) {
        s_m[slot][16 * t + col] = m[t];
        s_l[slot][16 * t + col] = l[t];
      }
#pragma unroll
      for (int e = 0; e < DPL; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_acc[slot][t * DPL + e][r][lane] = acc[t][e][r];
    }
  };
  auto take = [&](int slot) {
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      const float mo = s_m[slot][16 * t + col], lo = s_l[slot][16 * t + col];
      const float mn = fmaxf(m[t], mo);
      const float c0 = exp2_hw(m[t] - mn), c1 = exp2_hw(mo - mn);
      l[t] = fmaf(l[t], c0, lo * c1);
      m[t] = mn;
#pragma unroll
      for (int e = 0; e < DPL; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][e][r] = fmaf(acc[t][e][r], c0, s_acc[slot][t * DPL + e][r][lane] * c1);
    }
  };
  if (wave >= 2) give(wave - 2);
  __syncthreads();
  if (wave < 2) take(wave);
  __syncthreads();
  if (wave == 1) give(0);
  __syncthreads();
  if (wave != 0) return;
  take(0);

  const bool alone = rq.L <= kSeg;
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    const int row = row0 + 16 * t + col;
    if (row >= rows) continue;
    const int node = row / p.G, head = g * p.G + row % p.G;
    if (bad_page) l[t] = __builtin_nanf("");
    if (alone) {
      const bool nothing = ctx == 0 && seen[t] == 0;
      const int64_t at = (int64_t)(rq.q0 + node) * p.sot + (int64_t)head * p.soh;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < DPL; ++e)
          store_f32_as(p.out, p.out_dtype, at + (4 * grp + r) * DPL + e, nothing && !bad_page ? 0.0f : acc[t][e][r] / l[t]);
    } else {
      const int64_t part = ((int64_t)(rq.q0 + node) * H + head) * p.ns + seg;
      if (grp == 0) {
        p.mp[part] = m[t];
        p.lp[part] = l[t];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < DPL; ++e) p.ap[part * D + (4 * grp + r) * DPL + e] = acc[t][e][r];
    }
  }
}

// Joins a row's segments in order: a wave per (node, head). A row longer than a segment attends to its context, so
// its sum is not empty.
template <int D>
__global__ __launch_bounds__(64 * kWaves) void tree_merge_kernel(TreeParams p) {
  constexpr int DPW = D / 64;
  const int lane = threadIdx.x & 63;
  const int H = p.KV * p.G;
  const int64_t id = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int head = (int)(id % H);
  const int64_t bn = id / H;
  const int b = (int)(bn / p.max_nodes), node = (int)(bn % p.max_nodes);
  if (b >= p.n) return;
  const Request rq = request_of(p, b);
  if (rq.bad || node >= rq.T || rq.L <= kSeg) return;
  const int segs = (rq.L + kSeg - 1) / kSeg;
  const int64_t part = ((int64_t)(rq.q0 + node) * H + head) * p.ns;
  float top = kLowest;
  for (int s = lane; s < segs; s += 64) top = fmaxf(top, p.mp[part + s]);
#pragma unroll
  for (int x = 1; x < 64; x *= 2) top = fmaxf(top, shfl_xor_f32(top, x));
  float l = 0.0f, a[DPW];
#pragma unroll
  for (int j = 0; j < DPW; ++j) a[j] = 0.0f;
#pragma unroll 8
  for (int s = 0; s < segs; ++s) {
    const float c = exp2_hw(p.mp[part + s] - top);
    l = fmaf(p.lp[part + s], c, l);
#pragma unroll
    for (int j = 0; j < DPW; ++j) a[j] = fmaf(p.ap[(part + s) * D + DPW * lane + j], c, a[j]);
  }
  const int64_t at = (int64_t)(rq.q0 + node) * p.sot + (int64_t)head * p.soh;
#pragma unroll
  for (int j = 0; j < DPW; ++j) store_f32_as(p.out, p.out_dtype, at + DPW * lane + j, a[j] / l);
}

int row_blocks16(int64_t rows, int64_t D) { return rows <= 16 ? 1 : rows <= 32 || D == 256 ? 2 : 4; }

template <typename T, bool INT8, int D>
hipError_t launch_tree(TreeParams p, hipStream_t st) {
  const int64_t rows = (int64_t)p.max_nodes * p.G;
  const int nq = row_blocks16(rows, D);
  p.row_blocks = (int32_t)cdiv<int64_t>(rows, 16 * nq);
  const int64_t blocks = (int64_t)p.row_blocks * p.KV * p.n * p.ns;
  const int64_t merges = cdiv<int64_t>((int64_t)p.n * p.max_nodes * p.KV * p.G, kWaves);
  if (blocks > 0x7FFFFFFFLL || merges > 0x7FFFFFFFLL) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks), threads(64 * kWaves);
  if (nq == 1) {
    hipLaunchKernelGGL((tree_partial_kernel<T, INT8, D, 1>), grid, threads, 0, st, p);
  } else if (nq == 2) {
    hipLaunchKernelGGL((tree_partial_kernel<T, INT8, D, 2>), grid, threads, 0, st, p);
  } else {
    if constexpr (D < 256) hipLaunchKernelGGL((tree_partial_kernel<T, INT8, D, 4>), grid, threads, 0, st, p);
  }
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.ns == 1) return err;
  hipLaunchKernelGGL((tree_merge_kernel<D>), dim3((unsigned)merges), threads, 0, st, p);
  return hipGetLastError();
}

template <typename T, bool INT8>
hipError_t dispatch_dim(int64_t D, const TreeParams& p, hipStream_t st) {
  if (D == 64) return launch_tree<T, INT8, 64>(p, st);
  if (D == 128) return launch_tree<T, INT8, 128>(p, st);
  return launch_tree<T, INT8, 256>(p, st);
}

int64_t num_segments(int64_t keys) { return std::max<int64_t>(1, cdiv<int64_t>(keys, kSeg)); }

}  // namespace

extern "C" int vxa_tree_decode_workspace(int64_t tokens, int64_t num_heads, int64_t head_dim, int64_t max_seq_len,
                                         size_t* ws_bytes) {
  if (tokens < 0 || num_heads <= 0 || head_dim <= 0 || max_seq_len < 0 || !ws_bytes) return VXA_ERR_ARG;
  const int64_t ns = num_segments(max_seq_len);
  *ws_bytes = ns > 1 ? (size_t)tokens * num_heads * ns * (head_dim + 2) * sizeof(float) : 0;
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
  const int64_t ns = num_segments(max_seq_len);
  size_t need = 0;
  vxa_tree_decode_workspace(tokens, num_heads, head_dim, max_seq_len, &need);
  if (need > 0 && (!ws || ws_bytes < need)) return VXA_ERR_WORKSPACE;

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
  p.ns = (int32_t)ns, p.row_blocks = 1, p.max_nodes = (int32_t)max_nodes, p.max_len = (int32_t)max_seq_len;
  const int64_t parts = tokens * num_heads * ns;
  float* w = reinterpret_cast<float*>(ws);
  p.mp = w, p.lp = ns > 1 ? w + parts : nullptr, p.ap = ns > 1 ? w + 2 * parts : nullptr;
  p.out = out, p.sot = sot, p.soh = soh, p.out_dtype = out_dtype;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipError_t err;
  if (q_dtype == VXA_BF16)
    err = int8 ? dispatch_dim<BF16, true>(head_dim, p, st) : dispatch_dim<BF16, false>(head_dim, p, st);
  else
    err = int8 ? dispatch_dim<FP16, true>(head_dim, p, st) : dispatch_dim<FP16, false>(head_dim, p, st);
  if (err == hipErrorInvalidConfiguration) return VXA_ERR_UNSUPPORTED;
  return err == hipSuccess ? VXA_OK : VXA_ERR_LAUNCH;
}
