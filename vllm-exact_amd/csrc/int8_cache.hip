// A paged KV cache in 8 bits (gfx950): quantising new tokens as they are written, and reading ranges back.
//
// Each (token, KV head) has one scale for its key and one for its value: top = max |x| over the head's D
// elements, scale = top / 127, q = round(127 x / top) to the nearest whole number, ties to even, so q lies in
// [-127, 127] and stands for q * scale. 127 x is exact in fp32 for 16-bit x and the quotient of two such
// inputs is either a half exactly or further from it than its fp32 rounding, so q is the nearest whole number
// of the quotient itself. A row with an infinity or NaN gets q = 0 and the scale NaN: it reads back as NaN.
// A row of zeros gets the scale 0.
//
// Both kernels move each byte once and are bound by HBM, and by the latency of a few dependent loads at a decode step's
// sizes. Measured: 16 contexts of up to 8192 tokens (8 heads of 128 dims) read back as bf16 in 134 us, 4.6 TB/s, where a
// large copy reaches 4.9; 64 tokens written in 3.6 us and read back in 3.8.

#include <algorithm>

#include "attention_common.h"

namespace {

struct CacheWrite {
  const void* x[2];       // key, value rows
  int64_t sxt[2], sxh[2];
  int8_t* c[2];           // key, value caches
  int64_t scb[2], scp[2], sch[2];
  float* s[2];            // key, value scales
  int64_t ssb[2], ssp[2], ssh[2];
  const int64_t* slots;
  int64_t tokens;
  int32_t KV, page;
  Divisor by_token, by_page;  // by a token's units, by the tokens of a page
  int64_t rows_total;     // slots of the cache: blocks * page
  int32_t per_group;      // tokens of a workgroup
};

// The largest value of the LPR lanes of a row, in each of them.
template <int CTRL>
__device__ inline uint32_t max_with(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false));
}
template <int LPR>
__device__ inline uint32_t row_max(uint32_t x) {
  x = max_with<0xB1>(x);   // lane ^ 1
  x = max_with<0x4E>(x);   // lane ^ 2
  x = max_with<0x141>(x);  // the other end of 8 lanes
  if constexpr (LPR >= 16) x = max_with<0x140>(x);  // ... of 16
  if constexpr (LPR == 32) x = max(x, (uint32_t)__shfl_xor((int)x, 16));
  return x;
}

// A unit is 8 elements of a row; a token's units are those of its heads in turn. The lanes of a row are neighbours in a wave.
// A workgroup takes per_group tokens' keys or values, a unit for every thread where a token has no more than that: several
// loads ahead in a thread were slower (10,000 tokens of 2 heads of 256 dims: 14 us with four, 11 with one).
template <int DTYPE, int D, bool VEC>
__global__ __launch_bounds__(256) void int8_write_kernel(CacheWrite p) {
  constexpr int LPR = D / 8;
  const int per_token = p.KV * LPR, w = blockIdx.y;
  const int64_t t0 = (int64_t)blockIdx.x * p.per_group;
  const int units = (int)min((int64_t)p.per_group, p.tokens - t0) * per_token;
  const int lane = threadIdx.x & (LPR - 1);
  for (int u = threadIdx.x; u < units; u += 256) {  // a row's lanes are all in or all out
    const int tok = divide(u, p.by_token), h = (u - tok * per_token) / LPR;
    const int64_t slot = p.slots[t0 + tok];
    const int64_t at = (t0 + tok) * p.sxt[w] + (int64_t)h * p.sxh[w] + 8 * lane;
    float x[8];
    if constexpr (DTYPE == VXA_F32) {
      const float* src = reinterpret_cast<const float*>(p.x[w]) + at;
      if constexpr (VEC) {
        const v4f a = *reinterpret_cast<const v4f*>(src), b = *reinterpret_cast<const v4f*>(src + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = src[j];
      }
    } else {
      using T = std::conditional_t<DTYPE == VXA_BF16, BF16, FP16>;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(p.x[w]) + at;
      if constexpr (VEC) {
        const v4u32 a = *reinterpret_cast<const v4u32*>(src);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const v2f f = T::unpack(a[j]);
          x[2 * j] = f[0], x[2 * j + 1] = f[1];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = T::to_f32(src[j]);
      }
    }
    // The largest magnitude as bits: NaN and infinities order above every finite value.
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    top = row_max<LPR>(top);
    if (slot < 0 || slot >= p.rows_total) continue;
    const float ftop = __uint_as_float(top);
    const bool special = top >= 0x7F800000u;
    const int32_t block = divide((int32_t)slot, p.by_page);
    const int32_t off = (int32_t)slot - block * p.page;
    if (lane == 0)
      p.s[w][(int64_t)block * p.ssb[w] + (int64_t)off * p.ssp[w] + (int64_t)h * p.ssh[w]] = special ? __builtin_nanf("") : ftop / 127.0f;
    // x times 127 / top is off by at most 2^-16; adding 1.5 2^23 rounds it to a whole number in the low byte. Next to a half,
    // and where 127 / top overflows, the quotient decides.
    constexpr float kWhole = 12582912.0f;
    const float mul = 127.0f / ftop;
    uint32_t q[8];
    float away = 0.0f;  // from the whole numbers
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float r = x[j] * mul, a = r + kWhole;
      q[j] = __float_as_uint(a);
      away = fmaxf(away, fabsf(r - (a - kWhole)));
    }
    if (away > 0.4999f || ftop < 0x1p-110f || special) {
      // Above 2^100 the products 127 x could overflow: both sides are scaled by 2^-32, which rounds nothing that counts.
      const float down = ftop > 0x1p100f ? 0x1p-32f : 1.0f;
      const float div = ftop * down;
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = special || top == 0 ? 0u : (uint32_t)(int)rintf((x[j] * down) * 127.0f / div);
    }
    uint32_t out[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t lo = __builtin_amdgcn_perm(q[4 * j + 1], q[4 * j], 0x0C0C0400u);
      out[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[4 * j + 3], q[4 * j + 2], 0x0C0C0400u), lo, 0x05040100u);
    }
    int8_t* dst = p.c[w] + (int64_t)block * p.scb[w] + (int64_t)off * p.scp[w] + (int64_t)h * p.sch[w] + 8 * lane;
    *reinterpret_cast<v2u32*>(dst) = v2u32{out[0], out[1]};
  }
}

struct CacheRead {
  const int8_t* c[2];
  int64_t scb[2], scp[2], sch[2];
  const float* s[2];
  int64_t ssb[2], ssp[2], ssh[2];
  const int32_t* bt;
  int64_t sbt;
  const int32_t* cu;     // [n + 1] packed starts of the sequences' rows
  const int32_t* first;  // [n] or null: the first token read of each sequence
  int64_t n, total;      // sequences, packed rows
  int32_t KV, page, cols;  // cols: block-table entries of a sequence
  Divisor by_token, by_page;  // by a token's units, by the tokens of a page
  int32_t per_group;      // tokens of a workgroup
  int64_t blocks;
  void* o[2];
  int64_t sot[2], soh[2];
};

constexpr int kReadTokens = 16;  // tokens of a workgroup, at most

// A workgroup reads up to 16 packed tokens, all heads, keys and values: whole lines of the cache's pages (a page's tokens follow
// each other) and whole lines of the output (a token's heads do). A unit is 16 bytes of output; a token's units are those
// of its heads in turn, keys first, then values. A thread has kReadUnits units on their way together.
constexpr int kReadUnits = 4;
constexpr int64_t kNone = -0x7FFFFFFFFFFFFFFFLL;  // no place: a unit past the end or in no sequence
template <int OUT, int D>
__global__ __launch_bounds__(256) void int8_read_kernel(CacheRead p) {
  constexpr int EPU = OUT == VXA_F32 ? 4 : 8, LPR = D / EPU;  // elements of a unit, units of a row
  __shared__ int32_t s_block[kReadTokens], s_off[kReadTokens];
  const int64_t t0 = (int64_t)blockIdx.x * p.per_group;
  if (threadIdx.x < 64) {
    // A token's sequence is the number of sequences that end at or before it: lanes compare 64 ends at a time.
    const int lane = threadIdx.x;
    int seq = 0;
    for (int64_t j0 = 0; j0 < p.n; j0 += 64) {
      const int64_t j = j0 + lane;
      const int32_t end = j < p.n ? p.cu[j + 1] : 0x7FFFFFFF;
      for (int i = 0; i < p.per_group; ++i) {
        const int c = __popcll(__ballot((int64_t)end <= t0 + i));
        if (lane == i) seq += c;
      }
    }
    if (lane < p.per_group) {
      int32_t block = -1, off = 0;  // -1: the row is in no sequence, -2: its page does not exist
      const int64_t in_seq = t0 + lane < p.total && seq < p.n ? t0 + lane - p.cu[seq] : -1;
      if (in_seq >= 0) {
        const int64_t pos = in_seq + (p.first != nullptr ? p.first[seq] : 0);
        block = -2;
        if (pos >= 0 && pos < (int64_t)p.cols * p.page) {
          const int32_t pg = divide((int)pos, p.by_page);
          const int32_t id = p.bt[(int64_t)seq * p.sbt + pg];
          off = (int32_t)pos - pg * p.page;
          if (id >= 0 && id < p.blocks) block = id;
        }
      }
      s_block[lane] = block;
      s_off[lane] = off;
    }
  }
  __syncthreads();
  const int per_token = p.KV * LPR, units = p.per_group * per_token;
  static_for<2>([&](auto wc) {
    constexpr int wh = decltype(wc)::value;
    for (int u0 = threadIdx.x; u0 < units; u0 += 256 * kReadUnits) {
      uint32_t w[kReadUnits][EPU / 4];
      float scale[kReadUnits];
      int64_t at[kReadUnits];
#pragma unroll
      for (int n = 0; n < kReadUnits; ++n) {
        const int u = u0 + 256 * n;
        at[n] = kNone;
        if (u >= units) continue;
        const int i = divide(u, p.by_token), rest = u - i * per_token;
        const int lane = rest & (LPR - 1), h = rest / LPR;
        const int32_t block = s_block[i], off = s_off[i];
        if (block == -1) continue;
        at[n] = (t0 + i) * p.sot[wh] + (int64_t)h * p.soh[wh] + EPU * lane;
        scale[n] = __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < EPU / 4; ++j) w[n][j] = 0;
        if (block >= 0) {
          scale[n] = p.s[wh][(int64_t)block * p.ssb[wh] + (int64_t)off * p.ssp[wh] + (int64_t)h * p.ssh[wh]];
          const int8_t* src = p.c[wh] + (int64_t)block * p.scb[wh] + (int64_t)off * p.scp[wh] + (int64_t)h * p.sch[wh] + EPU * lane;
          if constexpr (EPU == 8) {
            const v2u32 x = *reinterpret_cast<const v2u32*>(src);
            w[n][0] = x.x, w[n][1] = x.y;
          } else {
            w[n][0] = *reinterpret_cast<const uint32_t*>(src);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < kReadUnits; ++n) {
        if (at[n] == kNone) continue;
        float f[EPU];
#pragma unroll
        for (int j = 0; j < EPU; ++j) f[j] = (float)(int8_t)(w[n][j / 4] >> (8 * (j % 4))) * scale[n];
        if constexpr (OUT == VXA_F32) {
          *reinterpret_cast<v4f*>(reinterpret_cast<float*>(p.o[wh]) + at[n]) = v4f{f[0], f[1], f[2], f[3]};
        } else {
          using T = std::conditional_t<OUT == VXA_BF16, BF16, FP16>;
          *reinterpret_cast<v4u32*>(reinterpret_cast<uint16_t*>(p.o[wh]) + at[n]) =
              v4u32{T::pack(f[0], f[1]), T::pack(f[2], f[3]), T::pack(f[4], f[5]), T::pack(f[6], f[7])};
        }
      }
    }
  });
}

template <int DTYPE, int D>
hipError_t launch_write(CacheWrite p, bool vec, hipStream_t st) {
  const int64_t per_token = p.KV * (D / 8);
  p.per_group = (int32_t)std::max<int64_t>(1, 256 / per_token);
  p.by_token = make_divisor(per_token);
  const int64_t blocks = cdiv<int64_t>(p.tokens, p.per_group);
  if (!launchable(blocks, 256)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks, 2), threads(256);
  if (vec)
    hipLaunchKernelGGL((int8_write_kernel<DTYPE, D, true>), grid, threads, 0, st, p);
  else
    hipLaunchKernelGGL((int8_write_kernel<DTYPE, D, false>), grid, threads, 0, st, p);
  return hipGetLastError();
}

template <int OUT, int D>
hipError_t launch_read(CacheRead p, hipStream_t st) {
  // Fewer tokens a workgroup where 16 would leave places on the GPU empty.
  p.per_group = (int32_t)std::clamp<int64_t>(p.total / 2048, 1, kReadTokens);
  const int64_t blocks = cdiv<int64_t>(p.total, p.per_group);
  if (!launchable(blocks, 256)) return hipErrorInvalidConfiguration;
  p.by_token = make_divisor(p.KV * (D / (OUT == VXA_F32 ? 4 : 8)));
  hipLaunchKernelGGL((int8_read_kernel<OUT, D>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  return hipGetLastError();
}

// launch(std::integral_constant<int, dtype>, std::integral_constant<int, D>) for the call's type and head size.
template <typename F>
hipError_t dispatch(int dtype, int64_t D, F&& launch) {
  auto by_dim = [&](auto t) {
    if (D == 64) return launch(t, std::integral_constant<int, 64>{});
    if (D == 128) return launch(t, std::integral_constant<int, 128>{});
    return launch(t, std::integral_constant<int, 256>{});
  };
  if (dtype == VXA_F32) return by_dim(std::integral_constant<int, VXA_F32>{});
  if (dtype == VXA_BF16) return by_dim(std::integral_constant<int, VXA_BF16>{});
  return by_dim(std::integral_constant<int, VXA_F16>{});
}

bool known_dtype(int d) { return d == VXA_F32 || d == VXA_BF16 || d == VXA_F16; }
bool known_dim(int64_t d) { return d == 64 || d == 128 || d == 256; }

// Sizes both entry points take: 32-bit slot arithmetic, and 8-bit rows that start on 16 bytes.
int check_cache(const void* kc, const void* vc, const int64_t* sk, const int64_t* sv, int64_t blocks, int64_t page,
                int64_t KV, int64_t D) {
  if (!known_dim(D) || KV > (1 << 16) || page > (1 << 30) || blocks > 0x7FFFFFFFLL / page) return VXA_ERR_UNSUPPORTED;
  if ((uintptr_t)kc % 16 || (uintptr_t)vc % 16) return VXA_ERR_UNSUPPORTED;
  for (int i = 0; i < 3; ++i)
    if (sk[i] % 16 || sv[i] % 16) return VXA_ERR_UNSUPPORTED;
  return VXA_OK;
}

}  // namespace

extern "C" int vxa_int8_cache_write(const void* key, int64_t skt, int64_t skh, const void* value, int64_t svt,
                                    int64_t svh, int dtype, int64_t tokens, int64_t num_kv_heads, int64_t head_dim,
                                    int8_t* k_cache, int64_t skcb, int64_t skcp, int64_t skch, int8_t* v_cache,
                                    int64_t svcb, int64_t svcp, int64_t svch, float* k_scale, int64_t sksb,
                                    int64_t sksp, int64_t sksh, float* v_scale, int64_t svsb, int64_t svsp,
                                    int64_t svsh, int64_t num_blocks, int64_t block_size, const int64_t* slots,
                                    vxa_stream_t stream) {
  if (tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || num_blocks < 0 || block_size <= 0 || !known_dtype(dtype))
    return VXA_ERR_ARG;
  if (tokens == 0 || num_blocks == 0) return VXA_OK;
  if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !slots) return VXA_ERR_ARG;
  const int64_t sk[3] = {skcb, skcp, skch}, sv[3] = {svcb, svcp, svch};
  const int rc = check_cache(k_cache, v_cache, sk, sv, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != VXA_OK) return rc;
  if (tokens > (int64_t)1 << 40) return VXA_ERR_UNSUPPORTED;
  const int64_t piece = dtype == VXA_F32 ? 4 : 8;  // elements of 16 bytes
  const bool vec = (uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0 && skt % piece == 0 && skh % piece == 0 &&
                   svt % piece == 0 && svh % piece == 0;
  const CacheWrite p{{key, value}, {skt, svt}, {skh, svh}, {k_cache, v_cache}, {skcb, svcb}, {skcp, svcp}, {skch, svch},
                     {k_scale, v_scale}, {sksb, svsb}, {sksp, svsp}, {sksh, svsh}, slots, tokens, (int32_t)num_kv_heads,
                     (int32_t)block_size, Divisor{}, make_divisor(block_size), num_blocks * block_size, 1};
  const hipError_t err = dispatch(dtype, head_dim, [&](auto t, auto d) {
    return launch_write<decltype(t)::value, decltype(d)::value>(p, vec, reinterpret_cast<hipStream_t>(stream));
  });
  if (err == hipErrorInvalidConfiguration) return VXA_ERR_UNSUPPORTED;
  return err == hipSuccess ? VXA_OK : VXA_ERR_LAUNCH;
}

extern "C" int vxa_int8_cache_read(const int8_t* k_cache, int64_t skcb, int64_t skcp, int64_t skch,
                                   const int8_t* v_cache, int64_t svcb, int64_t svcp, int64_t svch,
                                   const float* k_scale, int64_t sksb, int64_t sksp, int64_t sksh,
                                   const float* v_scale, int64_t svsb, int64_t svsp, int64_t svsh, int64_t num_blocks,
                                   int64_t block_size, const int32_t* block_table, int64_t sbt, int64_t bt_cols,
                                   const int32_t* starts, const int32_t* first, int64_t n, int64_t tokens,
                                   int64_t num_kv_heads, int64_t head_dim, void* key, int64_t skt, int64_t skh,
                                   void* value, int64_t svt, int64_t svh, int dtype, vxa_stream_t stream) {
  if (tokens < 0 || n < 0 || num_kv_heads <= 0 || head_dim <= 0 || num_blocks < 0 || block_size <= 0 || bt_cols < 0 ||
      !known_dtype(dtype))
    return VXA_ERR_ARG;
  if (tokens == 0 || n == 0) return VXA_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !block_table || !starts || !key || !value) return VXA_ERR_ARG;
  const int64_t sk[3] = {skcb, skcp, skch}, sv[3] = {svcb, svcp, svch};
  const int rc = check_cache(k_cache, v_cache, sk, sv, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != VXA_OK) return rc;
  if (tokens > 0x7FFFFFFFLL || n > 0x7FFFFFFFLL || bt_cols > 0x7FFFFFFFLL / block_size) return VXA_ERR_UNSUPPORTED;
  const int64_t piece = dtype == VXA_F32 ? 4 : 8;
  if ((uintptr_t)key % 16 || (uintptr_t)value % 16 || skt % piece || skh % piece || svt % piece || svh % piece)
    return VXA_ERR_UNSUPPORTED;
  const CacheRead p{{k_cache, v_cache}, {skcb, svcb}, {skcp, svcp}, {skch, svch}, {k_scale, v_scale}, {sksb, svsb},
                    {sksp, svsp}, {sksh, svsh}, block_table, sbt, starts, first, n, tokens, (int32_t)num_kv_heads,
                    (int32_t)block_size, (int32_t)bt_cols, Divisor{}, make_divisor(block_size), kReadTokens, num_blocks, {key, value}, {skt, svt}, {skh, svh}};
  const hipError_t err = dispatch(dtype, head_dim, [&](auto t, auto d) {
    return launch_read<decltype(t)::value, decltype(d)::value>(p, reinterpret_cast<hipStream_t>(stream));
  });
  if (err == hipErrorInvalidConfiguration) return VXA_ERR_UNSUPPORTED;
  return err == hipSuccess ? VXA_OK : VXA_ERR_LAUNCH;
}
