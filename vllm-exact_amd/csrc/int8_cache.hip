// A paged KV cache in 8 bits (gfx950): quantising new tokens as they are written, and reading ranges back.
//
// Each (token, KV head) has one scale for its key and one for its value: top = max |x| over the head's D
// elements, scale = top / 127, q = round(127 x / top) to the nearest whole number, ties to even, so q lies in
// [-127, 127] and stands for q * scale. 127 x is exact in fp32 for 16-bit x and the quotient of two such
// inputs is either a half exactly or further from it than its fp32 rounding, so q is the nearest whole number
// of the quotient itself. A row with an infinity or NaN gets q = 0 and the scale NaN: it reads back as NaN.
// A row of zeros gets the scale 0.
//
// Both kernels move each byte once and are bound by HBM, and by launch latency at a decode step's sizes.

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
  int64_t rows_total;     // slots of the cache: blocks * page
};

// LPR lanes hold a row, 8 elements each; a workgroup's rows are consecutive (token, KV head, key or value).
template <int DTYPE, int D, bool VEC>
__global__ __launch_bounds__(256) void int8_write_kernel(CacheWrite p) {
  constexpr int LPR = D / 8;
  const int lane = threadIdx.x & (LPR - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int which = (int)(row & 1);
  const int64_t th = row >> 1;
  const int64_t t = th / p.KV;
  const int h = (int)(th - t * p.KV);
  const bool live = t < p.tokens;
  float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  int64_t slot = -1;
  if (live) {
    slot = p.slots[t];
    const int64_t at = t * p.sxt[which] + (int64_t)h * p.sxh[which] + 8 * lane;
    if constexpr (DTYPE == VXA_F32) {
      const float* src = reinterpret_cast<const float*>(p.x[which]) + at;
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
      const uint16_t* src = reinterpret_cast<const uint16_t*>(p.x[which]) + at;
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
  }
  // The largest magnitude as bits: NaN and infinities order above every finite value.
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
#pragma unroll
  for (int m = 1; m < LPR; m *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, m));
  if (!live || slot < 0 || slot >= p.rows_total) return;
  const float ftop = __uint_as_float(top);
  const bool special = top >= 0x7F800000u;
  const int32_t block = (int32_t)((uint32_t)slot / (uint32_t)p.page);
  const int32_t off = (int32_t)slot - block * p.page;
  if (lane == 0)
    p.s[which][(int64_t)block * p.ssb[which] + (int64_t)off * p.ssp[which] + (int64_t)h * p.ssh[which]] =
        special ? __builtin_nanf("") : ftop / 127.0f;
  // Above 2^100 the products 127 x could overflow: both sides are scaled by 2^-32, which rounds nothing that counts.
  const float down = ftop > 0x1p100f ? 0x1p-32f : 1.0f;
  const float div = ftop * down;
  const bool zero = special || top == 0;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int q = zero ? 0 : (int)rintf((x[j] * down) * 127.0f / div);
    w[j / 4] |= ((uint32_t)q & 0xFFu) << (8 * (j % 4));
  }
  int8_t* dst = p.c[which] + (int64_t)block * p.scb[which] + (int64_t)off * p.scp[which] + (int64_t)h * p.sch[which] + 8 * lane;
  *reinterpret_cast<v2u32*>(dst) = v2u32{w[0], w[1]};
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
  int64_t blocks;
  void* o[2];
  int64_t sot[2], soh[2];
};

constexpr int kReadTokens = 16;  // tokens of a workgroup

// A workgroup reads 16 packed tokens, all heads, keys and values: whole lines of the cache's pages (a page's
// tokens follow each other) and whole lines of the output (a token's heads do). A lane moves 16 elements.
template <int OUT, int D>
__global__ __launch_bounds__(256) void int8_read_kernel(CacheRead p) {
  constexpr int LPR = D / 16;
  __shared__ int32_t s_block[kReadTokens], s_off[kReadTokens];
  const int64_t t0 = (int64_t)blockIdx.x * kReadTokens;
  if (threadIdx.x < 64) {
    // A token's sequence is the number of sequences that end at or before it: lanes compare 64 ends at a time.
    const int lane = threadIdx.x;
    int seq = 0;
    for (int64_t j0 = 0; j0 < p.n; j0 += 64) {
      const int64_t j = j0 + lane;
      const int32_t end = j < p.n ? p.cu[j + 1] : 0x7FFFFFFF;
#pragma unroll
      for (int i = 0; i < kReadTokens; ++i) {
        const int c = __popcll(__ballot((int64_t)end <= t0 + i));
        if (lane == i) seq += c;
      }
    }
    if (lane < kReadTokens) {
      int32_t block = -1, off = 0;  // -1: the row is in no sequence, -2: its page does not exist
      const int64_t in_seq = t0 + lane < p.total && seq < p.n ? t0 + lane - p.cu[seq] : -1;
      if (in_seq >= 0) {
        const int64_t pos = in_seq + (p.first != nullptr ? p.first[seq] : 0);
        block = -2;
        if (pos >= 0 && pos < (int64_t)p.cols * p.page) {
          const int32_t pg = (int32_t)((uint32_t)pos / (uint32_t)p.page);
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
  const int units = kReadTokens * p.KV * 2 * LPR;
  for (int u = threadIdx.x; u < units; u += 256) {
    const int lane = u & (LPR - 1);
    const int r = u / LPR;
    const int which = r & 1;
    const int i = (r >> 1) / p.KV;
    const int h = (r >> 1) - i * p.KV;
    const int32_t block = s_block[i], off = s_off[i];
    if (block == -1) continue;
    float scale = __builtin_nanf("");
    v4u32 w = {0, 0, 0, 0};
    if (block >= 0) {
      scale = p.s[which][(int64_t)block * p.ssb[which] + (int64_t)off * p.ssp[which] + (int64_t)h * p.ssh[which]];
      w = *reinterpret_cast<const v4u32*>(p.c[which] + (int64_t)block * p.scb[which] + (int64_t)off * p.scp[which] +
                                          (int64_t)h * p.sch[which] + 16 * lane);
    }
    float f[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = (float)(int8_t)(w[j / 4] >> (8 * (j % 4))) * scale;
    const int64_t at = (t0 + i) * p.sot[which] + (int64_t)h * p.soh[which] + 16 * lane;
    if constexpr (OUT == VXA_F32) {
      float* dst = reinterpret_cast<float*>(p.o[which]) + at;
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<v4f*>(dst + 4 * j) = v4f{f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]};
    } else {
      using T = std::conditional_t<OUT == VXA_BF16, BF16, FP16>;
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = T::pack(f[2 * j], f[2 * j + 1]);
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.o[which]) + at;
      *reinterpret_cast<v4u32*>(dst) = v4u32{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<v4u32*>(dst + 8) = v4u32{o[4], o[5], o[6], o[7]};
    }
  }
}

template <int DTYPE, int D>
hipError_t launch_write(const CacheWrite& p, bool vec, hipStream_t st) {
  const int64_t blocks = cdiv<int64_t>(p.tokens * p.KV * 2, 256 / (D / 8));
  if (blocks > 0x7FFFFFFFLL) return hipErrorInvalidConfiguration;
  if (vec)
    hipLaunchKernelGGL((int8_write_kernel<DTYPE, D, true>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((int8_write_kernel<DTYPE, D, false>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  return hipGetLastError();
}

template <int OUT, int D>
hipError_t launch_read(const CacheRead& p, hipStream_t st) {
  const int64_t blocks = cdiv<int64_t>(p.total, kReadTokens);
  if (blocks > 0x7FFFFFFFLL) return hipErrorInvalidConfiguration;
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
  if (!known_dim(D) || KV > (1 << 20) || page > (1 << 30) || blocks > 0x7FFFFFFFLL / page) return VXA_ERR_UNSUPPORTED;
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
                     (int32_t)block_size, num_blocks * block_size};
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
                    (int32_t)block_size, (int32_t)bt_cols, num_blocks, {key, value}, {skt, svt}, {skh, svh}};
  const hipError_t err = dispatch(dtype, head_dim, [&](auto t, auto d) {
    return launch_read<decltype(t)::value, decltype(d)::value>(p, reinterpret_cast<hipStream_t>(stream));
  });
  if (err == hipErrorInvalidConfiguration) return VXA_ERR_UNSUPPORTED;
  return err == hipSuccess ? VXA_OK : VXA_ERR_LAUNCH;
}
