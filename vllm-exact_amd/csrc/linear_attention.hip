// Linear attention with a decay for each head (gfx950): whole prompts, and one new token of every sequence.
//
//   S_t = exp(g) S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
// for every row t of a sequence, S a D x D matrix of each head in fp32, g the head's log_decay. A sequence starts from a slot of
// a pool of states (or zeros) and ends in one.

#include "attention_common.h"

namespace {

struct LinearParams {
  const uint16_t* q;
  int64_t sqt, sqh;
  const uint16_t* k;
  int64_t skt, skh;
  const uint16_t* v;
  int64_t svt, svh;
  const int32_t* cu;  // null: sequence i is row i
  int32_t n, total, H, G;
  const float* log_decay;
  float scale;
  void* out;
  int64_t sot, soh;
  int32_t out_dtype;
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
  if (p.write)
    for (int j = threadIdx.x; j < p.n; j += blockDim.x) {
      const int w = p.write[j];
      if (j != seq) bad |= (w >= 0 && (w == s.write || w == s.read)) || (p.read && s.write >= 0 && p.read[j] == s.write);
    }
  s.bad = __syncthreads_or(bad);
  return s;
}

constexpr int kCols = 32;    // columns of a state that a workgroup keeps
constexpr int kTokens = 16;  // staged at a time

// The recurrence as it stands: a workgroup keeps kCols columns of one head's state in registers.
template <typename T, int D>
__global__ __launch_bounds__(256) void linear_recurrent_kernel(LinearParams p) {
  constexpr int kRows = D / 8;  // of the state, of a thread
  __shared__ float s_q[kTokens][D], s_k[kTokens][D], s_v[kTokens][kCols], s_o[8][kTokens][kCols];
  const int slabs = D / kCols;
  const int slab = blockIdx.x % slabs, head = (int)(blockIdx.x / slabs) % p.H, seq = (int)(blockIdx.x / slabs) / p.H;
  const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
  int lo = seq, hi = seq + 1;
  if (p.cu) {
    lo = min(max(p.cu[seq], 0), p.total);
    hi = min(max(p.cu[seq + 1], lo), p.total);
  }
  const Slots slots = find_slots(p, seq);
  const int64_t at = (int64_t)head * p.soh + slab * kCols + col;
  if (slots.bad) {
    for (int t = lo + part; t < hi; t += 8) store_f32_as(p.out, p.out_dtype, t * p.sot + at, __builtin_nanf(""));
    return;
  }
  const int64_t place = (int64_t)head * p.ssh + (int64_t)part * kRows * D + slab * kCols + col;
  float s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) s[i] = slots.read >= 0 ? p.state[slots.read * p.sss + place + (int64_t)i * D] : 0.0f;
  const float decay = expf(p.log_decay[head]);
  for (int t0 = lo; t0 < hi; t0 += kTokens) {
    const int count = min(kTokens, hi - t0);
    __syncthreads();
    for (int x = threadIdx.x; x < count * D; x += 256) {
      const int64_t t = t0 + x / D;
      s_q[x / D][x % D] = T::to_f32(p.q[t * p.sqt + head * p.sqh + x % D]);
      s_k[x / D][x % D] = T::to_f32(p.k[t * p.skt + head / p.G * p.skh + x % D]);
    }
    for (int x = threadIdx.x; x < count * kCols; x += 256)
      s_v[x / kCols][x % kCols] = T::to_f32(p.v[(int64_t)(t0 + x / kCols) * p.svt + head / p.G * p.svh + slab * kCols + x % kCols]);
    __syncthreads();
    for (int t = 0; t < count; ++t) {
      const float v = s_v[t][col];
      float o = 0.0f;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        s[i] = fmaf(s_k[t][part * kRows + i], v, decay * s[i]);
        o = fmaf(s_q[t][part * kRows + i], s[i], o);
      }
      s_o[part][t][col] = o;
    }
    __syncthreads();
    for (int t = part; t < count; t += 8) {
      float o = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o += s_o[i][t][col];
      store_f32_as(p.out, p.out_dtype, (t0 + t) * p.sot + at, o * p.scale);
    }
  }
  if (slots.write >= 0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) p.state[slots.write * p.sss + place + (int64_t)i * D] = s[i];
  }
}

template <typename T>
hipError_t launch_recurrent(int64_t D, const LinearParams& p, hipStream_t st) {
  const int64_t blocks = (int64_t)p.n * p.H * (D / kCols);
  if (!launchable(blocks, 256)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks);
  if (D == 64)
    hipLaunchKernelGGL((linear_recurrent_kernel<T, 64>), grid, dim3(256), 0, st, p);
  else if (D == 128)
    hipLaunchKernelGGL((linear_recurrent_kernel<T, 128>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((linear_recurrent_kernel<T, 256>), grid, dim3(256), 0, st, p);
  return hipGetLastError();
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
  // Rows are read in 16-byte pieces.
  if ((uintptr_t)q % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || sqt % 8 || sqh % 8 || skt % 8 || skh % 8 || svt % 8 || svh % 8 ||
      (uintptr_t)state % 16 || sss % 4 || ssh % 4)
    return VXA_ERR_UNSUPPORTED;
  p.q = reinterpret_cast<const uint16_t*>(q), p.sqt = sqt, p.sqh = sqh;
  p.k = reinterpret_cast<const uint16_t*>(k), p.skt = skt, p.skh = skh;
  p.v = reinterpret_cast<const uint16_t*>(v), p.svt = svt, p.svh = svh;
  p.cu = nullptr;
  p.n = (int32_t)n, p.total = (int32_t)tokens, p.H = (int32_t)H, p.G = (int32_t)(H / KV);
  p.log_decay = log_decay, p.scale = scale;
  p.out = out, p.sot = sot, p.soh = soh, p.out_dtype = out_dtype;
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
  *ws_bytes = 0;
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
  p.cu = starts;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return status_of(dtype == VXA_BF16 ? launch_recurrent<BF16>(head_dim, p, st) : launch_recurrent<FP16>(head_dim, p, st));
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
  return status_of(dtype == VXA_BF16 ? launch_recurrent<BF16>(head_dim, p, st) : launch_recurrent<FP16>(head_dim, p, st));
}
