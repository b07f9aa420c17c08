// Pages of a cache (gfx950): copied, shared by forked rows, given out and taken back, and the kept tokens of drafted trees moved
// side by side.
//
// A page belongs to as many holders as its reference count says; 0: it is free. Rows of a block table hold the pages of their
// tokens, each from place 0 on; entries behind are -1. Nothing here goes through the host, and no result depends on the order in
// which workgroups run: counts are whole numbers, and new pages are the lowest free ones, in the order of rows and places.
//
// fork and resize are two launches: one workgroup decides which places get a page and finds the free ones, while others copy the
// counts; then a workgroup for each row writes its entries and counts, and others copy the pages. They move few bytes (2.4 us at a
// copy's rate for 256 rows and 4 layers) and are bound by launches and chains of dependent reads: parents, lengths, entries, counts,
// then the page. fork of 256 rows, 16 views: 5.3 + 7.9 us, resize 4.7 + 4.0; keep of 64 trees of 40 nodes, 16 views: 6.4, resize 2.4 + 3.1.
// A call takes 4 to 9 us on the host besides, most of it the views that it is given.

#include <algorithm>

#include "attention_common.h"

namespace {

constexpr int kViews = 32;       // of a launch
constexpr int kPlan = 1024;      // threads of the planning kernel
constexpr int kMostRows = 8192;  // of a table: the plan keeps two numbers of each in LDS

// Tokens of a cache, [block][place][head] rows of `bytes` bytes.
struct View {
  char* data;
  int64_t block, token, head;  // strides in bytes
  int32_t heads, bytes, unit;  // unit: bytes that are moved at once, all of the above are multiples of it
};
struct Views {
  View at[kViews];
};

// f(a value of the type that the view's rows are moved in)
template <typename F>
__device__ inline void with_unit(const View& v, F&& f) {
  if (v.unit == 16)
    f(v4u32{});
  else if (v.unit == 4)
    f(uint32_t{});
  else if (v.unit == 2)
    f(uint16_t{});
  else
    f(uint8_t{});
}

__device__ inline int pages_of(int tokens, int page) { return tokens <= 0 ? 0 : (int)(((int64_t)tokens + page - 1) / page); }

// By a workgroup of 256 threads.
__device__ inline void copy_page(const View& v, int page, int from, int to) {
  const bool by_head = v.token < v.head;  // which of the two is the inner dimension in memory
  const uint32_t inner = by_head ? page : v.heads;
  const char* src = v.data + from * v.block;
  char* dst = v.data + to * v.block;
  with_unit(v, [&](auto unit) {
    using U = decltype(unit);
    const uint32_t chunks = v.bytes / (int)sizeof(U), all = (uint32_t)page * v.heads * chunks;
    for (uint32_t i = threadIdx.x; i < all; i += 256) {
      const uint32_t x = i / chunks, c = i - x * chunks, b = x / inner, a = x - b * inner;
      const int64_t at = (by_head ? a * v.token + b * v.head : b * v.token + a * v.head) + c * (int64_t)sizeof(U);
      *reinterpret_cast<U*>(dst + at) = *reinterpret_cast<const U*>(src + at);
    }
  });
}

// Workgroup (x, y): pair x of view y. Of pairs with one target the last counts: every workgroup looks through the pairs behind its own, so a
// launch has at most 1024 of them, and later launches write over what earlier ones did. 16 views of four layers' 8-bit caches, 8 heads of
// 128, pages of 16: 1000 pairs 48 us, 4000 262, 16000 1056 (1685 with one launch), 4.1 TB/s read and written where a large copy
// reaches 4.9. A page of 528 tokens is one workgroup's, too: 31 us for one pair.
constexpr int kPairs = 1024;
__global__ __launch_bounds__(256) void pages_copy_kernel(Views views, int num_blocks, int page, const int32_t* source, const int32_t* target, int n) {
  const int from = source[blockIdx.x], to = target[blockIdx.x];
  if (from < 0 || from >= num_blocks || to < 0 || to >= num_blocks || from == to) return;
  bool later = false;
  for (int j = blockIdx.x + 1 + threadIdx.x; j < n; j += 256) later |= target[j] == to && source[j] >= 0 && source[j] < num_blocks;
  if (__syncthreads_or(later)) return;
  copy_page(views.at[blockIdx.y], page, from, to);
}

struct TableParams {
  const int32_t* table;
  int64_t stride;
  int32_t cols, rows;
  const int32_t* lens;      // of the old rows
  const int32_t* new_lens;  // resize
  const int32_t* parents;   // fork
  int32_t new_rows;
  int32_t* out_table;
  int64_t out_stride;
  int32_t* out_lens;  // fork
  const int32_t* refs;
  int32_t* out_refs;
  int32_t num_blocks, page;
  int32_t* missing;  // one number: places that wanted a page and got none
  int32_t* ws;
  // ws of fork: children[rows], source[new_rows], target[new_rows]; of resize: base[rows + 1], list[num_blocks]
};

// Running sum of x over the workgroup's threads, this one's included, and the sum of all.
__device__ inline int block_scan(int x, int* s_wave, int& all) {
  const int wave = threadIdx.x >> 6;
  const int mine = wave_scan(x, [](int a, int b) { return a + b; });
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s_wave[wave] = mine;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kPlan / 64; ++w) {
    if (w < wave) before += s_wave[w];
    all += s_wave[w];
  }
  return mine + before;
}

// give(rank, page) for the `wanted` lowest free pages; how many there were. A wave looks at 64 counts with each load, all of them at
// once; the free ones are the bits of a ballot. (8 counts a thread, one after the other in memory: 3.5 us for each
// 8192 of them in place of 2. 16 loads a wave: more instructions than a small pool's plan has time to fetch, 7.0 us for a resize in place of 6.2.)
template <typename F>
__device__ int find_free(const TableParams& p, int wanted, int* s_wave, F&& give) {
  constexpr int kMost = 8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int loads = min(kMost, (p.num_blocks + kPlan - 1) / kPlan);  // of a wave: few counts are for all waves too
  int found = 0;
  for (int b0 = 0; b0 < p.num_blocks && found < wanted; b0 += loads * kPlan) {
    const int first = b0 + wave * 64 * loads + lane;
    int32_t x[kMost];
    uint64_t free[kMost];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kMost; ++j)
      if (j < loads) x[j] = p.refs[min(first + 64 * j, p.num_blocks - 1)];
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
      free[j] = 0;
      if (j < loads) free[j] = __ballot(first + 64 * j < p.num_blocks && x[j] == 0);
      mine += __popcll(free[j]);
    }
    __syncthreads();  // the sums before have been read
    if (lane == 0) s_wave[wave] = mine;
    __syncthreads();
    int rank = found;
#pragma unroll
    for (int w = 0; w < kPlan / 64; ++w) {
      if (w < wave) rank += s_wave[w];
      found += s_wave[w];
    }
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
      if (free[j] == 0) continue;
      const int at = rank + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(free[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)free[j], 0u));
      if ((free[j] >> lane & 1) && at < wanted) give(at, first + 64 * j);
      rank += __popcll(free[j]);
    }
  }
  return min(found, wanted);
}

__device__ inline void copy_refs(const TableParams& p, int share, int shares) {
  constexpr int N = 4;  // at once
  const int step = shares * kPlan;
  for (int i0 = share * kPlan + (int)threadIdx.x; i0 < p.num_blocks; i0 += N * step) {
    int32_t x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = p.refs[min(i0 + j * step, p.num_blocks - 1)];
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i0 + j * step < p.num_blocks) p.out_refs[i0 + j * step] = x[j];
  }
}

// Length of row r's parent, and the page of its partly filled end (-1: there is none, or not one of the cache).
struct Parent {
  int row, len, tail;
};
__device__ inline Parent parent_of(const TableParams& p, int r) {
  Parent a{p.parents[r], 0, -1};
  if (a.row < 0 || a.row >= p.rows) return Parent{-1, 0, -1};
  a.len = min(max(p.lens[a.row], 0), (int)min((int64_t)p.cols * p.page, (int64_t)0x7FFFFFFF));
  if (a.len % p.page) {
    const int page = p.table[a.row * p.stride + a.len / p.page];
    if (page >= 0 && page < p.num_blocks) a.tail = page;
  }
  return a;
}

__global__ __launch_bounds__(kPlan) void pages_fork_plan_kernel(TableParams p) {
  __shared__ int s_first[kMostRows], s_children[kMostRows], s_wave[kPlan / 64];
  if (blockIdx.x > 0) return copy_refs(p, blockIdx.x - 1, gridDim.x - 1);
  int32_t *children = p.ws, *source = p.ws + p.rows, *target = source + p.new_rows;
  for (int i = threadIdx.x; i < p.rows; i += kPlan) s_first[i] = 0x7FFFFFFF, s_children[i] = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < p.new_rows; r += kPlan) {
    const int a = p.parents[r];
    if (a >= 0 && a < p.rows) atomicMin(&s_first[a], r), atomicAdd(&s_children[a], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.rows; i += kPlan) children[i] = s_children[i];
  // A row gets a page of its own for a partly filled end, unless it is the first of its parent and nobody else holds that page.
  int wanted = 0;
  for (int r0 = 0; r0 < p.new_rows; r0 += kPlan) {
    const int r = r0 + threadIdx.x;
    Parent a{-1, 0, -1};
    if (r < p.new_rows) a = parent_of(p, r);
    const bool copied = a.tail >= 0 && !(s_first[a.row] == r && p.refs[a.tail] == 1);
    int all;
    const int rank = wanted + block_scan(copied, s_wave, all) - 1;
    if (r < p.new_rows) source[r] = copied ? a.tail : -1, target[r] = copied ? rank : -1;  // the page's number in the order of free ones, for now
    wanted += all;
  }
  // Rows' ranks rise: the row of a rank is found again from them.
  __syncthreads();
  int* order = s_first;  // row of each rank
  for (int r = threadIdx.x; r < p.new_rows; r += kPlan)
    if (target[r] >= 0) order[target[r]] = r;
  __syncthreads();
  for (int r = threadIdx.x; r < p.new_rows; r += kPlan)
    if (source[r] >= 0) target[r] = -1;
  __syncthreads();
  const int found = find_free(p, wanted, s_wave, [&](int rank, int page) { target[order[rank]] = page; });
  if (threadIdx.x == 0) *p.missing = wanted - found;
}

// Workgroup (x, 0): row x's entries, and the counts of the pages that the old row x held. (x, 1 + y): the copy of row x's end in view y.
__global__ __launch_bounds__(256) void pages_fork_kernel(TableParams p, Views views) {
  const int32_t *children = p.ws, *source = p.ws + p.rows, *target = source + p.new_rows;
  const int r = blockIdx.x;
  if (blockIdx.y > 0) {
    if (r < p.new_rows && source[r] >= 0 && target[r] >= 0) copy_page(views.at[blockIdx.y - 1], p.page, source[r], target[r]);
    return;
  }
  if (r < p.rows) {  // its pages have as many holders more as it has children, but for itself
    const int len = min(max(p.lens[r], 0), (int)min((int64_t)p.cols * p.page, (int64_t)0x7FFFFFFF)), all = pages_of(len, p.page), more = children[r] - 1;
    const bool part = len % p.page != 0;
    if (more != 0)
      for (int j = threadIdx.x; j < all - part; j += 256) {
        const int b = p.table[r * p.stride + j];
        if (b >= 0 && b < p.num_blocks) atomicAdd(&p.out_refs[b], more);
      }
    if (part && threadIdx.x == 0) {
      const int b = p.table[r * p.stride + all - 1];
      if (b >= 0 && b < p.num_blocks) atomicAdd(&p.out_refs[b], -1);
    }
  }
  if (r < p.new_rows) {
    const Parent a = parent_of(p, r);
    const int all = pages_of(a.len, p.page);
    for (int j = threadIdx.x; j < p.cols; j += 256) {
      int b = j < all ? p.table[a.row * p.stride + j] : -1;
      if (j == all - 1 && a.tail >= 0) {
        if (source[r] >= 0) b = target[r];
        if (b >= 0) atomicAdd(&p.out_refs[b], 1);
      }
      p.out_table[r * p.out_stride + j] = b;
    }
    if (threadIdx.x == 0) p.out_lens[r] = a.len;
  }
}

// The copies in further views.
__global__ __launch_bounds__(256) void pages_fork_copy_kernel(TableParams p, Views views) {
  const int32_t *source = p.ws + p.rows, *target = source + p.new_rows;
  const int r = blockIdx.x;
  if (source[r] >= 0 && target[r] >= 0) copy_page(views.at[blockIdx.y], p.page, source[r], target[r]);
}

// Where each row's new pages are in the list of free ones, and the list.
__device__ inline void plan_resize(const TableParams& p, int* s_wave) {
  int32_t *base = p.ws, *list = p.ws + p.rows + 1;
  int wanted = 0;
  for (int r0 = 0; r0 < p.rows; r0 += kPlan) {
    const int r = r0 + threadIdx.x;
    int more = 0;
    if (r < p.rows) more = max(min(pages_of(p.new_lens[r], p.page), p.cols) - min(pages_of(p.lens[r], p.page), p.cols), 0);
    int all;
    const int upto = block_scan(more, s_wave, all);
    if (r < p.rows) base[r] = wanted + upto - more;
    wanted += all;
  }
  const int found = find_free(p, min(wanted, p.num_blocks), s_wave, [&](int rank, int page) { list[rank] = page; });
  if (threadIdx.x == 0) base[p.rows] = found, *p.missing = wanted - found;
}
// Entry j of row r.
__device__ inline void resize_entry(const TableParams& p, int r, int j) {
  const int32_t *base = p.ws, *list = p.ws + p.rows + 1;
  const int had = min(pages_of(p.lens[r], p.page), p.cols), has = min(pages_of(p.new_lens[r], p.page), p.cols);
  int b = p.table[r * p.stride + j];
  if (j >= has && j < had && b >= 0 && b < p.num_blocks) atomicAdd(&p.out_refs[b], -1);
  if (j >= has) b = -1;
  if (j >= had && j < has) {
    const int rank = base[r] + j - had;
    b = rank < base[p.rows] ? list[rank] : -1;
    if (b >= 0) atomicAdd(&p.out_refs[b], 1);
  }
  p.out_table[r * p.out_stride + j] = b;
}

__global__ __launch_bounds__(kPlan) void pages_resize_plan_kernel(TableParams p) {
  __shared__ int s_wave[kPlan / 64];
  if (blockIdx.x > 0) return copy_refs(p, blockIdx.x - 1, gridDim.x - 1);
  plan_resize(p, s_wave);
}
__global__ __launch_bounds__(256) void pages_resize_kernel(TableParams p) {
  for (int j = threadIdx.x; j < p.cols; j += 256) resize_entry(p, blockIdx.x, j);
}
// All of it by one workgroup, an entry a thread.
__global__ __launch_bounds__(kPlan) void pages_resize_small_kernel(TableParams p) {
  __shared__ int s_wave[kPlan / 64];
  if (p.out_refs != p.refs) copy_refs(p, 0, 1);
  plan_resize(p, s_wave);
  __syncthreads();  // the copied counts, the plan
  if ((int)threadIdx.x < p.rows * p.cols) resize_entry(p, threadIdx.x / p.cols, threadIdx.x % p.cols);
}

struct KeepParams {
  const int32_t* table;
  int64_t stride;
  int32_t cols;
  const int32_t *lens, *starts;
  const int64_t* keep;
  int32_t* out_lens;
  int32_t num_blocks, page;
};
constexpr int kKeepUnits = 8;                       // that a thread holds
constexpr int kKeepWidth = kKeepUnits * 256 / 64;   // columns of a slab: a workgroup holds 64 rows of it

// Workgroup (request, view, slab): the kept rows of columns (head, chunk) of the view. A kept token moves to a place that another one
// may still lie in, so all are read, into registers, before any is written: 64 rows of 32 chunks for 256 threads of 8.
__global__ __launch_bounds__(256) void pages_keep_kernel(KeepParams p, Views views, bool lens) {
  __shared__ int64_t s_src[64], s_dst[64];  // of kept row j, -1: it stays where it is
  const int r = blockIdx.x;
  const int64_t count = (int64_t)p.starts[r + 1] - p.starts[r], context = p.lens[r] - count;
  const bool bad = count < 0 || count > 64 || context < 0;
  const uint64_t kept = bad || count == 0 ? 0 : (uint64_t)p.keep[r] & ~0ull >> (64 - count);
  const int moved = __popcll(kept);
  if (lens && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) p.out_lens[r] = bad ? p.lens[r] : (int)context + moved;
  if (moved == 0) return;
  const View v = views.at[blockIdx.y];
  auto place = [&](int64_t at) {
    const int64_t col = at / p.page;
    const int b = col < p.cols ? p.table[r * p.stride + col] : -1;
    return b >= 0 && b < p.num_blocks ? b * v.block + at % p.page * v.token : -1;
  };
  if (threadIdx.x < 64 && kept >> threadIdx.x & 1) {
    const int rank = __popcll(kept & ((1ull << threadIdx.x) - 1));
    const int64_t from = place(context + threadIdx.x), to = place(context + rank);
    const bool go = rank != (int)threadIdx.x && from >= 0 && to >= 0;
    s_src[rank] = go ? from : -1, s_dst[rank] = to;
  }
  __syncthreads();
  with_unit(v, [&](auto unit) {
    using U = decltype(unit);
    const int chunks = v.bytes / (int)sizeof(U), columns = v.heads * chunks;
    for (int c0 = blockIdx.z * kKeepWidth; c0 < columns; c0 += gridDim.z * kKeepWidth) {
      U held[kKeepUnits];
      const int col = c0 + (int)threadIdx.x % kKeepWidth;
      const int64_t at = col < columns ? col / chunks * v.head + col % chunks * (int64_t)sizeof(U) : 0;
      auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kKeepUnits; ++i) {
          const int j = (int)threadIdx.x / kKeepWidth + i * (256 / kKeepWidth);
          if (j < moved && col < columns && s_src[j] >= 0) f(i, j);
        }
      };
      each([&](int i, int j) { held[i] = *reinterpret_cast<const U*>(v.data + s_src[j] + at); });
      __syncthreads();
      each([&](int i, int j) { *reinterpret_cast<U*>(v.data + s_dst[j] + at) = held[i]; });
    }
  });
}

int check_views(const vxa_cache_view* caches, int64_t count, int64_t page) {
  for (int64_t i = 0; i < count; ++i) {
    const vxa_cache_view& c = caches[i];
    if (!c.data || c.heads <= 0 || c.row_bytes <= 0) return VXA_ERR_ARG;
    if (product({page, c.heads, c.row_bytes}) >= 1LL << 31) return VXA_ERR_UNSUPPORTED;
  }
  return VXA_OK;
}
Views views_of(const vxa_cache_view* caches, int64_t first, int64_t count) {
  Views v;
  for (int64_t i = 0; i < std::min<int64_t>(kViews, count - first); ++i) {
    const vxa_cache_view& c = caches[first + i];
    const uint64_t bits = (uint64_t)(uintptr_t)c.data | (uint64_t)c.stride_block | (uint64_t)c.stride_token | (uint64_t)c.stride_head | (uint64_t)c.row_bytes;
    const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
    v.at[i] = View{reinterpret_cast<char*>(c.data), c.stride_block, c.stride_token, c.stride_head, (int32_t)c.heads, (int32_t)c.row_bytes, unit};
  }
  return v;
}

constexpr int64_t kMostBlocks = 1 << 28;
// A resize that one workgroup does, an entry and four counts a thread: 16 rows of 64 entries and 4096 counts, in a replayed graph, 5.7 us in place of
// two launches' 6.0, and 4 us less of the host where it is called eagerly. Four entries a thread took 8.2 us in place of 6.0, 16 counts
// besides 9.6 in place of 6.6.
constexpr int64_t kSmallTable = kPlan, kSmallPool = 4 * kPlan;

// What fork and resize check of a table and its counts.
int check_table(int64_t rows, int64_t cols, int64_t num_blocks, int64_t page) {
  if (rows < 0 || cols < 0 || num_blocks < 0 || page <= 0) return VXA_ERR_ARG;
  if (rows > kMostRows || product({rows, cols}) >= 1LL << 31 || num_blocks > kMostBlocks || page >= 1LL << 31) return VXA_ERR_UNSUPPORTED;
  return VXA_OK;
}
// Workgroups of a plan: the first one plans, the others copy the counts.
unsigned plan_grid(const TableParams& p) { return p.out_refs == p.refs ? 1 : 1 + (unsigned)std::min<int64_t>(64, cdiv<int64_t>(p.num_blocks, kPlan)); }

}  // namespace

extern "C" int vxa_pages_copy(const vxa_cache_view* caches, int64_t count, int64_t num_blocks, int64_t block_size, const int32_t* source,
                              const int32_t* target, int64_t n, vxa_stream_t stream) {
  if (count < 0 || num_blocks < 0 || block_size <= 0 || n < 0 || (count && !caches)) return VXA_ERR_ARG;
  if (num_blocks > kMostBlocks || n > (1 << 22)) return VXA_ERR_UNSUPPORTED;
  const int rc = check_views(caches, count, block_size);
  if (rc != VXA_OK) return rc;
  if (n == 0 || count == 0 || num_blocks == 0) return VXA_OK;
  if (!source || !target) return VXA_ERR_ARG;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int64_t i = 0; i < count; i += kViews) {
    const Views views = views_of(caches, i, count);
    for (int64_t j = 0; j < n; j += kPairs) {
      const int pairs = (int)std::min<int64_t>(kPairs, n - j);
      hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)pairs, (unsigned)std::min<int64_t>(kViews, count - i)), dim3(256), 0, st, views, (int)num_blocks, (int)block_size, source + j,
                         target + j, pairs);
      VXA_CHECK_LAUNCH();
    }
  }
  return VXA_OK;
}

extern "C" int vxa_pages_fork_workspace(int64_t rows, int64_t new_rows, size_t* ws_bytes) {
  if (rows < 0 || new_rows < 0 || !ws_bytes) return VXA_ERR_ARG;
  if (std::max(rows, new_rows) > kMostRows) return VXA_ERR_UNSUPPORTED;
  *ws_bytes = (size_t)product({product({2, new_rows}) + rows, 4});
  return VXA_OK;
}

extern "C" int vxa_pages_fork(const vxa_cache_view* caches, int64_t count, const int32_t* block_table, int64_t stride_bt, int64_t cols,
                              const int32_t* seq_lens, int64_t rows, const int32_t* parents, int64_t new_rows, const int32_t* ref_count,
                              int64_t num_blocks, int64_t block_size, int32_t* out_table, int64_t stride_ot, int32_t* out_lens,
                              int32_t* out_ref_count, int32_t* missing, void* ws, size_t ws_bytes, vxa_stream_t stream) {
  int rc = check_table(rows, cols, num_blocks, block_size);
  if (rc == VXA_OK) rc = check_table(new_rows, cols, num_blocks, block_size);
  if (rc != VXA_OK) return rc;
  if (count < 0 || (count && !caches) || !missing || (num_blocks && (!ref_count || !out_ref_count))) return VXA_ERR_ARG;
  rc = check_views(caches, count, block_size);
  if (rc != VXA_OK) return rc;
  if ((rows && (!seq_lens || (cols && !block_table))) || (new_rows && (!parents || !out_lens || (cols && !out_table)))) return VXA_ERR_ARG;
  if (rows && new_rows && ((cols && block_table == out_table) || seq_lens == out_lens)) return VXA_ERR_ARG;  // rows read each other's
  size_t bytes = 0;
  vxa_pages_fork_workspace(rows, new_rows, &bytes);
  if (bytes && (!ws || (uintptr_t)ws % 4 || ws_bytes < bytes)) return VXA_ERR_WORKSPACE;
  TableParams p{};
  p.table = block_table, p.stride = stride_bt, p.cols = (int32_t)cols, p.rows = (int32_t)rows, p.lens = seq_lens;
  p.parents = parents, p.new_rows = (int32_t)new_rows, p.out_table = out_table, p.out_stride = stride_ot, p.out_lens = out_lens;
  p.refs = ref_count, p.out_refs = out_ref_count, p.num_blocks = (int32_t)num_blocks, p.page = (int32_t)block_size;
  p.missing = missing, p.ws = reinterpret_cast<int32_t*>(ws);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(pages_fork_plan_kernel, dim3(plan_grid(p)), dim3(kPlan), 0, st, p);
  VXA_CHECK_LAUNCH();
  const unsigned most = (unsigned)std::max(rows, new_rows);
  if (most == 0) return VXA_OK;
  hipLaunchKernelGGL(pages_fork_kernel, dim3(most, 1 + (unsigned)std::min<int64_t>(kViews, count)), dim3(256), 0, st, p, views_of(caches, 0, count));
  VXA_CHECK_LAUNCH();
  for (int64_t i = kViews; i < count && new_rows; i += kViews) {
    hipLaunchKernelGGL(pages_fork_copy_kernel, dim3((unsigned)new_rows, (unsigned)std::min<int64_t>(kViews, count - i)), dim3(256), 0, st, p, views_of(caches, i, count));
    VXA_CHECK_LAUNCH();
  }
  return VXA_OK;
}

extern "C" int vxa_pages_resize_workspace(int64_t rows, int64_t num_blocks, size_t* ws_bytes) {
  if (rows < 0 || num_blocks < 0 || !ws_bytes) return VXA_ERR_ARG;
  if (rows > kMostRows) return VXA_ERR_UNSUPPORTED;
  *ws_bytes = (size_t)product({rows + 1 + num_blocks, 4});
  return VXA_OK;
}

extern "C" int vxa_pages_resize(const int32_t* block_table, int64_t stride_bt, int64_t cols, const int32_t* seq_lens, const int32_t* new_lens,
                                int64_t rows, const int32_t* ref_count, int64_t num_blocks, int64_t block_size, int32_t* out_table,
                                int64_t stride_ot, int32_t* out_ref_count, int32_t* missing, void* ws, size_t ws_bytes, vxa_stream_t stream) {
  const int rc = check_table(rows, cols, num_blocks, block_size);
  if (rc != VXA_OK) return rc;
  if (!missing || (num_blocks && (!ref_count || !out_ref_count))) return VXA_ERR_ARG;
  if (rows && (!seq_lens || !new_lens || (cols && (!block_table || !out_table)))) return VXA_ERR_ARG;
  if (block_table == out_table && stride_bt != stride_ot) return VXA_ERR_ARG;
  size_t bytes = 0;
  vxa_pages_resize_workspace(rows, num_blocks, &bytes);
  if (!ws || (uintptr_t)ws % 4 || ws_bytes < bytes) return VXA_ERR_WORKSPACE;
  TableParams p{};
  p.table = block_table, p.stride = stride_bt, p.cols = (int32_t)cols, p.rows = (int32_t)rows, p.lens = seq_lens, p.new_lens = new_lens;
  p.out_table = out_table, p.out_stride = stride_ot, p.refs = ref_count, p.out_refs = out_ref_count;
  p.num_blocks = (int32_t)num_blocks, p.page = (int32_t)block_size, p.missing = missing, p.ws = reinterpret_cast<int32_t*>(ws);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (rows * cols <= kSmallTable && num_blocks <= kSmallPool) {
    hipLaunchKernelGGL(pages_resize_small_kernel, dim3(1), dim3(kPlan), 0, st, p);
    VXA_CHECK_LAUNCH();
    return VXA_OK;
  }
  hipLaunchKernelGGL(pages_resize_plan_kernel, dim3(plan_grid(p)), dim3(kPlan), 0, st, p);
  VXA_CHECK_LAUNCH();
  if (rows == 0) return VXA_OK;
  hipLaunchKernelGGL(pages_resize_kernel, dim3((unsigned)rows), dim3(256), 0, st, p);
  VXA_CHECK_LAUNCH();
  return VXA_OK;
}

extern "C" int vxa_pages_keep(const vxa_cache_view* caches, int64_t count, const int32_t* block_table, int64_t stride_bt, int64_t cols,
                              const int32_t* seq_lens, const int32_t* starts, const int64_t* keep, int64_t n, int64_t num_blocks,
                              int64_t block_size, int32_t* out_lens, vxa_stream_t stream) {
  if (n < 0 || cols < 0 || num_blocks < 0 || block_size <= 0 || count < 0 || (count && !caches)) return VXA_ERR_ARG;
  if (n > (1 << 22) || cols >= 1LL << 31 || num_blocks > kMostBlocks || block_size >= 1LL << 31) return VXA_ERR_UNSUPPORTED;
  const int rc = check_views(caches, count, block_size);
  if (rc != VXA_OK) return rc;
  if (n == 0) return VXA_OK;
  if ((cols && !block_table) || !seq_lens || !starts || !keep || !out_lens || out_lens == seq_lens) return VXA_ERR_ARG;
  const KeepParams p{block_table, stride_bt, (int32_t)cols, seq_lens, starts, keep, out_lens, (int32_t)num_blocks, (int32_t)block_size};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // Without caches the lengths alone are written, by a launch with a view of nothing.
  int64_t i = 0;
  do {
    const Views views = views_of(caches, i, count);
    int64_t slabs = 1;
    for (int64_t j = i; j < std::min(count, i + kViews); ++j)
      slabs = std::max(slabs, cdiv<int64_t>((int64_t)views.at[j - i].heads * (views.at[j - i].bytes / views.at[j - i].unit), kKeepWidth));
    Views none{};
    none.at[0].unit = 1;
    hipLaunchKernelGGL(pages_keep_kernel, dim3((unsigned)n, (unsigned)std::max<int64_t>(1, std::min<int64_t>(kViews, count - i)), (unsigned)std::min<int64_t>(slabs, 256)),
                       dim3(256), 0, st, p, count ? views : none, i == 0);
    VXA_CHECK_LAUNCH();
    i += kViews;
  } while (i < count);
  return VXA_OK;
}
