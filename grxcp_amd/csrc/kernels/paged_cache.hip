// grxDNN paged key-value cache on gfx950: new rows into the pages, and eviction
// by the weights that the slots accumulated.
//
// New: the reference plans attention for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships neither it nor a cache.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"

#include <algorithm>

namespace grxk {
namespace {

PagedView view_of(const PagedCache& c) {
  return {c.table, c.table_rs, c.lengths, c.pages, c.page, c.W * c.page, page_div(c.page)};
}

// A pool as the kernels address it: strides in 16-byte chunks.
struct Pool {
  u32x4* p;
  int64_t sp, sh, ss;
  __device__ __forceinline__ u32x4* row(int page, int h, int slot) const { return p + page * sp + h * sh + slot * ss; }
};
Pool k_pool(const PagedCache& c) { return {(u32x4*)c.k, c.k_sp / 8, c.k_sh / 8, c.k_ss / 8}; }
Pool v_pool(const PagedCache& c) { return {(u32x4*)c.v, c.v_sp / 8, c.v_sh / 8, c.v_ss / 8}; }

// ---- append ------------------------------------------------------------------

struct AppendParams {
  PagedView view;
  Pool k, v;
  const u32x4* kn; int64_t kn_sb, kn_sh, kn_st;   // chunks
  const u32x4* vn; int64_t vn_sb, vn_sh, vn_st;
  const int* counts;
  int B, heads, T, chunks;                        // 16-byte chunks of a row
};

// One 16-byte chunk of a key and of a value per thread.
__global__ __launch_bounds__(256) void paged_append(AppendParams p) {
  const int64_t total = (int64_t)p.B * p.T * p.heads * p.chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int c = (int)(i % p.chunks);
    int64_t r = i / p.chunks;
    const int h = (int)(r % p.heads);
    r /= p.heads;
    const int t = (int)(r % p.T), b = (int)(r / p.T);
    if (p.counts && t >= p.counts[b]) continue;
    const int64_t slot = (int64_t)clamp_length(p.view.lengths[b], p.view.room) + t;
    int page, row;
    if (slot >= p.view.room || !find_slot(p.view, b, (int)slot, &page, &row)) continue;
    p.k.row(page, h, row)[c] = p.kn[b * p.kn_sb + h * p.kn_sh + t * p.kn_st + c];
    p.v.row(page, h, row)[c] = p.vn[b * p.vn_sb + h * p.vn_sh + t * p.vn_st + c];
  }
}

// ---- evict -------------------------------------------------------------------

struct EvictParams {
  PagedView view, to;
  Pool k, v;
  const float* w; int64_t w_sb, w_sh;
  float* nw; int64_t nw_sb, nw_sh; int nw_slots;
  int* kept;
  int* new_lengths;
  int B, heads, budget, recent, chunks;
};

__device__ __forceinline__ uint32_t key_at(const float* w, int j) { return order_key(__float_as_uint(w[j])); }

// Sum of v over the 256 threads, in every thread.
__device__ __forceinline__ int block_sum(int v, int* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// Which slots a head keeps: one workgroup per (sequence, head). The key of the
// last slot that stays is found bit by bit from the top.
__global__ __launch_bounds__(256) void evict_select(EvictParams p) {
  __shared__ int red[4];
  const int bh = blockIdx.x, b = bh / p.heads, h = bh - b * p.heads, tid = threadIdx.x;
  const int n = clamp_length(p.view.lengths[b], p.view.room), m = min(n, p.budget);
  const int old = n <= p.budget ? 0 : max(0, n - p.recent);   // slots that the weights decide on
  const int want = n <= p.budget ? 0 : p.budget - p.recent;   // how many of them stay
  const float* w = p.w + b * p.w_sb + h * p.w_sh;
  uint32_t last = 0;       // largest key that at least `want` slots reach
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = last | (1u << bit);
    int c = 0;
    for (int j = tid; j < old; j += 256) c += key_at(w, j) >= t;
    if (block_sum(c, red) >= want) last = t;
  }
  int c = 0;
  for (int j = tid; j < old; j += 256) c += key_at(w, j) > last;
  int ties = want - block_sum(c, red);                        // lowest slots with the last key
  int* kept = p.kept + (int64_t)bh * p.budget;
  float* nw = p.nw + b * p.nw_sb + h * p.nw_sh;
  // In slot order, 256 slots at a time: tied ones before, kept ones before.
  __shared__ int before[2][4];
  int at = 0;
  for (int j0 = 0; j0 < n; j0 += 256) {
    const int j = j0 + tid;
    const uint32_t key = j < old ? key_at(w, j) : 0;
    const bool tie = j < old && key == last;
    const uint64_t tmask = __ballot(tie), below = (1ull << (tid & 63)) - 1;
    __syncthreads();
    if ((tid & 63) == 0) before[0][tid >> 6] = __popcll(tmask);
    __syncthreads();
    int rank = __popcll(tmask & below);
    for (int i = 0; i < tid >> 6; ++i) rank += before[0][i];
    const bool stay = j < n && (j >= old || key > last || (tie && rank < ties));
    ties -= before[0][0] + before[0][1] + before[0][2] + before[0][3];
    const uint64_t smask = __ballot(stay);
    if ((tid & 63) == 0) before[1][tid >> 6] = __popcll(smask);
    __syncthreads();
    int to = at + __popcll(smask & below);
    for (int i = 0; i < tid >> 6; ++i) to += before[1][i];
    if (stay) {
      kept[to] = j;
      nw[to] = w[j];
    }
    at += before[1][0] + before[1][1] + before[1][2] + before[1][3];
  }
  for (int i = m + tid; i < p.budget; i += 256) kept[i] = -1;
  for (int i = m + tid; i < p.nw_slots; i += 256) nw[i] = 0.0f;
}

// The kept rows into the new pages, a 16-byte chunk of a key and of a value per
// thread; the new lengths (after every reader of lengths, which they may replace).
__global__ __launch_bounds__(256) void evict_copy(EvictParams p) {
  const int64_t total = (int64_t)p.B * p.heads * p.budget * p.chunks;
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t i = first; i < total; i += step) {
    const int c = (int)(i % p.chunks);
    const int64_t r = i / p.chunks;
    const int slot = p.kept[r];
    if (slot < 0) continue;
    const int to = (int)(r % p.budget);
    const int bh = (int)(r / p.budget), b = bh / p.heads, h = bh - b * p.heads;
    int page, row, new_page, new_row;
    if (!find_slot(p.view, b, slot, &page, &row) || !find_slot(p.to, b, to, &new_page, &new_row)) continue;
    p.k.row(new_page, h, new_row)[c] = p.k.row(page, h, row)[c];
    p.v.row(new_page, h, new_row)[c] = p.v.row(page, h, row)[c];
  }
  for (int64_t b = first; b < p.B; b += step)
    p.new_lengths[b] = min(clamp_length(p.view.lengths[b], p.view.room), p.budget);
}

unsigned blocks(int64_t threads) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 1 << 20));
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendDesc& d, hipStream_t s) {
  AppendParams p{};
  p.view = view_of(d.c);
  p.k = k_pool(d.c);
  p.v = v_pool(d.c);
  p.kn = (const u32x4*)d.k; p.kn_sb = d.k_sb / 8; p.kn_sh = d.k_sh / 8; p.kn_st = d.k_st / 8;
  p.vn = (const u32x4*)d.v; p.vn_sb = d.v_sb / 8; p.vn_sh = d.v_sh / 8; p.vn_st = d.v_st / 8;
  p.counts = d.counts;
  p.B = d.c.B; p.heads = d.c.heads; p.T = d.T; p.chunks = d.c.D / 8;
  const int64_t total = (int64_t)p.B * p.T * p.heads * p.chunks;
  hipLaunchKernelGGL(paged_append, dim3(blocks(total)), dim3(256), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_paged_evict(const PagedEvictDesc& d, hipStream_t s) {
  EvictParams p{};
  p.view = view_of(d.c);
  p.to = p.view;
  p.to.table = d.new_table;
  p.to.table_rs = d.new_table_rs;
  p.to.room = d.new_W * d.c.page;
  p.k = k_pool(d.c);
  p.v = v_pool(d.c);
  p.w = d.weights; p.w_sb = d.w_sb; p.w_sh = d.w_sh;
  p.nw = d.new_weights; p.nw_sb = d.nw_sb; p.nw_sh = d.nw_sh; p.nw_slots = d.nw_slots;
  p.kept = d.kept;
  p.new_lengths = d.new_lengths;
  p.B = d.c.B; p.heads = d.c.heads; p.budget = d.budget; p.recent = d.recent; p.chunks = d.c.D / 8;
  if ((int64_t)p.B * p.heads > max_workgroups(256)) return hipErrorNotSupported;
  hipLaunchKernelGGL(evict_select, dim3((unsigned)(p.B * p.heads)), dim3(256), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t total = (int64_t)p.B * p.heads * p.budget * p.chunks;
  hipLaunchKernelGGL(evict_copy, dim3(blocks(total)), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace grxk
