// grxDNN paged key-value cache on gfx950: new rows into the pages, and eviction
// by the weights that the slots accumulated.
//
// New: the reference plans attention for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships neither it nor a cache.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"

#include <algorithm>
#include <climits>

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
  PageDiv by_heads;
  int B, T, heads, tokens;    // tokens: of a tile
};

// Tiles of `tokens` new tokens of one sequence (blockIdx.y), their heads side by side: a
// thread copies a 16-byte chunk of a key and of a value of a row. Bound by memory, each row
// read and written once. The rows are written to stay in the caches: the next attention
// reads them. us, 8 x 4000 tokens of 8 heads of 128: 51.5 (5.1 TB/s); with four rows a
// thread, all loaded before the first is stored, 53.6; that and stores past the caches 50.5
// (but 8 x 2250 30.6 for 28.2); 64 tokens 4.9, 256 tokens 4.9.
template <int C>       // chunks of a row
__global__ __launch_bounds__(256) void paged_append(AppendParams p) {
  constexpr int R = 256 / C;
  const int c = threadIdx.x % C, first = threadIdx.x / C;
  const int rows = p.tokens * p.heads;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int n = clamp_length(p.view.lengths[b], p.view.room);
    const int T = min(p.counts ? min(p.counts[b], p.T) : p.T, p.view.room - n);   // the others have no place
    for (int64_t t0 = (int64_t)blockIdx.x * p.tokens; t0 < T; t0 += (int64_t)gridDim.x * p.tokens) {
      for (int r = first; r < rows; r += R) {
        const int i = div_page(p.by_heads, r), h = r - i * p.heads;
        const int64_t t = t0 + i;
        if (t >= T) break;
        int page, row;
        if (!find_slot(p.view, b, n + (int)t, &page, &row)) continue;
        const u32x4 key = __builtin_nontemporal_load(p.kn + b * p.kn_sb + h * p.kn_sh + t * p.kn_st + c);
        const u32x4 value = __builtin_nontemporal_load(p.vn + b * p.vn_sb + h * p.vn_sh + t * p.vn_st + c);
        p.k.row(page, h, row)[c] = key;
        p.v.row(page, h, row)[c] = value;
      }
    }
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
  int B, heads, budget, recent;
  int first;           // (sequence, head) of workgroup 0 of evict_select
};

constexpr int kWaves = 16;    // of a selecting workgroup

// Which slots a head keeps: one workgroup per (sequence, head). Wave w has the slots
// from 64 E w on, E to a lane, 64 neighbours at a time; E <= N of them in registers
// (N = 0: read again in every pass).
//  * The key of the last slot that stays is found from the top, two bits a step: how
//    many slots reach each of three keys, summed over the waves. Weights that differ
//    are told apart long before the last bit: the steps end when exactly as many slots
//    reach a key as stay, and once 64 or fewer lie between a key that too few reach and
//    one that enough do, those go on in registers without a barrier.
//  * Where every slot goes follows from the numbers of kept ones and of ties in the
//    waves before and ballots within the wave: no loop over the slots with a barrier.
// 128 heads of 6000 to 8192 slots to 2048: 19 us on the 128 CUs that have one, bound by the
// steps' latency: waves wait for loads, LDS and barriers in 59 % of their cycles, the VALU is
// at work in 38 %. A binary search over passes through memory, 256 threads, took 187. Where
// slots are read again (more than 32 a lane), 8 heads of 131072: 375 us.
template <int N>
__global__ __launch_bounds__(64 * kWaves) void evict_select(EvictParams p) {
  __shared__ int sums[2][3][kWaves], above_of[kWaves], ties_of[kWaves], few_n;
  __shared__ uint32_t few[64];
  const int bh = p.first + blockIdx.x, b = bh / p.heads, h = bh - b * p.heads, tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = clamp_length(p.view.lengths[b], p.view.room), m = min(n, p.budget);
  const int old = n <= p.budget ? 0 : max(0, n - p.recent);   // slots that the weights decide on
  const int want = n <= p.budget ? 0 : p.budget - p.recent;   // how many of them stay
  const float* w = p.w + b * p.w_sb + h * p.w_sh;
  const int E = (n + 64 * kWaves - 1) / (64 * kWaves), first = 64 * E * wave + lane;
  // A slot's key, 0 (which no weight has) where the weights do not decide.
  auto key_of = [&](int q) __attribute__((always_inline)) {
    const int j = first + 64 * q;
    return j < old ? order_key(__float_as_uint(w[j])) : 0;
  };
  uint32_t mine[N ? N : 1];
  if constexpr (N > 0)
#pragma unroll
    for (int q = 0; q < N; ++q) mine[q] = q < E ? key_of(q) : 0;
  // f(slot, key) for every row of 64 slots of the wave
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (N > 0) {
#pragma unroll
      for (int q = 0; q < (N ? N : 1); ++q)
        if (q < E) f(first + 64 * q, mine[q]);
    } else {
      for (int q = 0; q < E; ++q) f(first + 64 * q, key_of(q));
    }
  };

  uint32_t last = 0;       // slots whose key reaches it stay, or (ties) those above it and some of it
  bool ties = want > 0;
  int upper = 0, lower = INT_MAX;     // slots that reach last + 4 << bit, and last
  if (tid == 0) few_n = 0;
  for (int bit = 30, turn = 0; bit >= 0 && ties; bit -= 2, turn ^= 1) {
    uint32_t c[3] = {0, 0, 0};
    each([&](int, uint32_t key) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t d = 0; d < 3; ++d) c[d] += key >= (last | (d + 1) << bit);
    });
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      c[d] = wave_upto(c[d]);
      if (lane == 63) sums[turn][d][wave] = (int)c[d];
    }
    // One barrier a step: a wave that is a step ahead writes the other turn's sums.
    __syncthreads();
    uint32_t got = lane < 3 * kWaves ? (uint32_t)sums[turn][lane / kWaves][lane % kWaves] : 0;
    got = dpp_add<0x111, 0xf>(got);    // row_shr 1, 2, 4, 8: lanes 15, 31, 47 get their 16's sum
    got = dpp_add<0x112, 0xf>(got);
    got = dpp_add<0x114, 0xf>(got);
    got = dpp_add<0x118, 0xf>(got);
    static_assert(kWaves == 16, "a row of lanes per sum");
#pragma unroll
    for (int d = 2; d >= 0; --d) {
      const int s = __builtin_amdgcn_readlane((int)got, 16 * d + 15);
      if (s >= want) {
        last |= (uint32_t)(d + 1) << bit;
        lower = s;
        ties = s != want;
        break;
      }
      upper = s;
    }
    if (ties && bit && lower - upper <= 64) {
      // What is left between: each wave goes on by itself, a key to a lane.
      each([&](int, uint32_t key) __attribute__((always_inline)) {
        if ((key - last) >> bit) return;       // (as unsigned: below last too)
        const int at = atomicAdd(&few_n, 1);
        if (at < 64) few[at] = key;
      });
      __syncthreads();
      const uint32_t key = lane < lower - upper ? few[lane] : 0;
      for (int low = bit - 1; low >= 0 && ties; --low) {
        const int c = __popcll(__ballot(key >= (last | 1u << low)));
        if (c >= want - upper) {
          last |= 1u << low;
          ties = c != want - upper;
        }
      }
      break;
    }
  }
  // What stays: newer slots, old ones above `last`, and of those at it all or, where
  // more than fit tie, the lowest.
  auto above = [&](int j, uint32_t key) __attribute__((always_inline)) {
    return j < old ? want && (ties ? key > last : key >= last) : j < n;
  };
  auto tied = [&](int j, uint32_t key) __attribute__((always_inline)) { return ties && j < old && key == last; };
  int up = 0, at = 0;
  each([&](int j, uint32_t key) __attribute__((always_inline)) {
    up += __popcll(__ballot(above(j, key)));
    at += __popcll(__ballot(tied(j, key)));
  });
  if (lane == 0) {
    above_of[wave] = up;
    ties_of[wave] = at;
  }
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int x = 0; x < kWaves; ++x) total += above_of[x];
  int room = m - total, to = 0;      // ties that stay
#pragma unroll
  for (int x = 0; x < kWaves; ++x)
    if (x < wave) {
      const int some = min(room, ties_of[x]);
      to += above_of[x] + some;
      room -= some;
    }
  int* kept = p.kept + (int64_t)bh * p.budget;
  float* nw = p.nw + b * p.nw_sb + h * p.nw_sh;
  const uint64_t below = (1ull << lane) - 1;
  each([&](int j, uint32_t key) __attribute__((always_inline)) {
    const uint64_t tie = __ballot(tied(j, key));
    const bool stay = above(j, key) || (tied(j, key) && __popcll(tie & below) < room);
    const uint64_t all = __ballot(stay);
    const int i = to + __popcll(all & below);
    // (weights that change while they are read must not lead out of the arrays)
    if (stay && i < m) {
      kept[i] = j;
      nw[i] = w[j];
    }
    room -= min(room, __popcll(tie));
    to += __popcll(all);
  });
  for (int i = m + tid; i < p.budget; i += 64 * kWaves) kept[i] = -1;
  for (int64_t i = m + tid; i < p.nw_slots; i += 64 * kWaves) nw[i] = 0.0f;
}

// The kept rows of (sequence, head) blockIdx.y into the new pages: a thread copies a 16-byte
// chunk of a key and of a value of a row. Bound by memory: 128 heads of 2048 kept rows of
// 256 bytes, a quarter of those that lie between them, 268 MB in 56 us; four rows a thread
// took as long, and 1.6 us more in a call of 8 heads. The new lengths after every reader of
// lengths, which they may replace.
template <int C>
__global__ __launch_bounds__(256) void evict_copy(EvictParams p) {
  constexpr int R = 256 / C;
  const int c = threadIdx.x % C, first = threadIdx.x / C;
  for (int bh = blockIdx.y; bh < p.B * p.heads; bh += gridDim.y) {
    const int b = bh / p.heads, h = bh - b * p.heads;
    const int* kept = p.kept + (int64_t)bh * p.budget;
    for (int64_t r = (int64_t)blockIdx.x * R + first; r < p.budget; r += (int64_t)gridDim.x * R) {
      const int slot = kept[r];
      int page, row, new_page, new_row;
      const bool from = find_slot(p.view, b, max(slot, 0), &page, &row);
      const bool to = find_slot(p.to, b, (int)r, &new_page, &new_row);
      if (!((slot >= 0) & from & to)) continue;
      const u32x4 key = __builtin_nontemporal_load(p.k.row(page, h, row) + c);
      const u32x4 value = __builtin_nontemporal_load(p.v.row(page, h, row) + c);
      __builtin_nontemporal_store(key, p.k.row(new_page, h, new_row) + c);
      __builtin_nontemporal_store(value, p.v.row(new_page, h, new_row) + c);
    }
    if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0)
      p.new_lengths[b] = min(clamp_length(p.view.lengths[b], p.view.room), p.budget);
  }
}

// x by y workgroups, which loop where that is more than a million.
dim3 tiles_by(int64_t x, int64_t y) {
  y = std::min<int64_t>(y, 65535);
  return dim3((unsigned)std::min(x, std::max<int64_t>(1, (1 << 20) / y)), (unsigned)y);
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
  p.B = d.c.B; p.heads = d.c.heads; p.T = d.T;
  p.by_heads = page_div(p.heads);
  const int chunks = d.c.D / 8;
  p.tokens = (int)std::max<int64_t>(1, 256 / ((int64_t)p.heads * chunks));
  const int64_t tiles = ((int64_t)p.T + p.tokens - 1) / p.tokens;
  const dim3 grid = tiles_by(tiles, p.B);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, p); };
  if (chunks == 16) go(paged_append<16>);
  else go(paged_append<8>);
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
  p.B = d.c.B; p.heads = d.c.heads; p.budget = d.budget; p.recent = d.recent;
  const int64_t heads = (int64_t)p.B * p.heads;
  const int each = (p.view.room + 64 * kWaves - 1) / (64 * kWaves);
  for (int64_t first = 0; first < heads; first += max_workgroups(64 * kWaves)) {
    p.first = (int)first;
    const dim3 some((unsigned)std::min(heads - first, max_workgroups(64 * kWaves))), threads(64 * kWaves);
    if (each <= 8) hipLaunchKernelGGL(evict_select<8>, some, threads, 0, s, p);
    else if (each <= 32) hipLaunchKernelGGL(evict_select<32>, some, threads, 0, s, p);
    else hipLaunchKernelGGL(evict_select<0>, some, threads, 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int chunks = d.c.D / 8, rows = 256 / chunks;
  const dim3 grid = tiles_by((p.budget + (int64_t)rows - 1) / rows, heads);
  if (chunks == 16) hipLaunchKernelGGL(evict_copy<16>, grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL(evict_copy<8>, grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace grxk
