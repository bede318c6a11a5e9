// grxDNN attention of one new token per sequence over a paged key-value cache, on
// gfx950.
//
// New: the reference plans attention for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships no code.
//
// Every key and value is read once, for the whole group of query heads that share
// it, so the call is bound by reading the cache: 4 flops per query head and byte
// pair. What carries that:
//
//  * the cache of all sequences and key heads is one list of units of 128 slots of
//    one head, which the workgroups divide evenly (decode_split): whatever the
//    sequences' lengths, every CU reads the same share. The lengths are device
//    data, so each workgroup finds its share by a scan of them. A share that ends
//    inside a sequence leaves a partial result (O without its division, running
//    maximum, sum) and decode_join adds those up, in the order of the slots;
//  * a unit's four tiles of 32 slots go to the workgroup's four waves, each with a
//    running maximum, sum and O of its own: no barrier until a share's part of a
//    sequence ends and the four meet in LDS;
//  * scores are S^T = K Q^T (v_mfma_16x16x32), 16 query heads at a time, the K rows
//    in registers straight from memory. A group of fewer heads leaves columns
//    empty: the matrix cores have the time (16 MFMAs per 16 KB of cache);
//  * O^T += V^T P^T: the scores' lanes hold P^T as the B operand wants it if the
//    contraction runs over slots in the order 4g .. 4g+3, 16+4g .. 16+4g+3 (g: 16
//    lanes), and the V^T operand comes from the row-major V tile in LDS by the
//    transposing LDS read. V rows go to LDS without registers
//    (global_load_lds_dwordx4), chunks of 16 bytes XORed with the row so that a read
//    of 8 rows touches every bank once;
//  * the next tile's K and V are in flight while one is computed, and the page table
//    is read a tile further ahead: 16 KB per wave and tile, 8 waves per CU;
//  * slots that are not there (past the length, or on a page that does not exist)
//    read a row of zeros in place of what their page holds, and their scores are
//    -inf, so nothing stale reaches a sum.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"

#include <algorithm>

namespace grxk {
namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;                 // slots of a wave's tile
constexpr int kUnit = kWaves * kTile;     // slots of a unit
constexpr float kLowest = -__FLT_MAX__;
constexpr uint32_t kAbsent = 0x7fc0dead;  // a score of no slot (a NaN that no arithmetic gives)
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;

template <int N> struct Buf { static constexpr int value = N; };

// What a slot that is not there is read from: D values of zero.
__device__ __attribute__((aligned(256))) uint32_t zero_row[64];

template <AttnType T> struct PIo;
template <> struct PIo<AttnType::BF16> {
  // The weights' scale: exp2 of a score is at most 2^4 (kLazy) times this.
  static constexpr float kTop = 0.0f;
  __device__ static f32x4 mma(i32x4 a, i32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
  }
  __device__ static uint32_t pack2(float a, float b) { return pack_bf16x2(a, b); }
};
template <> struct PIo<AttnType::F16> {
  // Up to 2^15 of fp16's 65504, so that weights down to 2^-25 of the largest one keep
  // all of their bits: thousands of small ones may outweigh it together.
  static constexpr float kTop = 11.0f;
  __device__ static f32x4 mma(i32x4 a, i32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                  0, 0, 0);
  }
  __device__ static uint32_t pack2(float a, float b) { return pack_f16x2(a, b); }
};
// The running maximum moves only when a tile's exceeds it by more than this, so
// that O is rarely rescaled.
constexpr float kLazy = 4.0f;

struct DParams {
  PagedView view;
  const uint8_t* k; int64_t k_sp, k_sh, k_ss;   // byte strides of page, head, slot
  const uint8_t* v; int64_t v_sp, v_sh, v_ss;
  const uint8_t* q; int64_t q_sb, q_sh;
  uint8_t* o; int64_t o_sb, o_sh;
  float* w; int64_t w_sb, w_sh;
  float decay;
  float* ml;           // partial maxima and sums [parts, rows, 2]
  float* po;           // partial O [parts, rows, D]
  float* scores;       // [B, H, slots], or null: no weights asked for
  int64_t slots;
  int B, H, heads, group;
  int gtiles;          // tiles of 16 * NT query heads in a group
  int items;           // (key head, tile) pairs of a sequence
  int rows;            // query heads of a tile
  int wgs;             // workgroups of decode_split
  int whole;           // one workgroup per item, nothing to join
  float c;             // scale * log2(e)
};

// ---- who does what -----------------------------------------------------------

__device__ __forceinline__ int units_of(int len) { return max(1, (len + kUnit - 1) / kUnit); }

__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor((long long)v, o);
  return v;
}

// Units of one head of the sequences before b (b = B: of all).
__device__ __forceinline__ int64_t units_before(const DParams& p, int b, int lane) {
  int64_t s = 0;
  for (int i = lane; i < b; i += 64) s += units_of(clamp_length(p.view.lengths[i], p.view.room));
  return wave_sum64(s);
}

// Of `total` units share w of n is [total w / n, total (w + 1) / n): one to each
// workgroup, but none is empty.
__device__ __forceinline__ int64_t shares(const DParams& p, int64_t total) { return min((int64_t)p.wgs, total); }
// The share that holds unit u.
__device__ __forceinline__ int share_of(int64_t u, int64_t total, int64_t n) {
  return (int)((uint64_t)((u + 1) * n - 1) / (uint64_t)total);
}

// ---- the split -----------------------------------------------------------------

__device__ __forceinline__ void wait_all() {
  __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_ptr_t)p; }
// 16 bytes per lane from memory straight into LDS (lane L writes lds + 16 L), as
// assembly so that the compiler does not make every LDS read wait for it: the
// tile loop waits itself, before the tile is used. M0 holds the LDS address and
// needs a wait state before the load that reads it.
__device__ __forceinline__ void dma16(const uint8_t* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}

// 16-byte chunk of a V row in LDS: chunk ^ vswz(row).
template <int D> __device__ __forceinline__ int vswz(int row) {
  if constexpr (D == 128) return 2 * (row & 7);
  else return 2 * ((row >> 1) & 3);
}

// op over the four lanes that hold one query: l, l ^ 16, l ^ 32, l ^ 48.
template <class Op> __device__ __forceinline__ float over_query(float v, Op op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <AttnType T, int D, int NT>
__global__ __launch_bounds__(64 * kWaves, 2) void decode_split(DParams p) {
  using IO = PIo<T>;
  constexpr int F = D / 32;          // contraction steps of a score
  constexpr int DT = D / 16;         // tiles of the head dimension
  constexpr int CH = D / 8;          // chunks of a row
  constexpr int RPI = 64 / CH;       // V rows per load
  constexpr int kStage = kTile * CH; // chunks of a V tile
  constexpr int kPitch = D + 4;
  constexpr int kV = kWaves * 2 * kStage * 16, kMerge = kWaves * 16 * kPitch * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kV > kMerge ? kV : kMerge];
  __shared__ uint64_t rows[kWaves][2][kTile];
  __shared__ float ml[kWaves][2][16];

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // The share: sequence b, item `it` of it, from unit `i` on, `left` units.
  int b = 0, it = 0, i = 0;
  int64_t left;
  if (p.whole) {
    b = blockIdx.x / p.items;
    it = blockIdx.x - b * p.items;
    left = units_of(clamp_length(p.view.lengths[b], p.view.room));
  } else {
    const int64_t total = units_before(p, p.B, lane) * p.items;
    const int64_t parts = shares(p, total);
    if (blockIdx.x >= parts) return;
    const int64_t u0 = total * blockIdx.x / parts;
    left = total * (blockIdx.x + 1) / parts - u0;
    int64_t base = 0;                // units of the sequences before this 64
    for (int b0 = 0;; b0 += 64) {
      const int mine = b0 + lane < p.B ? units_of(clamp_length(p.view.lengths[b0 + lane], p.view.room)) : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int64_t below = __shfl_up((long long)upto, o);
        if (lane >= o) upto += below;
      }
      const uint64_t past = __ballot((base + upto) * p.items > u0);
      if (past) {                    // u0 < total: some sequence ends past it
        const int at = __ffsll((unsigned long long)past) - 1;
        b = b0 + at;
        const int64_t first = (base + __shfl((long long)(upto - mine), at)) * p.items;
        const int n = __shfl(mine, at);
        it = (int)((u0 - first) / n);
        i = (int)((u0 - first) - (int64_t)it * n);
        break;
      }
      base += __shfl((long long)upto, 63);
    }
  }
  b = __builtin_amdgcn_readfirstlane(b);
  it = __builtin_amdgcn_readfirstlane(it);
  i = __builtin_amdgcn_readfirstlane(i);

  uint8_t* vt = smem + wave * 2 * kStage * 16;
  const int kk = lane & 31;
  const bool second = lane >= 32;    // this half of the wave finds the V rows

  while (left > 0) {
    const int len = __builtin_amdgcn_readfirstlane(clamp_length(p.view.lengths[b], p.view.room));
    const int n = units_of(len);
    const int take = (int)min(left, (int64_t)(n - i));
    const int h = it / p.gtiles, q0 = (it - h * p.gtiles) * 16 * NT;   // key head, first query head of the group
    const int* table = p.view.table + b * p.view.table_rs;
    const uint8_t* base = second ? p.v + h * p.v_sh : p.k + h * p.k_sh;
    const int64_t sp = second ? p.v_sp : p.k_sp, ss = second ? p.v_ss : p.k_ss;

    i32x4 qf[NT][F];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = q0 + 16 * t + l16;
      const uint8_t* src = r < p.group ? p.q + b * p.q_sb + (h * p.group + r) * p.q_sh : (const uint8_t*)zero_row;
#pragma unroll
      for (int f = 0; f < F; ++f) qf[t][f] = *(const i32x4*)(src + 64 * f + 16 * g);
    }

    f32x4 o[NT][DT];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -INFINITY;              // no slot yet
      l[t] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    i32x4 kf[2][2][F];
    uint32_t live[2];
    int key = i * kUnit + wave * kTile;                                // the wave's first slot
    const int end = min(len, (i + take) * kUnit);
    auto entry = [&](int key0) __attribute__((always_inline)) {
      const int j = key0 + kk;
      return j < end ? table[div_page(p.view.div, j)] : -1;
    };
    // Loads of the tile at key0, whose table entries are e, into buffer BUF.
    auto issue = [&](auto buf, int key0, int e) __attribute__((always_inline)) {
      constexpr int BUF = decltype(buf)::value;
      const int j = key0 + kk;
      const int page = j < end ? checked_page(e, p.view.pages) : -1;
      const int row = j - div_page(p.view.div, j) * p.view.page;
      rows[wave][second][kk] = (uint64_t)(page >= 0 ? base + page * sp + row * ss : (const uint8_t*)zero_row);
      live[BUF] = (uint32_t)__ballot(page >= 0);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const uint8_t* src = (const uint8_t*)rows[wave][0][16 * kt + l16] + 16 * g;
#pragma unroll
        for (int f = 0; f < F; ++f) kf[BUF][kt][f] = *(const i32x4*)(src + 64 * f);
      }
#pragma unroll
      for (int x = 0; x < kTile / RPI; ++x) {
        const int r = RPI * x + lane / CH;
        const uint8_t* src = (const uint8_t*)rows[wave][1][r] + 16 * ((lane % CH) ^ vswz<D>(r));
        dma16(src, lds_addr(vt + (BUF * kStage + 64 * x) * 16));
      }
    };
    auto compute = [&](auto buf, int key0) __attribute__((always_inline)) {
      constexpr int BUF = decltype(buf)::value;
      const uint32_t mask = live[BUF];
      if (!mask && !p.scores) return;            // nothing to add and nothing to say
      i32x4 pf[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 s[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          s[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int f = 0; f < F; ++f) s[kt] = IO::mma(kf[BUF][kt][f], qf[t][f], s[kt]);
          s[kt] *= p.c;
        }
        if (mask != 0xffffffffu) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!(mask >> (16 * kt + 4 * g + r) & 1)) s[kt][r] = -INFINITY;
        }
        if (p.scores) {
          const int r = q0 + 16 * t + l16;
          if (r < p.group) {
            float* to = p.scores + ((int64_t)b * p.H + h * p.group + r) * p.slots + key0 + 4 * g;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
              f32x4 x = s[kt];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(mask >> (16 * kt + 4 * g + e) & 1)) x[e] = __uint_as_float(kAbsent);
              *(f32x4*)(to + 16 * kt) = x;
            }
          }
        }
        if (!mask) continue;
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = over_query(mx, [](float a, float x) { return fmaxf(a, x); });
        mx = fmaxf(mx, kLowest);     // -inf scores weigh 0; a row of only such has l = 0 and is NaN
        const bool raise = mx - m[t] > kLazy;
        if (__ballot(raise)) {
          const float top = raise ? mx : m[t];
          const float alpha = raise ? __builtin_amdgcn_exp2f(m[t] - top) : 1.0f;
          m[t] = top;
          l[t] *= alpha;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[t][d] *= alpha;
        }
        float w[2][4];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // the difference first: it is exact where scores are so large that a
            // rounding of the sum would tell
            w[kt][r] = __builtin_amdgcn_exp2f((s[kt][r] - m[t]) + IO::kTop);
            l[t] += w[kt][r];
          }
        pf[t] = i32x4{(int)IO::pack2(w[0][0], w[0][1]), (int)IO::pack2(w[0][2], w[0][3]),
                      (int)IO::pack2(w[1][0], w[1][1]), (int)IO::pack2(w[1][2], w[1][3])};
      }
      if (!mask) return;
      const uint8_t* v0 = vt + BUF * kStage * 16;
      const int r0 = 4 * g + (l16 >> 2), r1 = r0 + 16;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int c = 2 * d + ((lane >> 1) & 1);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4_t)(v0 + r0 * 2 * D + 16 * (c ^ vswz<D>(r0)) + 8 * (lane & 1)));
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4_t)(v0 + r1 * 2 * D + 16 * (c ^ vswz<D>(r1)) + 8 * (lane & 1)));
        const u32x2 w0 = __builtin_bit_cast(u32x2, a), w1 = __builtin_bit_cast(u32x2, x);
        const i32x4 vf = {(int)w0.x, (int)w0.y, (int)w1.x, (int)w1.y};
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][d] = IO::mma(vf, pf[t], o[t][d]);
      }
    };
    int e = entry(key);
    int next = entry(key + kUnit);
    if (key < end) issue(Buf<0>{}, key, e);
    while (key < end) {
      wait_all();
      if (key + kUnit < end) {
        issue(Buf<1>{}, key + kUnit, next);
        next = entry(key + 2 * kUnit);
      }
      compute(Buf<0>{}, key);
      key += kUnit;
      if (key >= end) break;
      wait_all();
      if (key + kUnit < end) {
        issue(Buf<0>{}, key + kUnit, next);
        next = entry(key + 2 * kUnit);
      }
      compute(Buf<1>{}, key);
      key += kUnit;
    }

    // The waves' results meet: rows of 16 query heads at a time.
    const bool whole = take == n;
    const int64_t part = p.whole ? blockIdx.x : (int64_t)b * p.items + it + blockIdx.x;
    float* mo = (float*)smem;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      wait_all();
      __syncthreads();               // every wave is done with its tiles, or with the rows before
#pragma unroll
      for (int d = 0; d < DT; ++d) *(f32x4*)&mo[(wave * 16 + l16) * kPitch + 16 * d + 4 * g] = o[t][d];
      const float sum = over_query(l[t], [](float a, float x) { return a + x; });
      if (g == 0) {
        ml[wave][0][l16] = m[t];
        ml[wave][1][l16] = sum;
      }
      __syncthreads();
      constexpr int E = D / 16;      // values of a thread
      const int r = tid >> 4, d0 = (tid & 15) * E;
      float top = ml[0][0][r];
#pragma unroll
      for (int x = 1; x < kWaves; ++x) top = fmaxf(top, ml[x][0][r]);
      float lsum = 0.0f, acc[E];
#pragma unroll
      for (int y = 0; y < E; ++y) acc[y] = 0.0f;
#pragma unroll
      for (int x = 0; x < kWaves; ++x) {
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[x][0][r] - top);
        lsum = fmaf(f, ml[x][1][r], lsum);
#pragma unroll
        for (int y = 0; y < E; ++y) acc[y] = fmaf(f, mo[(x * 16 + r) * kPitch + d0 + y], acc[y]);
      }
      const int row = 16 * t + r;    // in the tile
      if (q0 + row < p.group) {
        if (whole) {
          const float inv = top == -INFINITY ? 0.0f : 1.0f / lsum;   // no slot: 0; only -inf scores: 0 * inf
          uint32_t out[E / 2];
#pragma unroll
          for (int y = 0; y < E / 2; ++y) out[y] = IO::pack2(acc[2 * y] * inv, acc[2 * y + 1] * inv);
          uint8_t* to = p.o + b * p.o_sb + (h * p.group + q0 + row) * p.o_sh + 2 * d0;
          if constexpr (E == 8) *(u32x4*)to = u32x4{out[0], out[1], out[2], out[3]};
          else *(u32x2*)to = u32x2{out[0], out[1]};
        } else {
          float* to = p.po + (part * p.rows + row) * D + d0;
#pragma unroll
          for (int y = 0; y < E; y += 4) *(f32x4*)(to + y) = f32x4{acc[y], acc[y + 1], acc[y + 2], acc[y + 3]};
        }
        if (d0 == 0 && (!whole || p.scores)) {
          p.ml[(part * p.rows + row) * 2] = top;
          p.ml[(part * p.rows + row) * 2 + 1] = lsum;
        }
      }
    }
    wait_all();
    __syncthreads();                 // the tiles' LDS is free again

    left -= take;
    i = 0;
    if (++it == p.items) {
      it = 0;
      ++b;
    }
  }
}

// ---- the join ------------------------------------------------------------------

// Parts [first, first + count) of item `it` of sequence b.
struct Parts {
  int64_t first;
  int count;
};
__device__ __forceinline__ Parts parts_of(const DParams& p, int b, int it, int64_t before, int64_t total, int n) {
  const int64_t item = (int64_t)b * p.items + it;
  if (p.whole) return {item, 1};
  const int64_t u = before * p.items + (int64_t)it * n;
  const int64_t wgs = shares(p, total);
  const int w0 = share_of(u, total, wgs), w1 = share_of(u + n - 1, total, wgs);
  return {item + w0, w1 - w0 + 1};
}

// Workgroups below `heads` of the grid add up the parts of one query head's O; the
// others give 1024 slots of a key head their weights.
template <AttnType T, int D>
__global__ __launch_bounds__(256) void decode_join(DParams p, int64_t outs, int64_t chunks, int64_t jobs) {
  using IO = PIo<T>;
  constexpr int LD = D / 4, NP = 256 / LD;   // lanes of a part, parts at a time
  __shared__ float red[NP][D], top4[4], lred[NP];
  __shared__ float stat[1024][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t total = p.whole ? 0 : units_before(p, p.B, lane) * p.items;
  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const bool weights = job >= outs;
    const int64_t bh = weights ? (job - outs) / chunks : job;
    const int b = (int)(bh / (weights ? p.heads : p.H));
    const int head = (int)(bh - (int64_t)b * (weights ? p.heads : p.H));
    const int len = clamp_length(p.view.lengths[b], p.view.room), n = units_of(len);
    const int64_t before = p.whole ? 0 : units_before(p, b, lane);
    if (!weights) {
      const int h = head / p.group, r = head - h * p.group;
      const int gt = r / p.rows, row = r - gt * p.rows;
      const Parts x = parts_of(p, b, h * p.gtiles + gt, before, total, n);
      if (x.count == 1) continue;            // decode_split had all of it
      const float* ml = p.ml + (x.first * p.rows + row) * 2;
      const float* po = p.po + (x.first * p.rows + row) * D;
      float top = -INFINITY;
      for (int y = tid; y < x.count; y += 256) top = fmaxf(top, ml[(int64_t)y * p.rows * 2]);
      top = wave_max(top);
      __syncthreads();
      if (lane == 0) top4[wave] = top;
      __syncthreads();
      top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
      const int part = tid / LD, d = (tid % LD) * 4;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
      float l = 0.0f;
      for (int y = part; y < x.count; y += NP) {
        const float* s = ml + (int64_t)y * p.rows * 2;
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s[0] - top);
        l = fmaf(f, s[1], l);
        acc += *(const f32x4*)(po + (int64_t)y * p.rows * D + d) * f;
      }
      *(f32x4*)&red[part][d] = acc;
      if (d == 0) lred[part] = l;
      __syncthreads();
      if (tid < D / 2) {
        float a0 = 0.0f, a1 = 0.0f, sum = 0.0f;
#pragma unroll
        for (int y = 0; y < NP; ++y) {
          a0 += red[y][2 * tid];
          a1 += red[y][2 * tid + 1];
          sum += lred[y];
        }
        const float inv = top == -INFINITY ? 0.0f : 1.0f / sum;
        *(uint32_t*)(p.o + b * p.o_sb + head * p.o_sh + 4 * tid) = IO::pack2(a0 * inv, a1 * inv);
      }
      __syncthreads();
      continue;
    }
    const int j0 = (int)((job - outs) % chunks) * 1024;
    if (j0 >= len) continue;
    __syncthreads();
    for (int r = tid; r < p.group; r += 256) {
      const int gt = r / p.rows, row = r - gt * p.rows;
      const Parts x = parts_of(p, b, head * p.gtiles + gt, before, total, n);
      const float* ml = p.ml + (x.first * p.rows + row) * 2;
      float top = -INFINITY, l = 0.0f;
      for (int y = 0; y < x.count; ++y) top = fmaxf(top, ml[(int64_t)y * p.rows * 2]);
      for (int y = 0; y < x.count; ++y) {
        const float* s = ml + (int64_t)y * p.rows * 2;
        if (top != -INFINITY) l = fmaf(__builtin_amdgcn_exp2f(s[0] - top), s[1], l);
      }
      stat[r][0] = top;
      stat[r][1] = __builtin_amdgcn_exp2f(IO::kTop) / l;   // the sum has the weights' scale
    }
    __syncthreads();
    float* w = p.w + b * p.w_sb + head * p.w_sh;
    const float* sc = p.scores + ((int64_t)b * p.H + head * p.group) * p.slots;
    for (int j = j0 + tid; j < min(len, j0 + 1024); j += 256) {
      float a = 0.0f;
      for (int r = 0; r < p.group; ++r) {
        const float s = sc[(int64_t)r * p.slots + j];
        if (__float_as_uint(s) != kAbsent) a = fmaf(__builtin_amdgcn_exp2f(s - stat[r][0]), stat[r][1], a);
      }
      w[j] = p.decay == 0.0f ? a : fmaf(p.decay, w[j], a);
    }
  }
}

// ---- launch --------------------------------------------------------------------

struct Plan {
  int nt, gtiles, rows, wgs;
  bool whole;
  int64_t items, slots;
  size_t ml, po, scores;     // floats of the workspace, 16-byte multiples
};

int compute_units() {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  return std::max(8, cus / 8 * 8);
}

Plan plan_of(int B, int H, int heads, int D, int W, int page, bool weights) {
  Plan x{};
  const int group = H / heads;
  x.nt = group > 16 ? 2 : 1;
  x.gtiles = (group + 16 * x.nt - 1) / (16 * x.nt);
  x.rows = std::min(group, 16 * x.nt);
  x.items = (int64_t)B * heads * x.gtiles;
  x.slots = ((int64_t)W * page + kUnit - 1) / kUnit * kUnit;
  x.whole = (int64_t)W * page <= 2 * kUnit && x.items <= (1 << 20);
  x.wgs = x.whole ? (int)x.items : 2 * compute_units();
  const size_t parts = x.whole ? (size_t)x.items : (size_t)x.items + x.wgs;
  if (weights || !x.whole) x.ml = (parts * x.rows * 2 + 3) / 4 * 4;
  if (!x.whole) x.po = parts * x.rows * D;
  if (weights) x.scores = (size_t)B * H * x.slots;
  return x;
}

template <AttnType T, int D>
hipError_t run(const PagedAttnDesc& d, hipStream_t s) {
  const Plan x = plan_of(d.c.B, d.H, d.c.heads, D, d.c.W, d.c.page, d.weights != nullptr);
  DParams p{};
  p.view = {d.c.table, d.c.table_rs, d.c.lengths, d.c.pages, d.c.page, d.c.W * d.c.page, page_div(d.c.page)};
  p.k = (const uint8_t*)d.c.k; p.k_sp = 2 * d.c.k_sp; p.k_sh = 2 * d.c.k_sh; p.k_ss = 2 * d.c.k_ss;
  p.v = (const uint8_t*)d.c.v; p.v_sp = 2 * d.c.v_sp; p.v_sh = 2 * d.c.v_sh; p.v_ss = 2 * d.c.v_ss;
  p.q = (const uint8_t*)d.q; p.q_sb = 2 * d.q_sb; p.q_sh = 2 * d.q_sh;
  p.o = (uint8_t*)d.o; p.o_sb = 2 * d.o_sb; p.o_sh = 2 * d.o_sh;
  p.w = d.weights; p.w_sb = d.w_sb; p.w_sh = d.w_sh;
  p.decay = d.decay;
  float* ws = (float*)d.ws;
  p.ml = ws;
  p.po = ws + x.ml;
  p.scores = d.weights ? ws + x.ml + x.po : nullptr;
  p.slots = x.slots;
  p.B = d.c.B; p.H = d.H; p.heads = d.c.heads; p.group = d.H / d.c.heads;
  p.gtiles = x.gtiles; p.items = d.c.heads * x.gtiles; p.rows = x.rows; p.wgs = x.wgs; p.whole = x.whole;
  p.c = d.scale * 1.4426950408889634f;
  if (x.nt == 1) hipLaunchKernelGGL((decode_split<T, D, 1>), dim3(x.wgs), dim3(64 * kWaves), 0, s, p);
  else hipLaunchKernelGGL((decode_split<T, D, 2>), dim3(x.wgs), dim3(64 * kWaves), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (x.whole && !d.weights)) return e;
  const int64_t outs = x.whole ? 0 : (int64_t)p.B * p.H;
  const int64_t chunks = ((int64_t)d.c.W * d.c.page + 1023) / 1024;
  const int64_t jobs = outs + (d.weights ? (int64_t)p.B * p.heads * chunks : 0);
  hipLaunchKernelGGL((decode_join<T, D>), dim3((unsigned)std::min<int64_t>(jobs, 1 << 20)), dim3(256), 0, s, p, outs,
                     chunks, jobs);
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_workspace(int B, int H, int heads, int D, int W, int page, bool weights) {
  const Plan x = plan_of(B, H, heads, D, W, page, weights);
  return (x.ml + x.po + x.scores) * sizeof(float);
}

hipError_t launch_paged_attention(AttnType t, const PagedAttnDesc& d, hipStream_t s) {
  if (t == AttnType::BF16) {
    if (d.c.D == 128) return run<AttnType::BF16, 128>(d, s);
    if (d.c.D == 64) return run<AttnType::BF16, 64>(d, s);
  } else {
    if (d.c.D == 128) return run<AttnType::F16, 128>(d, s);
    if (d.c.D == 64) return run<AttnType::F16, 64>(d, s);
  }
  return hipErrorNotSupported;
}

}  // namespace grxk
