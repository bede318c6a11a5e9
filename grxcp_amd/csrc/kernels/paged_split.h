// What the attention of one new token over a paged cache has in common, whatever its
// pools hold: the shares of the workgroups, loads into LDS, and the join of the parts.
#ifndef GRXCP_PAGED_SPLIT_H
#define GRXCP_PAGED_SPLIT_H

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"

#include <algorithm>

namespace grxk {
namespace {

constexpr int kWaves = 4;
constexpr float kLowest = -__FLT_MAX__;
constexpr uint32_t kAbsent = 0x7fc0dead;  // a score of no slot (a NaN that no arithmetic gives)
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;

template <int N> struct Buf { static constexpr int value = N; };

// What a slot that is not there is read from: D values of zero.
__device__ __attribute__((aligned(256))) uint32_t zero_row[64];

// split2: two weights x, y >= 0 as a + b in the value type, which the product with V takes
// one after the other: a is cut off, b what that leaves. That keeps 16 bits (bf16) or 21
// (f16) of a weight; rounding it once, 8 or 11, costs o up to as much as its own rounding
// (and more where values cancel). b is not 0 where a is not, so that an infinite value
// times either is the same infinity. us, rounded once / so: groups of up to 16 heads as
// before (48 sequences of 33 to 4096 slots 76.1 / 76.0), 32 x 2 groups of 32 heads of 128,
// 4000 slots, 36.8 / 38.0, 8 groups of 128 heads, 8000 slots, 32.3 / 34.3.
template <AttnType T> struct PIo;
template <> struct PIo<AttnType::BF16> {
  // The weights' scale: exp2 of a score is at most 2^4 (kLazy) times this.
  static constexpr float kTop = 0.0f;
  __device__ static void split2(float x, float y, int& a, int& b) {
    const uint32_t ux = __float_as_uint(x), uy = __float_as_uint(y);
    a = (int)((uy & 0xffff0000u) | ux >> 16);
    b = (int)pack_bf16x2(fmaf(x, 1.0f + 0x1p-20f, -__uint_as_float(ux & 0xffff0000u)),
                         fmaf(y, 1.0f + 0x1p-20f, -__uint_as_float(uy & 0xffff0000u)));
  }
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
  __device__ static void split2(float x, float y, int& a, int& b) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x, y));
    const f16x2 rest = __builtin_bit_cast(f16x2, pack_f16x2(x - (float)h[0], y - (float)h[1]));
    const _Float16 least = 0x1p-24f;
    a = __builtin_bit_cast(int, h);
    b = __builtin_bit_cast(int, __builtin_elementwise_max(rest, __builtin_elementwise_min(h, f16x2{least, least})));
  }
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
  const uint8_t* k; uint32_t k_sp, k_sh, k_ss;   // strides of page, head, slot in 16-byte chunks
  const uint8_t* v; uint32_t v_sp, v_sh, v_ss;
  const uint8_t* q; int64_t q_sb, q_sh;
  uint8_t* o; int64_t o_sb, o_sh;
  float* w; int64_t w_sb, w_sh;
  float decay;
  float* ml;           // partial maxima and sums [parts, rows, 2]
  float* po;           // partial O [parts, rows, D]
  float* scores;       // [B, H, slots], or null: no weights asked for
  int64_t slots;
  int B, H, heads, group;
  int hw;              // key heads of a workgroup: 1, 2 or 4 waves' worth
  int shift;           // a unit is 2^shift slots: kTile for each of a head's waves
  int gtiles;          // tiles of 16 * NT query heads in a group
  int items;           // (hw key heads, tile) pairs of a sequence
  int rows;            // query heads of a tile
  int wgs;             // workgroups of decode_split
  int whole;           // one workgroup per item, nothing to join
  float c;             // scale * log2(e)
};

// ---- who does what -----------------------------------------------------------

__device__ __forceinline__ uint32_t units_of(const DParams& p, int len) {
  return max(1u, ((uint32_t)len + (1u << p.shift) - 1) >> p.shift);
}

__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readlane((int)wave_upto(v), 63);
}

// `total` units in `n` shares, none empty: the first `more` have `per` + 1 units, the
// others `per`.
struct Shares {
  uint32_t n, per, more;
  __device__ __forceinline__ uint32_t begin(uint32_t w) const { return w * per + min(w, more); }
  // the share that holds unit u
  __device__ __forceinline__ uint32_t of(uint32_t u) const {
    const uint32_t big = more * (per + 1);
    return u < big ? u / (per + 1) : more + (u - big) / per;
  }
};
__device__ __forceinline__ Shares shares(const DParams& p, uint32_t total) {
  Shares s;
  s.n = min((uint32_t)p.wgs, total);
  s.per = total / s.n;
  s.more = total - s.per * s.n;
  return s;
}

// The workgroup's share: sequence b, item `it` of it, from unit `i` on, `left` units. False:
// it has none. Lengths of the first 64 sequences stay in the lanes (len64); the others' are
// read again.
__device__ __forceinline__ bool find_share(const DParams& p, int lane, uint32_t& b, uint32_t& it, uint32_t& i,
                                           uint32_t& share, uint32_t& left, int& len64) {
  b = it = i = 0;
  share = blockIdx.x;
  len64 = lane < p.B ? clamp_length(p.view.lengths[lane], p.view.room) : 0;
  if (p.whole) {
    b = blockIdx.x / p.items;
    it = blockIdx.x - b * p.items;
    left = 1;
  } else {
    const uint32_t first64 = lane < p.B ? units_of(p, len64) : 0;
    uint32_t total = first64;
    for (int x = lane + 64; x < p.B; x += 64) total += units_of(p, clamp_length(p.view.lengths[x], p.view.room));
    const Shares sh = shares(p, wave_total(total) * p.items);
    if (blockIdx.x >= sh.n) return false;
    // Neighbouring shares go to one XCD (workgroups are dealt over the eight in turn).
    if (sh.n == p.wgs) share = (blockIdx.x & 7) * (p.wgs >> 3) + (blockIdx.x >> 3);
    const uint32_t u0 = sh.begin(share);
    left = sh.begin(share + 1) - u0;
    uint32_t base = 0;               // units of the sequences before this 64
    for (int b0 = 0;; b0 += 64) {
      const uint32_t mine = b0 == 0 ? first64
                            : b0 + lane < p.B ? units_of(p, clamp_length(p.view.lengths[b0 + lane], p.view.room)) : 0;
      const uint32_t upto = wave_upto(mine);
      const uint64_t past = __ballot((base + upto) * p.items > u0);
      if (past) {                    // u0 < total: some sequence ends past it
        const int at = __ffsll((unsigned long long)past) - 1;
        b = b0 + at;
        const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
        const uint32_t first = (base + (uint32_t)__builtin_amdgcn_readlane((int)upto, at) - n) * p.items;
        it = (u0 - first) / n;
        i = (u0 - first) - it * n;
        break;
      }
      base += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
  }
  b = __builtin_amdgcn_readfirstlane(b);
  it = __builtin_amdgcn_readfirstlane(it);
  i = __builtin_amdgcn_readfirstlane(i);
  left = __builtin_amdgcn_readfirstlane(left);
  return true;
}

// ---- loads and lanes -----------------------------------------------------------

__device__ __forceinline__ void wait_all() {
  __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_ptr_t)p; }
// 16 bytes per lane from memory straight into LDS (lane L writes lds + 16 L), as
// assembly so that the compiler does not make every LDS read wait for it: the
// tile loop waits itself, before the tile is used. M0 holds the LDS address and
// needs a wait state before the load that reads it.
template <bool ONCE> __device__ __forceinline__ void dma16(const uint8_t* src, uint32_t lds) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds), "v"(src) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}

// op over the four lanes that hold one query: l, l ^ 16, l ^ 32, l ^ 48.
template <class Op> __device__ __forceinline__ float over_query(float v, Op op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The results of a workgroup's waves, of which `of` share a key head, for 16 query heads:
// O rows [wave][16][D + 4] in mo, maxima and sums in ml. To o where `whole`, else to `part`.
template <AttnType T, int D>
__device__ __forceinline__ void meet(const DParams& p, int tid, int of, int hg, int q0, int row0, uint32_t b,
                                     int64_t part, bool whole, const float* mo, const float (*ml)[2][16]) {
  using IO = PIo<T>;
  constexpr int kPitch = D + 4;
  constexpr int E = D / 16;      // values of a thread, of 16 to a row
  const int r = tid >> 4, d0 = (tid & 15) * E;
  const int row = row0 + r;      // in the tile
  if (q0 + row >= p.group) return;
  for (int y = 0; y < p.hw; ++y) {
    float top = -INFINITY;
    for (int x = y * of; x < (y + 1) * of; ++x) top = fmaxf(top, ml[x][0][r]);
    float lsum = 0.0f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int x = y * of; x < (y + 1) * of; ++x) {
      const float f = __builtin_amdgcn_exp2f(ml[x][0][r] - fmaxf(top, kLowest));
      lsum = fmaf(f, ml[x][1][r], lsum);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(f, mo[(x * 16 + r) * kPitch + d0 + e], acc[e]);
    }
    const int64_t at = (part * p.hw + y) * p.rows + row;
    if (whole) {
      const float inv = top == -INFINITY ? 0.0f : 1.0f / lsum;   // no slot: 0; only -inf scores: 0 * inf
      uint32_t out[E / 2];
#pragma unroll
      for (int e = 0; e < E / 2; ++e) out[e] = IO::pack2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
      uint8_t* to = p.o + (int64_t)b * p.o_sb + ((hg * p.hw + y) * p.group + q0 + row) * p.o_sh + 2 * d0;
      if constexpr (E == 8) *(u32x4*)to = u32x4{out[0], out[1], out[2], out[3]};
      else *(u32x2*)to = u32x2{out[0], out[1]};
    } else {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *(f32x4*)(p.po + at * D + d0 + e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
    }
    if (d0 == 0 && (!whole || p.scores)) {
      p.ml[2 * at] = top;
      p.ml[2 * at + 1] = lsum;
    }
  }
}

// ---- the join ------------------------------------------------------------------

// Parts [first, first + count) of item `it` of sequence b.
struct Parts {
  int64_t first;
  int count;
};
__device__ __forceinline__ Parts parts_of(const DParams& p, const Shares& sh, uint32_t before, uint32_t n, int b,
                                          int it) {
  const int64_t item = (int64_t)b * p.items + it;
  if (p.whole) return {item, 1};
  const uint32_t u = before + it * n, w0 = sh.of(u), w1 = sh.of(u + n - 1);
  return {item + w0, (int)(w1 - w0) + 1};
}

// The parts of a query head's O from part `y0` on in steps of `by`, added up by lanes
// of V values each: acc, maximum and sum over them.
template <int V>
__device__ __forceinline__ void add_parts(const float* ml, const float* po, int64_t each, int D, int count, int y0,
                                          int by, float (&acc)[V], float& m, float& l) {
  typedef float vec __attribute__((ext_vector_type(V)));
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.0f;
  m = -INFINITY;
  l = 0.0f;
  for (int y = y0; y < count; y += 4 * by) {
    vec v[4];
    float pm[4], pl[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {            // all loads first
      const int64_t at = min(y + u * by, count - 1) * each;
      v[u] = *(const vec*)(po + at * D);
      pm[u] = ml[2 * at];
      pl[u] = ml[2 * at + 1];
    }
#pragma unroll
    for (int u = 1; u < 4; ++u)              // a part too far is one of no slot, in what it weighs too
      if (y + u * by >= count) {
        v[u] = vec(0.0f);
        pm[u] = -INFINITY;
        pl[u] = 0.0f;
      }
    const float top = fmaxf(fmaxf(m, fmaxf(pm[0], pm[1])), fmaxf(pm[2], pm[3]));
    const float from = fmaxf(top, kLowest);  // -inf - from is -inf
    const float f = __builtin_amdgcn_exp2f(m - from);
    m = top;
    l *= f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float w = __builtin_amdgcn_exp2f(pm[u] - from);
      l = fmaf(w, pl[u], l);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(w, ((const float*)&v[u])[e], acc[e]);
    }
  }
}

// For sequence blockIdx.y: workgroups below `outs` add up the parts of `apiece` query
// heads' O (4: a wave each, 1: the workgroup together), the others give 1024 slots of
// a key head their weights.
template <AttnType T, int D>
__global__ __launch_bounds__(256) void decode_join(DParams p, uint32_t outs, int apiece, uint32_t chunks) {
  using IO = PIo<T>;
  constexpr int LD = D / 4, NP = 256 / LD;   // lanes of a part, parts at a time
  __shared__ float red[NP][D], mred[NP], lred[NP];
  __shared__ float stat[1024][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const bool weights = blockIdx.x >= outs;
  int head = weights ? (blockIdx.x - outs) / chunks : blockIdx.x;
  if (!weights && apiece == 4) head = __builtin_amdgcn_readfirstlane(4 * head + (tid >> 6));
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int len = clamp_length(p.view.lengths[b], p.view.room);
    const uint32_t n = units_of(p, len);
    uint32_t before = 0, total = 0;          // units of all sequences, of those before b
    if (!p.whole) {
      for (int x = lane; x < p.B; x += 64) {
        const uint32_t m = units_of(p, clamp_length(p.view.lengths[x], p.view.room));
        total += m;
        before += x < b ? m : 0;
      }
      total = wave_total(total) * p.items;
      before = wave_total(before) * p.items;
    } else {
      total = 1;
    }
    const Shares sh = shares(p, total);
    if (!weights) {
      if (head >= p.H) continue;             // (a wave that has none)
      const int h = head / p.group, r = head - h * p.group;
      const int gt = r / p.rows, row = r - gt * p.rows, each = p.hw * p.rows;
      const Parts x = parts_of(p, sh, before, n, b, h / p.hw * p.gtiles + gt);
      if (x.count == 1) continue;            // decode_split had all of it
      const int64_t from = x.first * each + h % p.hw * p.rows + row;
      const float* ml = p.ml + from * 2;
      const float* po = p.po + from * D;
      uint8_t* out = p.o + (int64_t)b * p.o_sb + (int64_t)head * p.o_sh;
      float m, l;
      if (apiece == 4) {
        float acc[D / 64];
        add_parts<D / 64>(ml, po + lane * (D / 64), each, D, x.count, 0, 1, acc, m, l);
        const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
        const uint32_t w = IO::pack2(acc[0] * inv, acc[D / 64 - 1] * inv);
        if constexpr (D == 128) *(uint32_t*)(out + 4 * lane) = w;
        else *(uint16_t*)(out + 2 * lane) = (uint16_t)w;
        continue;
      }
      const int part = tid / LD, d = (tid % LD) * 4;
      float acc[4];
      add_parts<4>(ml, po + d, each, D, x.count, part, NP, acc, m, l);
      *(f32x4*)&red[part][d] = f32x4{acc[0], acc[1], acc[2], acc[3]};
      if (d == 0) {
        mred[part] = m;
        lred[part] = l;
      }
      __syncthreads();
      if (tid < D / 2) {
        float top = mred[0];
#pragma unroll
        for (int y = 1; y < NP; ++y) top = fmaxf(top, mred[y]);
        float a0 = 0.0f, a1 = 0.0f, sum = 0.0f;
#pragma unroll
        for (int y = 0; y < NP; ++y) {
          const float f = __builtin_amdgcn_exp2f(mred[y] - fmaxf(top, kLowest));
          a0 = fmaf(f, red[y][2 * tid], a0);
          a1 = fmaf(f, red[y][2 * tid + 1], a1);
          sum = fmaf(f, lred[y], sum);
        }
        const float inv = top == -INFINITY ? 0.0f : 1.0f / sum;
        *(uint32_t*)(out + 4 * tid) = IO::pack2(a0 * inv, a1 * inv);
      }
      __syncthreads();
      continue;
    }
    const int j0 = (int)((blockIdx.x - outs) % chunks) * 1024;
    if (j0 >= len) continue;
    // What the past steps gave the thread's four slots, and the first head's scores: they
    // come meanwhile.
    float* w = p.w + b * p.w_sb + head * p.w_sh;
    const float* sc = p.scores + ((int64_t)b * p.H + head * p.group) * p.slots;
    float old[4], a[4], s[4], next[4];
    int at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      at[u] = min(j0 + 256 * u + tid, len - 1);
      old[u] = p.decay == 0.0f ? 0.0f : w[at[u]];
      s[u] = sc[at[u]];
      a[u] = 0.0f;
    }
    // Sixteen lanes to a query head's parts.
    for (int r0 = 0; r0 < p.group; r0 += 16) {
      const int r = r0 + (tid >> 4);
      float m = -INFINITY, l = 0.0f;
      if (r < p.group) {
        const int gt = r / p.rows, row = r - gt * p.rows;
        const Parts x = parts_of(p, sh, before, n, b, head / p.hw * p.gtiles + gt);
        const float* ml = p.ml + (x.first * p.hw * p.rows + head % p.hw * p.rows + row) * 2;
        for (int y = tid & 15; y < x.count; y += 16) {
          const float* s = ml + (int64_t)y * p.hw * p.rows * 2;
          const float top = fmaxf(m, s[0]), from = fmaxf(top, kLowest);
          l = fmaf(__builtin_amdgcn_exp2f(s[0] - from), s[1], l * __builtin_amdgcn_exp2f(m - from));
          m = top;
        }
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        const float om = __shfl_xor(m, o), ol = __shfl_xor(l, o);
        const float top = fmaxf(m, om), from = fmaxf(top, kLowest);
        l = fmaf(__builtin_amdgcn_exp2f(om - from), ol, l * __builtin_amdgcn_exp2f(m - from));
        m = top;
      }
      if (r < p.group && (tid & 15) == 0) {
        stat[r][0] = m;
        stat[r][1] = __builtin_amdgcn_exp2f(IO::kTop) / l;   // the sum has the weights' scale
      }
    }
    __syncthreads();
#pragma unroll 2
    for (int r = 0; r < p.group; ++r) {
#pragma unroll
      for (int u = 0; u < 4; ++u) next[u] = sc[(int64_t)min(r + 1, p.group - 1) * p.slots + at[u]];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float x = __builtin_amdgcn_exp2f(s[u] - stat[r][0]) * stat[r][1];
        a[u] += __float_as_uint(s[u]) == kAbsent ? 0.0f : x;
        s[u] = next[u];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (j0 + 256 * u + tid < len) w[at[u]] = p.decay == 0.0f ? a[u] : fmaf(p.decay, old[u], a[u]);
    __syncthreads();
  }
}

// ---- plans ---------------------------------------------------------------------

// Heads of a slot lie next to each other ([pages, P, Hkv, D] memory), rather than the
// slots of a head.
bool neighbours(int64_t head_stride, int64_t slot_stride) { return head_stride < slot_stride; }

struct Plan {
  int nt, hw, gtiles, rows, wgs;
  bool whole;
  int64_t items, room, slots;
  size_t ml, po, scores;     // floats of the workspace, 16-byte multiples
};

int compute_units() {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  return std::max(8, cus / 8 * 8);
}

// Workgroups of the join, for every sequence: `outs` for the outputs, then one per chunk
// of 1024 slots of a key head's weights.
struct JoinPlan {
  int apiece;
  int64_t outs, chunks, jobs;
};
JoinPlan join_plan(const Plan& x, int B, int H, int heads, bool weights) {
  JoinPlan j{};
  // A wave to a query head, or the workgroup: few heads have many parts each. us, wave /
  // workgroup: 128 sequences of 800, 32 heads, 79.5 / 87.1; 16 of 8192 93.8 / 93.6; 2 of
  // 131072 97.7 / 89.7; one of 8000 22.6 / 15.0.
  j.apiece = (int64_t)B * H >= 512 ? 4 : 1;
  j.outs = x.whole ? 0 : ((int64_t)H + j.apiece - 1) / j.apiece;
  j.chunks = (x.room + 1023) / 1024;
  j.jobs = j.outs + (weights ? heads * j.chunks : 0);
  return j;
}

}  // namespace
}  // namespace grxk

#endif  // GRXCP_PAGED_SPLIT_H
