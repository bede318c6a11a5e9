// grxDNN attention of one new token per sequence over a paged key-value cache, on
// gfx950.
//
// New: the reference plans attention for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships no code.
//
// Every key and value is read once, for the whole group of query heads that share
// it (32 of them at a time), so the call is bound by reading the cache: 4 flops per
// query head and byte pair. What carries that:
//
//  * the cache of all sequences and key heads is one list of units, of a tile of 32
//    slots for each of the workgroup's four waves: 128 slots of one key head, 64 of
//    two or 32 of four (plan_of says when). The workgroups divide it evenly
//    (decode_split): whatever the sequences' lengths, every CU reads the same share.
//    The lengths are device data, so each workgroup finds its share by a scan of
//    them. A share that ends inside a sequence leaves a partial result (O without its
//    division, running maximum, sum) and decode_join adds those up, in the order of
//    the slots. Where no sequence is long a workgroup takes a whole one instead;
//  * each wave has a running maximum, sum and O of its own: no barrier until a
//    share's part of a sequence ends and a head's waves meet in LDS;
//  * scores are S^T = K Q^T (v_mfma_16x16x32), 16 query heads at a time, the K rows
//    in registers straight from memory. A group of fewer heads leaves columns
//    empty: the matrix cores have the time (24 MFMAs per 16 KB of cache);
//  * O^T += V^T P^T: the scores' lanes hold P^T as the B operand wants it if the
//    contraction runs over slots in the order 4g .. 4g+3, 16+4g .. 16+4g+3 (g: 16
//    lanes), and the V^T operand comes from the row-major V tile in LDS by the
//    transposing LDS read. V rows go to LDS without registers
//    (global_load_lds_dwordx4), chunks of 16 bytes XORed with the row so that a read
//    of 8 rows touches every bank once;
//  * the next tile's K and V are in flight while one is computed, and the page table
//    is read a tile further ahead: 16 KB per wave and tile, 8 waves per CU. Rows that
//    nothing reads again are loaded past the caches (6.8 TB/s for 6.1 in a loop that
//    only reads); those of a group of more than 32 heads are read once per 32;
//  * slots that are not there (past the length, or on a page that does not exist)
//    read a row of zeros in place of what their page holds, and their scores are
//    -inf, so nothing stale reaches a sum.
//
// us for 32 query and 8 key heads of 128, bf16, pages of 16 slots: 48 sequences of 33 to
// 4096 slots 76 (5.3 TB/s; 72 the split, 5 the join), 16 of 8192 93.6 (5.7), 2 of
// 131072 with 4 key heads 90 (6.0), 64 of 500 26.9 (4.9), one of 201 6.7, one of 60 5.3.
// The workgroups, as many as the CUs' registers hold (plan_of: two or three per CU), start
// together, and each waits for lengths, a table entry and its first tile in turn before the
// memory is busy; with the second launch that is what a call has above its bytes.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"

#include <algorithm>
#include <cstdio>

namespace grxk {
namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;                 // slots of a wave's tile
constexpr float kLowest = -__FLT_MAX__;
constexpr uint32_t kAbsent = 0x7fc0dead;  // a score of no slot (a NaN that no arithmetic gives)
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;

// Workgroups that share a CU: registers (D = 64 has half the accumulators) and LDS. us at
// D = 64, three / four (28 bytes of registers spilled, shares a quarter shorter): 24 x 16
// heads of 500 to 3001 slots with weights 42.3 / 50.8, 16 x 16 of 8192 94.6 / 103.4; with two
// tiles of query heads, two / three: 32 x 2 of 4000 23.1 / 26.4.
template <int D, int NT> constexpr int wgs_per_cu() { return D == 64 && NT == 1 ? 3 : 2; }

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
template <bool ONCE> __device__ __forceinline__ void dma16(const uint8_t* src, uint32_t lds) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds), "v"(src) : "memory");
  else
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

template <AttnType T, int D, int NT, bool ONCE>
__global__ __launch_bounds__(64 * kWaves, (wgs_per_cu<D, NT>())) void decode_split(DParams p) {
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
  uint32_t b = 0, it = 0, i = 0, share = blockIdx.x, left;
  // Lengths of the first 64 sequences stay in the lanes; the others' are read again.
  const int len64 = lane < p.B ? clamp_length(p.view.lengths[lane], p.view.room) : 0;
  if (p.whole) {
    b = blockIdx.x / p.items;
    it = blockIdx.x - b * p.items;
    left = 1;
  } else {
    const uint32_t first64 = lane < p.B ? units_of(p, len64) : 0;
    uint32_t total = first64;
    for (int x = lane + 64; x < p.B; x += 64) total += units_of(p, clamp_length(p.view.lengths[x], p.view.room));
    const Shares sh = shares(p, wave_total(total) * p.items);
    if (blockIdx.x >= sh.n) return;
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

  uint8_t* vt = smem + wave * 2 * kStage * 16;
  const int kk = lane & 31;
  const bool second = lane >= 32;    // this half of the wave finds the V rows
  const int of = kWaves / p.hw;      // waves of a key head
  const int hd = wave / of, sub = wave - hd * of;
  const uint32_t sp = second ? p.v_sp : p.k_sp, ss = second ? p.v_ss : p.k_ss;

  while (left > 0) {
    const int len = b < 64 ? __builtin_amdgcn_readlane(len64, b)
                           : __builtin_amdgcn_readfirstlane(clamp_length(p.view.lengths[b], p.view.room));
    const uint32_t n = units_of(p, len);
    if (p.whole) left = n;
    const uint32_t take = min(left, n - i);
    const int hg = (int)it / p.gtiles, q0 = ((int)it - hg * p.gtiles) * 16 * NT;   // first query head of the group
    const int h = hg * p.hw + hd;                                       // the wave's key head
    const int* table = p.view.table + (int64_t)b * p.view.table_rs;
    const uint8_t* base = second ? p.v + 16ull * h * p.v_sh : p.k + 16ull * h * p.k_sh;

    i32x4 qf[NT][F];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = q0 + 16 * t + l16;
      const uint8_t* src = r < p.group ? p.q + (int64_t)b * p.q_sb + (h * p.group + r) * p.q_sh : (const uint8_t*)zero_row;
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
    const int step = 1 << p.shift;
    int key = (int)(i << p.shift) + sub * kTile;                        // the wave's first slot
    const int end = (int)min((uint32_t)len, (i + take) << p.shift);
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
      rows[wave][second][kk] = (uint64_t)(
          page >= 0 ? base + 16 * ((uint64_t)(uint32_t)page * sp + (uint64_t)(uint32_t)row * ss) : (const uint8_t*)zero_row);
      live[BUF] = (uint32_t)__ballot(page >= 0);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const uint8_t* src = (const uint8_t*)rows[wave][0][16 * kt + l16] + 16 * g;
#pragma unroll
        for (int f = 0; f < F; ++f) {
          if constexpr (ONCE) kf[BUF][kt][f] = __builtin_nontemporal_load((const i32x4*)(src + 64 * f));
          else kf[BUF][kt][f] = *(const i32x4*)(src + 64 * f);
        }
      }
#pragma unroll
      for (int x = 0; x < kTile / RPI; ++x) {
        const int r = RPI * x + lane / CH;
        const uint8_t* src = (const uint8_t*)rows[wave][1][r] + 16 * ((lane % CH) ^ vswz<D>(r));
        dma16<ONCE>(src, lds_addr(vt + (BUF * kStage + 64 * x) * 16));
      }
    };
    auto compute = [&](auto buf, int key0) __attribute__((always_inline)) {
      constexpr int BUF = decltype(buf)::value;
      const uint32_t mask = live[BUF];
      if (!mask && !p.scores) return;            // nothing to add and nothing to say
      f32x4 scores[NT][2];                       // of all heads first: the keys' registers are free then
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          scores[t][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int f = 0; f < F; ++f) scores[t][kt] = IO::mma(kf[BUF][kt][f], qf[t][f], scores[t][kt]);
        }
      i32x4 pf[NT], pr[NT];                      // the weights: leading bits, rest
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 (&s)[2] = scores[t];
        s[0] *= p.c;
        s[1] *= p.c;
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
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          int a, b;
          IO::split2(w[x / 2][x % 2 * 2], w[x / 2][x % 2 * 2 + 1], a, b);
          pf[t][x] = a;
          pr[t][x] = b;
        }
      }
      if (!mask) return;
      const uint8_t* v0 = vt + BUF * kStage * 16;
      const int r0 = 4 * g + (l16 >> 2), r1 = r0 + 16;
      // Two tiles of the head dimension at a time: the products with the leading bits, then
      // those with the rest, which wait for them.
#pragma unroll
      for (int d0 = 0; d0 < DT; d0 += 2) {
        i32x4 vf[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int c = 2 * (d0 + x) + ((lane >> 1) & 1);
          const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4_t)(v0 + r0 * 2 * D + 16 * (c ^ vswz<D>(r0)) + 8 * (lane & 1)));
          const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4_t)(v0 + r1 * 2 * D + 16 * (c ^ vswz<D>(r1)) + 8 * (lane & 1)));
          const u32x2 w0 = __builtin_bit_cast(u32x2, a), w1 = __builtin_bit_cast(u32x2, b);
          vf[x] = i32x4{(int)w0.x, (int)w0.y, (int)w1.x, (int)w1.y};
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) o[t][d0 + x] = IO::mma(vf[x], pf[t], o[t][d0 + x]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) o[t][d0 + x] = IO::mma(vf[x], pr[t], o[t][d0 + x]);
      }
    };
    int e = entry(key);
    int next = entry(key + step);
    if (key < end) issue(Buf<0>{}, key, e);
    while (key < end) {
      wait_all();
      if (key + step < end) {
        issue(Buf<1>{}, key + step, next);
        next = entry(key + 2 * step);
      }
      compute(Buf<0>{}, key);
      key += step;
      if (key >= end) break;
      wait_all();
      if (key + step < end) {
        issue(Buf<0>{}, key + step, next);
        next = entry(key + 2 * step);
      }
      compute(Buf<1>{}, key);
      key += step;
    }

    // The results of a key head's waves meet: 16 query heads at a time.
    const bool whole = take == n;
    const int64_t part = p.whole ? share : (int64_t)b * p.items + it + share;
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
      constexpr int E = D / 16;      // values of a thread, of 16 to a row
      const int r = tid >> 4, d0 = (tid & 15) * E;
      const int row = 16 * t + r;    // in the tile
      if (q0 + row >= p.group) continue;
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
          for (int e = 0; e < E; e += 4) *(f32x4*)(p.po + at * D + d0 + e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
        }
        if (d0 == 0 && (!whole || p.scores)) {
          p.ml[2 * at] = top;
          p.ml[2 * at + 1] = lsum;
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
__device__ __forceinline__ Parts parts_of(const DParams& p, const Shares& sh, uint32_t before, uint32_t n, int b, int it) {
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

// ---- launch --------------------------------------------------------------------

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

Plan plan_of(int B, int H, int heads, int D, int W, int page, bool neighbours, bool weights) {
  Plan x{};
  const int group = H / heads;
  x.nt = group > 16 ? 2 : 1;
  x.gtiles = (group + 16 * x.nt - 1) / (16 * x.nt);
  x.rows = std::min(group, 16 * x.nt);
  // A workgroup per (sequence, head) and no join where no sequence is long: up to 256
  // slots always, up to 512 where there are workgroups enough to read as fast as the
  // memory gives (a CU alone reads about 46 GB/s). us, split and joined / whole: 32 x 8
  // heads of 300 slots 20.0 / 11.4, of 500 21.1 / 15.9, 16 x 8 of 500 14.6 / 14.2, but
  // 4 x 8 of 500 10.9 / 12.4, 8 x 8 of 1000 14.4 / 23.0, 64 x 8 of 20 to 1000 35.8 / 38.2.
  x.room = (int64_t)W * page;
  x.slots = (x.room + 127) / 128 * 128;
  const int64_t each = (int64_t)B * heads * x.gtiles;
  x.whole = (x.room <= 256 || (x.room <= 512 && each >= 128)) && each <= (1 << 20);
  // Where the heads of a slot lie together, a workgroup takes up to four of them (a
  // wave each), so that what it reads at a time does: 16 sequences of 8192, 8 heads of
  // 128, 103 us with one head, 93 with four (90 where the slots of a head lie
  // together). Not where that leaves few items, of many parts each: one sequence of
  // 8000, 15.9 us with one head, 21.7 with four.
  x.hw = 1;
  if (!x.whole && neighbours)
    for (int hw = 4; hw > 1 && x.hw == 1; hw /= 2)
      if (heads % hw == 0 && (int64_t)B * (heads / hw) * x.gtiles >= 64) x.hw = hw;
  x.items = (int64_t)B * (heads / x.hw) * x.gtiles;
  x.wgs = x.whole ? (int)x.items : (D == 64 && x.nt == 1 ? 3 : 2) * compute_units();
  const size_t parts = x.whole ? (size_t)x.items : (size_t)x.items + x.wgs;
  if (weights || !x.whole) x.ml = (parts * x.hw * x.rows * 2 + 3) / 4 * 4;
  if (!x.whole) x.po = parts * x.hw * x.rows * D;
  if (weights) x.scores = (size_t)B * H * x.slots;
  return x;
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

template <AttnType T, int D>
hipError_t run(const PagedAttnDesc& d, hipStream_t s) {
  const Plan x = plan_of(d.c.B, d.H, d.c.heads, D, d.c.W, d.c.page, neighbours(d.c.k_sh, d.c.k_ss),
                         d.weights != nullptr);
  DParams p{};
  p.view = {d.c.table, d.c.table_rs, d.c.lengths, d.c.pages, d.c.page, d.c.W * d.c.page, page_div(d.c.page)};
  p.k = (const uint8_t*)d.c.k; p.k_sp = d.c.k_sp / 8; p.k_sh = d.c.k_sh / 8; p.k_ss = d.c.k_ss / 8;
  p.v = (const uint8_t*)d.c.v; p.v_sp = d.c.v_sp / 8; p.v_sh = d.c.v_sh / 8; p.v_ss = d.c.v_ss / 8;
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
  p.hw = x.hw; p.shift = x.hw == 4 ? 5 : x.hw == 2 ? 6 : 7;
  p.gtiles = x.gtiles; p.items = d.c.heads / x.hw * x.gtiles; p.rows = x.rows; p.wgs = x.wgs; p.whole = x.whole;
  p.c = d.scale * 1.4426950408889634f;
  if (log_dnn_launches())
    std::fprintf(stderr, "grxdnn: paged attention %s b=%d h=%d hkv=%d d=%d page=%d room=%d weights=%d kernel=%s%d\n",
                 T == AttnType::BF16 ? "bf16" : "f16", p.B, p.H, p.heads, D, p.view.page, p.view.room,
                 (int)(d.weights != nullptr), x.whole ? "whole" : "split", x.hw);
  const dim3 grid(x.wgs), threads(64 * kWaves);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, threads, 0, s, p); };
  if (x.nt == 1) go(decode_split<T, D, 1, true>);
  else if (x.gtiles == 1) go(decode_split<T, D, 2, true>);
  else go(decode_split<T, D, 2, false>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (x.whole && !d.weights)) return e;
  const JoinPlan j = join_plan(x, p.B, p.H, p.heads, d.weights != nullptr);
  hipLaunchKernelGGL((decode_join<T, D>), dim3((unsigned)j.jobs, (unsigned)std::min(p.B, 65535)), dim3(256), 0, s, p,
                     (uint32_t)j.outs, j.apiece, (uint32_t)j.chunks);
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_workspace(const PagedCache& c, int H, bool weights) {
  const Plan x = plan_of(c.B, H, c.heads, c.D, c.W, c.page, neighbours(c.k_sh, c.k_ss), weights);
  return (x.ml + x.po + x.scores) * sizeof(float);
}

bool paged_attention_fits(const PagedCache& c, int H, bool weights) {
  const Plan x = plan_of(c.B, H, c.heads, c.D, c.W, c.page, neighbours(c.k_sh, c.k_ss), weights);
  return (double)x.items * (x.slots / 32) < 0x1p31 &&
         join_plan(x, c.B, H, c.heads, weights).jobs <= max_workgroups(256);
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
